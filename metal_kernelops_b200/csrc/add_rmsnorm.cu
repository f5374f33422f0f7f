// Residual RMSNorm with an optional int8 output, its backward pass, and the
// row quantiser that shares its last step.
//
// Per row of F features, in fp32:
//     s     = x + residual, rounded to the residual stream's type (s = x without one)
//     rstd  = 1 / sqrt(mean(s^2) + eps),   y = w s rstd
//     int8: scale = max|y| / 127,  q = rint(y / scale)
// The norm reads s as it is stored, so that the backward pass, and a layer run
// again from the stored stream, see the very values the forward saw.
// max|y| = rstd max|w s| and y / scale = 127 w s / max|w s|, so the sum of
// squares and the maximum come from one pass over the row and one reduction.
// The maximum is taken over the bit patterns of |w s| as unsigned integers: for
// non-negative floats their order is the values' order, with infinities and then
// NaN above every finite value, so a row that holds one is recognised; its scale
// is NaN and its q zero, and what reads it is NaN rather than silently finite.
// Rows whose largest |y| (before the factor rstd) is below 2^-100 count as zero.  A finite row
// whose squares do not fit fp32 is added up a second time, scaled down; |w s| has to fit.
// Backward, with xh = s rstd and c = mean(w dy xh):
//     d  = rstd (w dy - xh c) + dstream,   dx = dresidual = d,   dw = sum_rows dy xh
//
// Bytes bound these kernels: each row is read once and kept in registers.  A row
// belongs to a group of `tx` threads (whole warps; tx NV vectors of V elements
// cover the row), a CTA holds several rows when they are narrow.  V is 8, or 1
// where the width or an alignment does not allow 16-byte accesses.  The backward
// CTAs walk rows blockIdx, blockIdx + grid, ..., keep their columns' dw sums in
// registers and leave one partial row each; the fold adds the partials in a
// fixed order, so results are reproducible.  Rows wider than the registers of a
// CTA hold (16384 features forward, 8192 backward) stream: a CTA reads such a row
// twice, the second time from L1 / L2.
#include <atomic>
#include <climits>

#include "common.cuh"

namespace ssm {
namespace anorm {

constexpr int kMaxThreads = 512;
constexpr int kMaxWarps = kMaxThreads / 32;
constexpr float kTiny = 7.888609052210118e-31f;     // 2^-100

struct Args {
    int64_t rows, features, xs, rs;          // rs: residual row stride
    float eps, inv_f;
    int weight_dtype;
    const void* x; const void* res; const void* w;
    void* stream; void* y; int8_t* q; float* scale; float* rstd;
    const void* dy; const void* ds; void* dx; void* dres; float* part;
    int64_t dys, dss;
};

// V consecutive elements: 8 with vector accesses, or 1.
template <typename T, int V> struct Vec;
template <typename T> struct Vec<T, 1> {
    T r;
    __device__ __forceinline__ void ld(const T* p) { r = *p; }
    __device__ __forceinline__ void get(float* v) const { v[0] = ldf(&r); }
    __device__ __forceinline__ void set(const float* v) { stf(&r, v[0]); }
    __device__ __forceinline__ void st(T* p) const { *p = r; }
};
template <> struct Vec<float, 8> {
    float4 a, b;
    __device__ __forceinline__ void ld(const float* p) {
        a = reinterpret_cast<const float4*>(p)[0];
        b = reinterpret_cast<const float4*>(p)[1];
    }
    __device__ __forceinline__ void get(float* v) const {
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
    __device__ __forceinline__ void set(const float* v) {
        a = make_float4(v[0], v[1], v[2], v[3]);
        b = make_float4(v[4], v[5], v[6], v[7]);
    }
    __device__ __forceinline__ void st(float* p) const {
        reinterpret_cast<float4*>(p)[0] = a;
        reinterpret_cast<float4*>(p)[1] = b;
    }
};
template <typename T> struct Vec8h {
    uint4 r;
    __device__ __forceinline__ void ld(const T* p) { r = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void get(float* v) const {
        const T* h = reinterpret_cast<const T*>(&r);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = Io2<T>::ld(h + 2 * i);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
    __device__ __forceinline__ void set(const float* v) {
        T* h = reinterpret_cast<T*>(&r);
#pragma unroll
        for (int i = 0; i < 4; ++i) Io2<T>::st(h + 2 * i, make_float2(v[2 * i], v[2 * i + 1]));
    }
    __device__ __forceinline__ void st(T* p) const { *reinterpret_cast<uint4*>(p) = r; }
};
template <> struct Vec<__nv_bfloat16, 8> : Vec8h<__nv_bfloat16> {};
template <> struct Vec<__half, 8> : Vec8h<__half> {};

template <typename TS> __device__ __forceinline__ float as_stored(float v);
template <> __device__ __forceinline__ float as_stored<float>(float v) { return v; }
template <> __device__ __forceinline__ float as_stored<__nv_bfloat16>(float v) {
    return __bfloat162float(__float2bfloat16_rn(v));
}
template <> __device__ __forceinline__ float as_stored<__half>(float v) { return __half2float(__float2half_rn(v)); }

template <int V>
__device__ __forceinline__ void ld_weight(const Args& a, int64_t e, float* w) {
    if (a.weight_dtype == SSM_F32) {
        Vec<float, V> v; v.ld(static_cast<const float*>(a.w) + e); v.get(w);
    } else if (a.weight_dtype == SSM_BF16) {
        Vec<__nv_bfloat16, V> v; v.ld(static_cast<const __nv_bfloat16*>(a.w) + e); v.get(w);
    } else {
        Vec<__half, V> v; v.ld(static_cast<const __half*>(a.w) + e); v.get(w);
    }
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Sum and maximum over the `warps` warps that share a row; `red` holds them.
// Every thread of the CTA calls it the same number of times.
struct SumMax { float sum; uint32_t mx; };
__device__ __forceinline__ SumMax row_reduce(SumMax v, int warps, SumMax* red) {
    v.sum = sum_low_lanes<32>(v.sum);
    v.mx = __reduce_max_sync(0xffffffffu, v.mx);
    if (warps == 1) return v;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    SumMax* mine = red + threadIdx.y * warps;
    if (lane == 0) mine[warp] = v;
    __syncthreads();
    v = mine[0];
    for (int i = 1; i < warps; ++i) {
        v.sum += mine[i].sum;
        v.mx = v.mx > mine[i].mx ? v.mx : mine[i].mx;
    }
    return v;
}

// The int8 step.  q = rint(v / scale) = rint(127 v / max|v|): the quotient is formed
// from 127 v, which is exact for 16-bit data, and is correctly rounded, so that a v
// that lies exactly between two steps (16-bit data often do) is seen as such and goes
// to the even one.  A product with a rounded 127 / max misses those: 2e-5 of the
// values then differ from the definition in 64 bits, 7e-7 (fp16) so.
// The division: with y the rounded reciprocal of the divisor b, t = n y and
// t + (n - t b) y in fused steps is the rounded quotient (Markstein, IBM J. Res. Dev.
// 34, 1990).  n and b carry a factor of 1 / 128, so that 127 v cannot overflow.  It
// costs 3 % (65536 x 2560 bf16 to int8: 176 -> 182 us, HBM-bound).
struct Quant { float b, y, scale; };             // y = 0: the row's q are zeros; q * scale stands for v
__device__ __forceinline__ Quant quant_of(uint32_t mx) {
    const float m = __uint_as_float(mx);
    if (mx >= 0x7f800000u) return {0.0f, 0.0f, __uint_as_float(0x7fc00000u)};
    if (m < kTiny) return {0.0f, 0.0f, 0.0f};
    const float b = m * 0.0078125f;
    return {b, 1.0f / b, m / 127.0f};
}
// Two q in the low bytes: adding 1.5 * 2^23 leaves the rounded integer (to nearest,
// ties to even) in the low bits of the sum.
__device__ __forceinline__ float2 q_bits(float2 v, const Quant& s) {
    const float2 n = mul2(v, f2(0.9921875f)), t = mul2(n, f2(s.y));
    return add2(fma2(fma2(t, f2(-s.b), n), f2(s.y), t), f2(12582912.0f));
}
// A row that is not finite has y = 0 and must store zeros, also where v is
// infinite or NaN.
__device__ __forceinline__ uint32_t pack4(const float* v, const Quant& s) {
    const float2 a = q_bits(make_float2(v[0], v[1]), s), b = q_bits(make_float2(v[2], v[3]), s);
    const uint32_t lo = __byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040);
    const uint32_t hi = __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040);
    return s.y != 0.0f ? __byte_perm(lo, hi, 0x5410) : 0u;
}

// V int8 values of a row at q.
template <int V>
__device__ __forceinline__ void st_q(int8_t* q, const float* v, const Quant& s) {
    if constexpr (V == 8) *reinterpret_cast<uint2*>(q) = make_uint2(pack4(v, s), pack4(v + 4, s));
    else *q = s.y != 0.0f ? (int8_t)(__float_as_uint(q_bits(f2(v[0]), s).x) & 0xffu) : (int8_t)0;
}

// x (+ residual) -> s, and s stored; the V values of s.
template <typename T, typename TS, int V>
__device__ __forceinline__ void sum_store(const Args& a, int64_t row, int64_t e, const Vec<T, V>& xr,
                                          const Vec<TS, V>& rr, float* v) {
    xr.get(v);
    if (a.res != nullptr) {
        float r[V];
        rr.get(r);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = v[i] + r[i];
        Vec<TS, V> s;
        s.set(v);
        s.get(v);
        s.st(static_cast<TS*>(a.stream) + row * a.features + e);
    }
}

// rstd of a row whose sum of squares left fp32's range (an |s| above 1.8e19 does that): every
// warp of the row adds the squares of 2^-84 s, from s as it is stored.  What overflowed adds up
// to at least 2^-40 then, and 2^31 of the largest squares to 2^119.  A row that holds an infinity
// gets 0, as 1 / sqrt(infinity) is.  Called behind the reduction's barrier, so the other
// warps' stores are seen; a row of a single warp has to order its lanes' itself.
template <typename T, typename TS>
__device__ __forceinline__ float rstd_of_large(const Args& a, int64_t row) {
    constexpr float kDown = 5.169878828456423e-26f;     // 2^-84
    __syncwarp();
    const T* x = static_cast<const T*>(a.x) + row * a.xs;
    const TS* s = static_cast<const TS*>(a.stream) + row * a.features;
    float sum = 0.0f;
#pragma unroll 1
    for (int64_t e = threadIdx.x & 31; e < a.features; e += 32) {
        const float v = (a.res != nullptr ? ldf(s + e) : ldf(x + e)) * kDown;
        sum = fmaf(v, v, sum);
    }
    return kDown / sqrtf(fmaf(sum_low_lanes<32>(sum), a.inv_f, a.eps * kDown * kDown));
}
template <typename T, typename TS>
__device__ __forceinline__ float rstd_of(const Args& a, int64_t row, float sum) {
    if (sum == __int_as_float(0x7f800000)) return rstd_of_large<T, TS>(a, row);
    return 1.0f / sqrtf(fmaf(sum, a.inv_f, a.eps));
}

enum Mode { kNorm, kNormInt8, kInt8 };    // y, q and scale, q and scale of x itself

template <typename T, typename TS, int V, int NV, int MODE>
__global__ void __launch_bounds__(kMaxThreads)
fwd_kernel(const Args a) {
    __shared__ SumMax red[kMaxWarps];
    const int64_t F = a.features;
    const int tx = blockDim.x, warps = tx >> 5;
    const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    const bool live = row < a.rows;
    float v[NV][V];
    Vec<T, V> xr[NV];
    Vec<TS, V> rr[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int64_t e = ((int64_t)k * tx + threadIdx.x) * V;
        if (live && e < F) {
            xr[k].ld(static_cast<const T*>(a.x) + row * a.xs + e);
            if (MODE != kInt8 && a.res != nullptr) rr[k].ld(static_cast<const TS*>(a.res) + row * a.rs + e);
        }
    }
    SumMax sm{0.0f, 0u};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int64_t e = ((int64_t)k * tx + threadIdx.x) * V;
        if (live && e < F) {
            if (MODE == kInt8) {
                xr[k].get(v[k]);
            } else {
                float w[V];
                ld_weight<V>(a, e, w);
                sum_store<T, TS, V>(a, row, e, xr[k], rr[k], v[k]);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    sm.sum = fmaf(v[k][i], v[k][i], sm.sum);
                    v[k][i] *= w[i];
                }
            }
            if (MODE != kNorm) {
#pragma unroll
                for (int i = 0; i < V; ++i) sm.mx = max(sm.mx, abs_bits(v[k][i]));
            }
        }
    }
    sm = row_reduce(sm, warps, red);
    if (!live) return;
    const float r = MODE == kInt8 ? 1.0f : rstd_of<T, TS>(a, row, sm.sum);
    if (MODE == kNorm) {
        if (a.rstd != nullptr && threadIdx.x == 0) a.rstd[row] = r;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int64_t e = ((int64_t)k * tx + threadIdx.x) * V;
            if (e < F) {
#pragma unroll
                for (int i = 0; i < V; ++i) v[k][i] *= r;
                Vec<T, V> o;
                o.set(v[k]);
                o.st(static_cast<T*>(a.y) + row * F + e);
            }
        }
    } else {
        const Quant qt = quant_of(sm.mx);
        if (threadIdx.x == 0) a.scale[row] = qt.scale * r;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int64_t e = ((int64_t)k * tx + threadIdx.x) * V;
            if (e < F)
                st_q<V>(a.q + row * F + e, v[k], qt);
        }
    }
}

// One row per CTA, element by element, in two passes over the row.
template <typename T, typename TS, int MODE>
__global__ void __launch_bounds__(kMaxThreads)
fwd_stream_kernel(const Args a) {
    __shared__ SumMax red[kMaxWarps];
    const int64_t F = a.features, row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.xs;
    const TS* res = a.res != nullptr ? static_cast<const TS*>(a.res) + row * a.rs : nullptr;
    TS* stream = static_cast<TS*>(a.stream) + (res ? row * F : 0);
    auto value = [&](int64_t e) {
        float v = ldf(x + e);
        return res ? as_stored<TS>(v + ldf(res + e)) : v;
    };
    SumMax sm{0.0f, 0u};
    for (int64_t e = threadIdx.x; e < F; e += blockDim.x) {
        float v = MODE == kInt8 ? ldf(x + e) : value(e);
        if (MODE != kInt8) {
            if (res) stf(stream + e, v);
            sm.sum = fmaf(v, v, sm.sum);
            v *= ld_any(a.w, e, a.weight_dtype);
        }
        if (MODE != kNorm) sm.mx = max(sm.mx, abs_bits(v));
    }
    sm = row_reduce(sm, blockDim.x >> 5, red);
    const float r = MODE == kInt8 ? 1.0f : rstd_of<T, TS>(a, row, sm.sum);
    const Quant qt = quant_of(sm.mx);
    if (threadIdx.x == 0) {
        if (MODE != kNorm) a.scale[row] = qt.scale * r;
        else if (a.rstd != nullptr) a.rstd[row] = r;
    }
    for (int64_t e = threadIdx.x; e < F; e += blockDim.x) {
        float v = MODE == kInt8 ? ldf(x + e) : value(e);
        if (MODE != kInt8) v *= ld_any(a.w, e, a.weight_dtype);
        if (MODE == kNorm) stf(static_cast<T*>(a.y) + row * F + e, v * r);
        else st_q<1>(a.q + row * F + e, &v, qt);
    }
}

template <typename T, typename TS, int V, int NV>
__global__ void __launch_bounds__(kMaxThreads)
bwd_kernel(const Args a) {
    __shared__ SumMax red[2][kMaxWarps];
    const int64_t F = a.features;
    const int tx = blockDim.x, warps = tx >> 5;
    const TS* s = static_cast<const TS*>(a.stream);
    const T* dy = static_cast<const T*>(a.dy);
    const TS* ds = static_cast<const TS*>(a.ds);
    float dw[NV][V] = {};
    float w[NV][V] = {};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int64_t e = ((int64_t)k * tx + threadIdx.x) * V;
        if (e < F) ld_weight<V>(a, e, w[k]);
    }
    const int64_t step = (int64_t)gridDim.x * blockDim.y;
    int turn = 0;
    for (int64_t r0 = (int64_t)blockIdx.x * blockDim.y; r0 < a.rows; r0 += step, turn ^= 1) {
        const int64_t row = r0 + threadIdx.y;
        const bool live = row < a.rows;
        Vec<TS, V> sr[NV], dsr[NV];
        Vec<T, V> dyr[NV];
        float rstd = 0.0f;
        if (live) {
            rstd = a.rstd[row];
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int64_t e = ((int64_t)k * tx + threadIdx.x) * V;
                if (e < F) {
                    sr[k].ld(s + row * a.xs + e);
                    dyr[k].ld(dy + row * a.dys + e);
                    if (ds) dsr[k].ld(ds + row * a.dss + e);
                }
            }
        }
        SumMax c{0.0f, 0u};
        float xh[NV][V], g[NV][V];
        if (live) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int64_t e = ((int64_t)k * tx + threadIdx.x) * V;
                if (e < F) {
                    sr[k].get(xh[k]);
                    dyr[k].get(g[k]);
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        xh[k][i] *= rstd;
                        dw[k][i] = fmaf(g[k][i], xh[k][i], dw[k][i]);
                        g[k][i] *= w[k][i];
                        c.sum = fmaf(g[k][i], xh[k][i], c.sum);
                    }
                }
            }
        }
        const float c1 = row_reduce(c, warps, red[turn]).sum * a.inv_f;
        if (live) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int64_t e = ((int64_t)k * tx + threadIdx.x) * V;
                if (e < F) {
                    float d[V];
                    if (ds) dsr[k].get(d);
#pragma unroll
                    for (int i = 0; i < V; ++i) d[i] = fmaf(rstd, fmaf(-xh[k][i], c1, g[k][i]), ds ? d[i] : 0.0f);
                    Vec<T, V> o;
                    o.set(d);
                    o.st(static_cast<T*>(a.dx) + row * F + e);
                    if (a.dres) {
                        Vec<TS, V> p;
                        p.set(d);
                        p.st(static_cast<TS*>(a.dres) + row * F + e);
                    }
                }
            }
        }
    }
    if (a.part == nullptr) return;
    float* part = a.part + ((int64_t)blockIdx.x * blockDim.y + threadIdx.y) * F;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int64_t e = ((int64_t)k * tx + threadIdx.x) * V;
        if (e < F) {
            Vec<float, V> o;
            o.set(dw[k]);
            o.st(part + e);
        }
    }
}

// Element by element; the CTA's dw partial lives in its own row of `part`.
template <typename T, typename TS>
__global__ void __launch_bounds__(kMaxThreads)
bwd_stream_kernel(const Args a) {
    __shared__ SumMax red[2][kMaxWarps];
    const int64_t F = a.features;
    float* part = a.part + blockIdx.x * F;
    for (int64_t e = threadIdx.x; e < F; e += blockDim.x) part[e] = 0.0f;
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
        const TS* s = static_cast<const TS*>(a.stream) + row * a.xs;
        const T* dy = static_cast<const T*>(a.dy) + row * a.dys;
        const TS* ds = a.ds ? static_cast<const TS*>(a.ds) + row * a.dss : nullptr;
        const float rstd = a.rstd[row];
        SumMax c{0.0f, 0u};
        for (int64_t e = threadIdx.x; e < F; e += blockDim.x) {
            const float xh = ldf(s + e) * rstd, up = ldf(dy + e);
            part[e] = fmaf(up, xh, part[e]);
            c.sum = fmaf(up * ld_any(a.w, e, a.weight_dtype), xh, c.sum);
        }
        const float c1 = row_reduce(c, blockDim.x >> 5, red[turn]).sum * a.inv_f;
        for (int64_t e = threadIdx.x; e < F; e += blockDim.x) {
            const float xh = ldf(s + e) * rstd, g = ldf(dy + e) * ld_any(a.w, e, a.weight_dtype);
            const float d = fmaf(rstd, fmaf(-xh, c1, g), ds ? ldf(ds + e) : 0.0f);
            stf(static_cast<T*>(a.dx) + row * F + e, d);
            if (a.dres) stf(static_cast<TS*>(a.dres) + row * F + e, d);
        }
    }
}

// dw[f] = the partial rows added in order: 32 columns a CTA, 32 runs of consecutive
// partial rows each summed by one warp, the runs added in order.
constexpr int kRuns = 32;
__global__ void __launch_bounds__(kRuns * 32) fold_kernel(const float* part, int64_t parts, int64_t F, float* dw) {
    __shared__ float run[kRuns][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t f = (int64_t)blockIdx.x * 32 + lane;
    const int64_t per = (parts + kRuns - 1) / kRuns, k0 = warp * per, k1 = min64(k0 + per, parts);
    float s = 0.0f;
    if (f < F) {
#pragma unroll 8
        for (int64_t k = k0; k < k1; ++k) s += part[k * F + f];
    }
    run[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && f < F) {
        s = run[0][lane];
#pragma unroll
        for (int i = 1; i < kRuns; ++i) s += run[i][lane];
        dw[f] = s;
    }
}

// ------------------------------------------------------------------- host ----
static bool al(const void* p, int64_t b) { return (reinterpret_cast<uintptr_t>(p) % b) == 0; }
static int64_t esize(int dtype) { return dtype == SSM_F32 ? 4 : 2; }

// v elements a vector (8, or 1 where width or alignment does not allow 8), nv
// vectors a thread, tx threads a row, ty rows a CTA; nv = 0: the streaming
// kernels.  The forward gives a thread four vectors where the row has them: with
// 65536 x 2560 bf16 to int8 (with the plain product for q), 177 us against 189 with
// two and 219 with one: fewer warps meet at the reduction, each with more loads on
// the way.  The backward,
// which keeps three tensors' vectors, weights and sums, takes two (65536 x 2560: 425
// us, 499 with one; four would spill), and one in rows of up to 1024, whose CTAs are
// small enough as they are.
struct Shape { int tx, ty, v, nv; };

static Shape shape_of(int64_t F, bool vec, bool bwd) {
    const int v = vec ? 8 : 1;
    const int64_t n = ceil_div(F, v);
    int nv = 0;
    if (vec && bwd) nv = n <= 128 ? 1 : n <= 2 * kMaxThreads ? 2 : 0;
    else if (vec) nv = n <= 32 ? 1 : n <= 64 ? 2 : n <= 4 * kMaxThreads ? 4 : 0;
    else nv = n <= 8 * kMaxThreads ? 8 : n <= 16 * kMaxThreads ? 16 : 0;
    if (nv == 0) return {kMaxThreads, 1, 1, 0};
    const int tx = (int)(ceil_div(ceil_div(n, nv), 32) * 32);
    return {tx, tx >= 128 ? 1 : 128 / tx, v, nv};
}

static int validate(const ssm_add_rmsnorm_params* p, const char* op) {
    if (p == nullptr) return fail(SSM_ERR_INVALID, std::string(op) + ": null params");
    if (p->rows < 0 || p->features < 1) return fail(SSM_ERR_INVALID, std::string(op) + ": rows and features");
    if (p->rows > INT32_MAX || p->features > INT32_MAX)
        return fail(SSM_ERR_UNSUPPORTED, std::string(op) + ": more than 2^31 - 1 rows or features");
    if (p->dtype < SSM_F32 || p->dtype > SSM_F16 || p->weight_dtype < SSM_F32 || p->weight_dtype > SSM_F16)
        return fail(SSM_ERR_UNSUPPORTED, std::string(op) + ": dtype");
    if (p->stream_dtype != p->dtype && p->stream_dtype != SSM_F32)
        return fail(SSM_ERR_UNSUPPORTED, std::string(op) + ": the residual stream has x's dtype or float32");
    for (int64_t st : {p->x_row_stride, p->residual_row_stride, p->dy_row_stride, p->dstream_row_stride})
        if (st && st < p->features) return fail(SSM_ERR_INVALID, std::string(op) + ": a row stride is below features");
    return SSM_OK;
}

static Args args_of(const ssm_add_rmsnorm_params* p) {
    Args a{};
    a.rows = p->rows; a.features = p->features;
    a.xs = p->x_row_stride ? p->x_row_stride : p->features;
    a.rs = p->residual_row_stride ? p->residual_row_stride : p->features;
    a.dys = p->dy_row_stride ? p->dy_row_stride : p->features;
    a.dss = p->dstream_row_stride ? p->dstream_row_stride : p->features;
    a.eps = p->eps;
    a.inv_f = 1.0f / (float)p->features;
    a.weight_dtype = p->weight_dtype;
    a.x = p->x; a.res = p->residual; a.w = p->weight;
    a.stream = p->stream; a.y = p->y; a.q = p->q; a.scale = p->scale; a.rstd = p->rstd;
    a.dy = p->dy; a.ds = p->dstream; a.dx = p->dx; a.dres = p->dresidual;
    return a;
}

template <typename T, typename TS, int MODE>
static int launch_fwd(const Args& a, const Shape& s, cudaStream_t st) {
    const dim3 block(s.tx, s.ty);
    const unsigned grid = (unsigned)ceil_div(a.rows, s.ty);
    switch (s.nv) {
        case 0: fwd_stream_kernel<T, TS, MODE><<<grid, block, 0, st>>>(a); break;
        case 1: fwd_kernel<T, TS, 8, 1, MODE><<<grid, block, 0, st>>>(a); break;
        case 2: fwd_kernel<T, TS, 8, 2, MODE><<<grid, block, 0, st>>>(a); break;
        case 4: fwd_kernel<T, TS, 8, 4, MODE><<<grid, block, 0, st>>>(a); break;
        case 8: fwd_kernel<T, TS, 1, 8, MODE><<<grid, block, 0, st>>>(a); break;
        default: fwd_kernel<T, TS, 1, 16, MODE><<<grid, block, 0, st>>>(a);
    }
    return check_launch(MODE == kInt8 ? "quantize_int8" : "add_rmsnorm fwd");
}

template <int MODE>
static int dispatch_fwd(const Args& a, const Shape& s, int dtype, int stream_dtype, cudaStream_t st) {
    if (dtype == SSM_F32) return launch_fwd<float, float, MODE>(a, s, st);
    if (dtype == SSM_BF16) {
        if (MODE == kInt8 || stream_dtype == SSM_BF16) return launch_fwd<__nv_bfloat16, __nv_bfloat16, MODE>(a, s, st);
        return launch_fwd<__nv_bfloat16, float, MODE>(a, s, st);
    }
    if (MODE == kInt8 || stream_dtype == SSM_F16) return launch_fwd<__half, __half, MODE>(a, s, st);
    return launch_fwd<__half, float, MODE>(a, s, st);
}

// Whether every tensor the forward touches allows 8-element vectors.
static bool vec_fwd(const ssm_add_rmsnorm_params* p, const Args& a, bool quant_only) {
    const int64_t e = esize(p->dtype), es = esize(p->stream_dtype);
    if (a.features % 8 || !al(a.x, 16) || (a.xs * e) % 16 || !al(a.q, 8) || !al(a.y, 16)) return false;
    if (quant_only) return true;
    if (!al(a.w, 16)) return false;
    return !a.res || (al(a.res, 16) && (a.rs * es) % 16 == 0 && al(a.stream, 16));
}

// The most CTAs the backward runs (each leaves ty partial rows): 1024 threads an SM.
static int64_t most_ctas(int64_t rows, const Shape& s) {
    return min64(ceil_div(max64(rows, 1), s.ty), 148 * max64(1, 1024 / (s.tx * s.ty)));
}
// As many of them as the GPU holds at once.
template <auto kernel>
static int64_t launch_rows(Args& a, const Shape& s, cudaStream_t st) {
    static std::atomic<int> room[kMaxThreads / 32 + 1];   // CTAs per SM by warps; 0: not asked yet
    std::atomic<int>& n = room[s.tx * s.ty / 32];
    if (n == 0) {
        int k = 0;
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&k, kernel, s.tx * s.ty, 0) != cudaSuccess || k < 1) {
            cudaGetLastError();
            k = 1;
        }
        n = k;
    }
    const int64_t ctas = min64(most_ctas(a.rows, s), 148 * n);
    kernel<<<(unsigned)ctas, dim3(s.tx, s.ty), 0, st>>>(a);
    return ctas;
}

// Returns the CTAs launched.
template <typename T, typename TS>
static int64_t launch_bwd(Args& a, const Shape& s, cudaStream_t st) {
    switch (s.nv) {
        case 0: return launch_rows<bwd_stream_kernel<T, TS>>(a, s, st);
        case 1: return launch_rows<bwd_kernel<T, TS, 8, 1>>(a, s, st);
        case 2: return launch_rows<bwd_kernel<T, TS, 8, 2>>(a, s, st);
        case 8: return launch_rows<bwd_kernel<T, TS, 1, 8>>(a, s, st);
        default: return launch_rows<bwd_kernel<T, TS, 1, 16>>(a, s, st);
    }
}

}  // namespace anorm
}  // namespace ssm

using namespace ssm;
using namespace ssm::anorm;

extern "C" int ssm_add_rmsnorm_sizes(const ssm_add_rmsnorm_params* p, size_t* workspace_bytes) {
    if (int s = validate(p, "add_rmsnorm")) return s;
    // the partial rows of either form (the pointers' alignment picks one): a CTA leaves one per row group
    int64_t parts = 0;
    for (bool vec : {false, true}) {
        const Shape sh = shape_of(p->features, vec && p->features % 8 == 0, true);
        parts = max64(parts, most_ctas(p->rows, sh) * sh.ty);
    }
    if (workspace_bytes) *workspace_bytes = (size_t)(parts * p->features) * 4;
    return SSM_OK;
}

extern "C" int ssm_add_rmsnorm_fwd(const ssm_add_rmsnorm_params* p, void* stream) {
    if (int s = validate(p, "add_rmsnorm")) return s;
    if (p->rows == 0) return SSM_OK;
    if (!p->x || !p->weight || (p->residual && !p->stream) || !(p->y || (p->q && p->scale)))
        return fail(SSM_ERR_INVALID, "add_rmsnorm fwd: null pointer");
    if (p->y && p->q) return fail(SSM_ERR_INVALID, "add_rmsnorm fwd: y and q are alternatives");
    const Args a = args_of(p);
    const Shape sh = shape_of(a.features, vec_fwd(p, a, false), false);
    const int sd = p->residual ? p->stream_dtype : p->dtype;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return p->q ? dispatch_fwd<kNormInt8>(a, sh, p->dtype, sd, st) : dispatch_fwd<kNorm>(a, sh, p->dtype, sd, st);
}

extern "C" int ssm_quantize_int8(const ssm_add_rmsnorm_params* p, void* stream) {
    if (int s = validate(p, "quantize_int8")) return s;
    if (p->rows == 0) return SSM_OK;
    if (!p->x || !p->q || !p->scale) return fail(SSM_ERR_INVALID, "quantize_int8: null pointer");
    const Args a = args_of(p);
    return dispatch_fwd<kInt8>(a, shape_of(a.features, vec_fwd(p, a, true), false), p->dtype, p->dtype,
                               static_cast<cudaStream_t>(stream));
}

extern "C" int ssm_add_rmsnorm_bwd(const ssm_add_rmsnorm_params* p, void* stream) {
    if (int s = validate(p, "add_rmsnorm")) return s;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (p->rows == 0) {
        if (p->dweight && cudaMemsetAsync(p->dweight, 0, (size_t)p->features * 4, st))
            return check_launch("add_rmsnorm bwd: zero dweight");
        return SSM_OK;
    }
    if (!p->stream || !p->weight || !p->dy || !p->rstd || !p->dx)
        return fail(SSM_ERR_INVALID, "add_rmsnorm bwd: null pointer");
    size_t need = 0;
    ssm_add_rmsnorm_sizes(p, &need);
    if (!p->workspace || p->workspace_bytes < need)
        return fail(SSM_ERR_WORKSPACE, "add_rmsnorm bwd: workspace smaller than ssm_add_rmsnorm_sizes");
    Args a = args_of(p);
    a.part = static_cast<float*>(p->workspace);
    const int64_t e = esize(p->dtype), es = esize(p->stream_dtype);
    // x_row_stride is the saved stream's here
    const bool vec = a.features % 8 == 0 && al(a.stream, 16) && (a.xs * es) % 16 == 0 && al(a.w, 16) &&
                     al(a.dy, 16) && (a.dys * e) % 16 == 0 && al(a.dx, 16) && al(a.part, 16) &&
                     (!a.ds || (al(a.ds, 16) && (a.dss * es) % 16 == 0)) && (!a.dres || al(a.dres, 16));
    const Shape sh = shape_of(a.features, vec, true);
    int64_t ctas;
    if (p->dtype == SSM_F32) ctas = launch_bwd<float, float>(a, sh, st);
    else if (p->dtype == SSM_BF16 && p->stream_dtype == SSM_BF16) ctas = launch_bwd<__nv_bfloat16, __nv_bfloat16>(a, sh, st);
    else if (p->dtype == SSM_BF16) ctas = launch_bwd<__nv_bfloat16, float>(a, sh, st);
    else if (p->stream_dtype == SSM_F16) ctas = launch_bwd<__half, __half>(a, sh, st);
    else ctas = launch_bwd<__half, float>(a, sh, st);
    if (int s = check_launch("add_rmsnorm bwd")) return s;
    if (p->dweight) {
        fold_kernel<<<(unsigned)ceil_div(a.features, 32), kRuns * 32, 0, st>>>(a.part, ctas * sh.ty, a.features, p->dweight);
        return check_launch("add_rmsnorm bwd: fold");
    }
    return SSM_OK;
}
