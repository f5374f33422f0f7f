// Gated linear recurrence for sm_100a: a diagonal recurrence with one state per
// channel whose forget gate comes with every token; forward over sequences, its
// backward pass, and the single-token step.
//
// Per batch row and channel, with span = 1 - lower (the channel's lower bound of
// the forget gate), all in fp32:
//     k_t = sigmoid(-forget_t),   g_t = span k_t
//     h'_t = 0 where reset_t, else h_{t-1}
//     h_t = a_t h'_t + g_t x_t,  a_t = 1 - g_t
//     y_t = h_t silu(z_t)                    (h_t without z)
// k_t is 1 / (1 + e^forget): the complement of the gate is computed as such, so that g of
// gates near one (long memory) keeps its digits.  e^forget is two to a rounded product, so g and
// k err by up to (1.25 |forget| + 10) 2^-24 of themselves.  a = 1 - g is rounded to
// 2^-25; what the products of a row lack by that is carried along (settle()), which costs a
// fused addition a step (2 % of the backward).  Without it a steady forget of 8 with a lower
// bound of 0.9 ended 1e-3 off after 65536 steps, with it 5e-6.
// Backward, with dh_t the gradient of h_t and a_t taken as 0 at a reset:
//     dh_t = dy_t silu(z_t) + a_{t+1} dh_{t+1}   (+ dfinal at the last step)
//     dx = g dh,  dg = dh (x - h'),  dforget = -dg g (1 - k),  dlower = -sum dg k,  1 - k = k e^forget
//     dz = dy h silu'(z),  dinitial = a_0 dh_0
//
// Both directions are scans of affine maps: a run of steps takes the state S to
// A S + H, with A the product of the a_t, and the gradient D that enters it from
// the later steps to A D + R.  A warp owns N consecutive steps of a tile of
// channels (a lane: one 4-byte word, two 16-bit channels or one fp32 channel),
// holds them in registers, and reduces them to (A, H); the warps' maps meet in
// shared memory, each warp composes those before it and walks its steps a second
// time from the right start.  A CTA's kWarps warps make a chunk.  Where the channel
// tiles of all batch rows do not fill the GPU, a cluster of CTAs takes consecutive
// chunks of one tile at a time, and its CTAs exchange their chunks' maps through
// distributed shared memory; the inputs are still read once.  Chunks come through a
// ring of shared-memory stages filled ahead: by TMA, by 4-byte asynchronous copies
// where rows do not start on 16-byte boundaries; odd widths of 16-bit data are
// read directly.
// A composition whose A is exactly 0 (a reset) takes H alone: neither a state that is not
// finite nor a NaN gate passes a reset, forward or backward.
// The forward saves the state that enters each chunk, in fp32, for the backward,
// which recomputes the chunk's states from it.
#include <cooperative_groups.h>
#include <cuda.h>
#include <cudaTypedefs.h>

#include <atomic>
#include <climits>
#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "tc.cuh"

namespace ssm {
namespace glr {

constexpr int kWarps = 8, kThreads = kWarps * 32;
// A warp's steps of a chunk.  The forward holds 16 (its two factors a step and z fill
// the 128 registers of two CTAs per SM): 2 x 16384 x 5120 bf16 with gate takes 271 us, 313
// with 8 and three CTAs per SM, whose exchange comes twice as often; 16 x 4096 x 5120 416
// and 431.  The backward holds more for a step, so 8.
constexpr int kFwdSteps = 16, kBwdSteps = 8;
constexpr int kMaxCluster = 8;
constexpr int kRow = 128;                           // bytes of a step of one tensor

struct Args {
    int64_t batch, length, dim, chunks;             // chunks of this pass
    int64_t saved;                                  // states saved per batch row (every kBwdSteps kWarps steps)
    int64_t xt, xb, ft, fb, zt, zb, dyt, dyb;      // token and batch strides
    const void* x; const void* forget; const void* z;
    const float* lower; const float* init; const uint8_t* reset;
    void* y; float* final_state; float* states;
    const void* dy; const float* dfinal;
    void* dx; void* dforget; void* dz; float* dinit; float* part;
    int words;                                      // 4-byte accesses are aligned
    int* status;
};

// x, forget, z, dy as (channel, token, batch row)
struct TmaArgs {
    Args a;
    alignas(64) CUtensorMap m[4];
    int cluster;                                    // host: the launch's cluster size
};

__device__ int g_glr_error;

// A bounded wait ran out: record the code in the device's flag and in the
// call's status word; the first failure wins.
__device__ __forceinline__ void report(const Args& a, int code) {
    atomicCAS(&g_glr_error, 0, code);
    if (a.status) atomicCAS(a.status, 0, code);
}

// A bounded wait of a CTA, for at most `polls` tries.  One that gives up leaves the others a single
// try: from then on no more copies are asked for and no more maps sent, so that the CTA gets to its
// end, where what is on its way still has the time of a whole wait to land.
constexpr uint32_t kPolls = 1u << 22;
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, volatile uint32_t* polls) {
    const bool ok = tc::mbar_wait(bar, parity, *polls);
    if (!ok) *polls = 1;
    return ok;
}
__device__ __forceinline__ void let_land(uint32_t bar) {
    if (threadIdx.x == 0)
        for (uint32_t parity = 0; parity < 2; ++parity) tc::mbar_wait(bar, parity);
}

// ------------------------------------------------- one or two channels a lane --
template <typename T> struct Lane { using F = float2; static constexpr int E = 2; };
template <> struct Lane<float> { using F = float; static constexpr int E = 1; };

__device__ __forceinline__ float fm(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float2 fm(float2 a, float2 b, float2 c) { return fma2(a, b, c); }
__device__ __forceinline__ float mu(float a, float b) { return a * b; }
__device__ __forceinline__ float2 mu(float2 a, float2 b) { return mul2(a, b); }
__device__ __forceinline__ float ad(float a, float b) { return a + b; }
__device__ __forceinline__ float2 ad(float2 a, float2 b) { return add2(a, b); }
template <typename F> __device__ __forceinline__ F same(float v);
template <> __device__ __forceinline__ float same<float>(float v) { return v; }
template <> __device__ __forceinline__ float2 same<float2>(float v) { return f2(v); }
template <typename F> __device__ __forceinline__ F sub(F a, F b) { return fm(b, same<F>(-1.0f), a); }

// 1 / (1 + e^v): two MUFU operations (e^v may overflow: the result is then 0).
__device__ __forceinline__ float sigmoid_neg(float v) { return rcp_mufu(1.0f + exp2_mufu(v * kLog2e)); }
__device__ __forceinline__ float2 sigmoid_neg(float2 v) {
    const float2 m = mul2(v, f2(kLog2e));
    const float2 d = add2(f2(1.0f), make_float2(exp2_mufu(m.x), exp2_mufu(m.y)));
    return make_float2(rcp_mufu(d.x), rcp_mufu(d.y));
}
// The same in two halves, for the backward: e^v, and k = 1 / (1 + e^v) from it.  1 - k
// is then e^v k with the digits that k near 1 has lost; where e^v overflowed (infinity
// times the 0 that k became) it is 1, which the minimum returns for a NaN.
__device__ __forceinline__ float exp_of(float v) { return exp2_mufu(v * kLog2e); }
__device__ __forceinline__ float2 exp_of(float2 v) {
    const float2 m = mul2(v, f2(kLog2e));
    return make_float2(exp2_mufu(m.x), exp2_mufu(m.y));
}
__device__ __forceinline__ float gate_of(float e) { return rcp_mufu(1.0f + e); }
__device__ __forceinline__ float2 gate_of(float2 e) {
    const float2 d = add2(f2(1.0f), e);
    return make_float2(rcp_mufu(d.x), rcp_mufu(d.y));
}
__device__ __forceinline__ float complement(float e, float k) { return fminf(e * k, 1.0f); }
__device__ __forceinline__ float2 complement(float2 e, float2 k) {
    const float2 c = mul2(e, k);
    return make_float2(fminf(c.x, 1.0f), fminf(c.y, 1.0f));
}
// 1 / (1 + e^-v)
__device__ __forceinline__ float sigmoid_pos(float v) { return rcp_mufu(1.0f + exp2_mufu(v * -kLog2e)); }
__device__ __forceinline__ float2 sigmoid_pos(float2 v) {
    const float2 m = mul2(v, f2(-kLog2e));
    const float2 d = add2(f2(1.0f), make_float2(exp2_mufu(m.x), exp2_mufu(m.y)));
    return make_float2(rcp_mufu(d.x), rcp_mufu(d.y));
}

// S -> A S + H; with resets, where A is 0 the state that enters does not matter.
template <bool RESET>
__device__ __forceinline__ float through(float A, float H, float S) {
    return RESET && A == 0.0f ? H : fmaf(A, S, H);
}
template <bool RESET>
__device__ __forceinline__ float2 through(float2 A, float2 H, float2 S) {
    if constexpr (!RESET) return fma2(A, S, H);
    return make_float2(through<true>(A.x, H.x, S.x), through<true>(A.y, H.y, S.y));
}

template <typename T> __device__ __forceinline__ typename Lane<T>::F unpack(uint32_t w);
template <> __device__ __forceinline__ float unpack<float>(uint32_t w) { return __uint_as_float(w); }
template <> __device__ __forceinline__ float2 unpack<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 unpack<__half>(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// A forget word whose gates keep the state (+infinity: g = 0), for steps past the end.
template <typename T> constexpr uint32_t kKeep = 0x7f800000u;
template <> constexpr uint32_t kKeep<__nv_bfloat16> = 0x7f807f80u;
template <> constexpr uint32_t kKeep<__half> = 0x7c007c00u;

// The lane's word at p: channels c (and c + 1) of `dim`; zero outside.
template <typename T>
__device__ __forceinline__ uint32_t ld_word(const T* p, int64_t c, int64_t dim, bool words) {
    if constexpr (sizeof(T) == 4) {
        return c < dim ? *reinterpret_cast<const uint32_t*>(p) : 0u;
    } else {
        if (words && c + 1 < dim) return *reinterpret_cast<const uint32_t*>(p);
        const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
        uint32_t w = c < dim ? h[0] : 0u;
        if (c + 1 < dim) w |= (uint32_t)h[1] << 16;
        return w;
    }
}
__device__ __forceinline__ void st_lane(float* p, float v) { *p = v; }
template <typename T> __device__ __forceinline__ void st_lane(T* p, float2 v) { Io2<T>::st(p, v); }
template <typename T>
__device__ __forceinline__ void st_word(T* p, typename Lane<T>::F v, int64_t c, int64_t dim, bool words) {
    if constexpr (sizeof(T) == 4) {
        if (c < dim) *p = v;
    } else {
        if (words && c + 1 < dim) {
            Io2<T>::st(p, v);
        } else {
            if (c < dim) stf(p, v.x);
            if (c + 1 < dim) stf(p + 1, v.y);
        }
    }
}
// The lane's words of one output tensor, step by step.  ODD: words may be unaligned or
// half outside; otherwise one predicated 4-byte store.
template <typename T, bool ODD>
struct Out {
    T* p;
    int live;                                       // steps to store: none for channels outside
    int64_t c, dim;
    __device__ __forceinline__ Out(void* base, int64_t at, int64_t c_, int64_t dim_, int n)
        : p(static_cast<T*>(base) + at), live(c_ < dim_ ? n : 0), c(c_), dim(dim_) {}
    __device__ __forceinline__ void put(int i, typename Lane<T>::F v) const {
        if (i < live) {
            if constexpr (ODD) st_word<T>(p, v, c, dim, false);
            else st_lane(p, v);
        }
    }
    __device__ __forceinline__ void move(int64_t by) { p += by; }
};
// The lane's channels of a per-channel fp32 array; `none` where absent or outside.
__device__ __forceinline__ void ld_chan(const float* p, int64_t c, int64_t dim, float none, float& v) {
    v = (p != nullptr && c < dim) ? p[c] : none;
}
__device__ __forceinline__ void ld_chan(const float* p, int64_t c, int64_t dim, float none, float2& v) {
    v.x = (p != nullptr && c < dim) ? p[c] : none;
    v.y = (p != nullptr && c + 1 < dim) ? p[c + 1] : none;
}
__device__ __forceinline__ void st_chan(float* p, int64_t c, int64_t dim, float v) {
    if (c < dim) p[c] = v;
}
__device__ __forceinline__ void st_chan(float* p, int64_t c, int64_t dim, float2 v) {
    if (c < dim) p[c] = v.x;
    if (c + 1 < dim) p[c + 1] = v.y;
}

// Whether the lane's one of the warp's N steps (from t) is a reset.  The warp votes on it where the mask is
// used, so that the load's time passes beside the gates'.
template <int N>
__device__ __forceinline__ uint8_t reset_at(const uint8_t* reset, int64_t row, int64_t t, int64_t length) {
    const int lane = threadIdx.x & 31;
    return lane < N && t + lane < length ? reset[row + t + lane] : (uint8_t)0;
}
// Bit i: step i is a reset.
__device__ __forceinline__ uint32_t reset_mask(uint8_t at) { return __ballot_sync(0xffffffffu, at != 0); }

template <typename T, int N>
__device__ __forceinline__ void ld_steps(const void* base, int64_t row, int64_t stride, int64_t t, int live, int64_t c,
                                         const Args& a, uint32_t* w) {
    const T* p = static_cast<const T*>(base) + row + t * stride + c;
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = i < live ? ld_word<T>(p + i * stride, c, a.dim, a.words) : 0u;
}

// The ring of chunk tiles in shared memory: stage s holds NT tensors' chunks, a warp's steps being N consecutive 128-byte rows of each.
// TMA: thread 0 issues, the wait of a stage is every thread's.  kWords: each lane
// copies the words that it will read itself, so its own wait is enough.
enum Loads { kDirect, kWords, kTma };
template <int NT, int ST, int N>
struct Ring {
    static constexpr int kTile = kWarps * N * kRow;   // bytes of one tensor's chunk
    uint8_t* base;                  // ST * NT * kTile bytes, then ST mbarriers
    static constexpr size_t bytes = (size_t)ST * NT * kTile + ST * 8;
    __device__ __forceinline__ uint32_t bar(int s) const {
        return tc::smem_u32(base + (size_t)ST * NT * kTile) + s * 8;
    }
    __device__ __forceinline__ void init() const {
        if (threadIdx.x == 0) {
            for (int s = 0; s < ST; ++s) tc::mbar_init(bar(s), 1);
            tc::fence_mbar_init();
        }
        __syncthreads();
    }
    // The chunk at token t of batch row b into stage s: tensor i of the stage is map which[i].
    __device__ __forceinline__ void load(const TmaArgs& ta, int s, int c0, int64_t t, int b, const int* which) const {
        tc::mbar_expect_tx(bar(s), NT * kTile);
        for (int i = 0; i < NT; ++i)
            tc::tma_load3(tc::smem_u32(base + (s * NT + i) * kTile), &ta.m[which[i]], c0, (int)t, b, bar(s));
    }
    __device__ __forceinline__ void drain() const {
        for (int s = 0; s < ST; ++s) let_land(bar(s));
    }
    // The lane's words of tensor i: N steps from p, `live` of them inside the sequence.
    template <typename T>
    __device__ __forceinline__ void copy(int s, int i, const void* tensor, int64_t row, int64_t stride, int64_t t,
                                         int live, int64_t c, int64_t dim) const {
        const T* p = static_cast<const T*>(tensor) + row + t * stride + c;
        const uint32_t d = tc::smem_u32(base + (s * NT + i) * kTile) + (threadIdx.x / 32 * N * 32 + (threadIdx.x & 31)) * 4;
        if (live == N && c < dim) {
#pragma unroll
            for (int k = 0; k < N; ++k, p += stride) tc::cp_async4_zfill(d + k * kRow, p, 4u);
        } else {
#pragma unroll 1
            for (int k = 0; k < N; ++k, p += stride) {
                const bool in = k < live && c < dim;
                tc::cp_async4_zfill(d + k * kRow, in ? static_cast<const void*>(p) : tensor, in ? 4u : 0u);
            }
        }
    }
    __device__ __forceinline__ void read(int s, int i, uint32_t* w) const {
        const uint32_t* p = reinterpret_cast<const uint32_t*>(base + (s * NT + i) * kTile) + threadIdx.x / 32 * N * 32 +
                            (threadIdx.x & 31);
#pragma unroll
        for (int k = 0; k < N; ++k) w[k] = p[k * 32];
    }
};

// The values as the compiler cannot know them: what is computed from them later is
// computed again rather than kept in registers from an earlier use.
template <int N>
__device__ __forceinline__ void again(uint32_t (&w)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(w[i]));
}
template <int N>
__device__ __forceinline__ void again(float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+f"(v[i]));
}
template <int N>
__device__ __forceinline__ void again(float2 (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+f"(v[i].x), "+f"(v[i].y));
}

template <typename F> struct Map { F A, H; };
// Factors joined: with resets, 0 whatever the other factor is (a gate may be NaN).
template <bool RESET>
__device__ __forceinline__ float joined(float A, float B) { return RESET && (A == 0.0f || B == 0.0f) ? 0.0f : A * B; }
template <bool RESET>
__device__ __forceinline__ float2 joined(float2 A, float2 B) {
    if constexpr (!RESET) return mul2(A, B);
    return make_float2(joined<true>(A.x, B.x), joined<true>(A.y, B.y));
}
template <bool RESET, typename F>
__device__ __forceinline__ Map<F> then(const Map<F>& first, const Map<F>& next) {
    return {joined<RESET>(first.A, next.A), through<RESET>(next.A, next.H, first.H)};
}

// A product A of factors near one is known to 2^-24 of itself a factor, and with steady gates the
// errors of a long row's products all go one way.  So a warp also adds up B, what its steps took
// from the product: (1 - B) - A is what A lacks, exact where A is in [1/2, 1].  That, and what
// was left over from the turn before, is added to A; what the sum's rounding leaves (at most 2^-25)
// waits for the next turn's product.  A state that remembers across turns thereby meets errors that
// cancel; where A is below a half nothing is remembered that long.
__device__ __forceinline__ void settle(float& A, float lacks, float& left) {
    if (A >= 0.5f && A <= 1.0f) {
        lacks += left;
        const float whole = A + lacks;
        left = lacks - (whole - A);
        A = whole;
    }
}
__device__ __forceinline__ void settle(float2& A, float2 lacks, float2& left) {
    settle(A.x, lacks.x, left.x);
    settle(A.y, lacks.y, left.y);
}
template <typename F>
__device__ __forceinline__ F lacking(F A, F B) { return sub(sub(same<F>(1.0f), A), B); }
// `first` then `next`, and what the rounded product lacks added to `lacks` (to first order: for products near one).
template <bool RESET, typename F>
__device__ __forceinline__ Map<F> then(const Map<F>& first, const Map<F>& next, F& lacks) {
    const Map<F> r = then<RESET>(first, next);
    lacks = ad(lacks, fm(first.A, next.A, mu(r.A, same<F>(-1.0f))));
    return r;
}

// A cluster of C CTAs takes C consecutive chunks at a time (a round): each CTA
// sends its chunk's map to all of them with asynchronous remote stores that
// count their bytes on the receiver's mbarrier, and waits for the C maps of the
// round.  No fence is involved: a cluster barrier's release would first wait for
// the round's global stores (a round of 4 x 64 steps took 4 us with one).
// Two buffers alternate: a CTA sends round n + 2 only after it has every map of
// round n + 1, which a peer sends after all its warps have read round n.
__device__ __forceinline__ uint32_t remote(uint32_t addr, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void send(uint32_t addr, uint32_t bar, float a, float h) {
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];"
                 :: "r"(addr), "r"(__float_as_uint(a)), "r"(__float_as_uint(h)), "r"(bar) : "memory");
}
__device__ __forceinline__ void send(uint32_t addr, uint32_t bar, float2 a, float2 h) {
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];"
                 :: "r"(addr), "r"(__float_as_uint(a.x)), "r"(__float_as_uint(a.y)), "r"(__float_as_uint(h.x)),
                    "r"(__float_as_uint(h.y)), "r"(bar) : "memory");
}
template <typename F>
struct alignas(128) Exchange {        // whole 128-byte lines: the ring behind it starts on one
    Map<F> far[2][kMaxCluster][32];
    uint64_t bars[2];
    __device__ __forceinline__ void arm(int s, int C) {
        tc::mbar_expect_tx(tc::smem_u32(&bars[s]), (uint32_t)(C * 32 * sizeof(Map<F>)));
    }
    __device__ __forceinline__ void init(int C) {
        if (threadIdx.x == 0) {
            for (int s = 0; s < 2; ++s) tc::mbar_init(tc::smem_u32(&bars[s]), 1);
            tc::fence_mbar_init();
            arm(0, C);
            arm(1, C);
        }
    }
    // One warp: its lanes' maps of the whole chunk to every CTA.
    __device__ __forceinline__ void put(int round, int rank, int C, const Map<F>& all) {
        const int s = round & 1;
        const uint32_t at = tc::smem_u32(&far[s][rank][threadIdx.x & 31]), bar = tc::smem_u32(&bars[s]);
        for (int r = 0; r < C; ++r) send(remote(at, r), remote(bar, r), all.A, all.H);
    }
    // Every thread: the round's maps are here.
    __device__ __forceinline__ bool wait(int round, int C, volatile uint32_t* polls) {
        const int s = round & 1;
        if (!wait_for(tc::smem_u32(&bars[s]), (uint32_t)(round >> 1) & 1u, polls)) return false;
        if (threadIdx.x == 0) arm(s, C);
        return true;
    }
    __device__ __forceinline__ void drain() {
        for (int s = 0; s < 2; ++s) let_land(tc::smem_u32(&bars[s]));
    }
};
__device__ __forceinline__ int cluster_size() { return (int)cooperative_groups::this_cluster().num_blocks(); }

template <typename T, bool GATE, bool RESET, int LOADS, int ST, int N>
__global__ void __launch_bounds__(kThreads, N > 8 ? 2 : 3)
fwd_kernel(const __grid_constant__ TmaArgs ta) {
    using F = typename Lane<T>::F;
    constexpr int E = Lane<T>::E, NT = GATE ? 3 : 2, kChunk = kWarps * N;
    const Args& a = ta.a;
    __shared__ Map<F> maps[2][kWarps][32];
    __shared__ Exchange<F> ex;
    __shared__ volatile uint32_t polls;
    extern __shared__ __align__(128) uint8_t smem[];
    const Ring<NT, ST, N> ring{smem};
    const int which[3] = {0, 1, 2};
    const auto cluster = cooperative_groups::this_cluster();
    const int C = cluster_size(), rank = (int)cluster.block_rank();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t b = blockIdx.y, tile = blockIdx.x / C, c = (tile * 32 + lane) * E;
    // tokens, chunks and rounds fit 31 bits, a last chunk's overhang included
    const int rounds = (int)((a.chunks + C - 1) / C);
    if (threadIdx.x == 0) polls = kPolls;
    __syncthreads();
    if (C > 1) {
        ex.init(C);
        cluster.sync();                                 // every CTA's barriers are there to write to
    }
    // the chunk of round n into its stage
    auto fill = [&](int n) {
        const int s = n % ST;
        const int t0 = (n * C + rank) * kChunk;
        if constexpr (LOADS == kTma) {
            if (threadIdx.x == 0 && polls == kPolls) ring.load(ta, s, (int)(tile * 32 * E), t0, (int)b, which);
        } else if constexpr (LOADS == kWords) {
            const int t = t0 + warp * N;
            const int live = max(0, min(N, (int)a.length - t));
            ring.template copy<T>(s, 0, a.x, b * a.xb, a.xt, t, live, c, a.dim);
            ring.template copy<T>(s, 1, a.forget, b * a.fb, a.ft, t, live, c, a.dim);
            if (GATE) ring.template copy<T>(s, 2, a.z, b * a.zb, a.zt, t, live, c, a.dim);
        }
    };
    if constexpr (LOADS == kTma) ring.init();
    for (int s = 0; s < ST; ++s) {
        if (s < rounds) fill(s);
        if constexpr (LOADS == kWords) tc::cp_async_commit();
    }
    F span, nspan, S;
    ld_chan(a.lower, c, a.dim, 0.0f, span);
    nspan = sub(span, same<F>(1.0f));
    span = sub(same<F>(1.0f), span);
    ld_chan(a.init ? a.init + b * a.dim : nullptr, c, a.dim, 0.0f, S);
    F left = same<F>(0.0f), left_all = same<F>(0.0f);
    for (int n = 0; n < rounds; ++n) {
        const int chunk = n * C + rank, t = chunk * kChunk + warp * N;
        const int live = max(0, min(N, (int)a.length - t));
        uint32_t zw[N];
        F av[N], bv[N];                   // h -> av h + bv
        Map<F> m{same<F>(1.0f), same<F>(0.0f)};
        F B = same<F>(0.0f);              // 1 - m.A, added up
        uint32_t rs = 0;                  // the resets among the steps
        const uint8_t reset = RESET ? reset_at<N>(a.reset, b * a.length, t, a.length) : (uint8_t)0;
        {
            uint32_t xw[N], fw[N];
            if constexpr (LOADS != kDirect) {
                const int s = n % ST;
                if constexpr (LOADS == kTma) {
                    if (!wait_for(ring.bar(s), (uint32_t)(n / ST) & 1u, &polls)) report(a, 111);
                } else {
                    tc::cp_async_wait<ST - 1>();
                }
                ring.read(s, 0, xw);
                ring.read(s, 1, fw);
                if (GATE) ring.read(s, 2, zw);
            } else {
                ld_steps<T, N>(a.x, b * a.xb, a.xt, t, live, c, a, xw);
                ld_steps<T, N>(a.forget, b * a.fb, a.ft, t, live, c, a, fw);
                if (GATE) ld_steps<T, N>(a.z, b * a.zb, a.zt, t, live, c, a, zw);
            }
            if (RESET) rs = reset_mask(reset);
            if (live < N) {
#pragma unroll
                for (int i = 0; i < N; ++i) fw[i] = i < live ? fw[i] : kKeep<T>;
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const F k = sigmoid_neg(unpack<T>(fw[i])), g = mu(span, k);
                av[i] = fm(nspan, k, same<F>(1.0f));
                bv[i] = mu(g, unpack<T>(xw[i]));
                if (RESET && (rs >> i & 1u)) m = {same<F>(0.0f), same<F>(0.0f)};
                B = fm(g, m.A, B);
                m.H = fm(av[i], m.H, bv[i]);
                m.A = mu(m.A, av[i]);
            }
        }
        if (RESET && rs) m.A = same<F>(0.0f);             // also where a later gate is NaN
        settle(m.A, lacking(m.A, B), left);
        Map<F>(*mw)[32] = maps[n & 1];
        mw[warp][lane] = m;
        __syncthreads();
        // every warp has its words in registers: the stage is free
        if (n + ST < rounds) fill(n + ST);
        if constexpr (LOADS == kWords) tc::cp_async_commit();          // one group a round
        F h;
        if (C == 1) {
            h = S;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const Map<F> o = mw[w][lane];
                if (w == warp) h = S;
                S = through<RESET>(o.A, o.H, S);
            }
        } else {
            Map<F> before{same<F>(1.0f), same<F>(0.0f)};
#pragma unroll
            for (int w = 0; w < kWarps - 2; ++w)
                if (w < warp && warp < kWarps - 1) before = then<RESET>(before, mw[w][lane]);
            if (warp == kWarps - 1) {
                F lacks = same<F>(0.0f);
                before = {same<F>(1.0f), same<F>(0.0f)};
#pragma unroll
                for (int w = 0; w < kWarps - 1; ++w) before = then<RESET>(before, mw[w][lane], lacks);
                Map<F> all = then<RESET>(before, m, lacks);
                settle(all.A, lacks, left_all);
                if (polls == kPolls) ex.put(n, rank, C, all);
            }
            if (!ex.wait(n, C, &polls)) report(a, 113);
            h = S;
#pragma unroll
            for (int r = 0; r < kMaxCluster; ++r) {
                if (r < C) {
                    if (r == rank) h = S;
                    const Map<F> o = ex.far[n & 1][r][lane];
                    S = through<RESET>(o.A, o.H, S);
                }
            }
            h = through<RESET>(before.A, before.H, h);
        }
        // the state that enters every kBwdSteps kWarps steps, for the backward
        if (a.states != nullptr && warp % (kBwdSteps * kWarps / N) == 0 && live > 0)
            st_chan(a.states + (b * a.saved + t / (kBwdSteps * kWarps)) * a.dim, c, a.dim, h);
        Out<T, LOADS == kDirect> y(a.y, (b * a.length + t) * a.dim + c, c, a.dim, live);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (RESET && (rs >> i & 1u)) h = same<F>(0.0f);
            h = fm(av[i], h, bv[i]);
            F o = h;
            if (GATE) {
                const F z = unpack<T>(zw[i]);
                o = mu(h, mu(z, sigmoid_pos(z)));
            }
            y.put(i, o);
            y.move(a.dim);
        }
    }
    if (LOADS == kTma && polls != kPolls) ring.drain();
    if (C > 1) {
        cluster.sync();                                 // nothing is on its way to a CTA that ends
        if (polls != kPolls) ex.drain();
    }
    if (warp == 0 && rank == 0) st_chan(a.final_state + b * a.dim, c, a.dim, S);
}

template <typename T, bool GATE, bool RESET, int LOADS, int ST, int N>
__global__ void __launch_bounds__(kThreads, 2)
bwd_kernel(const __grid_constant__ TmaArgs ta) {
    using F = typename Lane<T>::F;
    constexpr int E = Lane<T>::E, NT = GATE ? 4 : 3, kChunk = kWarps * N;
    const Args& a = ta.a;
    __shared__ struct { Map<F> m[32]; F R[32]; } maps[2][kWarps];
    __shared__ Exchange<F> ex;            // of (A, R)
    __shared__ volatile uint32_t polls;
    __shared__ F sums[kWarps][32];
    extern __shared__ __align__(128) uint8_t smem[];
    const Ring<NT, ST, N> ring{smem};
    const int which[4] = {0, 1, 3, 2};                  // x, forget, dy, z
    const auto cluster = cooperative_groups::this_cluster();
    const int C = cluster_size(), rank = (int)cluster.block_rank();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t b = blockIdx.y, tile = blockIdx.x / C, c = (tile * 32 + lane) * E;
    // tokens, chunks and rounds fit 31 bits, a last chunk's overhang included
    const int rounds = (int)((a.chunks + C - 1) / C);
    if (threadIdx.x == 0) polls = kPolls;
    __syncthreads();
    if (C > 1) {
        ex.init(C);
        cluster.sync();                                 // every CTA's barriers are there to write to
    }
    // the chunk of a turn into its stage
    auto fill = [&](int turn) {
        const int s = turn % ST;
        const int t0 = ((rounds - 1 - turn) * C + rank) * kChunk;
        if constexpr (LOADS == kTma) {
            if (threadIdx.x == 0 && polls == kPolls) ring.load(ta, s, (int)(tile * 32 * E), t0, (int)b, which);
        } else if constexpr (LOADS == kWords) {
            const int t = t0 + warp * N;
            const int live = max(0, min(N, (int)a.length - t));
            ring.template copy<T>(s, 0, a.x, b * a.xb, a.xt, t, live, c, a.dim);
            ring.template copy<T>(s, 1, a.forget, b * a.fb, a.ft, t, live, c, a.dim);
            ring.template copy<T>(s, 2, a.dy, b * a.dyb, a.dyt, t, live, c, a.dim);
            if (GATE) ring.template copy<T>(s, 3, a.z, b * a.zb, a.zt, t, live, c, a.dim);
        }
    };
    if constexpr (LOADS == kTma) ring.init();
    for (int s = 0; s < ST; ++s) {
        if (s < rounds) fill(s);
        if constexpr (LOADS == kWords) tc::cp_async_commit();
    }
    const F one = same<F>(1.0f), zero = same<F>(0.0f);
    F span, nspan, D;
    ld_chan(a.lower, c, a.dim, 0.0f, span);
    nspan = sub(span, one);
    span = sub(one, span);
    ld_chan(a.dfinal ? a.dfinal + b * a.dim : nullptr, c, a.dim, 0.0f, D);
    F dlower = zero, left = zero, left_all = zero;
    for (int turn = 0; turn < rounds; ++turn) {
        const int chunk = (rounds - 1 - turn) * C + rank, t = chunk * kChunk + warp * N;
        const int live = max(0, min(N, (int)a.length - t));
        uint32_t xw[N], zw[N], dw[N];
        F ev[N], h;                       // e^forget
        const uint8_t reset = RESET ? reset_at<N>(a.reset, b * a.length, t, a.length) : (uint8_t)0;
        ld_chan(chunk < a.chunks ? a.states + (b * a.saved + chunk) * a.dim : nullptr, c, a.dim, 0.0f, h);
        {
            uint32_t fw[N];
            if constexpr (LOADS != kDirect) {
                const int s = turn % ST;
                if constexpr (LOADS == kTma) {
                    if (!wait_for(ring.bar(s), (uint32_t)(turn / ST) & 1u, &polls)) report(a, 112);
                } else {
                    tc::cp_async_wait<ST - 1>();
                }
                ring.read(s, 0, xw);
                ring.read(s, 1, fw);
                ring.read(s, 2, dw);
                if (GATE) ring.read(s, 3, zw);
            } else {
                ld_steps<T, N>(a.x, b * a.xb, a.xt, t, live, c, a, xw);
                ld_steps<T, N>(a.forget, b * a.fb, a.ft, t, live, c, a, fw);
                if (GATE) ld_steps<T, N>(a.z, b * a.zb, a.zt, t, live, c, a, zw);
                ld_steps<T, N>(a.dy, b * a.dyb, a.dyt, t, live, c, a, dw);
            }
            if (live < N) {
#pragma unroll
                for (int i = 0; i < N; ++i) fw[i] = i < live ? fw[i] : kKeep<T>;
            }
#pragma unroll
            for (int i = 0; i < N; ++i) ev[i] = exp_of(unpack<T>(fw[i]));
        }
        const uint32_t rs = RESET ? reset_mask(reset) : 0u;
        Map<F> m{one, zero};
        F B = zero;                                     // 1 - m.A, added up
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const F k = gate_of(ev[i]), g = mu(span, k), av = fm(nspan, k, one);
            if (RESET && (rs >> i & 1u)) m = {zero, zero};
            B = fm(g, m.A, B);
            m.H = fm(av, m.H, mu(g, unpack<T>(xw[i])));
            m.A = mu(m.A, av);
        }
        if (RESET && rs) m.A = same<F>(0.0f);             // also where a later gate is NaN
        settle(m.A, lacking(m.A, B), left);
        F d = zero;
#pragma unroll
        for (int i = N - 1; i >= 0; --i) {
            F e = unpack<T>(dw[i]);
            if (GATE) {
                const F z = unpack<T>(zw[i]);
                e = mu(e, mu(z, sigmoid_pos(z)));
            }
            d = mu(ad(d, e), fm(nspan, gate_of(ev[i]), one));
            if (RESET && (rs >> i & 1u)) d = zero;
        }
        auto& mw = maps[turn & 1];
        mw[warp].m[lane] = m;
        mw[warp].R[lane] = d;
        __syncthreads();
        if (turn + ST < rounds) fill(turn + ST);
        if constexpr (LOADS == kWords) tc::cp_async_commit();          // one group a turn
        if (C == 1) {
            d = D;
#pragma unroll
            for (int w = kWarps - 1; w >= 0; --w) {
                const F A = mw[w].m[lane].A;
                if (w == warp) d = D;
                D = through<RESET>(A, mw[w].R[lane], D);
            }
        } else {
            Map<F> after{one, zero};
#pragma unroll
            for (int w = kWarps - 1; w > 1; --w)
                if (w > warp && warp > 0) after = then<RESET>(after, Map<F>{mw[w].m[lane].A, mw[w].R[lane]});
            if (warp == 0) {
                F lacks = zero;
#pragma unroll
                for (int w = kWarps - 1; w > 0; --w)
                    after = then<RESET>(after, Map<F>{mw[w].m[lane].A, mw[w].R[lane]}, lacks);
                Map<F> all = then<RESET>(after, Map<F>{m.A, d}, lacks);
                settle(all.A, lacks, left_all);
                if (polls == kPolls) ex.put(turn, rank, C, all);
            }
            if (!ex.wait(turn, C, &polls)) report(a, 114);
            d = D;
#pragma unroll
            for (int r = kMaxCluster - 1; r >= 0; --r) {
                if (r < C) {
                    if (r == rank) d = D;
                    const Map<F> o = ex.far[turn & 1][r][lane];
                    D = through<RESET>(o.A, o.H, D);
                }
            }
            d = through<RESET>(after.A, after.H, d);
        }
#pragma unroll
        for (int w = 0; w < kWarps - 1; ++w) {
            if (w < warp) {
                const Map<F> o = mw[w].m[lane];
                h = through<RESET>(o.A, o.H, h);
            }
        }
        F hp[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            hp[i] = h;
            if (RESET && (rs >> i & 1u)) h = zero;
            const F k = gate_of(ev[i]);
            h = fm(fm(nspan, k, one), h, mu(mu(span, k), unpack<T>(xw[i])));
        }
        again(xw);
        again(ev);
        again(dw);
        if (GATE) again(zw);
        const int64_t at = (b * a.length + t + N - 1) * a.dim + c;
        Out<T, LOADS == kDirect> dx(a.dx, at, c, a.dim, live), df(a.dforget, at, c, a.dim, live);
        Out<T, LOADS == kDirect> dz(GATE ? a.dz : nullptr, at, c, a.dim, live);
        F dl = zero;
#pragma unroll
        for (int i = N - 1; i >= 0; --i) {
            const F k = gate_of(ev[i]), x = unpack<T>(xw[i]), dy = unpack<T>(dw[i]);
            F e = dy;
            if (GATE) {
                const F z = unpack<T>(zw[i]), s = sigmoid_pos(z), zs = mu(z, s);
                e = mu(dy, zs);
                // silu'(z) = s + z s (1 - s)
                const F ds = fm(zs, sub(one, s), s);
                dz.put(i, mu(mu(dy, h), ds));
                dz.move(-a.dim);
            }
            d = ad(d, e);                          // dh of step i
            h = hp[i];                             // what step i - 1 left
            const F gd = mu(mu(span, k), d), before = RESET && (rs >> i & 1u) ? zero : h;
            const F back = sub(before, x);         // -dg = dh (h' - x)
            dx.put(i, gd);
            dx.move(-a.dim);
            df.put(i, mu(mu(gd, back), complement(ev[i], k)));
            df.move(-a.dim);
            dl = fm(mu(d, back), k, dl);
            d = RESET && (rs >> i & 1u) ? zero : sub(d, gd);
        }
        dlower = ad(dlower, dl);
    }
    if (LOADS == kTma && polls != kPolls) ring.drain();
    if (C > 1) {
        cluster.sync();                                 // nothing is on its way to a CTA that ends
        if (polls != kPolls) ex.drain();
    }
    if (warp == 0 && rank == 0 && a.dinit != nullptr) st_chan(a.dinit + b * a.dim, c, a.dim, D);
    if (a.part != nullptr) {
        sums[warp][lane] = dlower;
        __syncthreads();
        if (warp == 0) {
            F s = sums[0][lane];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) s = ad(s, sums[w][lane]);
            st_chan(a.part + (b * C + rank) * a.dim, c, a.dim, s);
        }
    }
}

// dlower[c] = the partial rows added in order.
__global__ void fold_kernel(const float* part, int64_t rows, int64_t dim, float* out) {
    const int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= dim) return;
    float s = 0.0f;
    for (int64_t r = 0; r < rows; ++r) s += part[r * dim + c];
    out[c] = s;
}

// ------------------------------------------------------------ one token a row --
struct StepArgs {
    int64_t batch, dim, xb, fb, zb, sb, lanes;      // batch strides; lanes per row
    const void* x; const void* forget; const void* z; const float* lower; float* state; void* y;
    int words;
};

// Open gates (g below a half): h + (g x - g h), as the rounding of 1 - g would add up over many
// calls; above, 1 - g is exact.  An infinite h stays so.
__device__ __forceinline__ float next_state(float g, float h, float gx) {
    return g < 0.5f && fabsf(h) < __int_as_float(0x7f800000) ? h + fmaf(-g, h, gx) : fmaf(1.0f - g, h, gx);
}
__device__ __forceinline__ float2 next_state(float2 g, float2 h, float2 gx) {
    return make_float2(next_state(g.x, h.x, gx.x), next_state(g.y, h.y, gx.y));
}

template <typename T, bool GATE>
__global__ void __launch_bounds__(kThreads)
step_kernel(const StepArgs a) {
    using F = typename Lane<T>::F;
    constexpr int E = Lane<T>::E;
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= a.batch * a.lanes) return;
    const int64_t b = i / a.lanes, c = (i % a.lanes) * E;
    const F x = unpack<T>(ld_word<T>(static_cast<const T*>(a.x) + b * a.xb + c, c, a.dim, a.words));
    const F f = unpack<T>(ld_word<T>(static_cast<const T*>(a.forget) + b * a.fb + c, c, a.dim, a.words));
    F z = same<F>(0.0f), span, h;
    if (GATE) z = unpack<T>(ld_word<T>(static_cast<const T*>(a.z) + b * a.zb + c, c, a.dim, a.words));
    ld_chan(a.lower, c, a.dim, 0.0f, span);
    ld_chan(a.state + b * a.sb, c, a.dim, 0.0f, h);
    const F g = mu(sub(same<F>(1.0f), span), sigmoid_neg(f));
    h = next_state(g, h, mu(g, x));
    st_chan(a.state + b * a.sb, c, a.dim, h);
    if (GATE) h = mu(h, mu(z, sigmoid_pos(z)));
    st_word<T>(static_cast<T*>(a.y) + b * a.dim + c, h, c, a.dim, a.words);
}

// ------------------------------------------------------------------- host ----
static int64_t esize(int dtype) { return dtype == SSM_F32 ? 4 : 2; }
static bool al(const void* p, int64_t b) { return (reinterpret_cast<uintptr_t>(p) % b) == 0; }

static int validate(const ssm_gated_recurrence_params* p) {
    if (p == nullptr) return fail(SSM_ERR_INVALID, "gated_linear_recurrence: null params");
    if (p->batch < 0 || p->length < 0 || p->dim < 1)
        return fail(SSM_ERR_INVALID, "gated_linear_recurrence: batch, length and dim");
    if (p->batch > 65535 || p->length > INT32_MAX - 65536 || p->dim > INT32_MAX - 65536)
        return fail(SSM_ERR_UNSUPPORTED,
                    "gated_linear_recurrence: batch above 65535, or length or dim above 2^31 - 65537");
    if (p->dtype < SSM_F32 || p->dtype > SSM_F16) return fail(SSM_ERR_UNSUPPORTED, "gated_linear_recurrence: dtype");
    for (int64_t s : {p->x_token_stride, p->forget_token_stride, p->z_token_stride, p->dy_token_stride})
        if (s && s < p->dim) return fail(SSM_ERR_INVALID, "gated_linear_recurrence: a token stride is below dim");
    return SSM_OK;
}

static Args args_of(const ssm_gated_recurrence_params* p, bool bwd) {
    Args a{};
    a.batch = p->batch; a.length = p->length; a.dim = p->dim;
    a.chunks = ceil_div(p->length, kWarps * (bwd ? kBwdSteps : kFwdSteps));
    a.saved = ceil_div(p->length, kWarps * kBwdSteps);
    auto token = [&](int64_t s) { return s ? s : p->dim; };
    auto row = [&](int64_t s, int64_t t) { return s ? s : t * p->length; };
    a.xt = token(p->x_token_stride); a.xb = row(p->x_batch_stride, a.xt);
    a.ft = token(p->forget_token_stride); a.fb = row(p->forget_batch_stride, a.ft);
    a.zt = token(p->z_token_stride); a.zb = row(p->z_batch_stride, a.zt);
    a.dyt = token(p->dy_token_stride); a.dyb = row(p->dy_batch_stride, a.dyt);
    a.x = p->x; a.forget = p->forget; a.z = p->z;
    a.lower = p->lower; a.init = p->initial_state; a.reset = p->reset;
    a.y = p->y; a.final_state = p->final_state; a.states = p->states;
    a.dy = p->dy; a.dfinal = p->dfinal;
    a.dx = p->dx; a.dforget = p->dforget; a.dz = p->dz; a.dinit = p->dinitial;
    a.status = p->status;
    a.words = 1;
    if (p->dtype != SSM_F32) {
        for (const void* q : {p->x, p->forget, p->z, (const void*)p->y, p->dy, (const void*)p->dx,
                              (const void*)p->dforget, (const void*)p->dz})
            if (!al(q, 4)) a.words = 0;
        for (int64_t s : {a.dim, a.xt, a.xb, a.ft, a.fb, p->z ? a.zt : 0, p->z ? a.zb : 0, p->dy ? a.dyt : 0,
                          p->dy ? a.dyb : 0})
            if (s & 1) a.words = 0;
    }
    return a;
}

static PFN_cuTensorMapEncodeTiled_v12000 encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
        else
            cudaGetLastError();
    });
    return fn;
}

// (batch, length, dim) as (channel, token, batch row); box: one chunk of 128-byte rows.
static int encode(CUtensorMap* m, const void* base, int64_t token, int64_t row, int dtype, int chunk, const Args& a) {
    const int64_t es = esize(dtype);
    cuuint64_t dims[3] = {(cuuint64_t)a.dim, (cuuint64_t)a.length, (cuuint64_t)a.batch};
    // a single row's stride is never used, but has to be a valid one
    cuuint64_t strides[2] = {(cuuint64_t)(token * es), (cuuint64_t)((a.batch > 1 ? row : token) * es)};
    cuuint32_t box[3] = {(cuuint32_t)(128 / es), (cuuint32_t)chunk, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    const CUtensorMapDataType type = dtype == SSM_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : dtype == SSM_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                         : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const CUresult r = encoder()(m, type, 3, const_cast<void*>(base), dims, strides, box, estr,
                                 CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r == CUDA_SUCCESS) return SSM_OK;
    return fail(SSM_ERR_CUDA, "gated_linear_recurrence: cuTensorMapEncodeTiled failed (" + std::to_string((int)r) + ")");
}

// TMA reads rows that start on 16-byte boundaries.
static bool tma_ok(const Args& a, int dtype, bool bwd) {
    const int64_t es = esize(dtype);
    auto ok = [&](const void* p, int64_t token, int64_t row) {
        return p == nullptr || (al(p, 16) && (token * es) % 16 == 0 &&
                                (a.batch == 1 || (row * es) % 16 == 0) && token * es < ((int64_t)1 << 40) &&
                                (a.batch == 1 || row * es < ((int64_t)1 << 40)));
    };
    return encoder() && a.length > 0 && ok(a.x, a.xt, a.xb) && ok(a.forget, a.ft, a.fb) && ok(a.z, a.zt, a.zb) &&
           (!bwd || ok(a.dy, a.dyt, a.dyb));
}

// CTAs of a cluster.  With C of them a tile takes ceil(chunks / C) rounds, and the
// tiles run in as many waves as the GPU's room for such clusters needs; a round of a
// cluster costs 12 % and 6 % more per CTA than a lone CTA's (the exchange, and the
// spread of its CTAs).  The C with the least product is taken.  Measured, forward, bf16
// with gate, room for 296 CTAs: 1 x 4096 x 5120 (80 tiles) 57 us with C = 1, 43 with 3,
// 50 with 4; 2 x 16384 x 5120 (160 tiles) 356 us with 1, 328 with 2, 271 with 4, 301
// with 8; 16 x 4096 x 5120 (1280 tiles) 416 us with 1, 470 with 2.
template <auto kernel>
static int cluster_of(int64_t tiles, int64_t chunks, size_t smem) {
    static std::atomic<int> room[kMaxCluster + 1]; // clusters that fit at once, by size; 0: not asked yet
    double best = 0.0;
    int size = 1;
    for (int c = 1; c <= kMaxCluster && c <= chunks; ++c) {
        if (room[c] == 0) {
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = dim3(c);
            cfg.blockDim = dim3(kThreads);
            cfg.dynamicSmemBytes = smem;
            cudaLaunchAttribute at[1];
            at[0].id = cudaLaunchAttributeClusterDimension;
            at[0].val.clusterDim.x = c;
            at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
            cfg.attrs = at;
            cfg.numAttrs = 1;
            int n = 0;
            if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
                cudaGetLastError();
                n = 148 * 2 / c;
            }
            room[c] = n;
        }
        const double cost = (double)ceil_div(tiles, room[c]) * (double)ceil_div(chunks, c) *
                            (c == 1 ? 1.0 : 1.0 + 0.06 * c);
        if (c == 1 || cost < best) {
            best = cost;
            size = c;
        }
    }
    return size;
}

template <auto kernel>
static int launch_kernel(TmaArgs& ta, unsigned tiles, size_t smem, cudaStream_t st, const char* what) {
    if (smem && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
        return check_launch(what);
    const int cluster = cluster_of<kernel>((int64_t)tiles * ta.a.batch, ta.a.chunks, smem);
    ta.cluster = cluster;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(tiles * cluster, (unsigned)ta.a.batch);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kernel, ta);
    return check_launch(what);
}

constexpr int kFwdStages = 2, kBwdStages = 2;

template <typename T, bool GATE, bool RESET, int LOADS>
static int launch(TmaArgs& ta, bool bwd, cudaStream_t st) {
    const unsigned tiles = (unsigned)ceil_div(ta.a.dim, 32 * Lane<T>::E);
    constexpr size_t fs = LOADS == kDirect ? 0 : Ring<GATE ? 3 : 2, kFwdStages, kFwdSteps>::bytes;
    constexpr size_t bs = LOADS == kDirect ? 0 : Ring<GATE ? 4 : 3, kBwdStages, kBwdSteps>::bytes;
    if (bwd)
        return launch_kernel<bwd_kernel<T, GATE, RESET, LOADS, kBwdStages, kBwdSteps>>(
            ta, tiles, bs, st, "gated_linear_recurrence bwd");
    return launch_kernel<fwd_kernel<T, GATE, RESET, LOADS, kFwdStages, kFwdSteps>>(
        ta, tiles, fs, st, "gated_linear_recurrence fwd");
}

template <typename T, bool GATE, bool RESET>
static int launch_loads(TmaArgs& ta, bool bwd, int loads, cudaStream_t st) {
    if (loads == kTma) return launch<T, GATE, RESET, kTma>(ta, bwd, st);
    if (loads == kWords || sizeof(T) == 4) return launch<T, GATE, RESET, kWords>(ta, bwd, st);
    if constexpr (sizeof(T) == 2) return launch<T, GATE, RESET, kDirect>(ta, bwd, st);
    return SSM_OK;
}

template <typename T>
static int launch_gate(TmaArgs& ta, bool bwd, int loads, cudaStream_t st) {
    if (ta.a.reset)
        return ta.a.z ? launch_loads<T, true, true>(ta, bwd, loads, st) : launch_loads<T, false, true>(ta, bwd, loads, st);
    return ta.a.z ? launch_loads<T, true, false>(ta, bwd, loads, st) : launch_loads<T, false, false>(ta, bwd, loads, st);
}

static int launch_any(const ssm_gated_recurrence_params* p, const Args& a, bool bwd, cudaStream_t st,
                      int* cluster = nullptr) {
    TmaArgs ta{};
    ta.a = a;
    const bool tma = tma_ok(a, p->dtype, bwd);
    const int loads = !a.words ? kDirect : tma ? kTma : kWords;
    const int chunk = kWarps * (bwd ? kBwdSteps : kFwdSteps);
    if (tma) {
        if (int s = ensure_context("gated_linear_recurrence")) return s;
        if (int s = encode(&ta.m[0], a.x, a.xt, a.xb, p->dtype, chunk, a)) return s;
        if (int s = encode(&ta.m[1], a.forget, a.ft, a.fb, p->dtype, chunk, a)) return s;
        if (a.z)
            if (int s = encode(&ta.m[2], a.z, a.zt, a.zb, p->dtype, chunk, a)) return s;
        if (bwd)
            if (int s = encode(&ta.m[3], a.dy, a.dyt, a.dyb, p->dtype, chunk, a)) return s;
    }
    const int s = p->dtype == SSM_F32 ? launch_gate<float>(ta, bwd, loads, st)
                  : p->dtype == SSM_BF16 ? launch_gate<__nv_bfloat16>(ta, bwd, loads, st)
                                         : launch_gate<__half>(ta, bwd, loads, st);
    if (cluster) *cluster = ta.cluster;
    return s;
}

template <typename T>
static void launch_step(const StepArgs& a, cudaStream_t st) {
    const unsigned grid = (unsigned)ceil_div(a.batch * a.lanes, kThreads);
    if (a.z) step_kernel<T, true><<<grid, kThreads, 0, st>>>(a);
    else step_kernel<T, false><<<grid, kThreads, 0, st>>>(a);
}

}  // namespace glr
}  // namespace ssm

using namespace ssm;
using namespace ssm::glr;

// The kernels' error flag on the current device, read and cleared; called by
// ssm_take_kernel_error.
int ssm_glr_take_error() {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, ssm::glr::g_glr_error, sizeof(int)) != cudaSuccess) return -1;
    if (v) {
        const int zero = 0;
        cudaMemcpyToSymbol(ssm::glr::g_glr_error, &zero, sizeof(int));
    }
    return v;
}

extern "C" int ssm_gated_recurrence_sizes(const ssm_gated_recurrence_params* p, size_t* states_bytes,
                                          size_t* workspace_bytes) {
    if (int s = validate(p)) return s;
    if (states_bytes) *states_bytes = (size_t)(p->batch * ceil_div(p->length, kWarps * kBwdSteps) * p->dim) * 4;
    if (workspace_bytes) *workspace_bytes = (size_t)(p->batch * kMaxCluster * p->dim) * 4;
    return SSM_OK;
}

extern "C" int ssm_gated_recurrence_fwd(const ssm_gated_recurrence_params* p, void* stream) {
    if (int s = validate(p)) return s;
    if (p->batch == 0) return SSM_OK;
    if (!p->final_state || (p->length && (!p->x || !p->forget || !p->y)))
        return fail(SSM_ERR_INVALID, "gated_linear_recurrence fwd: null pointer");
    return launch_any(p, args_of(p, false), false, static_cast<cudaStream_t>(stream));
}

extern "C" int ssm_gated_recurrence_bwd(const ssm_gated_recurrence_params* p, void* stream) {
    if (int s = validate(p)) return s;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (p->batch == 0) {
        if (p->dlower && cudaMemsetAsync(p->dlower, 0, (size_t)p->dim * 4, st))
            return check_launch("gated_linear_recurrence bwd: zero dlower");
        return SSM_OK;
    }
    if (p->length && (!p->x || !p->forget || !p->dy || !p->states || !p->dx || !p->dforget || (p->z && !p->dz)))
        return fail(SSM_ERR_INVALID, "gated_linear_recurrence bwd: null pointer");
    Args a = args_of(p, true);
    if (p->dlower) {
        size_t need = 0;
        ssm_gated_recurrence_sizes(p, nullptr, &need);
        if (!p->workspace || p->workspace_bytes < need)
            return fail(SSM_ERR_WORKSPACE, "gated_linear_recurrence bwd: workspace smaller than ssm_gated_recurrence_sizes");
        a.part = static_cast<float*>(p->workspace);
    }
    int cluster = 1;
    if (int s = launch_any(p, a, true, st, &cluster)) return s;
    if (p->dlower) {
        fold_kernel<<<(unsigned)ceil_div(a.dim, 256), 256, 0, st>>>(a.part, a.batch * cluster, a.dim, p->dlower);
        return check_launch("gated_linear_recurrence bwd: fold");
    }
    return SSM_OK;
}

extern "C" int ssm_gated_recurrence_step(const ssm_gated_recurrence_step_params* p, void* stream) {
    if (p == nullptr) return fail(SSM_ERR_INVALID, "gated_linear_recurrence_update: null params");
    if (p->batch < 0 || p->dim < 1) return fail(SSM_ERR_INVALID, "gated_linear_recurrence_update: batch and dim");
    if (p->dtype < SSM_F32 || p->dtype > SSM_F16)
        return fail(SSM_ERR_UNSUPPORTED, "gated_linear_recurrence_update: dtype");
    if (p->batch > INT32_MAX || p->dim > INT32_MAX || p->batch * p->dim > ((int64_t)1 << 38))
        return fail(SSM_ERR_UNSUPPORTED, "gated_linear_recurrence_update: too large");
    if (p->batch == 0) return SSM_OK;
    if (!p->x || !p->forget || !p->state || !p->y)
        return fail(SSM_ERR_INVALID, "gated_linear_recurrence_update: null pointer");
    StepArgs a{};
    a.batch = p->batch; a.dim = p->dim;
    auto row = [&](int64_t s) { return s ? s : p->dim; };
    a.xb = row(p->x_batch_stride); a.fb = row(p->forget_batch_stride); a.zb = row(p->z_batch_stride);
    a.sb = row(p->state_batch_stride);
    for (int64_t s : {a.xb, a.fb, a.zb, a.sb})
        if (s < p->dim) return fail(SSM_ERR_INVALID, "gated_linear_recurrence_update: a batch stride is below dim");
    a.x = p->x; a.forget = p->forget; a.z = p->z; a.lower = p->lower; a.state = p->state; a.y = p->y;
    a.lanes = ceil_div(p->dim * esize(p->dtype), 4);
    a.words = 1;
    if (p->dtype != SSM_F32) {
        for (const void* q : {p->x, p->forget, p->z, (const void*)p->y}) if (!al(q, 4)) a.words = 0;
        for (int64_t s : {a.dim, a.xb, a.fb, p->z ? a.zb : 0}) if (s & 1) a.words = 0;
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (p->dtype == SSM_F32) launch_step<float>(a, st);
    else if (p->dtype == SSM_BF16) launch_step<__nv_bfloat16>(a, st);
    else launch_step<__half>(a, st);
    return check_launch("gated_linear_recurrence_update");
}
