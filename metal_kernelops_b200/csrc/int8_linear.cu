// Linear layer in 8-bit integers for sm_100a:
//     out[m, n] = x_scale[m] w_scale[n] sum_k x[m, k] w[n, k] (+ bias[n])
// x (tokens, K) and w (features, K) int8 rows, the sum exact in int32 (K is at
// most 131071, so that 128 * 128 * K stays below 2^31), the two scales and the
// bias applied in fp32, one rounding to the output's type.
//
// The products run on the fifth-generation tensor cores (kind::i8), operands staged
// by TMA in the 128-byte swizzle, int32 accumulators in tensor memory.  Rows past the
// end and the last bytes of K arrive as zeros.  TMA wants rows on 16-byte
// boundaries: operands that are not are first copied to such rows in the workspace.
//
// Few tokens: reading w once is the whole cost.  `skinny_kernel` makes the features
// the 128 rows of the product and the tokens its columns (16 to 128), and cuts K
// over the CTAs of a cluster until the GPU is full; the slices' int32 sums are added
// through distributed shared memory, exactly, so the cut changes no result.
//
// Many tokens: `wide_kernel`, a persistent pair of CTAs per 256 x 256 tile
// (cta_group::2: each CTA loads 128 rows of either operand and keeps 128 token rows
// of the sums).  A 128 x 256 tile on one CTA would fetch 96 bytes a clock from L2 to
// feed its tensor core at the int8 rate, the pair fetches 64.  Warp-specialised: one
// warp loads, one multiplies, four write the previous tile out from the other half
// of tensor memory.
#include <cooperative_groups.h>
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <mutex>

#include "common.cuh"
#include "tc.cuh"

namespace ssm {
namespace i8 {

constexpr int kBlockK = 128;                        // bytes of K a stage holds: one swizzle row
constexpr int kFeatures = 128;                      // features of a skinny tile
constexpr int kMaxStages = 8;

struct Args {
    int64_t tokens, features, k;
    const float* xs; const float* ws; const float* bias;
    void* out;
    int vec, vec4;                                  // stores of 32 bytes, of four elements are aligned
    int* status;
};
struct TmaArgs {
    Args a;
    alignas(64) CUtensorMap mx, mw;
    int stages;
};

__device__ int g_i8_error;

__device__ __forceinline__ void report(const Args& a, int code) {
    atomicCAS(&g_i8_error, 0, code);
    if (a.status) atomicCAS(a.status, 0, code);
}

// Shared-memory descriptor of K-major rows of 128 bytes in the 128-byte swizzle:
// eight rows make an atom of 1024 bytes, the next eight follow.
__device__ __forceinline__ uint64_t sdesc_sw128(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)2 << 61;
}
// Instruction descriptor of kind::i8: signed 8-bit A and B, both K-major, int32 D.
__host__ __device__ constexpr uint32_t idesc_i8(uint32_t M, uint32_t N) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((N >> 3) << 17) | ((M >> 4) << 24);
}
__device__ __forceinline__ void mma_i8(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n"
        :: "r"(d_tmem), "l"(a), "l"(b), "r"(idesc), "r"(accum));
}
// 32 lanes x 16 columns of int32; wait_ld orders the registers' uses after the wait.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, int* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void wait_ld16(int* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :: "memory");
}

__device__ __forceinline__ uint32_t at_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ int4 ld_remote(uint32_t addr, uint32_t rank) {
    int4 v;
    asm volatile("ld.shared::cluster.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at_rank(addr, rank)) : "memory");
    return v;
}
template <typename O> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Four results of one token row.
template <typename O>
__device__ __forceinline__ void write4(const Args& a, O* row, int64_t f, float v0, float v1, float v2, float v3) {
    if (f + 4 <= a.features && a.vec4) {
        if constexpr (sizeof(O) == 4) *reinterpret_cast<float4*>(row + f) = make_float4(v0, v1, v2, v3);
        else *reinterpret_cast<uint2*>(row + f) = make_uint2(pack2<O>(v0, v1), pack2<O>(v2, v3));
    } else {
        if (f < a.features) stf(row + f, v0);
        if (f + 1 < a.features) stf(row + f + 1, v1);
        if (f + 2 < a.features) stf(row + f + 2, v2);
        if (f + 3 < a.features) stf(row + f + 3, v3);
    }
}

// ------------------------------------------------------------ few tokens --
template <int NT>
struct Skinny {
    static constexpr int kStage = kFeatures * kBlockK + NT * kBlockK;     // bytes: w rows, then x rows
    static constexpr uint32_t kTmem = NT < 32 ? 32 : NT;
    static size_t smem(int stages) { return (size_t)stages * kStage + 1024; }
    // the sums pass through the stages' memory
    static int min_stages() { return (NT * kFeatures * 4 + kStage - 1) / kStage; }
    // where the choice of stages begins (about 72 KB) and ends
    static int first_stages() { return std::max({min_stages(), 2, (72 << 10) / kStage}); }
    static int last_stages() { return std::max(first_stages(), std::min(kMaxStages, (200 << 10) / kStage)); }
};

// Grid: (feature tiles * C, token tiles); a cluster's C CTAs share a tile, each with
// its slice of K.  Warp 0 loads, warp 1 multiplies, all four write out.
template <typename O, int NT>
__global__ void __launch_bounds__(128)
skinny_kernel(const __grid_constant__ TmaArgs ta) {
    using L = Skinny<NT>;
    const Args& a = ta.a;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024 - (tc::smem_u32(smem_raw) & 1023)) & 1023);
    __shared__ uint64_t full[kMaxStages], empty[kMaxStages], done;
    __shared__ uint32_t tmem_at;
    const auto cluster = cooperative_groups::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t f0 = (int64_t)(blockIdx.x / C) * kFeatures, m0 = (int64_t)blockIdx.y * NT;
    const int stages = ta.stages;
    const int blocks = (int)((a.k + kBlockK - 1) / kBlockK);
    const int kb0 = (int)((int64_t)blocks * rank / C), kb1 = (int)((int64_t)blocks * (rank + 1) / C);
    const int nk = kb1 - kb0;
    auto load = [&](int i) {
        const int s = i % stages;
        const uint32_t bar = tc::smem_u32(&full[s]), at = tc::smem_u32(smem + (size_t)s * L::kStage);
        tc::mbar_expect_tx(bar, L::kStage);
        tc::tma_load2(at, &ta.mw, (kb0 + i) * kBlockK, (int)f0, bar);
        tc::tma_load2(at + kFeatures * kBlockK, &ta.mx, (kb0 + i) * kBlockK, (int)m0, bar);
    };
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            tc::mbar_init(tc::smem_u32(&full[s]), 1);
            tc::mbar_init(tc::smem_u32(&empty[s]), 1);
        }
        tc::mbar_init(tc::smem_u32(&done), 1);
        tc::fence_mbar_init();
        // the ring's first loads go out before the CTA has its tensor memory
        for (int i = 0; i < stages && i < nk; ++i) load(i);
    }
    if (warp == 1) tc::tmem_alloc(tc::smem_u32(&tmem_at), L::kTmem);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = tmem_at;
    int loads = nk < stages ? nk : stages;              // thread 0's, so far
    bool ok = true;
    if (warp == 0 && lane == 0) {
        for (; loads < nk; ++loads) {
            if (!tc::mbar_wait(tc::smem_u32(&empty[loads % stages]), (uint32_t)(loads / stages - 1) & 1u)) {
                report(a, 121);
                ok = false;
                break;
            }
            load(loads);
        }
    } else if (warp == 1 && lane == 0) {
        for (int i = 0; i < nk; ++i) {
            const int s = i % stages;
            if (!tc::mbar_wait(tc::smem_u32(&full[s]), (uint32_t)(i / stages) & 1u)) {
                report(a, 122);
                ok = false;
                break;
            }
            tc::fence_after();
            const uint32_t at = tc::smem_u32(smem + (size_t)s * L::kStage);
            const uint64_t dw = sdesc_sw128(at), dx = sdesc_sw128(at + kFeatures * kBlockK);
#pragma unroll
            for (int j = 0; j < kBlockK / 32; ++j)          // 32 bytes of K an instruction: two 16-byte units
                mma_i8(tmem, dw + 2 * j, dx + 2 * j, idesc_i8(kFeatures, NT), i || j);
            tc::commit(tc::smem_u32(&empty[s]));
        }
        tc::commit(tc::smem_u32(&done));
    }
    __syncwarp();
    if (!tc::mbar_wait(tc::smem_u32(&done), 0)) {
        if (lane == 0) report(a, 123);
        ok = false;
    }
    // a wait has given up: no copy may land in a CTA that has ended, and nothing is written
    ok = __syncthreads_and(ok);
    if (!ok && threadIdx.x == 0)
        for (int i = loads > stages ? loads - stages : 0; i < loads; ++i)
            tc::mbar_wait(tc::smem_u32(&full[i % stages]), (uint32_t)(i / stages) & 1u);
    tc::fence_after();
    // tensor memory (lane: feature, column: token) to shared memory (token, feature)
    const int live = ok ? (int)min64(NT, a.tokens - m0) : 0;
    int* part = reinterpret_cast<int*>(smem);
    for (int c0 = 0; c0 < live; c0 += 16) {
        int acc[16];
        tmem_ld16(tmem + ((uint32_t)warp << 21) + c0, acc); // lanes 32 warp ..., columns c0 ...
        wait_ld16(acc);
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (c0 + j < live) part[(c0 + j) * kFeatures + threadIdx.x] = acc[j];
    }
    if (C > 1) cluster.sync();
    else __syncthreads();
    // a thread: four features of every (4 C)-th token, the slices of K added
    const int64_t f = f0 + lane * 4;
    float ws[4], bias[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        ws[j] = f + j < a.features ? a.ws[f + j] : 0.0f;
        bias[j] = f + j < a.features && a.bias ? a.bias[f + j] : 0.0f;
    }
    const uint32_t mine = tc::smem_u32(part + lane * 4);
#pragma unroll 2
    for (int m = rank * 4 + warp; m < live; m += 4 * C) {
        const float xs = a.xs[m0 + m];
        int4 v[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            v[r] = make_int4(0, 0, 0, 0);
            if (r < C) v[r] = ld_remote(mine + m * kFeatures * 4, r);
        }
        int4 s = v[0];
#pragma unroll
        for (int r = 1; r < 8; ++r) { s.x += v[r].x; s.y += v[r].y; s.z += v[r].z; s.w += v[r].w; }
        write4<O>(a, static_cast<O*>(a.out) + (m0 + m) * a.features, f, fmaf((float)s.x * xs, ws[0], bias[0]),
                  fmaf((float)s.y * xs, ws[1], bias[1]), fmaf((float)s.z * xs, ws[2], bias[2]),
                  fmaf((float)s.w * xs, ws[3], bias[3]));
    }
    if (C > 1) cluster.sync();                              // the peers have read this CTA's sums
    tc::fence_before();
    __syncthreads();
    if (warp == 1) tc::tmem_dealloc(tmem, L::kTmem);
}

// ----------------------------------------------------------- many tokens --
constexpr int kTileM = 256, kTileN = 256;           // a CTA pair's tile
constexpr int kWideStage = 2 * 128 * kBlockK;       // bytes a CTA stages: 128 token rows, 128 feature rows
constexpr int kWideStages = 6;
constexpr size_t kWideSmem = (size_t)kWideStages * kWideStage + 1024;
constexpr int kWideThreads = 256;

// A load into this CTA's shared memory that counts its bytes on a barrier of the pair.
__device__ __forceinline__ void pair_load(uint32_t dst, const void* map, int c0, int c1, uint32_t mbar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
        "[%0], [%1, {%2, %3}], [%4];"
        :: "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(mbar) : "memory");
}
__device__ __forceinline__ void pair_mma(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n"
        :: "r"(d_tmem), "l"(a), "l"(b), "r"(idesc), "r"(accum));
}
// Arrive on the barrier at this offset in both CTAs once the MMAs issued so far are done.
__device__ __forceinline__ void pair_commit(uint32_t mbar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
        :: "r"(mbar), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void arrive_at(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" :: "r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, int* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void st32(void* p, const uint32_t* w) {       // 32 bytes, 32-byte aligned
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 :: "l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}
// 32 results of one token row at out + (columns f ... f + 31 of the features).
template <typename O>
__device__ __forceinline__ void write32(const Args& a, O* row, int64_t f, const float* v) {
    if (f + 32 <= a.features && a.vec) {
        uint32_t w[8];
        constexpr int per = 32 / sizeof(O);
#pragma unroll
        for (int i = 0; i < 32; i += per) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if constexpr (sizeof(O) == 4) w[j] = __float_as_uint(v[i + j]);
                else w[j] = pack2<O>(v[i + 2 * j], v[i + 2 * j + 1]);
            }
            st32(row + f + i, w);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (f + i < a.features) stf(row + f + i, v[i]);
    }
}

template <typename O>
__global__ void __launch_bounds__(kWideThreads, 1)
wide_kernel(const __grid_constant__ TmaArgs ta) {
    const Args& a = ta.a;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024 - (tc::smem_u32(smem_raw) & 1023)) & 1023);
    __shared__ uint64_t full[kWideStages], empty[kWideStages], tfull[2], tempty[2];
    __shared__ __align__(16) float cols[2][kTileN];          // the tile's feature scales and biases
    __shared__ uint32_t tmem_at;
    const auto cluster = cooperative_groups::this_cluster();
    const uint32_t rank = cluster.block_rank();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t mt = (a.tokens + kTileM - 1) / kTileM, nt = (a.features + kTileN - 1) / kTileN, tiles = mt * nt;
    const int64_t first = blockIdx.x / 2, step = gridDim.x / 2;
    const int nk = (int)((a.k + kBlockK - 1) / kBlockK);
    if (threadIdx.x == 0) {
        for (int s = 0; s < kWideStages; ++s) {
            tc::mbar_init(tc::smem_u32(&full[s]), 1);
            tc::mbar_init(tc::smem_u32(&empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            tc::mbar_init(tc::smem_u32(&tfull[b]), 1);
            tc::mbar_init(tc::smem_u32(&tempty[b]), 8);      // four warps of either CTA
        }
        tc::fence_mbar_init();
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;"
                     :: "r"(tc::smem_u32(&tmem_at)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc::fence_before();
    cluster.sync();
    tc::fence_after();
    const uint32_t tmem = tmem_at;

    if (warp == 0 && lane == 0) {
        // loads: either CTA its own 128 rows of both operands, counted on the first CTA's barrier
        int64_t it = 0;
        bool ok = true;
        for (int64_t tile = first; tile < tiles && ok; tile += step) {
            const int m0 = (int)(tile / nt * kTileM + rank * 128), n0 = (int)(tile % nt * kTileN + rank * 128);
            for (int kb = 0; kb < nk; ++kb, ++it) {
                const int s = (int)(it % kWideStages);
                if (it >= kWideStages &&
                    !tc::mbar_wait(tc::smem_u32(&empty[s]), (uint32_t)(it / kWideStages - 1) & 1u)) {
                    report(a, 131);
                    ok = false;
                    break;
                }
                const uint32_t bar = tc::smem_u32(&full[s]), at = tc::smem_u32(smem + (size_t)s * kWideStage);
                if (rank == 0) tc::mbar_expect_tx(bar, 2 * kWideStage);
                const uint32_t lead = at_rank(bar, 0);
                pair_load(at, &ta.mx, kb * kBlockK, m0, lead);
                pair_load(at + 128 * kBlockK, &ta.mw, kb * kBlockK, n0, lead);
            }
        }
        // every stage's last use is over before the CTA may end
        for (int64_t i = max64(0, it - kWideStages); ok && i < it; ++i)
            if (!tc::mbar_wait(tc::smem_u32(&empty[i % kWideStages]), (uint32_t)(i / kWideStages) & 1u)) {
                report(a, 132);
                ok = false;
            }
        // a wait has given up: the pair's copies, which count on the first CTA's barriers, land before either ends
        if (!ok && rank == 0)
            for (int64_t i = max64(0, it - kWideStages); i < it; ++i)
                tc::mbar_wait(tc::smem_u32(&full[i % kWideStages]), (uint32_t)(i / kWideStages) & 1u);
    } else if (warp == 1 && lane == 0 && rank == 0) {
        int64_t it = 0;
        int64_t n = 0;
        bool ok = true;
        for (int64_t tile = first; tile < tiles && ok; tile += step, ++n) {
            const int b = (int)(n & 1);
            if (n >= 2 && !tc::mbar_wait(tc::smem_u32(&tempty[b]), (uint32_t)(n / 2 - 1) & 1u)) {
                report(a, 133);
                break;
            }
            tc::fence_after();
            for (int kb = 0; kb < nk; ++kb, ++it) {
                const int s = (int)(it % kWideStages);
                if (!tc::mbar_wait(tc::smem_u32(&full[s]), (uint32_t)(it / kWideStages) & 1u)) {
                    report(a, 134);
                    ok = false;
                    break;
                }
                tc::fence_after();
                const uint32_t at = tc::smem_u32(smem + (size_t)s * kWideStage);
                const uint64_t dx = sdesc_sw128(at), dw = sdesc_sw128(at + 128 * kBlockK);
#pragma unroll
                for (int j = 0; j < kBlockK / 32; ++j)
                    pair_mma(tmem + b * kTileN, dx + 2 * j, dw + 2 * j, idesc_i8(kTileM, kTileN), kb || j);
                pair_commit(tc::smem_u32(&empty[s]));
            }
            pair_commit(tc::smem_u32(&tfull[b]));
        }
    } else if (warp >= 4) {
        // a wait that gave up is not tried again, so that the named barriers below stay in step
        const int et = threadIdx.x - 128, ew = warp - 4;
        int64_t n = 0;
        bool ok = true;
        for (int64_t tile = first; tile < tiles; tile += step, ++n) {
            const int b = (int)(n & 1);
            const int64_t m = tile / nt * kTileM + rank * 128 + et, n0 = tile % nt * kTileN;
            asm volatile("bar.sync 1, 128;" ::: "memory");       // the previous tile's scales are read
            for (int i = et; i < kTileN; i += 128) {
                const int64_t f = n0 + i;
                cols[0][i] = f < a.features ? a.ws[f] : 0.0f;
                cols[1][i] = f < a.features && a.bias ? a.bias[f] : 0.0f;
            }
            const float xs = m < a.tokens ? a.xs[m] : 0.0f;
            asm volatile("bar.sync 1, 128;" ::: "memory");
            if (ok && !tc::mbar_wait(tc::smem_u32(&tfull[b]), (uint32_t)(n / 2) & 1u)) {
                if (lane == 0) report(a, 135);
                ok = false;
            }
            __syncwarp();
            tc::fence_after();
            O* row = static_cast<O*>(a.out) + m * a.features;
#pragma unroll 1
            for (int c0 = 0; c0 < kTileN; c0 += 32) {
                int acc[32];
                tmem_ld32(tmem + b * kTileN + c0 + ((uint32_t)ew << 21), acc);
                wait_ld16(acc);
                wait_ld16(acc + 16);
                if (c0 + 32 == kTileN) {
                    tc::fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_at(at_rank(tc::smem_u32(&tempty[b]), 0));
                }
                float v[32];
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    const float4 w = *reinterpret_cast<const float4*>(&cols[0][c0 + i]);
                    const float4 bb = *reinterpret_cast<const float4*>(&cols[1][c0 + i]);
                    v[i] = fmaf((float)acc[i] * xs, w.x, bb.x);
                    v[i + 1] = fmaf((float)acc[i + 1] * xs, w.y, bb.y);
                    v[i + 2] = fmaf((float)acc[i + 2] * xs, w.z, bb.z);
                    v[i + 3] = fmaf((float)acc[i + 3] * xs, w.w, bb.w);
                }
                if (m < a.tokens && ok) write32<O>(a, row, n0 + c0, v);
            }
        }
    }
    __syncwarp();
    tc::fence_before();
    cluster.sync();
    if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" :: "r"(tmem) : "memory");
}

// Rows of K bytes at any stride to rows of `padded` bytes (a multiple of 16).
__global__ void pack_kernel(const int8_t* src, int64_t stride, int8_t* dst, int64_t padded, int64_t rows, int64_t k) {
    const int64_t words = padded / 4, n = rows * words;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t r = i / words, c = (i % words) * 4;
        const int8_t* p = src + r * stride + c;
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c + j < k) w |= (uint32_t)(uint8_t)p[j] << (8 * j);
        *reinterpret_cast<uint32_t*>(dst + r * padded + c) = w;
    }
}

// ------------------------------------------------------------------- host ----
constexpr int64_t kMaxK = 131071;

static bool al(const void* p, int64_t b) { return (reinterpret_cast<uintptr_t>(p) % b) == 0; }

static int validate(const ssm_int8_linear_params* p) {
    if (p == nullptr) return fail(SSM_ERR_INVALID, "int8_linear: null params");
    if (p->tokens < 0 || p->in_features < 1 || p->out_features < 1)
        return fail(SSM_ERR_INVALID, "int8_linear: tokens, in_features and out_features");
    if (p->in_features > kMaxK)
        return fail(SSM_ERR_UNSUPPORTED, "int8_linear: in_features above 131071 (the int32 sums could overflow)");
    // tile coordinates are 32-bit, a tile's overhang included
    if (p->tokens > INT32_MAX - 1024 || p->out_features > INT32_MAX - 1024)
        return fail(SSM_ERR_UNSUPPORTED, "int8_linear: more than 2^31 - 1025 tokens or out_features");
    if (p->out_dtype < SSM_F32 || p->out_dtype > SSM_F16) return fail(SSM_ERR_UNSUPPORTED, "int8_linear: out_dtype");
    if ((p->x_row_stride && p->x_row_stride < p->in_features) || (p->w_row_stride && p->w_row_stride < p->in_features))
        return fail(SSM_ERR_INVALID, "int8_linear: a row stride is below in_features");
    return SSM_OK;
}

static int64_t padded(int64_t k) { return (k + 15) / 16 * 16; }
static bool rows_ok(const void* p, int64_t stride, int64_t rows) {
    return al(p, 16) && (rows == 1 || stride % 16 == 0) && stride < ((int64_t)1 << 40);
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

static int encode(CUtensorMap* m, const void* base, int64_t k, int64_t rows, int64_t stride, int box_rows) {
    if (!encoder()) return fail(SSM_ERR_CUDA, "int8_linear: cuTensorMapEncodeTiled unavailable");
    cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)(rows == 1 ? padded(k) : stride)};    // one row: never used
    cuuint32_t box[2] = {kBlockK, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    const CUresult r = encoder()(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                                 CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r == CUDA_SUCCESS) return SSM_OK;
    return fail(SSM_ERR_CUDA, "int8_linear: cuTensorMapEncodeTiled failed (" + std::to_string((int)r) + ")");
}

// How many clusters of C CTAs with S stages each the GPU holds at once.  The
// occupancy query counts kernels that allocate tensor memory as one CTA an SM; shared
// and tensor memory say how many more share it.
template <typename O, int NT>
static int64_t clusters_at_once(int S, int C) {
    static std::atomic<int> alone[9];                // with one CTA an SM; 0: not asked yet
    if (alone[C] == 0) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(C);
        cfg.blockDim = dim3(128);
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = C;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, skinny_kernel<O, NT>, &cfg) != cudaSuccess || n < 1) {
            cudaGetLastError();
            n = 128 / C;
        }
        alone[C] = n;
    }
    // 228 KB an SM; a CTA also has its barriers and 1 KB of the system's
    const int64_t by_smem = (228 << 10) / (int64_t)(Skinny<NT>::smem(S) + 2048);
    return alone[C] * max64(1, min64(by_smem, 512 / Skinny<NT>::kTmem));
}

template <typename O, int NT>
static int launch_skinny(TmaArgs& ta, cudaStream_t st) {
    using L = Skinny<NT>;
    const Args& a = ta.a;
    const int64_t ftiles = ceil_div(a.features, kFeatures), mtiles = ceil_div(a.tokens, NT);
    const int64_t blocks = ceil_div(a.k, kBlockK);
    // As many K slices as let every cluster run at once (at most eight, at least two
    // blocks each), with about 72 KB of stages a CTA; then more stages while all still
    // fit.  One cluster too many costs a second wave: 1 x 2560 -> 12368 takes 10.1 us with
    // three slices of four stages, 14.9 us with six stages, of which one of the 97
    // clusters has to wait; 11.5 us uncut.
    const int64_t tiles = ftiles * mtiles;
    auto fits = [&](int s, int c) { return tiles <= clusters_at_once<O, NT>(s, c); };
    int S = L::first_stages(), C = 1;
    while (C < 8 && blocks >= 2 * (C + 1) && fits(S, C + 1)) ++C;
    while (S < L::last_stages() && (int64_t)S * C < blocks && fits(S + 1, C)) ++S;
    ta.stages = S;
    const size_t smem = L::smem(ta.stages);
    // the limit belongs to the kernel, not to this call: one value for every call, so that
    // another thread's cannot lower it before this launch
    if (cudaFuncSetAttribute(skinny_kernel<O, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)L::smem(L::last_stages())) != cudaSuccess)
        return check_launch("int8_linear");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(ftiles * C), (unsigned)mtiles);
    cfg.blockDim = dim3(128);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = C;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, skinny_kernel<O, NT>, ta);
    return check_launch("int8_linear");
}

template <typename O>
static int launch_few(TmaArgs& ta, int nt, cudaStream_t st) {
    switch (nt) {
        case 16: return launch_skinny<O, 16>(ta, st);
        case 32: return launch_skinny<O, 32>(ta, st);
        case 64: return launch_skinny<O, 64>(ta, st);
        default: return launch_skinny<O, 128>(ta, st);
    }
}

template <typename O>
static int launch_wide(TmaArgs& ta, cudaStream_t st) {
    const Args& a = ta.a;
    const int64_t tiles = ceil_div(a.tokens, kTileM) * ceil_div(a.features, kTileN);
    if (cudaFuncSetAttribute(wide_kernel<O>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kWideSmem) != cudaSuccess)
        return check_launch("int8_linear");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(2 * min64(tiles, 148 / 2)));
    cfg.blockDim = dim3(kWideThreads);
    cfg.dynamicSmemBytes = kWideSmem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 2;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, wide_kernel<O>, ta);
    return check_launch("int8_linear");
}

// From this many tokens on the wide kernel runs: with 2560 -> 12368, whose tiles fill the
// GPU, the skinny one takes 19.4 us at 256 tokens, 22.8 at 257 and 26.4 at 400, the wide one 18.2 at 257 and 19.9 at
// 400.  Narrow layers, whose tiles do not, would do better with the skinny one for longer: 300 x 5120
// -> 2560 14.5 us (wide 17.9), 512 tokens 16.8 (18.2), 1024 tokens 24.0 (18.3); 300 x 8192 -> 256 10.8 (24.9).
constexpr int64_t kWideTokens = 257;

}  // namespace i8
}  // namespace ssm

using namespace ssm;
using namespace ssm::i8;

// The kernels' error flag on the current device, read and cleared; called by
// ssm_take_kernel_error.
int ssm_i8_take_error() {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, ssm::i8::g_i8_error, sizeof(int)) != cudaSuccess) return -1;
    if (v) {
        const int zero = 0;
        cudaMemcpyToSymbol(ssm::i8::g_i8_error, &zero, sizeof(int));
    }
    return v;
}

extern "C" int ssm_int8_linear_sizes(const ssm_int8_linear_params* p, size_t* workspace_bytes) {
    if (int s = validate(p)) return s;
    const int64_t xs = p->x_row_stride ? p->x_row_stride : p->in_features;
    const int64_t ws = p->w_row_stride ? p->w_row_stride : p->in_features;
    size_t need = 0;
    if (!rows_ok(p->x, xs, p->tokens)) need += align_up((size_t)(p->tokens * padded(p->in_features)), 256);
    if (!rows_ok(p->w, ws, p->out_features)) need += align_up((size_t)(p->out_features * padded(p->in_features)), 256);
    if (workspace_bytes) *workspace_bytes = need;
    return SSM_OK;
}

extern "C" int ssm_int8_linear_fwd(const ssm_int8_linear_params* p, void* stream) {
    if (int s = validate(p)) return s;
    if (p->tokens == 0) return SSM_OK;
    if (!p->x || !p->x_scale || !p->w || !p->w_scale || !p->out)
        return fail(SSM_ERR_INVALID, "int8_linear: null pointer");
    size_t need = 0;
    ssm_int8_linear_sizes(p, &need);
    if (need && (!p->workspace || p->workspace_bytes < need || !al(p->workspace, 16)))
        return fail(SSM_ERR_WORKSPACE, "int8_linear: workspace smaller than ssm_int8_linear_sizes");
    if (int s = ensure_context("int8_linear")) return s;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int8_t* x = p->x;
    const int8_t* w = p->w;
    int64_t xs = p->x_row_stride ? p->x_row_stride : p->in_features;
    int64_t ws = p->w_row_stride ? p->w_row_stride : p->in_features;
    int8_t* room = static_cast<int8_t*>(p->workspace);
    const int64_t k = p->in_features, kp = padded(k);
    auto pack = [&](const int8_t*& src, int64_t& stride, int64_t rows) {
        pack_kernel<<<(unsigned)min64(ceil_div(rows * kp / 4, 256), 148 * 16), 256, 0, st>>>(src, stride, room, kp, rows, k);
        src = room;
        stride = kp;
        room += align_up((size_t)(rows * kp), 256);
        return check_launch("int8_linear: pack");
    };
    if (!rows_ok(x, xs, p->tokens))
        if (int s = pack(x, xs, p->tokens)) return s;
    if (!rows_ok(w, ws, p->out_features))
        if (int s = pack(w, ws, p->out_features)) return s;
    TmaArgs ta{};
    Args& a = ta.a;
    a.tokens = p->tokens; a.features = p->out_features; a.k = k;
    a.xs = p->x_scale; a.ws = p->w_scale; a.bias = p->bias;
    a.out = p->out;
    const int64_t es = p->out_dtype == SSM_F32 ? 4 : 2;
    a.vec = al(p->out, 32) && (a.features * es) % 32 == 0;
    a.vec4 = al(p->out, 4 * es) && a.features % 4 == 0;
    a.status = p->status;
    if (a.tokens >= kWideTokens) {
        if (int s = encode(&ta.mx, x, k, a.tokens, xs, 128)) return s;
        if (int s = encode(&ta.mw, w, k, a.features, ws, 128)) return s;
        if (p->out_dtype == SSM_F32) return launch_wide<float>(ta, st);
        return p->out_dtype == SSM_BF16 ? launch_wide<__nv_bfloat16>(ta, st) : launch_wide<__half>(ta, st);
    }
    const int nt = a.tokens <= 16 ? 16 : a.tokens <= 32 ? 32 : a.tokens <= 64 ? 64 : 128;
    if (int s = encode(&ta.mx, x, k, a.tokens, xs, nt)) return s;
    if (int s = encode(&ta.mw, w, k, a.features, ws, kFeatures)) return s;
    if (p->out_dtype == SSM_F32) return launch_few<float>(ta, nt, st);
    return p->out_dtype == SSM_BF16 ? launch_few<__nv_bfloat16>(ta, nt, st) : launch_few<__half>(ta, nt, st);
}
