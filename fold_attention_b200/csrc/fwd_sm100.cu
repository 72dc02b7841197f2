// Attention forward on Blackwell tensor cores (tcgen05 + TMEM), head dim 128, bf16 or fp16:
// O and the log-sum-exp the backward consumes. One CTA owns 256 query rows of one
// head as two tiles of 128; a query row is one TMEM lane of its tile, so a row's
// maximum and sum need no shuffle.
//
//   S  = Q K^T   tcgen05.mma kind::f16, M=128 queries, N=128 keys, 8 steps of 16 channels,
//                both operands K-major from shared memory (TMA, 128-byte swizzle) -> TMEM fp32
//   P  = exp2(S c log2e - m)  by the row's thread, written over S in TMEM as packed 16-bit
//   O += P V     A = P from TMEM, B = V as stored (MN-major), 8 steps of 16 keys -> TMEM fp32
//
// The two tiles share each K/V stage and take turns on the tensor core: while one tile's
// rows are in their softmax, the other's scores or P V product run. A row's softmax
// reference only ever rises, and only when the row's maximum passed it by more than 2^8; O is
// rescaled in TMEM when a row's reference moved (skipped, with the wait for the tile's previous
// product, by warps in which no row's did).
//
// Warps: 0 TMA producer, 1 MMA issuer (owns all 512 TMEM columns), 4-7 and 8-11 the two
// tiles' softmax, O rescale and epilogue. Every wait is bounded (about a second); on expiry
// a status word is raised, nobody waits any more, TMEM is freed and the kernel returns.
// Replaces the third-party forward called at src/fold_attention/interface.py:42-44,
// :70-81 and kv_cache.py:252-262 (the algorithm is the usual online softmax; the
// schedule is this kernel's own).
#include <cuda.h>

#include <algorithm>
#include <type_traits>

#include "bwd_common.cuh"
#include "common.cuh"
#include "fold_b200.h"

namespace fold {
namespace fsm100 {

constexpr int BM = 128, BN = 128;   // a query tile, a key tile
constexpr int CTA_M = 2 * BM;       // a CTA owns two query tiles
constexpr int NTHREADS = 384;
constexpr long long WAIT_CYCLES = 1ll << 31;
constexpr long long DRAIN_CYCLES = 1ll << 22;   // two milliseconds: a copy takes microseconds
constexpr float LAZY = 8.0f;        // log2 of how far a row's maximum may pass its softmax reference before the reference moves

// shared memory map (1024-aligned base)
constexpr int SM_Q = 0;                        // 2 tiles x [2 boxes of 64 channels][128 rows][128 B]
constexpr int SM_KV = 65536;                   // 2 stages x { K 32 KB, V 32 KB }
constexpr int STAGE = 65536;
constexpr int SM_BAR = SM_KV + 2 * STAGE;
constexpr int SMEM_BYTES = SM_BAR + 256 + 1024;   // + room to align the base

enum {
    B_Q = 0,
    B_KVFULL = 1,      // [2] the stage's K and V have landed
    B_KVEMPTY = 3,     // [2] both query tiles' products with the stage retired
    B_SFULL = 5,       // [2 query tiles] the tile's scores against this key tile are in TMEM
    B_PREADY = 7,      // [2 query tiles] 128 arrivals: P is in TMEM and O is rescaled
    B_ODONE = 9,       // [2 query tiles] the tile's P V product retired
    B_COUNT = 11,
};

// TMEM columns: per query tile 128 of S (P is written over its first 64 as the row's thread
// goes), then 128 of O per tile
constexpr uint32_t T_S = 0, T_O = 256;

__device__ __forceinline__ void mbar_init(uint32_t bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// Bounded wait. `abort` (shared) is raised by whoever runs out first; once it is up
// nobody waits any more, so every role runs to its end.
__device__ __forceinline__ void mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status) {
    if (mbar_try(bar, parity)) return;
    if (*abort_flag) return;
    const long long t0 = clock64();
    for (int i = 0;; ++i) {
        if (mbar_try(bar, parity)) return;
        if ((i & 63) == 63) {
            if (*abort_flag) return;
            if (clock64() - t0 > WAIT_CYCLES) break;
        }
    }
    *abort_flag = 1;
    atomicExch(status, FOLD_ERR_TIMEOUT);
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
                 "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
                   "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
                   "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
                 "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Two fp32 FMAs per instruction and a three-input maximum (same results as the scalar forms): the
// softmax warps are what this kernel waits for.
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void fma2(float& d0, float& d1, float a0, float a1, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(pack2(a0, a1)), "l"(b), "l"(c));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(d0), "=f"(d1) : "l"(d));
}
__device__ __forceinline__ float max3f(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float ex2f(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// shared-memory matrix descriptor, 128-byte swizzle; offsets in bytes
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((addr & 0x3FFFF) >> 4);
    d |= static_cast<uint64_t>((lbo >> 4) & 0x3FFF) << 16;
    d |= static_cast<uint64_t>((sbo >> 4) & 0x3FFF) << 32;
    d |= 1ull << 46;
    d |= 2ull << 61;
    return d;
}
// instruction descriptor: 16-bit x 16-bit -> f32 (format 1 bf16, 0 fp16), M x N, operand majors (0 K, 1 MN)
__host__ __device__ constexpr uint32_t instr_desc(int fmt, int M, int N, int a_mn, int b_mn) {
    return (1u << 4) | (static_cast<uint32_t>(fmt) << 7) | (static_cast<uint32_t>(fmt) << 10) | (static_cast<uint32_t>(a_mn) << 15) |
           (static_cast<uint32_t>(b_mn) << 16) | (static_cast<uint32_t>(N >> 3) << 17) |
           (static_cast<uint32_t>(M >> 4) << 24);
}

struct Params {
    TensorView o;
    float* lse;
    int64_t lse_sb, lse_sh;
    const int* cu;
    int B, H, HKV, G, S, causal;
    float scale;
    int* status;
    // fwd_window_sm100_kernel's: a row sees the `window` newest keys up to its own position and the first
    // `sinks` keys; with `plan` the queries are request b's last positions and its keys plan[b].x rows of
    // (row, head) tensors from row plan[b].y on, without the plan[b].z tiles of 128 keys between the sinks'
    // tiles and the window's that no query of the chunk sees
    int window, sinks;
    const int4* plan;
    int total;       // packed rows
    void* o_rest;    // what rounding took from o, laid out as o, or null
    int blocks;      // blocks of 256 rows (dense), or slots of 256 packed rows and one per request; with `plan` its own count
};
struct Maps {
    CUtensorMap q, k, v;   // (channel, row, head, batch), boxes (64, 128, 1, 1)
};

template <bool F16>
__global__ void __launch_bounds__(NTHREADS, 1) fwd_sm100_kernel(const Params p, const __grid_constant__ Maps maps) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = static_cast<uint32_t>(__cvta_generic_to_shared(smem_raw));
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (base - raw);
    auto bar = [&](int i) { return base + SM_BAR + 8 * i; };
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + SM_BAR + 8 * B_COUNT);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + SM_BAR + 8 * B_COUNT + 8);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // the last query rows first: under a causal mask they meet the most key tiles
    const int mb = gridDim.x - 1 - blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    int start = 0, len = p.S;
    if (p.cu) {
        start = p.cu[b];
        len = p.cu[b + 1] - start;
    }
    const int m0 = mb * CTA_M;
    if (m0 >= len) return;
    const int hkv = h / p.G;
    const int bb = p.cu ? 0 : b;
    // key tiles each of the two query tiles meets (the second tile may lie past the sequence)
    int nt[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int mx = m0 + x * BM;
        const int kv_end = mx >= len ? 0 : (p.causal ? min(len, mx + BM) : len);
        nt[x] = (kv_end + BN - 1) / BN;
    }
    const int n_tiles = max(nt[0], nt[1]);

    if (tid == 0) {
        *abort_flag = 0;
        mbar_init(bar(B_Q), 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(B_KVFULL + i), 1);
            mbar_init(bar(B_KVEMPTY + i), 1);
            mbar_init(bar(B_SFULL + i), 1);
            mbar_init(bar(B_PREADY + i), 128);
            mbar_init(bar(B_ODONE + i), 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;"
                     ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(tmem_slot))) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        // ================= TMA producer =================
        if (lane == 0) {
            mbar_expect_tx(bar(B_Q), nt[1] > 0 ? 65536 : 32768);
            for (int x = 0; x < 2; ++x) {
                if (nt[x] == 0) continue;
                for (int c = 0; c < 2; ++c)
                    tma_load_4d(base + SM_Q + x * 32768 + c * 16384, &maps.q, 64 * c, start + m0 + x * BM, h, bb, bar(B_Q));
            }
            for (int j = 0; j < n_tiles; ++j) {
                const int s = j & 1;
                if (j >= 2) mbar_wait(bar(B_KVEMPTY + s), ((j >> 1) - 1) & 1, abort_flag, p.status);
                const uint32_t st = base + SM_KV + s * STAGE;
                mbar_expect_tx(bar(B_KVFULL + s), 65536);
                for (int c = 0; c < 2; ++c) {
                    tma_load_4d(st + c * 16384, &maps.k, 64 * c, start + j * BN, hkv, bb, bar(B_KVFULL + s));
                    tma_load_4d(st + 32768 + c * 16384, &maps.v, 64 * c, start + j * BN, hkv, bb, bar(B_KVFULL + s));
                }
            }
        }
    } else if (warp == 1) {
        // ================= MMA issuer =================
        if (lane == 0) {
            constexpr uint32_t ID_S = instr_desc(F16 ? 0 : 1, 128, 128, 0, 0);    // Q (K-major) x K (K-major)
            constexpr uint32_t ID_PV = instr_desc(F16 ? 0 : 1, 128, 128, 0, 1);   // P (TMEM) x V (MN-major)
            mbar_wait(bar(B_Q), 0, abort_flag, p.status);
            auto issue_s = [&](int x, int j) {
                const int s = j & 1;
                mbar_wait(bar(B_KVFULL + s), (j >> 1) & 1, abort_flag, p.status);
                tc_fence_after();
                const uint32_t kt = base + SM_KV + s * STAGE, qt = base + SM_Q + x * 32768;
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) {   // 16 channels per step; 4 steps per 64-channel box
                    const uint32_t off = (ks >> 2) * 16384 + (ks & 3) * 32;
                    mma_ss(tmem + T_S + 128 * x, smem_desc(qt + off, 16, 1024), smem_desc(kt + off, 16, 1024), ID_S, ks > 0);
                }
                tc_commit(bar(B_SFULL + x));
            };
            for (int x = 0; x < 2; ++x)
                if (nt[x] > 0) issue_s(x, 0);
            for (int j = 0; j < n_tiles; ++j) {
                const int s = j & 1;
                const uint32_t vt = base + SM_KV + s * STAGE + 32768;
                for (int x = 0; x < 2; ++x) {
                    if (j >= nt[x]) continue;
                    mbar_wait(bar(B_PREADY + x), j & 1, abort_flag, p.status);
                    tc_fence_after();
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks)   // 16 keys per step: 8 TMEM columns of P, 2048 bytes of V per box
                        mma_ts(tmem + T_O + 128 * x, tmem + T_S + 128 * x + 8 * ks, smem_desc(vt + ks * 2048, 16384, 1024), ID_PV,
                               (j > 0) || (ks > 0));
                    tc_commit(bar(B_ODONE + x));
                    // the next scores overwrite S (and the P just consumed): the tensor pipe runs a
                    // thread's MMAs in the order it issued them
                    if (j + 1 < nt[x]) issue_s(x, j + 1);
                }
                tc_commit(bar(B_KVEMPTY + s));
            }
        }
    } else if (warp >= 4) {
        // ================= softmax: two groups, one per query tile; thread = query row = TMEM lane =================
        const int x = (warp - 4) >> 2;
        const int r = 32 * (warp & 3) + lane;
        const uint32_t lane_addr = static_cast<uint32_t>(32 * (warp & 3)) << 16;
        const float c2 = p.scale * kLog2e;
        const uint64_t c2x2 = pack2(c2, c2);
        const int mx = m0 + x * BM;
        const int qi = mx + r;                 // the row's position in its sequence
        const int my_tiles = nt[x];
        float m_run = -INFINITY, l_run = 0.f;  // running maximum (log2 domain) and sum
        const uint32_t ts = tmem + lane_addr + T_S + 128 * x;
        const uint32_t to = tmem + lane_addr + T_O + 128 * x;
        for (int j = 0; j < my_tiles; ++j) {
            const int n0 = j * BN;
            const bool need_mask = (p.causal && n0 + BN > mx) || (n0 + BN > len);
            const int kmax = min(len - 1, p.causal ? qi : len - 1) - n0;   // last key column this row may see
            mbar_wait(bar(B_SFULL + x), j & 1, abort_flag, p.status);
            tc_fence_after();
            // pass 1: the row's maximum over the tile
            float mxv = -INFINITY;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t sv[32];
                tmem_ld32(ts + 32 * c, sv);
                tmem_wait_ld();
                if (need_mask) {
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (32 * c + e > kmax) sv[e] = 0xff800000u;   // -inf
                }
#pragma unroll
                for (int e = 0; e < 32; e += 2) mxv = max3f(mxv, __uint_as_float(sv[e]), __uint_as_float(sv[e + 1]));
            }
            // The reference point only moves when the row's maximum rose by more than 2^LAZY: weights
            // up to 2^LAZY are as exact in 16 bits as weights up to 1, the final O / l cancels the
            // choice, and a row whose reference stays has alpha = 1 exactly, so its warp neither
            // waits for the previous product nor rescales O. After a sequence's first tiles that is
            // nearly every warp.
            const float m_cand = fmaxf(m_run, mxv * c2);
            const float m_new = m_cand > m_run + LAZY ? m_cand : m_run;
            // a row that sees no key yet keeps m = -inf; its weights are exp2(-inf) = 0
            const float m_use = m_new == -INFINITY ? 0.f : m_new;
            const float alpha = ex2f(m_run - m_use);   // 0 on the first tile that holds a key, 1 where the reference stays
            // pass 2: weights over the scores as packed bf16 (P chunk c lands on columns the row's
            // thread has already read), and their sum
            uint64_t sum2 = 0ull;   // two partial sums, added at the end of the tile
            const uint64_t nm2 = pack2(-m_use, -m_use);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t sv[32];
                tmem_ld32(ts + 32 * c, sv);
                tmem_wait_ld();
                uint32_t pp[16];
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    float x0, x1;
                    fma2(x0, x1, __uint_as_float(sv[e]), __uint_as_float(sv[e + 1]), c2x2, nm2);
                    x0 = ex2f(x0);
                    x1 = ex2f(x1);
                    if (need_mask) {
                        if (32 * c + e > kmax) x0 = 0.f;
                        if (32 * c + e + 1 > kmax) x1 = 0.f;
                    }
                    asm("add.rn.f32x2 %0, %0, %1;" : "+l"(sum2) : "l"(pack2(x0, x1)));   // even and odd columns apart
                    pp[e >> 1] = F16 ? pack_f16x2(x0, x1) : pack_bf16x2(x0, x1);
                }
                tmem_st16(ts + 16 * c, pp);
            }
            float sum_e, sum_o;
            asm("mov.b64 {%0, %1}, %2;" : "=f"(sum_e), "=f"(sum_o) : "l"(sum2));
            l_run = l_run * alpha + (sum_e + sum_o);
            m_run = m_new;
            // O was last written by key tile j-1's product: rescale it where a row's maximum rose
            if (j > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
                mbar_wait(bar(B_ODONE + x), (j - 1) & 1, abort_flag, p.status);
                tc_fence_after();
                {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t ov[32];
                        tmem_ld32(to + 32 * c, ov);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
                        tmem_st32(to + 32 * c, ov);
                    }
                }
            }
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(bar(B_PREADY + x));
        }
        // ---- epilogue: O / l -> bf16, LSE in nats ----
        if (my_tiles > 0) {
            mbar_wait(bar(B_ODONE + x), (my_tiles - 1) & 1, abort_flag, p.status);
            tc_fence_after();
            // the warp's tcgen05.ld is collective: every lane reads, rows past the sequence store nothing
            const bool row_ok = qi < len;
            auto pk2 = [](float a, float b2) { return F16 ? pack_f16x2(a, b2) : pack_bf16x2(a, b2); };
            const float inv = l_run > 0.f ? 1.0f / l_run : 0.f;
            uint16_t* orow = row_ptr<uint16_t>(p.o, b, start + (row_ok ? qi : 0), h);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t ov[32];
                tmem_ld32(to + 32 * c, ov);
                tmem_wait_ld();
                if (row_ok) {
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        uint4 w;
                        w.x = pk2(__uint_as_float(ov[8 * u]) * inv, __uint_as_float(ov[8 * u + 1]) * inv);
                        w.y = pk2(__uint_as_float(ov[8 * u + 2]) * inv, __uint_as_float(ov[8 * u + 3]) * inv);
                        w.z = pk2(__uint_as_float(ov[8 * u + 4]) * inv, __uint_as_float(ov[8 * u + 5]) * inv);
                        w.w = pk2(__uint_as_float(ov[8 * u + 6]) * inv, __uint_as_float(ov[8 * u + 7]) * inv);
                        *reinterpret_cast<uint4*>(orow + 32 * c + 8 * u) = w;
                    }
                }
            }
            if (row_ok) {
                const float lse = l_run > 0.f ? (m_run + log2f(l_run)) * 0.6931471805599453f : -INFINITY;
                p.lse[static_cast<int64_t>(b) * p.lse_sb + static_cast<int64_t>(h) * p.lse_sh + start + qi] = lse;
            }
            tc_fence_before();
        }
    }
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// ---- a sliding window with sinks, and keys of another length than the queries ------------------
// The same tiles and the same softmax under another mask, as a persistent kernel: a window's CTA has ten
// key tiles or so to walk, and what a CTA of its own costs each block (launch, TMEM, barriers, the first
// loads, and the epilogue with nothing behind it) was half of its time. One CTA per SM walks the work items
// in stride, and the next item's Q and first tiles are loaded, and its first scores issued, while the last
// one's O is written. Barrier phases count key tiles and items since the CTA started.
// Measured (D=128, 32 heads, 8 KV heads): 6 packed sequences of 16384 tokens in all, window 512: 250 us; 2 x 8192, window 1024,
// 4 sinks: 360-390; chunks of 2 x 2048 behind 16384-24576 keys: 1660 (1.0 PFLOP/s). The tensor and the transcendental
// pipe are busy 54 % of the time each: a tile's softmax waits for its scores and its product for the softmax, and two query
// tiles a CTA cover one another in part. Taking the weights in one pass over the scores (the maximum found
// on the way, a second pass where it rose) was slower, 2068 us for the chunks: the weights wait in registers for the verdict.
// In a loop of seconds the power cap holds the SMs at 1.7 GHz and the chunks take 1850.

// What an item walks: key tiles [0, ns), then [lo, lo + n - ns); query tile x takes tiles
// [low[x], end[x]) and those of the sinks (st of them).
struct Item {
    int m0, h, b, start, len, klen, qoff, kstart, kshift;
    int ns, lo, n, st;
    int end[2], low[2], nt[2];      // nt: key tiles that query tile x takes
    bool half;                      // 128 rows: there is no second query tile
    __device__ __forceinline__ int tile(int j) const { return j < ns ? j : lo + j - ns; }
    __device__ __forceinline__ bool takes(int e, int l, int j) const {
        const int t = tile(j);
        return j < n && t < e && (t >= l || t < st);
    }
    // the first row of the j-th tile (tiles that a chunk leaves out have none)
    __device__ __forceinline__ int row(int j) const {
        const int t = tile(j);
        return kstart + (t < st ? t : t - kshift) * BN;
    }
};

// Work item i, longest rows first in a dense call; false if it is empty.
struct List {
    int blocks;      // of 256 rows
    int whole;       // blocks x heads, of which so many are walked whole and the others as two items of 128 rows
    int items;       // so many in all
    const int* first;   // with `plan`: each request's first block
};
__device__ __forceinline__ List list_of(const Params& p) {
    List l;
    l.first = p.plan ? reinterpret_cast<const int*>(p.plan + p.B) : nullptr;
    l.blocks = p.plan ? __ldg(l.first + p.B) : p.blocks;
    // The last wave: where at most half of the CTAs would have an item of 256 rows, it is walked as twice as many
    // of 128: the 512 items of a 2 x 2048-token chunk are 3.46 waves of 148 (1658 -> 1624 us).
    const int n = l.blocks * p.H, ctas = static_cast<int>(gridDim.x), rest = n % ctas;
    l.whole = n > ctas && 2 * rest <= ctas ? n - rest : n;
    l.items = l.whole + 2 * (n - l.whole);
    return l;
}
__device__ __forceinline__ bool load_item(const Params& p, const List& l, int i, Item& w) {
    w.half = i >= l.whole;
    const int second = w.half ? (i - l.whole) & 1 : 0;
    if (w.half) i = l.whole + ((i - l.whole) >> 1);
    const int blk = i / p.H;
    w.h = i - blk * p.H;
    if (p.cu) {
        // packed: request b's blocks sit in slots from cu[b] / 256 + b on (at least as many as it needs)
        // (a chunk's plan counts them exactly)
        const int slot = l.blocks - 1 - blk;
        auto first_of = [&](int b) { return l.first ? __ldg(l.first + b) : __ldg(p.cu + b) / CTA_M + b; };
        int lo = 0, hi = p.B;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (first_of(mid) <= slot) lo = mid;
            else hi = mid;
        }
        w.b = lo;
        w.start = __ldg(p.cu + lo);
        w.len = __ldg(p.cu + lo + 1) - w.start;
        w.m0 = (slot - first_of(lo)) * CTA_M;
    } else {
        const int nb = (p.S + CTA_M - 1) / CTA_M;
        w.b = blk % p.B;
        w.start = 0;
        w.len = p.S;
        w.m0 = (nb - 1 - blk / p.B) * CTA_M;
    }
    if (w.m0 < 0) return false;
    w.m0 += second * BM;
    if (w.m0 >= w.len) return false;
    if (p.plan && (w.start < 0 || w.len > p.total - w.start)) {   // counts that q has no rows for
        atomicExch(p.status, FOLD_ERR_ARGUMENT);
        return false;
    }
    w.klen = w.len;
    w.qoff = w.kshift = 0;
    w.kstart = w.start;
    if (p.plan) {
        const int4 pl = __ldg(p.plan + w.b);
        if (pl.x < 0) return false;   // another kernel's
        w.klen = pl.x;
        w.qoff = pl.x - w.len;
        w.kstart = pl.y;
        w.kshift = pl.z;
    }
    w.st = w.ns = (p.sinks + BN - 1) / BN;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int mx = w.m0 + x * BM;
        const int kv_end = mx >= w.len || (x == 1 && w.half) ? 0 : max(0, min(w.klen, w.qoff + min(mx + BM, w.len)));
        w.end[x] = (kv_end + BN - 1) / BN;
        w.low[x] = max(0, w.qoff + mx - p.window + 1) / BN;
        w.nt[x] = min(w.end[x], w.st) + max(0, w.end[x] - max(w.low[x], w.st));
    }
    w.lo = w.low[0];
    if (w.ns >= w.lo) w.ns = w.lo = 0;   // the sinks' tiles run into the window's
    w.n = max(0, w.ns + max(w.end[0], w.end[1]) - w.lo);
    return true;
}
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

template <bool F16>
__global__ void __launch_bounds__(NTHREADS, 1) fwd_window_sm100_kernel(const Params p, const __grid_constant__ Maps maps) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = static_cast<uint32_t>(__cvta_generic_to_shared(smem_raw));
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (base - raw);
    auto bar = [&](int i) { return base + SM_BAR + 8 * i; };
    constexpr int B_QEMPTY = B_COUNT;      // the item's last scores are out of Q
    constexpr int B_CUT = B_COUNT + 1;     // a sequence's last tile has landed, its V still with the rows behind it
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + SM_BAR + 8 * (B_COUNT + 2));
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + SM_BAR + 8 * (B_COUNT + 2) + 8);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        *abort_flag = 0;
        mbar_init(bar(B_Q), 1);
        mbar_init(bar(B_QEMPTY), 1);
        mbar_init(bar(B_CUT), 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(B_KVFULL + i), 1);
            mbar_init(bar(B_KVEMPTY + i), 1);
            mbar_init(bar(B_SFULL + i), 1);
            mbar_init(bar(B_PREADY + i), 128);
            mbar_init(bar(B_ODONE + i), 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;"
                     ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(tmem_slot))) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const List list = list_of(p);

    if (warp == 0) {
        // ================= TMA producer =================
        if (lane == 0) {
            int jk = 0, items = 0, cuts = 0;         // key tiles, items with any, and tiles cut short, so far
            for (int i = blockIdx.x; i < list.items; i += gridDim.x) {
                Item w;
                if (!load_item(p, list, i, w) || w.nt[0] + w.nt[1] == 0) continue;
                if (*abort_flag) break;
                const int hkv = w.h / p.G, bb = p.cu ? 0 : w.b;
                if (items > 0) mbar_wait(bar(B_QEMPTY), (items - 1) & 1, abort_flag, p.status);
                mbar_expect_tx(bar(B_Q), w.nt[0] > 0 && w.nt[1] > 0 ? 65536 : 32768);
#pragma unroll
                for (int x = 0; x < 2; ++x)
                    if (w.nt[x] > 0)
                        for (int c = 0; c < 2; ++c)
                            tma_load_4d(base + SM_Q + x * 32768 + c * 16384, &maps.q, 64 * c, w.start + w.m0 + x * BM, w.h, bb, bar(B_Q));
                for (int j = 0; j < w.n; ++j, ++jk) {
                    const int s = jk & 1;
                    if (jk >= 2) mbar_wait(bar(B_KVEMPTY + s), ((jk >> 1) - 1) & 1, abort_flag, p.status);
                    if (*abort_flag) break;    // nothing new once a wait ran out
                    const uint32_t st = base + SM_KV + s * STAGE;
                    // A packed sequence's last tile holds rows behind its end: their scores are masked, but a NaN in V there
                    // would pass through P's zeros, so V's are made zeros before the tile is handed on.
                    const int live = max(0, w.klen - w.tile(j) * BN);
                    const bool cut = p.cu && !p.plan && live < BN;
                    const uint32_t full = bar(cut ? B_CUT : B_KVFULL + s);
                    mbar_expect_tx(full, 65536);
                    for (int c = 0; c < 2; ++c) {
                        tma_load_4d(st + c * 16384, &maps.k, 64 * c, w.row(j), hkv, bb, full);
                        tma_load_4d(st + 32768 + c * 16384, &maps.v, 64 * c, w.row(j), hkv, bb, full);
                    }
                    if (cut) {
                        mbar_wait(full, cuts++ & 1, abort_flag, p.status);
                        for (int c = 0; c < 2; ++c) {
                            uint4* dead = reinterpret_cast<uint4*>(smem + SM_KV + s * STAGE + 32768 + c * 16384 + live * 128);
                            for (int u = 0; u < 8 * (BN - live); ++u) dead[u] = make_uint4(0u, 0u, 0u, 0u);
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        mbar_arrive(bar(B_KVFULL + s));
                    }
                }
                ++items;
            }
        }
    } else if (warp == 1) {
        // ================= MMA issuer =================
        if (lane == 0) {
            constexpr uint32_t ID_S = instr_desc(F16 ? 0 : 1, 128, 128, 0, 0);    // Q (K-major) x K (K-major)
            constexpr uint32_t ID_PV = instr_desc(F16 ? 0 : 1, 128, 128, 0, 1);   // P (TMEM) x V (MN-major)
            int jk = 0, items = 0, done[2] = {0, 0};
            for (int i = blockIdx.x; i < list.items; i += gridDim.x) {
                Item w;
                if (!load_item(p, list, i, w) || w.nt[0] + w.nt[1] == 0) continue;
                mbar_wait(bar(B_Q), items & 1, abort_flag, p.status);
                int left = w.nt[0] + w.nt[1];      // scores still to issue
                auto issue_s = [&](int x, int j) {
                    const int g = jk + j, s = g & 1;
                    mbar_wait(bar(B_KVFULL + s), (g >> 1) & 1, abort_flag, p.status);
                    tc_fence_after();
                    const uint32_t kt = base + SM_KV + s * STAGE, qt = base + SM_Q + x * 32768;
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) {
                        const uint32_t off = (ks >> 2) * 16384 + (ks & 3) * 32;
                        mma_ss(tmem + T_S + 128 * x, smem_desc(qt + off, 16, 1024), smem_desc(kt + off, 16, 1024), ID_S, ks > 0);
                    }
                    tc_commit(bar(B_SFULL + x));
                    if (--left == 0) tc_commit(bar(B_QEMPTY));
                };
                bool now[2], next[2], first[2] = {true, true};
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    next[x] = w.takes(w.end[x], w.low[x], 0);
                    if (next[x]) issue_s(x, 0);
                }
                for (int j = 0; j < w.n; ++j) {
                    const int s = (jk + j) & 1;
                    const uint32_t vt = base + SM_KV + s * STAGE + 32768;
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        now[x] = next[x];
                        next[x] = w.takes(w.end[x], w.low[x], j + 1);
                    }
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        if (now[x]) {
                            mbar_wait(bar(B_PREADY + x), done[x] & 1, abort_flag, p.status);
                            tc_fence_after();
#pragma unroll
                            for (int ks = 0; ks < 8; ++ks)   // 16 keys per step: 8 TMEM columns of P, 2048 bytes of V per box
                                mma_ts(tmem + T_O + 128 * x, tmem + T_S + 128 * x + 8 * ks, smem_desc(vt + ks * 2048, 16384, 1024), ID_PV,
                                       !first[x] || ks > 0);
                            tc_commit(bar(B_ODONE + x));
                            ++done[x];
                            first[x] = false;
                        }
                        // the next scores overwrite S and the P just consumed: a thread's MMAs run in the order it issued
                        // them. (Only ever the next key tile's: a later one's stage is not free before this tile is done with it.)
                        if (next[x]) issue_s(x, j + 1);
                    }
                    // a tile that no product reads has still to land before its stage is filled again
                    if (!now[0] && !now[1]) mbar_wait(bar(B_KVFULL + s), ((jk + j) >> 1) & 1, abort_flag, p.status);
                    tc_commit(bar(B_KVEMPTY + s));
                }
                jk += w.n;
                ++items;
            }
        }
    } else if (warp == 2) {
        // rows behind the last packed sequence: zeros
        if (p.cu && !p.plan)
            for (int64_t i = max(__ldg(p.cu + p.B), 0) + static_cast<int64_t>(blockIdx.x); i < p.total; i += gridDim.x)
                for (int h = 0; h < p.H; ++h) {
                    if (lane < 16) *reinterpret_cast<uint4*>(row_ptr<uint16_t>(p.o, 0, i, h) + 8 * lane) = make_uint4(0u, 0u, 0u, 0u);
                    if (lane == 0 && p.lse) p.lse[h * p.lse_sh + i] = -INFINITY;
                }
    } else if (warp >= 4) {
        // ================= softmax: two groups, one per query tile; thread = query row = TMEM lane =================
        const int x = (warp - 4) >> 2;
        const int r = 32 * (warp & 3) + lane;
        const uint32_t lane_addr = static_cast<uint32_t>(32 * (warp & 3)) << 16;
        const float c2 = p.scale * kLog2e;
        const uint64_t c2x2 = pack2(c2, c2);
        const uint32_t ts = tmem + lane_addr + T_S + 128 * x;
        const uint32_t to = tmem + lane_addr + T_O + 128 * x;
        // A chunk's fp16 weights, of rows that may see millions of keys, and their sums carry 2^7, which O / l cancels: up to
        // 2^(LAZY + 7) of 65504, and a weight loses 2^-32 of its row's largest at most instead of 2^-25
        const float lift = F16 && p.plan ? 7.0f : 0.0f;
        int it = 0;                                // the query tile's key tiles so far
        for (int i = blockIdx.x; i < list.items; i += gridDim.x) {
            Item w;
            if (!load_item(p, list, i, w) || (x == 1 && w.half)) continue;
            const int mx = w.m0 + x * BM;
            const int qr = mx + r;                 // the query's row in its sequence
            const int qi = qr + w.qoff;            // its position among the keys
            const int my_end = x ? w.end[1] : w.end[0], my_low = x ? w.low[1] : w.low[0], my_tiles = x ? w.nt[1] : w.nt[0];
            float m_run = -INFINITY, l_run = 0.f;  // running maximum (log2 domain) and sum
            bool first = true;
            for (int j = 0; j < w.n; ++j) {
                if (!w.takes(my_end, my_low, j)) continue;
                const int n0 = w.tile(j) * BN;
                // the tile's last row has moved past its first key, or its first row does not see the last
                const bool need_mask = n0 + BN > w.qoff + mx || n0 + BN > w.klen || (n0 <= w.qoff + mx + BM - 1 - p.window && n0 + BN > p.sinks);
                const int kmax = min(w.klen - 1, qi) - n0, kmin = qi - p.window + 1 - n0, ksink = p.sinks - n0;
                // columns [32 c, 32 c + 32) that the row sees, as bits
                auto seen = [&](int c) { return bits_below(kmax + 1 - 32 * c) & (~bits_below(kmin - 32 * c) | bits_below(ksink - 32 * c)); };
                mbar_wait(bar(B_SFULL + x), it & 1, abort_flag, p.status);
                tc_fence_after();
                // pass 1: the row's maximum over the tile. The masked and the unmasked form are two pieces of code: left to
                // itself the compiler evaluates this mask for every tile, at 1.6 times the kernel's time.
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};   // apart: one chain of 64 would be latency
                auto row_max = [&](auto masked) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t sv[32];
                        tmem_ld32(ts + 32 * c, sv);
                        const uint32_t vis = decltype(masked)::value ? seen(c) : 0u;
                        tmem_wait_ld();
                        if (decltype(masked)::value) {
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (!(vis & (1u << e))) sv[e] = 0xff800000u;   // -inf
                        }
#pragma unroll
                        for (int e = 0; e < 32; e += 2)
                            mx4[(e >> 1) & 3] = max3f(mx4[(e >> 1) & 3], __uint_as_float(sv[e]), __uint_as_float(sv[e + 1]));
                    }
                };
                if (need_mask) row_max(std::true_type{});
                else row_max(std::false_type{});
                const float mxv = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
                // The reference point only moves when the row's maximum rose by more than 2^LAZY (fwd_sm100_kernel)
                const float m_cand = fmaxf(m_run, mxv * c2);
                const float m_new = m_cand > m_run + LAZY ? m_cand : m_run;
                const float m_use = m_new == -INFINITY ? 0.f : m_new;     // a row that sees no key yet
                const float alpha = m_run == -INFINITY ? 1.f : ex2f(m_run - m_use);   // (its O is zero: nothing to rescale)
                uint64_t sum2 = 0ull;
                const uint64_t nm2 = pack2(lift - m_use, lift - m_use);
                auto weights = [&](auto masked) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t sv[32];
                        tmem_ld32(ts + 32 * c, sv);
                        const uint32_t vis = decltype(masked)::value ? seen(c) : 0u;
                        tmem_wait_ld();
                        uint32_t pp[16];
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            float x0, x1;
                            fma2(x0, x1, __uint_as_float(sv[e]), __uint_as_float(sv[e + 1]), c2x2, nm2);
                            x0 = ex2f(x0);
                            x1 = ex2f(x1);
                            if (decltype(masked)::value) {
                                if (!(vis & (1u << e))) x0 = 0.f;
                                if (!(vis & (2u << e))) x1 = 0.f;
                            }
                            asm("add.rn.f32x2 %0, %0, %1;" : "+l"(sum2) : "l"(pack2(x0, x1)));   // even and odd columns apart
                            pp[e >> 1] = F16 ? pack_f16x2(x0, x1) : pack_bf16x2(x0, x1);
                        }
                        tmem_st16(ts + 16 * c, pp);
                    }
                };
                if (need_mask) weights(std::true_type{});
                else weights(std::false_type{});
                float sum_e, sum_o;
                asm("mov.b64 {%0, %1}, %2;" : "=f"(sum_e), "=f"(sum_o) : "l"(sum2));
                l_run = l_run * alpha + (sum_e + sum_o);
                m_run = m_new;
                // O was last written by the product of the key tile before: rescale it where a row's maximum rose
                if (!first && __any_sync(0xffffffffu, alpha != 1.0f)) {
                    mbar_wait(bar(B_ODONE + x), (it - 1) & 1, abort_flag, p.status);
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t ov[32];
                        tmem_ld32(to + 32 * c, ov);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
                        tmem_st32(to + 32 * c, ov);
                    }
                }
                first = false;
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(bar(B_PREADY + x));
                ++it;
            }
            // ---- epilogue: O / l -> 16-bit, LSE in nats ----
            const bool row_ok = qr < w.len;
            uint16_t* orow = row_ptr<uint16_t>(p.o, w.b, w.start + (row_ok ? qr : 0), w.h);
            uint16_t* rrow = static_cast<uint16_t*>(p.o_rest) + (orow - static_cast<uint16_t*>(p.o.ptr));
            if (my_tiles > 0) {
                mbar_wait(bar(B_ODONE + x), (it - 1) & 1, abort_flag, p.status);
                tc_fence_after();
                auto pk2 = [](float a, float b2) { return F16 ? pack_f16x2(a, b2) : pack_bf16x2(a, b2); };
                const float inv = l_run > 0.f ? 1.0f / l_run : 0.f;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t ov[32];
                    tmem_ld32(to + 32 * c, ov);
                    tmem_wait_ld();
                    if (row_ok) {
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            uint4 v;
                            v.x = pk2(__uint_as_float(ov[8 * u]) * inv, __uint_as_float(ov[8 * u + 1]) * inv);
                            v.y = pk2(__uint_as_float(ov[8 * u + 2]) * inv, __uint_as_float(ov[8 * u + 3]) * inv);
                            v.z = pk2(__uint_as_float(ov[8 * u + 4]) * inv, __uint_as_float(ov[8 * u + 5]) * inv);
                            v.w = pk2(__uint_as_float(ov[8 * u + 6]) * inv, __uint_as_float(ov[8 * u + 7]) * inv);
                            *reinterpret_cast<uint4*>(orow + 32 * c + 8 * u) = v;
                            if (p.o_rest) {
                                auto rest = [&](int e, uint32_t w) {
                                    return pk2(__uint_as_float(ov[8 * u + e]) * inv - half_bits_to_float<F16>(static_cast<uint16_t>(w & 0xFFFFu)),
                                               __uint_as_float(ov[8 * u + e + 1]) * inv - half_bits_to_float<F16>(static_cast<uint16_t>(w >> 16)));
                                };
                                *reinterpret_cast<uint4*>(rrow + 32 * c + 8 * u) = make_uint4(rest(0, v.x), rest(2, v.y), rest(4, v.z), rest(6, v.w));
                            }
                        }
                    }
                }
                tc_fence_before();
            } else if (row_ok) {   // rows that see no key at all
                for (int u = 0; u < 16; ++u) *reinterpret_cast<uint4*>(orow + 8 * u) = make_uint4(0u, 0u, 0u, 0u);
            }
            if (row_ok && p.lse) {
                const float lse = l_run > 0.f ? (m_run - lift + log2f(l_run)) * 0.6931471805599453f : -INFINITY;
                p.lse[static_cast<int64_t>(w.b) * p.lse_sb + static_cast<int64_t>(w.h) * p.lse_sh + w.start + qr] = lse;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {        // a wait ran out: what was under way lands before this memory is another CTA's
        const long long t0 = clock64();
        while (clock64() - t0 < DRAIN_CYCLES) {}
        __syncthreads();
    }
    if (warp == 1) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

}  // namespace fsm100
}  // namespace fold

using namespace fold;

namespace {

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                              CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                              CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
    static EncodeFn fn = nullptr;
    if (!fn) {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeFn>(ptr);
    }
    return fn;
}

// (channel, row, head, batch) view of a (batch, row, head, channel)-strided bf16 tensor; a box is
// 64 channels of 128 rows. Rows past the tensor read as zeros.
bool make_map(CUtensorMap* m, const void* ptr, int64_t sb, int64_t sr, int64_t sh, int64_t rows, int heads, int batch, bool f16) {
    EncodeFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[4] = {128, static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(batch)};
    if (!sb) sb = sr * rows;
    cuuint64_t strides[3] = {static_cast<cuuint64_t>(sr * 2), static_cast<cuuint64_t>(sh * 2), static_cast<cuuint64_t>(sb * 2)};
    cuuint32_t box[4] = {64, 128, 1, 1};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    return fn(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(ptr), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

extern "C" int fold_fwd_sm100_supported(int head_dim, int is_f16) {
    (void)is_f16;   // bf16 and fp16
    return head_dim == 128 && encode_fn() != nullptr;
}

namespace {

// The causal and full forward, or (`ext`) the windowed one.
int run_sm100(const char* what, const void* q, const void* k, const void* v, void* o, float* lse, void* o_rest, const int64_t* strides,
              const int32_t* cu_seqlens, int batch, int n_heads, int n_kv_heads, int max_seqlen, int total, int head_dim,
              int causal, int is_f16, float softmax_scale, int ext, int window, int sinks, const int32_t* plan, int krows,
              int32_t* status, void* stream) {
    FOLD_CHECK_ARG(q && k && v && o && (lse || plan) && strides && status, "%s: null pointer", what);
    FOLD_CHECK_ARG(n_kv_heads > 0 && n_heads % n_kv_heads == 0, "the query heads must be a multiple of the KV heads");
    FOLD_CHECK_ARG(batch > 0 && max_seqlen > 0, "%s: empty call", what);
    FOLD_CHECK_ARG(n_heads <= 65535 && batch <= 65535, "%s: %d heads, %d requests (65535 at most)", what, n_heads, batch);
    if (!fold_fwd_sm100_supported(head_dim, 0)) {
        set_error("the tcgen05 forward takes head_dim 128");
        return FOLD_ERR_UNSUPPORTED;
    }
    const void* ptrs[4] = {q, k, v, o};
    for (int i = 0; i < 4; ++i)
        FOLD_CHECK_ARG(strides[3 * i] % 8 == 0 && strides[3 * i + 1] % 8 == 0 && strides[3 * i + 2] % 8 == 0 &&
                           reinterpret_cast<uintptr_t>(ptrs[i]) % 16 == 0,
                       "%s: rows must be 16-byte aligned", what);
    fsm100::Params p;
    p.o.ptr = o; p.o.sb = strides[9]; p.o.sr = strides[10]; p.o.sh = strides[11];
    p.lse = lse;
    p.o_rest = o_rest;
    p.cu = cu_seqlens;
    if (cu_seqlens) {
        p.lse_sb = 0;
        p.lse_sh = total;
    } else {
        p.lse_sb = static_cast<int64_t>(n_heads) * max_seqlen;
        p.lse_sh = max_seqlen;
    }
    p.B = batch; p.H = n_heads; p.HKV = n_kv_heads; p.G = n_heads / n_kv_heads;
    p.S = max_seqlen; p.causal = causal; p.scale = softmax_scale; p.status = status;
    p.window = window; p.sinks = sinks; p.plan = reinterpret_cast<const int4*>(plan);
    const int64_t rows = cu_seqlens ? total : max_seqlen;
    const int mbatch = cu_seqlens ? 1 : batch;
    const int64_t kvrows = plan ? krows : rows;
    fsm100::Maps maps;
    const bool f16 = is_f16 != 0;
    if (!make_map(&maps.q, q, strides[0], strides[1], strides[2], rows, n_heads, mbatch, f16) ||
        !make_map(&maps.k, k, strides[3], strides[4], strides[5], kvrows, n_kv_heads, mbatch, f16) ||
        !make_map(&maps.v, v, strides[6], strides[7], strides[8], kvrows, n_kv_heads, mbatch, f16)) {
        set_error("%s: cuTensorMapEncodeTiled failed", what);
        return FOLD_ERR_LAUNCH;
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (ext) {
        // packed: a slot per 256 rows and one per request (fsm100::load_item); dense: the blocks themselves
        const int64_t blocks = cu_seqlens ? static_cast<int64_t>(total) / fsm100::CTA_M + batch
                                          : static_cast<int64_t>((max_seqlen + fsm100::CTA_M - 1) / fsm100::CTA_M) * batch;
        FOLD_CHECK_ARG(2 * blocks * n_heads < (1ll << 31), "%s: %lld blocks of %d heads", what, static_cast<long long>(blocks), n_heads);
        p.blocks = static_cast<int>(blocks);
        p.total = total;
        int dev = 0, sms = 1;
        cudaGetDevice(&dev);
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
        auto kern = f16 ? fsm100::fwd_window_sm100_kernel<true> : fsm100::fwd_window_sm100_kernel<false>;
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, fsm100::SMEM_BYTES);
        kern<<<static_cast<int>(std::min<int64_t>(blocks * n_heads, sms)), fsm100::NTHREADS, fsm100::SMEM_BYTES, st>>>(p, maps);
        return check_launch(what);
    }
    p.blocks = p.total = 0;
    dim3 grid((max_seqlen + fsm100::CTA_M - 1) / fsm100::CTA_M, n_heads, batch);
    auto kern = f16 ? fsm100::fwd_sm100_kernel<true> : fsm100::fwd_sm100_kernel<false>;
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, fsm100::SMEM_BYTES);
    kern<<<grid, fsm100::NTHREADS, fsm100::SMEM_BYTES, st>>>(p, maps);
    return check_launch(what);
}

}  // namespace

extern "C" int fold_fwd_run_sm100(const void* q, const void* k, const void* v, void* o, float* lse,
                                  const int64_t* strides, const int32_t* cu_seqlens, int batch, int n_heads,
                                  int n_kv_heads, int max_seqlen, int total, int head_dim, int causal, int is_f16,
                                  float softmax_scale, int32_t* status, void* stream) {
    FOLD_CHECK_ARG(lse, "fold_fwd_run_sm100: null pointer");
    return run_sm100("fold_fwd_run_sm100", q, k, v, o, lse, nullptr, strides, cu_seqlens, batch, n_heads, n_kv_heads, max_seqlen, total,
                     head_dim, causal, is_f16, softmax_scale, 0, 0, 0, nullptr, 0, status, stream);
}

extern "C" int fold_fwd_window_sm100(const void* q, const void* k, const void* v, void* o, float* lse, void* o_rest,
                                     const int64_t* strides, const int32_t* cu_seqlens, int batch, int n_heads,
                                     int n_kv_heads, int max_seqlen, int total, int head_dim, int is_f16,
                                     float softmax_scale, int window, int sinks, const int32_t* plan, int key_rows,
                                     int32_t* status, void* stream) {
    FOLD_CHECK_ARG(window > 0 && window <= FOLD_MAX_WINDOW && sinks >= 0 && sinks <= FOLD_MAX_WINDOW,
                   "fold_fwd_window_sm100: a window of %d keys and %d sinks (1 .. 2^30 and 0 .. 2^30)", window, sinks);
    FOLD_CHECK_ARG(!plan || key_rows > 0, "fold_fwd_window_sm100: %d key rows", key_rows);
    FOLD_CHECK_ARG(reinterpret_cast<uintptr_t>(o_rest) % 16 == 0 && !(plan && o_rest), "fold_fwd_window_sm100: o_rest is 16-byte aligned, without a plan");
    return run_sm100("fold_fwd_window_sm100", q, k, v, o, lse, o_rest, strides, cu_seqlens, batch, n_heads, n_kv_heads, max_seqlen, total,
                     head_dim, 1, is_f16, softmax_scale, 1, window, sinks, plan, key_rows, status, stream);
}
