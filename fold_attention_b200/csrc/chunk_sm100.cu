// Attention of a few new tokens per request over the paged, quantised cache: each KV head's query
// rows (new tokens x query heads of the group, 128 at most) meet every key the request's window
// holds, straight from the pool's codes. Bytes bound it (a key is 4 D + 2 of them, and a row group
// does at most 128 rows' work with it), so the codes are what travels and nothing is written back but O.
//
//   S1 = Qa Ka^T, S2 = Qa Kb^T + Qb Ka^T    tcgen05.mma kind::i8, M=128 rows, N=128 keys, on the planes as
//                stored (their XOR swizzle is the tensor core's), exact int32 in TMEM
//   logit = (256 S1 + S2) ek (eq / 256)     the query's planes as a decode step's (16 bits of its largest); the
//                product of the two second planes, under 2^-16 of the largest logit, is left out
//   P  = exp2(logit - m)                    per row, written as 16-bit to TMEM (fp16 queries on a bf16 V: as two
//                bf16 terms, or P would be 8 bits where the output has 11); a row's reference m moves only when
//                the row's maximum passes it by more than 2^8
//   O += P V     kind::f16, A = P from TMEM, B = V (MN-major): a bf16 V as TMA lays it down; an 8-bit V's two
//                planes converted to fp16 in shared memory, where a + b / 8 fits but for its last bits
//
// Few rows would leave most of the 128 TMEM lanes, and three of the four softmax warps, without work:
// a group of up to 32 (64) rows is stacked four (two) times, each copy's warp takes a quarter (half)
// of a tile's keys, with zeros in P for the others, and the copies' sums meet in the epilogue.
// Between two (request, head)s the next one's Q and first tiles are on their way while O is written out.
//
// Work is one list of 128-key tiles, request by request and head by head, cut evenly over one
// persistent CTA per SM: a (request, head) spans neighbouring CTAs at most where their ranges meet.
// Each leaves its piece (m, l, O) in the workspace and the last to arrive adds the pieces in list
// order, so the bits do not depend on who that is.
//
// Measured: 64 requests of up to 32768 keys, 8 KV heads, D=128, an 8-bit V, one token each under a window of 1024 with 4
// sinks: 80-84 us of 41 that its bytes take at the copy's rate (3.3 TB/s): a CTA has some twenty tiles in three or four
// (request, head)s, and what each of those costs beside its tiles is a quarter of its time; the conversion of V's
// two planes to fp16 is most of the rest. (The decode kernel feeds them to kind::f8f6f4 as stored, its weights as four E5M2
// terms; P in such terms has not been tried here.) 32 requests of up to 32768 keys, 3-8 tokens each, a
// bf16 V: 290-300 us of 276 (6.2 TB/s); 370 in a loop of seconds, where the power cap holds the SMs at 1.4 GHz.
//
// Warps: 0 K producer (both planes, scales), 3 V producer, 1 MMA issuer, 2 Q and V's dead rows (bf16 V),
// 4-7 softmax and epilogue, 2 (8-bit V) or 8-11 (bf16 V) join pieces, 8-11 V's conversion (8-bit V). Every wait is bounded.
#include <cuda.h>

#include <type_traits>

#include "cache_common.cuh"
#include "fold_b200.h"

namespace fold {
namespace csm100 {

constexpr int BN = 128;
constexpr long long WAIT_CYCLES = 1ll << 31;
constexpr long long DRAIN_CYCLES = 1ll << 22;    // two milliseconds: a copy takes microseconds
constexpr float LAZY = 8.0f;
// An 8-bit V's weights are fp16, whose least step is 2^-24: they and their sum carry 2^LIFT, which O / l cancels. At most
// 2^(LAZY + LIFT) of 65504, and a row's weights lose 2^-32 each of its largest at most instead of 2^-25, which a million keys
// far under one would have added up to 3 % of the row.
constexpr float LIFT = 7.0f;
constexpr int SLOTS = 4;         // a CTA's pieces: of the item it starts in, of the one it ends in, two for the items between
constexpr int MIN_TILES = 4;     // tiles a CTA takes at least: its fixed costs are two or three tiles' time
// What a (request, head) costs a CTA beside its tiles, in tiles: its first tile's way through the pipeline and
// its last one's, and its O. Each item is that much longer in the list that the shares are cut from
// (without it the CTA that met ten short requests finished a third later than the others).
constexpr int ITEM_TILES = 5;

constexpr int N_GEO = 6;         // requests a CTA keeps the lengths of (a share of a long list spans two or three)

template <int D, bool V8>
struct Lay {
    static constexpr int PLANE = 128 * D;                  // a tile of one 8-bit plane
    static constexpr int NK = D == 128 ? (V8 ? 2 : 3) : (V8 ? 5 : 6), NV = D == 128 ? (V8 ? 2 : 3) : 5;
    static constexpr int KSLOT = 2 * PLANE, VSLOT = 2 * PLANE;
    static constexpr int SM_Q = 0;                         // plane A, plane B
    static constexpr int SM_V16 = 2 * PLANE;               // two converted tiles (8-bit V)
    static constexpr int SM_K = SM_V16 + (V8 ? 4 * PLANE : 0);
    static constexpr int SM_V = SM_K + NK * KSLOT;
    static constexpr int SM_EK = SM_V + NV * VSLOT;        // [NK][128] bf16
    static constexpr int SM_ROW = SM_EK + NK * 256;        // m, l [128] f32
    static constexpr int SM_BAR = SM_ROW + 2 * 512;
    static constexpr int SM_MISC = SM_BAR + 304;           // scan [12], walk [3] and the last piece's number, flags [2], TMEM address
    static constexpr int SM_GEO = SM_MISC + 80;            // the share's first requests
    static constexpr int USED = SM_GEO + N_GEO * 28;
    static constexpr int SLACK = 232448 - USED < 1024 ? 232448 - USED : 1024;   // room to align the base
    static constexpr int BYTES = USED + SLACK;
    static constexpr int W_JOIN = V8 ? 2 : 8, N_JOIN = V8 ? 1 : 4;   // the warps that join pieces
    static constexpr int NTHREADS = 384;
    static_assert(SLACK >= 0, "shared memory");
};

// barriers: [6] K slots, [5] V slots, [2] converted tiles, then one each
enum { B_KFULL = 0, B_KEMPTY = 6, B_VFULL = 12, B_VEMPTY = 17, B_VREADY = 22, B_CEMPTY = 27, B_SFULL = 29, B_SEMPTY = 30, B_PREADY = 31, B_ODONE = 32, B_QFULL = 33, B_QEMPTY = 34, B_PIECE = 35, B_JOINED = 36 };

constexpr uint32_t T_S1 = 0, T_S2 = 128, T_P = 256, T_P2 = 320, T_O = 384;   // TMEM columns: 128, 128, 64, 64, D

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
// Bounded wait: `abort` (shared) is raised by whoever runs out first, and then nobody waits any more.
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
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(bar) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p; }"
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
__device__ __forceinline__ float ex2f(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3f(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ float4 as_float4(uint4 v) {
    return make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
}
__device__ __forceinline__ uint4 as_uint4(float4 v) {
    return make_uint4(__float_as_uint(v.x), __float_as_uint(v.y), __float_as_uint(v.z), __float_as_uint(v.w));
}
// shared-memory matrix descriptor; layout 2 = 128-byte swizzle, 4 = 64-byte
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo, uint32_t layout) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((addr & 0x3FFFF) >> 4);
    d |= static_cast<uint64_t>((lbo >> 4) & 0x3FFF) << 16;
    d |= static_cast<uint64_t>((sbo >> 4) & 0x3FFF) << 32;
    d |= 1ull << 46;
    d |= static_cast<uint64_t>(layout) << 61;
    return d;
}
// instruction descriptor: c_fmt (1 f32, 2 s32), a/b formats, majors (0 K, 1 MN), N, M
__host__ __device__ constexpr uint32_t instr_desc(int c_fmt, int a_fmt, int b_fmt, int a_mn, int b_mn, int N, int M) {
    return (static_cast<uint32_t>(c_fmt) << 4) | (static_cast<uint32_t>(a_fmt) << 7) |
           (static_cast<uint32_t>(b_fmt) << 10) | (static_cast<uint32_t>(a_mn) << 15) |
           (static_cast<uint32_t>(b_mn) << 16) | (static_cast<uint32_t>(N >> 3) << 17) |
           (static_cast<uint32_t>(M >> 4) << 24);
}

struct Params {
    const uint16_t* q;
    int64_t q_st, q_sh;     // token, head
    int8_t* qa;             // Q's planes and scales / 256 by (request, KV head, row), from chunk_q_kernel
    int8_t* qb;
    float* eq;
    uint16_t* o;
    int64_t o_st, o_sh;
    const int* cu;
    const int* lens;
    const int* table;
    int batch, hkv, G, ppr, page_size, piece;   // piece: keys that one load may take (a page's power of two, 128 at most)
    int max_keys, total, window, sinks;
    const int8_t* ka;
    const int8_t* kb;
    const uint16_t* ek;
    const uint8_t* va;
    const uint8_t* vb;
    float evs;
    int* counters;          // [batch * hkv], zero
    float* parts;           // [SLOTS * CTAs][128 * D + 256]: pieces, O, then m and l
    int* status;
    int others;             // whether another kernel takes the requests with more rows
};

// One request as this kernel sees it; nt = 0: not its (no new tokens, or more rows than 128).
struct Geo {
    int tok0, n, L, first, shift, nt;
    int wide;       // more rows than the kernel takes
};
__device__ __forceinline__ Geo geo_of(const Params& p, int b) {
    Geo g;
    const int t0 = __ldg(p.cu + b), t1 = __ldg(p.cu + b + 1);
    g.tok0 = t0;
    g.n = t0 < 0 || t1 > p.total ? -1 : t1 - t0;     // (negative: counts that q has no rows for)
    g.L = max(0, min(__ldg(p.lens + b), p.max_keys));
    g.first = g.L - g.n;                       // position of the first new token
    const int ns = (p.sinks + BN - 1) / BN;
    g.shift = max(0, max(0, g.first - p.window + 1) / BN - ns);   // tiles between the sinks' and the window's first
    g.wide = static_cast<int64_t>(g.n) * p.G > 128;
    g.nt = g.n <= 0 || g.wide ? 0 : max(1, (g.L + BN - 1) / BN - g.shift);
    return g;
}
// A CTA's walk over its share of the list, a segment (tiles [t0, t1) of one (request, head)) at a time. In
// the list an item is ITEM_TILES + nt long, its tiles last.
struct Walk {
    int b, h, v;        // the next place: request, head, place in the item
    int left;
    Geo g;
    int t0, t1, segment;
    int64_t start;      // the item's first place in the list
    const Geo* kept;    // requests [b0, b0 + N_GEO)
    int b0;
    // the next segment; false, with the last one left standing, when the share is through
    __device__ __forceinline__ bool next(const Params& p) {
        int nb = b, nh = h, nv = v, nleft = left;
        int64_t ns = start;
        Geo ng = g;
        for (;;) {
            if (nleft <= 0) return false;
            if (nv < 0) {                          // the next item
                nv = 0;
                ns += ITEM_TILES + ng.nt;
                if (++nh == p.hkv) {
                    nh = 0;
                    do {
                        if (++nb >= p.batch) return false;
                        if (nb - b0 < N_GEO) ng = kept[nb - b0];
                        else ng = geo_of(p, nb);
                    } while (ng.nt == 0);
                }
            }
            const int v1 = min(ITEM_TILES + ng.nt, nv + nleft);
            const int n0 = max(0, nv - ITEM_TILES), n1 = max(0, v1 - ITEM_TILES);
            nleft -= v1 - nv;
            nv = v1 == ITEM_TILES + ng.nt ? -1 : v1;
            if (n1 > n0) {                         // (a share may end before an item's tiles begin)
                t0 = n0;
                t1 = n1;
                break;
            }
        }
        b = nb; h = nh; v = nv; left = nleft; start = ns; g = ng;
        ++segment;
        return true;
    }
    __device__ __forceinline__ int pos(const Params& p, int j) const {     // first position of the item's j-th tile
        return (j * BN < p.sinks ? j : j + g.shift) * BN;
    }
};

__device__ __forceinline__ int copies_of(int R) { return R <= 32 ? 4 : R <= 64 ? 2 : 1; }

// the first place of CTA c's share of the list, and whose share place x is in
__device__ __forceinline__ int64_t share_start(int64_t total, int n, int c) { return total * c / n; }
__device__ __forceinline__ int share_of(int64_t total, int n, int64_t x) { return static_cast<int>(((x + 1) * n - 1) / total); }

// Q's planes and scales, laid out as the attention's CTAs load them: row (token i, head g of the group) of
// (request b, KV head h) at cu[b] H + h n G + i G + g, its 16-byte units swizzled for the tensor core. A
// row costs a load and two thousand cycles of latency, which every CTA that meets the (request, head)
// would pay between its tiles; here all rows pay it at once (the first form did: 16 thousand cycles a
// (request, head) of which Q was half). Also zeroes the counters and the status word, in place of a memset.
template <int D, bool F16>
__global__ void __launch_bounds__(NT) chunk_q_kernel(const Params p, int heads, int64_t n_rows) {
    constexpr int TPR = D / 16, RPB = NT / TPR;
    const int64_t gt = static_cast<int64_t>(blockIdx.x) * NT + threadIdx.x;
    for (int64_t i = gt; i < static_cast<int64_t>(p.batch) * p.hkv; i += static_cast<int64_t>(gridDim.x) * NT) p.counters[i] = 0;
    if (gt == 0) *p.status = 0;
    const int lane = threadIdx.x % TPR;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * RPB + threadIdx.x / TPR;
    const int64_t rr = row < n_rows ? row : 0;
    const int tok = static_cast<int>(rr / heads), hd = static_cast<int>(rr % heads);
    float x[16];
    uint4 raw[2];
    load16<F16>(p.q + static_cast<int64_t>(tok) * p.q_st + static_cast<int64_t>(hd) * p.q_sh + lane * 16, x, raw);
    int lo = 0, hi = p.batch;      // the last request that starts at or before the token
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(p.cu + mid) <= tok) lo = mid;
        else hi = mid;
    }
    const int t0 = __ldg(p.cu + lo), t1 = __ldg(p.cu + lo + 1), n = t1 - t0;
    const bool ok = row < n_rows && tok >= t0 && tok < t1 && t1 <= p.total && static_cast<int64_t>(n) * p.G <= 128;
    const float qscale = D == 64 ? 0.18033688011112042f : 0.12751743082459868f;   // log2(e) / sqrt(D)
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = __fmul_rn(x[i], qscale);
    rotate16<TPR>(x, lane, D == 64 ? 0.125f : 0.08838834764831845f);
    const float e = __fmul_rn(fmaxf(row_amax16<TPR>(x), 1e-30f), INV127);
    uint4 wa, wb;
    int8_planes16(x, e, wa, wb);
    if (ok) {
        const int r = (tok - t0) * p.G + hd % p.G;
        const int64_t at = static_cast<int64_t>(t0) * heads + static_cast<int64_t>(hd / p.G) * n * p.G + r;
        const int64_t unit = at * D + ((lane ^ (D == 128 ? r & 7 : (r >> 1) & 3)) << 4);
        *reinterpret_cast<uint4*>(p.qa + unit) = wa;
        *reinterpret_cast<uint4*>(p.qb + unit) = wb;
        // codes hold neither NaN nor infinity: the row's scale does (the rotation has spread a NaN over the row)
        if (lane == 0) p.eq[at] = x[0] == x[0] && e < INFINITY ? e * 0.00390625f : NAN;
    }
}

template <int D, bool V8, bool F16>
__global__ void __launch_bounds__(Lay<D, V8>::NTHREADS, 1) chunk_sm100_kernel(const Params p, const __grid_constant__ CUtensorMap vmap) {
    using L = Lay<D, V8>;
    constexpr int TERMS = F16 && !V8 ? 2 : 1;      // of P
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = static_cast<uint32_t>(__cvta_generic_to_shared(smem_raw));
    const uint32_t base = (raw + 1023u) & ~1023u;
    if (base - raw > static_cast<uint32_t>(L::SLACK)) {   // the map would not fit: refuse, loudly
        if (threadIdx.x == 0) atomicExch(p.status, FOLD_ERR_LAUNCH);
        return;
    }
    uint8_t* smem = smem_raw + (base - raw);
    int* s_scan = reinterpret_cast<int*>(smem + L::SM_MISC);
    int* s_walk = s_scan + 12;
    int* s_flag = s_scan + 16;
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(s_scan + 18);
    auto bar = [&](int i) { return base + L::SM_BAR + 8 * i; };
    volatile int* abort_flag = s_flag;
    volatile int* last_flag = s_flag + 1;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        s_flag[0] = s_flag[1] = 0;
        s_walk[0] = -1;
        for (int i = 0; i < L::NK; ++i) {
            mbar_init(bar(B_KFULL + i), 1);
            mbar_init(bar(B_KEMPTY + i), 1 + 4);      // the tile's logits are out, and the softmax warps have its scales
        }
        for (int i = 0; i < L::NV; ++i) {
            mbar_init(bar(B_VFULL + i), 1);
            mbar_init(bar(B_VEMPTY + i), V8 ? 4 : 1);
            mbar_init(bar(B_VREADY + i), V8 ? 4 : 1);
        }
        mbar_init(bar(B_SFULL), 1);
        mbar_init(bar(B_SEMPTY), 128);
        mbar_init(bar(B_PREADY), 128);
        mbar_init(bar(B_ODONE), 1);
        mbar_init(bar(B_QFULL), 1);
        mbar_init(bar(B_QEMPTY), 1);
        mbar_init(bar(B_PIECE), 128);
        mbar_init(bar(B_JOINED), L::N_JOIN);
        mbar_init(bar(B_CEMPTY), 1);
        mbar_init(bar(B_CEMPTY + 1), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;"
                     ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(s_tmem))) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // ---- this CTA's share of the list: a block scan over the requests, twice (the total, then the place) ----
    int64_t total = 0;
    int n_cta = 1;
    int64_t g0 = 0, g1 = 0;
    Geo mg = {};
    int64_t mine = 0;
    for (int pass = 0; pass < 2; ++pass) {
        int64_t run = 0;
        for (int b0 = 0; b0 < p.batch; b0 += L::NTHREADS) {
            const int b = b0 + tid;
            if (pass == 0 || p.batch > L::NTHREADS) {
                mine = 0;
                if (b < p.batch) {
                    mg = geo_of(p, b);
                    mine = mg.nt ? static_cast<int64_t>(mg.nt + ITEM_TILES) * p.hkv : 0;
                    if (mg.n < 0 || (mg.wide && !p.others)) atomicExch(p.status, FOLD_ERR_ARGUMENT);   // counts the host did not plan for
                }
            }
            int x = static_cast<int>(mine);      // (a request's places fit 31 bits: 2^30 keys are 2^23 tiles, of 128 heads)
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            __syncthreads();
            if (lane == 31) s_scan[warp] = x;
            __syncthreads();
            int64_t before = 0, sum = 0;
            for (int wi = 0; wi < L::NTHREADS / 32; ++wi) {
                if (wi < warp) before += s_scan[wi];
                sum += s_scan[wi];
            }
            const int64_t at = run + before + x - mine;
            if (pass == 1 && mine > 0 && g0 >= at && g0 < at + mine && g0 < g1) {
                const int per = mg.nt + ITEM_TILES, off = static_cast<int>(g0 - at);
                s_walk[0] = b;
                s_walk[1] = off / per;
                s_walk[2] = off % per;
            }
            run += sum;
        }
        total = run;
        if (pass == 0) {
            n_cta = static_cast<int>(max(static_cast<int64_t>(1), min(static_cast<int64_t>(gridDim.x), (total + MIN_TILES + ITEM_TILES - 1) / (MIN_TILES + ITEM_TILES))));
            if (static_cast<int>(blockIdx.x) < n_cta) {
                g0 = share_start(total, n_cta, blockIdx.x);
                g1 = share_start(total, n_cta, blockIdx.x + 1);
            }
        }
    }
    __syncthreads();
    Walk w;
    w.b = w.b0 = s_walk[0];
    w.h = s_walk[1];
    w.v = s_walk[2];
    w.left = w.b < 0 ? 0 : static_cast<int>(g1 - g0);
    w.segment = -1;
    w.kept = reinterpret_cast<const Geo*>(smem + L::SM_GEO);
    w.start = g0 - w.v;
    if (w.left > 0) {
        w.g = geo_of(p, w.b);
        if (tid < N_GEO && w.b + tid < p.batch) reinterpret_cast<Geo*>(smem + L::SM_GEO)[tid] = geo_of(p, w.b + tid);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;

    const int np = BN / p.piece;
    // Whether any new token sees a key of [a, a + len): what is loaded; the rest of a tile's rows are masked in
    // the logits and zeroed in V, whatever the pool (or the ring) holds there
    auto wanted = [&](const Geo& g, int a, int len) { return a < g.L && (a + len - 1 > g.first - p.window || a < p.sinks); };
    auto pool_row = [&](const Walk& x, int pos) -> int64_t {
        const int pg = __ldg(p.table + static_cast<int64_t>(x.b) * p.ppr + pos / p.page_size);
        return (static_cast<int64_t>(pg) * p.hkv + x.h) * p.page_size + pos % p.page_size;
    };

    // A segment's piece: whole items alternate between two slots, the item the share starts in and the one it
    // ends in keep theirs for whoever joins them. A whole item of 128-row groups needs none. A piece is
    // [D / 4 units][128 rows] of four channels, so that a warp's store is 512 bytes in a row, then m and l.
    auto is_whole = [&](const Walk& x) { return x.t0 == 0 && x.t1 == x.g.nt; };
    auto slot_of = [&](int c, int k) { return p.parts + (static_cast<int64_t>(SLOTS) * c + k) * (128 * D + 256); };
    // Join a (request, head)'s pieces: a row's pieces (each the copies' plain sums under one reference) are added
    // in list order and copies within, by this CTA for an item of its own, by the last CTA to get here for
    // one that several share.
    // `end`: the share's last item, which every thread of the CTA joins once nothing else is left to do.
    auto join = [&](const Walk& x, int& joins, auto end) {
        constexpr bool END = decltype(end)::value;
        const int R = x.g.n * p.G, copies = copies_of(R), rows = 128 / copies;
        const bool whole = is_whole(x);
        if (whole && copies == 1) return;
        const int jl = END ? tid : (warp - L::W_JOIN) * 32 + lane;
        constexpr int NJ = END ? L::NTHREADS : 32 * L::N_JOIN;
        if (!END) {
            Walk y = x;
            if (!y.next(p)) return;
            mbar_wait(bar(B_PIECE), joins & 1, abort_flag, p.status);
        }
        int c_first = blockIdx.x, c_last = blockIdx.x;
        bool mine = true;
        if (!whole) {
            c_first = share_of(total, n_cta, x.start + ITEM_TILES);
            c_last = share_of(total, n_cta, x.start + ITEM_TILES + x.g.nt - 1);
            __threadfence();
            if (jl == 0) *last_flag = atomicAdd(p.counters + static_cast<int64_t>(x.b) * p.hkv + x.h, 1) == c_last - c_first;
            if (END) __syncthreads();
            else if (L::N_JOIN > 1) asm volatile("bar.sync 2, 128;" ::: "memory");
            else __syncwarp();
            mine = *last_flag != 0;
            __threadfence();
        }
        if (mine) {
            auto piece = [&](int c) { return whole ? slot_of(c, 2 + (joins & 1)) : slot_of(c, c == c_first ? 1 : 0); };
            auto pk2 = [](float a, float b2) { return F16 ? pack_f16x2(a, b2) : pack_bf16x2(a, b2); };
            const int n_work = R * (D / 8);
            for (int i = jl; i < n_work; i += NJ) {
                const int row = i % R, u = i / R;      // 8 channels of a row
                float mm = -INFINITY, ll = 0.f;
                if (!whole) {
                    for (int c = c_first; c <= c_last; ++c) mm = fmaxf(mm, __ldcg(piece(c) + 128 * D + row));
                    if (mm == -INFINITY) mm = 0.f;
                }
                float4 a0 = make_float4(0.f, 0.f, 0.f, 0.f), a1 = a0;
                for (int c = c_first; c <= c_last; ++c) {
                    const float* pc = piece(c);
                    const float4* src = reinterpret_cast<const float4*>(pc) + 2 * u * 128 + row;
                    float4 v0[4], v1[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (k < copies) {
                            v0[k] = __ldcg(src + k * rows);
                            v1[k] = __ldcg(src + k * rows + 128);
                        }
                    const float lc = __ldcg(pc + 128 * D + 128 + row);
                    const float fc = whole ? 1.f : ex2f(__ldcg(pc + 128 * D + row) - mm);
                    ll = fmaf(lc, fc, ll);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (k < copies) {
                            a0.x = fmaf(v0[k].x, fc, a0.x); a0.y = fmaf(v0[k].y, fc, a0.y); a0.z = fmaf(v0[k].z, fc, a0.z); a0.w = fmaf(v0[k].w, fc, a0.w);
                            a1.x = fmaf(v1[k].x, fc, a1.x); a1.y = fmaf(v1[k].y, fc, a1.y); a1.z = fmaf(v1[k].z, fc, a1.z); a1.w = fmaf(v1[k].w, fc, a1.w);
                        }
                }
                const float inv = ll > 0.f ? (V8 ? p.evs : 1.f) / ll : 0.f;
                uint16_t* out = p.o + static_cast<int64_t>(x.g.tok0 + row / p.G) * p.o_st + static_cast<int64_t>(x.h * p.G + row % p.G) * p.o_sh + 8 * u;
                *reinterpret_cast<uint4*>(out) = make_uint4(pk2(a0.x * inv, a0.y * inv), pk2(a0.z * inv, a0.w * inv),
                                                            pk2(a1.x * inv, a1.y * inv), pk2(a1.z * inv, a1.w * inv));
            }
        }
        if (END) return;
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_JOINED));
        if (L::N_JOIN > 1 && !whole) asm volatile("bar.sync 2, 128;" ::: "memory");   // the flag has been read
        ++joins;
    };

    if (warp == 0 || warp == 3) {
        // ================= producers: a lane per piece of the tile =================
        const bool is_k = warp == 0;
        int j = 0;
        while (w.next(p)) {
            for (int t = w.t0; t < w.t1; ++t, ++j) {
                const int s = j % (is_k ? L::NK : L::NV), round = j / (is_k ? L::NK : L::NV);
                const int pos = w.pos(p, t) + lane * p.piece;
                const bool mine = lane < np && wanted(w.g, pos, p.piece) && !*abort_flag;   // (nothing new once a wait ran out)
                const int64_t row = mine ? pool_row(w, pos) : 0;
                const int count = __popc(__ballot_sync(0xffffffffu, mine));
                const uint32_t full = bar((is_k ? B_KFULL : B_VFULL) + s);
                if (lane == 0) {
                    if (round > 0) mbar_wait(bar((is_k ? B_KEMPTY : B_VEMPTY) + s), (round - 1) & 1, abort_flag, p.status);
                    mbar_expect_tx(full, static_cast<uint32_t>(count) * p.piece * (2 * D + (is_k ? 2 : 0)));
                }
                __syncwarp();
                if (mine) {
                    const uint32_t r0 = lane * p.piece;
                    if (is_k) {
                        const uint32_t dst = base + L::SM_K + s * L::KSLOT + r0 * D;
                        bulk_load(dst, p.ka + row * D, p.piece * D, full);
                        bulk_load(dst + L::PLANE, p.kb + row * D, p.piece * D, full);
                        bulk_load(base + L::SM_EK + s * 256 + r0 * 2, p.ek + row, p.piece * 2, full);
                    } else if (V8) {
                        const uint32_t dst = base + L::SM_V + s * L::VSLOT + r0 * D;
                        bulk_load(dst, p.va + row * D, p.piece * D, full);
                        bulk_load(dst + L::PLANE, p.vb + row * D, p.piece * D, full);
                    } else {
                        for (int c = 0; c < D / 64; ++c)
                            tma_load_2d(base + L::SM_V + s * L::VSLOT + c * 16384 + r0 * 128, &vmap, 64 * c, static_cast<int>(row), full);
                    }
                }
            }
        }
    } else if (warp == 1) {
        // ================= MMA issuer =================
        if (lane == 0) {
            constexpr uint32_t ID_S = instr_desc(2, 1, 1, 0, 0, 128, 128);                             // s8 x s8 -> s32
            constexpr uint32_t ID_PV = instr_desc(1, V8 ? 0 : 1, V8 ? 0 : 1, 0, 1, D, 128);            // P x V, V MN-major
            constexpr uint32_t SW = D == 128 ? 2 : 4, SBO = 8 * D;
            const uint64_t qa = smem_desc(base + L::SM_Q, 16, SBO, SW), qb = smem_desc(base + L::SM_Q + L::PLANE, 16, SBO, SW);
            int j = 0;
            while (w.next(p)) {
                mbar_wait(bar(B_QFULL), w.segment & 1, abort_flag, p.status);
                auto issue_pv = [&](int jj, bool acc) {
                    const int vs = jj % L::NV;
                    mbar_wait(bar(B_PREADY), jj & 1, abort_flag, p.status);
                    if (V8) mbar_wait(bar(B_VREADY + (jj & 1)), (jj >> 1) & 1, abort_flag, p.status);
                    else mbar_wait(bar(B_VREADY + vs), (jj / L::NV) & 1, abort_flag, p.status);
                    tc_fence_after();
                    const uint32_t vt = base + (V8 ? L::SM_V16 + (jj & 1) * 2 * L::PLANE : L::SM_V + vs * L::VSLOT);
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks)     // 16 keys per step
                        mma_ts(tmem + T_O, tmem + T_P + 8 * ks, smem_desc(vt + ks * 2048, 16384, 1024, 2), ID_PV, acc || ks > 0);
                    if (TERMS == 2) {
#pragma unroll
                        for (int ks = 0; ks < 8; ++ks)
                            mma_ts(tmem + T_O, tmem + T_P2 + 8 * ks, smem_desc(vt + ks * 2048, 16384, 1024, 2), ID_PV, 1u);
                    }
                    tc_commit(bar(V8 ? B_CEMPTY + (jj & 1) : B_VEMPTY + vs));
                    tc_commit(bar(B_ODONE));
                };
                for (int t = w.t0; t < w.t1; ++t, ++j) {
                    const int s = j % L::NK;
                    mbar_wait(bar(B_KFULL + s), (j / L::NK) & 1, abort_flag, p.status);
                    if (j > 0) mbar_wait(bar(B_SEMPTY), (j - 1) & 1, abort_flag, p.status);
                    tc_fence_after();
                    const uint64_t ka = smem_desc(base + L::SM_K + s * L::KSLOT, 16, SBO, SW);
                    const uint64_t kb = smem_desc(base + L::SM_K + s * L::KSLOT + L::PLANE, 16, SBO, SW);
#pragma unroll
                    for (int ks = 0; ks < D / 32; ++ks) mma_i8(tmem + T_S1, qa + 2 * ks, ka + 2 * ks, ID_S, ks > 0);
#pragma unroll
                    for (int ks = 0; ks < D / 32; ++ks) mma_i8(tmem + T_S2, qa + 2 * ks, kb + 2 * ks, ID_S, ks > 0);
#pragma unroll
                    for (int ks = 0; ks < D / 32; ++ks) mma_i8(tmem + T_S2, qb + 2 * ks, ka + 2 * ks, ID_S, 1u);
                    tc_commit(bar(B_SFULL));
                    tc_commit(bar(B_KEMPTY + s));
                    if (t + 1 == w.t1) tc_commit(bar(B_QEMPTY));   // the next item's Q may land
                    if (t > w.t0) issue_pv(j - 1, t - 1 > w.t0);
                }
                // the item's last product: its epilogue waits for it
                issue_pv(j - 1, w.t1 - w.t0 > 1);
            }
        }
    } else if (warp == 2) {
        // ================= Q of each item; bf16 V: rows that no new token sees are zeroed in shared memory; 8-bit V: pieces =================
        [[maybe_unused]] int j = 0, joins = 0;
        Walk before = w;
        bool had = false;
        while (w.next(p)) {
            {
                const int R = w.g.n * p.G, copies = copies_of(R), rows = 128 / copies;
                const int64_t row0 = static_cast<int64_t>(w.g.tok0) * p.hkv * p.G + static_cast<int64_t>(w.h) * R;
                if (lane == 0 && w.segment > 0) mbar_wait(bar(B_QEMPTY), (w.segment - 1) & 1, abort_flag, p.status);
                __syncwarp();
                const bool go = !__any_sync(0xffffffffu, *abort_flag != 0);
                if (lane == 0 && go) mbar_expect_tx(bar(B_QFULL), static_cast<uint32_t>(2 * copies * R * D));
                __syncwarp();
                if (lane < 2 * copies && go)
                    bulk_load(base + L::SM_Q + (lane & 1) * L::PLANE + (lane >> 1) * rows * D, ((lane & 1) ? p.qb : p.qa) + row0 * D,
                              static_cast<uint32_t>(R * D), bar(B_QFULL));
            }
            if constexpr (V8) {
                if (had) join(before, joins, std::false_type{});     // the item before, while this one's tiles run
                before = w;
                had = true;
            } else {
                for (int t = w.t0; t < w.t1; ++t, ++j) {
                    const int s = j % L::NV, pos = w.pos(p, t);
                    mbar_wait(bar(B_VFULL + s), (j / L::NV) & 1, abort_flag, p.status);
                    if (pos + BN > w.g.L || (pos <= w.g.first - p.window && pos + BN > p.sinks)) {
                        for (int r = lane >> 4; r < BN; r += 2) {
                            if (wanted(w.g, pos + r, 1)) continue;
                            if ((lane & 15) < D / 8)
                                sts128(base + L::SM_V + s * L::VSLOT + ((lane & 15) >> 3) * 16384 + r * 128 + (lane & 7) * 16, make_uint4(0u, 0u, 0u, 0u));
                        }
                        fence_async_smem();
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(B_VREADY + s));
                }
            }
        }
    } else if (!V8 && warp >= L::W_JOIN) {
        int joins = 0;
        while (w.next(p)) join(w, joins, std::false_type{});
    } else if (warp < 8) {
        // ================= Q, softmax, epilogue: thread = TMEM lane =================
        const int wq = warp - 4, m_row = 32 * wq + lane;
        const uint32_t lane_addr = static_cast<uint32_t>(32 * wq) << 16;
        float* s_m = reinterpret_cast<float*>(smem + L::SM_ROW);
        float* s_l = s_m + 128;
        int j = 0, joins = 0;
        auto scale_of = [&](const Walk& x) {
            const int R = x.g.n * p.G, r = m_row & (128 / copies_of(R) - 1);
            return r < R ? __ldg(p.eq + static_cast<int64_t>(x.g.tok0) * p.hkv * p.G + static_cast<int64_t>(x.h) * R + r) : 0.f;
        };
        float eq_next;
        {
            Walk x = w;
            eq_next = x.next(p) ? scale_of(x) : 0.f;
        }
        while (w.next(p)) {
            const Geo& g = w.g;
            const int R = g.n * p.G;
            const int copies = copies_of(R);
            const int rows = 128 / copies;                // a copy's lanes
            const int r = m_row & (rows - 1);             // the thread's query row: token r / G, head r % G of the group
            const int copy = m_row / rows;
            const bool live = r < R;
            const float eq = eq_next;
            {   // the next item's scale, while this one's tiles run
                Walk x = w;
                eq_next = x.next(p) ? scale_of(x) : 0.f;
            }
            const int rpos = g.first + r / p.G;           // the row's position (rows past R: never written)
            if (copies > 1) {       // P's columns of the other copies' keys stay zero
                uint32_t z[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) z[i] = 0u;
                tmem_st32(tmem + lane_addr + T_P, z);
                tmem_st32(tmem + lane_addr + T_P + 32, z);
                if (TERMS == 2) {
                    tmem_st32(tmem + lane_addr + T_P2, z);
                    tmem_st32(tmem + lane_addr + T_P2 + 32, z);
                }
                tmem_wait_st();
            }
            float m_run = -INFINITY, l_run = 0.f;
            const int seg0 = j;
            // one tile: a copy's 32, 64 or 128 keys, 32 at a time
            const int n_ch = 4 / copies;
            auto tile = [&](auto one, int t) {
                constexpr bool KEEP = decltype(one)::value;
                const int nch = KEEP ? 1 : n_ch;
                const int s = j % L::NK, pos = w.pos(p, t), k0 = copy * 32 * nch;
                const bool need_mask = pos + BN - 1 > g.first || (pos <= g.L - 1 - p.window && pos + BN > p.sinks);
                const int kmax = rpos - pos, kmin = rpos - p.window + 1 - pos, ksink = p.sinks - pos;
                mbar_wait(bar(B_SFULL), j & 1, abort_flag, p.status);
                tc_fence_after();
                // Chunk c's logits over the row's scale, from S1, S2 and the keys' scales. One chunk is kept in
                // registers; more would spill (168 a thread), and are made twice instead: for the maximum and for P.
                auto logits = [&](int c, float (&x)[32]) {
                    uint32_t a[32], b2[32];
                    tmem_ld32(tmem + lane_addr + T_S1 + k0 + 32 * c, a);
                    tmem_ld32(tmem + lane_addr + T_S2 + k0 + 32 * c, b2);
                    const uint4* es = reinterpret_cast<const uint4*>(smem + L::SM_EK + s * 256 + 2 * (k0 + 32 * c));
                    const uint4 ew[4] = {es[0], es[1], es[2], es[3]};
                    tmem_wait_ld();
                    const uint32_t* ep = reinterpret_cast<const uint32_t*>(ew);
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const float ekf = __uint_as_float((e & 1) ? (ep[e >> 1] & 0xFFFF0000u) : (ep[e >> 1] << 16));
                        x[e] = static_cast<float>(static_cast<int>(a[e]) * 256 + static_cast<int>(b2[e])) * ekf;
                    }
                    if (need_mask) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            const int k = k0 + 32 * c + e;
                            if (k > kmax || (k < kmin && k >= ksink)) x[e] = -INFINITY;
                        }
                    }
                };
                auto release = [&]() {                 // the logits are in registers: the next tile's may come
                    tc_fence_before();
                    mbar_arrive(bar(B_SEMPTY));
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(B_KEMPTY + s));
                };
                float x[32];
                float mx = -INFINITY, mx1 = -INFINITY;
#pragma unroll 1
                for (int c = 0; c < nch; ++c) {
                    logits(c, x);
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        mx = max3f(mx, x[e], x[e + 1]);
                        mx1 = max3f(mx1, x[e + 2], x[e + 3]);
                    }
                }
                if (KEEP) release();
                const float m_cand = max3f(m_run, mx * eq, mx1 * eq);
                const float m_new = m_cand > m_run + LAZY ? m_cand : m_run;
                const float m_use = m_new == -INFINITY ? 0.f : m_new;
                const float alpha = m_run == -INFINITY ? 1.f : ex2f(m_run - m_use);   // nothing summed yet: nothing to rescale
                if (j > seg0) {                        // P's columns and O: the product before has read and written them
                    mbar_wait(bar(B_ODONE), (j - 1) & 1, abort_flag, p.status);
                    tc_fence_after();
                    if (__any_sync(0xffffffffu, live && alpha != 1.0f)) {
#pragma unroll 1
                        for (int c = 0; c < D / 32; ++c) {
                            uint32_t ov[32];
                            tmem_ld32(tmem + lane_addr + T_O + 32 * c, ov);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
                            tmem_st32(tmem + lane_addr + T_O + 32 * c, ov);
                        }
                    }
                }
                const float m_ref = V8 ? m_use - LIFT : m_use;
                float sum = 0.f, sum2 = 0.f;
#pragma unroll 1
                for (int c = 0; c < nch; ++c) {
                    uint32_t pk[16], lo[16];
                    if (!KEEP) {
                        logits(c, x);
                        if (c == nch - 1) release();
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const float p0 = ex2f(fmaf(x[e], eq, -m_ref)), p1 = ex2f(fmaf(x[e + 1], eq, -m_ref));
                        sum += p0;
                        sum2 += p1;
                        pk[e >> 1] = V8 ? pack_f16x2(p0, p1) : pack_bf16x2(p0, p1);
                        if (TERMS == 2)
                            lo[e >> 1] = pack_bf16x2(p0 - __uint_as_float(pk[e >> 1] << 16), p1 - __uint_as_float(pk[e >> 1] & 0xFFFF0000u));
                    }
                    tmem_st16(tmem + lane_addr + T_P + (k0 + 32 * c) / 2, pk);
                    if (TERMS == 2) tmem_st16(tmem + lane_addr + T_P2 + (k0 + 32 * c) / 2, lo);
                }
                l_run = l_run * alpha + (sum + sum2);
                m_run = m_new;
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(bar(B_PREADY));
            };
            for (int t = w.t0; t < w.t1; ++t, ++j) {
                if (copies == 4) tile(std::true_type{}, t);
                else tile(std::false_type{}, t);
            }
            // ---- epilogue: O out, or O and its statistics to a piece that another warp joins ----
            mbar_wait(bar(B_ODONE), (j - 1) & 1, abort_flag, p.status);
            tc_fence_after();
            if (copies == 1 && is_whole(w)) {       // the whole row is this thread's
                auto pk2 = [](float a, float b2) { return F16 ? pack_f16x2(a, b2) : pack_bf16x2(a, b2); };
                const float inv = l_run > 0.f ? (V8 ? p.evs : 1.f) / l_run : 0.f;
                const int row = live ? r : 0;
                uint16_t* orow = p.o + static_cast<int64_t>(g.tok0 + row / p.G) * p.o_st + static_cast<int64_t>(w.h * p.G + row % p.G) * p.o_sh;
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t ov[32];
                    tmem_ld32(tmem + lane_addr + T_O + 32 * c, ov);
                    tmem_wait_ld();
                    if (live) {
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            uint4 v;
                            v.x = pk2(__uint_as_float(ov[8 * u]) * inv, __uint_as_float(ov[8 * u + 1]) * inv);
                            v.y = pk2(__uint_as_float(ov[8 * u + 2]) * inv, __uint_as_float(ov[8 * u + 3]) * inv);
                            v.z = pk2(__uint_as_float(ov[8 * u + 4]) * inv, __uint_as_float(ov[8 * u + 5]) * inv);
                            v.w = pk2(__uint_as_float(ov[8 * u + 6]) * inv, __uint_as_float(ov[8 * u + 7]) * inv);
                            *reinterpret_cast<uint4*>(orow + 32 * c + 8 * u) = v;
                        }
                    }
                }
                tc_fence_before();
                continue;
            }
            // the copies under one reference, so that a piece is plain sums
            s_m[m_row] = m_run;
            s_l[m_row] = l_run;
            asm volatile("bar.sync 1, 128;" ::: "memory");
            float mt = -INFINITY, lt = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (k < copies) mt = fmaxf(mt, s_m[k * rows + r]);
            const float mu = mt == -INFINITY ? 0.f : mt;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (k < copies) lt = fmaf(s_l[k * rows + r], ex2f(s_m[k * rows + r] - mu), lt);
            const float f = ex2f(m_run - mu);
            float* part = slot_of(blockIdx.x, is_whole(w) ? 2 + (joins & 1) : w.t0 > 0 ? 0 : 1);
            if (live && copy == 0) {
                part[128 * D + r] = mt;
                part[128 * D + 128 + r] = lt;
            }
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
                uint32_t ov[32];
                tmem_ld32(tmem + lane_addr + T_O + 32 * c, ov);
                tmem_wait_ld();
                if (live) {
                    uint4* d = reinterpret_cast<uint4*>(part) + 8 * c * 128 + m_row;
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        d[128 * u] = make_uint4(__float_as_uint(__uint_as_float(ov[4 * u]) * f), __float_as_uint(__uint_as_float(ov[4 * u + 1]) * f),
                                          __float_as_uint(__uint_as_float(ov[4 * u + 2]) * f), __float_as_uint(__uint_as_float(ov[4 * u + 3]) * f));
                }
            }
            tc_fence_before();
            // (the arrival releases the piece to the joining warps; what other CTAs see is their fence's matter)
            // one piece at a time is handed over: the joining warp tells phases apart by their parity, and the slot
            // of two pieces back is then free for the next
            if (joins >= 1) mbar_wait(bar(B_JOINED), (joins - 1) & 1, abort_flag, p.status);
            if (m_row == 0) s_walk[3] = joins;    // (the share's last piece is found by it)
            mbar_arrive(bar(B_PIECE));
            ++joins;
        }
    } else {
        // ================= 8-bit V: two planes -> fp16 rows, MN-major, swizzled; dead rows are zeros =================
        int j = 0;
        const int c0 = tid - 256;
        constexpr int UPR = D / 16;             // 16-channel units a row
        while (w.next(p)) {
            for (int t = w.t0; t < w.t1; ++t, ++j) {
                const int s = j % L::NV, pos = w.pos(p, t);
                const bool cut = pos + BN > w.g.L || (pos <= w.g.first - p.window && pos + BN > p.sinks);
                mbar_wait(bar(B_VFULL + s), (j / L::NV) & 1, abort_flag, p.status);
                if (j > 1) mbar_wait(bar(B_CEMPTY + (j & 1)), ((j >> 1) - 1) & 1, abort_flag, p.status);   // the product two tiles back has read its rows
                const uint4* src = reinterpret_cast<const uint4*>(smem + L::SM_V + s * L::VSLOT);
                uint4* dst = reinterpret_cast<uint4*>(smem + L::SM_V16 + (j & 1) * 2 * L::PLANE);
                // One unit a turn, the next one's loads ahead of its arithmetic, and not unrolled: what the warps of a
                // scheduler run must fit its instruction cache together (four units a turn took 94 us where this takes 84)
                uint4 a = src[c0], b2 = src[L::PLANE / 16 + c0];
#pragma unroll 1
                for (int i = c0; i < BN * UPR; i += 128) {
                    const int r = i / UPR, u = i % UPR;
                    const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b2.x, b2.y, b2.z, b2.w};
                    if (i + 128 < BN * UPR) {
                        a = src[i + 128];
                        b2 = src[L::PLANE / 16 + i + 128];
                    }
                    uint32_t o[8];
                    const bool keep = !cut || wanted(w.g, pos + r, 1);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        uint32_t ha, hb, x;
                        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(ha) : "h"(static_cast<uint16_t>(aw[k >> 1] >> (16 * (k & 1)))));
                        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hb) : "h"(static_cast<uint16_t>(bw[k >> 1] >> (16 * (k & 1)))));
                        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(x) : "r"(hb), "r"(0x30003000u), "r"(ha));   // a + b / 8
                        o[k] = keep ? x : 0u;
                    }
                    uint4* row = dst + (u >> 2) * 1024 + r * 8;
                    const int ch = 2 * (u & 3);
                    row[ch ^ (r & 7)] = make_uint4(o[0], o[1], o[2], o[3]);
                    row[(ch + 1) ^ (r & 7)] = make_uint4(o[4], o[5], o[6], o[7]);
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(bar(B_VREADY + (j & 1)));
                    mbar_arrive(bar(B_VEMPTY + s));
                }
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
    while (w.next(p)) {}      // (the issuing warp's other lanes have not walked)
    if (w.segment >= 0) {     // w is the share's last segment
        int joins = s_walk[3];
        join(w, joins, std::true_type{});
    }
    if (warp == 1) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

}  // namespace csm100
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

// the workspace: pieces, Q's planes and scales, counters (bytes from its start, each on 16)
struct Work {
    int64_t parts, qa, qb, eq, counters, total;
};
Work chunk_work(int batch, int total, int heads, int hkv, int D, int ctas) {
    auto up = [](int64_t x) { return (x + 15) / 16 * 16; };
    const int64_t rows = static_cast<int64_t>(total) * heads;
    Work w;
    w.parts = 0;
    w.qa = up(static_cast<int64_t>(csm100::SLOTS) * ctas * (128 * D + 256) * 4);
    w.qb = up(w.qa + rows * D);
    w.eq = up(w.qb + rows * D);
    w.counters = up(w.eq + rows * 4);
    w.total = up(w.counters + static_cast<int64_t>(batch) * hkv * 4);
    return w;
}

template <int D, bool V8, bool F16>
int launch(const csm100::Params& p, const CUtensorMap& vmap, int ctas, cudaStream_t st) {
    using L = csm100::Lay<D, V8>;
    const int heads = p.hkv * p.G, rpb = NT / (D / 16);
    const int64_t rows = static_cast<int64_t>(p.total) * heads;
    csm100::chunk_q_kernel<D, F16><<<static_cast<unsigned>((rows + rpb - 1) / rpb), NT, 0, st>>>(p, heads, rows);
    auto kern = csm100::chunk_sm100_kernel<D, V8, F16>;
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::BYTES);
    kern<<<ctas, L::NTHREADS, L::BYTES, st>>>(p, vmap);
    return check_launch("fold_chunk_sm100");
}

}  // namespace

extern "C" int64_t fold_chunk_workspace_bytes(int batch, int total, int n_heads, int n_kv_heads, int head_dim, int ctas) {
    if (batch <= 0 || total <= 0 || n_heads <= 0 || n_kv_heads <= 0 || head_dim <= 0 || ctas <= 0) return 0;
    return chunk_work(batch, total, n_heads, n_kv_heads, head_dim, ctas).total;
}

extern "C" int fold_chunk_sm100(const void* q, int64_t q_token_stride, int64_t q_head_stride, void* o, int64_t o_token_stride, int64_t o_head_stride,
                                int is_f16, const int32_t* cu_seqlens, const int32_t* seq_lens, int batch, int total, int n_heads, int n_kv_heads,
                                int head_dim, const int32_t* page_table, int pages_per_request, int page_size, int64_t pool_rows, const int8_t* ka,
                                const int8_t* kb, const void* va, const void* vb, const void* ek, float v_scale, int window, int sinks, int others, int ctas,
                                void* workspace, int64_t workspace_bytes, int32_t* status, void* stream) {
    FOLD_CHECK_ARG(head_dim == 64 || head_dim == 128, "head_dim %d: the cache holds 64 or 128", head_dim);
    FOLD_CHECK_ARG(q && o && cu_seqlens && seq_lens && page_table && ka && kb && va && ek && workspace && status, "fold_chunk_sm100: null pointer");
    FOLD_CHECK_ARG(n_kv_heads > 0 && n_heads % n_kv_heads == 0 && n_heads / n_kv_heads <= 128, "fold_chunk_sm100: %d query heads over %d KV heads (128 a group at most)", n_heads, n_kv_heads);
    FOLD_CHECK_ARG(batch > 0 && total > 0 && pages_per_request > 0 && ctas > 0 && pool_rows > 0 && pool_rows < (1ll << 31),
                   "fold_chunk_sm100: %d requests, %d tokens, %d pages a request, %d CTAs, %lld pool rows", batch, total, pages_per_request, ctas, static_cast<long long>(pool_rows));
    FOLD_CHECK_ARG(page_size > 0 && page_size % 16 == 0, "fold_chunk_sm100: pages of %d keys (a multiple of 16)", page_size);
    FOLD_CHECK_ARG(window > 0 && window <= FOLD_MAX_WINDOW && sinks >= 0 && sinks <= FOLD_MAX_WINDOW, "fold_chunk_sm100: a window of %d keys and %d sinks", window, sinks);
    FOLD_CHECK_ARG(q_token_stride % 8 == 0 && q_head_stride % 8 == 0 && o_token_stride % 8 == 0 && o_head_stride % 8 == 0 &&
                       reinterpret_cast<uintptr_t>(q) % 16 == 0 && reinterpret_cast<uintptr_t>(o) % 16 == 0 &&
                       reinterpret_cast<uintptr_t>(workspace) % 16 == 0 && reinterpret_cast<uintptr_t>(ka) % 16 == 0 && reinterpret_cast<uintptr_t>(kb) % 16 == 0 &&
                       reinterpret_cast<uintptr_t>(va) % 16 == 0 && reinterpret_cast<uintptr_t>(vb) % 16 == 0 && reinterpret_cast<uintptr_t>(ek) % 16 == 0,
                   "fold_chunk_sm100: rows must be 16-byte aligned");
    const Work w = chunk_work(batch, total, n_heads, n_kv_heads, head_dim, ctas);
    FOLD_CHECK_ARG(workspace_bytes >= w.total, "fold_chunk_sm100: a workspace of %lld bytes, %lld needed", static_cast<long long>(workspace_bytes),
                   static_cast<long long>(w.total));
    FOLD_CHECK_ARG((static_cast<int64_t>(total) * n_heads * head_dim / 16 + NT - 1) / NT < (1ll << 31), "fold_chunk_sm100: %d tokens of %d heads in one call", total, n_heads);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    csm100::Params p;
    p.qa = reinterpret_cast<int8_t*>(ws + w.qa); p.qb = reinterpret_cast<int8_t*>(ws + w.qb); p.eq = reinterpret_cast<float*>(ws + w.eq);
    p.q = static_cast<const uint16_t*>(q); p.q_st = q_token_stride; p.q_sh = q_head_stride;
    p.o = static_cast<uint16_t*>(o); p.o_st = o_token_stride; p.o_sh = o_head_stride;
    p.cu = cu_seqlens; p.lens = seq_lens; p.table = page_table;
    p.batch = batch; p.hkv = n_kv_heads; p.G = n_heads / n_kv_heads; p.ppr = pages_per_request; p.page_size = page_size;
    p.piece = 128;
    while (page_size % p.piece) p.piece >>= 1;
    const int64_t cap = static_cast<int64_t>(pages_per_request) * page_size;
    p.max_keys = static_cast<int>(cap < (1 << 30) ? cap : (1 << 30));
    p.total = total; p.window = window; p.sinks = sinks;
    p.ka = ka; p.kb = kb; p.ek = static_cast<const uint16_t*>(ek);
    p.va = static_cast<const uint8_t*>(va); p.vb = static_cast<const uint8_t*>(vb); p.evs = v_scale;
    p.counters = reinterpret_cast<int*>(ws + w.counters); p.parts = reinterpret_cast<float*>(ws + w.parts); p.status = status; p.others = others;
    CUtensorMap vmap = {};
    if (!vb) {   // a bf16 V: rows of the pool, boxes of 64 channels of a piece's keys
        EncodeFn fn = encode_fn();
        cuuint64_t dims[2] = {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(pool_rows)};
        cuuint64_t strides[1] = {static_cast<cuuint64_t>(head_dim) * 2};
        cuuint32_t box[2] = {64u, static_cast<cuuint32_t>(p.piece)};
        cuuint32_t estr[2] = {1, 1};
        if (!fn || fn(&vmap, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(va), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
            set_error("fold_chunk_sm100: cuTensorMapEncodeTiled failed");
            return FOLD_ERR_LAUNCH;
        }
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (head_dim == 64) {
        if (vb) return is_f16 ? launch<64, true, true>(p, vmap, ctas, st) : launch<64, true, false>(p, vmap, ctas, st);
        return is_f16 ? launch<64, false, true>(p, vmap, ctas, st) : launch<64, false, false>(p, vmap, ctas, st);
    }
    if (vb) return is_f16 ? launch<128, true, true>(p, vmap, ctas, st) : launch<128, true, false>(p, vmap, ctas, st);
    return is_f16 ? launch<128, false, true>(p, vmap, ctas, st) : launch<128, false, false>(p, vmap, ctas, st);
}
