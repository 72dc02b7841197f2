// The paged cache a piece at a time: block tables and slots from request lengths, any number of
// new tokens per request into the pool, and pool rows back out as 16- or 32-bit keys and values.
//
// A token's slot is page * page_size + offset, the same for every head and layer that share the
// table; its pool row for KV head h is (page * n_kv_heads + h) * page_size + offset. A slot of -1
// stands for "no place": writers skip it, readers return zeros.
#include "cache_common.cuh"
#include "fold_b200.h"

namespace fold {

__device__ __forceinline__ int64_t slot_row(int slot, int page_size, int hkv, int h, int& off) {
    off = slot % page_size;
    return (static_cast<int64_t>(slot / page_size) * hkv + h) * page_size + off;
}

// ------------------------------------------------- block tables and slots ----
// One CTA per request. Where its new pages start in the free list is the number of pages that the
// requests before it take, which every CTA adds up for itself (two integers a request, in L2 after
// the first CTA): no scan pass, no order between CTAs, one launch. A step's work is a few kilobytes,
// so the launch is what it costs: 3 us for 256 requests of one token, 12 for 48 prompts of up to 4096 tokens and
// pages of 16 (a CTA a prompt writes its slots 128 at a time); 14 us a call with the host's part of it.
constexpr int TB_THREADS = 128;

__device__ __forceinline__ int pages_of(int n, int page_size) { return (n + page_size - 1) / page_size; }

__global__ void __launch_bounds__(TB_THREADS) build_tables_kernel(const int* __restrict__ cu, const int* __restrict__ lens, int batch,
                                                                  int* table, int ppr, int page_size, int total,
                                                                  const int* __restrict__ free_pages, int n_free,
                                                                  const int* __restrict__ taken, int* __restrict__ slots,
                                                                  int* __restrict__ lens_out, int* __restrict__ taken_out) {
    __shared__ int s_part[TB_THREADS / 32];
    const int b = blockIdx.x, tid = threadIdx.x;
    int before = 0;
    if (free_pages) {
        for (int i = tid; i < b; i += TB_THREADS) {
            const int len = lens[i], n = max(cu[i + 1] - cu[i], 0);
            before += pages_of(len + n, page_size) - pages_of(len, page_size);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
        if ((tid & 31) == 0) s_part[tid >> 5] = before;
        __syncthreads();
        before = *taken;
        for (int i = 0; i < TB_THREADS / 32; ++i) before += s_part[i];
    }
    const int t0 = cu[b], n = max(cu[b + 1] - t0, 0), len = lens[b];
    const int p0 = pages_of(len, page_size), p1 = pages_of(len + n, page_size);
    int* row = table + static_cast<int64_t>(b) * ppr;
    // the request's j-th page, or -1 where the table or the pool ends
    auto page = [&](int j) -> int {
        if (j < 0 || j >= ppr) return -1;
        if (!free_pages || j < p0) return row[j];
        const int at = before + j - p0;
        return at >= 0 && at < n_free ? free_pages[at] : -1;
    };
    if (free_pages)
        for (int j = p0 + tid; j < min(p1, ppr); j += TB_THREADS) {
            const int pg = page(j);
            if (pg >= 0) row[j] = pg;
        }
    for (int i = tid; i < n; i += TB_THREADS) {
        const int t = t0 + i, pos = len + i;
        if (t < 0 || t >= total) continue;
        const int pg = pos < 0 ? -1 : page(pos / page_size);
        slots[t] = pg < 0 ? -1 : pg * page_size + pos % page_size;
    }
    if (tid == 0) {
        lens_out[b] = len + n;
        if (b == batch - 1 && taken_out) *taken_out = free_pages ? before + p1 - p0 : *taken;
    }
    // rows of `slots` that no request covers
    if (b == 0)
        for (int t = tid; t < min(t0, total); t += TB_THREADS) slots[t] = -1;
    if (b == batch - 1)
        for (int t = max(t0 + n, 0) + tid; t < total; t += TB_THREADS) slots[t] = -1;
}

// ------------------------------------------------------ tokens in and out ----
// Bytes are all these two move: a thread's 16-byte units are its only accesses, a row's lanes are
// neighbours, and no row waits for another. 16384 tokens of 8 heads, D=128, a bf16 V: written in 30 us and read as fp32
// in 34, 5.3 TB/s; 256 tokens: 3 us each, the launch.
template <int D, bool V8, bool F16>
__global__ void __launch_bounds__(NT) write_tokens_kernel(const uint16_t* __restrict__ k, const uint16_t* __restrict__ v, int64_t k_st,
                                                          int64_t k_sh, int64_t v_st, int64_t v_sh, const int* __restrict__ slots,
                                                          int64_t n_rows, int hkv, int page_size, int64_t pool_rows, int8_t* ka, int8_t* kb, void* va,
                                                          void* vb, __nv_bfloat16* ek, float ievs) {
    constexpr int TPR = D / 16, RPB = NT / TPR;
    const int lane = threadIdx.x % TPR;
    const int64_t r = static_cast<int64_t>(blockIdx.x) * RPB + threadIdx.x / TPR;
    const int64_t rr = r < n_rows ? r : 0;      // the row's shuffles want every lane
    const int64_t t = rr / hkv;
    const int h = static_cast<int>(rr % hkv);
    const int slot = slots[t];
    // a slot outside the pool is no place either (a page's rows end (hkv * page_size) after they begin)
    const bool ok = r < n_rows && slot >= 0 && (static_cast<int64_t>(slot / page_size) + 1) * hkv * page_size <= pool_rows;
    float xk[16], xv[16];
    uint4 wk[2], wv[2];
    load16<F16>(k + t * k_st + h * k_sh + lane * 16, xk, wk);
    load16<F16>(v + t * v_st + h * v_sh + lane * 16, xv, wv);
    int off;
    const int64_t prow = slot_row(ok ? slot : 0, page_size, hkv, h, off);
    rotate16<TPR>(xk, lane, D == 64 ? 0.125f : 0.08838834764831845f);
    put_key<D>(xk, ka, kb, ek, prow, off, lane, ok);
    put_value<D, V8, F16>(xv, wv, va, vb, prow, lane, ok, ievs);
}

struct Planes {
    const int8_t* ka;
    const int8_t* kb;
    const uint16_t* ek;
    const uint8_t* va;
    const uint8_t* vb;
    float evs;
};

// A pool row's 16 channels of this lane: the key in its own basis (the codes' value is exact in fp32,
// the rotation is 7 rounded adds and a multiply) and the value.
template <int D, bool V8>
__device__ __forceinline__ void load_row(const Planes& p, int64_t prow, int off, int lane, bool ok, float (&xk)[16], float (&xv)[16]) {
    constexpr int LANES = D / 16;
    constexpr int NU = LANES < 8 ? LANES : 8;
    constexpr int SH = NU == 8 ? 0 : (NU == 4 ? 1 : (NU == 2 ? 2 : 3));
    const uint4 z = make_uint4(0u, 0u, 0u, 0u);
    uint4 a = z, b = z, v0 = z, v1 = z;
    float e = 0.f;
    if (ok) {
        const int64_t addr = prow * D + ((lane ^ ((off >> SH) & (NU - 1))) * 16);
        a = __ldg(reinterpret_cast<const uint4*>(p.ka + addr));
        b = __ldg(reinterpret_cast<const uint4*>(p.kb + addr));
        e = bf16_bits_to_float(__ldg(p.ek + prow));
        if constexpr (V8) {
            v0 = __ldg(reinterpret_cast<const uint4*>(p.va + prow * D + lane * 16));
            v1 = __ldg(reinterpret_cast<const uint4*>(p.vb + prow * D + lane * 16));
        } else {
            const uint4* s = reinterpret_cast<const uint4*>(p.va + (prow * D + lane * 16) * 2);
            v0 = __ldg(s);
            v1 = __ldg(s + 1);
        }
    }
    const uint32_t* aw = reinterpret_cast<const uint32_t*>(&a);
    const uint32_t* bw = reinterpret_cast<const uint32_t*>(&b);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int sa = static_cast<int8_t>(aw[i >> 2] >> (8 * (i & 3))), sb = static_cast<int8_t>(bw[i >> 2] >> (8 * (i & 3)));
        xk[i] = __fmul_rn(static_cast<float>(sa * 256 + sb) * 0.00390625f, e);
    }
    rotate16<LANES>(xk, lane, D == 64 ? 0.125f : 0.08838834764831845f);
    const uint32_t* w0 = reinterpret_cast<const uint32_t*>(&v0);
    const uint32_t* w1 = reinterpret_cast<const uint32_t*>(&v1);
    if constexpr (V8) {
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            uint32_t ha, hb;
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(ha) : "h"(static_cast<uint16_t>(w0[i >> 2] >> (8 * (i & 3)))));
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hb) : "h"(static_cast<uint16_t>(w1[i >> 2] >> (8 * (i & 3)))));
            const float2 fa = __half22float2(*reinterpret_cast<const __half2*>(&ha)), fb = __half22float2(*reinterpret_cast<const __half2*>(&hb));
            xv[i] = __fmul_rn(__fadd_rn(fa.x, fb.x * 0.125f), p.evs);
            xv[i + 1] = __fmul_rn(__fadd_rn(fa.y, fb.y * 0.125f), p.evs);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t w = i < 8 ? w0[i >> 1] : w1[(i - 8) >> 1];
            xv[i] = bf16_bits_to_float(static_cast<uint16_t>((i & 1) ? w >> 16 : w & 0xFFFF));
        }
    }
}

enum { OUT_F32 = 0, OUT_BF16 = 1, OUT_F16 = 2 };

__device__ __forceinline__ float to_f16_range(float x) {
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(-65504.f));
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(65504.f));
    return x;
}

// A row's channels as 16-bit values, 16 to a lane.
template <int OUT>
__device__ __forceinline__ void store16(void* base, int64_t at, const float (&x)[16]) {
    static_assert(OUT != OUT_F32, "fp32 rows are store_f32's");
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (OUT == OUT_BF16) w[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
        // the pool holds bf16's range: fp16 takes what it can, and a NaN stays one
        else w[i] = pack_f16x2(to_f16_range(x[2 * i]), to_f16_range(x[2 * i + 1]));
    }
    uint4* d = reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + at);
    d[0] = make_uint4(w[0], w[1], w[2], w[3]);
    d[1] = make_uint4(w[4], w[5], w[6], w[7]);
}

// A row's fp32 channels, 16 to a lane, stored by whole cache lines: within groups of four lanes the 4 x 4 matrix
// of 16-byte units is transposed (lane l's unit t to lane t's unit l), so that a group's store is 64 bytes in a row.
template <int TPR>
__device__ __forceinline__ void store_f32(float* row, int lane, bool ok, const float (&x)[16]) {
    float4 u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
    const int q = lane & 3;
    auto swap = [](float4& a, float4& b, bool upper, int off) {     // exchange the lower lane's b with the upper lane's a
        const float4 give = upper ? a : b;
        float4 got;
        got.x = __shfl_xor_sync(0xffffffffu, give.x, off);
        got.y = __shfl_xor_sync(0xffffffffu, give.y, off);
        got.z = __shfl_xor_sync(0xffffffffu, give.z, off);
        got.w = __shfl_xor_sync(0xffffffffu, give.w, off);
        if (upper) a = got;
        else b = got;
    };
    swap(u[0], u[1], q & 1, 1);
    swap(u[2], u[3], q & 1, 1);
    swap(u[0], u[2], q & 2, 2);
    swap(u[1], u[3], q & 2, 2);
    // lane q now holds unit q of lanes 0..3 of its group
    float4* d = reinterpret_cast<float4*>(row) + (lane & ~3) * 4 + q;
    if (ok)
#pragma unroll
        for (int i = 0; i < 4; ++i) d[4 * i] = u[i];
}

template <int D, bool V8, int OUT>
__global__ void __launch_bounds__(NT) read_tokens_kernel(const int* __restrict__ slots, int64_t n_rows, int hkv, int page_size, int64_t pool_rows, const Planes p,
                                                         void* k, void* v) {
    constexpr int TPR = D / 16, RPB = NT / TPR;
    const int lane = threadIdx.x % TPR;
    const int64_t r = static_cast<int64_t>(blockIdx.x) * RPB + threadIdx.x / TPR;
    const int64_t rr = r < n_rows ? r : 0;
    const int slot = slots[rr / hkv];
    const bool ok = slot >= 0 && (static_cast<int64_t>(slot / page_size) + 1) * hkv * page_size <= pool_rows;
    int off;
    const int64_t prow = slot_row(ok ? slot : 0, page_size, hkv, static_cast<int>(rr % hkv), off);
    float xk[16], xv[16];
    load_row<D, V8>(p, prow, off, lane, ok, xk, xv);
    if constexpr (OUT == OUT_F32) {      // 64 bytes a lane, by whole lines (with every lane of the warp, for its shuffles)
        store_f32<TPR>(static_cast<float*>(k) + r * D, lane, r < n_rows, xk);
        store_f32<TPR>(static_cast<float*>(v) + r * D, lane, r < n_rows, xv);
    } else if (r < n_rows) {
        store16<OUT>(k, r * D + lane * 16, xk);
        store16<OUT>(v, r * D + lane * 16, xv);
    }
}

// ------------------------------------------------------------- the sums ----
// A chunk's share of the running V sums and means, and the lengths moved: one CTA per (KV head,
// request). Token i goes to slot i % 16 and the slots are added in order, so the sum depends on the
// chunk alone. With the tokens' places (`slots`), those without one do not count. They are a request's last
// (pages are handed out in order); where a page was missing the length stops at the last key that has a place, so that no
// reader meets a page that is not there, and past the table's end (`room` keys), where every reader stops, it moves on.
template <int D, bool F16>
__global__ void __launch_bounds__(16 * D / 4) chunk_sums_kernel(const uint16_t* __restrict__ v, int64_t v_st, int64_t v_sh, int hkv,
                                                                const int* __restrict__ cu, int total, const int* __restrict__ slots, int64_t room,
                                                                const int* __restrict__ lens_new, int* lens, float evs, float* vsum, float* vmean) {
    constexpr int TPR = D / 4;
    __shared__ float s_part[16][D];
    __shared__ int s_placed[16];
    const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x % TPR, slot = threadIdx.x / TPR;
    const int t0 = max(cu[b], 0), t1 = min(cu[b + 1], total);
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    int placed = 0;
    for (int t = t0 + slot; t < t1; t += 16) {
        if (slots && __ldg(slots + t) < 0) continue;
        ++placed;
        const uint2 w = __ldg(reinterpret_cast<const uint2*>(v + t * v_st + h * v_sh + lane * 4));
        s[0] = __fadd_rn(s[0], half_bits_to_float<F16>(static_cast<uint16_t>(w.x & 0xFFFF)));
        s[1] = __fadd_rn(s[1], half_bits_to_float<F16>(static_cast<uint16_t>(w.x >> 16)));
        s[2] = __fadd_rn(s[2], half_bits_to_float<F16>(static_cast<uint16_t>(w.y & 0xFFFF)));
        s[3] = __fadd_rn(s[3], half_bits_to_float<F16>(static_cast<uint16_t>(w.y >> 16)));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) s_part[slot][lane * 4 + i] = s[i];
    if (lane == 0) s_placed[slot] = placed;
    __syncthreads();
    int len = lens_new[b], keys = len;
    placed = 0;
    for (int i = 0; i < 16; ++i) placed += s_placed[i];
    if (slots) {
        const int n = cu[b + 1] - cu[b], before = len - n;
        if (placed < n && before + placed < room) len = before + placed;
        keys = static_cast<int>(min(static_cast<int64_t>(len), room));
    }
    if (threadIdx.x < D && placed > 0) {
        const int64_t at = (static_cast<int64_t>(b) * hkv + h) * D + threadIdx.x;
        float acc = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) acc = __fadd_rn(acc, s_part[i][threadIdx.x]);
        acc = __fadd_rn(vsum[at], acc);
        vsum[at] = acc;
        vmean[at] = __fdiv_rn(acc, __fmul_rn(static_cast<float>(keys), evs));
    }
    if (h == 0 && threadIdx.x == 0) lens[b] = len;
}

// ------------------------------------------- a chunk's keys, dequantised ----
// Long chunks attend 16-bit keys and values: every key is met by hundreds of query rows, so the
// pool's codes are turned into rows a matrix product can take once, ahead of the attention, instead
// of in every CTA that meets them (two requests of up to 26624 keys, 8 heads, D=128, an 8-bit V: 75 us beside the
// attention's 1660; bytes bound it). The rows of each request that its window (or its sinks) can see
// are laid out in whole tiles of 128 keys, requests one after another: [KV head][row][channel].
//
// chunk_plan_kernel (one CTA) lays them out: plan[b] = (keys, first row, tiles left out between the
// sinks' tiles and the window's, last position before the first query's window); keys -1: the request is
// another kernel's; then each request's first block of 256 query rows and their count, and for each 128-row tile (request, tile
// in the request).
constexpr int CP_THREADS = 256;
__global__ void __launch_bounds__(CP_THREADS) chunk_plan_kernel(const int* __restrict__ cu, const int* __restrict__ lens, int batch, int max_keys,
                                                                int window, int sinks, int rows_over, int group, int cap_tiles, int4* plan, int2* tiles, int* status) {
    __shared__ int s_warp[CP_THREADS / 32], s_warpq[CP_THREADS / 32];
    if (rows_over == 0 && threadIdx.x == 0) *status = 0;    // no other kernel of the call has a say in it
    __syncthreads();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ns = (sinks + 127) / 128;
    int* qfirst = reinterpret_cast<int*>(plan + batch);
    int base = 0, qbase = 0;
    for (int b0 = 0; b0 < batch; b0 += CP_THREADS) {
        const int b = b0 + tid;
        int klen = 0, shift = 0, nt = 0, before = -1, nq = 0;
        if (b < batch) {
            const int n = cu[b + 1] - cu[b], len = lens[b];
            nq = n > 0 && static_cast<int64_t>(n) * group > rows_over ? (n + 255) / 256 : 0;
            if (static_cast<int64_t>(n) * group <= rows_over) {
                klen = -1;                     // another kernel's
            } else if (n > 0 && len > 0) {
                klen = min(len, max_keys);
                before = klen - n - window;    // (of the keys that the table holds: the attention counts its queries back from klen)
                const int low = max(0, before + 1) / 128;
                shift = max(0, low - ns);
                nt = max(0, (klen + 127) / 128 - shift);
            }
        }
        int x = nt, xq = nq;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o), yq = __shfl_up_sync(0xffffffffu, xq, o);
            if (lane >= o) {
                x += y;
                xq += yq;
            }
        }
        if (lane == 31) {
            s_warp[warp] = x;
            s_warpq[warp] = xq;
        }
        __syncthreads();
        int add = base, sum = 0, addq = qbase, sumq = 0;
        for (int w = 0; w < CP_THREADS / 32; ++w) {
            if (w < warp) {
                add += s_warp[w];
                addq += s_warpq[w];
            }
            sum += s_warp[w];
            sumq += s_warpq[w];
        }
        if (b < batch) {
            const int first = add + x - nt;
            const bool fits = first + nt <= cap_tiles;
            if (!fits) atomicExch(status, FOLD_ERR_ARGUMENT);   // lengths the host did not plan for: the request sees nothing
            qfirst[b] = addq + xq - nq;
            plan[b] = make_int4(fits || klen < 0 ? klen : 0, first * 128, shift, before);
        }
        base += sum;
        qbase += sumq;
        __syncthreads();
    }
    if (tid == 0) qfirst[batch] = qbase;
    for (int g = tid; g < cap_tiles; g += CP_THREADS) {
        int lo = 0, hi = batch;          // the last request that starts at or before tile g
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (plan[mid].y <= g * 128) lo = mid;
            else hi = mid;
        }
        const int4 pl = plan[lo];
        const int local = g - pl.y / 128;
        tiles[g] = g < base && pl.x > 0 ? make_int2(lo, local < ns ? local : local + pl.z) : make_int2(-1, 0);
    }
}

template <int D, bool V8, int OUT>
__global__ void __launch_bounds__(NT) chunk_gather_kernel(const int4* __restrict__ plan, const int2* __restrict__ tiles,
                                                          const int* __restrict__ table, int ppr, int page_size, int hkv, int sinks, const Planes p,
                                                          int64_t rows, uint16_t* kw, uint16_t* vw) {
    constexpr int TPR = D / 16, RPB = NT / TPR, PER = 128 / RPB;
    const int g = blockIdx.x / PER, h = blockIdx.y;
    const int2 tl = tiles[g];
    if (tl.x < 0) return;
    const int lane = threadIdx.x % TPR;
    const int r = blockIdx.x % PER * RPB + threadIdx.x / TPR;
    const int pos = tl.y * 128 + r;
    // rows that no query sees (past the request's end, before its first query's window) are zeros, whatever
    // the pool holds there: their weights are 0, but 0 times a NaN is not
    const int4 pl = plan[tl.x];
    const bool ok = pos < pl.x && (pos > pl.w || pos < sinks);
    int64_t prow = 0;
    int off = 0;
    if (ok) {
        const int pg = __ldg(table + static_cast<int64_t>(tl.x) * ppr + pos / page_size);
        off = pos % page_size;
        prow = (static_cast<int64_t>(pg) * hkv + h) * page_size + off;
    }
    float xk[16], xv[16];
    load_row<D, V8>(p, prow, off, lane, ok, xk, xv);
    const int64_t at = (h * rows + static_cast<int64_t>(g) * 128 + r) * D + lane * 16;
    store16<OUT>(kw, at, xk);
    store16<OUT>(vw, at, xv);
}

}  // namespace fold

using namespace fold;

static bool planes_aligned(const void* ka, const void* kb, const void* va, const void* vb) {   // (16 bytes; vb may be null)
    return ((reinterpret_cast<uintptr_t>(ka) | reinterpret_cast<uintptr_t>(kb) | reinterpret_cast<uintptr_t>(va) | reinterpret_cast<uintptr_t>(vb)) & 15) == 0;
}

extern "C" int fold_build_tables(const int32_t* cu_seqlens, const int32_t* seq_lens, int batch, int32_t* page_table, int pages_per_request,
                                 int page_size, int total, const int32_t* free_pages, int n_free, const int32_t* taken, int32_t* slots,
                                 int32_t* lens_out, int32_t* taken_out, void* stream) {
    FOLD_CHECK_ARG(cu_seqlens && seq_lens && page_table && lens_out && (slots || total == 0), "fold_build_tables: null pointer");
    FOLD_CHECK_ARG(batch > 0 && pages_per_request > 0 && page_size > 0 && total >= 0 && n_free >= 0,
                   "fold_build_tables: %d requests, %d pages of %d keys, %d tokens, %d free pages", batch, pages_per_request, page_size, total, n_free);
    FOLD_CHECK_ARG(!free_pages || (taken && taken_out && taken != taken_out), "fold_build_tables: a free list comes with the count taken from it, in and out");
    FOLD_CHECK_ARG(lens_out != seq_lens, "fold_build_tables: lens_out is another tensor than seq_lens");
    build_tables_kernel<<<batch, TB_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(cu_seqlens, seq_lens, batch, page_table, pages_per_request, page_size,
                                                                                     total, free_pages, n_free, taken, slots, lens_out, taken_out);
    return check_launch("fold_build_tables");
}

extern "C" int fold_write_tokens(const void* k, const void* v, int is_f16, int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride,
                                 int64_t v_head_stride, const int32_t* slots, int64_t total, int n_kv_heads, int head_dim, int page_size, int64_t pool_rows,
                                 int8_t* ka, int8_t* kb, void* va, void* vb, void* ek, float v_scale, void* stream) {
    FOLD_CHECK_ARG(head_dim == 64 || head_dim == 128, "head_dim %d: the cache writers take 64 or 128", head_dim);
    FOLD_CHECK_ARG(total >= 0 && n_kv_heads > 0 && page_size > 0, "fold_write_tokens: %lld tokens, %d heads, pages of %d", static_cast<long long>(total), n_kv_heads, page_size);
    if (total == 0) return FOLD_OK;
    FOLD_CHECK_ARG(k && v && slots && ka && kb && va && ek, "fold_write_tokens: null pointer");
    FOLD_CHECK_ARG(k_token_stride % 8 == 0 && k_head_stride % 8 == 0 && v_token_stride % 8 == 0 && v_head_stride % 8 == 0 &&
                       reinterpret_cast<uintptr_t>(k) % 16 == 0 && reinterpret_cast<uintptr_t>(v) % 16 == 0 && planes_aligned(ka, kb, va, vb),
                   "fold_write_tokens: rows must be 16-byte aligned");
    const int rpb = NT / (head_dim / 16);
    const int64_t rows = total * n_kv_heads, grid = (rows + rpb - 1) / rpb;
    FOLD_CHECK_ARG(grid < (1ll << 31), "fold_write_tokens: %lld rows in one call", static_cast<long long>(rows));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const uint16_t *kp = static_cast<const uint16_t*>(k), *vp = static_cast<const uint16_t*>(v);
    const float ievs = 1.0f / v_scale;
#define FOLD_WT(DD, VV, FF)                                                                                                       \
    write_tokens_kernel<DD, VV, FF><<<static_cast<unsigned>(grid), NT, 0, st>>>(kp, vp, k_token_stride, k_head_stride, v_token_stride, \
        v_head_stride, slots, rows, n_kv_heads, page_size, pool_rows, ka, kb, va, vb, static_cast<__nv_bfloat16*>(ek), ievs)
    if (head_dim == 64) {
        if (vb) { if (is_f16) FOLD_WT(64, true, true); else FOLD_WT(64, true, false); }
        else    { if (is_f16) FOLD_WT(64, false, true); else FOLD_WT(64, false, false); }
    } else {
        if (vb) { if (is_f16) FOLD_WT(128, true, true); else FOLD_WT(128, true, false); }
        else    { if (is_f16) FOLD_WT(128, false, true); else FOLD_WT(128, false, false); }
    }
#undef FOLD_WT
    return check_launch("fold_write_tokens");
}

extern "C" int fold_read_tokens(const int32_t* slots, int64_t total, int n_kv_heads, int head_dim, int page_size, int64_t pool_rows, const int8_t* ka, const int8_t* kb,
                                const void* va, const void* vb, const void* ek, float v_scale, void* k, void* v, int out_dtype, void* stream) {
    FOLD_CHECK_ARG(head_dim == 64 || head_dim == 128, "head_dim %d: the cache holds 64 or 128", head_dim);
    FOLD_CHECK_ARG(total >= 0 && n_kv_heads > 0 && page_size > 0, "fold_read_tokens: %lld tokens, %d heads, pages of %d", static_cast<long long>(total), n_kv_heads, page_size);
    FOLD_CHECK_ARG(out_dtype >= 0 && out_dtype <= 2, "fold_read_tokens: output type %d", out_dtype);
    if (total == 0) return FOLD_OK;
    FOLD_CHECK_ARG(slots && ka && kb && va && ek && k && v, "fold_read_tokens: null pointer");
    FOLD_CHECK_ARG(reinterpret_cast<uintptr_t>(k) % 16 == 0 && reinterpret_cast<uintptr_t>(v) % 16 == 0 && planes_aligned(ka, kb, va, vb), "fold_read_tokens: rows must be 16-byte aligned");
    const int rpb = NT / (head_dim / 16);
    const int64_t rows = total * n_kv_heads, grid = (rows + rpb - 1) / rpb;
    FOLD_CHECK_ARG(grid < (1ll << 31), "fold_read_tokens: %lld rows in one call", static_cast<long long>(rows));
    const Planes p = {ka, kb, static_cast<const uint16_t*>(ek), static_cast<const uint8_t*>(va), static_cast<const uint8_t*>(vb), v_scale};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
#define FOLD_RT(DD, VV, OO) read_tokens_kernel<DD, VV, OO><<<static_cast<unsigned>(grid), NT, 0, st>>>(slots, rows, n_kv_heads, page_size, pool_rows, p, k, v)
#define FOLD_RT3(DD, VV)                                    \
    do {                                                    \
        if (out_dtype == OUT_F32) FOLD_RT(DD, VV, OUT_F32); \
        else if (out_dtype == OUT_BF16) FOLD_RT(DD, VV, OUT_BF16); \
        else FOLD_RT(DD, VV, OUT_F16);                      \
    } while (0)
    if (head_dim == 64) { if (vb) FOLD_RT3(64, true); else FOLD_RT3(64, false); }
    else                { if (vb) FOLD_RT3(128, true); else FOLD_RT3(128, false); }
#undef FOLD_RT3
#undef FOLD_RT
    return check_launch("fold_read_tokens");
}

extern "C" int fold_chunk_sums(const void* v, int is_f16, int64_t v_token_stride, int64_t v_head_stride, int batch, int n_kv_heads, int head_dim,
                               const int32_t* cu_seqlens, int total, const int32_t* lens_new, int32_t* lens, float v_scale, float* vsum, float* vmean,
                               void* stream) {
    return fold_chunk_sums_placed(v, is_f16, v_token_stride, v_head_stride, batch, n_kv_heads, head_dim, cu_seqlens, total, nullptr, 0, lens_new, lens,
                                  v_scale, vsum, vmean, stream);
}

extern "C" int fold_chunk_sums_placed(const void* v, int is_f16, int64_t v_token_stride, int64_t v_head_stride, int batch, int n_kv_heads, int head_dim,
                                      const int32_t* cu_seqlens, int total, const int32_t* slots, int64_t room, const int32_t* lens_new, int32_t* lens,
                                      float v_scale, float* vsum, float* vmean, void* stream) {
    FOLD_CHECK_ARG(head_dim == 64 || head_dim == 128, "head_dim %d: the cache writers take 64 or 128", head_dim);
    FOLD_CHECK_ARG(cu_seqlens && lens_new && lens && vsum && vmean && (v || total == 0), "fold_chunk_sums: null pointer");
    FOLD_CHECK_ARG(batch > 0 && batch <= 65535 && n_kv_heads > 0 && total >= 0, "fold_chunk_sums: %d requests, %d heads", batch, n_kv_heads);
    FOLD_CHECK_ARG(v_token_stride % 4 == 0 && v_head_stride % 4 == 0 && reinterpret_cast<uintptr_t>(v) % 8 == 0, "fold_chunk_sums: rows must be 8-byte aligned");
    const dim3 grid(n_kv_heads, batch);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const uint16_t* vp = static_cast<const uint16_t*>(v);
#define FOLD_CS(DD, FF) \
    chunk_sums_kernel<DD, FF><<<grid, 16 * DD / 4, 0, st>>>(vp, v_token_stride, v_head_stride, n_kv_heads, cu_seqlens, total, slots, room, lens_new, lens, v_scale, vsum, vmean)
    if (head_dim == 64) { if (is_f16) FOLD_CS(64, true); else FOLD_CS(64, false); }
    else                { if (is_f16) FOLD_CS(128, true); else FOLD_CS(128, false); }
#undef FOLD_CS
    return check_launch("fold_chunk_sums");
}

extern "C" int fold_chunk_gather(const int32_t* cu_seqlens, const int32_t* seq_lens, int batch, const int32_t* page_table, int pages_per_request,
                                 int page_size, int n_kv_heads, int head_dim, int window, int sinks, const int8_t* ka, const int8_t* kb, const void* va,
                                 const void* vb, const void* ek, float v_scale, int is_f16, int rows_over, int group, int cap_tiles, int32_t* plan, int32_t* tiles, void* kw,
                                 void* vw, int32_t* status, void* stream) {
    FOLD_CHECK_ARG(head_dim == 64 || head_dim == 128, "head_dim %d: the cache holds 64 or 128", head_dim);
    FOLD_CHECK_ARG(cu_seqlens && seq_lens && page_table && ka && kb && va && ek && plan && tiles && kw && vw && status, "fold_chunk_gather: null pointer");
    FOLD_CHECK_ARG(batch > 0 && n_kv_heads > 0 && n_kv_heads <= 65535 && pages_per_request > 0 && page_size > 0 && cap_tiles > 0 && cap_tiles <= (1 << 24) &&
                       rows_over >= 0 && group > 0,
                   "fold_chunk_gather: %d requests, %d heads, %d pages of %d keys, %d tiles", batch, n_kv_heads, pages_per_request, page_size, cap_tiles);
    FOLD_CHECK_ARG(planes_aligned(ka, kb, va, vb) && planes_aligned(kw, vw, plan, nullptr) && reinterpret_cast<uintptr_t>(tiles) % 8 == 0, "fold_chunk_gather: rows must be 16-byte aligned");
    FOLD_CHECK_ARG(window > 0 && window <= FOLD_MAX_WINDOW && sinks >= 0 && sinks <= FOLD_MAX_WINDOW, "fold_chunk_gather: a window of %d keys and %d sinks", window, sinks);
    const int64_t cap = static_cast<int64_t>(pages_per_request) * page_size;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    chunk_plan_kernel<<<1, CP_THREADS, 0, st>>>(cu_seqlens, seq_lens, batch, static_cast<int>(cap < (1 << 30) ? cap : (1 << 30)), window, sinks, rows_over, group, cap_tiles,
                                                reinterpret_cast<int4*>(plan), reinterpret_cast<int2*>(tiles), status);
    const Planes p = {ka, kb, static_cast<const uint16_t*>(ek), static_cast<const uint8_t*>(va), static_cast<const uint8_t*>(vb), v_scale};
    const int rpb = NT / (head_dim / 16);
    const dim3 grid(static_cast<unsigned>(cap_tiles) * (128 / rpb), n_kv_heads);
    const int64_t rows = static_cast<int64_t>(cap_tiles) * 128;
#define FOLD_CG(DD, VV, OO)                                                                                                                  \
    chunk_gather_kernel<DD, VV, OO><<<grid, NT, 0, st>>>(reinterpret_cast<const int4*>(plan), reinterpret_cast<const int2*>(tiles), page_table, \
        pages_per_request, page_size, n_kv_heads, sinks, p, rows, static_cast<uint16_t*>(kw), static_cast<uint16_t*>(vw))
    if (head_dim == 64) {
        if (vb) { if (is_f16) FOLD_CG(64, true, OUT_F16); else FOLD_CG(64, true, OUT_BF16); }
        else    { if (is_f16) FOLD_CG(64, false, OUT_F16); else FOLD_CG(64, false, OUT_BF16); }
    } else {
        if (vb) { if (is_f16) FOLD_CG(128, true, OUT_F16); else FOLD_CG(128, true, OUT_BF16); }
        else    { if (is_f16) FOLD_CG(128, false, OUT_F16); else FOLD_CG(128, false, OUT_BF16); }
    }
#undef FOLD_CG
    return check_launch("fold_chunk_gather");
}
