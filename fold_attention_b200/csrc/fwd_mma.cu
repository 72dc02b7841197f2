// Attention forward producing O and the log-sum-exp the backward consumes.
// The reference takes both from a third-party forward
// (src/fold_attention/interface.py:42-44,70-81); this is a self-contained
// online-softmax kernel on mma.sync so the package has no such dependency.
// One CTA: 64 query rows of one head; four warps of 16 rows each.
#include "bwd_common.cuh"
#include "mma_utils.cuh"

namespace fold {

struct FwdParams {
    TensorView q, k, v, o;
    float* lse;
    int64_t lse_sb, lse_sh;
    const int* cu;
    int B, H, HKV, G, S, D, causal, f16;
    float scale;
    // a build with EXT = true only (it is causal): a row sees the `window` newest keys up to its own
    // position and the first `sinks` keys; with `plan` the queries are request b's last positions and its
    // keys plan[b].x rows of (row, head) tensors from row plan[b].y on, without the plan[b].z tiles of 128
    // keys between the sinks' tiles and the window's that no query of the chunk sees
    int window, sinks;
    const int4* plan;
    int total;       // packed rows
    void* o_rest;    // what rounding took from o, laid out as o, or null (a window's)
};

// KIND: the causal and full forward, a window, or a chunk. A chunk's blocks are few and their keys many, and
// with four warps a block each scheduler has one, whose matrix instructions wait for one another: there two
// groups of four warps take the key tiles in turn, and their sums meet at the end (9 requests of up to 300 new
// tokens behind 1500, 6 heads: 46 -> 36 us).
enum { KIND_PLAIN, KIND_WINDOW, KIND_CHUNK };

template <int D, bool F16, bool CAUSAL, int KIND>
__global__ void __launch_bounds__(KIND == KIND_CHUNK ? 256 : 128) fwd_mma_kernel(const FwdParams p) {
    constexpr int PITCH = D * 2 + 16, TILE = 64 * PITCH, NTO = D / 8;
    constexpr bool EXT = KIND != KIND_PLAIN;
    constexpr int GROUPS = KIND == KIND_CHUNK ? 2 : 1;
    // a chunk's fp16 weights (1 at most, of rows that may see millions of keys) and their sums carry 2^14, which
    // O / l cancels: fp16's least step is then 2^-38 of a row's largest weight
    constexpr float LIFT = KIND == KIND_CHUNK && F16 ? 14.f : 0.f;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* sQ = smem;
    const int grp = GROUPS == 2 ? threadIdx.x >> 7 : 0;
    uint8_t* sK = smem + (1 + 2 * grp) * TILE;
    uint8_t* sV = sK + TILE;
    const int mb = gridDim.x - 1 - blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    int start = 0, len = p.S;
    if (p.cu) {
        start = p.cu[b];
        len = p.cu[b + 1] - start;
    }
    const int m0 = mb * 64;
    if (KIND == KIND_WINDOW && p.cu && b == p.B - 1 && mb == 0)   // rows behind the last packed sequence: zeros
        for (int64_t i = max(start + len, 0) + static_cast<int64_t>(threadIdx.x >> 5); i < p.total; i += 4) {
            for (int c = threadIdx.x & 31; c < D / 2; c += 32) reinterpret_cast<uint32_t*>(row_ptr<uint16_t>(p.o, 0, i, h))[c] = 0u;
            if ((threadIdx.x & 31) == 0 && p.lse) p.lse[h * p.lse_sh + i] = -INFINITY;
        }
    if (m0 >= len) return;
    const int tid = threadIdx.x & 127, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, tq = lane & 3;
    const int hkv = h / p.G;
    const float c2 = p.scale * kLog2e;
    int klen = len, qoff = 0, kstart = start, kshift = 0;   // keys, and the first query's position among them
    if constexpr (KIND == KIND_CHUNK) {
        const int4 pl = p.plan[b];
        if (pl.x < 0 || start < 0 || len > p.total - start) return;   // another kernel's, or counts that q has no rows for
        klen = pl.x;
        qoff = klen - len;
        kstart = pl.y;
        kshift = 128 * pl.z;
    }

    load_tile_async<D, PITCH, 128 * GROUPS>(sQ, row_ptr<const uint16_t>(p.q, b, start + m0, h), p.q.sr, 64, min(64, len - m0), threadIdx.x);
    cp_async_commit();

    float o[NTO][4];
#pragma unroll
    for (int i = 0; i < NTO; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    float mx[2] = {-INFINITY, -INFINITY}, ls[2] = {0.f, 0.f};

    const int n_end = EXT ? max(0, min(klen, qoff + min(len, m0 + 64))) : CAUSAL ? min(len, m0 + 64) : len;
    // EXT: the first key tile of the block's window; between the sinks' tiles and it nothing is seen
    const int n_low = EXT ? max(0, qoff + m0 - p.window + 1) / 64 * 64 : 0;
    auto seen_from = [&](int n0) { return EXT && n0 >= p.sinks && n0 < n_low ? n_low : n0; };
    int next = seen_from(0);
    while (next < n_end) {
        int n0 = next;
        next = seen_from(n0 + 64);
        if (GROUPS == 2) {
            if (grp) n0 = next;
            next = seen_from(next + 64);
        }
        __syncthreads();  // previous tile's reads are done
        const int kvalid = min(64, klen - n0);
        const int krow = kstart + (EXT && n0 >= (p.sinks + 127) / 128 * 128 ? n0 - kshift : n0);   // whole tiles of 128 keys are left out
        if (GROUPS == 1 || n0 < n_end) {
            load_tile_async<D, PITCH, 128>(sK, row_ptr<const uint16_t>(p.k, b, krow, hkv), p.k.sr, 64, kvalid, tid);
            load_tile_async<D, PITCH, 128>(sV, row_ptr<const uint16_t>(p.v, b, krow, hkv), p.v.sr, 64, kvalid, tid);
        }
        cp_async_commit();
        cp_async_wait<0>();
        __syncthreads();
        if (GROUPS == 2 && n0 >= n_end) break;   // the second group's: the last tile is the first's

        float s[8][4];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[i][e] = 0.f;
        const int arow = 16 * warp + (lane & 7) + 8 * ((lane >> 3) & 1);
        const int brow = (lane & 7) + 8 * (lane >> 4);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            uint32_t a[4];
            ldmatrix_x4(a, smem_u32(sQ + arow * PITCH + (2 * ks + (lane >> 4)) * 16));
#pragma unroll
            for (int np = 0; np < 4; ++np) {
                uint32_t bk[4];
                ldmatrix_x4(bk, smem_u32(sK + (brow + 16 * np) * PITCH + (2 * ks + ((lane >> 3) & 1)) * 16));
                mma_16816<F16>(s[2 * np], a, bk[0], bk[1]);
                mma_16816<F16>(s[2 * np + 1], a, bk[2], bk[3]);
            }
        }
        const bool need_mask = (CAUSAL && n0 + 64 > qoff + m0) || (n0 + 64 > klen) ||
                               (EXT && n0 <= qoff + m0 + 63 - p.window && n0 + 64 > p.sinks);
        float rmax[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x = s[nt][e] * c2;
                if (need_mask) {
                    const int kj = n0 + 8 * nt + 2 * tq + (e & 1);
                    const int qi = qoff + m0 + 16 * warp + gid + 8 * (e >> 1);
                    if (kj >= klen || (CAUSAL && kj > qi)) x = -INFINITY;
                    if (EXT && qi - kj >= p.window && kj >= p.sinks) x = -INFINITY;
                }
                s[nt][e] = x;
                rmax[e >> 1] = fmaxf(rmax[e >> 1], x);
            }
        float corr[2], mnew[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            rmax[r] = fmaxf(rmax[r], __shfl_xor_sync(0xffffffffu, rmax[r], 1));
            rmax[r] = fmaxf(rmax[r], __shfl_xor_sync(0xffffffffu, rmax[r], 2));
            mnew[r] = fmaxf(mx[r], rmax[r]);
            const float ms = mnew[r] == -INFINITY ? 0.f : mnew[r];
            corr[r] = ex2_approx(mx[r] - ms);
            mx[r] = mnew[r];
            mnew[r] = LIFT > 0.f ? ms - LIFT : ms;
        }
        float rsum[2] = {0.f, 0.f};
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float pv = ex2_approx(s[nt][e] - mnew[e >> 1]);
                s[nt][e] = pv;
                rsum[e >> 1] += pv;
            }
#pragma unroll
        for (int r = 0; r < 2; ++r) ls[r] = ls[r] * corr[r] + rsum[r];
#pragma unroll
        for (int i = 0; i < NTO; ++i) {
            o[i][0] *= corr[0];
            o[i][1] *= corr[0];
            o[i][2] *= corr[1];
            o[i][3] *= corr[1];
        }
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            uint32_t a[4];
            a[0] = pack16x2<F16>(s[2 * kk][0], s[2 * kk][1]);
            a[1] = pack16x2<F16>(s[2 * kk][2], s[2 * kk][3]);
            a[2] = pack16x2<F16>(s[2 * kk + 1][0], s[2 * kk + 1][1]);
            a[3] = pack16x2<F16>(s[2 * kk + 1][2], s[2 * kk + 1][3]);
            const int vrow = 16 * kk + (lane & 7) + 8 * ((lane >> 3) & 1);
#pragma unroll
            for (int np = 0; np < NTO / 2; ++np) {
                uint32_t bv[4];
                ldmatrix_x4_trans(bv, smem_u32(sV + vrow * PITCH + (2 * np + (lane >> 4)) * 16));
                mma_16816<F16>(o[2 * np], a, bv[0], bv[1]);
                mma_16816<F16>(o[2 * np + 1], a, bv[2], bv[3]);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        ls[r] += __shfl_xor_sync(0xffffffffu, ls[r], 1);
        ls[r] += __shfl_xor_sync(0xffffffffu, ls[r], 2);
    }
    if constexpr (GROUPS == 2) {
        float* part = reinterpret_cast<float*>(smem + TILE) + tid;   // over the key tiles: [4 NTO + 4][128]
        __syncthreads();
        if (grp) {
#pragma unroll
            for (int i = 0; i < NTO; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) part[(4 * i + e) * 128] = o[i][e];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                part[(4 * NTO + r) * 128] = mx[r];
                part[(4 * NTO + 2 + r) * 128] = ls[r];
            }
        }
        __syncthreads();
        if (grp) return;
        float f[2], g[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const float m2 = part[(4 * NTO + r) * 128], l2 = part[(4 * NTO + 2 + r) * 128], mm = fmaxf(mx[r], m2);
            const float ms = mm == -INFINITY ? 0.f : mm;
            f[r] = ex2_approx(mx[r] - ms);
            g[r] = ex2_approx(m2 - ms);
            ls[r] = ls[r] * f[r] + l2 * g[r];
            mx[r] = mm;
        }
#pragma unroll
        for (int i = 0; i < NTO; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][e] = o[i][e] * f[e >> 1] + part[(4 * i + e) * 128] * g[e >> 1];
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int qi = m0 + 16 * warp + gid + 8 * r;
        if (qi >= len) continue;
        const float inv = ls[r] > 0.f ? 1.f / ls[r] : 0.f;
        uint16_t* orow = row_ptr<uint16_t>(p.o, b, start + qi, h);
#pragma unroll
        for (int i = 0; i < NTO; ++i)
            *reinterpret_cast<uint32_t*>(orow + 8 * i + 2 * tq) = pack16x2<F16>(o[i][2 * r] * inv, o[i][2 * r + 1] * inv);
        if (KIND == KIND_WINDOW && p.o_rest) {
            uint16_t* rest = static_cast<uint16_t*>(p.o_rest) + (orow - static_cast<uint16_t*>(p.o.ptr));
#pragma unroll
            for (int i = 0; i < NTO; ++i) {
                const float x = o[i][2 * r] * inv, y = o[i][2 * r + 1] * inv;
                const uint32_t w = pack16x2<F16>(x, y);
                *reinterpret_cast<uint32_t*>(rest + 8 * i + 2 * tq) =
                    pack16x2<F16>(x - half_bits_to_float<F16>(static_cast<uint16_t>(w & 0xFFFFu)), y - half_bits_to_float<F16>(static_cast<uint16_t>(w >> 16)));
            }
        }
        if (tq == 0 && (!EXT || p.lse))
            p.lse[b * p.lse_sb + h * p.lse_sh + start + qi] =
                ls[r] > 0.f ? ((LIFT > 0.f ? mx[r] - LIFT : mx[r]) + log2f(ls[r])) * 0.6931471805599453f : -INFINITY;
    }
}

template <int D, bool F16, bool CAUSAL, int KIND>
static int fwd_launch_one(const FwdParams& p, cudaStream_t st) {
    constexpr int GROUPS = KIND == KIND_CHUNK ? 2 : 1;
    constexpr int BYTES = (1 + 2 * GROUPS) * 64 * (D * 2 + 16);
    auto kern = fwd_mma_kernel<D, F16, CAUSAL, KIND>;
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, BYTES);
    dim3 grid((p.S + 63) / 64, p.H, p.B);
    kern<<<grid, 128 * GROUPS, BYTES, st>>>(p);
    return check_launch("fwd_mma");
}

template <int D>
static int fwd_launch_d(const FwdParams& p, cudaStream_t st) {
    if (p.plan) {
        if constexpr (D == 64) return p.f16 ? fwd_launch_one<D, true, true, KIND_CHUNK>(p, st) : fwd_launch_one<D, false, true, KIND_CHUNK>(p, st);
        set_error("head_dim %d: a plan comes with 64", D);
        return FOLD_ERR_UNSUPPORTED;
    }
    if (p.window > 0) return p.f16 ? fwd_launch_one<D, true, true, KIND_WINDOW>(p, st) : fwd_launch_one<D, false, true, KIND_WINDOW>(p, st);
    if (p.f16) return p.causal ? fwd_launch_one<D, true, true, KIND_PLAIN>(p, st) : fwd_launch_one<D, true, false, KIND_PLAIN>(p, st);
    return p.causal ? fwd_launch_one<D, false, true, KIND_PLAIN>(p, st) : fwd_launch_one<D, false, false, KIND_PLAIN>(p, st);
}

}  // namespace fold

using namespace fold;

// The causal and full forward (window 0, plan null), a window's or a chunk's.
static int fwd_run(const char* what, const void* q, const void* k, const void* v, void* o, float* lse, void* o_rest,
                   const int64_t* strides, const int32_t* cu_seqlens, int batch, int n_heads, int n_kv_heads,
                   int max_seqlen, int total, int head_dim, int causal, int is_f16, float softmax_scale, int window,
                   int sinks, const int32_t* plan, int krows, void* stream) {
    FOLD_CHECK_ARG(q && k && v && o && (lse || plan) && strides, "%s: null pointer", what);
    FOLD_CHECK_ARG(n_kv_heads > 0 && n_heads % n_kv_heads == 0, "the query heads must be a multiple of the KV heads");
    FOLD_CHECK_ARG(batch > 0 && max_seqlen > 0, "%s: empty call", what);
    FOLD_CHECK_ARG(n_heads <= 65535 && batch <= 65535, "%s: %d heads, %d requests (65535 at most)", what, n_heads, batch);
    FwdParams p;
    const void* ptrs[4] = {q, k, v, o};
    TensorView* views[4] = {&p.q, &p.k, &p.v, &p.o};
    for (int i = 0; i < 4; ++i) {
        views[i]->ptr = const_cast<void*>(ptrs[i]);
        views[i]->sb = strides[3 * i];
        views[i]->sr = strides[3 * i + 1];
        views[i]->sh = strides[3 * i + 2];
        FOLD_CHECK_ARG(views[i]->sr % 8 == 0 && views[i]->sh % 8 == 0 && views[i]->sb % 8 == 0 &&
                           reinterpret_cast<uintptr_t>(ptrs[i]) % 16 == 0,
                       "%s: rows must be 16-byte aligned", what);
    }
    p.lse = lse;
    p.cu = cu_seqlens;
    if (cu_seqlens) {
        p.lse_sb = 0;
        p.lse_sh = total;
    } else {
        p.lse_sb = static_cast<int64_t>(n_heads) * max_seqlen;
        p.lse_sh = max_seqlen;
    }
    p.B = batch; p.H = n_heads; p.HKV = n_kv_heads; p.G = n_heads / n_kv_heads;
    p.S = max_seqlen; p.D = head_dim; p.causal = causal; p.f16 = is_f16; p.scale = softmax_scale;
    p.window = window; p.sinks = sinks; p.plan = reinterpret_cast<const int4*>(plan);
    p.total = total; p.o_rest = o_rest;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (head_dim) {
        case 64: return fwd_launch_d<64>(p, st);
        case 96: return fwd_launch_d<96>(p, st);
        case 128: return fwd_launch_d<128>(p, st);
    }
    set_error("head_dim %d: 64, 96 and 128 are supported", head_dim);
    return FOLD_ERR_UNSUPPORTED;
}

extern "C" int fold_fwd_run(const void* q, const void* k, const void* v, void* o, float* lse,
                            const int64_t* strides, const int32_t* cu_seqlens, int batch,
                            int n_heads, int n_kv_heads, int max_seqlen, int total, int head_dim,
                            int causal, int is_f16, float softmax_scale, void* stream) {
    FOLD_CHECK_ARG(lse, "fold_fwd_run: null pointer");
    return fwd_run("fold_fwd_run", q, k, v, o, lse, nullptr, strides, cu_seqlens, batch, n_heads, n_kv_heads, max_seqlen, total,
                   head_dim, causal, is_f16, softmax_scale, 0, 0, nullptr, 0, stream);
}

extern "C" int fold_fwd_window(const void* q, const void* k, const void* v, void* o, float* lse, void* o_rest,
                               const int64_t* strides, const int32_t* cu_seqlens, int batch, int n_heads,
                               int n_kv_heads, int max_seqlen, int total, int head_dim, int is_f16,
                               float softmax_scale, int window, int sinks, const int32_t* plan, int key_rows,
                               void* stream) {
    FOLD_CHECK_ARG(window > 0 && window <= FOLD_MAX_WINDOW && sinks >= 0 && sinks <= FOLD_MAX_WINDOW,
                   "fold_fwd_window: a window of %d keys and %d sinks (1 .. 2^30 and 0 .. 2^30)", window, sinks);
    FOLD_CHECK_ARG(!plan || key_rows > 0, "fold_fwd_window: %d key rows", key_rows);
    FOLD_CHECK_ARG(reinterpret_cast<uintptr_t>(o_rest) % 16 == 0 && !(plan && o_rest), "fold_fwd_window: o_rest is 16-byte aligned, without a plan");
    return fwd_run("fold_fwd_window", q, k, v, o, lse, o_rest, strides, cu_seqlens, batch, n_heads, n_kv_heads, max_seqlen, total,
                   head_dim, 1, is_f16, softmax_scale, window, sinks, plan, key_rows, stream);
}
