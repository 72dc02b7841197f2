// Shared definitions of the deterministic attention backward.
//
// One call handles B sequences ("requests"), dense (B, S, H, D) or packed
// (total, H, D) with cu_seqlens. Per-row workspaces are laid out [head][padded
// row]: a sequence's rows start on a 128-row boundary so every query tile
// belongs to one sequence.
#pragma once
#include "common.cuh"

namespace fold {

constexpr int ROW_PAD = 128;  // sequences start on this boundary in the workspaces

struct TensorView {
    void* ptr;
    int64_t sb, sr, sh;  // element strides: batch, row (token), head; channels are contiguous
};

struct BwdParams {
    TensorView q, k, v, o, dout, dq, dk, dv;
    const void* o_rest;    // what rounding took from o, laid out as o, or null: Delta then is dO's product with both
    const float* lse;      // natural log; dense (B, H, S), packed (H, total)
    int64_t lse_sb, lse_sh;
    const int* cu;         // (B + 1) int32 on the device, or null for dense
    int B, H, HKV, G, S, total, D;
    int causal, f16;
    float scale;
    // workspace
    int* dq_acc;    // int32 [H][rows_p][D], the fixed-point dQ / scale * 2^s
    float* dpsum;   // [H][rows_p]  Delta_i = sum_d dO O
    float* lse2;    // [H][rows_p]  s - lse * log2(e) (fp16: -lse * log2(e)); -inf on padded rows
    int* stats;     // [B][HKV][N_STATS] float bits of the order-free maxima
    int* status;    // one word after the stats: raised if a device-side wait ran out
    int64_t rows_p; // padded rows per head
    int dq_bias;    // the main loop adds 0x4B400000 with every partial: the accumulator starts at minus their sum
    // how the tcgen05 main loop's work is cut (the other main loop takes whole groups and ranges)
    int subgroup;   // query heads per work item; it divides G
    int record;     // query blocks per work item, 0: every block that sees the key block
    int fold;       // a key block's dK, dV are summed across work items, on integer grids
    int dv_bits;    // dV's accumulator when folding: 32 (30-bit grid) or 64 (61-bit grid)
    long long* dk_acc;   // int64 [HKV][rows_p][D], zero before the main loop (fold)
    void* dv_acc;        // int32 or int64 [HKV][rows_p][D] (fold)
    int* work;      // the work list: n_items x 8 ints, written in-stream ahead of the main loop
    int n_items;
    int* sched;     // [2]: the list's claim counter and the count of finished CTAs, zero between launches
    int S_r;        // dense: S rounded up to ROW_PAD
    // A causal call under a sliding window (window > 0): query i sees key j <= i when i - j < window or
    // j < sinks. Key blocks past the sinks meet the few query blocks their window reaches and stay
    // private to a CTA; a block that holds sinks meets every later query block, so its items are cut
    // into records of `sink_record` query blocks and its dK, dV meet in the integer accumulators
    // (dk_acc, dv_acc), which then hold [HKV][B][sink_stride][D] for the sinks' blocks alone.
    int window, sinks, sink_record;
    // Packed sequences under a window, on the tcgen05 main loop: each one's last block of 128 rows of Q, dO
    // [B][H][128][D] and K, V [B][HKV][128][D], zeros past its end, or null. A tile that TMA takes from the
    // tensor there holds the next sequence's first rows, or what lies behind the last one's, and a NaN among them would
    // pass through the products' zeros.
    uint16_t* last;
    int sink_rows;      // rows of a sequence whose dK, dV the accumulators hold: the sinks' whole key blocks
    int sink_stride;    // and how many are laid out
};

// Whether each query of a sequence sees one key: P = 1 whatever its score, so dS = 0. dP - Delta would
// leave the rounding of two sums there, and gradients that are zero throughout would come back as noise.
__device__ __forceinline__ bool lone_keys(const BwdParams& p, int len) { return len == 1 || (p.window == 1 && p.sinks == 0); }

// The longest a window's key block is walked before an item is cut, in the main loop's query blocks:
// about what a block past the sinks walks, so the launch's longest items stay its ordinary ones. It
// depends on the window alone: a sequence's bits do not depend on its neighbours.
// (Never under 3: an item's exit adds its block to the accumulators. At 3 x 1037 tokens, 6 heads, window 77
// the launch takes 42 us with records of 3, 53 of 4 and 97 of 8.)
inline int sink_record_blocks(int window, int tile) {
    const int r = window / tile + 2;
    return r < 3 ? 3 : r > (1 << 20) ? (1 << 20) : r;
}
// one past the last query block of `tile` rows that sees any key of [n0, n0 + tile) by the window
__host__ __device__ inline int window_end(int n0, int tile, int window) { return (n0 + tile - 1 + window - 1) / tile + 1; }


struct SeqInfo {
    int start;       // first row in the packed tensors (0 for dense)
    int len;
    int64_t pstart;  // first row in the padded workspaces
};

__device__ __forceinline__ SeqInfo seq_info(const BwdParams& p, int b) {
    SeqInfo s;
    if (p.cu) {
        s.start = p.cu[b];
        s.len = p.cu[b + 1] - s.start;
        s.pstart = (static_cast<int64_t>(s.start) + static_cast<int64_t>(b) * ROW_PAD) / ROW_PAD * ROW_PAD;
    } else {
        s.start = 0;
        s.len = p.S;
        s.pstart = static_cast<int64_t>(b) * p.S_r;
    }
    return s;
}

// first row of a (request, KV head) in dk_acc, dv_acc
__device__ __forceinline__ int64_t dkv_acc_row(const BwdParams& p, const SeqInfo& sq, int b, int hkv) {
    return p.window > 0 ? (static_cast<int64_t>(hkv) * p.B + b) * p.sink_stride : static_cast<int64_t>(hkv) * p.rows_p + sq.pstart;
}

template <typename T>
__device__ __forceinline__ T* row_ptr(const TensorView& t, int b, int64_t row, int h) {
    return static_cast<T*>(t.ptr) + b * t.sb + row * t.sr + h * t.sh;
}

inline int64_t padded_rows(int B, int S, int total, bool varlen) {
    if (!varlen) return static_cast<int64_t>(B) * ((S + ROW_PAD - 1) / ROW_PAD * ROW_PAD);
    int64_t r = static_cast<int64_t>(total) + static_cast<int64_t>(B + 1) * ROW_PAD - 1;
    return (r + ROW_PAD - 1) / ROW_PAD * ROW_PAD;
}

// kernels
int launch_bwd_preprocess(const BwdParams& p, cudaStream_t st);
int launch_bwd_postprocess(const BwdParams& p, int layout, cudaStream_t st);
// how many work items the tcgen05 main loop's list holds for a call (0 for the other main loop)
int64_t bwd_sm100_work_items(int B, int H, int HKV, int S, int subgroup, int record, int window, int sinks);
int launch_bwd_main_mma(const BwdParams& p, cudaStream_t st);
int launch_bwd_main_sm100(const BwdParams& p, bool build_list, bool run_main, cudaStream_t st);
bool bwd_sm100_supported(const BwdParams& p);
bool bwd_sm100_biased();   // whether the tcgen05 main loop leaves its rounding constant in the partials

// dq accumulator tile layouts
enum { DQ_LAYOUT_ROW_MAJOR = 0, DQ_LAYOUT_SM100 = 1 };

}  // namespace fold
