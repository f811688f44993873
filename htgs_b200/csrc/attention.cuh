// Shared by the kernels of attention over packed sequences (attention.cu, attention_tiles.cu): which rows a block works on, and what a row sees.
//
//   S = scale q k^T over the rows that a row sees,  P = softmax(S),  out = P v            (a key head serves heads / key_heads query heads)
//   dP = dout v^T,  D = sum(dout * out) of a row,  dS = P * (dP - D),  dq = scale dS k,  dk = scale dS^T q,  dv = P^T dout
//
// Exponentials are powers of two: S carries scale * log2(e), and a row's statistic is log2 of the sum of 2^S.
#pragma once

#include "tensor_core.cuh"

namespace htgs {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kStatisticRows = 128, kStatisticBytes = kStatisticRows * 2 * 4;

// Sequences and what stands before and behind them (rows of no sequence, with offsets only) share tiles with nobody: sequence v begins at tile bound(v) / ROWS + v.  That leaves
// room for the tiles of all before it, needs no sum over the sequences, and is found by a search over the offsets alone.
struct SequenceTile {
    int sequence;            // counted with the rows before the first one
    int begin, end;          // its rows
    int first;               // of the tile; not below `end` where the tile holds nothing
    bool outside;            // rows of no sequence
};
__host__ __device__ __forceinline__ int64_t sequence_tiles(const HtgsAttention& a, int rows_of_tile) {
    if (a.offsets) return a.rows / rows_of_tile + a.n_sequences + 2;
    const int64_t each = a.rows / a.n_sequences;
    return (each + rows_of_tile - 1) / rows_of_tile * a.n_sequences;
}
// By a whole warp.
template <int ROWS> __device__ __forceinline__ SequenceTile find_tile(const HtgsAttention& a, int tile) {
    if (!a.offsets) {
        const int each = int(a.rows / a.n_sequences), tiles = (each + ROWS - 1) / ROWS, s = tile / tiles;
        return {s, s * each, (s + 1) * each, s * each + (tile - s * tiles) * ROWS, false};
    }
    const int rows = int(a.rows), n = a.n_sequences, lane = int(threadIdx.x & 31);
    const auto bound = [&](int v) { return v <= 0 ? 0 : v > n + 1 ? rows : min(max(__ldg(a.offsets + v - 1), 0), rows); };      // no offset reaches behind the rows
    int low = 0, high = n + 2;
    while (high - low > 1) {
        const int step = (high - low + 31) / 32, probe = low + lane * step;
        const uint32_t before = __ballot_sync(0xffffffffu, probe < high && bound(probe) / ROWS + probe <= tile);
        const int last = before ? 31 - __clz(before) : 0;
        low += last * step;
        high = min(high, low + step);
    }
    const int begin = bound(low), end = bound(low + 1);
    return {low, begin, end, begin + (tile - begin / ROWS - low) * ROWS, low == 0 || low == n + 1};
}

// Statistics of rows for the backward pass, log2 of the sum and D, in order of tiles of 128 rows: 128 of the one, 128 of the other, so that a tile's lie side by side on 16 bytes.  Where those of a
// sequence begin, in rows.
__host__ __device__ __forceinline__ int64_t statistic_rows(const HtgsAttention& a) { return sequence_tiles(a, kStatisticRows) * kStatisticRows; }
__device__ __forceinline__ int64_t statistic_base(const HtgsAttention& a, const SequenceTile& t) {
    if (a.offsets) return (int64_t(t.begin / kStatisticRows) + t.sequence) * kStatisticRows;
    const int64_t each = a.rows / a.n_sequences;
    return t.sequence * ((each + kStatisticRows - 1) / kStatisticRows) * kStatisticRows;
}

// The rows that row i of a sequence sees, and those that see it: [first, last].
__device__ __forceinline__ int first_seen(const HtgsAttention& a, int begin, int i) { return a.window < 0 || i - begin <= a.window ? begin : i - a.window; }
__device__ __forceinline__ int last_seen(const HtgsAttention& a, int end, int i) { return a.causal ? i : a.window < 0 || end - 1 - i <= a.window ? end - 1 : i + a.window; }
__device__ __forceinline__ int first_seeing(const HtgsAttention& a, int begin, int j) { return a.causal ? j : first_seen(a, begin, j); }
__device__ __forceinline__ int last_seeing(const HtgsAttention& a, int end, int j) { return a.window < 0 || end - 1 - j <= a.window ? end - 1 : j + a.window; }

// The least b with n <= 2^b, of a positive n.
__device__ __forceinline__ int bits_of(int n) { return 32 - __clz(n - 1); }

__device__ __forceinline__ float exp2_approx(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float infinity() { return __uint_as_float(0x7f800000u); }

struct AttentionBackward {
    const void* grad; int64_t grad_stride, grad_head_stride;
    void* grad_q; void* grad_k; void* grad_v;
    const float* statistics; int64_t statistics_rows;        // of a head
    const uint32_t* largest;                                 // of each sequence (counted as in SequenceTile): the largest finite |dout|^2 and |v|^2 of a row and head, as bits; fp16 only
};

// attention_tiles.cu: 16-bit types, widths that are a multiple of 8, everything on 16 bytes
bool attention_tiles_take(const HtgsAttention& a, const void* out, const void* rest);
int attention_tiles_forward(const HtgsAttention& a, void* out, void* rest, float* sums, cudaStream_t stream);
bool attention_tiles_take(const HtgsAttention& a, const AttentionBackward& b);
int attention_tiles_backward(const HtgsAttention& a, const AttentionBackward& b, cudaStream_t stream);
unsigned int* attention_error_word(int device);

}  // namespace htgs
