// Attention of one more row for each of many sequences over their caches (htgs_attention_step):
//
//   out = sum over cached rows j of softmax_j(scale * q . k_j) v_j,   the new row among them.
//
// A cache is read once: bound by HBM where caches are long (a million rows of 2 key heads of 64: 46 us, 5.6 TB/s; 32 scenes of up to 8192 rows, 2 key heads of 128: 40 us, 4.2 TB/s), by the launch where they are short (7 us).  The rows of a sequence are split over blocks, by its length, which only the device knows;
// each leaves its largest score, its sum and its unnormalised output, and a second kernel joins them, always in the same order.
#include "attention.cuh"

namespace htgs {

namespace {

constexpr int kStepThreads = 256, kStepWarps = kStepThreads / 32, kMostStepWidth = 128, kStepColumns = kMostStepWidth / 32, kStepPiece = 32, kMostSplits = 256;

struct StepRows { int low, length; bool left_out, full; };        // rows [low, length], the last one new

__device__ __forceinline__ StepRows rows_of(const HtgsAttentionStep& a, int b) {
    const int n = __ldg(a.lengths + b);
    return {a.window >= 0 && n > a.window ? n - a.window : 0, n, n < 0, n >= a.capacity};
}
// Rows of a sequence that is not left out, as a power of two that they do not pass: weights carry its inverse (fp16: see kStepLift), so that a row's add up to 1 at most and no sum of values passes the
// largest of them.  (Without it some 300 values of 1e36 became infinite.)
__device__ __forceinline__ int row_bits(const StepRows& r) { return bits_of(r.length + 1 - r.low); }
// Rows [first, last) of a split, in whole pieces but for the last.
__device__ __forceinline__ int2 rows_of_split(const StepRows& r, int split, int splits) {
    const int rows = r.length + 1 - r.low, pieces = (rows + kStepPiece - 1) / kStepPiece;
    return make_int2(r.low + int(int64_t(pieces) * split / splits) * kStepPiece, min(r.length + 1, r.low + int(int64_t(pieces) * (split + 1) / splits) * kStepPiece));
}
// What a split leaves: {largest score, sum} and the output, in 32 bits.
__host__ __device__ __forceinline__ int part_floats(int width) { return 4 + (width + 3) / 4 * 4; }

template <typename T> __device__ __forceinline__ void append(const HtgsAttentionStep& a, int b, int key_head, int length) {
    T* keys = static_cast<T*>(a.keys) + b * a.keys_stride + length * a.keys_row_stride + key_head * a.keys_head_stride;
    T* values = static_cast<T*>(a.values) + b * a.values_stride + length * a.values_row_stride + key_head * a.values_head_stride;
    for (int c = threadIdx.x; c < a.width; c += blockDim.x) {
        keys[c] = static_cast<const T*>(a.k)[b * a.k_stride + key_head * a.k_head_stride + c];
        values[c] = static_cast<const T*>(a.v)[b * a.v_stride + key_head * a.v_head_stride + c];
    }
}

// One head and split to a block, a row at a time to a warp, columns to its lanes.  Bound by a warp's sum for each row (a million rows, 8 heads of 64: 1.07 ms).
template <typename T> __global__ void __launch_bounds__(kStepThreads) step_lanes_kernel(const HtgsAttentionStep a, T* out, float* parts, int splits) {
    __shared__ float2 warps[kStepWarps];
    __shared__ float outputs[kStepWarps][kMostStepWidth];
    grid_dependency();
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, split = int(blockIdx.x % splits), head = int(blockIdx.x / splits % a.heads), b = int(blockIdx.x / splits / a.heads);
    const int group = a.heads / a.key_heads, key_head = head / group;
    const StepRows r = rows_of(a, b);
    float m = -infinity(), l = 0.0f, o[kStepColumns] = {};
    const bool any = !r.left_out && !r.full;
    if (any) {
        const int2 rows = rows_of_split(r, split, splits);
        const float scale = a.scale * kLog2e, unit = __uint_as_float(uint32_t(127 - row_bits(r)) << 23);
        float q[kStepColumns];
        #pragma unroll
        for (int i = 0; i < kStepColumns; ++i) {
            const int c = lane + 32 * i;
            q[i] = c < a.width ? to_float<T>(static_cast<const T*>(a.q)[b * a.q_stride + head * a.q_head_stride + c]) : 0.0f;
        }
        for (int j = rows.x + warp; j < rows.y; j += kStepWarps) {
            const T* k = j == r.length ? static_cast<const T*>(a.k) + b * a.k_stride + key_head * a.k_head_stride
                                       : static_cast<const T*>(a.keys) + b * a.keys_stride + j * a.keys_row_stride + key_head * a.keys_head_stride;
            const T* v = j == r.length ? static_cast<const T*>(a.v) + b * a.v_stride + key_head * a.v_head_stride
                                       : static_cast<const T*>(a.values) + b * a.values_stride + j * a.values_row_stride + key_head * a.values_head_stride;
            float s = 0.0f, value[kStepColumns];
            #pragma unroll
            for (int i = 0; i < kStepColumns; ++i) {
                const int c = lane + 32 * i;
                s = c < a.width ? fmaf(q[i], to_float<T>(k[c]), s) : s;
                value[i] = c < a.width ? to_float<T>(v[c]) : 0.0f;
            }
            s = warp_sum(s) * scale;
            const float most = fmaxf(m, s), base = most == -infinity() ? 0.0f : most, factor = exp2_approx(m - base), p = exp2_approx(s - base) * unit;
            m = most;
            l = fmaf(l, factor, p);
            #pragma unroll
            for (int i = 0; i < kStepColumns; ++i) o[i] = fmaf(p, value[i], o[i] * factor);
        }
        if (head % group == 0 && rows.y == r.length + 1 && rows.x < rows.y) append<T>(a, b, key_head, r.length);
    }
    if (lane == 0) warps[warp] = make_float2(m, l);
    #pragma unroll
    for (int i = 0; i < kStepColumns; ++i) outputs[warp][lane + 32 * i] = o[i];
    __syncthreads();
    const int64_t at = int64_t(b) * a.heads + head;
    float most = -infinity(), sum = 0.0f;
    #pragma unroll
    for (int w = 0; w < kStepWarps; ++w) most = fmaxf(most, warps[w].x);
    const float base = most == -infinity() ? 0.0f : most;
    #pragma unroll
    for (int w = 0; w < kStepWarps; ++w) sum = fmaf(warps[w].y, exp2_approx(warps[w].x - base), sum);
    for (int c = threadIdx.x; c < a.width; c += kStepThreads) {
        float total = 0.0f;
        #pragma unroll
        for (int w = 0; w < kStepWarps; ++w) total = fmaf(outputs[w][c], exp2_approx(warps[w].x - base), total);
        if (splits > 1) parts[(at * splits + split) * part_floats(a.width) + 4 + c] = total;
        else out[at * a.width + c] = from_float<T>(r.left_out ? 0.0f : any ? total / sum : __uint_as_float(0x7fffffffu));
    }
    if (splits > 1 && threadIdx.x == 0) *reinterpret_cast<float2*>(parts + (at * splits + split) * part_floats(a.width)) = make_float2(most, sum);
}

// ---- 16-bit heads on 16 bytes: matrix instructions of a warp ---------------------------------------------------------------------------
//
// A block has the query heads of a key head, up to 16 rows of a matrix, and a split of the sequence.  Each of its warps brings 16 or 32 keys and values at a time into places of its own in shared memory, one
// set on its way while one is used, and goes its own way until the end: no barrier of the block.  (Two sets on their way: a million rows 49 us instead of 46, 32 scenes 44 instead of 40.)  Products are m16n8k16; the arithmetic is a tenth of what they could do, so rows that no head fills cost nothing.
// (tcgen05 takes 64 rows at least, of which 4 to 16 would be used; its accumulators would have to come out of tensor memory for every 32 keys, and the step is bound by HBM.)

constexpr int kTileWarps = 4, kTileStages = 2, kTileHeads = 16, kMostClusters = 8;
template <int W> constexpr int kKeysOfSet = W == 128 ? 16 : 32;          // 64 KB to a block at most, so that some fit an SM, and one's way in and out is the others' time
// Weights are at most 1: fp16 ones carry 2^15, so that one of 2^-29 is a normal number (sums of such values are far from the end of 32 bits).
constexpr float kStepLift = 15.0f;

// Where piece `piece` (16 bytes) of a row of W values lies: eight rows of a piece are in banks of their own.
template <int W> __device__ __forceinline__ uint32_t place_of(int row, int piece) {
    return uint32_t(row * W * 2 + (W >= 64 ? piece ^ (row & 7) : piece ^ (row >> 1 & 3)) * 16);
}
__device__ __forceinline__ void load_matrices(uint32_t address, uint32_t (&v)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(address) : "memory");
}
__device__ __forceinline__ void load_turned(uint32_t address, uint32_t (&v)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(address) : "memory");
}
template <typename T> __device__ __forceinline__ void multiply_add(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// W: the width rounded up to 32, 64 or 128.  CLUSTER: the splits of a sequence are a cluster of blocks, which join them through shared memory.
template <typename T, int W, bool CLUSTER>
__global__ void __launch_bounds__(kTileWarps * 32) step_tiles_kernel(const HtgsAttentionStep a, T* out, float* parts, int splits, int chunks) {
    constexpr int kTileKeys = kKeysOfSet<W>, kSteps = W / 16, kPieces = W / 8, kCopies = kTileKeys * kPieces / 32, kRowsOfCopy = 32 / kPieces, kSetBytes = kTileKeys * W * 2;
    extern __shared__ __align__(16) unsigned char shared[];
    grid_dependency();
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    int rest = int(blockIdx.x);
    // a cluster is splits that follow one another; else blocks that run at once read the same rows' heads
    int split = 0, chunk = 0;
    if (CLUSTER) { split = rest % splits; rest /= splits; }
    chunk = rest % chunks; rest /= chunks;
    const int key_head = rest % a.key_heads;
    rest /= a.key_heads;
    if (!CLUSTER) { split = rest % splits; rest /= splits; }
    const int b = rest;
    const int group = a.heads / a.key_heads, first_head = key_head * group + chunk * kTileHeads, heads = min(kTileHeads, group - chunk * kTileHeads);
    const StepRows r = rows_of(a, b);
    const bool any = !r.left_out && !r.full;
    float most[2] = {-infinity(), -infinity()}, sum[2] = {0.0f, 0.0f}, o[kPieces][4] = {};
    if (any) {
        const int2 rows = rows_of_split(r, split, splits);
        unsigned char* const mine = shared + warp * kTileStages * 2 * kSetBytes;
        const uint32_t mine_at = smem_u32(mine);
        if (a.width < W) {               // columns that are not there: zeros, which no copy overwrites
            for (int i = lane; i < kTileStages * 2 * kTileKeys * kPieces; i += 32) {
                const int row = i / kPieces, piece = i % kPieces;
                if (piece * 8 >= a.width) *reinterpret_cast<uint4*>(mine + row / kTileKeys * kSetBytes + place_of<W>(row % kTileKeys, piece)) = make_uint4(0, 0, 0, 0);
            }
            __syncwarp();
        }
        // a lane copies piece lane % kPieces of every kRowsOfCopy-th row
        const int piece = lane % kPieces, row0 = lane / kPieces;
        const T* const keys = static_cast<const T*>(a.keys) + b * a.keys_stride + key_head * a.keys_head_stride + piece * 8;
        const T* const values = static_cast<const T*>(a.values) + b * a.values_stride + key_head * a.values_head_stride + piece * 8;
        const T* const new_key = static_cast<const T*>(a.k) + b * a.k_stride + key_head * a.k_head_stride + piece * 8;
        const T* const new_value = static_cast<const T*>(a.v) + b * a.v_stride + key_head * a.v_head_stride + piece * 8;
        const bool mine_there = piece * 8 < a.width;
        const auto begin = [&](int first, int stage) {          // rows of a set; what lies behind the split's last row is zero
            const uint32_t to = mine_at + stage * 2 * kSetBytes;
            if (mine_there && first < rows.y) {
                #pragma unroll
                for (int i = 0; i < kCopies; ++i) {
                    const int row = row0 + i * kRowsOfCopy, j = first + row;
                    const T* k = j == r.length ? new_key : keys + j * a.keys_row_stride;
                    const T* v = j == r.length ? new_value : values + j * a.values_row_stride;
                    const uint32_t bytes = j < rows.y ? 16u : 0u;
                    if (bytes == 0) { k = new_key; v = new_value; }
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + place_of<W>(row, piece)), "l"(k), "r"(bytes) : "memory");
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + kSetBytes + place_of<W>(row, piece)), "l"(v), "r"(bytes) : "memory");
                }
            }
            copies_begun();
        };
        // queries: rows lane / 4 and 8 more, columns 2 (lane % 4) and 8 more of each step
        uint32_t q[kSteps][4];
        #pragma unroll
        for (int k = 0; k < kSteps; ++k)
            #pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int head = lane / 4 + (i & 1) * 8, column = k * 16 + (lane & 3) * 2 + (i >> 1) * 8;
                q[k][i] = head < heads && column < a.width ? __ldg(reinterpret_cast<const uint32_t*>(static_cast<const T*>(a.q) + b * a.q_stride + (first_head + head) * a.q_head_stride + column)) : 0u;
            }
        const float scale = a.scale * kLog2e, lift = std::is_same<T, __half>::value ? kStepLift : -float(row_bits(r) + 1);          // bf16 weights are rounded: a half in all
        int first = rows.x + warp * kTileKeys, stage = 0;
        #pragma unroll
        for (int i = 0; i < kTileStages - 1; ++i) begin(first + i * kTileWarps * kTileKeys, i);
        for (; first < rows.y; first += kTileWarps * kTileKeys) {
            begin(first + (kTileStages - 1) * kTileWarps * kTileKeys, stage == 0 ? kTileStages - 1 : stage - 1);
            copies_done<kTileStages - 1>();
            const uint32_t at = mine_at + stage * 2 * kSetBytes;
            float s[kTileKeys / 8][4] = {};
            #pragma unroll
            for (int k = 0; k < kSteps; ++k)
                #pragma unroll
                for (int n = 0; n < kTileKeys / 16; ++n) {
                    uint32_t m[4];
                    load_matrices(at + place_of<W>(n * 16 + (lane >> 4) * 8 + (lane & 7), 2 * k + (lane >> 3 & 1)), m);
                    multiply_add<T>(s[2 * n], q[k], m[0], m[1]);
                    multiply_add<T>(s[2 * n + 1], q[k], m[2], m[3]);
                }
            float now[2] = {most[0], most[1]};
            #pragma unroll
            for (int n = 0; n < kTileKeys / 8; ++n)
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[n][i] = first + n * 8 + (lane & 3) * 2 + (i & 1) < rows.y ? s[n][i] * scale : -infinity();
                    now[i >> 1] = fmaxf(now[i >> 1], s[n][i]);
                }
            #pragma unroll
            for (int i = 0; i < 2; ++i) {
                now[i] = fmaxf(now[i], __shfl_xor_sync(0xffffffffu, now[i], 1));
                now[i] = fmaxf(now[i], __shfl_xor_sync(0xffffffffu, now[i], 2));
            }
            if (__any_sync(0xffffffffu, now[0] > most[0] || now[1] > most[1])) {
                #pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float factor = now[i] == most[i] ? 1.0f : exp2_approx(most[i] - now[i]);
                    most[i] = now[i];
                    sum[i] *= factor;
                    #pragma unroll
                    for (int c = 0; c < kPieces; ++c) { o[c][2 * i] *= factor; o[c][2 * i + 1] *= factor; }
                }
            }
            uint32_t p[kTileKeys / 8][2];
            #pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float base = (most[i] == -infinity() ? 0.0f : most[i]) - lift;
                #pragma unroll
                for (int n = 0; n < kTileKeys / 8; ++n) {
                    const float p0 = exp2_approx(s[n][2 * i] - base), p1 = exp2_approx(s[n][2 * i + 1] - base);
                    sum[i] += p0 + p1;
                    p[n][i] = floats_pair<T>(p0, p1);
                }
            }
            #pragma unroll
            for (int n = 0; n < kTileKeys / 16; ++n) {
                const uint32_t weights[4] = {p[2 * n][0], p[2 * n][1], p[2 * n + 1][0], p[2 * n + 1][1]};
                #pragma unroll
                for (int c = 0; c < kPieces; c += 2) {
                    uint32_t m[4];
                    load_turned(at + kSetBytes + place_of<W>(n * 16 + (lane >> 3 & 1) * 8 + (lane & 7), c + (lane >> 4)), m);
                    multiply_add<T>(o[c], weights, m[0], m[1]);
                    multiply_add<T>(o[c + 1], weights, m[2], m[3]);
                }
            }
            stage = stage + 1 == kTileStages ? 0 : stage + 1;
            __syncwarp();                // before the place is filled again
        }
        copies_done<0>();
        if (chunk == 0 && rows.y == r.length + 1 && rows.x < rows.y) append<T>(a, b, key_head, r.length);
        #pragma unroll
        for (int i = 0; i < 2; ++i) {
            sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
            sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
        }
    }
    // the warps' parts, joined: [warp][head]{largest, sum} and [warp][head][W]
    constexpr int kPitch = W + 4;
    float2* const tops = reinterpret_cast<float2*>(shared);
    float* const outputs = reinterpret_cast<float*>(tops + kTileWarps * kTileHeads);
    float* const joined = outputs + kTileWarps * kTileHeads * kPitch;
    __syncthreads();
    #pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int head = lane / 4 + 8 * i;
        if ((lane & 3) == 0) tops[warp * kTileHeads + head] = make_float2(most[i], sum[i]);
        #pragma unroll
        for (int c = 0; c < kPieces; ++c)
            *reinterpret_cast<float2*>(outputs + (warp * kTileHeads + head) * kPitch + c * 8 + (lane & 3) * 2) = make_float2(o[c][2 * i], o[c][2 * i + 1]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < heads * (a.width / 8); i += kTileWarps * 32) {
        const int head = i / (a.width / 8), c = i % (a.width / 8) * 8;
        float largest = -infinity(), all = 0.0f, total[8] = {};
        #pragma unroll
        for (int w = 0; w < kTileWarps; ++w) largest = fmaxf(largest, tops[w * kTileHeads + head].x);
        const float base = largest == -infinity() ? 0.0f : largest;
        #pragma unroll
        for (int w = 0; w < kTileWarps; ++w) {
            const float2 top = tops[w * kTileHeads + head];
            const float factor = exp2_approx(top.x - base);
            all = fmaf(top.y, factor, all);
            float v[8];
            load_floats<float, 4>(outputs + (w * kTileHeads + head) * kPitch + c, *reinterpret_cast<float (*)[4]>(v));
            load_floats<float, 4>(outputs + (w * kTileHeads + head) * kPitch + c + 4, *reinterpret_cast<float (*)[4]>(v + 4));
            #pragma unroll
            for (int k = 0; k < 8; ++k) total[k] = fmaf(v[k], factor, total[k]);
        }
        const int64_t at = int64_t(b) * a.heads + first_head + head;
        if (CLUSTER) {
            *reinterpret_cast<float4*>(joined + head * kPitch + c) = make_float4(total[0], total[1], total[2], total[3]);
            *reinterpret_cast<float4*>(joined + head * kPitch + c + 4) = make_float4(total[4], total[5], total[6], total[7]);
            if (c == 0) *reinterpret_cast<float4*>(joined + head * kPitch + W) = make_float4(largest, all, 0.0f, 0.0f);
        } else if (splits > 1) {
            float* to = parts + (at * splits + split) * part_floats(a.width);
            *reinterpret_cast<float4*>(to + 4 + c) = make_float4(total[0], total[1], total[2], total[3]);
            *reinterpret_cast<float4*>(to + 8 + c) = make_float4(total[4], total[5], total[6], total[7]);
            if (c == 0) *reinterpret_cast<float2*>(to) = make_float2(largest, all);
        } else {
            #pragma unroll
            for (int k = 0; k < 8; ++k) total[k] = r.left_out ? 0.0f : any ? total[k] / all : __uint_as_float(0x7fffffffu);
            store_floats<T, 8>(out + at * a.width + c, total);
        }
    }
    if constexpr (CLUSTER) {
        cluster_barrier();
        const uint32_t joined_at = smem_u32(joined);
        for (int i = split * kTileWarps * 32 + int(threadIdx.x); i < heads * (a.width / 4); i += splits * kTileWarps * 32) {
            const int head = i / (a.width / 4), c = i % (a.width / 4) * 4;
            float4 tops[kMostClusters], v[kMostClusters];
            float largest = -infinity(), all = 0.0f;
            #pragma unroll
            for (int k = 0; k < kMostClusters; ++k) {
                if (k >= splits) break;
                tops[k] = peer_float4(joined_at + uint32_t(head * kPitch + W) * 4, k);
                v[k] = peer_float4(joined_at + uint32_t(head * kPitch + c) * 4, k);
                largest = fmaxf(largest, tops[k].x);
            }
            const float base = largest == -infinity() ? 0.0f : largest;
            float total[4] = {};
            #pragma unroll
            for (int k = 0; k < kMostClusters; ++k) {
                if (k >= splits) break;
                const float factor = exp2_approx(tops[k].x - base);
                all = fmaf(tops[k].y, factor, all);
                total[0] = fmaf(v[k].x, factor, total[0]);
                total[1] = fmaf(v[k].y, factor, total[1]);
                total[2] = fmaf(v[k].z, factor, total[2]);
                total[3] = fmaf(v[k].w, factor, total[3]);
            }
            #pragma unroll
            for (int k = 0; k < 4; ++k) total[k] = r.left_out ? 0.0f : any ? total[k] / all : __uint_as_float(0x7fffffffu);
            store_floats<T, 4>(out + (int64_t(b) * a.heads + first_head + head) * a.width + c, total);
        }
        cluster_barrier();           // no block's shared memory goes before the others have read it
    }
}

// The splits of a head, joined: a warp's lanes have four columns each and its splits are every eighth; then the warps' sums.
constexpr int kJoinThreads = 256, kJoinWarps = kJoinThreads / 32;
template <typename T> __global__ void __launch_bounds__(kJoinThreads) step_join_kernel(const HtgsAttentionStep a, T* out, const float* parts, int splits) {
    __shared__ float factors[kMostSplits];
    __shared__ float4 sums[kJoinWarps][32];
    __shared__ float warps[2][kJoinWarps];
    grid_dependency();
    const int64_t at = blockIdx.x;
    const int pitch = part_floats(a.width), lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    const float* mine = parts + at * splits * pitch;
    static_assert(kMostSplits <= kJoinThreads, "a split for each thread");
    const float2 top = int(threadIdx.x) < splits ? *reinterpret_cast<const float2*>(mine + int64_t(threadIdx.x) * pitch) : make_float2(-infinity(), 0.0f);
    float most = lanes_max<32>(top.x);
    if (lane == 0) warps[0][warp] = most;
    __syncthreads();
    #pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) most = fmaxf(most, warps[0][w]);
    const float factor = exp2_approx(top.x - (most == -infinity() ? 0.0f : most)), part = warp_sum(top.y * factor);
    if (int(threadIdx.x) < splits) factors[threadIdx.x] = factor;
    if (lane == 0) warps[1][warp] = part;
    __syncthreads();
    float sum = 0.0f;
    #pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) sum += warps[1][w];
    float4 total = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (lane * 4 < a.width) {
        #pragma unroll 8
        for (int s = warp; s < splits; s += kJoinWarps) {
            const float4 v = *reinterpret_cast<const float4*>(mine + int64_t(s) * pitch + 4 + lane * 4);
            const float f = factors[s];
            total.x = fmaf(v.x, f, total.x); total.y = fmaf(v.y, f, total.y); total.z = fmaf(v.z, f, total.z); total.w = fmaf(v.w, f, total.w);
        }
    }
    sums[warp][lane] = total;
    __syncthreads();
    const int c = threadIdx.x;
    if (c >= a.width) return;
    float all = 0.0f;
    #pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) all += reinterpret_cast<const float*>(sums[w])[c];
    const StepRows r = rows_of(a, int(at / a.heads));
    out[at * a.width + c] = from_float<T>(r.left_out ? 0.0f : r.full ? __uint_as_float(0x7fffffffu) : all / sum);
}

const char* wrong(const HtgsAttentionStep* a) {
    if (!a) return "htgs_attention_step: no arguments";
    if (!known_type(a->type)) return "htgs_attention_step: unknown element type";
    if (a->batch < 0 || a->capacity < 0 || a->capacity > 0x7fffff00) return "htgs_attention_step: batch must not be negative, and the capacity below 2^31 - 256";
    if (a->key_heads < 1 || a->heads < 1 || a->heads % a->key_heads || a->heads > 65536) return "htgs_attention_step: heads must be a multiple of key_heads, at most 65536";
    if (a->width < 1 || a->width > kMostStepWidth) return "htgs_attention_step: heads must be 1 to 128 values wide";
    if (!(a->scale > 0.0f && a->scale <= FLT_MAX)) return "htgs_attention_step: scale must be positive and finite";
    if (a->q_stride < 0 || a->k_stride < 0 || a->v_stride < 0 || a->q_head_stride < 0 || a->k_head_stride < 0 || a->v_head_stride < 0 || a->keys_stride < 0 || a->values_stride < 0 ||
        a->keys_row_stride < 0 || a->values_row_stride < 0 || a->keys_head_stride < 0 || a->values_head_stride < 0) return "htgs_attention_step: strides must not be negative";
    if (a->batch && (!a->q || !a->k || !a->v || !a->lengths || (a->capacity && (!a->keys || !a->values)))) return "htgs_attention_step: no pointer may be null";
    if (int64_t(a->batch) * a->heads * kMostSplits > 0x7fffffff) return "htgs_attention_step: too many sequences and heads for one call";
    return nullptr;
}

bool step_aligned(const HtgsAttentionStep& a) {
    const auto ok = [](const void* p, int64_t n0, int64_t s0, int64_t n1, int64_t s1) { return aligned(p, 16) && (n0 == 1 || s0 % 8 == 0) && (n1 == 1 || s1 % 8 == 0); };
    return a.type != HTGS_FLOAT32 && a.width % 8 == 0 && ok(a.q, a.batch, a.q_stride, a.heads, a.q_head_stride) && ok(a.k, a.batch, a.k_stride, a.key_heads, a.k_head_stride) &&
           ok(a.v, a.batch, a.v_stride, a.key_heads, a.v_head_stride) && ok(a.keys, a.batch, a.keys_stride, a.key_heads, a.keys_head_stride) && (a.capacity <= 1 || a.keys_row_stride % 8 == 0) &&
           ok(a.values, a.batch, a.values_stride, a.key_heads, a.values_head_stride) && (a.capacity <= 1 || a.values_row_stride % 8 == 0);
}

struct StepPlan { bool tiles; int64_t blocks; int chunks, splits; bool cluster; };       // blocks: of one split
// Splits of a sequence, for caches that are full: what they hold only the device knows, and the plan has to bear the most.  (Plans for caches half or five eighths full are the same or a few splits apart, and
// within 4 % in time at an eighth, a half and all of the capacity.)  A block costs about as much as 128 rows beside its own, or 256 while it takes from others.  One sequence: the rounds of all places for a
// block, by a block's rows.  Several, whose lengths differ: blocks come and go, so all their rows spread over the places, and then the last block's.  Places are two on an SM for heads of more than 32, though
// three fit: with splits for three a million rows of 2 key heads of 64 take 114 us instead of 108 (caches out of L2), 32 full caches of 8192 rows, 2 of 128, 58 instead of 54, 100 of 3000 rows, 1 of 96, 39
// instead of 40.  Up to eight splits can be a cluster, whose join costs about 128 rows' time, where half the places are enough for all (32 scenes, 8 splits: 49 us in clusters, 42 without); else a kernel of
// its own joins them, about 512.
StepPlan plan_of(const HtgsAttentionStep& a) {
    StepPlan p{step_aligned(a), 0, 1, 1, false};
    const int group = a.heads / a.key_heads;
    if (p.tiles) p.chunks = (group + kTileHeads - 1) / kTileHeads;
    p.blocks = int64_t(a.batch) * (p.tiles ? a.key_heads * p.chunks : a.heads);
    const int64_t rows = (a.window >= 0 && a.window < a.capacity ? a.window + 1 : a.capacity) + 1, slots = 148 * (p.tiles ? (a.width <= 32 ? 4 : 2) : 8);
    int64_t best = INT64_MAX;
    for (int splits = 1; splits <= kMostSplits && (splits == 1 || rows >= splits * 128); ++splits) {
        const bool cluster = p.tiles && splits > 1 && splits <= kMostClusters && p.blocks * splits <= slots / 2;
        const int64_t time = a.batch == 1 ? (p.blocks * splits + slots - 1) / slots * (rows / splits + 128) : p.blocks * (rows + 256 * splits) / slots + rows / splits;
        const int64_t cost = time + (splits == 1 ? 0 : cluster ? 128 : 512);
        if (cost < best) { best = cost; p.splits = splits; p.cluster = cluster; }
    }
    return p;
}

template <typename T, int W, bool CLUSTER> cudaError_t launch_step(const HtgsAttentionStep& a, T* out, float* parts, const StepPlan& plan, cudaStream_t stream) {
    constexpr int smem = kTileWarps * kTileStages * 2 * kKeysOfSet<W> * W * 2;
    static_assert(kTileWarps * kTileHeads * (8 + (W + 4) * 4) + kTileHeads * (W + 4) * 4 <= smem, "the warps' parts and the block's fit the places of keys and values");
    static PerDeviceOnce once;
    const cudaError_t err = once.run([] { return cudaFuncSetAttribute(step_tiles_kernel<T, W, CLUSTER>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
    if (err != cudaSuccess) return err;
    const dim3 grid(unsigned(plan.blocks * plan.splits));
    if (!CLUSTER) return launch_after(step_tiles_kernel<T, W, CLUSTER>, grid, kTileWarps * 32, smem, stream, a, out, parts, plan.splits, plan.chunks);
    cudaLaunchAttribute attributes[2]{};
    attributes[0].id = cudaLaunchAttributeClusterDimension;
    attributes[0].val.clusterDim.x = unsigned(plan.splits); attributes[0].val.clusterDim.y = attributes[0].val.clusterDim.z = 1;
    attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = grid; config.blockDim = kTileWarps * 32; config.dynamicSmemBytes = smem; config.stream = stream;
    config.attrs = attributes; config.numAttrs = 2;
    return cudaLaunchKernelEx(&config, step_tiles_kernel<T, W, CLUSTER>, a, out, parts, plan.splits, plan.chunks);
}
template <typename T, bool CLUSTER> cudaError_t launch_step(const HtgsAttentionStep& a, T* out, float* parts, const StepPlan& plan, cudaStream_t stream) {
    return a.width <= 32 ? launch_step<T, 32, CLUSTER>(a, out, parts, plan, stream) : a.width <= 64 ? launch_step<T, 64, CLUSTER>(a, out, parts, plan, stream)
                                                                                    : launch_step<T, 128, CLUSTER>(a, out, parts, plan, stream);
}

template <typename T> int step_typed(const HtgsAttentionStep& a, void* to, float* parts, cudaStream_t stream) {
    const StepPlan plan = plan_of(a);
    T* const out = static_cast<T*>(to);
    cudaError_t err = cudaSuccess;
    bool done = false;
    if constexpr (sizeof(T) == 2) {
        if (plan.tiles) {
            err = plan.cluster ? launch_step<T, true>(a, out, parts, plan, stream) : launch_step<T, false>(a, out, parts, plan, stream);
            done = true;
        }
    }
    if (!done) err = launch_after(step_lanes_kernel<T>, dim3(unsigned(int64_t(a.batch) * a.heads * plan.splits)), kStepThreads, 0, stream, a, out, parts, plan.splits);
    if (err == cudaSuccess && plan.splits > 1 && !plan.cluster) err = launch_after(step_join_kernel<T>, dim3(unsigned(int64_t(a.batch) * a.heads)), kJoinThreads, 0, stream, a, out, parts, plan.splits);
    return err == cudaSuccess ? sequence_status("htgs_attention_step") : sequence_fail(HTGS_ERR_CUDA, cudaGetErrorString(err));
}

}  // namespace

}  // namespace htgs

extern "C" {

size_t htgs_attention_step_workspace_bytes(const HtgsAttentionStep* step) {
    using namespace htgs;
    if (wrong(step) || step->batch == 0) return 0;
    const StepPlan plan = plan_of(*step);
    return plan.splits == 1 || plan.cluster ? 0 : size_t(step->batch) * step->heads * plan.splits * part_floats(step->width) * sizeof(float);
}

int htgs_attention_step(const HtgsAttentionStep* step, void* out, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace htgs;
    if (const char* message = wrong(step)) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, message);
    if (step->batch == 0) return HTGS_OK;
    if (!out || !aligned(out, 16)) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_attention_step: out must not be null, and begin on 16 bytes");
    const size_t size = htgs_attention_step_workspace_bytes(step);
    if (size && (!workspace || !aligned(workspace, 16) || workspace_bytes < size)) return sequence_fail(HTGS_ERR_WORKSPACE_TOO_SMALL, "htgs_attention_step: the workspace is too small or not on 16 bytes");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    float* parts = static_cast<float*>(workspace);
    if (step->type == HTGS_FLOAT32) return step_typed<float>(*step, out, parts, s);
    if (step->type == HTGS_FLOAT16) return step_typed<__half>(*step, out, parts, s);
    return step_typed<__nv_bfloat16>(*step, out, parts, s);
}

}  // extern "C"
