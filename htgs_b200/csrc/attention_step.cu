// Attention of one more row for each of many sequences over their caches (htgs_attention_step):
//
//   out = sum over cached rows j of softmax_j(scale * q . k_j) v_j,   the new row among them.
//
// A cache is read once: bound by HBM where caches are long, by the launch where they are short.  The rows of a sequence are split over blocks, by its length, which only the device knows;
// each leaves its largest score, its sum and its unnormalised output, and a second kernel joins them, always in the same order.
#include "attention.cuh"

namespace htgs {

namespace {

constexpr int kStepThreads = 256, kStepWarps = kStepThreads / 32, kMostStepWidth = 128, kStepColumns = kMostStepWidth / 32, kStepPiece = 16, kMostSplits = 256;

struct StepRows { int low, length; bool left_out, full; };        // rows [low, length], the last one new

__device__ __forceinline__ StepRows rows_of(const HtgsAttentionStep& a, int b) {
    const int n = __ldg(a.lengths + b);
    return {a.window >= 0 && n > a.window ? n - a.window : 0, n, n < 0, n >= a.capacity};
}
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

// One head and split to a block, a row at a time to a warp, columns to its lanes.
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
        const float scale = a.scale * kLog2e;
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
            const float most = fmaxf(m, s), base = most == -infinity() ? 0.0f : most, factor = exp2_approx(m - base), p = exp2_approx(s - base);
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

// The splits of a head, joined.
template <typename T> __global__ void __launch_bounds__(kMostStepWidth) step_join_kernel(const HtgsAttentionStep a, T* out, const float* parts, int splits) {
    __shared__ float factors[kMostSplits];
    grid_dependency();
    const int64_t at = blockIdx.x;
    const int pitch = part_floats(a.width), lane = threadIdx.x & 31;
    const StepRows r = rows_of(a, int(at / a.heads));
    const float* mine = parts + at * splits * pitch;
    if (threadIdx.x < 32) {
        float most = -infinity(), sum = 0.0f;
        for (int s = lane; s < splits; s += 32) most = fmaxf(most, mine[s * pitch]);
        most = lanes_max<32>(most);
        const float base = most == -infinity() ? 0.0f : most;
        for (int s = lane; s < splits; s += 32) {
            const float2 part = *reinterpret_cast<const float2*>(mine + s * pitch);
            factors[s] = exp2_approx(part.x - base);
            sum = fmaf(part.y, factors[s], sum);
        }
        sum = warp_sum(sum);
        for (int s = lane; s < splits; s += 32) factors[s] /= sum;
    }
    __syncthreads();
    const int c = threadIdx.x;
    if (c >= a.width) return;
    float total = 0.0f;
    for (int s = 0; s < splits; ++s) total = fmaf(mine[s * pitch + 4 + c], factors[s], total);
    out[at * a.width + c] = from_float<T>(r.left_out ? 0.0f : r.full ? __uint_as_float(0x7fffffffu) : total);
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

// Blocks for each head (or key head and its query heads): enough to fill the GPU, none with fewer than 256 rows of a full cache.
int splits_of(const HtgsAttentionStep& a, int64_t blocks) {
    const int64_t rows = a.window >= 0 && a.window < a.capacity ? a.window + 1 : a.capacity;
    const int64_t most = (rows + 255) / 256, wanted = (148 * 4 + blocks - 1) / blocks;
    const int64_t splits = wanted < most ? wanted : most;
    return int(splits < 1 ? 1 : splits > kMostSplits ? kMostSplits : splits);
}

template <typename T> int step_typed(const HtgsAttentionStep& a, void* out, float* parts, cudaStream_t stream) {
    const int64_t blocks = int64_t(a.batch) * a.heads;
    const int splits = splits_of(a, blocks);
    cudaError_t err = launch_after(step_lanes_kernel<T>, dim3(unsigned(blocks * splits)), kStepThreads, 0, stream, a, static_cast<T*>(out), parts, splits);
    if (err == cudaSuccess && splits > 1) err = launch_after(step_join_kernel<T>, dim3(unsigned(blocks)), kMostStepWidth, 0, stream, a, static_cast<T*>(out), parts, splits);
    return err == cudaSuccess ? sequence_status("htgs_attention_step") : sequence_fail(HTGS_ERR_CUDA, cudaGetErrorString(err));
}

}  // namespace

}  // namespace htgs

extern "C" {

size_t htgs_attention_step_workspace_bytes(const HtgsAttentionStep* step) {
    using namespace htgs;
    if (wrong(step) || step->batch == 0) return 0;
    const int64_t blocks = int64_t(step->batch) * step->heads;
    const int splits = splits_of(*step, blocks);
    return splits == 1 ? 0 : size_t(blocks) * splits * part_floats(step->width) * sizeof(float);
}

int htgs_attention_step(const HtgsAttentionStep* step, void* out, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace htgs;
    if (const char* message = wrong(step)) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, message);
    if (step->batch == 0) return HTGS_OK;
    if (!out) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_attention_step: out must not be null");
    const size_t size = htgs_attention_step_workspace_bytes(step);
    if (size && (!workspace || !aligned(workspace, 16) || workspace_bytes < size)) return sequence_fail(HTGS_ERR_WORKSPACE_TOO_SMALL, "htgs_attention_step: the workspace is too small or not on 16 bytes");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    float* parts = static_cast<float*>(workspace);
    if (step->type == HTGS_FLOAT32) return step_typed<float>(*step, out, parts, s);
    if (step->type == HTGS_FLOAT16) return step_typed<__half>(*step, out, parts, s);
    return step_typed<__nv_bfloat16>(*step, out, parts, s);
}

}  // extern "C"
