// Attention over packed sequences: the entry points, the statistics of the backward pass, and kernels for what the tensor cores' (attention_tiles.cu) do not take: 32-bit
// values, widths that are no multiple of 8, rows that do not begin on 16 bytes.
#include "attention.cuh"

#include <algorithm>

namespace htgs {

namespace {

constexpr int kLanesThreads = 256, kLanesRows = 32, kRowsOfWarp = 4, kMostWidth = 128, kColumns = kMostWidth / 32;

// rows first + [0, 32) of a head into shared memory, zeros where there is none.
template <typename T> __device__ __forceinline__ void fill_rows(float* to, int pitch, const void* from, int64_t stride, int64_t offset, int first, int end, int width) {
    const T* p = static_cast<const T*>(from) + offset;
    for (int r = threadIdx.x / 32; r < kLanesRows; r += kLanesThreads / 32)
        for (int c = threadIdx.x & 31; c < width; c += 32) to[r * pitch + c] = first + r < end ? to_float<T>(p[(first + r) * stride + c]) : 0.0f;
}
template <typename T> __device__ __forceinline__ void store_row(T* to, const float (&v)[kColumns], float factor, int width, int lane) {
    #pragma unroll
    for (int i = 0; i < kColumns; ++i)
        if (lane + 32 * i < width) to[lane + 32 * i] = from_float<T>(v[i] * factor);
}

// 32 rows of a head, four to a warp, against 32 rows at a time of those that they see, a lane for each.  Values that a row does not see meet nothing of it: neither its sums nor, by a
// product with zero, its output.  Weights carry `unit`, so little that a row's add up to 1 at most, and no sum of values passes the largest of them.  Bound by loads from shared memory, five for four multiply-adds: 11 TFLOP/s (20011 rows in 33 sequences, 8 heads of 64: 4.98 ms).
template <typename T> __global__ void __launch_bounds__(kLanesThreads) attention_lanes_kernel(const HtgsAttention a, T* out, T* rest, float* sums) {
    extern __shared__ float shared[];
    grid_dependency();
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, pitch = a.width | 1;
    const int head = int(blockIdx.x % a.heads), key_head = head / (a.heads / a.key_heads);
    const SequenceTile t = find_tile<kLanesRows>(a, int(blockIdx.x / a.heads));
    if (t.first >= t.end) return;
    float *const qs = shared, *const ks = qs + kLanesRows * pitch, *const vs = ks + kLanesRows * pitch;
    const int rows = min(kLanesRows, t.end - t.first);
    float unit = 1.0f, m[kRowsOfWarp], l[kRowsOfWarp] = {}, o[kRowsOfWarp][kColumns] = {};
    #pragma unroll
    for (int r = 0; r < kRowsOfWarp; ++r) m[r] = -infinity();
    if (!t.outside) {
        fill_rows<T>(qs, pitch, a.q, a.q_stride, head * a.q_head_stride, t.first, t.end, a.width);
        const float scale = a.scale * kLog2e;
        const int low = first_seen(a, t.begin, t.first), high = last_seen(a, t.end, t.first + rows - 1);
        unit = __uint_as_float(uint32_t(127 - bits_of(high - low + 1)) << 23);
        for (int at = low; at <= high; at += kLanesRows) {
            __syncthreads();
            fill_rows<T>(ks, pitch, a.k, a.k_stride, key_head * a.k_head_stride, at, high + 1, a.width);
            fill_rows<T>(vs, pitch, a.v, a.v_stride, key_head * a.v_head_stride, at, high + 1, a.width);
            __syncthreads();
            float s[kRowsOfWarp] = {};
            for (int c = 0; c < a.width; ++c) {
                const float k = ks[lane * pitch + c];
                #pragma unroll
                for (int r = 0; r < kRowsOfWarp; ++r) s[r] = fmaf(qs[(warp * kRowsOfWarp + r) * pitch + c], k, s[r]);
            }
            uint32_t seen[kRowsOfWarp];
            #pragma unroll
            for (int r = 0; r < kRowsOfWarp; ++r) {
                const int i = t.first + warp * kRowsOfWarp + r, j = at + lane;
                const bool sees = i < t.end && j >= first_seen(a, t.begin, i) && j <= last_seen(a, t.end, i);
                seen[r] = __ballot_sync(0xffffffffu, sees);
                const float x = sees ? s[r] * scale : -infinity(), most = fmaxf(m[r], lanes_max<32>(x)), base = most == -infinity() ? 0.0f : most, factor = exp2_approx(m[r] - base);
                m[r] = most;
                s[r] = exp2_approx(x - base) * unit;
                l[r] = l[r] * factor + warp_sum(s[r]);
                #pragma unroll
                for (int i2 = 0; i2 < kColumns; ++i2) o[r][i2] *= factor;
            }
            for (int j = 0; j < kLanesRows; ++j) {
                float v[kColumns];
                #pragma unroll
                for (int i = 0; i < kColumns; ++i) v[i] = lane + 32 * i < a.width ? vs[j * pitch + lane + 32 * i] : 0.0f;
                #pragma unroll
                for (int r = 0; r < kRowsOfWarp; ++r) {
                    const float p = __shfl_sync(0xffffffffu, s[r], j);
                    if (!(seen[r] >> j & 1)) continue;
                    #pragma unroll
                    for (int i = 0; i < kColumns; ++i) o[r][i] = fmaf(p, v[i], o[r][i]);
                }
            }
        }
    }
    #pragma unroll
    for (int r = 0; r < kRowsOfWarp; ++r) {
        const int i = t.first + warp * kRowsOfWarp + r;
        if (i >= t.end) break;
        const int64_t at = (int64_t(i) * a.heads + head) * a.width;
        const float factor = t.outside ? 0.0f : 1.0f / l[r];
        store_row<T>(out + at, o[r], factor, a.width, lane);
        if (rest) {                    // what the rounding takes away
            #pragma unroll
            for (int c = 0; c < kColumns; ++c) o[r][c] = o[r][c] * factor - to_float<T>(from_float<T>(o[r][c] * factor));
            store_row<T>(rest + at, o[r], 1.0f, a.width, lane);
        }
        if (sums && lane == 0) sums[head * a.rows + i] = t.outside ? 0.0f : m[r] + log2f(l[r] / unit);
    }
}

// Statistics of the rows of a tile of 128 and some heads.  Bound by HBM: reads the output and its gradient once.  LANES lanes have a row, N values of it at a time each.
template <typename T, int N, int LANES> __global__ void __launch_bounds__(kLanesThreads) statistics_kernel(const HtgsAttention a, const T* out, const T* rest, const float* sums, const AttentionBackward b, float* statistics,
                                                                                                          uint32_t* largest, int heads_of_block) {
    grid_dependency();
    const int lane = threadIdx.x % LANES, group = a.heads / a.key_heads, blocks = (a.heads + heads_of_block - 1) / heads_of_block;
    const int first_head = int(blockIdx.x % blocks) * heads_of_block, last_head = min(first_head + heads_of_block, a.heads);
    const SequenceTile t = find_tile<kStatisticRows>(a, int(blockIdx.x / blocks));
    if (t.first >= t.end) return;
    const int64_t base = statistic_base(a, t) + (t.first - t.begin);
    float grads = 0.0f, values = 0.0f;
    const int count = (last_head - first_head) * kStatisticRows;
    #pragma unroll 4
    for (int x = threadIdx.x / LANES; x < count; x += kLanesThreads / LANES) {           // rows of a head, then of the next
        const int head = first_head + x / kStatisticRows, r = x % kStatisticRows;
        const int64_t i = t.first + r;
        const bool there = i < t.end && !t.outside;
        float mean = 0.0f, grad = 0.0f, value = 0.0f;
        if (there) {
            const T *o = out + (i * a.heads + head) * a.width, *g = static_cast<const T*>(b.grad) + i * b.grad_stride + head * b.grad_head_stride;
            for (int c = lane * N; c < a.width; c += LANES * N) {
                float x[N], y[N];
                load_floats<T, N>(o + c, x);
                load_floats<T, N>(g + c, y);
                #pragma unroll
                for (int k = 0; k < N; ++k) { mean = fmaf(x[k], y[k], mean); grad = fmaf(y[k], y[k], grad); }
                if (rest) {
                    load_floats<T, N>(rest + (o - out) + c, x);
                    #pragma unroll
                    for (int k = 0; k < N; ++k) mean = fmaf(x[k], y[k], mean);
                }
            }
            if (largest && head % group == 0) {
                const T* v = static_cast<const T*>(a.v) + i * a.v_stride + head / group * a.v_head_stride;
                for (int c = lane * N; c < a.width; c += LANES * N) {
                    float x[N];
                    load_floats<T, N>(v + c, x);
                    #pragma unroll
                    for (int k = 0; k < N; ++k) value = fmaf(x[k], x[k], value);
                }
            }
        }
        #pragma unroll
        for (int d = LANES / 2; d > 0; d >>= 1) {
            mean += __shfl_xor_sync(0xffffffffu, mean, d);
            if (largest) { grad += __shfl_xor_sync(0xffffffffu, grad, d); value += __shfl_xor_sync(0xffffffffu, value, d); }
        }
        if (lane == 0) {
            float* to = statistics + (head * b.statistics_rows + base) * 2;
            to[r] = there ? sums[head * a.rows + i] : 0.0f;
            to[kStatisticRows + r] = mean;
        }
        grads = fmaxf(grads, finite_magnitude(grad));
        values = fmaxf(values, finite_magnitude(value));
    }
    if (!largest || t.outside) return;
    grads = lanes_max<32>(grads);
    values = lanes_max<32>(values);
    if ((threadIdx.x & 31) == 0) {
        atomicMax(largest + 2 * t.sequence, __float_as_uint(grads));
        atomicMax(largest + 2 * t.sequence + 1, __float_as_uint(values));
    }
}

// Gradients of 32 rows of q and a head (KEYS false), or of k, v and a key head, over its query heads, against 32 rows at a time of the others, a lane for each.  Bound as the forward pass.
template <typename T, bool KEYS> __global__ void __launch_bounds__(kLanesThreads) attention_lanes_backward_kernel(const HtgsAttention a, const AttentionBackward b) {
    extern __shared__ float shared[];
    __shared__ float2 statistics[kLanesRows];
    grid_dependency();
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, pitch = a.width | 1, group = a.heads / a.key_heads, own_heads = KEYS ? a.key_heads : a.heads;
    const int own_head = int(blockIdx.x % own_heads);
    const SequenceTile t = find_tile<kLanesRows>(a, int(blockIdx.x / own_heads));
    if (t.first >= t.end) return;
    float *const own1 = shared, *const own2 = own1 + kLanesRows * pitch, *const other1 = own2 + kLanesRows * pitch, *const other2 = other1 + kLanesRows * pitch;
    const int rows = min(kLanesRows, t.end - t.first);
    const int64_t base = statistic_base(a, t);
    const float scale = a.scale * kLog2e;
    float first[kRowsOfWarp][kColumns] = {}, second[kRowsOfWarp][kColumns] = {};        // of q or k; of v
    if (!t.outside) {
        const int key_head = KEYS ? own_head : own_head / group;
        const auto fill_queries = [&](float* q, float* grad, int head, int at, int end) {
            fill_rows<T>(q, pitch, a.q, a.q_stride, head * a.q_head_stride, at, end, a.width);
            fill_rows<T>(grad, pitch, b.grad, b.grad_stride, head * b.grad_head_stride, at, end, a.width);
            if (threadIdx.x < kLanesRows && at + int(threadIdx.x) < end) {
                const int64_t r = base + (at - t.begin) + threadIdx.x;
                const float* from = b.statistics + (head * b.statistics_rows + r / kStatisticRows * kStatisticRows) * 2 + r % kStatisticRows;
                statistics[threadIdx.x] = make_float2(from[0], from[kStatisticRows]);
            }
        };
        const auto fill_keys = [&](float* k, float* v, int at, int end) {
            fill_rows<T>(k, pitch, a.k, a.k_stride, key_head * a.k_head_stride, at, end, a.width);
            fill_rows<T>(v, pitch, a.v, a.v_stride, key_head * a.v_head_stride, at, end, a.width);
        };
        if (KEYS) fill_keys(own1, own2, t.first, t.end);
        else fill_queries(own1, own2, own_head, t.first, t.end);
        const int low = KEYS ? first_seeing(a, t.begin, t.first) : first_seen(a, t.begin, t.first);
        const int high = KEYS ? last_seeing(a, t.end, t.first + rows - 1) : last_seen(a, t.end, t.first + rows - 1);
        for (int head = KEYS ? own_head * group : own_head; head < (KEYS ? (own_head + 1) * group : own_head + 1); ++head) {
            for (int at = low; at <= high; at += kLanesRows) {
                __syncthreads();
                if (KEYS) fill_queries(other1, other2, head, at, high + 1);
                else fill_keys(other1, other2, at, high + 1);
                __syncthreads();
                float s[kRowsOfWarp] = {}, ds[kRowsOfWarp] = {};
                for (int c = 0; c < a.width; ++c) {
                    const float x = other1[lane * pitch + c], y = other2[lane * pitch + c];
                    #pragma unroll
                    for (int r = 0; r < kRowsOfWarp; ++r) {
                        s[r] = fmaf(own1[(warp * kRowsOfWarp + r) * pitch + c], x, s[r]);
                        ds[r] = fmaf(own2[(warp * kRowsOfWarp + r) * pitch + c], y, ds[r]);
                    }
                }
                uint32_t seen[kRowsOfWarp];
                #pragma unroll
                for (int r = 0; r < kRowsOfWarp; ++r) {
                    const int own = t.first + warp * kRowsOfWarp + r, i = KEYS ? at + lane : own, j = KEYS ? own : at + lane;
                    const bool sees = i < t.end && j < t.end && j >= first_seen(a, t.begin, i) && j <= last_seen(a, t.end, i);
                    seen[r] = __ballot_sync(0xffffffffu, sees);
                    const float2 st = sees ? statistics[KEYS ? lane : warp * kRowsOfWarp + r] : make_float2(0.0f, 0.0f);
                    s[r] = sees ? exp2_approx(fmaf(s[r], scale, -st.x)) : 0.0f;
                    ds[r] = sees ? s[r] * (ds[r] - st.y) : 0.0f;
                }
                for (int j = 0; j < kLanesRows; ++j) {
                    float x[kColumns], y[kColumns];
                    #pragma unroll
                    for (int i = 0; i < kColumns; ++i) {
                        x[i] = lane + 32 * i < a.width ? other1[j * pitch + lane + 32 * i] : 0.0f;
                        if (KEYS) y[i] = lane + 32 * i < a.width ? other2[j * pitch + lane + 32 * i] : 0.0f;
                    }
                    #pragma unroll
                    for (int r = 0; r < kRowsOfWarp; ++r) {
                        const float w = __shfl_sync(0xffffffffu, ds[r], j), p = KEYS ? __shfl_sync(0xffffffffu, s[r], j) : 0.0f;
                        if (!(seen[r] >> j & 1)) continue;
                        #pragma unroll
                        for (int i = 0; i < kColumns; ++i) {
                            first[r][i] = fmaf(w, x[i], first[r][i]);
                            if (KEYS) second[r][i] = fmaf(p, y[i], second[r][i]);
                        }
                    }
                }
            }
        }
    }
    #pragma unroll
    for (int r = 0; r < kRowsOfWarp; ++r) {
        const int i = t.first + warp * kRowsOfWarp + r;
        if (i >= t.end) break;
        const int64_t at = (int64_t(i) * own_heads + own_head) * a.width;
        store_row<T>(static_cast<T*>(KEYS ? b.grad_k : b.grad_q) + at, first[r], a.scale, a.width, lane);
        if (KEYS) store_row<T>(static_cast<T*>(b.grad_v) + at, second[r], 1.0f, a.width, lane);
    }
}

template <typename T, typename Kernel, typename... Args>
int launch_lanes(Kernel kernel, PerDeviceOnce& once, const HtgsAttention& a, int heads, int buffers, cudaStream_t stream, const Args&... args) {
    const int most = buffers * kLanesRows * (kMostWidth | 1) * int(sizeof(float));
    cudaError_t err = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most); });
    if (err == cudaSuccess)
        err = launch_after(kernel, dim3(unsigned(sequence_tiles(a, kLanesRows) * heads)), kLanesThreads, size_t(buffers) * kLanesRows * (a.width | 1) * sizeof(float), stream, a, args...);
    return err == cudaSuccess ? sequence_status("htgs_attention") : sequence_fail(HTGS_ERR_CUDA, cudaGetErrorString(err));
}

template <typename T> int forward_lanes(const HtgsAttention& a, void* out, void* rest, float* sums, cudaStream_t stream) {
    static PerDeviceOnce once;
    return launch_lanes<T>(attention_lanes_kernel<T>, once, a, a.heads, 3, stream, static_cast<T*>(out), static_cast<T*>(rest), sums);
}
template <typename T> int backward_lanes(const HtgsAttention& a, const AttentionBackward& b, cudaStream_t stream) {
    static PerDeviceOnce once, once_keys;
    const int code = launch_lanes<T>(attention_lanes_backward_kernel<T, false>, once, a, a.heads, 4, stream, b);
    return code != HTGS_OK ? code : launch_lanes<T>(attention_lanes_backward_kernel<T, true>, once_keys, a, a.key_heads, 4, stream, b);
}
template <typename T, int N, int LANES>
int launch_statistics(const HtgsAttention& a, const void* out, const void* rest, const float* sums, const AttentionBackward& b, float* statistics, uint32_t* largest, cudaStream_t stream) {
    // Some heads to a block, as long as there are eight blocks for each SM: the way in costs as much as a head (100003 rows, 8 heads of 32 in 7 sequences: 41 us with one head to a block, 39 with four).
    const int64_t tiles = sequence_tiles(a, kStatisticRows);
    const int heads = int(std::max<int64_t>(1, std::min<int64_t>(a.heads, tiles * a.heads / (148 * 8))));
    const cudaError_t err = launch_after(statistics_kernel<T, N, LANES>, dim3(unsigned(tiles * ((a.heads + heads - 1) / heads))), kLanesThreads, 0, stream, a, static_cast<const T*>(out), static_cast<const T*>(rest), sums, b,
                                         statistics, largest, heads);
    return err == cudaSuccess ? sequence_status("htgs_attention_backward") : sequence_fail(HTGS_ERR_CUDA, cudaGetErrorString(err));
}
template <typename T> int backward_typed(const HtgsAttention& a, const void* out, const void* rest, const float* sums, AttentionBackward b, float* statistics, uint32_t* largest, cudaStream_t stream) {
    const bool tiles = aligned(out, 16) && aligned(rest, 16) && attention_tiles_take(a, b);
    if constexpr (sizeof(T) == 2) {
        if (tiles) {
            if (std::is_same<T, __half>::value) {
                const cudaError_t err = cudaMemsetAsync(largest, 0, (size_t(a.n_sequences) + 2) * 2 * sizeof(uint32_t), stream);
                if (err != cudaSuccess) return sequence_fail(HTGS_ERR_CUDA, cudaGetErrorString(err));
                b.largest = largest;
            } else largest = nullptr;
            const int code = a.width <= 32 ? launch_statistics<T, 8, 4>(a, out, rest, sums, b, statistics, largest, stream)
                             : a.width <= 64 ? launch_statistics<T, 8, 8>(a, out, rest, sums, b, statistics, largest, stream) : launch_statistics<T, 8, 16>(a, out, rest, sums, b, statistics, largest, stream);
            return code != HTGS_OK ? code : attention_tiles_backward(a, b, stream);
        }
    }
    const int code = launch_statistics<T, 1, 32>(a, out, rest, sums, b, statistics, nullptr, stream);
    return code != HTGS_OK ? code : backward_lanes<T>(a, b, stream);
}

ErrorWords& error_words() {
    static ErrorWords words;
    return words;
}
int reported(unsigned int* word) { return htgs::reported(word, "htgs_attention: a wait in an earlier call on this device ran out, and its result is not complete"); }

// What a call may not be; nullptr if all is well.
const char* wrong(const HtgsAttention* a) {
    if (!a) return "htgs_attention: no arguments";
    if (!known_type(a->type)) return "htgs_attention: unknown element type";
    if (a->rows < 0 || a->rows > 0x7fffff00 || a->n_sequences < 1 || a->n_sequences > 0x7fffff00) return "htgs_attention: rows and n_sequences must be below 2^31 - 256, and n_sequences at least 1";
    if (!a->offsets && a->rows % a->n_sequences) return "htgs_attention: rows must be a multiple of n_sequences where there are no offsets";
    if (a->key_heads < 1 || a->heads < 1 || a->heads % a->key_heads || a->heads > 65536) return "htgs_attention: heads must be a multiple of key_heads, at most 65536";
    if (a->width < 1 || a->width > kMostWidth) return "htgs_attention: heads must be 1 to 128 values wide";
    if (!(a->scale > 0.0f && a->scale <= FLT_MAX)) return "htgs_attention: scale must be positive and finite";
    if (a->q_stride < 0 || a->k_stride < 0 || a->v_stride < 0 || a->q_head_stride < 0 || a->k_head_stride < 0 || a->v_head_stride < 0) return "htgs_attention: strides must not be negative";
    if (a->rows && (!a->q || !a->k || !a->v)) return "htgs_attention: q, k and v must not be null";
    if (sequence_tiles(*a, kLanesRows) * a->heads > 0x7fffffff) return "htgs_attention: too many rows and heads for one call";
    return nullptr;
}

}  // namespace

unsigned int* attention_error_word(int device) { return error_words().of(device); }

}  // namespace htgs

extern "C" {

unsigned int* htgs_attention_error_word(int32_t device) { return htgs::attention_error_word(device); }

int htgs_attention_status(int32_t device) {
    using namespace htgs;
    if (device < 0 || device >= ErrorWords::kMostDevices) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_attention_status: no such device");
    return reported(attention_error_word(device));
}

int htgs_attention(const HtgsAttention* attention, void* out, void* rest, float* sums, void* stream) {
    using namespace htgs;
    if (const char* message = wrong(attention)) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, message);
    if (attention->rows == 0) return HTGS_OK;
    if (!out) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_attention: out must not be null");
    if (const int code = reported(attention_error_word(current_device())); code != HTGS_OK) return code;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const HtgsAttention& a = *attention;
    if (attention_tiles_take(a, out, rest)) return attention_tiles_forward(a, out, rest, sums, s);
    if (a.type == HTGS_FLOAT32) return forward_lanes<float>(a, out, rest, sums, s);
    if (a.type == HTGS_FLOAT16) return forward_lanes<__half>(a, out, rest, sums, s);
    return forward_lanes<__nv_bfloat16>(a, out, rest, sums, s);
}

size_t htgs_attention_backward_workspace_bytes(const HtgsAttention* attention) {
    using namespace htgs;
    if (wrong(attention) || attention->rows == 0) return 0;
    const size_t largest = attention->type == HTGS_FLOAT16 ? (size_t(attention->n_sequences) + 2) * 2 * sizeof(uint32_t) : 0;
    return size_t(statistic_rows(*attention)) * attention->heads * 2 * sizeof(float) + largest;
}

int htgs_attention_backward(const HtgsAttention* attention, const void* out, const void* rest, const float* sums, const void* grad_out, int64_t grad_out_stride, int64_t grad_out_head_stride,
                            void* grad_q, void* grad_k, void* grad_v, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace htgs;
    if (const char* message = wrong(attention)) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, message);
    if (attention->rows == 0) return HTGS_OK;
    if (!out || !sums || !grad_out || !grad_q || !grad_k || !grad_v) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_attention_backward: no pointer may be null");
    if (grad_out_stride < 0 || grad_out_head_stride < 0) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_attention_backward: strides must not be negative");
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < htgs_attention_backward_workspace_bytes(attention))
        return sequence_fail(HTGS_ERR_WORKSPACE_TOO_SMALL, "htgs_attention_backward: the workspace is too small or not on 16 bytes");
    if (const int code = reported(attention_error_word(current_device())); code != HTGS_OK) return code;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const HtgsAttention& a = *attention;
    float* statistics = static_cast<float*>(workspace);
    const int64_t rows = statistic_rows(a);
    uint32_t* largest = reinterpret_cast<uint32_t*>(statistics + rows * a.heads * 2);
    const AttentionBackward b{grad_out, grad_out_stride, grad_out_head_stride, grad_q, grad_k, grad_v, statistics, rows, nullptr};
    if (a.type == HTGS_FLOAT32) return backward_typed<float>(a, out, rest, sums, b, statistics, largest, s);
    if (a.type == HTGS_FLOAT16) return backward_typed<__half>(a, out, rest, sums, b, statistics, largest, s);
    return backward_typed<__nv_bfloat16>(a, out, rest, sums, b, statistics, largest, s);
}

}  // extern "C"
