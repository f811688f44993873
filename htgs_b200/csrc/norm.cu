// Root-mean-square norm of a residual stream, with the residual's addition, forward and backward, and with an 8-bit output.
//
//   u = x + residual;   rho = 1 / sqrt(mean(u^2) + eps);   y = u * rho * weight;   sum = u in the stream's type
//   backward, with unit = u * rho and z = weight * grad_y:
//       grad_x = grad_residual = rho * (z - unit * mean(z * unit)) + grad_sum;      grad_weight = sum over rows of grad_y * unit
//
// A row stays in registers between its statistics and its output, so every value crosses HBM once: read x and residual, write sum
// and y (or 8-bit codes and a scale byte for each 128 columns); backward read grad_y, grad_sum, x and residual, write one gradient that
// serves x and residual alike.  Bound by HBM.  Forward, a warp holds a row of up to 1024 columns (32 values a lane), eight warps a wider one.
// Sums are 32-bit and u is never rounded where it is computed with: the backward pass adds x and residual again rather than read the stream, whose
// rounding to 16 bits would show in grad_weight (relative error 0.0028 instead of 0.0018 at 65537 x 1024 in bf16) for 2 bytes less of 16 a value.
#include "sequence.cuh"

namespace htgs {

namespace {

constexpr int kNormBlock = 256;
constexpr int kNormWarps = kNormBlock / 32;
constexpr int kBackwardColumns = 8;                // a thread
constexpr int kNarrowBlock = 128, kNarrowBlocks = 4, kWideBlock = 1024;
constexpr int kMaxNormWidth = kNormBlock * 32;

struct NormArgs {
    const void* x; const void* residual; const void* weight;
    int64_t x_stride, residual_stride;
    void* y; void* sum; float* rstd; uint8_t* codes; uint8_t* scales;
    int64_t y_stride, sum_stride, codes_stride, scales_stride;
    int64_t rows;
    int32_t width;
    float eps;
};

struct NormBackwardArgs {
    const void* grad_y; const void* grad_sum; const void* x; const void* residual; const void* weight; const float* rstd;
    int64_t grad_y_stride, grad_sum_stride, x_stride, residual_stride, grad_x_stride;
    void* grad_x; float* partial;
    int64_t rows;
    int32_t width;
};

// Sum over the WPR warps that share a row.
template <int WPR> __device__ __forceinline__ float row_sum(float v, float* shared) {
    v = warp_sum(v);
    if (WPR == 1) return v;
    __syncthreads();                    // the previous use of `shared` is over
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    float total = 0.0f;
    #pragma unroll
    for (int w = 0; w < WPR; ++w) total += shared[w];
    return total;
}

// E values a lane, in groups of VEC side by side; group j of a warp starts at column (32 * j + lane) * VEC of the warp's 32 * E, so
// that a block of 128 columns is held by 16 or 32 lanes of one group (VEC 8, 4) or by two or four groups (VEC 2, 1) of one warp.
template <typename T, int VEC, int E, int WPR, bool FP8>
__global__ void __launch_bounds__(kNormBlock) norm_kernel(const NormArgs a) {
    __shared__ float shared[kNormWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = int64_t(blockIdx.x) * (kNormWarps / WPR) + (WPR == 1 ? warp : 0);
    if (row >= a.rows) return;          // whole warps where WPR is 1, never where it is 8
    const int base = WPR == 1 ? 0 : warp * 32 * E;
    constexpr int G = E / VEC;
    float u[G][VEC];
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* residual = a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride : nullptr;
    float squares = 0.0f;
    #pragma unroll
    for (int j = 0; j < G; ++j) {
        const int column = base + (32 * j + lane) * VEC;
        if (column < a.width) load_floats<T, VEC>(x + column, u[j]);
        else {
            #pragma unroll
            for (int i = 0; i < VEC; ++i) u[j][i] = 0.0f;
        }
    }
    if (residual) {
        #pragma unroll
        for (int j = 0; j < G; ++j) {
            const int column = base + (32 * j + lane) * VEC;
            if (column >= a.width) continue;
            float r[VEC];
            load_floats<T, VEC>(residual + column, r);
            #pragma unroll
            for (int i = 0; i < VEC; ++i) u[j][i] += r[i];
        }
    }
    #pragma unroll
    for (int j = 0; j < G; ++j) {
        #pragma unroll
        for (int i = 0; i < VEC; ++i) squares += u[j][i] * u[j][i];
    }
    const float rho = rsqrtf(row_sum<WPR>(squares, shared) / float(a.width) + a.eps);
    if (a.rstd && threadIdx.x % (32 * WPR) == 0) a.rstd[row] = rho;
    T* sum = a.sum ? static_cast<T*>(a.sum) + row * a.sum_stride : nullptr;
    const T* weight = static_cast<const T*>(a.weight);
    #pragma unroll
    for (int j = 0; j < G; ++j) {
        const int column = base + (32 * j + lane) * VEC;
        if (column < a.width) {
            if (sum) store_floats<T, VEC>(sum + column, u[j]);
            float w[VEC];
            load_floats<T, VEC>(weight + column, w);
            #pragma unroll
            for (int i = 0; i < VEC; ++i) u[j][i] = u[j][i] * rho * w[i];
            if (!FP8) store_floats<T, VEC>(static_cast<T*>(a.y) + row * a.y_stride + column, u[j]);
        }
    }
    if (FP8) {
        uint8_t* codes = a.codes + row * a.codes_stride;
        uint8_t* scales = a.scales + row * a.scales_stride;
        constexpr int kGroups = VEC < 4 ? 4 / VEC : 1;               // groups in a block of 128 columns
        constexpr int kLanes = VEC == 8 ? 16 : 32;                   // lanes
        #pragma unroll
        for (int j = 0; j < G; j += kGroups) {
            float largest = 0.0f;
            #pragma unroll
            for (int k = 0; k < kGroups; ++k) largest = largest_magnitude(u[j + k], largest);
            const bool careful = __any_sync(0xffffffffu, largest > FLT_MAX);
            if (careful) {
                largest = 0.0f;
                #pragma unroll
                for (int k = 0; k < kGroups; ++k) largest = largest_finite(u[j + k], largest);
            }
            const int e = scale_exponent(lanes_max<kLanes>(largest));
            const float inverse = inverse_scale(e);
            #pragma unroll
            for (int k = 0; k < kGroups; ++k) {
                const int column = base + (32 * (j + k) + lane) * VEC;
                if (column >= a.width) continue;
                if (careful) store_codes<true>(codes + column, u[j + k], inverse);
                else store_codes<false>(codes + column, u[j + k], inverse);
                if (k == 0 && lane % kLanes == 0) scales[column / kScaleBlock] = uint8_t(e + 127);
            }
        }
    }
}

// A block holds whole rows, eight columns a thread, and takes R of them at a time, so that enough loads are on their way; persistent, with
// each thread's part of grad_weight in registers until the end.  Groups of VEC columns as in norm_kernel, 256 columns a warp.
// Blocks of up to 128 threads (1024 columns), four per SM, have registers for four rows of 16-bit groups (two of others); wider ones take one.
template <typename T, int VEC, int MOST>
__global__ void __launch_bounds__(MOST, MOST == kNarrowBlock ? kNarrowBlocks : 1) norm_backward_kernel(const NormBackwardArgs a) {
    constexpr int G = kBackwardColumns / VEC, R = MOST != kNarrowBlock ? 1 : VEC > 1 && sizeof(T) == 2 ? 4 : 2;
    __shared__ float shared[2][32][R];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int base = warp * 32 * kBackwardColumns;
    float w[G][VEC] = {}, grad_weight[G][VEC] = {};
    #pragma unroll
    for (int j = 0; j < G; ++j) {
        const int column = base + (32 * j + lane) * VEC;
        if (column < a.width) load_floats<T, VEC>(static_cast<const T*>(a.weight) + column, w[j]);
    }
    const float per_width = 1.0f / float(a.width);
    int buffer = 0;
    for (int64_t row0 = int64_t(blockIdx.x) * R; row0 < a.rows; row0 += int64_t(gridDim.x) * R, buffer ^= 1) {
        Pack<T, VEC> g[R][G], x[R][G], r[R][G], d[R][G];          // as they are in memory: half the registers of 32-bit values
        float rho[R];
        #pragma unroll
        for (int k = 0; k < R; ++k) {
            const int64_t row = min(row0 + k, a.rows - 1);
            rho[k] = row0 + k < a.rows ? a.rstd[row] : 0.0f;
            #pragma unroll
            for (int j = 0; j < G; ++j) {
                const int column = base + (32 * j + lane) * VEC;
                if (column < a.width && row0 + k < a.rows) {
                    g[k][j] = *reinterpret_cast<const Pack<T, VEC>*>(static_cast<const T*>(a.grad_y) + row * a.grad_y_stride + column);
                    x[k][j] = *reinterpret_cast<const Pack<T, VEC>*>(static_cast<const T*>(a.x) + row * a.x_stride + column);
                    if (a.residual) r[k][j] = *reinterpret_cast<const Pack<T, VEC>*>(static_cast<const T*>(a.residual) + row * a.residual_stride + column);
                    if (a.grad_sum) d[k][j] = *reinterpret_cast<const Pack<T, VEC>*>(static_cast<const T*>(a.grad_sum) + row * a.grad_sum_stride + column);
                } else {
                    #pragma unroll
                    for (int i = 0; i < VEC; ++i) g[k][j].v[i] = x[k][j].v[i] = r[k][j].v[i] = from_float<T>(0.0f);
                }
            }
        }
        float mean[R];
        #pragma unroll
        for (int k = 0; k < R; ++k) {
            float dot = 0.0f;
            #pragma unroll
            for (int j = 0; j < G; ++j) {
                float gy[VEC], u[VEC];
                to_floats<T, VEC>(g[k][j], gy);
                to_floats<T, VEC>(x[k][j], u);
                if (a.residual) {
                    float v[VEC];
                    to_floats<T, VEC>(r[k][j], v);
                    #pragma unroll
                    for (int i = 0; i < VEC; ++i) u[i] += v[i];
                }
                #pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float term = gy[i] * (u[i] * rho[k]);
                    grad_weight[j][i] += term;
                    dot = fmaf(term, w[j][i], dot);
                }
            }
            mean[k] = warp_sum(dot);
        }
        if (warps > 1) {
            if (lane == 0) {
                #pragma unroll
                for (int k = 0; k < R; ++k) shared[buffer][warp][k] = mean[k];
            }
            __syncthreads();            // one per trip: the other buffer is read before the next one
            #pragma unroll
            for (int k = 0; k < R; ++k) mean[k] = 0.0f;
            for (int v = 0; v < warps; ++v) {
                #pragma unroll
                for (int k = 0; k < R; ++k) mean[k] += shared[buffer][v][k];
            }
        }
        #pragma unroll
        for (int k = 0; k < R; ++k) {
            if (row0 + k >= a.rows) break;
            T* grad_x = static_cast<T*>(a.grad_x) + (row0 + k) * a.grad_x_stride;
            const float slope = mean[k] * per_width * rho[k];
            #pragma unroll
            for (int j = 0; j < G; ++j) {
                const int column = base + (32 * j + lane) * VEC;
                if (column >= a.width) continue;
                float gy[VEC], u[VEC], out[VEC];
                to_floats<T, VEC>(g[k][j], gy);
                to_floats<T, VEC>(x[k][j], u);
                if (a.residual) {
                    float v[VEC];
                    to_floats<T, VEC>(r[k][j], v);
                    #pragma unroll
                    for (int i = 0; i < VEC; ++i) u[i] += v[i];
                }
                #pragma unroll
                for (int i = 0; i < VEC; ++i) out[i] = rho[k] * (gy[i] * w[j][i] - u[i] * slope);
                if (a.grad_sum) {
                    float v[VEC];
                    to_floats<T, VEC>(d[k][j], v);
                    #pragma unroll
                    for (int i = 0; i < VEC; ++i) out[i] += v[i];
                }
                store_floats<T, VEC>(grad_x + column, out);
            }
        }
    }
    float* partial = a.partial + int64_t(blockIdx.x) * a.width;
    #pragma unroll
    for (int j = 0; j < G; ++j) {
        const int column = base + (32 * j + lane) * VEC;
        if (column >= a.width) continue;
        #pragma unroll
        for (int i = 0; i < VEC; ++i) partial[column + i] = grad_weight[j][i];
    }
}

// Sums the blocks' partial gradients of the weight, always in the same order.  32 columns by 32 slices of the blocks, four of a slice's on their way at a time.
template <typename T> __global__ void __launch_bounds__(1024) norm_weight_kernel(const float* partial, int blocks, int width, T* grad_weight) {
    __shared__ float shared[32][33];
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, column = blockIdx.x * 32 + lane;
    grid_dependency();
    float sum[4] = {};
    if (column < width) {
        for (int b = slice; b < blocks; b += 128) {
            #pragma unroll
            for (int i = 0; i < 4; ++i)
                if (b + 32 * i < blocks) sum[i] += partial[int64_t(b + 32 * i) * width + column];
        }
    }
    shared[slice][lane] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    __syncthreads();
    const float total = warp_sum(shared[lane][slice]);       // of column `slice`
    if (lane == 0 && int(blockIdx.x) * 32 + slice < width) grad_weight[blockIdx.x * 32 + slice] = from_float<T>(total);
}

int backward_threads(int width) { return (width + 32 * kBackwardColumns - 1) / (32 * kBackwardColumns) * 32; }
// Persistent blocks, each with one partial sum of grad_weight: as many threads per SM as their registers allow.
int backward_blocks(int64_t rows, int width) {
    const int threads = backward_threads(width), per_sm = (threads <= kNarrowBlock ? kNarrowBlock * kNarrowBlocks : kWideBlock) / threads;
    const int64_t blocks = (rows + 1) / 2, most = 148 * per_sm;
    return int(blocks < most ? blocks : most);
}

template <typename T, int VEC, int E, int WPR> void launch_norm(const NormArgs& a, cudaStream_t stream) {
    const unsigned int blocks = unsigned((a.rows + kNormWarps / WPR - 1) / (kNormWarps / WPR));
    if (a.codes) norm_kernel<T, VEC, E, WPR, true><<<blocks, kNormBlock, 0, stream>>>(a);
    else norm_kernel<T, VEC, E, WPR, false><<<blocks, kNormBlock, 0, stream>>>(a);
}

// The fewest values a lane that hold a row: one warp up to 1024 columns, then eight.
#define HTGS_NORM_WIDTHS(launch, args)                                                              \
    do {                                                                                            \
        if (args.width <= 32 * 8) launch<T, VEC, 8, 1>(args, stream);                               \
        else if (args.width <= 32 * 16) launch<T, VEC, 16, 1>(args, stream);                        \
        else if (args.width <= 32 * 32) launch<T, VEC, 32, 1>(args, stream);                        \
        else if (args.width <= 256 * 8) launch<T, VEC, 8, 8>(args, stream);                         \
        else if (args.width <= 256 * 16) launch<T, VEC, 16, 8>(args, stream);                       \
        else launch<T, VEC, 32, 8>(args, stream);                                                   \
    } while (0)

template <typename T, int VEC> void norm_widths(const NormArgs& a, cudaStream_t stream) { HTGS_NORM_WIDTHS(launch_norm, a); }
template <typename T, int VEC> void backward_launch(const NormBackwardArgs& a, cudaStream_t stream) {
    const int threads = backward_threads(a.width), blocks = backward_blocks(a.rows, a.width);
    if (threads <= kNarrowBlock) norm_backward_kernel<T, VEC, kNarrowBlock><<<blocks, threads, 0, stream>>>(a);
    else norm_backward_kernel<T, VEC, kWideBlock><<<blocks, threads, 0, stream>>>(a);
}

// Groups of 16 bytes where every row of every tensor allows them, of 4 where they allow that, single values otherwise.
template <typename T> void norm_typed(const NormArgs& a, cudaStream_t stream) {
    const auto allow = [&](int values) {
        const size_t e = sizeof(T), bytes = values * e;
        return a.width % values == 0 && rows_aligned(a.x, a.x_stride, a.rows, e, bytes) && rows_aligned(a.residual, a.residual_stride, a.rows, e, bytes) &&
               aligned(a.weight, bytes) && rows_aligned(a.y, a.y_stride, a.rows, e, bytes) && rows_aligned(a.sum, a.sum_stride, a.rows, e, bytes) &&
               rows_aligned(a.codes, a.codes_stride, a.rows, 1, values);
    };
    if (allow(16 / int(sizeof(T)))) norm_widths<T, 16 / int(sizeof(T))>(a, stream);
    else if (sizeof(T) == 2 && allow(2)) norm_widths<T, sizeof(T) == 2 ? 2 : 1>(a, stream);
    else norm_widths<T, 1>(a, stream);
}
template <typename T> void backward_typed(const NormBackwardArgs& a, void* grad_weight, cudaStream_t stream) {
    const auto allow = [&](int values) {
        const size_t e = sizeof(T), bytes = values * e;
        return a.width % values == 0 && rows_aligned(a.grad_y, a.grad_y_stride, a.rows, e, bytes) && rows_aligned(a.grad_sum, a.grad_sum_stride, a.rows, e, bytes) &&
               rows_aligned(a.x, a.x_stride, a.rows, e, bytes) && rows_aligned(a.residual, a.residual_stride, a.rows, e, bytes) && aligned(a.weight, bytes) &&
               rows_aligned(a.grad_x, a.grad_x_stride, a.rows, e, bytes);
    };
    if (allow(16 / int(sizeof(T)))) backward_launch<T, 16 / int(sizeof(T))>(a, stream);
    else if (sizeof(T) == 2 && allow(2)) backward_launch<T, sizeof(T) == 2 ? 2 : 1>(a, stream);
    else backward_launch<T, 1>(a, stream);
    (void)launch_after(norm_weight_kernel<T>, (a.width + 31) / 32, 1024, 0, stream, static_cast<const float*>(a.partial), backward_blocks(a.rows, a.width), int(a.width),
                       static_cast<T*>(grad_weight));      // the caller asks for the last error
}

}  // namespace

}  // namespace htgs

extern "C" {

int htgs_add_rms_norm(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride, const void* weight, int type, int64_t rows,
                      int32_t width, float eps, void* y, int64_t y_stride, void* sum, int64_t sum_stride, float* rstd, uint8_t* codes,
                      int64_t codes_stride, uint8_t* scales, int64_t scales_stride, void* stream) {
    using namespace htgs;
    if (!known_type(type)) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_add_rms_norm: unknown element type");
    if (rows < 0 || rows > 0x7fffffff || width < 1 || width > kMaxNormWidth)
        return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_add_rms_norm: rows must be in [0, 2^31), width in [1, 8192]");
    if (!(eps >= 0.0f)) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_add_rms_norm: eps must be >= 0");
    if (rows == 0) return HTGS_OK;
    if (!x || !weight || (y != nullptr) == (codes != nullptr) || (codes != nullptr) != (scales != nullptr))
        return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_add_rms_norm: x, weight and either y or codes with scales must be given");
    const NormArgs a{x, residual, weight, x_stride, residual_stride, y, sum, rstd, codes, scales, y_stride, sum_stride, codes_stride, scales_stride,
                     rows, width, eps};
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (type == HTGS_FLOAT32) norm_typed<float>(a, s);
    else if (type == HTGS_FLOAT16) norm_typed<__half>(a, s);
    else norm_typed<__nv_bfloat16>(a, s);
    return sequence_status("htgs_add_rms_norm");
}

size_t htgs_add_rms_norm_backward_scratch_bytes(int64_t rows, int32_t width) {
    if (rows <= 0 || width <= 0) return 0;
    return size_t(htgs::backward_blocks(rows, width)) * size_t(width) * sizeof(float);
}

int htgs_add_rms_norm_backward(const void* grad_y, int64_t grad_y_stride, const void* grad_sum, int64_t grad_sum_stride, const void* x, int64_t x_stride,
                               const void* residual, int64_t residual_stride, const void* weight, const float* rstd, int type, int64_t rows, int32_t width,
                               void* grad_x, int64_t grad_x_stride, void* grad_weight, void* scratch, size_t scratch_bytes, void* stream) {
    using namespace htgs;
    if (!known_type(type)) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_add_rms_norm_backward: unknown element type");
    if (rows < 0 || rows > 0x7fffffff || width < 1 || width > kMaxNormWidth)
        return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_add_rms_norm_backward: rows must be in [0, 2^31), width in [1, 8192]");
    if (!grad_weight) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_add_rms_norm_backward: grad_weight must not be null");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (rows == 0) {
        const cudaError_t err = cudaMemsetAsync(grad_weight, 0, size_t(width) * type_bytes(type), s);
        return err == cudaSuccess ? HTGS_OK : sequence_fail(HTGS_ERR_CUDA, cudaGetErrorString(err));
    }
    if (!grad_y || !x || !weight || !rstd || !grad_x) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_add_rms_norm_backward: null pointer");
    if (!scratch || !aligned(scratch, 16) || scratch_bytes < htgs_add_rms_norm_backward_scratch_bytes(rows, width))
        return sequence_fail(HTGS_ERR_WORKSPACE_TOO_SMALL, "htgs_add_rms_norm_backward: scratch too small or not 16-byte aligned");
    const NormBackwardArgs a{grad_y, grad_sum, x, residual, weight, rstd, grad_y_stride, grad_sum_stride, x_stride, residual_stride, grad_x_stride, grad_x,
                             static_cast<float*>(scratch), rows, width};
    if (type == HTGS_FLOAT32) backward_typed<float>(a, grad_weight, s);
    else if (type == HTGS_FLOAT16) backward_typed<__half>(a, grad_weight, s);
    else backward_typed<__nv_bfloat16>(a, grad_weight, s);
    return sequence_status("htgs_add_rms_norm_backward");
}

}  // extern "C"
