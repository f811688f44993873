// Root-mean-square norm of a residual stream, with the residual's addition, forward and backward, and with an 8-bit output.
//
//   u = x + residual;   rho = 1 / sqrt(mean(u^2) + eps);   y = u * rho * weight;   sum = u in the stream's type
//   backward, with unit = u * rho and z = weight * grad_y:
//       grad_x = grad_residual = rho * (z - unit * mean(z * unit)) + grad_sum;      grad_weight = sum over rows of grad_y * unit
//
// A row stays in registers between its statistics and its output, so every value crosses HBM once: read x and residual, write sum
// and y (or 8-bit codes and a scale byte for each 128 columns); backward read grad_y, grad_sum, x and residual, write one gradient that
// serves x and residual alike.  Forward, a warp holds a row of up to 1024 columns (32 values a lane), eight warps a wider one.  Bound by HBM:
// 65537 x 1024 in bf16 87 us forward (6.2 TB/s) and 114 us backward (5.9 TB/s), 100000 x 512 with 8-bit output 65 us (5.6 TB/s).  Rows that do not begin on 16 bytes
// come near that through shared memory: 100000 x 511 in bf16 82 us forward (5.0 TB/s) and 118 backward, 100003 x 333 in fp32 101 (5.3) and 135 (4.9).
// Sums are 32-bit and u is never rounded where it is computed with: the backward pass adds x and residual again rather than read the stream, whose
// rounding to 16 bits would show in grad_weight (relative error 0.0028 instead of 0.0018 at 65537 x 1024 in bf16) for 2 bytes less of 16 a value.
#include "sequence.cuh"

#include <type_traits>

namespace htgs {

namespace {

constexpr int kNormBlock = 256;
constexpr int kNormWarps = kNormBlock / 32;
constexpr int kBackwardColumns = 8;                // a thread
constexpr int kNarrowBlock = 128, kNarrowBlocks = 4, kWideBlock = 1024;
constexpr int kSharedBytes = 227 * 1024;           // of an SM; a block takes 1 KB of them besides its own
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

// Rows that begin anywhere, of any width: they come and go through shared memory, the next STAGES - 1 on their way while a warp deals with one; a lane has every 32nd
// column.  Persistent, with the weights as 32-bit values in shared memory.  More than LEAST * 32 columns a row, at most E * 32 a warp.
template <typename T, int E, int WPR> struct Anywhere {
    static constexpr int warps = WPR > 1 ? 8 : 4, together = warps / WPR;         // rows of a block
    static constexpr int stages = WPR == 1 && E * sizeof(T) <= 32 ? 4 : 2;
    static constexpr int blocks = WPR > 1 ? E > 16 ? 2 : 3 : E <= 16 ? 7 : E <= 32 ? 5 : 3;               // on an SM, as registers go
    static int slot(int width) { return (int(sizeof(T)) * (WPR == 1 ? width : 32 * E) + 31) / 16 * 16; }    // bytes
    static int memory(int width) { return (width * 4 + 15) / 16 * 16 + warps * stages * 2 * slot(width); }
};
template <typename T, int E, int LEAST, int WPR, bool FP8>
__global__ void __launch_bounds__(Anywhere<T, E, WPR>::warps * 32, Anywhere<T, E, WPR>::blocks) norm_anywhere_kernel(const NormArgs a, int slot) {
    using Shape = Anywhere<T, E, WPR>;
    extern __shared__ __align__(16) unsigned char memory[];
    __shared__ float shared[kNormWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, base = WPR == 1 ? 0 : warp * 32 * E, count = min(32 * E, a.width - base);
    float* weight = reinterpret_cast<float*>(memory);
    for (int i = threadIdx.x; i < a.width; i += Shape::warps * 32) weight[i] = to_float<T>(static_cast<const T*>(a.weight)[i]);
    weight += base;
    unsigned char* ring = memory + (a.width * 4 + 15) / 16 * 16 + warp * Shape::stages * 2 * slot;
    const int64_t step = int64_t(gridDim.x) * Shape::together;
    int64_t row = int64_t(blockIdx.x) * Shape::together + (WPR == 1 ? warp : 0), coming = row;
    const T* x = static_cast<const T*>(a.x) + base;
    const T* residual = a.residual ? static_cast<const T*>(a.residual) + base : nullptr;
    int to = 0, from = 0;
    const auto next = [&]() {
        if (coming < a.rows) {
            bring<32 * E>(ring + (2 * to) * slot, x + coming * a.x_stride, count, lane);
            if (residual) bring<32 * E>(ring + (2 * to + 1) * slot, residual + coming * a.residual_stride, count, lane);
        }
        copies_begun();
        coming += step;
        to = to + 1 == Shape::stages ? 0 : to + 1;
    };
    #pragma unroll
    for (int i = 0; i < Shape::stages - 1; ++i) next();
    __syncthreads();                    // the weights
    for (; row < a.rows; row += step) {
        next();
        copies_done<Shape::stages - 1>();
        unsigned char *first = ring + (2 * from) * slot, *second = first + slot;
        from = from + 1 == Shape::stages ? 0 : from + 1;
        const T* xs = in_slot(first, x + row * a.x_stride) + lane;
        float u[E], squares = 0.0f;
        #pragma unroll
        for (int j = 0; j < E; ++j) u[j] = j < LEAST || lane + 32 * j < count ? to_float<T>(xs[32 * j]) : 0.0f;
        if (residual) {
            const T* rs = in_slot(second, residual + row * a.residual_stride) + lane;
            #pragma unroll
            for (int j = 0; j < E; ++j)
                if (j < LEAST || lane + 32 * j < count) u[j] += to_float<T>(rs[32 * j]);
        }
        #pragma unroll
        for (int j = 0; j < E; ++j) squares = fmaf(u[j], u[j], squares);
        const float rho = rsqrtf(row_sum<WPR>(squares, shared) / float(a.width) + a.eps);
        if (a.rstd && threadIdx.x % (32 * WPR) == 0) a.rstd[row] = rho;
        __syncwarp();                   // the slots have been read
        T* sum = a.sum ? static_cast<T*>(a.sum) + row * a.sum_stride + base : nullptr;
        T* y = FP8 ? nullptr : static_cast<T*>(a.y) + row * a.y_stride + base;
        T *sums = in_slot(first, sum) + lane, *ys = in_slot(second, y) + lane;
        #pragma unroll
        for (int j = 0; j < E; ++j) {
            if (!(j < LEAST || lane + 32 * j < count)) continue;
            if (sum) sums[32 * j] = from_float<T>(u[j]);
            u[j] = u[j] * rho * weight[lane + 32 * j];
            if (!FP8) ys[32 * j] = from_float<T>(u[j]);
        }
        __syncwarp();
        if (sum) send<32 * E>(first, sum, count, lane);
        if (!FP8) send<32 * E>(second, y, count, lane);
        if (FP8) {
            uint8_t* codes = a.codes + row * a.codes_stride + base + lane;
            uint8_t* scales = a.scales + row * a.scales_stride + base / kScaleBlock;
            #pragma unroll
            for (int j = 0; j < E; j += 4) {
                if (32 * j >= count) break;
                const float v[4] = {u[j], u[j + 1], u[j + 2], u[j + 3]};
                float largest = largest_magnitude(v);
                const bool careful = __any_sync(0xffffffffu, largest > FLT_MAX);
                if (careful) largest = largest_finite(v);
                const int e = scale_exponent(lanes_max<32>(largest));
                const float inverse = inverse_scale(e);
                const uint32_t four = careful ? encode4<true>(v[0], v[1], v[2], v[3], inverse) : encode4<false>(v[0], v[1], v[2], v[3], inverse);
                #pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (j + i < LEAST || lane + 32 * (j + i) < count) codes[32 * (j + i)] = uint8_t(four >> (8 * i));
                if (lane == 0) scales[j / 4] = uint8_t(e + 127);
            }
        }
        __syncwarp();                   // what was in the slots is on its way
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

// The same for rows that begin anywhere, through shared memory as in norm_anywhere_kernel: a row at a time, the next ones on their way; a lane has every 32nd of its warp's 32 * C
// columns, and all of the first LEAST.  More than 2048 columns take more than 128 threads, whose shared memory holds one row of each tensor.
template <typename T, int C, bool WIDE> struct AnywhereBackward {
    static constexpr int most = WIDE ? 512 : 128, blocks = WIDE ? 1 : C <= 8 ? 6 : C <= 12 ? 5 : 4;
    static constexpr int stages = WIDE ? 1 : sizeof(T) == 4 && C > 8 ? 2 : 3, slot = 32 * C * int(sizeof(T)) + 16, per_warp = stages * 4 * slot;      // bytes: grad_y, x, residual, grad_sum
    static int threads(int width) { return (width + 32 * C - 1) / (32 * C) * 32; }
    static int grid(int64_t rows, int width) {                // as many as an SM's registers and shared memory hold
        const int n = threads(width), by_registers = most * blocks / n, by_memory = kSharedBytes / (n / 32 * per_warp + 1024);
        const int64_t most_blocks = 148 * (by_registers < by_memory ? by_registers : by_memory);
        return int(rows < most_blocks ? rows : most_blocks);
    }
};
template <typename T, int C, int LEAST, bool WIDE>
__global__ void __launch_bounds__(AnywhereBackward<T, C, WIDE>::most, AnywhereBackward<T, C, WIDE>::blocks) norm_backward_anywhere_kernel(const NormBackwardArgs a) {
    using Shape = AnywhereBackward<T, C, WIDE>;
    constexpr int kSlot = Shape::slot, kStages = Shape::stages;
    extern __shared__ __align__(16) unsigned char memory[];
    __shared__ float shared[2][16];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, base = warp * 32 * C, count = min(32 * C, a.width - base);
    unsigned char* ring = memory + warp * Shape::per_warp;
    const T *grad_y = static_cast<const T*>(a.grad_y) + base, *x = static_cast<const T*>(a.x) + base;
    const T* residual = a.residual ? static_cast<const T*>(a.residual) + base : nullptr;
    const T* grad_sum = a.grad_sum ? static_cast<const T*>(a.grad_sum) + base : nullptr;
    float w[C], grad_weight[C] = {};
    #pragma unroll
    for (int j = 0; j < C; ++j) w[j] = lane + 32 * j < count ? to_float<T>(static_cast<const T*>(a.weight)[base + lane + 32 * j]) : 0.0f;
    const float per_width = 1.0f / float(a.width);
    int to = 0, from = 0, buffer = 0;
    const auto next = [&](int64_t row) {
        if (row < a.rows) {
            unsigned char* slots = ring + to * 4 * kSlot;
            bring<32 * C>(slots, grad_y + row * a.grad_y_stride, count, lane);
            bring<32 * C>(slots + kSlot, x + row * a.x_stride, count, lane);
            if (residual) bring<32 * C>(slots + 2 * kSlot, residual + row * a.residual_stride, count, lane);
            if (grad_sum) bring<32 * C>(slots + 3 * kSlot, grad_sum + row * a.grad_sum_stride, count, lane);
        }
        copies_begun();
        to = to + 1 == kStages ? 0 : to + 1;
    };
    #pragma unroll
    for (int i = 0; i < kStages - 1; ++i) next(int64_t(blockIdx.x) + int64_t(i) * gridDim.x);
    const auto go = [&](auto whole) {               // whole: every lane has all its columns
        for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, buffer ^= 1) {
            const float rho = a.rstd[row];
            next(row + int64_t(kStages - 1) * gridDim.x);
            copies_done<kStages - 1>();
            unsigned char* slots = ring + from * 4 * kSlot;
            from = from + 1 == kStages ? 0 : from + 1;
            const T *gs = in_slot(slots, grad_y + row * a.grad_y_stride) + lane, *xs = in_slot(slots + kSlot, x + row * a.x_stride) + lane;
            float gy[C], u[C];
            #pragma unroll
            for (int j = 0; j < C; ++j) {
                gy[j] = whole || j < LEAST || lane + 32 * j < count ? to_float<T>(gs[32 * j]) : 0.0f;
                u[j] = whole || j < LEAST || lane + 32 * j < count ? to_float<T>(xs[32 * j]) : 0.0f;
            }
            if (residual) {
                const T* rs = in_slot(slots + 2 * kSlot, residual + row * a.residual_stride) + lane;
                #pragma unroll
                for (int j = 0; j < C; ++j)
                    if (whole || j < LEAST || lane + 32 * j < count) u[j] += to_float<T>(rs[32 * j]);
            }
            float mean = 0.0f;
            #pragma unroll
            for (int j = 0; j < C; ++j) {
                const float term = gy[j] * (u[j] * rho);
                grad_weight[j] += term;
                mean = fmaf(term, w[j], mean);
            }
            mean = warp_sum(mean);
            if (warps > 1) {
                if (lane == 0) shared[buffer][warp] = mean;
                asm volatile("barrier.cta.sync 0;" ::: "memory");          // one per row: the other buffer is read before the next one
                mean = 0.0f;
                for (int v = 0; v < warps; ++v) mean += shared[buffer][v];
            }
            __syncwarp();                           // grad_y's slot, which takes the output, has been read
            T* grad_x = static_cast<T*>(a.grad_x) + row * a.grad_x_stride + base;
            T* outs = in_slot(slots, grad_x) + lane;
            const float slope = mean * per_width * rho;
            #pragma unroll
            for (int j = 0; j < C; ++j) gy[j] = rho * (gy[j] * w[j] - u[j] * slope);
            if (grad_sum) {
                const T* ds = in_slot(slots + 3 * kSlot, grad_sum + row * a.grad_sum_stride) + lane;
                #pragma unroll
                for (int j = 0; j < C; ++j)
                    if (whole || j < LEAST || lane + 32 * j < count) gy[j] += to_float<T>(ds[32 * j]);
            }
            #pragma unroll
            for (int j = 0; j < C; ++j)
                if (whole || j < LEAST || lane + 32 * j < count) outs[32 * j] = from_float<T>(gy[j]);
            __syncwarp();
            send<32 * C>(slots, grad_x, count, lane);
            __syncwarp();                           // what was in the slots is on its way
        }
    };
    if (count >= 32 * C) go(std::true_type());
    else go(std::false_type());
    float* partial = a.partial + int64_t(blockIdx.x) * a.width + base + lane;
    #pragma unroll
    for (int j = 0; j < C; ++j)
        if (lane + 32 * j < count) partial[32 * j] = grad_weight[j];
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

template <typename T, int VEC, int E, int WPR> cudaError_t launch_norm(const NormArgs& a, cudaStream_t stream) {
    const unsigned int blocks = unsigned((a.rows + kNormWarps / WPR - 1) / (kNormWarps / WPR));
    if (a.codes) norm_kernel<T, VEC, E, WPR, true><<<blocks, kNormBlock, 0, stream>>>(a);
    else norm_kernel<T, VEC, E, WPR, false><<<blocks, kNormBlock, 0, stream>>>(a);
    return cudaSuccess;                 // the caller asks for the last error
}
// The fewest values a lane that hold a row: one warp up to 1024 columns, then eight.
template <typename T> cudaError_t norm_aligned(const NormArgs& a, cudaStream_t stream) {
    constexpr int V = 16 / int(sizeof(T));
    if (a.width <= 32 * 8) return launch_norm<T, V, 8, 1>(a, stream);
    if (a.width <= 32 * 16) return launch_norm<T, V, 16, 1>(a, stream);
    if (a.width <= 32 * 32) return launch_norm<T, V, 32, 1>(a, stream);
    if (a.width <= 256 * 8) return launch_norm<T, V, 8, 8>(a, stream);
    if (a.width <= 256 * 16) return launch_norm<T, V, 16, 8>(a, stream);
    return launch_norm<T, V, 32, 8>(a, stream);
}
template <typename T, int E, int LEAST, int WPR, bool FP8> cudaError_t launch_anywhere_as(const NormArgs& a, cudaStream_t stream) {
    using Shape = Anywhere<T, E, WPR>;
    const auto kernel = norm_anywhere_kernel<T, E, LEAST, WPR, FP8>;
    static PerDeviceOnce once;
    const cudaError_t err = once.run([kernel] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::memory((WPR == 1 ? 1 : 8) * 32 * E)); });
    if (err != cudaSuccess) return err;
    const int memory = Shape::memory(a.width), fit = kSharedBytes / (memory + 1024);
    const int64_t blocks = (a.rows + Shape::together - 1) / Shape::together, most = 148 * (fit < Shape::blocks ? fit : Shape::blocks);
    kernel<<<unsigned(blocks < most ? blocks : most), Shape::warps * 32, memory, stream>>>(a, Shape::slot(a.width));
    return cudaSuccess;
}
template <typename T, int E, int LEAST, int WPR> cudaError_t launch_anywhere(const NormArgs& a, cudaStream_t stream) {
    return a.codes ? launch_anywhere_as<T, E, LEAST, WPR, true>(a, stream) : launch_anywhere_as<T, E, LEAST, WPR, false>(a, stream);
}
template <typename T> cudaError_t norm_anywhere(const NormArgs& a, cudaStream_t stream) {         // more than 256 columns
    if (a.width <= 32 * 12) return launch_anywhere<T, 12, 8, 1>(a, stream);
    if (a.width <= 32 * 16) return launch_anywhere<T, 16, 12, 1>(a, stream);
    if (a.width <= 32 * 24) return launch_anywhere<T, 24, 16, 1>(a, stream);
    if (a.width <= 32 * 32) return launch_anywhere<T, 32, 24, 1>(a, stream);
    if constexpr (sizeof(T) == 2) {
        if (a.width <= 32 * 48) return launch_anywhere<T, 48, 32, 1>(a, stream);
        if (a.width <= 32 * 64) return launch_anywhere<T, 64, 48, 1>(a, stream);
    }
    if (a.width <= 256 * 16) return launch_anywhere<T, 16, 0, 8>(a, stream);
    return launch_anywhere<T, 32, 0, 8>(a, stream);
}

// Groups of 16 bytes where every row of every tensor begins and ends on them.  Else rows that are at most eight groups of 4 bytes or of single values a lane go directly (of one warp;
// of 32-bit values, whose slots would leave room for few warps, eight too), and others through shared memory.  (In us, direct and through shared memory:
// 200000 x 201 bf16 74 and 109, 80000 x 498 fp16 58 and 66, 100000 x 301 fp32 99 and 91, 60000 x 651 bf16 186 and 61, 30000 x 1111 fp16 79 and 64, fp32 89 and 100, 10000 x 4001 fp32 137 and 111.)
template <typename T> cudaError_t norm_typed(const NormArgs& a, cudaStream_t stream) {
    const auto allow = [&](int values) {
        const size_t e = sizeof(T), bytes = values * e;
        return a.width % values == 0 && rows_aligned(a.x, a.x_stride, a.rows, e, bytes) && rows_aligned(a.residual, a.residual_stride, a.rows, e, bytes) &&
               aligned(a.weight, bytes) && rows_aligned(a.y, a.y_stride, a.rows, e, bytes) && rows_aligned(a.sum, a.sum_stride, a.rows, e, bytes) &&
               rows_aligned(a.codes, a.codes_stride, a.rows, 1, values);
    };
    if (allow(16 / int(sizeof(T)))) return norm_aligned<T>(a, stream);
    if constexpr (sizeof(T) == 2) {
        if (a.width <= 32 * 8 && allow(2)) return launch_norm<T, 2, 8, 1>(a, stream);
        if (a.width <= 32 * 16 && allow(2)) return launch_norm<T, 2, 16, 1>(a, stream);
    }
    if (a.width <= 32 * 8) return launch_norm<T, 1, 8, 1>(a, stream);
    if constexpr (sizeof(T) == 4) {
        if (a.width > 32 * 32 && a.width <= 256 * 8) return launch_norm<T, 1, 8, 8>(a, stream);
    }
    return norm_anywhere<T>(a, stream);
}
template <typename T, int C, int LEAST, bool WIDE> cudaError_t launch_backward_anywhere(const NormBackwardArgs& a, int& blocks, cudaStream_t stream) {
    using Shape = AnywhereBackward<T, C, WIDE>;
    const auto kernel = norm_backward_anywhere_kernel<T, C, LEAST, WIDE>;
    static PerDeviceOnce once;
    const cudaError_t err = once.run([kernel] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::most / 32 * Shape::per_warp); });
    if (err != cudaSuccess) return err;
    const int threads = Shape::threads(a.width);
    blocks = Shape::grid(a.rows, a.width);
    kernel<<<blocks, threads, threads / 32 * Shape::per_warp, stream>>>(a);
    return cudaSuccess;
}
// The fewest warps that hold a row, and the fewest columns a lane that do with those; more than 128 columns.
template <typename F> auto with_backward_shape(int width, F f) {
    if (width <= 32 * 8) return f(std::integral_constant<int, 8>(), std::integral_constant<int, 4>(), std::false_type());
    if (width <= 32 * 12) return f(std::integral_constant<int, 12>(), std::integral_constant<int, 8>(), std::false_type());
    if (width <= 32 * 16) return f(std::integral_constant<int, 16>(), std::integral_constant<int, 12>(), std::false_type());
    if (width <= 2 * 32 * 12 || (width > 2 * 32 * 16 && width <= 3 * 32 * 12)) return f(std::integral_constant<int, 12>(), std::integral_constant<int, 0>(), std::false_type());
    if (width <= 4 * 32 * 16) return f(std::integral_constant<int, 16>(), std::integral_constant<int, 0>(), std::false_type());
    return f(std::integral_constant<int, 16>(), std::integral_constant<int, 0>(), std::true_type());
}
// The entry point for the workspace does not know the rows' addresses or type.
int most_backward_blocks(int64_t rows, int width) {
    const int aligned = backward_blocks(rows, width), anywhere = with_backward_shape(width, [&](auto c, auto, auto wide) {
        const int a = AnywhereBackward<__half, c.value, wide.value>::grid(rows, width), b = AnywhereBackward<float, c.value, wide.value>::grid(rows, width);
        return a > b ? a : b;
    });
    return aligned > anywhere ? aligned : anywhere;
}
// Groups of 16 bytes, or of 4 in blocks that have registers for several rows of them, where every row of every tensor begins and ends on them; else rows of up to 128 columns
// in single values and longer ones through shared memory.  (In us, direct and through shared memory: 80000 x 498 fp16 84 and 93, 60000 x 650 fp16 92 and 131,
// 200000 x 33 fp32 86 and 106, x 201 bf16 123 and 114, 50000 x 901 fp16 135 and 114.)
template <typename T> cudaError_t backward_typed(const NormBackwardArgs& a, void* grad_weight, cudaStream_t stream) {
    const auto allow = [&](int values) {
        const size_t e = sizeof(T), bytes = values * e;
        return a.width % values == 0 && rows_aligned(a.grad_y, a.grad_y_stride, a.rows, e, bytes) && rows_aligned(a.grad_sum, a.grad_sum_stride, a.rows, e, bytes) &&
               rows_aligned(a.x, a.x_stride, a.rows, e, bytes) && rows_aligned(a.residual, a.residual_stride, a.rows, e, bytes) && aligned(a.weight, bytes) &&
               rows_aligned(a.grad_x, a.grad_x_stride, a.rows, e, bytes);
    };
    constexpr int V = 16 / int(sizeof(T)), kPair = sizeof(T) == 2 ? 2 : 1;
    const int threads = backward_threads(a.width);
    const bool narrow = threads <= kNarrowBlock;
    int blocks = backward_blocks(a.rows, a.width);
    cudaError_t err = cudaSuccess;
    if (allow(V) && narrow) norm_backward_kernel<T, V, kNarrowBlock><<<blocks, threads, 0, stream>>>(a);
    else if (allow(V)) norm_backward_kernel<T, V, kWideBlock><<<blocks, threads, 0, stream>>>(a);
    else if (kPair == 2 && narrow && allow(2)) norm_backward_kernel<T, kPair, kNarrowBlock><<<blocks, threads, 0, stream>>>(a);
    else if (a.width <= 128) norm_backward_kernel<T, 1, kNarrowBlock><<<blocks, threads, 0, stream>>>(a);
    else err = with_backward_shape(a.width, [&](auto c, auto least, auto wide) { return launch_backward_anywhere<T, c.value, least.value, wide.value>(a, blocks, stream); });
    if (err != cudaSuccess) return err;
    return launch_after(norm_weight_kernel<T>, (a.width + 31) / 32, 1024, 0, stream, static_cast<const float*>(a.partial), blocks, int(a.width), static_cast<T*>(grad_weight));
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
    const cudaError_t err = type == HTGS_FLOAT32 ? norm_typed<float>(a, s) : type == HTGS_FLOAT16 ? norm_typed<__half>(a, s) : norm_typed<__nv_bfloat16>(a, s);
    return err == cudaSuccess ? sequence_status("htgs_add_rms_norm") : sequence_fail(HTGS_ERR_CUDA, cudaGetErrorString(err));
}

size_t htgs_add_rms_norm_backward_scratch_bytes(int64_t rows, int32_t width) {
    if (rows <= 0 || width <= 0) return 0;
    return size_t(htgs::most_backward_blocks(rows, width)) * size_t(width) * sizeof(float);
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
    const cudaError_t err = type == HTGS_FLOAT32   ? backward_typed<float>(a, grad_weight, s)
                            : type == HTGS_FLOAT16 ? backward_typed<__half>(a, grad_weight, s)
                                                   : backward_typed<__nv_bfloat16>(a, grad_weight, s);
    return err == cudaSuccess ? sequence_status("htgs_add_rms_norm_backward") : sequence_fail(HTGS_ERR_CUDA, cudaGetErrorString(err));
}

}  // extern "C"
