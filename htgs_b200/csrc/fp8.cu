// The 8-bit format of the matrix product: codes of type E4M3 with one power-of-two scale for each block of 128 columns, of one row
// (activations, gradients) or of 128 rows (weights).  For a block with largest finite magnitude m the scale is 2^e with the least e that has
// m <= 448 * 2^e, and a code is v * 2^-e rounded to nearest, ties to even.  Infinities and NaN become NaN codes and leave the scale alone.
//
// `quantize_rows_kernel` codes a matrix as it lies; `quantize_tiles_kernel` codes it, its transpose or both from one read through
// shared memory: the two gradients of a product sum over other axes than the product, and their operands' blocks run along those.
// Both are bound by HBM: 2 bytes read (16-bit input) and 1 written per value and orientation.
#include "sequence.cuh"

namespace htgs {

namespace {

constexpr int kQuantBlock = 256;

struct QuantArgs {
    const void* x;
    int64_t x_stride, rows, width;
    uint8_t* codes; uint8_t* scales; int64_t codes_stride, scales_stride;         // as it lies; may be null
    uint8_t* codes_t; uint8_t* scales_t; int64_t codes_t_stride, scales_t_stride; // transposed; may be null
};

// A warp takes 32 * VEC columns of a row at a time, VEC side by side in a lane; VEC 1: 128 columns, four of them 32 apart in a lane.
template <typename T, int VEC>
__global__ void __launch_bounds__(kQuantBlock) quantize_rows_kernel(const QuantArgs a) {
    const int lane = threadIdx.x & 31;
    constexpr int kColumns = VEC == 1 ? kScaleBlock : 32 * VEC, kValues = VEC == 1 ? 4 : VEC, kLanes = VEC == 8 ? 16 : 32;
    const int64_t units_per_row = (a.width + kColumns - 1) / kColumns, units = units_per_row * a.rows;
    const int64_t step = int64_t(gridDim.x) * (kQuantBlock / 32);
    for (int64_t unit = int64_t(blockIdx.x) * (kQuantBlock / 32) + (threadIdx.x >> 5); unit < units; unit += step) {
        const int64_t row = unit / units_per_row, first = (unit - row * units_per_row) * kColumns;
        const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
        uint8_t* codes = a.codes + row * a.codes_stride;
        float v[kValues];
        float largest = 0.0f;
        if (VEC == 1) {
            #pragma unroll
            for (int i = 0; i < kValues; ++i) v[i] = first + 32 * i + lane < a.width ? to_float<T>(x[first + 32 * i + lane]) : 0.0f;
        } else if (first + lane * VEC < a.width) {
            load_floats<T, kValues>(x + first + lane * VEC, v);
        } else {
            #pragma unroll
            for (int i = 0; i < kValues; ++i) v[i] = 0.0f;
        }
        #pragma unroll
        for (int i = 0; i < kValues; ++i) largest = fmaxf(largest, finite_magnitude(v[i]));
        const int e = scale_exponent(lanes_max<kLanes>(largest));
        const float inverse = inverse_scale(e);
        if (VEC == 1) {
            #pragma unroll
            for (int i = 0; i < kValues; ++i)
                if (first + 32 * i + lane < a.width) codes[first + 32 * i + lane] = uint8_t(encode2(v[i], 0.0f, inverse) & 0xffu);
        } else if (first + lane * VEC < a.width) {
            if (VEC == 8)
                *reinterpret_cast<uint2*>(codes + first + lane * VEC) =
                    make_uint2(encode4(v[0], v[1], v[2], v[3], inverse), encode4(v[4 % kValues], v[5 % kValues], v[6 % kValues], v[7 % kValues], inverse));
            else
                *reinterpret_cast<uint32_t*>(codes + first + lane * VEC) = encode4(v[0], v[1], v[2], v[3], inverse);
        }
        const int64_t at = first + (lane / kLanes) * kScaleBlock;
        if (lane % kLanes == 0 && at < a.width) a.scales[row * a.scales_stride + at / kScaleBlock] = uint8_t(e + 127);
    }
}

// One block per 128 x 128 values.  The tile lies in shared memory with a row pitch of an odd number of words, so that the 32 rows that a
// warp reads of one column come from 32 banks.  PER_TILE: one scale for the whole tile.
template <typename T, bool PER_TILE>
__global__ void __launch_bounds__(kQuantBlock) quantize_tiles_kernel(const QuantArgs a) {
    extern __shared__ unsigned char raw[];
    T* tile = reinterpret_cast<T*>(raw);
    constexpr int kPitch = sizeof(T) == 4 ? 129 : 130;
    __shared__ float block_largest[kQuantBlock / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row0 = int64_t(blockIdx.y) * kScaleBlock, column0 = int64_t(blockIdx.x) * kScaleBlock;
    float largest = 0.0f;
    for (int r = warp; r < kScaleBlock; r += kQuantBlock / 32) {
        const int64_t row = row0 + r;
        const T* x = static_cast<const T*>(a.x) + row * a.x_stride + column0;
        float v[4];
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = lane + 32 * i;
            const T value = row < a.rows && column0 + c < a.width ? x[c] : from_float<T>(0.0f);
            tile[r * kPitch + c] = value;
            v[i] = to_float<T>(value);
        }
        float most = fmaxf(fmaxf(finite_magnitude(v[0]), finite_magnitude(v[1])), fmaxf(finite_magnitude(v[2]), finite_magnitude(v[3])));
        if (PER_TILE) { largest = fmaxf(largest, most); continue; }
        if (!a.codes || row >= a.rows) continue;
        const int e = scale_exponent(lanes_max<32>(most));
        const float inverse = inverse_scale(e);
        uint8_t* codes = a.codes + row * a.codes_stride + column0;
        #pragma unroll
        for (int i = 0; i < 4; ++i)
            if (column0 + lane + 32 * i < a.width) codes[lane + 32 * i] = uint8_t(encode2(v[i], 0.0f, inverse) & 0xffu);
        if (lane == 0) a.scales[row * a.scales_stride + blockIdx.x] = uint8_t(e + 127);
    }
    int tile_e = 0;
    if (PER_TILE) {
        largest = lanes_max<32>(largest);
        if (lane == 0) block_largest[warp] = largest;
    }
    __syncthreads();
    if (PER_TILE) {
        #pragma unroll
        for (int w = 0; w < kQuantBlock / 32; ++w) largest = fmaxf(largest, block_largest[w]);
        tile_e = scale_exponent(largest);
        if (a.codes) {
            const float inverse = inverse_scale(tile_e);
            for (int r = warp; r < kScaleBlock && row0 + r < a.rows; r += kQuantBlock / 32) {
                uint8_t* codes = a.codes + (row0 + r) * a.codes_stride + column0;
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int c = lane + 32 * i;
                    if (column0 + c < a.width) codes[c] = uint8_t(encode2(to_float<T>(tile[r * kPitch + c]), 0.0f, inverse) & 0xffu);
                }
            }
            if (threadIdx.x == 0) a.scales[int64_t(blockIdx.y) * a.scales_stride + blockIdx.x] = uint8_t(tile_e + 127);
        }
        if (a.codes_t && threadIdx.x == 0) a.scales_t[int64_t(blockIdx.x) * a.scales_t_stride + blockIdx.y] = uint8_t(tile_e + 127);
    }
    if (!a.codes_t) return;
    for (int c = warp; c < kScaleBlock && column0 + c < a.width; c += kQuantBlock / 32) {
        float v[4];
        #pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = to_float<T>(tile[(lane + 32 * i) * kPitch + c]);
        int e = tile_e;
        if (!PER_TILE) {
            const float most = fmaxf(fmaxf(finite_magnitude(v[0]), finite_magnitude(v[1])), fmaxf(finite_magnitude(v[2]), finite_magnitude(v[3])));
            e = scale_exponent(lanes_max<32>(most));
            if (lane == 0) a.scales_t[(column0 + c) * a.scales_t_stride + blockIdx.y] = uint8_t(e + 127);
        }
        const float inverse = inverse_scale(e);
        uint8_t* codes = a.codes_t + (column0 + c) * a.codes_t_stride + row0;
        #pragma unroll
        for (int i = 0; i < 4; ++i)
            if (row0 + lane + 32 * i < a.rows) codes[lane + 32 * i] = uint8_t(encode2(v[i], 0.0f, inverse) & 0xffu);
    }
}

// Codes back to values: exact in every output type, except that what leaves the range of 16-bit floats becomes infinite or zero.
template <typename T, int VEC>
__global__ void __launch_bounds__(kQuantBlock) dequantize_kernel(const uint8_t* codes, int64_t codes_stride, const uint8_t* scales, int64_t scales_stride,
                                                                int rows_per_scale, int64_t rows, int64_t width, T* out, int64_t out_stride) {
    const int64_t per_row = (width + VEC - 1) / VEC, total = per_row * rows, step = int64_t(gridDim.x) * kQuantBlock;
    for (int64_t i = int64_t(blockIdx.x) * kQuantBlock + threadIdx.x; i < total; i += step) {
        const int64_t row = i / per_row, column = (i - row * per_row) * VEC;
        const float scale = scale_value(scales[row / rows_per_scale * scales_stride + column / kScaleBlock]);
        const uint8_t* at = codes + row * codes_stride + column;
        if (VEC == 8) {
            const uint2 packed = *reinterpret_cast<const uint2*>(at);
            const float2 a = decode2(packed.x), b = decode2(packed.x >> 16), c = decode2(packed.y), d = decode2(packed.y >> 16);
            const float v[8] = {a.x * scale, a.y * scale, b.x * scale, b.y * scale, c.x * scale, c.y * scale, d.x * scale, d.y * scale};
            if (sizeof(T) == 2) store_floats<T, 8>(out + row * out_stride + column, v);
            else {
                *reinterpret_cast<float4*>(out + row * out_stride + column) = make_float4(v[0], v[1], v[2], v[3]);
                *reinterpret_cast<float4*>(out + row * out_stride + column + 4) = make_float4(v[4], v[5], v[6], v[7]);
            }
        } else {
            out[row * out_stride + column] = from_float<T>(decode2(*at).x * scale);
        }
    }
}

unsigned int capped_blocks(int64_t work, int64_t per_block) {
    const int64_t blocks = (work + per_block - 1) / per_block;
    return unsigned(blocks < 148 * 8 ? blocks : 148 * 8);
}

template <typename T> void quantize_typed(const QuantArgs& a, int rows_per_scale, cudaStream_t stream) {
    if (rows_per_scale == 1 && !a.codes_t) {
        constexpr int V = 16 / int(sizeof(T));
        if (a.width % V == 0 && rows_aligned(a.x, a.x_stride, a.rows, sizeof(T), 16) && rows_aligned(a.codes, a.codes_stride, a.rows, 1, V))
            quantize_rows_kernel<T, V><<<capped_blocks(a.rows * ((a.width + 32 * V - 1) / (32 * V)), kQuantBlock / 32), kQuantBlock, 0, stream>>>(a);
        else
            quantize_rows_kernel<T, 1><<<capped_blocks(a.rows * ((a.width + kScaleBlock - 1) / kScaleBlock), kQuantBlock / 32), kQuantBlock, 0, stream>>>(a);
        return;
    }
    const dim3 grid(unsigned((a.width + kScaleBlock - 1) / kScaleBlock), unsigned((a.rows + kScaleBlock - 1) / kScaleBlock));
    constexpr size_t smem = size_t(kScaleBlock) * (sizeof(T) == 4 ? 129 : 130) * sizeof(T);
    if (rows_per_scale == 1) {
        static PerDeviceOnce once;
        once.run([] { return cudaFuncSetAttribute(quantize_tiles_kernel<T, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)); });
        quantize_tiles_kernel<T, false><<<grid, kQuantBlock, smem, stream>>>(a);
    } else {
        static PerDeviceOnce once;
        once.run([] { return cudaFuncSetAttribute(quantize_tiles_kernel<T, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)); });
        quantize_tiles_kernel<T, true><<<grid, kQuantBlock, smem, stream>>>(a);
    }
}

template <typename T> void dequantize_typed(const HtgsFp8Matrix& m, void* out, int64_t out_stride, cudaStream_t stream) {
    if (m.width % 8 == 0 && rows_aligned(m.codes, m.codes_stride, m.rows, 1, 8) && rows_aligned(out, out_stride, m.rows, sizeof(T), 16))
        dequantize_kernel<T, 8><<<capped_blocks(m.rows * (m.width / 8), kQuantBlock), kQuantBlock, 0, stream>>>(
            m.codes, m.codes_stride, m.scales, m.scales_stride, m.rows_per_scale, m.rows, m.width, static_cast<T*>(out), out_stride);
    else
        dequantize_kernel<T, 1><<<capped_blocks(m.rows * m.width, kQuantBlock), kQuantBlock, 0, stream>>>(
            m.codes, m.codes_stride, m.scales, m.scales_stride, m.rows_per_scale, m.rows, m.width, static_cast<T*>(out), out_stride);
}

}  // namespace

}  // namespace htgs

extern "C" {

int htgs_quantize_fp8(const void* x, int64_t x_stride, int type, int64_t rows, int64_t width, int rows_per_scale, uint8_t* codes, int64_t codes_stride,
                      uint8_t* scales, int64_t scales_stride, uint8_t* codes_t, int64_t codes_t_stride, uint8_t* scales_t, int64_t scales_t_stride,
                      void* stream) {
    using namespace htgs;
    if (!known_type(type)) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_quantize_fp8: unknown element type");
    if (rows < 0 || width < 0 || rows > 0x7fffffff || width > 0x7fffffff) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_quantize_fp8: rows and width must be in [0, 2^31)");
    if (rows_per_scale != 1 && rows_per_scale != kScaleBlock) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_quantize_fp8: rows_per_scale must be 1 or 128");
    if (rows == 0 || width == 0) return HTGS_OK;
    if (!x || (!codes && !codes_t) || (codes && !scales) || (codes_t && !scales_t)) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_quantize_fp8: null pointer");
    if ((codes_t || rows_per_scale != 1) && rows > 65535ll * kScaleBlock) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_quantize_fp8: at most 8388480 rows with tiles or a transpose");
    const QuantArgs a{x, x_stride, rows, width, codes, scales, codes_stride, scales_stride, codes_t, scales_t, codes_t_stride, scales_t_stride};
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (type == HTGS_FLOAT32) quantize_typed<float>(a, rows_per_scale, s);
    else if (type == HTGS_FLOAT16) quantize_typed<__half>(a, rows_per_scale, s);
    else quantize_typed<__nv_bfloat16>(a, rows_per_scale, s);
    return sequence_status("htgs_quantize_fp8");
}

int htgs_dequantize_fp8(const HtgsFp8Matrix* matrix, void* out, int64_t out_stride, int out_type, void* stream) {
    using namespace htgs;
    if (!matrix || !known_type(out_type)) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_dequantize_fp8: null matrix or unknown element type");
    if (matrix->rows < 0 || matrix->width < 0 || (matrix->rows_per_scale != 1 && matrix->rows_per_scale != kScaleBlock))
        return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_dequantize_fp8: bad sizes, or rows_per_scale other than 1 or 128");
    if (matrix->rows == 0 || matrix->width == 0) return HTGS_OK;
    if (!matrix->codes || !matrix->scales || !out) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_dequantize_fp8: null pointer");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (out_type == HTGS_FLOAT32) dequantize_typed<float>(*matrix, out, out_stride, s);
    else if (out_type == HTGS_FLOAT16) dequantize_typed<__half>(*matrix, out, out_stride, s);
    else dequantize_typed<__nv_bfloat16>(*matrix, out, out_stride, s);
    return sequence_status("htgs_dequantize_fp8");
}

}  // extern "C"
