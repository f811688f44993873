// The 8-bit format of the matrix product: codes of type E4M3 with one power-of-two scale for each block of 128 columns, of one row
// (activations, gradients) or of 128 rows (weights).  For a block with largest finite magnitude m the scale is 2^e with the least e that has
// m <= 448 * 2^e, and a code is v * 2^-e rounded to nearest, ties to even.  Infinities and NaN become NaN codes and leave the scale alone.
//
// `quantize_rows_kernel` codes a matrix as it lies; `quantize_tiles_kernel` codes it, its transpose or both from one
// read: the two gradients of a product sum over other axes than the product, and their operands' blocks run along those.
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

// A warp takes 32 * VEC columns, VEC side by side in a lane, but 128 at least (VEC 1, 2: in a lane several, 32 * VEC apart), of several rows, four at a
// time, so that enough loads are on their way.
template <typename T, int VEC>
__global__ void __launch_bounds__(kQuantBlock, 6) quantize_rows_kernel(const QuantArgs a) {
    const int lane = threadIdx.x & 31;
    constexpr int kColumns = VEC < 4 ? kScaleBlock : 32 * VEC, kValues = kColumns / 32, kLanes = VEC == 8 ? 16 : 32, R = 4;
    const uint32_t across = uint32_t((a.width + kColumns - 1) / kColumns), warp = blockIdx.x * (kQuantBlock / 32) + (threadIdx.x >> 5);
    const uint32_t down = gridDim.x * (kQuantBlock / 32) / across;        // rows that are begun side by side
    if (warp >= across * down) return;
    const int64_t first = int64_t(warp % across) * kColumns, at = first + (lane / kLanes) * kScaleBlock;
    for (int64_t row0 = warp / across; row0 < a.rows; row0 += int64_t(down) * R) {
        Pack<T, VEC> raw[R][kValues / VEC];          // as they are in memory: half the registers of 32-bit values
        #pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t row = row0 + int64_t(down) * r;
            const T* x = static_cast<const T*>(a.x) + row * a.x_stride + first + lane * VEC;
            #pragma unroll
            for (int i = 0; i < kValues / VEC; ++i) {
                if (row < a.rows && first + (32 * i + lane) * VEC < a.width) raw[r][i] = *reinterpret_cast<const Pack<T, VEC>*>(x + 32 * VEC * i);
                else {
                    #pragma unroll
                    for (int k = 0; k < VEC; ++k) raw[r][i].v[k] = from_float<T>(0.0f);
                }
            }
        }
        #pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t row = row0 + int64_t(down) * r;
            if (row >= a.rows) break;
            uint8_t* codes = a.codes + row * a.codes_stride;
            float v[kValues];
            #pragma unroll
            for (int i = 0; i < kValues / VEC; ++i) {
                float f[VEC];
                to_floats<T, VEC>(raw[r][i], f);
                #pragma unroll
                for (int k = 0; k < VEC; ++k) v[i * VEC + k] = f[k];
            }
            float largest = largest_magnitude(v);
            const bool careful = __any_sync(0xffffffffu, largest > FLT_MAX);
            if (careful) largest = largest_finite(v);
            const int e = scale_exponent(lanes_max<kLanes>(largest));
            const float inverse = inverse_scale(e);
            #pragma unroll
            for (int i = 0; i < kValues / VEC; ++i) {
                const int64_t column = first + (32 * i + lane) * VEC;
                if (column >= a.width) continue;
                float f[VEC];
                #pragma unroll
                for (int k = 0; k < VEC; ++k) f[k] = v[i * VEC + k];
                if (careful) store_codes<true>(codes + column, f, inverse);
                else store_codes<false>(codes + column, f, inverse);
            }
            if (lane % kLanes == 0 && at < a.width) a.scales[row * a.scales_stride + at / kScaleBlock] = uint8_t(e + 127);
        }
    }
}

// One block per 128 x 128 values, which lie in shared memory as they came: 16 bytes at a time without passing through registers where the rows allow it (WIDE).
// A thread deals with eight rows by eight columns: half a warp has the 128 columns of its eight rows, so a row's largest value is found by
// shuffles, a column's through shared memory.  Transposed codes go through shared memory too, in the tile's place, so that they leave as rows of 128: the
// eight bytes of half-warp h and column c lie in slot h ^ (c / 8 % 16) of the column's sixteen, which spreads the 16 lanes of a store over all
// banks.  PER_TILE: one scale for the whole tile.
// (With the tile in registers, 98 a thread, two blocks were on an SM: 32768 x 1024 with its transpose in 26.6 us.)
template <typename T, bool WIDE, bool PER_TILE>
__global__ void __launch_bounds__(kQuantBlock, 4) quantize_tiles_kernel(const QuantArgs a) {
    constexpr int VEC = 16 / int(sizeof(T)), G = 8 / VEC;                 // values in 16 bytes, and of those in a thread's eight columns
    extern __shared__ __align__(16) unsigned char raw[];
    T (*tile)[kScaleBlock] = reinterpret_cast<T (*)[kScaleBlock]>(raw);
    uint2 (*turned)[16] = reinterpret_cast<uint2 (*)[16]>(raw);
    __shared__ float column_largest[16][kScaleBlock];
    __shared__ float column_all[kScaleBlock];
    const int l = threadIdx.x & 15, h = threadIdx.x >> 4;
    const int64_t row0 = int64_t(blockIdx.y) * kScaleBlock, column0 = int64_t(blockIdx.x) * kScaleBlock;
    const int rows = int(min(int64_t(kScaleBlock), a.rows - row0)), columns = int(min(int64_t(kScaleBlock), a.width - column0));
    const T* x = static_cast<const T*>(a.x) + row0 * a.x_stride + column0;
    if (WIDE) {
        constexpr int kPieces = kScaleBlock / VEC;                       // of a row
        #pragma unroll
        for (int i = 0; i < kScaleBlock * kPieces / kQuantBlock; ++i) {
            const int at = i * kQuantBlock + int(threadIdx.x), r = at / kPieces, c = at % kPieces * VEC;
            const bool there = r < rows && c < columns;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(&tile[r][c])), "l"(there ? x + r * a.x_stride + c : x), "r"(there ? 16 : 0) : "memory");
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (a.x_stride * sizeof(T) % 4 == 0 && reinterpret_cast<uintptr_t>(a.x) % 4 == 0 && (sizeof(T) == 4 || columns % 2 == 0)) {
        constexpr int kTogether = 4 / int(sizeof(T)), kPieces = kScaleBlock / kTogether;
        #pragma unroll 8
        for (int i = 0; i < kScaleBlock * kPieces / kQuantBlock; ++i) {
            const int at = i * kQuantBlock + int(threadIdx.x), r = at / kPieces, c = at % kPieces * kTogether;
            const bool there = r < rows && c < columns;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(&tile[r][c])), "l"(there ? x + r * a.x_stride + c : x), "r"(there ? 4 : 0) : "memory");
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else {
        #pragma unroll 8
        for (int i = 0; i < kScaleBlock * kScaleBlock / kQuantBlock; ++i) {
            const int at = i * kQuantBlock + int(threadIdx.x), r = at / kScaleBlock, c = at % kScaleBlock;
            tile[r][c] = r < rows && c < columns ? x[r * a.x_stride + c] : from_float<T>(0.0f);
        }
    }
    __syncthreads();
    const auto column = [&](int c) { return c / VEC * 16 * VEC + l * VEC + c % VEC; };      // of the thread's c-th value in the tile
    const auto values = [&](int r, float (&v)[8]) {
        #pragma unroll
        for (int j = 0; j < G; ++j) {
            float f[VEC];
            load_floats<T, VEC>(&tile[h * 8 + r][(j * 16 + l) * VEC], f);
            #pragma unroll
            for (int i = 0; i < VEC; ++i) v[j * VEC + i] = f[i];
        }
    };
    float most[8] = {};                      // of the thread's columns
    #pragma unroll
    for (int r = 0; r < 8; ++r) {
        float v[8];
        values(r, v);
        #pragma unroll
        for (int c = 0; c < 8; ++c) most[c] = fmaxf(most[c], fabsf(v[c]));
    }
    const bool careful = __syncthreads_or(largest_magnitude(most) > FLT_MAX) != 0;      // an infinity in the tile
    if (careful) {
        #pragma unroll
        for (int c = 0; c < 8; ++c) most[c] = 0.0f;
        #pragma unroll 1
        for (int r = 0; r < 8; ++r) {
            float v[8];
            values(r, v);
            #pragma unroll
            for (int c = 0; c < 8; ++c) most[c] = fmaxf(most[c], finite_magnitude(v[c]));
        }
    }
    #pragma unroll
    for (int c = 0; c < 8; ++c) column_largest[h][column(c)] = most[c];
    __syncthreads();
    if (threadIdx.x < kScaleBlock) {
        float largest = 0.0f;
        #pragma unroll
        for (int i = 0; i < 16; ++i) largest = fmaxf(largest, column_largest[i][threadIdx.x]);
        if (PER_TILE) largest = lanes_max<32>(largest);
        column_all[threadIdx.x] = largest;
        if (!PER_TILE && a.codes_t && int(threadIdx.x) < columns) a.scales_t[(column0 + threadIdx.x) * a.scales_t_stride + blockIdx.y] = uint8_t(scale_exponent(largest) + 127);
    }
    __syncthreads();
    int tile_e = 0;
    if (PER_TILE) {
        tile_e = scale_exponent(fmaxf(fmaxf(column_all[0], column_all[32]), fmaxf(column_all[64], column_all[96])));
        if (threadIdx.x == 0 && a.codes) a.scales[int64_t(blockIdx.y) * a.scales_stride + blockIdx.x] = uint8_t(tile_e + 127);
        if (threadIdx.x == 0 && a.codes_t) a.scales_t[int64_t(blockIdx.x) * a.scales_t_stride + blockIdx.y] = uint8_t(tile_e + 127);
    }
    if (a.codes) {
        const bool together = a.width % VEC == 0 && a.codes_stride % VEC == 0 && reinterpret_cast<uintptr_t>(a.codes) % VEC == 0;
        #pragma unroll 2
        for (int r = 0; r < 8; ++r) {
            float v[8];
            values(r, v);
            const int e = PER_TILE ? tile_e : scale_exponent(lanes_max<16>(careful ? largest_finite(v) : largest_magnitude(v)));
            if (h * 8 + r >= rows) continue;
            const float inverse = inverse_scale(e);
            uint8_t* codes = a.codes + (row0 + h * 8 + r) * a.codes_stride + column0;
            #pragma unroll
            for (int j = 0; j < G; ++j) {
                float f[VEC];
                #pragma unroll
                for (int i = 0; i < VEC; ++i) f[i] = v[j * VEC + i];
                if (together) {
                    if (column(j * VEC) >= columns) continue;
                    if (careful) store_codes<true>(codes + column(j * VEC), f, inverse);
                    else store_codes<false>(codes + column(j * VEC), f, inverse);
                } else {
                    #pragma unroll
                    for (int i = 0; i < VEC; ++i)
                        if (column(j * VEC + i) < columns) codes[column(j * VEC + i)] = uint8_t(encode2<true>(f[i], 0.0f, inverse) & 0xffu);
                }
            }
            if (!PER_TILE && l == 0) a.scales[(row0 + h * 8 + r) * a.scales_stride + blockIdx.x] = uint8_t(e + 127);
        }
    }
    if (!a.codes_t) return;
    #pragma unroll
    for (int c = 0; c < 8; ++c) most[c] = inverse_scale(PER_TILE ? tile_e : scale_exponent(column_all[column(c)]));
    uint32_t words[2][8];                    // four rows' codes of each column
    #pragma unroll
    for (int q = 0; q < 2; ++q) {
        float v[4][8];
        #pragma unroll
        for (int r = 0; r < 4; ++r) values(4 * q + r, v[r]);
        #pragma unroll
        for (int c = 0; c < 8; ++c)
            words[q][c] = careful ? encode4<true>(v[0][c], v[1][c], v[2][c], v[3][c], most[c]) : encode4<false>(v[0][c], v[1][c], v[2][c], v[3][c], most[c]);
    }
    __syncthreads();                         // nothing more is read of the tile
    #pragma unroll
    for (int c = 0; c < 8; ++c) turned[column(c)][h ^ (column(c) / 8 % 16)] = make_uint2(words[0][c], words[1][c]);
    __syncthreads();
    const bool whole = rows == kScaleBlock && a.codes_t_stride % 16 == 0 && reinterpret_cast<uintptr_t>(a.codes_t) % 16 == 0;
    for (int i = threadIdx.x; i < columns * 8; i += kQuantBlock) {
        const int c = i >> 3, s = i & 7;                  // rows 16 s .. 16 s + 15 of column c
        const uint2 lo = turned[c][(2 * s) ^ (c / 8 % 16)], hi = turned[c][(2 * s + 1) ^ (c / 8 % 16)];
        uint8_t* to = a.codes_t + (column0 + c) * a.codes_t_stride + row0 + 16 * s;
        if (whole) *reinterpret_cast<uint4*>(to) = make_uint4(lo.x, lo.y, hi.x, hi.y);
        else {
            const uint32_t four[4] = {lo.x, lo.y, hi.x, hi.y};
            #pragma unroll 1
            for (int k = 0; k < 16 && 16 * s + k < rows; ++k) to[k] = uint8_t((k < 8 ? k < 4 ? four[0] : four[1] : k < 12 ? four[2] : four[3]) >> (8 * (k & 3)));
        }
    }
}

// Codes back to values: exact in every output type, except that what leaves the range of 16-bit floats becomes infinite or zero.
template <typename T, int VEC>
__global__ void __launch_bounds__(kQuantBlock, 6) dequantize_kernel(const uint8_t* codes, int64_t codes_stride, const uint8_t* scales, int64_t scales_stride,
                                                                int shift, int64_t rows, int64_t width, T* out, int64_t out_stride) {
    const int lane = threadIdx.x & 31;
    constexpr int kColumns = VEC < 4 ? kScaleBlock : 32 * VEC, G = kColumns / 32 / VEC, R = 4;       // as in quantize_rows_kernel
    const uint32_t across = uint32_t((width + kColumns - 1) / kColumns), warp = blockIdx.x * (kQuantBlock / 32) + (threadIdx.x >> 5);
    const uint32_t down = gridDim.x * (kQuantBlock / 32) / across;
    const int64_t column = int64_t(warp % across) * kColumns + lane * VEC;
    grid_dependency();
    if (warp >= across * down || column >= width) return;
    for (int64_t row0 = warp / across; row0 < rows; row0 += int64_t(down) * R) {
        Pack<uint8_t, VEC> packed[R][G];
        uint32_t exponent[R];
        #pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t row = row0 + int64_t(down) * r;
            if (row >= rows) break;
            #pragma unroll
            for (int j = 0; j < G; ++j)
                if (column + 32 * VEC * j < width) packed[r][j] = *reinterpret_cast<const Pack<uint8_t, VEC>*>(codes + row * codes_stride + column + 32 * VEC * j);
            exponent[r] = scales[(row >> shift) * scales_stride + column / kScaleBlock];
        }
        #pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t row = row0 + int64_t(down) * r;
            if (row >= rows) break;
            const float scale = scale_value(exponent[r]);
            #pragma unroll
            for (int j = 0; j < G; ++j) {
                if (column + 32 * VEC * j >= width) break;
                float v[VEC];
                if constexpr (VEC == 1) v[0] = decode2(packed[r][j].v[0]).x * scale;
                else {
                    uint32_t words[(VEC + 3) / 4];
                    if constexpr (VEC == 2) words[0] = *reinterpret_cast<const uint16_t*>(&packed[r][j]);
                    else {
                        #pragma unroll
                        for (int k = 0; k < VEC / 4; ++k) words[k] = reinterpret_cast<const uint32_t*>(&packed[r][j])[k];
                    }
                    #pragma unroll
                    for (int k = 0; k < VEC; k += 2) {
                        const float2 f = decode2(words[k / 4] >> (k % 4 * 8));
                        v[k] = f.x * scale; v[k + 1] = f.y * scale;
                    }
                }
                store_floats<T, VEC>(out + row * out_stride + column + 32 * VEC * j, v);
            }
        }
    }
}

// Blocks for warps that take `columns` columns of four rows each: as many as the SMs hold at once, and at least one row's worth.
unsigned int blocks_for(int64_t rows, int64_t width, int columns) {
    const int64_t across = (width + columns - 1) / columns, per_block = kQuantBlock / 32;
    int64_t blocks = (across * ((rows + 3) / 4) + per_block - 1) / per_block;
    if (blocks > 148 * 6) blocks = 148 * 6;
    const int64_t least = (across + per_block - 1) / per_block;
    return unsigned(blocks > least ? blocks : least);
}

template <typename T, int VEC> void launch_rows(const QuantArgs& a, cudaStream_t stream) {
    quantize_rows_kernel<T, VEC><<<blocks_for(a.rows, a.width, VEC < 4 ? kScaleBlock : 32 * VEC), kQuantBlock, 0, stream>>>(a);
}
template <typename T, bool WIDE, bool PER_TILE> cudaError_t launch_tiles(const QuantArgs& a, cudaStream_t stream) {
    const dim3 grid(unsigned((a.width + kScaleBlock - 1) / kScaleBlock), unsigned((a.rows + kScaleBlock - 1) / kScaleBlock));
    constexpr int smem = kScaleBlock * kScaleBlock * int(sizeof(T));
    static PerDeviceOnce once;
    const cudaError_t err = once.run([] { return cudaFuncSetAttribute(quantize_tiles_kernel<T, WIDE, PER_TILE>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
    if (err == cudaSuccess) quantize_tiles_kernel<T, WIDE, PER_TILE><<<grid, kQuantBlock, smem, stream>>>(a);
    return err;
}
template <typename T> int quantize_typed(const QuantArgs& a, int rows_per_scale, cudaStream_t stream) {
    constexpr int V = 16 / int(sizeof(T));
    const bool wide = a.width % V == 0 && rows_aligned(a.x, a.x_stride, a.rows, sizeof(T), 16);
    cudaError_t err = cudaSuccess;
    if (rows_per_scale != 1) err = wide ? launch_tiles<T, true, true>(a, stream) : launch_tiles<T, false, true>(a, stream);
    else if (a.codes_t) err = wide ? launch_tiles<T, true, false>(a, stream) : launch_tiles<T, false, false>(a, stream);
    else if (wide && rows_aligned(a.codes, a.codes_stride, a.rows, 1, V)) launch_rows<T, V>(a, stream);
    else if (sizeof(T) == 2 && a.width % 2 == 0 && rows_aligned(a.x, a.x_stride, a.rows, 2, 4) && rows_aligned(a.codes, a.codes_stride, a.rows, 1, 2))
        launch_rows<T, sizeof(T) == 2 ? 2 : 1>(a, stream);
    else launch_rows<T, 1>(a, stream);
    return err == cudaSuccess ? sequence_status("htgs_quantize_fp8") : sequence_fail(HTGS_ERR_CUDA, cudaGetErrorString(err));
}

template <typename T, int VEC> void launch_dequantize(const HtgsFp8Matrix& m, void* out, int64_t out_stride, cudaStream_t stream) {
    (void)launch_after(dequantize_kernel<T, VEC>, blocks_for(m.rows, m.width, VEC < 4 ? kScaleBlock : 32 * VEC), kQuantBlock, 0, stream, m.codes, m.codes_stride, m.scales, m.scales_stride,
                       m.rows_per_scale == 1 ? 0 : 7, m.rows, m.width, static_cast<T*>(out), out_stride);       // the caller asks for the last error
}
template <typename T> void dequantize_typed(const HtgsFp8Matrix& m, void* out, int64_t out_stride, cudaStream_t stream) {
    constexpr int V = 16 / int(sizeof(T));        // 16 bytes to store: with 32 a lane every store would write half sectors
    const auto allow = [&](int values) {
        return m.width % values == 0 && rows_aligned(m.codes, m.codes_stride, m.rows, 1, values) && rows_aligned(out, out_stride, m.rows, sizeof(T), values * sizeof(T));
    };
    if (allow(V)) launch_dequantize<T, V>(m, out, out_stride, stream);
    else if (allow(2)) launch_dequantize<T, 2>(m, out, out_stride, stream);
    else launch_dequantize<T, 1>(m, out, out_stride, stream);
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
    if (type == HTGS_FLOAT32) return quantize_typed<float>(a, rows_per_scale, s);
    if (type == HTGS_FLOAT16) return quantize_typed<__half>(a, rows_per_scale, s);
    return quantize_typed<__nv_bfloat16>(a, rows_per_scale, s);
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
