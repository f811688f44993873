// The 8-bit format of the matrix product: codes of type E4M3 with one power-of-two scale for each block of 128 columns, of one row
// (activations, gradients) or of 128 rows (weights).  For a block with largest finite magnitude m the scale is 2^e with the least e that has
// m <= 448 * 2^e, and a code is v * 2^-e rounded to nearest, ties to even.  Infinities and NaN become NaN codes and leave the scale alone.
//
// `quantize_rows_kernel` codes a matrix as it lies; `quantize_tiles_kernel` codes it, its transpose or both from one
// read: the two gradients of a product sum over other axes than the product, and their operands' blocks run along those.
// Both are bound by HBM: 2 bytes read (16-bit input) and 1 written per value and orientation: 100000 x 1024 in bf16 58 us as it lies (5.3 TB/s), 62 us turned (4.9 TB/s);
// back to bf16 100000 x 512 in 34 us (4.5 TB/s).  Rows that do not begin on 16 bytes: 100000 x 511 46, 63 and 51 us, where instructions are the bound.
#include "sequence.cuh"

#include <type_traits>

namespace htgs {

namespace {

constexpr int kQuantBlock = 256;

struct QuantArgs {
    const void* x;
    int64_t x_stride, rows, width;
    uint8_t* codes; uint8_t* scales; int64_t codes_stride, scales_stride;         // as it lies; may be null
    uint8_t* codes_t; uint8_t* scales_t; int64_t codes_t_stride, scales_t_stride; // transposed; may be null
};

// Rows that begin and end on 16 bytes.  A warp takes 16 bytes a lane of several rows, four at a time, so that enough loads are on their way.
constexpr int kTogether = 4;
template <typename T>
__global__ void __launch_bounds__(kQuantBlock, 6) quantize_rows_kernel(const QuantArgs a) {
    const int lane = threadIdx.x & 31;
    constexpr int VEC = 16 / int(sizeof(T)), kColumns = 32 * VEC, kLanes = kScaleBlock / VEC, R = kTogether;
    const uint32_t across = uint32_t((a.width + kColumns - 1) / kColumns), warp = blockIdx.x * (kQuantBlock / 32) + (threadIdx.x >> 5);
    const uint32_t down = gridDim.x * (kQuantBlock / 32) / across;        // rows that are begun side by side
    if (warp >= across * down) return;
    const int64_t column = int64_t(warp % across) * kColumns + lane * VEC;
    for (int64_t row0 = warp / across; row0 < a.rows; row0 += int64_t(down) * R) {
        Pack<T, VEC> raw[R];                         // as they are in memory: half the registers of 32-bit values
        #pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t row = row0 + int64_t(down) * r;
            if (row < a.rows && column < a.width) raw[r] = *reinterpret_cast<const Pack<T, VEC>*>(static_cast<const T*>(a.x) + row * a.x_stride + column);
            else {
                #pragma unroll
                for (int k = 0; k < VEC; ++k) raw[r].v[k] = from_float<T>(0.0f);
            }
        }
        #pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t row = row0 + int64_t(down) * r;
            if (row >= a.rows) break;
            float v[VEC];
            to_floats<T, VEC>(raw[r], v);
            float largest = largest_magnitude(v);
            const bool careful = __any_sync(0xffffffffu, largest > FLT_MAX);
            if (careful) largest = largest_finite(v);
            const int e = scale_exponent(lanes_max<kLanes>(largest));
            const float inverse = inverse_scale(e);
            if (column >= a.width) continue;
            uint8_t* codes = a.codes + row * a.codes_stride + column;
            if (careful) store_codes<true>(codes, v, inverse);
            else store_codes<false>(codes, v, inverse);
            if (lane % kLanes == 0) a.scales[row * a.scales_stride + column / kScaleBlock] = uint8_t(e + 127);
        }
    }
}

// Rows that begin anywhere, of any width, through shared memory: a warp takes 256 columns of a row while those of the next rows are on their way; a lane has every 32nd
// column.  Addresses go from row to row by one addition.
constexpr int kStretch = 256, kOnTheWay = 3;
template <typename T> constexpr int kStretchSlot = kStretch * int(sizeof(T)) + 16;         // bytes
template <typename T>
__global__ void __launch_bounds__(kQuantBlock, 6) quantize_anywhere_kernel(const QuantArgs a) {
    extern __shared__ __align__(16) unsigned char memory[];
    constexpr int kSlot = kStretchSlot<T>;
    const int lane = threadIdx.x & 31;
    const uint32_t across = uint32_t((a.width + kStretch - 1) / kStretch), warp = blockIdx.x * (kQuantBlock / 32) + (threadIdx.x >> 5);
    const uint32_t down = gridDim.x * (kQuantBlock / 32) / across;
    if (warp >= across * down) return;
    const int64_t first = int64_t(warp % across) * kStretch, row = warp / across;
    const int count = int(min(int64_t(kStretch), a.width - first)), rows = int((a.rows - row + down - 1) / down);
    const int64_t step = int64_t(down) * a.x_stride, codes_step = int64_t(down) * a.codes_stride, scales_step = int64_t(down) * a.scales_stride;
    const T *x = static_cast<const T*>(a.x) + row * a.x_stride + first, *coming = x;
    uint8_t *codes = a.codes + row * a.codes_stride + first + lane, *scales = a.scales + row * a.scales_stride + first / kScaleBlock;
    unsigned char* ring = memory + (threadIdx.x >> 5) * (kOnTheWay + 1) * kSlot;
    #pragma unroll
    for (int i = 0; i < kOnTheWay; ++i, coming += step) {
        if (i < rows) bring<kStretch>(ring + i * kSlot, coming, count, lane);
        copies_begun();
    }
    const auto go = [&](auto whole) {               // whole: every lane has all its columns
        for (int i = 0; i < rows; ++i, x += step, coming += step, codes += codes_step, scales += scales_step) {
            if (i + kOnTheWay < rows) bring<kStretch>(ring + (i + kOnTheWay) % (kOnTheWay + 1) * kSlot, coming, count, lane);
            copies_begun();
            copies_done<kOnTheWay>();
            const T* from = in_slot(ring + i % (kOnTheWay + 1) * kSlot, x) + lane;
            #pragma unroll
            for (int b = 0; b < kStretch / kScaleBlock; ++b) {
                const int there = count - b * kScaleBlock - lane;
                if (!whole && b * kScaleBlock >= count) break;
                float v[4];
                #pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = whole || 32 * j < there ? to_float<T>(from[b * kScaleBlock + 32 * j]) : 0.0f;
                float largest = largest_magnitude(v);
                const bool careful = __any_sync(0xffffffffu, largest > FLT_MAX);
                if (careful) largest = largest_finite(v);
                const int e = scale_exponent(lanes_max<32>(largest));
                const float inverse = inverse_scale(e);
                const uint32_t four = careful ? encode4<true>(v[0], v[1], v[2], v[3], inverse) : encode4<false>(v[0], v[1], v[2], v[3], inverse);
                #pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (whole || 32 * j < there) codes[b * kScaleBlock + 32 * j] = uint8_t(four >> (8 * j));
                if (lane == 0) scales[b] = uint8_t(e + 127);
            }
            __syncwarp();                           // the slot has been read
        }
    };
    if (count == kStretch) go(std::true_type());
    else go(std::false_type());
}

// One block per 128 x 128 values, which lie in shared memory as they came: 16 bytes at a time without passing through registers where the rows allow it (WIDE).
// A thread deals with eight rows by eight columns: half a warp has the 128 columns of its eight rows, so a row's largest value is found by
// shuffles, a column's through shared memory.  Transposed codes go through shared memory too, in the tile's place, so that they leave as rows of 128: the
// eight bytes of half-warp h and column c lie in slot h ^ (c / 8 % 16) of the column's sixteen, which spreads the 16 lanes of a store over all
// banks.  PER_TILE: one scale for the whole tile.
// Rows that do not begin and end on 16 bytes come in pairs of 16-bit values, or as they lie and are moved to the beginning of their slots (in us, coded and turned, pairs
// and slots: 50000 x 1002 fp16 51 and 55; single values and slots: 50000 x 1001 fp32 78 and 67, 80000 x 499 bf16 53 and 41).
// (32768 x 1024 in bf16 with its transpose: 23 us; with the tile in registers, 98 a thread, two blocks were on an SM, 26.6 us.)
template <typename T, bool WIDE> constexpr int kTilePitch = kScaleBlock + (WIDE ? 0 : 16 / int(sizeof(T)));
template <typename T, bool WIDE, bool PER_TILE>
__global__ void __launch_bounds__(kQuantBlock, 4) quantize_tiles_kernel(const QuantArgs a) {
    constexpr int VEC = 16 / int(sizeof(T)), G = 8 / VEC;                 // values in 16 bytes, and of those in a thread's eight columns
    extern __shared__ __align__(16) unsigned char raw[];
    constexpr int kPitch = kTilePitch<T, WIDE>;
    T (*tile)[kPitch] = reinterpret_cast<T (*)[kPitch]>(raw);
    uint2 (*turned)[16] = reinterpret_cast<uint2 (*)[16]>(raw);
    __shared__ float column_largest[16][kScaleBlock];
    __shared__ float column_all[kScaleBlock];
    const int l = threadIdx.x & 15, h = threadIdx.x >> 4;
    const uint32_t right = blockIdx.x, down = blockIdx.z * gridDim.y + blockIdx.y;       // of the tiles; a grid has 65535 blocks in its second direction
    const int64_t row0 = int64_t(down) * kScaleBlock, column0 = int64_t(right) * kScaleBlock;
    const int rows = int(min(int64_t(kScaleBlock), a.rows - row0)), columns = int(min(int64_t(kScaleBlock), a.width - column0));
    if (rows <= 0) return;
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
    } else if (sizeof(T) == 2 && columns % 2 == 0 && a.x_stride % 2 == 0 && reinterpret_cast<uintptr_t>(a.x) % 4 == 0) {
        #pragma unroll 8
        for (int i = 0; i < kScaleBlock * kScaleBlock / 2 / kQuantBlock; ++i) {
            const int at = i * kQuantBlock + int(threadIdx.x), r = at / (kScaleBlock / 2), c = at % (kScaleBlock / 2) * 2;
            const bool there = r < rows && c < columns;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(&tile[r][c])), "l"(there ? x + r * a.x_stride + c : x), "r"(there ? 4 : 0) : "memory");
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else {
        const int lane = threadIdx.x & 31, first = int(threadIdx.x >> 5) * 16;             // of the warp's 16 rows
        const T zero = from_float<T>(0.0f);
        for (int r = first; r < min(rows, first + 16); ++r) bring<kScaleBlock>(reinterpret_cast<unsigned char*>(tile[r]), x + r * a.x_stride, columns, lane);
        copies_begun();
        copies_done<0>();
        #pragma unroll 4
        for (int r = first; r < first + 16; ++r) {
            const T* from = in_slot(reinterpret_cast<unsigned char*>(tile[r]), x + r * a.x_stride) + lane;
            T v[4];
            #pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = r < rows && lane + 32 * i < columns ? from[32 * i] : zero;
            __syncwarp();
            #pragma unroll
            for (int i = 0; i < 4; ++i) tile[r][lane + 32 * i] = v[i];
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
        if (!PER_TILE && a.codes_t && int(threadIdx.x) < columns) a.scales_t[(column0 + threadIdx.x) * a.scales_t_stride + down] = uint8_t(scale_exponent(largest) + 127);
    }
    __syncthreads();
    int tile_e = 0;
    if (PER_TILE) {
        tile_e = scale_exponent(fmaxf(fmaxf(column_all[0], column_all[32]), fmaxf(column_all[64], column_all[96])));
        if (threadIdx.x == 0 && a.codes) a.scales[int64_t(down) * a.scales_stride + right] = uint8_t(tile_e + 127);
        if (threadIdx.x == 0 && a.codes_t) a.scales_t[int64_t(right) * a.scales_t_stride + down] = uint8_t(tile_e + 127);
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
            if (!PER_TILE && l == 0) a.scales[(row0 + h * 8 + r) * a.scales_stride + right] = uint8_t(e + 127);
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

// Codes back to values: exact in every output type, except that what leaves the range of 16-bit floats becomes infinite or zero.  VEC values side by side in a lane, and 128
// columns of a warp at least (VEC 1, 2: in a lane several groups, 32 * VEC apart).
template <typename T, int VEC>
__global__ void __launch_bounds__(kQuantBlock, 6) dequantize_kernel(const uint8_t* codes, int64_t codes_stride, const uint8_t* scales, int64_t scales_stride,
                                                                int shift, int64_t rows, int64_t width, T* out, int64_t out_stride) {
    const int lane = threadIdx.x & 31;
    constexpr int kColumns = VEC < 4 ? kScaleBlock : 32 * VEC, G = kColumns / 32 / VEC, R = kTogether;
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

// The same for rows that begin anywhere, of any width, through shared memory as in quantize_anywhere_kernel.
template <typename T> constexpr int kDecodeBytes = (kOnTheWay + 1) * (kStretch + 16) + kStretchSlot<T>;         // of a warp
template <typename T>
__global__ void __launch_bounds__(kQuantBlock, 6) dequantize_anywhere_kernel(const uint8_t* codes, int64_t codes_stride, const uint8_t* scales, int64_t scales_stride,
                                                                         int shift, int64_t rows, int64_t width, T* out, int64_t out_stride) {
    extern __shared__ __align__(16) unsigned char memory[];
    constexpr int kSlot = kStretch + 16, kBlocks = kStretch / kScaleBlock;
    const int lane = threadIdx.x & 31;
    const uint32_t across = uint32_t((width + kStretch - 1) / kStretch), warp = blockIdx.x * (kQuantBlock / 32) + (threadIdx.x >> 5);
    const uint32_t down = gridDim.x * (kQuantBlock / 32) / across;
    grid_dependency();
    if (warp >= across * down) return;
    const int64_t first = int64_t(warp % across) * kStretch;
    const int count = int(min(int64_t(kStretch), width - first)), trips = int((rows - warp / across + down - 1) / down);
    int64_t row = warp / across;                    // that comes next
    codes += row * codes_stride + first; out += row * out_stride + first;
    scales += first / kScaleBlock + (lane * kScaleBlock < count ? lane : 0);
    const int64_t step = int64_t(down) * codes_stride, out_step = int64_t(down) * out_stride;
    unsigned char* ring = memory + (threadIdx.x >> 5) * kDecodeBytes<T>;
    unsigned char* outs = ring + (kOnTheWay + 1) * kSlot;
    const uint8_t* coming = codes;
    uint32_t exponents[kOnTheWay + 1];              // lane b has block b's
    #pragma unroll
    for (int i = 0; i < kOnTheWay; ++i, coming += step, row += down) {
        exponents[i] = i < trips ? scales[(row >> shift) * scales_stride] : 0u;
        if (i < trips) bring<kStretch>(ring + i * kSlot, coming, count, lane);
        copies_begun();
    }
    const auto go = [&](auto whole) {               // whole: every lane has all its columns
        for (int i = 0; i < trips; ++i, codes += step, coming += step, out += out_step, row += down) {
            exponents[kOnTheWay] = 0u;
            if (i + kOnTheWay < trips) {
                exponents[kOnTheWay] = scales[(row >> shift) * scales_stride];
                bring<kStretch>(ring + (i + kOnTheWay) % (kOnTheWay + 1) * kSlot, coming, count, lane);
            }
            copies_begun();
            copies_done<kOnTheWay>();               // what the lanes read of the row before, and of its output, lies behind them
            const uint8_t* from = in_slot(ring + i % (kOnTheWay + 1) * kSlot, codes) + lane;
            T* to = in_slot(outs, out) + lane;
            #pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                const float scale = scale_value(__shfl_sync(0xffffffffu, exponents[0], b));
                #pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int c = b * kScaleBlock + 32 * j;
                    if (whole || lane + c < count) to[c] = from_float<T>(decode2(from[c]).x * scale);
                }
            }
            __syncwarp();
            send<kStretch>(outs, out, count, lane);
            #pragma unroll
            for (int k = 0; k < kOnTheWay; ++k) exponents[k] = exponents[k + 1];
        }
    };
    if (count == kStretch) go(std::true_type());
    else go(std::false_type());
}

// Blocks for warps that take `columns` columns of four rows each: as many as the SMs hold at once (six by the kernels' registers), and at least one row's worth.
constexpr int kSharedBytes = 227 * 1024;        // of an SM; a block takes 1 KB of them besides its own
unsigned int blocks_for(int64_t rows, int64_t width, int columns, int per_sm = 6) {
    if (per_sm > 6) per_sm = 6;
    const int64_t across = (width + columns - 1) / columns, per_block = kQuantBlock / 32;
    int64_t blocks = (across * ((rows + 3) / 4) + per_block - 1) / per_block;
    if (blocks > 148 * per_sm) blocks = 148 * per_sm;
    const int64_t least = (across + per_block - 1) / per_block;
    return unsigned(blocks > least ? blocks : least);
}

template <typename T> cudaError_t quantize_anywhere(const QuantArgs& a, cudaStream_t stream) {
    constexpr int smem = kQuantBlock / 32 * (kOnTheWay + 1) * kStretchSlot<T>;
    static PerDeviceOnce once;
    const cudaError_t err = once.run([] { return cudaFuncSetAttribute(quantize_anywhere_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
    if (err == cudaSuccess) quantize_anywhere_kernel<T><<<blocks_for(a.rows, a.width, kStretch, kSharedBytes / (smem + 1024)), kQuantBlock, smem, stream>>>(a);
    return err;
}
template <typename T, bool WIDE, bool PER_TILE> cudaError_t launch_tiles(const QuantArgs& a, cudaStream_t stream) {
    const unsigned down = unsigned((a.rows + kScaleBlock - 1) / kScaleBlock), deep = (down + 65534) / 65535;
    const dim3 grid(unsigned((a.width + kScaleBlock - 1) / kScaleBlock), (down + deep - 1) / deep, deep);
    constexpr int smem = kScaleBlock * kTilePitch<T, WIDE> * int(sizeof(T));
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
    else if (wide && rows_aligned(a.codes, a.codes_stride, a.rows, 1, V)) quantize_rows_kernel<T><<<blocks_for(a.rows, a.width, 32 * V), kQuantBlock, 0, stream>>>(a);
    else err = quantize_anywhere<T>(a, stream);
    return err == cudaSuccess ? sequence_status("htgs_quantize_fp8") : sequence_fail(HTGS_ERR_CUDA, cudaGetErrorString(err));
}

template <typename T, int VEC> cudaError_t launch_dequantize(const HtgsFp8Matrix& m, void* out, int64_t out_stride, cudaStream_t stream) {
    return launch_after(dequantize_kernel<T, VEC>, blocks_for(m.rows, m.width, VEC < 4 ? kScaleBlock : 32 * VEC), kQuantBlock, 0, stream, m.codes, m.codes_stride, m.scales, m.scales_stride,
                        m.rows_per_scale == 1 ? 0 : 7, m.rows, m.width, static_cast<T*>(out), out_stride);
}
// 16 bytes to store (with 32 a lane every store would write half sectors) or two values where every row allows it; else values of narrow matrices one by one, and those of others
// through shared memory.  (In us, one by one and through shared memory: 200000 x 101 bf16 32 and 53, x 201 64 and 54, 50000 x 1001 fp32 85 and 53; two by two and
// through shared memory 60000 x 650 fp16 34 and 46.)
template <typename T> int dequantize_typed(const HtgsFp8Matrix& m, void* out, int64_t out_stride, cudaStream_t stream) {
    constexpr int V = 16 / int(sizeof(T));
    const auto allow = [&](int values) {
        return m.width % values == 0 && rows_aligned(m.codes, m.codes_stride, m.rows, 1, values) && rows_aligned(out, out_stride, m.rows, sizeof(T), values * sizeof(T));
    };
    cudaError_t err = cudaSuccess;
    if (allow(V)) err = launch_dequantize<T, V>(m, out, out_stride, stream);
    else if (allow(2)) err = launch_dequantize<T, 2>(m, out, out_stride, stream);
    else if (m.width <= kScaleBlock) err = launch_dequantize<T, 1>(m, out, out_stride, stream);
    else {
        constexpr int smem = kQuantBlock / 32 * kDecodeBytes<T>;
        static PerDeviceOnce once;
        err = once.run([] { return cudaFuncSetAttribute(dequantize_anywhere_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
        if (err == cudaSuccess)
            err = launch_after(dequantize_anywhere_kernel<T>, blocks_for(m.rows, m.width, kStretch, kSharedBytes / (smem + 1024)), kQuantBlock, smem, stream, m.codes, m.codes_stride, m.scales,
                               m.scales_stride, m.rows_per_scale == 1 ? 0 : 7, m.rows, m.width, static_cast<T*>(out), out_stride);
    }
    return err == cudaSuccess ? sequence_status("htgs_dequantize_fp8") : sequence_fail(HTGS_ERR_CUDA, cudaGetErrorString(err));
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
    if (out_type == HTGS_FLOAT32) return dequantize_typed<float>(*matrix, out, out_stride, s);
    if (out_type == HTGS_FLOAT16) return dequantize_typed<__half>(*matrix, out, out_stride, s);
    return dequantize_typed<__nv_bfloat16>(*matrix, out, out_stride, s);
}

}  // extern "C"
