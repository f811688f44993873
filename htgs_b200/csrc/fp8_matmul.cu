// out = a * b^T for 8-bit matrices with a power-of-two scale for each block of 128 columns (fp8.cu):
//
//   out[m, n] = sum over k of  sa[m, k / 128] sb[n / (1 or 128), k / 128]  a[m, k] b[n, k]
//
// The product of two E4M3 codes is exact in 32 bits, and a scale shifts its exponent, so the only roundings are those of the 32-bit
// sum and the last one to the output's type.
//
// Few rows: `matmul_rows_kernel`, a warp per row of b, bound by reading b.  Otherwise `matmul_tiles_kernel` on the tensor cores, which take the
// scales themselves (kind::mxf8f6f4, one scale per row and 32 columns; a block of 128 uses the same one four times).
#include "sequence.cuh"

#include <cuda.h>

namespace htgs {

namespace {

constexpr int kRowsBlock = 256;

struct MatmulArgs {
    HtgsFp8Matrix a, b;
    void* out;
    int64_t out_stride;
};

// Few rows of a: a warp per row of b, 16 codes of it in a lane at a time, against ROWS rows of a.
template <typename T, int ROWS>
__global__ void __launch_bounds__(kRowsBlock) matmul_rows_kernel(const MatmulArgs args) {
    const int lane = threadIdx.x & 31;
    const int64_t n = int64_t(blockIdx.x) * (kRowsBlock / 32) + (threadIdx.x >> 5), m0 = int64_t(blockIdx.y) * ROWS;
    if (n >= args.b.rows) return;
    const uint8_t* b = args.b.codes + n * args.b.codes_stride;
    const uint8_t* sb = args.b.scales + n / args.b.rows_per_scale * args.b.scales_stride;
    float acc[ROWS] = {};
    for (int64_t k = lane * 16; k < args.a.width; k += 512) {
        const uint4 packed = *reinterpret_cast<const uint4*>(b + k);
        uint32_t words[4] = {packed.x, packed.y, packed.z, packed.w};
        if (k + 16 > args.a.width) {           // codes behind the row's end are no part of it
            #pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int64_t rest = args.a.width - k - 4 * w;
                words[w] = rest >= 4 ? words[w] : rest <= 0 ? 0u : words[w] & ((1u << (8 * int(rest))) - 1u);
            }
        }
        float2 vb[8];
        #pragma unroll
        for (int w = 0; w < 4; ++w) { vb[2 * w] = decode2(words[w]); vb[2 * w + 1] = decode2(words[w] >> 16); }
        const float scale_b = scale_value(sb[k / kScaleBlock]);
        #pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const int64_t m = m0 + r;
            if (m >= args.a.rows) break;
            const uint4 pa = *reinterpret_cast<const uint4*>(args.a.codes + m * args.a.codes_stride + k);
            uint32_t wa[4] = {pa.x, pa.y, pa.z, pa.w};
            if (k + 16 > args.a.width) {
                #pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const int64_t rest = args.a.width - k - 4 * w;
                    wa[w] = rest >= 4 ? wa[w] : rest <= 0 ? 0u : wa[w] & ((1u << (8 * int(rest))) - 1u);
                }
            }
            float sum = 0.0f;
            #pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float2 lo = decode2(wa[w]), hi = decode2(wa[w] >> 16);
                sum = fmaf(lo.x, vb[2 * w].x, sum);
                sum = fmaf(lo.y, vb[2 * w].y, sum);
                sum = fmaf(hi.x, vb[2 * w + 1].x, sum);
                sum = fmaf(hi.y, vb[2 * w + 1].y, sum);
            }
            acc[r] = fmaf(sum * scale_value(args.a.scales[m / args.a.rows_per_scale * args.a.scales_stride + k / kScaleBlock]), scale_b, acc[r]);
        }
    }
    #pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const float total = warp_sum(acc[r]);
        if (lane == 0 && m0 + r < args.a.rows) static_cast<T*>(args.out)[(m0 + r) * args.out_stride + n] = from_float<T>(total);
    }
}

// ---- tensor cores ------------------------------------------------------------------------------------------------------------
//
// A tile is 128 rows of a by BN rows of b.  Persistent blocks of twelve warps, each with its role, go through the tiles:
//   warp 0        loads 128 columns of a's and b's rows at a time into a ring of shared-memory stages (TMA, 128-byte swizzle)
//   warp 1        issues the matrix instructions (one thread) into one of two accumulators in tensor memory
//   warps 4 .. 7  put the scale bytes of four blocks of 128 columns into tensor memory: the word of row r in lane r % 32 of each quarter, column r / 32
//   warps 8 .. 11 bring an accumulator's rows out, round them and store them while the next tile is computed
// With few tiles the sum over the columns is split over the blocks of a cluster; each leaves its 32-bit part in its shared memory, and every
// block adds up some of the rows, always in the same order.
// Every wait has a time limit.  A role whose wait runs out reports it (MatmulArgs::error, which the next call returns), and the others follow.

constexpr int kTileRows = 128;
constexpr int kTileThreads = 384;
constexpr int kAccumulators = 2, kScaleStages = 2, kScaleColumns = 12;       // 4 columns of a's scales and up to 8 of b's
constexpr uint64_t kWaitNanoseconds = 2000000000ull;

template <int BN> struct Tile {
    static constexpr int stage_bytes = kTileRows * kScaleBlock + BN * kScaleBlock;
    static constexpr int stages = BN <= 64 ? 8 : BN <= 128 ? 6 : BN <= 192 ? 5 : 4;
    static constexpr int barriers = 2 * stages + 2 * kScaleStages + 2 * kAccumulators + 1;
    static constexpr int smem = 1024 + stages * stage_bytes + 256;             // the ring begins on a multiple of 1024; over half of an SM's, so that one block has it alone
    static constexpr int partial_pitch = BN + 4;                                // floats
    static_assert(barriers * 8 + 16 <= 256 && smem > 116 * 1024 && smem <= 227 * 1024, "shared memory");
    static_assert(kTileRows * partial_pitch * 4 <= stages * stage_bytes, "a part's sums fit the ring");
    static_assert(kAccumulators * BN + kScaleStages * kScaleColumns <= 512, "tensor memory");
};

struct TileArgs {
    const uint8_t* scales_a; const uint8_t* scales_b;
    int64_t scales_a_stride, scales_b_stride;
    int32_t rows_a, rows_b, shift_a, shift_b;       // shift: 0 or 7, rows per scale
    int32_t blocks_k, tiles_n, tiles;
    void* out; int64_t out_stride;
    int32_t wide;                                   // out takes 16-byte stores
    unsigned int* error;
};

__device__ __forceinline__ uint64_t nanoseconds() { uint64_t t; asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t)); return t; }

__device__ __forceinline__ void arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// False if the time limit ran out or another role has given up.
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, volatile uint32_t* failed) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t begin = nanoseconds();
    while (!mbar_try_wait(bar, parity)) {
        if (*failed) return false;
        if (nanoseconds() - begin > kWaitNanoseconds) { *failed = 1; return false; }
    }
    return true;
}

__device__ __forceinline__ void tma_load(void* to, const CUtensorMap* map, int column, int row, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(smem_u32(to)), "l"(map), "r"(column), "r"(row), "r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tmem_store4(uint32_t address, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(address), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void tmem_load32(uint32_t address, uint32_t (&v)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
                   "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]),
                   "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(address));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// Shared-memory operand: rows of 128 bytes under the 128-byte swizzle, groups of 8 rows 1024 bytes apart (the leading offset says nothing there).
__device__ __forceinline__ uint64_t operand(uint32_t address) {
    return uint64_t((address & 0x3ffffu) >> 4) | uint64_t(1) << 16 | uint64_t(1024 >> 4) << 32 | uint64_t(1) << 46 | uint64_t(2) << 61;
}
// E4M3 by E4M3, both along the columns, power-of-two scales; `which`: the byte of the scale words.
template <int BN> __device__ __forceinline__ uint32_t instruction(uint32_t which) {
    return which << 4 | uint32_t(BN >> 3) << 17 | 1u << 23 | uint32_t(kTileRows >> 7) << 27 | which << 29;
}
__device__ __forceinline__ void multiply(uint32_t d, uint64_t a, uint64_t b, uint32_t instruction, uint32_t scale_a, uint32_t scale_b, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(instruction), "r"(scale_a), "r"(scale_b), "r"(uint32_t(add)) : "memory");
}

// One row's 32 columns, rounded and stored.
template <typename T> __device__ __forceinline__ void store_row(T* row, int column, int columns, const uint32_t (&v)[32], bool wide) {
    constexpr int V = 16 / int(sizeof(T));
    #pragma unroll
    for (int i = 0; i < 32; i += V) {
        float f[V];
        #pragma unroll
        for (int k = 0; k < V; ++k) f[k] = __uint_as_float(v[i + k]);
        if (wide && column + i + V <= columns) store_floats<T, V>(row + column + i, f);
        else {
            #pragma unroll
            for (int k = 0; k < V; ++k)
                if (column + i + k < columns) row[column + i + k] = from_float<T>(f[k]);
        }
    }
}

// SPLIT: gridDim.x = tiles * parts in clusters of `parts` blocks, one tile each; else parts is 1.
template <typename T, int BN, bool SPLIT>
__global__ void __launch_bounds__(kTileThreads, 1) matmul_tiles_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                                                                      const TileArgs args, const int parts) {
    using S = Tile<BN>;
    extern __shared__ unsigned char raw[];
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    unsigned char* ring = raw + (base - smem_u32(raw));
    uint64_t* full = reinterpret_cast<uint64_t*>(ring + S::stages * S::stage_bytes);
    uint64_t* empty = full + S::stages;
    uint64_t* scale_full = empty + S::stages;
    uint64_t* scale_empty = scale_full + kScaleStages;
    uint64_t* sum_full = scale_empty + kScaleStages;
    uint64_t* sum_empty = sum_full + kAccumulators;
    uint64_t* drained = sum_empty + kAccumulators;
    uint32_t* tmem_at = reinterpret_cast<uint32_t*>(drained + 1);
    volatile uint32_t* failed = tmem_at + 1;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::stages; ++i) { mbar_init(full + i, 1); mbar_init(empty + i, 1); }
        for (int i = 0; i < kScaleStages; ++i) { mbar_init(scale_full + i, 4); mbar_init(scale_empty + i, 1); }
        for (int i = 0; i < kAccumulators; ++i) { mbar_init(sum_full + i, 1); mbar_init(sum_empty + i, 4); }
        mbar_init(drained, 1);
        *failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_at)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tmem_fence_before();
    }
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = *tmem_at;
    const uint32_t tmem_scales = tmem + kAccumulators * BN;

    const int part = SPLIT ? int(blockIdx.x) % parts : 0;
    const int first_tile = SPLIT ? int(blockIdx.x) / parts : int(blockIdx.x), tile_step = SPLIT ? args.tiles : int(gridDim.x);
    const int k_begin = SPLIT ? int(int64_t(args.blocks_k) * part / parts) : 0;
    const int k_end = SPLIT ? int(int64_t(args.blocks_k) * (part + 1) / parts) : args.blocks_k;

    if (warp == 0) {
        if (lane == 0) {
            uint32_t use = 0;
            bool ok = true;
            for (int tile = first_tile; ok && tile < args.tiles; tile += tile_step) {
                const int row_a = tile / args.tiles_n * kTileRows, row_b = tile % args.tiles_n * BN;
                for (int k = k_begin; k < k_end; ++k, ++use) {
                    const uint32_t stage = use % S::stages, round = use / S::stages;
                    ok = wait_for(empty + stage, (round & 1) ^ 1, failed);
                    if (!ok) break;
                    mbar_arrive_expect_tx(full + stage, S::stage_bytes);
                    unsigned char* at = ring + stage * S::stage_bytes;
                    tma_load(at, &map_a, k * kScaleBlock, row_a, full + stage);
                    tma_load(at + kTileRows * kScaleBlock, &map_b, k * kScaleBlock, row_b, full + stage);
                }
            }
            if (!ok)            // no copy may be on its way when the block ends
                for (uint32_t u = use > S::stages ? use - S::stages : 0; u < use; ++u) {
                    const uint64_t begin = nanoseconds();
                    while (!mbar_try_wait(full + u % S::stages, u / S::stages & 1) && nanoseconds() - begin < kWaitNanoseconds) {}
                }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            uint32_t use = 0, scale_use = 0, tile_use = 0;
            bool ok = true;
            for (int tile = first_tile; ok && tile < args.tiles; tile += tile_step, ++tile_use) {
                const uint32_t sum = tile_use % kAccumulators;
                ok = wait_for(sum_empty + sum, (tile_use / kAccumulators & 1) ^ 1, failed);
                if (!ok) break;
                tmem_fence_after();
                for (int k = k_begin; k < k_end; ++k, ++use) {
                    const uint32_t scale_stage = scale_use % kScaleStages;
                    if (k == k_begin || (k & 3) == 0) {
                        ok = wait_for(scale_full + scale_stage, scale_use / kScaleStages & 1, failed);
                        if (!ok) break;
                    }
                    const uint32_t stage = use % S::stages;
                    ok = wait_for(full + stage, use / S::stages & 1, failed);
                    if (!ok) break;
                    tmem_fence_after();
                    const uint32_t scales = tmem_scales + scale_stage * kScaleColumns;
                    const uint64_t a = operand(base + stage * S::stage_bytes), b = operand(base + stage * S::stage_bytes + kTileRows * kScaleBlock);
                    #pragma unroll
                    for (int i = 0; i < 4; ++i)          // 32 columns each, 32 bytes further on
                        multiply(tmem + sum * BN, a + 2 * i, b + 2 * i, instruction<BN>(k & 3), scales, scales + 4, k > k_begin || i > 0);
                    tmem_commit(empty + stage);
                    if (k + 1 == k_end || (k & 3) == 3) { tmem_commit(scale_empty + scale_stage); ++scale_use; }
                }
                if (ok) tmem_commit(sum_full + sum);
            }
            if (!ok) {
                tmem_commit(drained);
                const uint64_t begin = nanoseconds();
                while (!mbar_try_wait(drained, 0) && nanoseconds() - begin < kWaitNanoseconds) {}
            }
        }
    } else if (warp >= 4 && warp < 8) {
        const uint32_t quarter = uint32_t(warp - 4) * 32 << 16;
        uint32_t scale_use = 0;
        bool ok = true;
        for (int tile = first_tile; ok && tile < args.tiles; tile += tile_step) {
            const int row_a = tile / args.tiles_n * kTileRows, row_b = tile % args.tiles_n * BN;
            for (int group = k_begin >> 2; group <= (k_end - 1) >> 2; ++group, ++scale_use) {
                uint32_t a[4], b[8];
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = row_a + 32 * i + lane;
                    a[i] = row < args.rows_a ? __ldg(reinterpret_cast<const uint32_t*>(args.scales_a + (row >> args.shift_a) * args.scales_a_stride) + group) : 0x7f7f7f7fu;
                }
                #pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int row = row_b + 32 * i + lane;
                    b[i] = 32 * i < BN && row < args.rows_b ? __ldg(reinterpret_cast<const uint32_t*>(args.scales_b + (row >> args.shift_b) * args.scales_b_stride) + group) : 0x7f7f7f7fu;
                }
                const uint32_t stage = scale_use % kScaleStages;
                ok = wait_for(scale_empty + stage, (scale_use / kScaleStages & 1) ^ 1, failed);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tmem_fence_after();
                const uint32_t to = tmem_scales + stage * kScaleColumns + quarter;
                tmem_store4(to, a[0], a[1], a[2], a[3]);
                tmem_store4(to + 4, b[0], b[1], b[2], b[3]);
                if (BN > 128) tmem_store4(to + 8, b[4], b[5], b[6], b[7]);
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) arrive(scale_full + stage);
            }
        }
    } else if (warp >= 8) {
        const uint32_t quarter = uint32_t(warp - 8) * 32;
        uint32_t tile_use = 0;
        for (int tile = first_tile; tile < args.tiles; tile += tile_step, ++tile_use) {
            const uint32_t sum = tile_use % kAccumulators;
            bool ok = wait_for(sum_full + sum, tile_use / kAccumulators & 1, failed);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tmem_fence_after();
            const int column0 = tile % args.tiles_n * BN;
            const int64_t row = int64_t(tile / args.tiles_n) * kTileRows + quarter + lane;
            #pragma unroll 1
            for (int c = 0; c < BN; c += 32) {
                uint32_t v[32];
                tmem_load32(tmem + sum * BN + c + (quarter << 16), v);
                if (SPLIT) {
                    float* to = reinterpret_cast<float*>(ring) + (quarter + lane) * S::partial_pitch + c;
                    #pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *reinterpret_cast<uint4*>(to + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                } else if (row < args.rows_a && column0 + c < args.rows_b) {
                    store_row<T>(static_cast<T*>(args.out) + row * args.out_stride, column0 + c, args.rows_b, v, args.wide != 0);
                }
            }
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) arrive(sum_empty + sum);
        }
    }
    __syncwarp();
    if (SPLIT) {
        cluster_barrier();
        const int rows = kTileRows / parts, column0 = first_tile % args.tiles_n * BN;
        const int64_t row0 = int64_t(first_tile / args.tiles_n) * kTileRows;
        for (int i = threadIdx.x; i < rows * BN; i += kTileThreads) {
            const int r = part * rows + i / BN, c = i % BN;
            if (row0 + r >= args.rows_a || column0 + c >= args.rows_b) continue;
            float total = 0.0f;
            for (int p = 0; p < parts; ++p) total += peer_float(base + uint32_t(r * S::partial_pitch + c) * 4, p);
            static_cast<T*>(args.out)[(row0 + r) * args.out_stride + column0 + c] = from_float<T>(total);
        }
        cluster_barrier();           // no block's shared memory goes before the others have read it
    }
    __syncthreads();
    if (warp == 1) {
        tmem_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
    if (threadIdx.x == 0 && *failed) {
        *reinterpret_cast<volatile unsigned int*>(args.error) = 1;
        __threadfence_system();
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                 CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
    static const EncodeTiled found = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult result;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &result) != cudaSuccess || result != cudaDriverEntryPointSuccess) f = nullptr;
        return reinterpret_cast<EncodeTiled>(f);
    }();
    return found;
}

bool make_map(CUtensorMap* map, const HtgsFp8Matrix& m, int box_rows) {
    const cuuint64_t sizes[2] = {cuuint64_t(m.width), cuuint64_t(m.rows)}, strides[1] = {cuuint64_t(m.codes_stride)};
    const cuuint32_t box[2] = {kScaleBlock, cuuint32_t(box_rows)}, steps[2] = {1, 1};
    const EncodeTiled encode = encode_tiled();
    return encode && encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(m.codes), sizes, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A word in the host's memory that a kernel sets when one of its waits runs out; the next product reports it.  One per process.
unsigned int* error_word() {
    static unsigned int* const word = [] {
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;       // the first call may be inside a capture
        cudaThreadExchangeStreamCaptureMode(&mode);
        void* p = nullptr;
        if (cudaHostAlloc(&p, sizeof(unsigned int), cudaHostAllocPortable | cudaHostAllocMapped) != cudaSuccess) p = nullptr;
        cudaThreadExchangeStreamCaptureMode(&mode);
        if (p) *static_cast<volatile unsigned int*>(p) = 0;
        return static_cast<unsigned int*>(p);
    }();
    return word;
}

template <typename T, int BN> int launch_tiles(const MatmulArgs& m, int parts, cudaStream_t stream) {
    using S = Tile<BN>;
    unsigned int* error = error_word();
    if (!error) return sequence_fail(HTGS_ERR_CUDA, "htgs_fp8_matmul: no host memory for the error word");
    CUtensorMap map_a, map_b;
    if (!make_map(&map_a, m.a, kTileRows) || !make_map(&map_b, m.b, BN)) return sequence_fail(HTGS_ERR_CUDA, "htgs_fp8_matmul: the tensor maps cannot be made");
    TileArgs args{};
    args.scales_a = m.a.scales; args.scales_b = m.b.scales; args.scales_a_stride = m.a.scales_stride; args.scales_b_stride = m.b.scales_stride;
    args.rows_a = int32_t(m.a.rows); args.rows_b = int32_t(m.b.rows);
    args.shift_a = m.a.rows_per_scale == 1 ? 0 : 7; args.shift_b = m.b.rows_per_scale == 1 ? 0 : 7;
    args.blocks_k = int32_t((m.a.width + kScaleBlock - 1) / kScaleBlock);
    args.tiles_n = int32_t((m.b.rows + BN - 1) / BN);
    const int64_t tiles = (m.a.rows + kTileRows - 1) / kTileRows * args.tiles_n;
    if (tiles > 0x3fffffff) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_fp8_matmul: too many tiles");
    args.tiles = int32_t(tiles);
    args.out = m.out; args.out_stride = m.out_stride;
    args.wide = rows_aligned(m.out, m.out_stride, m.a.rows, sizeof(T), 16);
    args.error = error;
    cudaLaunchConfig_t config{};
    config.blockDim = kTileThreads; config.dynamicSmemBytes = S::smem; config.stream = stream;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = unsigned(parts); attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    cudaError_t err;
    if (parts > 1) {
        static PerDeviceOnce once;
        err = once.run([] { return cudaFuncSetAttribute(matmul_tiles_kernel<T, BN, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::smem); });
        config.gridDim = unsigned(args.tiles) * unsigned(parts);
        config.attrs = &attribute; config.numAttrs = 1;
        if (err == cudaSuccess) err = cudaLaunchKernelEx(&config, matmul_tiles_kernel<T, BN, true>, map_a, map_b, args, parts);
    } else {
        static PerDeviceOnce once;
        err = once.run([] { return cudaFuncSetAttribute(matmul_tiles_kernel<T, BN, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::smem); });
        config.gridDim = unsigned(args.tiles < 148 ? args.tiles : 148);
        if (err == cudaSuccess) err = cudaLaunchKernelEx(&config, matmul_tiles_kernel<T, BN, false>, map_a, map_b, args, 1);
    }
    return err == cudaSuccess ? sequence_status("htgs_fp8_matmul") : sequence_fail(HTGS_ERR_CUDA, cudaGetErrorString(err));
}

template <typename T> int matmul_typed(const MatmulArgs& args, cudaStream_t stream) {
    if (args.a.rows <= 8) {
        constexpr int R = 8;
        const dim3 grid(unsigned((args.b.rows + kRowsBlock / 32 - 1) / (kRowsBlock / 32)), unsigned((args.a.rows + R - 1) / R));
        matmul_rows_kernel<T, R><<<grid, kRowsBlock, 0, stream>>>(args);
        return sequence_status("htgs_fp8_matmul");
    }
    // The time of a tile goes with its width, and the tiles go in waves of one per SM.
    const int64_t tiles_m = (args.a.rows + kTileRows - 1) / kTileRows;
    const int64_t blocks_k = (args.a.width + kScaleBlock - 1) / kScaleBlock;
    const int64_t tiles128 = tiles_m * ((args.b.rows + 127) / 128);
    int parts = 1;
    while (parts < 8 && tiles128 * parts * 2 <= 148 && blocks_k >= 2 * parts) parts *= 2;
    if (parts > 1) return launch_tiles<T, 128>(args, parts, stream);
    const int widths[] = {64, 128, 192, 224};
    int best = 224;
    int64_t least = INT64_MAX;
    for (int w : widths) {
        const int64_t tiles = tiles_m * ((args.b.rows + w - 1) / w), time = (tiles + 147) / 148 * (w < 128 ? 128 : w);
        if (time <= least) { least = time; best = w; }
    }
    if (best == 64) return launch_tiles<T, 64>(args, 1, stream);
    if (best == 128) return launch_tiles<T, 128>(args, 1, stream);
    if (best == 192) return launch_tiles<T, 192>(args, 1, stream);
    return launch_tiles<T, 224>(args, 1, stream);
}

bool matrix_ok(const HtgsFp8Matrix* m) {
    return m && m->rows >= 0 && m->rows <= 0x7fffff00 && m->width >= 0 && m->width <= 0x7fffffff && (m->rows_per_scale == 1 || m->rows_per_scale == kScaleBlock) &&
           (m->rows == 0 || m->width == 0 ||
            (m->codes && m->scales && rows_aligned(m->codes, m->codes_stride, m->rows, 1, 16) && rows_aligned(m->scales, m->scales_stride, m->rows, 1, 4) &&
             m->codes_stride >= m->width && m->scales_stride >= (m->width + kScaleBlock - 1) / kScaleBlock));
}

}  // namespace

}  // namespace htgs

extern "C" {

int htgs_fp8_matmul(const HtgsFp8Matrix* a, const HtgsFp8Matrix* b, void* out, int64_t out_stride, int out_type, void* stream) {
    using namespace htgs;
    if (!matrix_ok(a) || !matrix_ok(b))
        return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_fp8_matmul: matrices need sizes below 2^31 - 256, codes on 16 bytes, scales on 4 bytes, rows_per_scale 1 or 128");
    if (a->width != b->width) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_fp8_matmul: a and b must have the same width");
    if (!known_type(out_type)) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_fp8_matmul: unknown element type");
    if (a->rows == 0 || b->rows == 0) return HTGS_OK;
    if (!out || out_stride < b->rows) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_fp8_matmul: out must not be null, and its rows must hold b.rows values");
    if (volatile unsigned int* error = error_word(); error && *error) {
        *error = 0;
        return sequence_fail(HTGS_ERR_DEVICE_FLAG, "htgs_fp8_matmul: a wait in an earlier product ran out, and its result is not complete");
    }
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a->width == 0) {
        const cudaError_t err = cudaMemset2DAsync(out, size_t(out_stride) * type_bytes(out_type), 0, size_t(b->rows) * type_bytes(out_type), size_t(a->rows), s);
        return err == cudaSuccess ? HTGS_OK : sequence_fail(HTGS_ERR_CUDA, cudaGetErrorString(err));
    }
    const MatmulArgs args{*a, *b, out, out_stride};
    if (out_type == HTGS_FLOAT32) return matmul_typed<float>(args, s);
    if (out_type == HTGS_FLOAT16) return matmul_typed<__half>(args, s);
    return matmul_typed<__nv_bfloat16>(args, s);
}

}  // extern "C"
