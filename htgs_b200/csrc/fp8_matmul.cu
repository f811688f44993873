// out = a * b^T for 8-bit matrices with a power-of-two scale for each block of 128 columns (fp8.cu):
//
//   out[m, n] = sum over k of  sa[m, k / 128] sb[n / (1 or 128), k / 128]  a[m, k] b[n, k]
//
// The product of two E4M3 codes is exact in 32 bits, and a scale shifts its exponent, so the only roundings are those of the 32-bit
// sum and the last one to the output's type.
//
// Up to eight rows: `matmul_rows_kernel`, a warp per row of b.  Otherwise `matmul_tiles_kernel` on the tensor cores, which take the scales themselves (kind::mxf8f6f4, one scale
// per row and 32 columns; a block of 128 uses the same one four times).
#include "tensor_core.cuh"

namespace htgs {

namespace {

constexpr int kRowsBlock = 256;

struct MatmulArgs {
    HtgsFp8Matrix a, b;
    void* out;
    int64_t out_stride;
};

// Sixteen codes from column k on of a row of `width`, without what lies behind its end.
__device__ __forceinline__ void load_codes(const uint8_t* row, int64_t k, int64_t width, uint32_t (&words)[4]) {
    const uint4 packed = *reinterpret_cast<const uint4*>(row + k);
    words[0] = packed.x; words[1] = packed.y; words[2] = packed.z; words[3] = packed.w;
    if (k + 16 <= width) return;
    #pragma unroll
    for (int w = 0; w < 4; ++w) {
        const int64_t rest = width - k - 4 * w;
        words[w] = rest >= 4 ? words[w] : rest <= 0 ? 0u : words[w] & ((1u << (8 * int(rest))) - 1u);
    }
}

// Few rows of a: a warp per row of b, 16 codes of it in a lane at a time, against ROWS rows of a.  Bound by the launch for small b, else by instructions: a multiply-add and a part of
// decoding for each code and row of a.  us, one row / eight rows, and the tensor cores' tiles for either (of codes, calls close behind one another; b up to 2048 x 2048 in L2, beyond it from HBM): 512 x 512 1.9 / 5.8 and 3.4, 1024 x 2048
// 2.8 / 10.4 and 4.5, 2048 x 2048 5.1 / 18.6 and 6.7, 4096 x 4096 10.6 / 46 and 8.6, 8192 x 8192 34 / 152 and 19.  What it saves is a launch, with VALUES: the coding's.
// With VALUES a comes as values of type X and each block codes them itself into shared memory, as quantize_rows_kernel would (fp8.cu): a launch less.
struct ValuesArgs { const void* x; int64_t stride; };
constexpr int kMostRows = 8, kMostValues = 32768;       // of a
template <typename T, int ROWS, typename X, bool VALUES>
__global__ void __launch_bounds__(kRowsBlock) matmul_rows_kernel(const MatmulArgs args, const ValuesArgs values) {
    extern __shared__ __align__(16) uint8_t coded[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t n = int64_t(blockIdx.x) * (kRowsBlock / 32) + warp, m0 = int64_t(blockIdx.y) * ROWS, width = args.a.width;
    const int across = int((width + kScaleBlock - 1) / kScaleBlock);
    const int pitch = across * kScaleBlock;
    uint8_t* exponents = coded + args.a.rows * pitch;                            // with VALUES all rows of a are the block's
    grid_dependency();
    if (VALUES) {
        for (int unit = warp; unit < int(args.a.rows) * across; unit += kRowsBlock / 32) {
            const int row = unit / across, block = unit - row * across;
            const X* x = static_cast<const X*>(values.x) + row * values.stride + block * kScaleBlock;
            float v[4];
            #pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = block * kScaleBlock + lane + 32 * i < width ? to_float<X>(x[lane + 32 * i]) : 0.0f;
            const int e = scale_exponent(lanes_max<32>(largest_finite(v)));
            #pragma unroll
            for (int i = 0; i < 4; ++i) coded[row * pitch + block * kScaleBlock + lane + 32 * i] = uint8_t(encode2<true>(v[i], 0.0f, inverse_scale(e)) & 0xffu);
            if (lane == 0) exponents[row * across + block] = uint8_t(e + 127);
        }
        __syncthreads();
    }
    if (n >= args.b.rows) return;
    const uint8_t* b = args.b.codes + n * args.b.codes_stride;
    const uint8_t* sb = args.b.scales + n / args.b.rows_per_scale * args.b.scales_stride;
    float acc[ROWS] = {};
    for (int64_t k = lane * 16; k < width; k += 512) {
        uint32_t words[4];
        load_codes(b, k, width, words);
        float2 vb[8];
        #pragma unroll
        for (int w = 0; w < 4; ++w) { vb[2 * w] = decode2(words[w]); vb[2 * w + 1] = decode2(words[w] >> 16); }
        const uint32_t scale_b = sb[k / kScaleBlock];
        #pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const int64_t m = m0 + r;
            if (m >= args.a.rows) break;
            uint32_t wa[4];
            uint32_t scale_a;
            if (VALUES) {
                const uint4 packed = *reinterpret_cast<const uint4*>(coded + r * pitch + k);
                wa[0] = packed.x; wa[1] = packed.y; wa[2] = packed.z; wa[3] = packed.w;
                scale_a = exponents[r * across + k / kScaleBlock];
            } else {
                load_codes(args.a.codes + m * args.a.codes_stride, k, width, wa);
                scale_a = args.a.scales[m / args.a.rows_per_scale * args.a.scales_stride + k / kScaleBlock];
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
            const float2 factors = scale_factors(scale_a, scale_b);
            acc[r] = fmaf(sum * factors.x, factors.y, acc[r]);
        }
    }
    #pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        if (m0 + r >= args.a.rows) break;
        const float total = warp_sum(acc[r]);
        if (lane == 0) static_cast<T*>(args.out)[(m0 + r) * args.out_stride + n] = from_float<T>(total);
    }
}

template <typename T, int ROWS, typename X, bool VALUES> int launch_rows(const MatmulArgs& args, const ValuesArgs& values, cudaStream_t stream) {
    const int across = int((args.a.width + kScaleBlock - 1) / kScaleBlock);
    const size_t smem = VALUES ? size_t(args.a.rows) * across * (kScaleBlock + 1) : 0;
    const dim3 grid(unsigned((args.b.rows + kRowsBlock / 32 - 1) / (kRowsBlock / 32)), unsigned((args.a.rows + ROWS - 1) / ROWS));
    const cudaError_t err = launch_after(matmul_rows_kernel<T, ROWS, X, VALUES>, grid, kRowsBlock, smem, stream, args, values);
    return err == cudaSuccess ? sequence_status("htgs_fp8_matmul") : sequence_fail(HTGS_ERR_CUDA, cudaGetErrorString(err));
}
template <typename T, typename X> int matmul_values(const MatmulArgs& args, const ValuesArgs& values, cudaStream_t stream) {
    return args.a.rows == 1 ? launch_rows<T, 1, X, true>(args, values, stream) : launch_rows<T, kMostRows, X, true>(args, values, stream);
}
template <typename T> int matmul_values(const MatmulArgs& args, const ValuesArgs& values, int type, cudaStream_t stream) {
    if (type == HTGS_FLOAT32) return matmul_values<T, float>(args, values, stream);
    if (type == HTGS_FLOAT16) return matmul_values<T, __half>(args, values, stream);
    return matmul_values<T, __nv_bfloat16>(args, values, stream);
}

// ---- tensor cores ------------------------------------------------------------------------------------------------------------
//
// A tile is 128 rows of a, or 256 for a pair of blocks, by BN rows of b.  Persistent blocks of twelve warps, each with its role, go through the tiles:
//   warp 0        loads 128 columns of a's and b's rows at a time into a ring of shared-memory stages (TMA, 128-byte swizzle)
//   warp 1        issues the matrix instructions (one thread) into one of two accumulators in tensor memory
//   warps 4 .. 7  put the scale bytes of four blocks of 128 columns into tensor memory: the word of row r in lane r % 32 of each quarter, column r / 32
//   warps 8 .. 11 bring an accumulator's rows out, round them and store them while the next tile is computed
// Pair: two blocks of a cluster, on two SMs, work on one tile (cta_group::2).  Each loads its own 128 rows of a and half of the rows of b, and the first one's
// instruction reads both halves, which is a third less to copy into shared memory.
// The output leaves through shared memory, 32 rows by 32 columns at a time, by TMA where its rows begin on 16 bytes and else as rows of 32 values: lanes that
// stored their own rows took 264 us for 100000 x 1024 by 2048 instead of 207, and 48 instead of 12 for 4099 x 1080 by 1001.
// Measured (bf16 out): 100000 x 1024 by 2048 2029 TFLOP/s, 8192 x 8192 by 8192 2487; without any loads the matrix instructions alone reach 2391 and 3354.
// Split: with few tiles the sum over the columns is split over the blocks of a cluster; each leaves its 32-bit part in its shared memory, and every
// block adds up some of the rows, always in the same order.
// Every wait has a time limit (WaitLimit).  A role whose wait runs out reports it (TileArgs::error: htgs_fp8_matmul_status), the others follow,
// and the block's tiles are left full of NaN.

constexpr int kTileRows = 128;                 // of a block
constexpr int kSms = 148;
constexpr int kMostParts = 8;
constexpr int kTileThreads = 384;
constexpr int kAccumulators = 2, kScaleStages = 4, kScaleColumns = 12;       // 4 columns of a's scales and up to 8 of b's

enum TileMode { kSingle, kSplit, kPair };

constexpr int kPatch = 32;                       // rows and columns that a warp of the output's stores at a time

template <typename T, int BN, int MODE> struct Tile {
    static constexpr int blocks = MODE == kPair ? 2 : 1;                            // of a tile
    static constexpr int b_rows = BN / blocks;                                      // loaded by a block
    static constexpr int stage_bytes = kTileRows * kScaleBlock + b_rows * kScaleBlock;
    static constexpr int patch_bytes = kPatch * kPatch * int(sizeof(T));
    static constexpr int out_bytes = 4 * 2 * patch_bytes;                          // two for each of four warps
    static constexpr int word_bytes = MODE == kSplit ? 2 * kScaleColumns * 32 * 4 : 0;       // two groups' scale words
    static constexpr int room = (227 * 1024 - 1024 - 256 - word_bytes - out_bytes) / stage_bytes, stages = room < 8 ? room : 8;
    static constexpr int barriers = 2 * stages + 2 * kScaleStages + 2 * kAccumulators + 1;
    static constexpr int smem = 1024 + stages * stage_bytes + out_bytes + word_bytes + 256;  // the ring begins on a multiple of 1024; over half of an SM's, so that one block has it alone
    static constexpr int partial_pitch = BN + 4;                                // floats
    static_assert(barriers * 8 + 16 <= 256 && smem > 116 * 1024 && smem <= 227 * 1024 && stage_bytes % 1024 == 0, "shared memory");
    static_assert(MODE != kSplit || kTileRows * partial_pitch * 4 <= stages * stage_bytes, "a part's sums fit the ring");
    static_assert(kAccumulators * BN + kScaleStages * kScaleColumns <= 512 && smem >= kLeastTensorShared && alone_with_tensor_memory(smem), "tensor memory");
};

struct TileArgs {
    const uint8_t* scales_a; const uint8_t* scales_b;
    int64_t scales_a_stride, scales_b_stride;
    int32_t rows_a, rows_b, shift_a, shift_b;       // shift: 0 or 7, rows per scale
    int32_t blocks_k, tiles_n, tiles;
    void* out; int64_t out_stride;
    int32_t mapped;                                 // out has a tensor map: its rows begin on 16 bytes
    unsigned int* error;
};

__device__ __forceinline__ void arrive_there(uint32_t bar) { asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }

// `bar`: in a pair, a barrier of the first block.
template <int MODE> __device__ __forceinline__ void tma_load(void* to, const CUtensorMap* map, int column, int row, uint32_t bar) {
    if constexpr (MODE == kPair)
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                     ::"r"(smem_u32(to)), "l"(map), "r"(column), "r"(row), "r"(bar) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                     ::"r"(smem_u32(to)), "l"(map), "r"(column), "r"(row), "r"(bar) : "memory");
}

// An arrival, once the instructions so far are done; in a pair at both blocks' barriers.
template <int MODE> __device__ __forceinline__ void tmem_commit(uint64_t* bar) {
    if constexpr (MODE == kPair)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"(uint16_t(3)) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tmem_store4(uint32_t address, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(address), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// Shared-memory operands: rows of 128 bytes under the 128-byte swizzle, groups of 8 rows 1024 bytes apart (the leading offset says nothing there).  The
// lower word of a descriptor has the address in units of 16 bytes, the upper one is the same for all.
constexpr uint32_t kOperandHigh = 1024 >> 4 | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t operand_low(uint32_t address) { return (address & 0x3ffffu) >> 4 | 1u << 16; }
// E4M3 by E4M3, both along the columns, power-of-two scales; bits 4 and 29: which byte of the scale words.
template <int BN, int MODE> constexpr uint32_t kInstruction = uint32_t(BN >> 3) << 17 | 1u << 23 | uint32_t(MODE == kPair ? 2 : 1) << 27;
template <int MODE>
__device__ __forceinline__ void multiply(uint32_t d, uint32_t a, uint32_t b, uint32_t instruction, uint32_t scale_a, uint32_t scale_b, uint32_t add) {
    if constexpr (MODE == kPair)
        asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %6, 0;\n\tmov.b64 da, {%1, %7};\n\tmov.b64 db, {%2, %7};\n\t"
                     "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], da, db, %3, [%4], [%5], p;\n\t}"
                     ::"r"(d), "r"(a), "r"(b), "r"(instruction), "r"(scale_a), "r"(scale_b), "r"(add), "n"(kOperandHigh) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %6, 0;\n\tmov.b64 da, {%1, %7};\n\tmov.b64 db, {%2, %7};\n\t"
                     "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], da, db, %3, [%4], [%5], p;\n\t}"
                     ::"r"(d), "r"(a), "r"(b), "r"(instruction), "r"(scale_a), "r"(scale_b), "r"(add), "n"(kOperandHigh) : "memory");
}

// 32 columns of a lane's row, rounded, into a patch of 32 rows.  Pieces of 16 bytes change places as the tensor map's swizzle says (64 bytes for
// 16-bit types, 128 for 32), which also keeps the lanes of a store in banks of their own.
template <typename T> __device__ __forceinline__ uint32_t patch_piece(int row, int piece) { return sizeof(T) == 2 ? piece ^ (row >> 1 & 3) : piece ^ (row & 7); }
template <typename T> __device__ __forceinline__ void fill_patch(unsigned char* patch, int row, const uint32_t (&v)[32]) {
    constexpr int V = 16 / int(sizeof(T));
    #pragma unroll
    for (int i = 0; i < kPatch / V; ++i) {
        float f[V];
        #pragma unroll
        for (int k = 0; k < V; ++k) f[k] = __uint_as_float(v[i * V + k]);
        store_floats<T, V>(reinterpret_cast<T*>(patch + row * kPatch * int(sizeof(T)) + patch_piece<T>(row, i) * 16), f);
    }
}
__device__ __forceinline__ void tma_store(const CUtensorMap* map, int column, int row, const void* from) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];\n\tcp.async.bulk.commit_group;"
                 ::"l"(map), "r"(column), "r"(row), "r"(smem_u32(from)) : "memory");
}

// After a wait that ran out: NaN in every tile that the block had a part in, so that what it left there cannot pass for a result.  The block's own stores have ended,
// and where sums are split the cluster's.
template <typename T> __device__ __noinline__ void leave_nan(T* out, int64_t out_stride, int rows_a, int rows_b, int tiles_n, int tiles, int first_tile, int tile_step,
                                                            int rows_of_tile, int row_in_tile, int columns) {
    for (int tile = first_tile; tile < tiles; tile += tile_step) {
        const int64_t row0 = int64_t(tile / tiles_n) * rows_of_tile + row_in_tile, column0 = int64_t(tile % tiles_n) * columns;
        for (int i = threadIdx.x; i < kTileRows * columns; i += kTileThreads) {
            const int64_t row = row0 + i / columns, column = column0 + i % columns;
            if (row < rows_a && column < rows_b) out[row * out_stride + column] = from_float<T>(__uint_as_float(0x7fffffffu));
        }
    }
}

// kSplit: gridDim.x = tiles * parts in clusters of `parts` blocks, one tile each; kPair: clusters of two blocks, and parts is 2; kSingle: parts is 1.
template <typename T, int BN, int MODE>
__global__ void __launch_bounds__(kTileThreads, 1) matmul_tiles_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                                                                      const __grid_constant__ CUtensorMap map_out, const TileArgs args, const int parts) {
    using S = Tile<T, BN, MODE>;
    constexpr bool SPLIT = MODE == kSplit, PAIR = MODE == kPair;
    extern __shared__ unsigned char raw[];
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    unsigned char* ring = raw + (base - smem_u32(raw));
    uint64_t* full = reinterpret_cast<uint64_t*>(ring + S::stages * S::stage_bytes + S::out_bytes + S::word_bytes);
    uint64_t* empty = full + S::stages;
    uint64_t* scale_full = empty + S::stages;
    uint64_t* scale_empty = scale_full + kScaleStages;
    uint64_t* sum_full = scale_empty + kScaleStages;
    uint64_t* sum_empty = sum_full + kAccumulators;
    uint64_t* drained = sum_empty + kAccumulators;
    uint32_t* tmem_at = reinterpret_cast<uint32_t*>(drained + 1);
    volatile uint32_t* failed = tmem_at + 1;

    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::stages; ++i) { mbar_init(full + i, 1); mbar_init(empty + i, 1); }
        for (int i = 0; i < kScaleStages; ++i) { mbar_init(scale_full + i, 4 * S::blocks); mbar_init(scale_empty + i, 1); }
        for (int i = 0; i < kAccumulators; ++i) { mbar_init(sum_full + i, 1); mbar_init(sum_empty + i, 4 * S::blocks); }
        mbar_init(drained, 1);
        *failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_at)) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_at)) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
        tmem_fence_before();
    }
    __syncthreads();
    if constexpr (PAIR) cluster_barrier();          // the other block's barriers can be reached from here on
    grid_dependency();                               // the operands may come from the kernel before
    tmem_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_at, 0);
    const uint32_t tmem_scales = tmem + kAccumulators * BN;

    const int part = MODE == kSingle ? 0 : int(blockIdx.x) % parts;
    const int first_tile = MODE == kSingle ? int(blockIdx.x) : int(blockIdx.x) / parts, tile_step = SPLIT ? args.tiles : int(gridDim.x) / parts;
    constexpr int kRowsOfTile = kTileRows * S::blocks;
    const int row_in_tile = PAIR ? part * kTileRows : 0;       // where this block's rows of a begin
    const int k_begin = SPLIT ? int(int64_t(args.blocks_k) * part / parts) : 0;
    const int k_end = SPLIT ? int(int64_t(args.blocks_k) * (part + 1) / parts) : args.blocks_k;

    if (warp == 0) {
        // The whole warp goes round the loop and one lane issues: the compiler then keeps the operands in uniform registers.  With the loop inside
        // `if (lane == 0)` each matrix instruction took 145 clocks, whatever its size.
        const bool one = elect_one();
        uint32_t uses = 0;
        const uint32_t full_there = PAIR ? peer_address(smem_u32(full), 0) : 0;
        Ring<S::stages> stage;
        bool ok = true;
        for (int tile = first_tile; ok && tile < args.tiles; tile += tile_step) {
            const int row_a = tile / args.tiles_n * kRowsOfTile + row_in_tile, row_b = tile % args.tiles_n * BN + (PAIR ? part * S::b_rows : 0);
            for (int k = k_begin; k < k_end; ++k, ++uses, stage.next()) {
                ok = __all_sync(0xffffffffu, wait_for(empty + stage.at, stage.round ^ 1, failed));
                if (!ok) break;
                unsigned char* at = ring + stage.at * S::stage_bytes;
                const uint32_t bar = PAIR ? full_there + stage.at * 8 : smem_u32(full + stage.at);
                if (one) {
                    if (!PAIR || part == 0) mbar_arrive_expect_tx(full + stage.at, S::stage_bytes * S::blocks);
                    tma_load<MODE>(at, &map_a, k * kScaleBlock, row_a, bar);
                    tma_load<MODE>(at + kTileRows * kScaleBlock, &map_b, k * kScaleBlock, row_b, bar);
                }
                __syncwarp();
            }
        }
        if (!ok && PAIR) {      // no copy may be on its way when the block ends; a pair's second block has no barrier to ask
            WaitLimit limit(20000000, nanoseconds());
            while (!limit.over(nanoseconds())) {}
        }
        if (!ok && !PAIR)
            for (uint32_t u = uses > S::stages ? uses - S::stages : 0; u < uses; ++u) {
                WaitLimit limit(kWaitNanoseconds, nanoseconds());
                while (!mbar_try_wait(full + u % S::stages, u / S::stages & 1) && !limit.over(nanoseconds())) {}
            }
    } else if (warp == 1) {
        if (!PAIR || part == 0) {
            const bool one = elect_one();
            Ring<S::stages> stage;
            Ring<kScaleStages> scale;
            Ring<kAccumulators> sum;
            const uint32_t low = operand_low(base);
            bool ok = true;
            for (int tile = first_tile; ok && tile < args.tiles; tile += tile_step, sum.next()) {
                ok = __all_sync(0xffffffffu, wait_for(sum_empty + sum.at, sum.round ^ 1, failed));
                if (!ok) break;
                tmem_fence_after();
                const uint32_t to = tmem + sum.at * BN;
                for (int k = k_begin; k < k_end; ++k, stage.next()) {
                    if (k == k_begin || (k & 3) == 0) {
                        ok = __all_sync(0xffffffffu, wait_for(scale_full + scale.at, scale.round, failed));
                        if (!ok) break;
                    }
                    ok = __all_sync(0xffffffffu, wait_for(full + stage.at, stage.round, failed));
                    if (!ok) break;
                    tmem_fence_after();
                    const uint32_t scales = tmem_scales + scale.at * kScaleColumns, instruction = kInstruction<BN, MODE> | (k & 3) << 4 | (k & 3) << 29;
                    const uint32_t a = low + stage.at * (S::stage_bytes >> 4), b = a + (kTileRows * kScaleBlock >> 4);
                    const bool last_of_scale = k + 1 == k_end || (k & 3) == 3;
                    if (one) {
                        #pragma unroll
                        for (int i = 0; i < 4; ++i)          // 32 columns each, 32 bytes further on
                            multiply<MODE>(to, a + 2 * i, b + 2 * i, instruction, scales, scales + 4, k > k_begin || i > 0);
                        tmem_commit<MODE>(empty + stage.at);
                        if (last_of_scale) tmem_commit<MODE>(scale_empty + scale.at);
                        if (k + 1 == k_end) tmem_commit<MODE>(sum_full + sum.at);
                    }
                    __syncwarp();
                    if (last_of_scale) scale.next();
                }
            }
            if (!ok && one) {
                tmem_commit<MODE>(drained);
                WaitLimit limit(kWaitNanoseconds, nanoseconds());
                while (!mbar_try_wait(drained, 0) && !limit.over(nanoseconds())) {}
            }
        }
    } else if (warp >= 4 && warp < 8) {
        const uint32_t quarter = uint32_t(warp - 4) * 32 << 16, there = PAIR ? peer_address(smem_u32(scale_full), 0) : 0;
        Ring<kScaleStages> scale;
        constexpr int kWords = 4 + (BN + 31) / 32;           // of a's rows, then of b's
        const int group_begin = k_begin >> 2, groups = ((k_end - 1) >> 2) - group_begin + 1;
        // Each warp needs all words.  Split, where the rows of a long sum lie far apart and a load takes as many lines as lanes, a warp loads a quarter of
        // them and has the rest through shared memory (1024 x 32768 by 512: 33 -> 25 us); else it loads all (8192 x 8192 by 8192: 429 us, shared 484).
        constexpr int kLoads = SPLIT ? 3 : kWords;
        uint32_t next[kLoads];
        uint32_t (*shared)[kScaleColumns][32] = reinterpret_cast<uint32_t (*)[kScaleColumns][32]>(ring + S::stages * S::stage_bytes + S::out_bytes);
        const auto load = [&](int tile, int group) {         // rows that do not exist have scale 1 (their codes are loaded as zeros)
            const int row_a = tile / args.tiles_n * kRowsOfTile + row_in_tile, row_b = tile % args.tiles_n * BN;      // of b's scales each block needs all
            #pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                const int i = SPLIT ? 4 * j + warp - 4 : j;
                const bool of_a = SPLIT ? j == 0 : j < 4;
                const int row = (of_a ? row_a + 32 * i : row_b + 32 * (i - 4)) + lane;
                const uint8_t* at = of_a ? args.scales_a + (row >> args.shift_a) * args.scales_a_stride : args.scales_b + (row >> args.shift_b) * args.scales_b_stride;
                next[j] = i < kWords && row < (of_a ? args.rows_a : args.rows_b) ? __ldg(reinterpret_cast<const uint32_t*>(at) + group) : 0x7f7f7f7fu;
            }
        };
        int tile = first_tile, group = 0, turn = 0;
        bool ok = true;
        if (tile < args.tiles) load(tile, group_begin);
        while (tile < args.tiles) {
            uint32_t words[12];
            if (SPLIT) {
                #pragma unroll
                for (int j = 0; j < kLoads; ++j) shared[turn][4 * j + warp - 4][lane] = next[j];
                __syncwarp();                // the barrier is of whole warps
                asm volatile("bar.sync 1, 128;" ::: "memory");    // one per trip: the other buffer is written before the next one
                #pragma unroll
                for (int i = 0; i < 12; ++i) words[i] = shared[turn][i][lane];
                turn ^= 1;
            } else {
                #pragma unroll
                for (int i = 0; i < 12; ++i) words[i] = i < kLoads ? next[i < kLoads ? i : 0] : 0;
            }
            if (++group == groups) { group = 0; tile += tile_step; }
            if (tile < args.tiles) load(tile, group_begin + group);          // the next four blocks' are on their way meanwhile
            // a warp whose wait ran out still goes round for the others' barrier
            ok = ok && __all_sync(0xffffffffu, wait_for(scale_empty + scale.at, scale.round ^ 1, failed));
            if (!ok) continue;
            tmem_fence_after();
            const uint32_t to = tmem_scales + scale.at * kScaleColumns + quarter;
            tmem_store4(to, words[0], words[1], words[2], words[3]);
            tmem_store4(to + 4, words[4], words[5], words[6], words[7]);
            if (BN > 128) tmem_store4(to + 8, words[8], words[9], words[10], words[11]);
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) { if (PAIR) arrive_there(there + scale.at * 8); else arrive(scale_full + scale.at); }
            scale.next();
        }
    } else if (warp >= 8) {
        const uint32_t quarter = uint32_t(warp - 8) * 32, there = PAIR ? peer_address(smem_u32(sum_empty), 0) : 0;
        Ring<kAccumulators> sum;
        unsigned char* patches = ring + S::stages * S::stage_bytes + (warp - 8) * 2 * S::patch_bytes;
        int patch_at = 0;
        for (int tile = first_tile; tile < args.tiles; tile += tile_step, sum.next()) {
            bool ok = wait_for(sum_full + sum.at, sum.round, failed);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tmem_fence_after();
            const int column0 = tile % args.tiles_n * BN, row0 = tile / args.tiles_n * kRowsOfTile + row_in_tile + int(quarter);
            #pragma unroll 1
            for (int c = 0; c < BN; c += kPatch) {
                uint32_t v[32];
                tmem_load32(tmem + sum.at * BN + c + (quarter << 16), v);
                if (SPLIT) {
                    float* to = reinterpret_cast<float*>(ring) + (quarter + lane) * S::partial_pitch + c;
                    #pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *reinterpret_cast<uint4*>(to + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                    continue;
                }
                if (row0 >= args.rows_a || column0 + c >= args.rows_b) continue;
                unsigned char* patch = patches + patch_at * S::patch_bytes;
                patch_at ^= 1;
                asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");       // the copy before the last has left this patch
                __syncwarp();
                fill_patch<T>(patch, lane, v);
                if (args.mapped) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) tma_store(&map_out, column0 + c, row0, patch);
                    __syncwarp();            // the next columns are read by the whole warp (.aligned)
                } else {                     // rows that begin anywhere: a row's 32 values by the 32 lanes
                    __syncwarp();
                    const int column = column0 + c + lane, rows = min(kPatch, args.rows_a - row0);
                    T* to = static_cast<T*>(args.out) + int64_t(row0) * args.out_stride + column;
                    constexpr int V = 16 / int(sizeof(T));
                    if (column < args.rows_b) {
                        #pragma unroll 8
                        for (int r = 0; r < rows; ++r)
                            to[r * args.out_stride] = *reinterpret_cast<const T*>(patch + r * kPatch * int(sizeof(T)) + patch_piece<T>(r, lane / V) * 16 + lane % V * int(sizeof(T)));
                    }
                    __syncwarp();
                }
            }
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) { if (PAIR) arrive_there(there + sum.at * 8); else arrive(sum_empty + sum.at); }
        }
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    __syncwarp();
    if (SPLIT) {
        cluster_barrier();
        const int rows = kTileRows / parts, column0 = first_tile % args.tiles_n * BN;
        const int64_t row0 = int64_t(first_tile / args.tiles_n) * kTileRows;
        for (int i = threadIdx.x; i < rows * (BN / 4); i += kTileThreads) {
            const int r = part * rows + i / (BN / 4), c = i % (BN / 4) * 4;
            if (row0 + r >= args.rows_a || column0 + c >= args.rows_b) continue;
            float4 v[kMostParts];
            #pragma unroll
            for (int p = 0; p < kMostParts; ++p)
                if (p < parts) v[p] = peer_float4(base + uint32_t(r * S::partial_pitch + c) * 4, p);
            float4 total = v[0];
            #pragma unroll
            for (int p = 1; p < kMostParts; ++p)
                if (p < parts) total += v[p];
            T* to = static_cast<T*>(args.out) + (row0 + r) * args.out_stride + column0 + c;
            const float f[4] = {total.x, total.y, total.z, total.w};
            if (args.mapped && column0 + c + 4 <= args.rows_b) store_floats<T, 4>(to, f);
            else {
                #pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (column0 + c + k < args.rows_b) to[k] = from_float<T>(f[k]);
            }
        }
        cluster_barrier();           // no block's shared memory goes before the others have read it
    }
    if constexpr (PAIR) cluster_barrier();      // nor a block's barriers before the other's last arrival
    __syncthreads();
    if (warp == 1) {
        tmem_fence_after();
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
    if (*failed) {
        leave_nan<T>(static_cast<T*>(args.out), args.out_stride, args.rows_a, args.rows_b, args.tiles_n, args.tiles, first_tile, tile_step, kRowsOfTile, row_in_tile, BN);
        if (threadIdx.x == 0) {
            *reinterpret_cast<volatile unsigned int*>(args.error) = 1;
            __threadfence_system();
        }
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------

bool make_map(CUtensorMap* map, CUtensorMapDataType type, CUtensorMapSwizzle swizzle, const void* base, int64_t columns, int64_t rows, int64_t stride_bytes, int box_columns,
              int box_rows) {
    const cuuint64_t sizes[2] = {cuuint64_t(columns), cuuint64_t(rows)}, strides[1] = {cuuint64_t(stride_bytes)};
    const cuuint32_t box[2] = {cuuint32_t(box_columns), cuuint32_t(box_rows)}, steps[2] = {1, 1};
    const EncodeTiled encode = encode_tiled();
    return encode && encode(map, type, 2, const_cast<void*>(base), sizes, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool make_operand_map(CUtensorMap* map, const HtgsFp8Matrix& m, int box_rows) {
    return make_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_SWIZZLE_128B, m.codes, m.width, m.rows, m.codes_stride, kScaleBlock, box_rows);
}
template <typename T> bool make_out_map(CUtensorMap* map, const MatmulArgs& m) {
    return make_map(map, sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, sizeof(T) == 4 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                    m.out, m.b.rows, m.a.rows, m.out_stride * int64_t(sizeof(T)), kPatch, kPatch);
}

ErrorWords& error_words() {
    static ErrorWords words;
    return words;
}
unsigned int* error_word(int device) { return error_words().of(device); }
int reported(unsigned int* word) { return htgs::reported(word, "htgs_fp8_matmul: a wait in an earlier product on this device ran out, and its result is not complete"); }

// parts: blocks of a cluster (kSplit), else the mode's own number.
template <typename T, int BN, int MODE> int launch_tiles(const MatmulArgs& m, int parts, cudaStream_t stream) {
    using S = Tile<T, BN, MODE>;
    unsigned int* error = error_word(current_device());
    if (!error) return sequence_fail(HTGS_ERR_CUDA, "htgs_fp8_matmul: no host memory for the error word");
    CUtensorMap map_a, map_b, map_out{};
    const bool mapped = rows_aligned(m.out, m.out_stride, 2, sizeof(T), 16);
    if (!make_operand_map(&map_a, m.a, kTileRows) || !make_operand_map(&map_b, m.b, S::b_rows) || (mapped && !make_out_map<T>(&map_out, m))) return sequence_fail(HTGS_ERR_CUDA, "htgs_fp8_matmul: the tensor maps cannot be made");
    TileArgs args{};
    args.scales_a = m.a.scales; args.scales_b = m.b.scales; args.scales_a_stride = m.a.scales_stride; args.scales_b_stride = m.b.scales_stride;
    args.rows_a = int32_t(m.a.rows); args.rows_b = int32_t(m.b.rows);
    args.shift_a = m.a.rows_per_scale == 1 ? 0 : 7; args.shift_b = m.b.rows_per_scale == 1 ? 0 : 7;
    args.blocks_k = int32_t((m.a.width + kScaleBlock - 1) / kScaleBlock);
    args.tiles_n = int32_t((m.b.rows + BN - 1) / BN);
    const int64_t tiles = (m.a.rows + kTileRows * S::blocks - 1) / (kTileRows * S::blocks) * args.tiles_n;
    if (tiles > 0x3fffffff) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_fp8_matmul: too many tiles");
    args.tiles = int32_t(tiles);
    args.out = m.out; args.out_stride = m.out_stride;
    args.mapped = mapped;
    args.error = error;
    static PerDeviceOnce once;
    cudaError_t err = once.run([] { return cudaFuncSetAttribute(matmul_tiles_kernel<T, BN, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::smem); });
    if (err != cudaSuccess) return sequence_fail(HTGS_ERR_CUDA, cudaGetErrorString(err));
    cudaLaunchConfig_t config{};
    cudaLaunchAttribute attributes[2]{};
    attributes[0].id = cudaLaunchAttributeClusterDimension;
    attributes[0].val.clusterDim.x = unsigned(parts); attributes[0].val.clusterDim.y = attributes[0].val.clusterDim.z = 1;
    attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[1].val.programmaticStreamSerializationAllowed = 1;
    config.blockDim = kTileThreads; config.dynamicSmemBytes = S::smem; config.stream = stream;
    config.attrs = attributes; config.numAttrs = 2;
    config.gridDim = MODE == kSplit ? unsigned(args.tiles) * unsigned(parts) : unsigned(args.tiles < kSms / parts ? args.tiles : kSms / parts) * unsigned(parts);
    err = cudaLaunchKernelEx(&config, matmul_tiles_kernel<T, BN, MODE>, map_a, map_b, map_out, args, parts);
    return err == cudaSuccess ? sequence_status("htgs_fp8_matmul") : sequence_fail(HTGS_ERR_CUDA, cudaGetErrorString(err));
}

template <typename T> int matmul_typed(const MatmulArgs& args, cudaStream_t stream) {
    if (args.a.rows == 1) return launch_rows<T, 1, T, false>(args, {}, stream);
    if (args.a.rows <= kMostRows) return launch_rows<T, kMostRows, T, false>(args, {}, stream);
    const auto tiles_of = [&](int rows, int columns) { return (args.a.rows + rows - 1) / rows * ((args.b.rows + columns - 1) / columns); };
    const int64_t blocks_k = (args.a.width + kScaleBlock - 1) / kScaleBlock, tiles128 = tiles_of(128, 128), tiles224 = tiles_of(128, 224);
    // Few tiles and a long sum: split it.  Joining the parts costs 2 to 3 us, ten blocks of 128 columns' worth, so a part has eight blocks at least (us, unsplit /
    // in 4 / in 8: 128 x 2048 by 2048 7.1 / 7.4 / 14.3, 100 x 4096 by 256 10.7 / 7.7 / 7.5, 1024 x 32768 by 512 65 / 25 / 25).  Sixteen clusters of eight are not on
    // the SMs at once.
    int parts = 1;
    while (parts < kMostParts && blocks_k >= 32 && blocks_k >= 16 * parts && tiles128 * parts * 2 <= (parts < 4 ? kSms : 64)) parts *= 2;
    if (parts > 1) return launch_tiles<T, 128, kSplit>(args, parts, stream);
    // Many tiles: pairs, from sixteen rounds of all SMs on, so that the last, incomplete one weighs little.  us, pairs of 224 / single blocks of 224 / of 128:
    // 8192 x 8192 by 8192 442 / 478 / 554, 100000 x 1024 by 2048 207 / 213 / 226; with fewer rounds 32768 x 512 by 1024 29 / 24 / 25, 4099 x 1080 by 1008 15 / 13 / 11.
    if (tiles_of(256, 224) >= 16 * (kSms / 2)) return launch_tiles<T, 224, kPair>(args, 2, stream);
    // Between them a tile's time goes with its width, and the tiles go in rounds of one per SM.
    if ((tiles128 + kSms - 1) / kSms * 128 <= (tiles224 + kSms - 1) / kSms * 224) return launch_tiles<T, 128, kSingle>(args, 1, stream);
    return launch_tiles<T, 224, kSingle>(args, 1, stream);
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

unsigned int* htgs_fp8_matmul_error_word(int32_t device) { return htgs::error_word(device); }

int htgs_fp8_matmul_status(int32_t device) {
    using namespace htgs;
    if (device < 0 || device >= ErrorWords::kMostDevices) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_fp8_matmul_status: no such device");
    return reported(error_word(device));
}

int htgs_fp8_matmul_values(const void* x, int64_t x_stride, int type, int64_t rows, const HtgsFp8Matrix* b, void* out, int64_t out_stride, int out_type, void* stream) {
    using namespace htgs;
    if (!matrix_ok(b) || !known_type(type) || !known_type(out_type)) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_fp8_matmul_values: bad matrix or unknown element type");
    if (rows < 0 || rows > kMostRows || rows * ((b->width + kScaleBlock - 1) / kScaleBlock * kScaleBlock) > kMostValues)
        return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_fp8_matmul_values: at most 8 rows and 32768 values (the width rounded up to 128)");
    if (rows == 0 || b->rows == 0) return HTGS_OK;
    if (b->width < 1 || !x || !out || out_stride < b->rows)
        return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_fp8_matmul_values: x and out must not be null, the width at least 1, and out's rows must hold b.rows values");
    if (const int code = reported(error_word(current_device())); code != HTGS_OK) return code;
    const HtgsFp8Matrix a{nullptr, nullptr, rows, b->width, 0, 0, 1};
    const MatmulArgs args{a, *b, out, out_stride};
    const ValuesArgs values{x, x_stride};
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (out_type == HTGS_FLOAT32) return matmul_values<float>(args, values, type, s);
    if (out_type == HTGS_FLOAT16) return matmul_values<__half>(args, values, type, s);
    return matmul_values<__nv_bfloat16>(args, values, type, s);
}

int htgs_fp8_matmul(const HtgsFp8Matrix* a, const HtgsFp8Matrix* b, void* out, int64_t out_stride, int out_type, void* stream) {
    using namespace htgs;
    if (!matrix_ok(a) || !matrix_ok(b))
        return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_fp8_matmul: matrices need sizes below 2^31 - 256, codes on 16 bytes, scales on 4 bytes, rows_per_scale 1 or 128");
    if (a->width != b->width) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_fp8_matmul: a and b must have the same width");
    if (!known_type(out_type)) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_fp8_matmul: unknown element type");
    if (a->rows == 0 || b->rows == 0) return HTGS_OK;
    if (!out || out_stride < b->rows) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_fp8_matmul: out must not be null, and its rows must hold b.rows values");
    if (const int code = reported(error_word(current_device())); code != HTGS_OK) return code;
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
