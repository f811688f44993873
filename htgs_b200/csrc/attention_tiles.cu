// Attention over packed sequences on the tensor cores (tcgen05): 16-bit values, heads of 8, 16, ... 128 values, rows and heads that begin on 16 bytes.
//
// Tiles are 128 rows by 128 rows.  Operands come by TMA into shared memory as panels of 64 columns under the 128-byte swizzle: [128 rows][128 bytes], which serve as they lie both for
// products along the columns (q k^T) and along the rows (P v, where a panel is a transposed operand).  Scores, weights (over the scores, in the type) and outputs stay in tensor memory.
#include "attention.cuh"

namespace htgs {

namespace {

constexpr int kTile = 128, kPanel = 64, kPanelBytes = kTile * kPanel * 2;
constexpr int kTilesThreads = 384;
constexpr uint32_t kPanelUnits = kPanelBytes >> 4;

// Operand descriptors.  The upper word is the same for all: groups of 8 rows 1024 bytes apart, 128-byte swizzle.  Lower word, along the columns: the address (the leading offset says
// nothing); along the rows: the address and the distance from panel to panel.
constexpr uint32_t kPanelHigh = 1024 >> 4 | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t along_columns(uint32_t address) { return (address & 0x3ffffu) >> 4 | 1u << 16; }
__device__ __forceinline__ uint32_t along_rows(uint32_t address) { return (address & 0x3ffffu) >> 4 | kPanelUnits << 16; }
// 32-bit sums of products of T; the second operand along its rows or columns.
template <typename T> __device__ __forceinline__ uint32_t instruction(int columns, bool second_along_rows) {
    constexpr uint32_t format = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return 1u << 4 | format << 7 | format << 10 | uint32_t(second_along_rows) << 16 | uint32_t(columns >> 3) << 17 | uint32_t(kTile >> 4) << 24;
}
__device__ __forceinline__ void multiply(uint32_t d, uint32_t a, uint32_t b, uint32_t instruction, uint32_t add) {                 // a in shared memory
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "r"(b), "r"(instruction), "r"(add), "n"(kPanelHigh) : "memory");
}
__device__ __forceinline__ void multiply_tmem(uint32_t d, uint32_t a, uint32_t b, uint32_t instruction, uint32_t add) {            // a in tensor memory
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 db, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "r"(b), "r"(instruction), "r"(add), "n"(kPanelHigh) : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void load_panel(void* to, const CUtensorMap* map, int column, int head, int row, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(smem_u32(to)), "l"(map), "r"(column), "r"(head), "r"(row), "r"(smem_u32(bar)) : "memory");
}
// 32 columns of a lane's row; begun, and all done.
__device__ __forceinline__ void tmem_begin32(uint32_t address, uint32_t* v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
                   "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]),
                   "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(address));
}
__device__ __forceinline__ void tmem_begin16(uint32_t address, uint32_t* v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
                   "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(address));
}
__device__ __forceinline__ void tmem_loaded() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_store16(uint32_t address, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 ::"r"(address), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]),
                   "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t address, const uint32_t (&v)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
                 "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
                 ::"r"(address), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]),
                 "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]),
                 "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31]) : "memory");
}
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ---- pieces of work ----------------------------------------------------------------------------------------------------------------
// The grid has a block for each piece.  A block that runs takes further ones from those that have not begun (clusterlaunchcontrol), so long and short pieces spread by themselves, and its roles go on from
// one to the next without the 9000 clocks that a block needs on its way in and out.
constexpr int kRecent = 8;
struct PieceShared { uint4 response[2]; uint64_t come[2]; int recent[kRecent]; };      // recent: what a failed wait may have left incomplete

// One warp's.  A request is made a piece ahead.
struct Pieces {
    PieceShared* shared;
    volatile uint32_t* failed;
    uint32_t asked = 0, got = 0, taken = 0;
    bool one;
    __device__ __forceinline__ void note(int piece) {
        if (one) shared->recent[taken % kRecent] = piece;
        ++taken;
    }
    __device__ __forceinline__ void ask() {
        if (one) {
            uint64_t* const bar = shared->come + (asked & 1);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_arrive_expect_tx(bar, 16);
            asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(smem_u32(shared->response + (asked & 1))), "r"(smem_u32(bar)) : "memory");
        }
        __syncwarp();
        ++asked;
    }
    __device__ __forceinline__ int first() {
        note(int(blockIdx.x));
        ask();
        return int(blockIdx.x);
    }
    // The piece asked for last, and -1 if there is none or the answer does not come.
    __device__ __forceinline__ int next() {
        if (!__all_sync(0xffffffffu, wait_in_line(shared->come + (got & 1), got >> 1 & 1, failed))) return -1;
        const uint32_t at = smem_u32(shared->response + (got & 1));
        uint32_t there, piece;
        asm volatile("{\n\t.reg .b128 r;\n\t.reg .pred p;\n\tld.shared.b128 r, [%2];\n\tclusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\tselp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
                     "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t}" : "=r"(there), "=r"(piece) : "r"(at) : "memory");
        ++got;
        if (!there) return -1;
        note(int(piece));
        return int(piece);
    }
    __device__ __forceinline__ int following() {
        const int piece = next();
        if (piece >= 0) ask();
        return piece;
    }
    // After a failure: an answer that is on its way is still a piece that nobody else will do.
    __device__ __forceinline__ void finish() {
        WaitLimit limit(kWaitNanoseconds, nanoseconds());
        while (got < asked) {
            if (mbar_try_wait(shared->come + (got & 1), got >> 1 & 1)) { next(); break; }
            if (limit.over(nanoseconds())) break;
        }
    }
};

// ---- values that are not finite ------------------------------------------------------------------------------------------------
// A weight of zero takes a finite value out of a sum, not an infinite one or a NaN.  So in tiles where not every row sees every other the operand is looked through before it is used, by warps that have
// nothing else to do, and where something is not finite a thread adds up what its row sees itself (some 50 us a tile).  Nothing of this costs the other tiles anything.

// Whether so much of a tile holds such values; by a warp.
template <typename T, int BYTES> __device__ __forceinline__ bool not_finite(const unsigned char* tile, int lane) {
    using Two = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const uint32_t zero = 0;
    Two sum = *reinterpret_cast<const Two*>(&zero);
    #pragma unroll 4
    for (int i = lane; i < BYTES / 16; i += 32) {
        const uint4 piece = *reinterpret_cast<const uint4*>(tile + i * 16);
        const Two* v = reinterpret_cast<const Two*>(&piece);
        #pragma unroll
        for (int k = 0; k < 4; ++k) sum = __hfma2(v[k], *reinterpret_cast<const Two*>(&zero), sum);          // NaN from then on
    }
    const float2 both = pair_floats<T>(*reinterpret_cast<const uint32_t*>(&sum));
    return __any_sync(0xffffffffu, both.x != 0.0f || both.y != 0.0f);
}
// Columns [from, to) of a lane's row of sums in tensor memory: plus (add), or set to, its weights times the rows [low, high] of a tile.  Weights: words of two, 64 at `weights`, 64 at weights + second.
template <typename T> __device__ __forceinline__ void multiply_seen(uint32_t sums, int from, int to, bool add, uint32_t weights, uint32_t second, const unsigned char* tile, int low, int high, int blocks = 4) {
    #pragma unroll 1
    for (int c = from; c < to; c += 16) {
        uint32_t o[16] = {};
        if (add) {
            tmem_begin16(sums + c, o);
            tmem_loaded();
        }
        #pragma unroll 1
        for (int block = 0; block < blocks; ++block) {
            uint32_t w[16];
            tmem_begin16(weights + (block >> 1) * second + (block & 1) * 16, w);
            tmem_loaded();
            #pragma unroll
            for (int k = 0; k < 32; ++k) {
                const int row = block * 32 + k;
                if (row < low || row > high) continue;
                const float2 pair = pair_floats<T>(w[k / 2]);
                const float weight = k & 1 ? pair.y : pair.x;
                const unsigned char* at = tile + (c >> 6) * kPanelBytes + row * 128;
                #pragma unroll
                for (int piece = 0; piece < 2; ++piece) {
                    float v[8];
                    load_floats<T, 8>(reinterpret_cast<const T*>(at + (((c >> 3 & 7) + piece) ^ (row & 7)) * 16), v);
                    #pragma unroll
                    for (int i = 0; i < 8; ++i) o[piece * 8 + i] = __float_as_uint(fmaf(weight, v[i], __uint_as_float(o[piece * 8 + i])));
                }
            }
            __syncwarp();
        }
        tmem_store16(sums + c, o);
    }
    tmem_stored();
}

// ---- forward -------------------------------------------------------------------------------------------------------------------

// NaN if one of them is.
__device__ __forceinline__ float largest3(float a, float b, float c) { float d; asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c)); return d; }
__device__ __forceinline__ float largest2(float a, float b) { float d; asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b)); return d; }

__device__ __forceinline__ f32x2 exp2_pair(f32x2 x) {
    const float2 v = unpack2(x);
    return pack2(exp2_approx(v.x), exp2_approx(v.y));
}
// 2^x = 2^n 2^r with n = x rounded (by adding 1.5 * 2^23, whose low bits then are n) and -1/2 <= r <= 1/2, where 2^r is a polynomial, 1 at 0, of least maximal relative error (found by linear programming):
// degree 3 for bf16, 2^-13.2, and 4 for fp16, 2^-18.4, both far below half a step of the type.  From x = -127 down it is exactly zero.  NaN is for the caller to keep out.
//
// The unit for exponentials makes 16 a clock and SM, 1024 clocks for a tile, as long as the products of heads of 128 and twice as long as those of 64.  Four pairs of 16 go this way instead, through
// multiply-adds that would idle (16384 rows, causal, heads of 64: 460 -> 425 us; more of them, or a second copy of the loop without them, cost more in instructions than they give).
constexpr int kPolynomials = 4;
template <typename T> __device__ __forceinline__ f32x2 exp2_polynomial(f32x2 x) {
    constexpr bool kHalf = std::is_same<T, __half>::value;
    const float2 v = unpack2(x);
    x = pack2(fmaxf(v.x, -127.0f), fmaxf(v.y, -127.0f));
    const f32x2 magic = pack2(12582912.0f, 12582912.0f), back = pack2(-12582912.0f, -12582912.0f), minus = pack2(-1.0f, -1.0f);
    const f32x2 n = add2(x, magic), r = fma2(add2(n, back), minus, x);
    const auto both = [](float c) { return pack2(c, c); };
    f32x2 p = kHalf ? fma2(both(0.009582853876054287f), r, both(0.055906426161527634f)) : both(0.05500892922282219f);
    p = fma2(p, r, both(kHalf ? 0.24024099111557007f : 0.24221095442771912f));
    p = fma2(p, r, both(kHalf ? 0.6931241750717163f : 0.6932829022407532f));
    p = fma2(p, r, both(1.0f));
    const float2 low = unpack2(p), whole = unpack2(n);
    return pack2(__uint_as_float(__float_as_uint(low.x) + (__float_as_uint(whole.x) << 23)), __uint_as_float(__float_as_uint(low.y) + (__float_as_uint(whole.y) << 23)));
}

// What an exponent may pass the running maximum by before the output is scaled down to a new one: weights up to 2^8 are as precise as those up to 1, and most tiles then leave the output alone.
// (What is lost is that the largest weight is a power of two, which is not rounded: the output is off by 0.0023 of its size in bf16, where 0.0019 would be possible and its own rounding is 0.0017; a scaling at each new maximum costs 10 % for heads of
// 64 and up to 30 % for those of 128.  In training with heads of more than 64 it is done all the same: the gradients of q and k, which the output's error reaches through D, have their score gradients rounded once more.)
constexpr float kSlack = 8.0f;
// Powers of two that weights carry.  fp16: 2^6, so that one of 2^-20 of the row's largest is a normal number (and the largest is 2^14); sums of such values are far from the end of 32 bits.  bf16, whose
// values reach as far as 32 bits do: so little that the weights of n tiles of keys, 2^8 each at most, add up to a half at most, and no sum of values passes the largest of them.  (Without it 1.3e36, or a
// thousand times 4e35, became infinite.  Exponents lose their last bits by it, 2^-19 of a weight.  By the piece's own tiles, so that a sequence gets the same bits whatever it is packed with.)
template <typename T> __device__ __forceinline__ float lift_of(int n) { return std::is_same<T, __half>::value ? 6.0f : -(kSlack + 1.0f + float(bits_of(n * kTile))); }

constexpr int kItems = 2;            // pieces of work that a block knows of: the present one and the next

// QUERIES: tiles of queries of a block.  Two have an SM and its tensor memory alone, one shares it with another block.
template <int PANELS, int QUERIES> struct ForwardTile {
    static constexpr int threads = 128 + 128 * QUERIES, blocks = 3 - QUERIES, columns = 512 / blocks;      // of an SM; of tensor memory
    static constexpr int bytes = PANELS * kPanelBytes, stages = 5;
    static constexpr bool apart = PANELS == 1 && QUERIES == 1;       // weights have columns of their own
    static constexpr int weights = apart ? kTile : 0, outputs = apart ? kTile + kTile / 2 : QUERIES * kTile;     // where they begin; another tile's 128 further
    static constexpr int barriers = 2 * kItems + 3 * stages + 7 * QUERIES;
    static constexpr int smem = 1024 + (QUERIES + stages) * bytes + 1024;
    static_assert(barriers * 8 + 8 + stages * 4 + kItems * 24 + 16 + int(sizeof(PieceShared)) <= 1024 && smem <= 227 * 1024 / blocks - (blocks - 1) * 1024 && smem * (blocks + 1) > 227 * 1024, "shared memory");
    static_assert(smem >= kLeastTensorShared && columns * blocks <= 512, "tensor memory");
};
// Registers of the warps that compute, and of the others; together those of the launch.
template <int GROUPS> __device__ __forceinline__ void take_registers() {
    if constexpr (GROUPS == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
}
template <int GROUPS> __device__ __forceinline__ void give_registers() {
    if constexpr (GROUPS == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
}

struct ForwardArgs { HtgsAttention a; void* out; void* rest; float* sums; unsigned int* error; };

// A piece is a head and one or two tiles of queries, one behind the other, against tiles of keys.  Warp 0 finds the pieces and loads; warps 1 and 2 issue the products, for one tile of queries while the other's softmax (or the other block's) is
// computed, and the next piece's first scores while the last one's output is stored; warp 3 looks through values of which some are not seen; warps 4 to 7 and 8 to 11 have a tile of queries each, a thread
// for each row.  Tensor memory of two tiles: scores (weights over them) at 0 and 128, outputs at 256 and 384.  Of one, up to 64 columns wide: scores 0, weights 128, output 192; the next scores are
// computed as soon as the softmax has read the last ones.
template <typename T, int PANELS, int QUERIES>
__global__ void __launch_bounds__(128 + 128 * QUERIES, 3 - QUERIES) attention_tiles_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                                                          const __grid_constant__ CUtensorMap map_v, const __grid_constant__ ForwardArgs args) {
    using S = ForwardTile<PANELS, QUERIES>;
    extern __shared__ unsigned char raw[];
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    unsigned char* const queries = raw + (base - smem_u32(raw));
    unsigned char* const ring = queries + QUERIES * S::bytes;
    uint64_t* const item_full = reinterpret_cast<uint64_t*>(ring + S::stages * S::bytes);
    uint64_t* const item_empty = item_full + kItems;
    uint64_t* const full = item_empty + kItems;
    uint64_t* const empty = full + S::stages;
    uint64_t* const searched = empty + S::stages;        // values have been looked through
    uint64_t* const q_full = searched + S::stages;
    uint64_t* const q_empty = q_full + QUERIES;
    uint64_t* const scored = q_empty + QUERIES;          // the scores of a tile are there
    uint64_t* const weighed = scored + QUERIES;          // its weights are
    uint64_t* const summed = weighed + QUERIES;          // they are in the output
    uint64_t* const taken = summed + QUERIES;            // the scores have been read (weights apart)
    uint64_t* const drained = taken + QUERIES;           // the output has been read
    uint32_t* const tmem_at = reinterpret_cast<uint32_t*>(drained + QUERIES);
    volatile uint32_t* const failed = tmem_at + 1;
    volatile uint32_t* const dirty = failed + 1;         // [stages], of tiles of values
    volatile int* const items = reinterpret_cast<volatile int*>(dirty + S::stages);        // [kItems] of 6 words
    PieceShared* const shared = reinterpret_cast<PieceShared*>((reinterpret_cast<uintptr_t>(items + kItems * 6) + 15) & ~uintptr_t(15));

    const HtgsAttention& a = args.a;
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31, group = a.heads / a.key_heads;
    T* const out = static_cast<T*>(args.out);
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) mbar_init(shared->come + i, 1);
        for (int i = 0; i < kRecent; ++i) shared->recent[i] = -1;
        for (int i = 0; i < kItems; ++i) { mbar_init(item_full + i, 1); mbar_init(item_empty + i, (S::apart ? 2 : 1) + 1 + 4 * QUERIES); }
        for (int i = 0; i < QUERIES; ++i) {
            mbar_init(q_full + i, 1); mbar_init(q_empty + i, 1); mbar_init(scored + i, 1); mbar_init(weighed + i, 4); mbar_init(summed + i, 1); mbar_init(taken + i, 4); mbar_init(drained + i, 4);
        }
        for (int i = 0; i < S::stages; ++i) { mbar_init(full + i, 1); mbar_init(empty + i, 2); mbar_init(searched + i, 1); }
        *failed = 0;
        mbar_fence_init();
    }
    grid_dependency();               // before tensor memory is taken, which a block of the kernel before may still have to get
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_at)), "n"(S::columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tmem_fence_before();
    }
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_at, 0);
    const int total = int(gridDim.x);
    // Piece `item`: the last tiles of a sequence first, as they have the most keys where attention is causal.
    const auto tile_of = [&](int item) { return find_tile<QUERIES * kTile>(a, (total - 1 - item) / a.heads); };
    const auto head_of = [&](int item) { return item % a.heads; };

    // What the roles know of a piece: keys low + [0, 128 n) for the block; tile s of queries sees tiles [from(s), to(s)) of them.
    struct Piece {
        const HtgsAttention& a;
        int begin, end, first, head, low, n;
        __device__ Piece(const HtgsAttention& a_) : a(a_), n(0) {}
        __device__ void set(int begin_, int end_, int first_, int head_) {
            begin = begin_; end = end_; first = first_; head = head_;
            low = first_seen(a, begin, first);
            n = (last_seen(a, end, min(first + QUERIES * kTile, end) - 1) - low) / kTile + 1;
        }
        __device__ int from(int s) const { return QUERIES == 1 ? 0 : first + s * kTile < end ? (first_seen(a, begin, first + s * kTile) - low) / kTile : 0; }
        __device__ int to(int s) const { return QUERIES == 1 ? n : first + s * kTile < end ? (last_seen(a, end, min(first + (s + 1) * kTile, end) - 1) - low) / kTile + 1 : 0; }
        // tiles [x, y) of keys are seen by all rows of tile s
        __device__ int2 whole(int s) const {
            const int row = first + s * kTile;
            return make_int2((first_seen(a, begin, min(row + kTile, end) - 1) - low + kTile - 1) / kTile, (last_seen(a, end, min(row, end - 1)) - low + 1) / kTile);
        }
    };
    // The next piece, for a warp of a role that is not the loading one; false behind the last.
    Ring<kItems> item_at;
    Piece piece(a);
    const auto next_piece = [&] {
        if (!__all_sync(0xffffffffu, wait_in_line(item_full + item_at.at, item_at.round, failed))) return false;
        volatile int* const from = items + 6 * item_at.at;
        const bool there = from[4];
        if (there) piece.set(from[0], from[1], from[2], from[3]);
        __syncwarp();
        if (lane == 0) arrive(item_empty + item_at.at);
        item_at.next();
        return there;
    };

    if (warp < 4) {
        give_registers<QUERIES>();
        if (warp == 0) {
            const bool one = elect_one();
            Ring<S::stages> stage;
            uint32_t uses = 0, loads[QUERIES] = {};
            bool ok = true;
            const auto wait = [&](uint64_t* bar, uint32_t parity) { ok = ok && __all_sync(0xffffffffu, wait_in_line(bar, parity, failed)); };
            const auto publish = [&](const SequenceTile& t, int head, int there) {
                wait(item_empty + item_at.at, item_at.round ^ 1);
                if (!ok) return;
                if (lane == 0) {
                    volatile int* const to = items + 6 * item_at.at;
                    to[0] = t.begin; to[1] = t.end; to[2] = t.first; to[3] = head; to[4] = there;
                    arrive(item_full + item_at.at);
                }
                __syncwarp();
                item_at.next();
            };
            Pieces pieces{shared, failed};
            pieces.one = one;
            for (int item = pieces.first(); item >= 0 && ok; item = pieces.following()) {
                const SequenceTile t = tile_of(item);
                if (t.first >= t.end) continue;
                const int head = head_of(item);
                if (t.outside) {
                    const int rows = min(QUERIES * kTile, t.end - t.first), pieces = a.width / 8;
                    for (int i = lane; i < rows * pieces; i += 32)
                        *reinterpret_cast<uint4*>(out + (int64_t(t.first + i / pieces) * a.heads + head) * a.width + i % pieces * 8) = make_uint4(0, 0, 0, 0);
                    for (int i = lane; i < rows && args.sums; i += 32) args.sums[head * a.rows + t.first + i] = 0.0f;
                    __syncwarp();
                    continue;
                }
                publish(t, head, 1);
                piece.set(t.begin, t.end, t.first, head);
                #pragma unroll
                for (int s = 0; s < QUERIES; ++s) {
                    if (piece.to(s) == 0) continue;
                    wait(q_empty + s, (loads[s] & 1) ^ 1);
                    if (!ok) break;
                    ++loads[s];
                    if (one) {
                        mbar_arrive_expect_tx(q_full + s, S::bytes);
                        for (int p = 0; p < PANELS; ++p) load_panel(queries + s * S::bytes + p * kPanelBytes, &map_q, p * kPanel, head, t.first + s * kTile, q_full + s);
                    }
                    __syncwarp();
                }
                for (int i = 0; i < 2 * piece.n && ok; ++i) {           // keys and values of a tile by turns
                    wait(empty + stage.at, stage.round ^ 1);
                    if (!ok) break;
                    if (one) {
                        mbar_arrive_expect_tx(full + stage.at, S::bytes);
                        for (int p = 0; p < PANELS; ++p) load_panel(ring + stage.at * S::bytes + p * kPanelBytes, i & 1 ? &map_v : &map_k, p * kPanel, head / group, piece.low + (i >> 1) * kTile, full + stage.at);
                    }
                    __syncwarp();
                    ++uses;
                    stage.next();
                }
            }
            ok = ok && !*failed;
            if (ok) publish({0, 0, 0, 0, false}, 0, 0);
            if (!ok) {              // no copy may be on its way when the block ends
                pieces.finish();
                for (uint32_t u = uses > S::stages ? uses - S::stages : 0; u < uses; ++u) {
                    WaitLimit limit(kWaitNanoseconds, nanoseconds());
                    while (!mbar_try_wait(full + u % S::stages, u / S::stages & 1) && !limit.over(nanoseconds())) {}
                }
                for (int s = 0; s < QUERIES; ++s) {
                    WaitLimit limit(kWaitNanoseconds, nanoseconds());
                    while (loads[s] && !mbar_try_wait(q_full + s, (loads[s] - 1) & 1) && !limit.over(nanoseconds())) {}
                }
            }
        } else if (warp == 1 || (S::apart && warp == 2)) {
            const bool one = elect_one();
            const uint32_t score = instruction<T>(kTile, false), weigh = instruction<T>((a.width + 15) & ~15, true);
            const int steps = (a.width + 15) / 16;
            Ring<S::stages> stage;
            int2 all[QUERIES] = {};
            uint32_t scores_done[QUERIES] = {}, outputs_done[QUERIES] = {}, pieces_done[QUERIES] = {};            // so far, whose lowest bits are the parities
            bool ok = true;
            const auto wait = [&](uint64_t* bar, uint32_t parity) { ok = ok && __all_sync(0xffffffffu, wait_in_line(bar, parity, failed)); };
            // scores of tile s of queries; the piece's last free the place of the queries
            const auto scores = [&](int s, bool last) {
                const uint32_t q = along_columns(base + s * S::bytes), k = along_columns(base + QUERIES * S::bytes + stage.at * S::bytes);
                if (one) {
                    for (int i = 0; i < steps; ++i) {
                        const uint32_t at = (i >> 2) * kPanelUnits + (i & 3) * 2;
                        multiply(tmem + s * kTile, q + at, k + at, score, i > 0);
                    }
                    commit(scored + s);
                    if (last) commit(q_empty + s);
                }
                __syncwarp();
            };
            const auto outputs = [&](int s, int j, bool first, uint32_t slot) {
                const bool added = (j < all[s].x || j >= all[s].y) && dirty[slot];       // by the softmax's threads
                const uint32_t v = along_rows(base + QUERIES * S::bytes + slot * S::bytes);
                if (one) {
                    #pragma unroll
                    for (int i = 0; i < (added ? 0 : kTile / 16); ++i) multiply_tmem(tmem + S::outputs + s * kTile, tmem + S::weights + s * kTile + i * 8, v + i * (2048 >> 4), weigh, !first || i > 0);
                    commit(summed + s);
                }
                __syncwarp();
            };
            const auto used = [&](uint32_t slot) {
                if (one) commit(empty + slot);
                __syncwarp();
            };
            if (S::apart && warp == 2) stage.next();
            while (ok && next_piece()) {
                const int n = piece.n;
                #pragma unroll
                for (int s = 0; s < QUERIES; ++s) all[s] = piece.whole(s);
                if constexpr (S::apart) {             // one warp has the scores, the other the output
                    if (warp == 1) wait(q_full, pieces_done[0] & 1);
                    else wait(drained, (pieces_done[0] & 1) ^ 1);
                    ++pieces_done[0];
                    for (int j = 0; j < n && ok; ++j) {
                        wait(full + stage.at, stage.round);
                        if (warp == 1) wait(taken, (scores_done[0] & 1) ^ 1);
                        else wait(weighed, outputs_done[0] & 1);
                        if (!ok) break;
                        tmem_fence_after();
                        if (warp == 1) { scores(0, j + 1 == n); ++scores_done[0]; }
                        else { outputs(0, j, j == 0, stage.at); ++outputs_done[0]; }
                        used(stage.at);
                        stage.next(); stage.next();
                    }
                } else {                              // by turns: two warps would take the tensor cores from each other (32768 rows, causal, heads of 128: 1.73 -> 2.08 ms)
                    int from[QUERIES], to[QUERIES];
                    #pragma unroll
                    for (int s = 0; s < QUERIES; ++s) { from[s] = piece.from(s); to[s] = piece.to(s); }
                    for (int j = -1; j < n && ok; ++j) {              // the output's part of tile j, then the scores of tile j + 1
                        uint32_t value_slot = 0;
                        if (j >= 0) {
                            wait(full + stage.at, stage.round);
                            value_slot = stage.at;
                            stage.next();
                        }
                        if (j + 1 < n) wait(full + stage.at, stage.round);
                        #pragma unroll
                        for (int s = 0; s < QUERIES; ++s) {
                            if (j >= from[s] && j < to[s]) {
                                if (j == from[s]) wait(drained + s, pieces_done[s] & 1);        // pieces_done counts the present one
                                wait(weighed + s, outputs_done[s] & 1);
                                if (!ok) break;
                                ++outputs_done[s];
                                tmem_fence_after();
                                outputs(s, j, j == from[s], value_slot);
                            }
                            if (j + 1 >= from[s] && j + 1 < to[s]) {
                                if (j + 1 == from[s]) wait(q_full + s, pieces_done[s]++ & 1);
                                if (!ok) break;
                                tmem_fence_after();
                                scores(s, j + 2 == to[s]);
                            }
                        }
                        if (!ok) break;
                        if (j >= 0) used(value_slot);
                        if (j + 1 < n) {
                            used(stage.at);
                            stage.next();
                        }
                    }
                }
            }
        } else if (warp == 3) {
            Ring<S::stages> stage;
            bool ok = true;
            while (ok && next_piece()) {
                int2 all[QUERIES], any[QUERIES];
                #pragma unroll
                for (int s = 0; s < QUERIES; ++s) { all[s] = piece.whole(s); any[s] = make_int2(piece.from(s), piece.to(s)); }
                for (int i = 0; i < 2 * piece.n && ok; ++i, stage.next()) {
                    ok = __all_sync(0xffffffffu, wait_in_line(full + stage.at, stage.round, failed));
                    if (!ok) break;
                    const int j = i >> 1;
                    bool seen = true;
                    #pragma unroll
                    for (int s = 0; s < QUERIES; ++s) seen = seen && (!(i & 1) || j < any[s].x || j >= any[s].y || (j >= all[s].x && j < all[s].y));
                    const bool found = !seen && not_finite<T, S::bytes>(ring + stage.at * S::bytes, lane);
                    if (lane == 0) {
                        dirty[stage.at] = found;
                        arrive(searched + stage.at);
                        arrive(empty + stage.at);
                    }
                    __syncwarp();
                }
            }
        }
    } else {
        take_registers<QUERIES>();
        const int s = (warp >> 2) - 1, quarter = (warp & 3) * 32;
        const uint32_t lanes = uint32_t(quarter) << 16, score = tmem + s * kTile + lanes, weights = score + S::weights, sum_at = tmem + S::outputs + s * kTile + lanes;
        const float scale = a.scale * kLog2e;
        const f32x2 scale2 = pack2(scale, scale);
        const float slack = PANELS == 2 && args.rest ? 0.0f : kSlack;
        uint32_t tiles_done = 0, uses = 0;                     // so far: of this tile of queries; places of the ring, by the block
        bool ok = true;
        while (ok && next_piece()) {
            const int first = piece.first + s * kTile, row = min(first + quarter + lane, piece.end - 1);
            const bool there = first + quarter + lane < piece.end;
            const int row_low = first_seen(a, piece.begin, row), row_high = last_seen(a, piece.end, row);
            const int from = piece.from(s), to = piece.to(s);
            const int2 all = piece.whole(s);
            const float lift = lift_of<T>(piece.n);
            float most = -infinity();
            f32x2 total2 = pack2(0.0f, 0.0f);
            for (int j = from; j < to; ++j, ++tiles_done) {
                ok = __all_sync(0xffffffffu, wait_in_line(scored + s, tiles_done & 1, failed));
                if (!ok) break;
                const bool used = S::apart && j > from && __all_sync(0xffffffffu, mbar_test(summed + s, (tiles_done - 1) & 1));      // the last tile's weights: asked here, where nothing waits for it
                tmem_fence_after();              // behind both: what the last tile's product read is written over too
                uint32_t v[128];
                tmem_begin32(score, v);
                tmem_begin32(score + 32, v + 32);
                tmem_loaded();
                tmem_begin32(score + 64, v + 64);
                tmem_begin32(score + 96, v + 96);
                float m[8];
                #pragma unroll
                for (int i = 0; i < 8; ++i) m[i] = __uint_as_float(v[i]);
                const int from_column = row_low - (piece.low + j * kTile), to_column = row_high - (piece.low + j * kTile);
                const bool masked = j < all.x || j >= all.y;
                if (masked) {
                    #pragma unroll
                    for (int c = 0; c < 64; ++c) v[c] = c < from_column || c > to_column ? 0xff800000u : v[c];
                    #pragma unroll
                    for (int i = 0; i < 8; ++i) m[i] = __uint_as_float(v[i]);
                }
                #pragma unroll
                for (int c = 8; c < 56; c += 16)
                    #pragma unroll
                    for (int i = 0; i < 8; ++i) m[i] = largest3(m[i], __uint_as_float(v[c + i]), __uint_as_float(v[c + 8 + i]));
                tmem_loaded();
                if constexpr (S::apart) {
                    tmem_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive(taken + s);
                }
                if (masked) {
                    #pragma unroll
                    for (int c = 64; c < 128; ++c) v[c] = c < from_column || c > to_column ? 0xff800000u : v[c];
                }
                #pragma unroll
                for (int c = 56; c < 120; c += 16)
                    #pragma unroll
                    for (int i = 0; i < 8; ++i) m[i] = largest3(m[i], __uint_as_float(v[c + i]), __uint_as_float(v[c + 8 + i]));
                #pragma unroll
                for (int i = 0; i < 8; ++i) m[i] = largest2(m[i], __uint_as_float(v[120 + i]));
                const float tile_most = largest3(largest3(m[0], m[1], m[2]), largest3(m[3], m[4], m[5]), largest2(m[6], m[7])) * scale;
                if (__any_sync(0xffffffffu, !(tile_most <= most + slack))) {
                    float now = largest2(most, tile_most);           // NaN makes the row's weights NaN, and so does infinity, which could only be taken from itself
                    now = now == infinity() ? __uint_as_float(0x7fffffffu) : now;
                    const float factor = most == now ? 1.0f : exp2_approx(most - now);
                    most = now;
                    total2 = mul2(total2, pack2(factor, factor));
                    if (j > from) {
                        ok = __all_sync(0xffffffffu, wait_in_line(summed + s, (tiles_done - 1) & 1, failed));
                        if (!ok) break;
                        tmem_fence_after();
                        #pragma unroll 1
                        for (int c = 0; c < a.width; c += 16) {
                            uint32_t o[16];
                            tmem_begin16(sum_at + c, o);
                            tmem_loaded();
                            #pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
                            tmem_store16(sum_at + c, o);
                        }
                        tmem_stored();
                    }
                }
                const float shift = lift - (most == -infinity() ? 0.0f : most);
                const f32x2 shift2 = pack2(shift, shift);
                f32x2 sums[2] = {total2, pack2(0.0f, 0.0f)};
                #pragma unroll
                for (int c = 0; c < 128; c += 32) {
                    uint32_t words[16];
                    #pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const f32x2 x = fma2(pack2(__uint_as_float(v[c + 2 * i]), __uint_as_float(v[c + 2 * i + 1])), scale2, shift2);
                        const f32x2 p = i * kPolynomials / 16 != (i + 1) * kPolynomials / 16 ? exp2_polynomial<T>(x) : exp2_pair(x);
                        sums[i & 1] = add2(sums[i & 1], p);
                        const float2 both = unpack2(p);
                        words[i] = floats_pair<T>(both.x, both.y);
                    }
                    if constexpr (S::apart) {
                        if (c == 0 && j > from && !used) {
                            ok = __all_sync(0xffffffffu, wait_in_line(summed + s, (tiles_done - 1) & 1, failed));
                            tmem_fence_after();
                        }
                    }
                    tmem_store16(weights + c / 2, words);
                }
                if (S::apart && !ok) break;
                total2 = add2(sums[0], sums[1]);
                tmem_stored();
                if (masked) {
                    const uint32_t use = uses + 2 * j + 1, at = use % S::stages, round = use / S::stages & 1;
                    ok = __all_sync(0xffffffffu, wait_in_line(searched + at, round, failed));
                    if (!ok) break;
                    if (dirty[at]) {
                        ok = __all_sync(0xffffffffu, wait_in_line(full + at, round, failed));
                        if (ok && j > from) ok = __all_sync(0xffffffffu, wait_in_line(summed + s, (tiles_done - 1) & 1, failed));
                        if (!ok) break;
                        tmem_fence_after();
                        multiply_seen<T>(sum_at, 0, a.width, j > from, weights, 32, ring + at * S::bytes, from_column, to_column);
                    }
                }
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) arrive(weighed + s);
            }
            uses += 2 * piece.n;
            if (!ok || to <= from) continue;
            ok = __all_sync(0xffffffffu, wait_in_line(summed + s, (tiles_done - 1) & 1, failed));
            if (!ok) break;
            tmem_fence_after();
            const float2 parts = unpack2(total2);
            const float sum = parts.x + parts.y, inverse = 1.0f / sum;
            T* const at = out + (int64_t(row) * a.heads + piece.head) * a.width;
            for (int c = 0; c < a.width; c += 32) {
                uint32_t o[32];
                tmem_begin32(sum_at + c, o);
                tmem_loaded();
                #pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    float f[8];
                    #pragma unroll
                    for (int k = 0; k < 8; ++k) f[k] = __uint_as_float(o[i + k]) * inverse;
                    if (there && c + i < a.width) {
                        store_floats<T, 8>(at + c + i, f);
                        if (args.rest) {                    // what the rounding takes away
                            #pragma unroll
                            for (int k = 0; k < 8; ++k) f[k] -= to_float<T>(from_float<T>(f[k]));
                            store_floats<T, 8>(static_cast<T*>(args.rest) + (at - out) + c + i, f);
                        }
                    }
                }
            }
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) arrive(drained + s);
            if (args.sums && there) args.sums[piece.head * a.rows + row] = most - lift + log2f(sum);
        }
        tmem_fence_before();
    }
    __syncthreads();
    if (warp == 1) {
        tmem_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::columns) : "memory");
    }
    if (*failed) {               // a wait ran out: nothing that looks like a result
        for (int k = 0; k < kRecent; ++k) {
            const int item = shared->recent[k];
            if (item < 0) continue;
            const SequenceTile t = tile_of(item);
            const int rows = min(QUERIES * kTile, t.end - t.first);
            for (int i = threadIdx.x; i < rows * a.width && !t.outside; i += S::threads)
                out[(int64_t(t.first + i / a.width) * a.heads + head_of(item)) * a.width + i % a.width] = from_float<T>(__uint_as_float(0x7fffffffu));
        }
        if (threadIdx.x == 0) {
            *reinterpret_cast<volatile unsigned int*>(args.error) = 1;
            __threadfence_system();
        }
    }
}

// ---- backward ------------------------------------------------------------------------------------------------------------------
// Two kernels, one over tiles of keys (gradients of k and v, over all query heads of the key head) and one over tiles of queries, which compute the weights again from the rows' statistics. Seven products
// where one kernel could do with five, but that one's sums for q would come from many blocks, in an order of their own or in memory of 32 bits.  Here each sum stays in tensor memory from its first
// term to its last, in a fixed order.
//
// fp16: weights carry 2^14 (they are at most 1), and their gradients c, a power of two by a bound on them for the sequence, |dout| |v| / 2: at most 2^14, where small ones are normal numbers.

constexpr int kBackwardTail = 512;
template <typename T> constexpr float kWeightLift = std::is_same<T, __half>::value ? 14.0f : 0.0f;

// Heads of more than 64.
constexpr int kWidePanels = 2;
struct KeysTile {
    static constexpr int bytes = kWidePanels * kPanelBytes, stages = 2, stage_bytes = 2 * bytes + kStatisticBytes;
    static constexpr int smem = 1024 + 2 * bytes + stages * stage_bytes + kBackwardTail;
    static_assert((7 + 3 * stages) * 8 + 8 + stages * 8 <= kBackwardTail && smem <= 227 * 1024 && smem > 116 * 1024 && stage_bytes % 1024 == 0, "shared memory");
    static_assert(smem >= kLeastTensorShared, "tensor memory");
};
struct QueriesTile {
    static constexpr int bytes = kWidePanels * kPanelBytes, stages = 5;
    static constexpr int smem = 1024 + (2 + stages) * bytes + kBackwardTail;
    static_assert((8 + 3 * stages) * 8 + 8 + stages * 8 <= kBackwardTail && smem <= 227 * 1024 && smem > 116 * 1024, "shared memory");
    static_assert(smem >= kLeastTensorShared, "tensor memory");
};

struct BackwardArgs { HtgsAttention a; AttentionBackward b; unsigned int* error; };

// The power of two that a sequence's gradients of scores carry (fp16), and 1.
template <typename T> __device__ __forceinline__ float gradient_lift(const AttentionBackward& b, int sequence) {
    if (!std::is_same<T, __half>::value) return 1.0f;
    const float bound = sqrtf(__uint_as_float(b.largest[2 * sequence])) * sqrtf(__uint_as_float(b.largest[2 * sequence + 1]));
    if (!(bound >= 1e-30f && bound <= 1e30f)) return 1.0f;
    return __uint_as_float((254u - (__float_as_uint(bound) >> 23)) << 23) * 16384.0f;           // 2^14 / (the power of two that the bound reaches), which is above half of it
}
template <typename T> __device__ __forceinline__ void zero_rows(void* to, const SequenceTile& t, int heads, int head, int width, int thread, int threads) {
    const int rows = min(kTile, t.end - t.first), pieces = width / 8;
    for (int i = thread; i < rows * pieces; i += threads)
        *reinterpret_cast<uint4*>(static_cast<T*>(to) + (int64_t(t.first + i / pieces) * heads + head) * width + i % pieces * 8) = make_uint4(0, 0, 0, 0);
}
template <typename T> __device__ __forceinline__ void nan_rows(void* to, const SequenceTile& t, int heads, int head, int width) {
    const int rows = min(kTile, t.end - t.first);
    for (int i = threadIdx.x; i < rows * width; i += kTilesThreads)
        static_cast<T*>(to)[(int64_t(t.first + i / width) * heads + head) * width + i % width] = from_float<T>(__uint_as_float(0x7fffffffu));
}
// Columns [from, to) of a lane's row of sums, times a factor, rounded, into memory.
template <typename T> __device__ __forceinline__ void store_sums(uint32_t sums, T* row, int from, int to, float factor, bool there) {
    #pragma unroll 1
    for (int c = from; c < to; c += 16) {
        uint32_t o[16];
        tmem_begin16(sums + c, o);
        tmem_loaded();
        #pragma unroll
        for (int i = 0; i < 16; i += 8) {
            float f[8];
            #pragma unroll
            for (int k = 0; k < 8; ++k) f[k] = __uint_as_float(o[i + k]) * factor;
            if (there && c + i < to) store_floats<T, 8>(row + c + i, f);
        }
    }
}
// Columns [from, to] of 64, as words of two.  On what is stored and not before, so that what is not seen may be anything; and apart from the arithmetic, which else carried it in every tile (14 clocks a value).
__device__ __forceinline__ void mask_words(uint32_t (&words)[32], int from, int to) {
    #pragma unroll
    for (int k = 0; k < 32; ++k)
        words[k] &= (2 * k >= from && 2 * k <= to ? 0xffffu : 0u) | (2 * k + 1 >= from && 2 * k + 1 <= to ? 0xffff0000u : 0u);
}
// A barrier of the eight warps that share a tile's columns, with the limit of every wait.
__device__ __forceinline__ bool all_meet(uint64_t* met, uint32_t& meetings, int lane, volatile uint32_t* failed) {
    tmem_fence_before();
    __syncwarp();
    if (lane == 0) arrive(met);
    const bool ok = __all_sync(0xffffffffu, wait_in_line(met, meetings++ & 1, failed));
    tmem_fence_after();
    return ok;
}

// Heads of up to 64 (262144 rows within 512, 4 heads of 64: 950 us for k and v, 740 for q): the gradients of k and v (KEYS) or of q of a piece, 128 rows of a head ("own": k and v, or q and dout), against tiles of 64 of the others (q and dout, or k and v), in turns by two
// warpgroups, a thread for each own row.  Everything that a warpgroup writes or reads has columns of its own, so its next scores and weight gradients are computed while it works on the last ones, and it never
// waits for more than its own arithmetic.  Score gradients go into the sum in two parts, what their rounding takes away over the weight gradients that they were made of: the tensor cores have the time, and the gradients
// of q and k are then rounded where they are stored and nowhere else to speak of (100003 rows within 256, heads of 32: off by 0.0021 of their size, 0.0027 in one part, for 0.0017 of the last rounding alone).  Warp 0 finds pieces and loads; warp 1 issues the products for scores and weight gradients; warp 2 those that add up, in the tiles' order; warp 3 looks through tiles that
// are not seen whole.  Tensor memory: scores 0 and 64, weight gradients 128 and 192, weights 256 and 288, score gradients 320 and 352 (of q at both by turns), the sum for k or q 384, for v 448.
struct NarrowTile {
    static constexpr int own_bytes = kPanelBytes, other = 64, bytes = other * 128, statistic_bytes = 2 * other * 4, stage_bytes = 2 * bytes + 1024, stages = 6;
    static constexpr int smem = 1024 + 2 * 2 * own_bytes + stages * stage_bytes + 1024;
    static_assert((2 * kItems + 4 + 3 * stages + 20 + 2) * 8 + 8 + stages * 4 + kItems * 24 + 16 + int(sizeof(PieceShared)) <= 1024 && smem <= 227 * 1024 && smem > 116 * 1024, "shared memory");
    static_assert(smem >= kLeastTensorShared, "tensor memory");
};

template <typename T, bool KEYS>
__global__ void __launch_bounds__(kTilesThreads, 1) attention_narrow_kernel(const __grid_constant__ CUtensorMap map_own1, const __grid_constant__ CUtensorMap map_own2, const __grid_constant__ CUtensorMap map_other1,
                                                                           const __grid_constant__ CUtensorMap map_other2, const __grid_constant__ BackwardArgs args) {
    using S = NarrowTile;
    extern __shared__ unsigned char raw[];
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    unsigned char* const own = raw + (base - smem_u32(raw));            // two pieces' own rows, one panel and the other
    unsigned char* const ring = own + 2 * 2 * S::own_bytes;
    const uint32_t ring_at = base + 2 * 2 * S::own_bytes;
    uint64_t* const item_full = reinterpret_cast<uint64_t*>(ring + S::stages * S::stage_bytes);
    uint64_t* const item_empty = item_full + kItems;
    uint64_t* const own_full = item_empty + kItems;
    uint64_t* const own_empty = own_full + 2;
    uint64_t* const full = own_empty + 2;
    uint64_t* const empty = full + S::stages;
    uint64_t* const searched = empty + S::stages;
    // of each warpgroup
    uint64_t* const scored = searched + S::stages;       // its scores are there
    uint64_t* const scores_taken = scored + 2;           // and read
    uint64_t* const graded = scores_taken + 2;           // the gradients of its weights are there
    uint64_t* const weighed = graded + 2;                // its weights are there
    uint64_t* const changed = weighed + 2;               // the gradients of its scores are: two, by turns, as a warpgroup may be two tiles ahead of the sums
    uint64_t* const added = changed + 4;                 // and both are in the sums: two, by turns
    uint64_t* const granted = added + 4;                 // the sums are its to change
    uint64_t* const returned = granted + 2;              // and not any more
    uint64_t* const finished = returned + 2;
    uint64_t* const drained = finished + 1;
    uint32_t* const tmem_at = reinterpret_cast<uint32_t*>(drained + 1);
    volatile uint32_t* const failed = tmem_at + 1;
    volatile uint32_t* const dirty = failed + 1;         // [stages]
    volatile int* const items = reinterpret_cast<volatile int*>(dirty + S::stages);
    PieceShared* const shared = reinterpret_cast<PieceShared*>((reinterpret_cast<uintptr_t>(items + kItems * 6) + 15) & ~uintptr_t(15));

    const HtgsAttention& a = args.a;
    const AttentionBackward& b = args.b;
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31, group = a.heads / a.key_heads, own_heads = KEYS ? a.key_heads : a.heads;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) mbar_init(shared->come + i, 1);
        for (int i = 0; i < kRecent; ++i) shared->recent[i] = -1;
        for (int i = 0; i < kItems; ++i) { mbar_init(item_full + i, 1); mbar_init(item_empty + i, 3 + 8); }
        for (int i = 0; i < 2; ++i) {
            mbar_init(own_full + i, 1); mbar_init(own_empty + i, 1); mbar_init(scored + i, 1); mbar_init(scores_taken + i, 4); mbar_init(graded + i, 1);
            mbar_init(weighed + i, 4); mbar_init(changed + 2 * i, 4); mbar_init(changed + 2 * i + 1, 4); mbar_init(added + 2 * i, 1); mbar_init(added + 2 * i + 1, 1); mbar_init(granted + i, 1); mbar_init(returned + i, 4);
        }
        mbar_init(finished, 1);
        mbar_init(drained, 8);
        for (int i = 0; i < S::stages; ++i) { mbar_init(full + i, 1); mbar_init(empty + i, 2); mbar_init(searched + i, 1); }
        *failed = 0;
        mbar_fence_init();
    }
    grid_dependency();               // before tensor memory is taken, which a block of the kernel before may still have to get
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_at)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tmem_fence_before();
    }
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_at, 0);
    constexpr uint32_t kGrades = 128, kWeights = 256, kChanges = 320, kSums = 384;
    // Pieces with the most to do first, where attention is causal: the first tiles of keys, the last ones of queries.
    const auto tile_of = [&](int item) { return find_tile<kTile>(a, KEYS ? item / own_heads : int(gridDim.x - 1 - item) / own_heads); };
    const auto head_of = [&](int item) { return item % own_heads; };

    // A piece: `tiles` tiles of 64 others from row `low` on, for each of the `turns` query heads of a key head; tiles [whole.x, whole.y) are seen (or see) whole.
    struct Piece {
        int begin, end, first, head, sequence, low, tiles, n;
        int2 whole;
    };
    Piece piece;
    const auto set_piece = [&](int begin, int end, int first, int head, int sequence) {
        const int last = min(first + kTile, end) - 1;
        int low, high, all_low, all_high;
        if (KEYS) {
            low = begin + (first_seeing(a, begin, first) - begin) / S::other * S::other;      // the statistics' tiles begin with the sequence
            high = last_seeing(a, end, last); all_low = first_seeing(a, begin, last); all_high = last_seeing(a, end, first);
        } else {
            low = first_seen(a, begin, first);
            high = last_seen(a, end, last); all_low = first_seen(a, begin, last); all_high = last_seen(a, end, first);
        }
        const int tiles = (high - low) / S::other + 1;
        piece = {begin, end, first, head, sequence, low, tiles, KEYS ? group * tiles : tiles, make_int2((all_low - low + S::other - 1) / S::other, (all_high - low + 1) / S::other)};
    };
    Ring<kItems> item_at;
    const auto next_piece = [&] {
        if (!__all_sync(0xffffffffu, wait_in_line(item_full + item_at.at, item_at.round, failed))) return false;
        volatile int* const from = items + 6 * item_at.at;
        const bool there = from[5];
        if (there) set_piece(from[0], from[1], from[2], from[3], from[4]);
        __syncwarp();
        if (lane == 0) arrive(item_empty + item_at.at);
        item_at.next();
        return there;
    };
    // The tile that comes `step` behind a tile; the tiles begin again with each query head.
    const auto after = [&](int tile, int step) {
        tile += step;
        if (KEYS) while (tile >= piece.tiles) tile -= piece.tiles;
        return tile;
    };
    const auto seen_whole = [&](int tile) { return tile >= piece.whole.x && tile < piece.whole.y; };

    if (warp < 4) {
        give_registers<2>();
        const bool one = elect_one();
        bool ok = true;
        const auto wait = [&](uint64_t* bar, uint32_t parity) { ok = ok && __all_sync(0xffffffffu, wait_in_line(bar, parity, failed)); };
        uint32_t u = 0, pieces_done = 0;              // tiles of others and pieces so far
        if (warp == 0) {
            Ring<S::stages> stage;
            const auto publish = [&](const SequenceTile& t, int head, int there) {
                wait(item_empty + item_at.at, item_at.round ^ 1);
                if (!ok) return;
                if (lane == 0) {
                    volatile int* const to = items + 6 * item_at.at;
                    to[0] = t.begin; to[1] = t.end; to[2] = t.first; to[3] = head; to[4] = t.sequence; to[5] = there;
                    arrive(item_full + item_at.at);
                }
                __syncwarp();
                item_at.next();
            };
            Pieces pieces{shared, failed};
            pieces.one = one;
            for (int item = pieces.first(); item >= 0 && ok; item = pieces.following()) {
                const SequenceTile t = tile_of(item);
                if (t.first >= t.end) continue;
                const int head = head_of(item);
                if (t.outside) {
                    zero_rows<T>(KEYS ? b.grad_k : b.grad_q, t, own_heads, head, a.width, lane, 32);
                    if (KEYS) zero_rows<T>(b.grad_v, t, own_heads, head, a.width, lane, 32);
                    __syncwarp();
                    continue;
                }
                publish(t, head, 1);
                set_piece(t.begin, t.end, t.first, head, t.sequence);
                const uint32_t place = pieces_done & 1;
                wait(own_empty + place, (pieces_done >> 1 & 1) ^ 1);
                if (!ok) break;
                if (one) {
                    mbar_arrive_expect_tx(own_full + place, 2 * S::own_bytes);
                    load_panel(own + place * 2 * S::own_bytes, &map_own1, 0, head, t.first, own_full + place);
                    load_panel(own + (place * 2 + 1) * S::own_bytes, &map_own2, 0, head, t.first, own_full + place);
                }
                __syncwarp();
                ++pieces_done;
                int tile = 0, other_head = KEYS ? head * group : head / group;
                for (int i = 0; i < piece.n && ok; ++i) {
                    wait(empty + stage.at, stage.round ^ 1);
                    if (!ok) break;
                    if (one) {
                        const int row = piece.low + tile * S::other;
                        unsigned char* const at = ring + stage.at * S::stage_bytes;
                        mbar_arrive_expect_tx(full + stage.at, 2 * S::bytes + (KEYS ? S::statistic_bytes : 0));
                        load_panel(at, &map_other1, 0, other_head, row, full + stage.at);
                        load_panel(at + S::bytes, &map_other2, 0, other_head, row, full + stage.at);
                        if (KEYS) {
                            const int64_t r = statistic_base(a, t) + (row - t.begin);
                            const float* from = b.statistics + (other_head * b.statistics_rows + r / kStatisticRows * kStatisticRows) * 2 + r % kStatisticRows;
                            bulk_copy_g2s(at + 2 * S::bytes, from, S::statistic_bytes / 2, full + stage.at);
                            bulk_copy_g2s(at + 2 * S::bytes + S::statistic_bytes / 2, from + kStatisticRows, S::statistic_bytes / 2, full + stage.at);
                        }
                    }
                    __syncwarp();
                    ++u;
                    stage.next();
                    if (++tile == piece.tiles) { tile = 0; ++other_head; }
                }
            }
            ok = ok && !*failed;
            if (ok) publish({0, 0, 0, 0, false}, 0, 0);
            if (!ok) {              // no copy may be on its way when the block ends
                pieces.finish();
                for (uint32_t x = u > S::stages ? u - S::stages : 0; x < u; ++x) {
                    WaitLimit limit(kWaitNanoseconds, nanoseconds());
                    while (!mbar_try_wait(full + x % S::stages, x / S::stages & 1) && !limit.over(nanoseconds())) {}
                }
                for (uint32_t x = pieces_done > 2 ? pieces_done - 2 : 0; x < pieces_done; ++x) {
                    WaitLimit limit(kWaitNanoseconds, nanoseconds());
                    while (!mbar_try_wait(own_full + (x & 1), x >> 1 & 1) && !limit.over(nanoseconds())) {}
                }
            }
        } else if (warp == 1) {
            const uint32_t score = instruction<T>(S::other, false);
            const int steps = (a.width + 15) / 16;
            const auto product = [&](uint32_t to, uint32_t x, uint32_t y, uint64_t* bar) {
                if (one) {
                    for (int i = 0; i < steps; ++i) multiply(to, x + i * 2, y + i * 2, score, i > 0);
                    commit(bar);
                }
                __syncwarp();
            };
            while (ok && next_piece()) {
                const uint32_t place = pieces_done & 1, x = along_columns(base + place * 2 * S::own_bytes);
                wait(own_full + place, pieces_done >> 1 & 1);
                ++pieces_done;
                for (int i = 0; i < piece.n && ok; ++i, ++u) {
                    const uint32_t h = u & 1, parity = (u >> 1 & 1) ^ 1, slot = u % S::stages, y = along_columns(ring_at + slot * S::stage_bytes);
                    wait(full + slot, u / S::stages & 1);
                    wait(scores_taken + h, parity);
                    if (!ok) break;
                    tmem_fence_after();
                    product(tmem + h * 64, x, y, scored + h);
                    if (u > 1) wait(added + 2 * h + ((u >> 1) - 1 & 1), (u >> 1) - 1 >> 1 & 1);      // where they were lie the last score gradients' lower parts
                    if (!ok) break;
                    tmem_fence_after();
                    product(tmem + kGrades + h * 64, x + (S::own_bytes >> 4), y + (S::bytes >> 4), graded + h);
                }
                if (one && ok) commit(own_empty + place);
                __syncwarp();
            }
        } else if (warp == 2) {
            const uint32_t sum = instruction<T>((a.width + 15) & ~15, true);
            uint32_t grants[2] = {0, 0};
            const auto gather = [&](uint32_t to, uint32_t weights, uint32_t y, bool first) {
                if (one) {
                    #pragma unroll
                    for (int i = 0; i < S::other / 16; ++i) multiply_tmem(to, weights + i * 8, y + i * (2048 >> 4), sum, !first || i > 0);
                }
                __syncwarp();
            };
            while (ok && next_piece()) {
                wait(drained, (pieces_done & 1) ^ 1);
                ++pieces_done;
                int tile = 0;
                for (int i = 0; i < piece.n && ok; ++i, ++u, tile = after(tile, 1)) {
                    const uint32_t h = u & 1, parity = u >> 1 & 1, slot = u % S::stages, y = along_rows(ring_at + slot * S::stage_bytes);
                    const bool all = seen_whole(tile);
                    if (KEYS) {
                        wait(weighed + h, parity);
                        if (!ok) break;
                        tmem_fence_after();
                        if (all || !dirty[slot]) gather(tmem + kSums + 64, tmem + kWeights + h * 32, y + (S::bytes >> 4), i == 0);
                    }
                    wait(changed + 2 * h + parity, u >> 2 & 1);
                    if (!ok) break;
                    tmem_fence_after();
                    if (all || !dirty[slot]) {
                        gather(tmem + kSums, tmem + h * 32 + (KEYS || u >> 1 & 1 ? kChanges : kWeights), y, i == 0);
                        gather(tmem + kSums, tmem + kGrades + h * 64, y, false);
                    }
                    else {                         // the warpgroup adds them itself, when all before are in and before those behind
                        if (one) commit(granted + h);
                        __syncwarp();
                        wait(returned + h, (h ? grants[1]++ : grants[0]++) & 1);
                        if (!ok) break;
                        tmem_fence_after();
                    }
                    if (one) { commit(added + 2 * h + parity); commit(empty + slot); }
                    __syncwarp();
                }
                if (one && ok) commit(finished);
                __syncwarp();
            }
        } else {
            while (ok && next_piece()) {
                int tile = 0;
                for (int i = 0; i < piece.n && ok; ++i, ++u, tile = after(tile, 1)) {
                    const uint32_t slot = u % S::stages;
                    wait(full + slot, u / S::stages & 1);
                    if (!ok) break;
                    const unsigned char* const at = ring + slot * S::stage_bytes;
                    const bool found = !seen_whole(tile) && not_finite<T, 2 * S::bytes>(at, lane);
                    if (lane == 0) {
                        dirty[slot] = found;
                        arrive(searched + slot);
                        arrive(empty + slot);
                    }
                    __syncwarp();
                }
            }
        }
    } else {
        take_registers<2>();
        const uint32_t h = uint32_t(warp >> 2) - 1;
        const int quarter = (warp & 3) * 32;
        const uint32_t lanes = uint32_t(quarter) << 16, score = tmem + lanes + h * 64, grade = tmem + lanes + kGrades + h * 64, weights = tmem + lanes + kWeights + h * 32,
                       sums = tmem + lanes + kSums;
        const float scale = a.scale * kLog2e;
        const f32x2 scale2 = pack2(scale, scale), minus = pack2(-1.0f, -1.0f);
        constexpr float kLifted = KEYS ? kWeightLift<T> : 0.0f;                  // weights of keys go into a product themselves
        const f32x2 weight_lift2 = pack2(kLifted, kLifted);
        uint32_t u0 = 0, pieces_done = 0, grants = 0;
        bool ok = true;
        while (ok && next_piece()) {
            const int row = min(piece.first + quarter + lane, piece.end - 1);
            const bool there = piece.first + quarter + lane < piece.end;
            const int seen_low = (KEYS ? first_seeing(a, piece.begin, row) : first_seen(a, piece.begin, row)) - piece.low;
            const int seen_high = (KEYS ? last_seeing(a, piece.end, row) : last_seen(a, piece.end, row)) - piece.low;
            const float lift = gradient_lift<T>(b, piece.sequence), change_lift = lift * exp2f(-kLifted);
            const f32x2 lift2 = pack2(change_lift, change_lift);
            f32x2 row_off2 = weight_lift2, row_mean2 = weight_lift2;
            if (!KEYS) {
                const int64_t r = statistic_base(a, {piece.sequence, piece.begin, piece.end, piece.first, false}) + (row - piece.begin);
                const float* from = b.statistics + (piece.head * b.statistics_rows + r / kStatisticRows * kStatisticRows) * 2 + r % kStatisticRows;
                row_off2 = pack2(-from[0], -from[0]);
                row_mean2 = pack2(-from[kStatisticRows], -from[kStatisticRows]);
            }
            int tile = after(0, (u0 ^ h) & 1);
            for (uint32_t u = u0 + ((u0 ^ h) & 1); u < u0 + piece.n; u += 2, tile = after(tile, 2)) {
                const uint32_t parity = u >> 1 & 1, slot = u % S::stages;
                const int from = seen_low - tile * S::other, to = seen_high - tile * S::other;
                const bool masked = !seen_whole(tile);
                const float4* const statistics = reinterpret_cast<const float4*>(ring + slot * S::stage_bytes + 2 * S::bytes);
                const bool loaded = !KEYS || mbar_test(full + slot, u / S::stages & 1), there_yet = mbar_test(scored + h, parity);          // side by side: each takes a hundred clocks
                ok = __all_sync(0xffffffffu, loaded && there_yet);
                if (!ok) {
                    ok = __all_sync(0xffffffffu, wait_in_line(full + slot, u / S::stages & 1, failed) && wait_in_line(scored + h, parity, failed));
                    if (!ok) break;
                }
                // What this tile's weights and score gradients write over is in the sums: the last tile's, or of q, whose score gradients have two places, the last but one's.  Asked where nothing waits for it.
                const uint32_t turn = u >> 1, over = turn - (KEYS ? 1 : 2);
                uint64_t* const old = added + 2 * h + (over & 1);
                const bool free = turn < (KEYS ? 1 : 2) || __all_sync(0xffffffffu, mbar_test(old, over >> 1 & 1));
                tmem_fence_after();
                uint32_t p[64];
                tmem_begin32(score, p);
                tmem_begin32(score + 32, p + 32);
                tmem_loaded();
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) arrive(scores_taken + h);
                #pragma unroll
                for (int c = 0; c < 64; c += 4) {
                    const float4 off = KEYS ? statistics[c / 4] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    #pragma unroll
                    for (int k = 0; k < 4; k += 2) {
                        const f32x2 off2 = KEYS ? fma2(k ? pack2(off.z, off.w) : pack2(off.x, off.y), minus, weight_lift2) : row_off2;
                        const float2 x = unpack2(exp2_pair(fma2(pack2(__uint_as_float(p[c + k]), __uint_as_float(p[c + k + 1])), scale2, off2)));
                        p[c + k] = __float_as_uint(x.x);
                        p[c + k + 1] = __float_as_uint(x.y);
                    }
                }
                if (!free) {
                    ok = __all_sync(0xffffffffu, wait_in_line(old, over >> 1 & 1, failed));
                    if (!ok) break;
                    tmem_fence_after();
                }
                if (KEYS) {
                    uint32_t words[32];
                    #pragma unroll
                    for (int k = 0; k < 32; ++k) words[k] = floats_pair<T>(__uint_as_float(p[2 * k]), __uint_as_float(p[2 * k + 1]));
                    if (masked) mask_words(words, from, to);
                    tmem_store32(weights, words);
                    tmem_stored();
                    if (masked) {
                        ok = __all_sync(0xffffffffu, wait_in_line(searched + slot, u / S::stages & 1, failed));
                        if (!ok) break;
                    }
                    tmem_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive(weighed + h);
                }
                ok = __all_sync(0xffffffffu, wait_in_line(graded + h, parity, failed));
                if (!ok) break;
                tmem_fence_after();
                uint32_t g[64];
                tmem_begin32(grade, g);
                tmem_begin32(grade + 32, g + 32);
                tmem_loaded();
                const uint32_t changes = tmem + lanes + h * 32 + (KEYS || turn & 1 ? kChanges : kWeights);
                {
                    uint32_t words[32], lower[32];
                    #pragma unroll
                    for (int c = 0; c < 64; c += 4) {
                        const float4 mean = KEYS ? statistics[16 + c / 4] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        #pragma unroll
                        for (int k = 0; k < 4; k += 2) {
                            const f32x2 grad = pack2(__uint_as_float(g[c + k]), __uint_as_float(g[c + k + 1])), weight = pack2(__uint_as_float(p[c + k]), __uint_as_float(p[c + k + 1]));
                            const f32x2 away = KEYS ? fma2(k ? pack2(mean.z, mean.w) : pack2(mean.x, mean.y), minus, grad) : add2(grad, row_mean2);
                            const f32x2 change = mul2(std::is_same<T, __half>::value ? mul2(weight, lift2) : weight, away);
                            const float2 ds = unpack2(change);
                            words[(c + k) / 2] = floats_pair<T>(ds.x, ds.y);
                            const float2 upper = pair_floats<T>(words[(c + k) / 2]), rest = unpack2(fma2(pack2(upper.x, upper.y), minus, change));
                            lower[(c + k) / 2] = floats_pair<T>(rest.x, rest.y);
                        }
                    }
                    if (masked) { mask_words(words, from, to); mask_words(lower, from, to); }
                    tmem_store32(changes, words);
                    tmem_store32(grade, lower);
                }
                tmem_stored();
                if (!KEYS && masked) {
                    ok = __all_sync(0xffffffffu, wait_in_line(searched + slot, u / S::stages & 1, failed));
                    if (!ok) break;
                }
                const bool spoilt = masked && dirty[slot];
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) arrive(changed + 2 * h + parity);
                if (spoilt) {
                    ok = __all_sync(0xffffffffu, wait_in_line(full + slot, u / S::stages & 1, failed) && wait_in_line(granted + h, grants & 1, failed));
                    if (!ok) break;
                    ++grants;
                    tmem_fence_after();
                    multiply_seen<T>(sums, 0, a.width, u > u0, changes, 0, ring + slot * S::stage_bytes, from, to, 2);
                    multiply_seen<T>(sums, 0, a.width, true, grade, 0, ring + slot * S::stage_bytes, from, to, 2);
                    if (KEYS) multiply_seen<T>(sums + 64, 0, a.width, u > u0, weights, 0, ring + slot * S::stage_bytes + S::bytes, from, to, 2);
                    tmem_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive(returned + h);
                }
            }
            u0 += piece.n;
            if (!ok) break;
            ok = __all_sync(0xffffffffu, wait_in_line(finished, pieces_done & 1, failed));
            if (!ok) break;
            ++pieces_done;
            tmem_fence_after();
            const int64_t at = (int64_t(row) * own_heads + piece.head) * a.width;
            const int middle = min((a.width / 2 + 15) & ~15, a.width);
            if (!KEYS) store_sums<T>(sums, static_cast<T*>(b.grad_q) + at, h ? middle : 0, h ? a.width : middle, a.scale / lift, there);
            else if (h) store_sums<T>(sums + 64, static_cast<T*>(b.grad_v) + at, 0, a.width, exp2f(-kLifted), there);
            else store_sums<T>(sums, static_cast<T*>(b.grad_k) + at, 0, a.width, a.scale / lift, there);
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) arrive(drained);
        }
        tmem_fence_before();
    }
    __syncthreads();
    if (warp == 1) {
        tmem_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
    if (*failed) {
        for (int k = 0; k < kRecent; ++k) {
            if (shared->recent[k] < 0) continue;
            const SequenceTile t = tile_of(shared->recent[k]);
            if (t.outside) continue;
            nan_rows<T>(KEYS ? b.grad_k : b.grad_q, t, own_heads, head_of(shared->recent[k]), a.width);
            if (KEYS) nan_rows<T>(b.grad_v, t, own_heads, head_of(shared->recent[k]), a.width);
        }
        if (threadIdx.x == 0) {
            *reinterpret_cast<volatile unsigned int*>(args.error) = 1;
            __threadfence_system();
        }
    }
}

// Gradients of k and v of a tile.  Scores and their gradients are turned round, a row for each key, so that the weights are the first operand from tensor memory.  Warp 0 loads queries, output gradients and
// statistics of a tile of queries; warp 1 issues the products, [dv, next scores] while the score gradients are computed and [dk, next weight gradients] while the weights are; warps 4 to 7 and 8 to 11
// have 64 columns each.  Tensor memory: scores (weights) 0, weight gradients (score gradients) 128, dv 256, dk 384.  With the kernel behind it 16384 rows, causal, 8 heads of 128 take 1.5 to 1.8 ms, 1.0
// PFLOP/s of the seven products.
template <typename T>
__global__ void __launch_bounds__(kTilesThreads, 1) attention_keys_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                                         const __grid_constant__ CUtensorMap map_grad, const __grid_constant__ BackwardArgs args) {
    using S = KeysTile;
    extern __shared__ unsigned char raw[];
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    unsigned char* const own = raw + (base - smem_u32(raw));            // k, v
    unsigned char* const ring = own + 2 * S::bytes;
    const uint32_t ring_at = base + 2 * S::bytes;
    uint64_t* const own_full = reinterpret_cast<uint64_t*>(ring + S::stages * S::stage_bytes);
    uint64_t* const full = own_full + 1;
    uint64_t* const empty = full + S::stages;
    uint64_t* const searched = empty + S::stages;
    uint64_t* const scored = searched + S::stages;       // scores are there
    uint64_t* const weighed = scored + 1;                // weights are
    uint64_t* const graded = weighed + 1;                // gradients of the weights are
    uint64_t* const changed = graded + 1;                // gradients of the scores are
    uint64_t* const finished = changed + 1;
    uint64_t* const met = finished + 1;
    uint32_t* const tmem_at = reinterpret_cast<uint32_t*>(met + 1);
    volatile uint32_t* const failed = tmem_at + 1;
    volatile uint32_t* const dirty = failed + 1;         // [stages][2]: output gradients, queries

    const HtgsAttention& a = args.a;
    const AttentionBackward& b = args.b;
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    grid_dependency();
    // the first tiles of a sequence first: causal, they are seen by the most queries
    const int key_head = int(blockIdx.x % a.key_heads), group = a.heads / a.key_heads;
    const SequenceTile t = find_tile<kTile>(a, int(blockIdx.x / a.key_heads));
    if (t.first >= t.end) return;
    if (t.outside) {
        zero_rows<T>(b.grad_k, t, a.key_heads, key_head, a.width, threadIdx.x, kTilesThreads);
        zero_rows<T>(b.grad_v, t, a.key_heads, key_head, a.width, threadIdx.x, kTilesThreads);
        return;
    }
    const int last_row = min(t.first + kTile, t.end) - 1;
    const int first_tile = (first_seeing(a, t.begin, t.first) - t.begin) / kTile, tiles = (last_seeing(a, t.end, last_row) - t.begin) / kTile - first_tile + 1, n = group * tiles;
    const int whole_low = first_seeing(a, t.begin, last_row), whole_high = last_seeing(a, t.end, t.first);
    const auto query_row = [&](int i) { return t.begin + (first_tile + i % tiles) * kTile; };
    const auto whole = [&](int q0) { return q0 >= whole_low && q0 + kTile - 1 <= whole_high; };       // all keys are seen by all queries

    if (threadIdx.x == 0) {
        mbar_init(own_full, 1); mbar_init(scored, 1); mbar_init(weighed, 8); mbar_init(graded, 1); mbar_init(changed, 8); mbar_init(finished, 1); mbar_init(met, 8);
        for (int i = 0; i < S::stages; ++i) { mbar_init(full + i, 1); mbar_init(empty + i, 3); mbar_init(searched + i, 2); }
        *failed = 0;
        mbar_fence_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_at)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tmem_fence_before();
    }
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_at, 0);

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 0) {
            const bool one = elect_one();
            if (one) {
                mbar_arrive_expect_tx(own_full, 2 * S::bytes);
                for (int p = 0; p < kWidePanels; ++p) {
                    load_panel(own + p * kPanelBytes, &map_k, p * kPanel, key_head, t.first, own_full);
                    load_panel(own + S::bytes + p * kPanelBytes, &map_v, p * kPanel, key_head, t.first, own_full);
                }
            }
            __syncwarp();
            const float* statistics = b.statistics + (statistic_base(a, t) + first_tile * kTile) * 2;
            Ring<S::stages> stage;
            uint32_t uses = 0;
            bool ok = true;
            for (int i = 0; i < n; ++i, ++uses, stage.next()) {
                ok = __all_sync(0xffffffffu, wait_in_line(empty + stage.at, stage.round ^ 1, failed));
                if (!ok) break;
                if (one) {
                    unsigned char* at = ring + stage.at * S::stage_bytes;
                    const int head = key_head * group + i / tiles, row = query_row(i);
                    mbar_arrive_expect_tx(full + stage.at, S::stage_bytes);
                    for (int p = 0; p < kWidePanels; ++p) load_panel(at + p * kPanelBytes, &map_q, p * kPanel, head, row, full + stage.at);
                    for (int p = 0; p < kWidePanels; ++p) load_panel(at + S::bytes + p * kPanelBytes, &map_grad, p * kPanel, head, row, full + stage.at);
                    bulk_copy_g2s(at + 2 * S::bytes, statistics + (head * b.statistics_rows + i % tiles * kTile) * 2, kStatisticBytes, full + stage.at);
                }
                __syncwarp();
            }
            if (!ok) {              // no copy may be on its way when the block ends
                for (uint32_t u = uses > S::stages ? uses - S::stages : 0; u < uses; ++u) {
                    WaitLimit limit(kWaitNanoseconds, nanoseconds());
                    while (!mbar_try_wait(full + u % S::stages, u / S::stages & 1) && !limit.over(nanoseconds())) {}
                }
                WaitLimit limit(kWaitNanoseconds, nanoseconds());
                while (!mbar_try_wait(own_full, 0) && !limit.over(nanoseconds())) {}
            }
        } else if (warp == 1) {
            const bool one = elect_one();
            const uint32_t score = instruction<T>(kTile, false), sum = instruction<T>((a.width + 15) & ~15, true);
            const int steps = (a.width + 15) / 16;
            Ring<S::stages> stage, next;
            bool ok = true;
            const auto wait = [&](uint64_t* bar, uint32_t parity) { ok = ok && __all_sync(0xffffffffu, wait_in_line(bar, parity, failed)); };
            // scores (which 0) of keys and queries, or gradients of weights (1) of values and output gradients
            const auto product = [&](int which, uint32_t slot, uint64_t* bar) {
                const uint32_t x = along_columns(base + which * S::bytes), y = along_columns(ring_at + slot * S::stage_bytes + which * S::bytes);
                if (one) {
                    for (int i = 0; i < steps; ++i) {
                        const uint32_t at = (i >> 2) * kPanelUnits + (i & 3) * 2;
                        multiply(tmem + which * kTile, x + at, y + at, score, i > 0);
                    }
                    commit(bar);
                }
                __syncwarp();
            };
            // dv (1) of weights and output gradients, or dk (0) of score gradients and queries
            const auto gather = [&](int which, uint32_t slot, bool first, bool added) {
                const uint32_t w = tmem + (which ? 0 : kTile), y = along_rows(ring_at + slot * S::stage_bytes + which * S::bytes), to = tmem + (which ? 2 : 3) * kTile;
                if (one) {
                    #pragma unroll
                    for (int i = 0; i < (added ? 0 : kTile / 16); ++i) multiply_tmem(to, w + (i >> 2) * 64 + (i & 3) * 8, y + i * (2048 >> 4), sum, !first || i > 0);
                }
                __syncwarp();
            };
            wait(own_full, 0);
            wait(full, 0);
            if (ok) {
                tmem_fence_after();
                product(0, 0, scored);
                product(1, 0, graded);
                next.next();
            }
            for (int i = 0; i < n && ok; ++i, stage.next()) {
                const bool all = whole(query_row(i));
                wait(weighed, i & 1);
                if (!ok) break;
                tmem_fence_after();
                gather(1, stage.at, i == 0, !all && dirty[2 * stage.at]);
                if (i + 1 < n) {
                    wait(full + next.at, next.round);
                    if (!ok) break;
                    product(0, next.at, scored);
                }
                wait(changed, i & 1);
                if (!ok) break;
                tmem_fence_after();
                gather(0, stage.at, i == 0, !all && dirty[2 * stage.at + 1]);
                if (one) commit(empty + stage.at);
                __syncwarp();
                if (i + 1 < n) {
                    product(1, next.at, graded);
                    next.next();
                }
            }
            if (one && ok) commit(finished);
            __syncwarp();
        } else {
            Ring<S::stages> stage;
            for (int i = 0; i < n; ++i, stage.next()) {
                if (!__all_sync(0xffffffffu, wait_in_line(full + stage.at, stage.round, failed))) break;
                bool found = false;
                if (!whole(query_row(i))) {
                    const unsigned char* tile = ring + stage.at * S::stage_bytes + (warp == 2 ? S::bytes : 0);
                    found = not_finite<T, S::bytes>(tile, lane);
                }
                if (lane == 0) {
                    dirty[2 * stage.at + warp - 2] = found;
                    arrive(searched + stage.at);
                    arrive(empty + stage.at);
                }
                __syncwarp();
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int half = (warp >> 2) - 1, quarter = (warp & 3) * 32;
        const int row = min(t.first + quarter + lane, t.end - 1);
        const bool there = t.first + quarter + lane < t.end;
        const uint32_t lanes = uint32_t(quarter) << 16, score = tmem + lanes + half * 64, grade = score + kTile;
        const float scale = a.scale * kLog2e, lift = gradient_lift<T>(b, t.sequence);
        const f32x2 scale2 = pack2(scale, scale), lift2 = pack2(lift * exp2f(-kWeightLift<T>), lift * exp2f(-kWeightLift<T>)), weight_lift2 = pack2(kWeightLift<T>, kWeightLift<T>);
        const f32x2 minus = pack2(-1.0f, -1.0f);
        const int seen_low = first_seeing(a, t.begin, row), seen_high = last_seeing(a, t.end, row);
        const int middle = min((a.width / 2 + 15) & ~15, a.width);                // columns of sums, where the two warpgroups share them
        uint32_t meetings = 0;
        const auto meet = [&] { return all_meet(met, meetings, lane, failed); };
        Ring<S::stages> stage;
        bool ok = true;
        for (int i = 0; i < n; ++i, stage.next()) {
            const int q0 = query_row(i), from = seen_low - q0, to = seen_high - q0;
            const bool masked = !whole(q0);
            const unsigned char* place = ring + stage.at * S::stage_bytes;
            const float4* statistics = reinterpret_cast<const float4*>(place + 2 * S::bytes) + half * 16;
            ok = __all_sync(0xffffffffu, wait_in_line(full + stage.at, stage.round, failed) && wait_in_line(scored, i & 1, failed));
            if (!ok) break;
            tmem_fence_after();
            uint32_t p[64];
            tmem_begin32(score, p);
            tmem_begin32(score + 32, p + 32);
            tmem_loaded();
            uint32_t words[32];
            #pragma unroll
            for (int c = 0; c < 64; c += 32) {
                #pragma unroll
                for (int k = 0; k < 32; k += 4) {
                    const float4 sums = statistics[(c + k) / 4];
                    #pragma unroll
                    for (int h = 0; h < 4; h += 2) {
                        const f32x2 off = fma2(h ? pack2(sums.z, sums.w) : pack2(sums.x, sums.y), minus, weight_lift2);
                        const float2 x = unpack2(fma2(pack2(__uint_as_float(p[c + k + h]), __uint_as_float(p[c + k + h + 1])), scale2, off));
                        const float p0 = exp2_approx(x.x), p1 = exp2_approx(x.y);
                        p[c + k + h] = __float_as_uint(p0);
                        p[c + k + h + 1] = __float_as_uint(p1);
                        words[(c + k + h) / 2] = floats_pair<T>(p0, p1);
                    }
                }
            }
            if (masked) mask_words(words, from - half * 64, to - half * 64);
            tmem_store32(score, words);
            tmem_stored();
            uint32_t spoilt[2] = {0, 0};
            if (masked) {
                ok = __all_sync(0xffffffffu, wait_in_line(searched + stage.at, stage.round, failed));
                if (!ok) break;
                spoilt[0] = dirty[2 * stage.at]; spoilt[1] = dirty[2 * stage.at + 1];
                if (spoilt[0]) {
                    ok = meet();             // the other columns' weights
                    if (!ok) break;
                    multiply_seen<T>(tmem + lanes + 2 * kTile, half ? middle : 0, half ? a.width : middle, i > 0, tmem + lanes, 64, place + S::bytes, from, to);
                }
            }
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) arrive(weighed);
            ok = __all_sync(0xffffffffu, wait_in_line(graded, i & 1, failed));
            if (!ok) break;
            tmem_fence_after();
            #pragma unroll
            for (int c = 0; c < 64; c += 32) {
                uint32_t g[32];
                tmem_begin32(grade + c, g);
                tmem_loaded();
                #pragma unroll
                for (int k = 0; k < 32; k += 4) {
                    const float4 means = statistics[32 + (c + k) / 4];
                    #pragma unroll
                    for (int h = 0; h < 4; h += 2) {
                        const f32x2 away = fma2(h ? pack2(means.z, means.w) : pack2(means.x, means.y), minus, pack2(__uint_as_float(g[k + h]), __uint_as_float(g[k + h + 1])));
                        const f32x2 weight = pack2(__uint_as_float(p[c + k + h]), __uint_as_float(p[c + k + h + 1]));
                        const float2 ds = unpack2(mul2(std::is_same<T, __half>::value ? mul2(weight, lift2) : weight, away));
                        words[(c + k + h) / 2] = floats_pair<T>(ds.x, ds.y);
                    }
                }
            }
            if (masked) mask_words(words, from - half * 64, to - half * 64);
            tmem_store32(grade, words);
            tmem_stored();
            if (spoilt[1]) {
                ok = meet();
                if (!ok) break;
                multiply_seen<T>(tmem + lanes + 3 * kTile, half ? middle : 0, half ? a.width : middle, i > 0, tmem + lanes + kTile, 64, place, from, to);
            }
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) arrive(changed);
        }
        ok = ok && __all_sync(0xffffffffu, wait_in_line(finished, 0, failed));
        if (ok) {
            tmem_fence_after();
            const int64_t at = (int64_t(row) * a.key_heads + key_head) * a.width;
            if (half == 0) store_sums<T>(tmem + lanes + 2 * kTile, static_cast<T*>(b.grad_v) + at, 0, a.width, exp2f(-kWeightLift<T>), there);
            else store_sums<T>(tmem + lanes + 3 * kTile, static_cast<T*>(b.grad_k) + at, 0, a.width, a.scale / lift, there);
        }
        tmem_fence_before();
    }
    __syncthreads();
    if (warp == 1) {
        tmem_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
    if (*failed) {
        nan_rows<T>(b.grad_k, t, a.key_heads, key_head, a.width);
        nan_rows<T>(b.grad_v, t, a.key_heads, key_head, a.width);
        if (threadIdx.x == 0) {
            *reinterpret_cast<volatile unsigned int*>(args.error) = 1;
            __threadfence_system();
        }
    }
}

// Gradient of q of a tile.  Scores are computed a tile ahead.  Tensor memory: scores (score gradients) by turns at 0 and 128, weight gradients 256, dq 384.
template <typename T>
__global__ void __launch_bounds__(kTilesThreads, 1) attention_queries_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                                            const __grid_constant__ CUtensorMap map_grad, const __grid_constant__ BackwardArgs args) {
    using S = QueriesTile;
    extern __shared__ unsigned char raw[];
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    unsigned char* const own = raw + (base - smem_u32(raw));            // q, dout
    unsigned char* const ring = own + 2 * S::bytes;
    const uint32_t ring_at = base + 2 * S::bytes;
    uint64_t* const own_full = reinterpret_cast<uint64_t*>(ring + S::stages * S::bytes);
    uint64_t* const full = own_full + 1;
    uint64_t* const empty = full + S::stages;
    uint64_t* const searched = empty + S::stages;
    uint64_t* const scored = searched + S::stages;       // [2]
    uint64_t* const graded = scored + 2;
    uint64_t* const changed = graded + 1;
    uint64_t* const finished = changed + 1;
    uint64_t* const met = finished + 1;
    uint32_t* const tmem_at = reinterpret_cast<uint32_t*>(met + 1);
    volatile uint32_t* const failed = tmem_at + 1;
    volatile uint32_t* const dirty = failed + 1;         // [stages][2], of halves of a tile of keys

    const HtgsAttention& a = args.a;
    const AttentionBackward& b = args.b;
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    grid_dependency();
    const int head = int(blockIdx.x % a.heads), key_head = head / (a.heads / a.key_heads);
    const SequenceTile t = find_tile<kTile>(a, int(gridDim.x / a.heads - 1 - blockIdx.x / a.heads));
    if (t.first >= t.end) return;
    if (t.outside) {
        zero_rows<T>(b.grad_q, t, a.heads, head, a.width, threadIdx.x, kTilesThreads);
        return;
    }
    const int last_row = min(t.first + kTile, t.end) - 1;
    const int low = first_seen(a, t.begin, t.first), n = (last_seen(a, t.end, last_row) - low) / kTile + 1;
    const int whole_low = first_seen(a, t.begin, last_row), whole_high = last_seen(a, t.end, t.first);
    const auto whole = [&](int j) { return low + j * kTile >= whole_low && low + j * kTile + kTile - 1 <= whole_high; };

    if (threadIdx.x == 0) {
        mbar_init(own_full, 1); mbar_init(scored, 1); mbar_init(scored + 1, 1); mbar_init(graded, 1); mbar_init(changed, 8); mbar_init(finished, 1); mbar_init(met, 8);
        for (int i = 0; i < S::stages; ++i) { mbar_init(full + i, 1); mbar_init(empty + i, 3); mbar_init(searched + i, 2); }
        *failed = 0;
        mbar_fence_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_at)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tmem_fence_before();
    }
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_at, 0);

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 0) {
            const bool one = elect_one();
            if (one) {
                mbar_arrive_expect_tx(own_full, 2 * S::bytes);
                for (int p = 0; p < kWidePanels; ++p) {
                    load_panel(own + p * kPanelBytes, &map_q, p * kPanel, head, t.first, own_full);
                    load_panel(own + S::bytes + p * kPanelBytes, &map_grad, p * kPanel, head, t.first, own_full);
                }
            }
            __syncwarp();
            Ring<S::stages> stage;
            uint32_t uses = 0;
            bool ok = true;
            for (int i = 0; i < 2 * n; ++i, ++uses, stage.next()) {           // keys and values of a tile by turns
                ok = __all_sync(0xffffffffu, wait_in_line(empty + stage.at, stage.round ^ 1, failed));
                if (!ok) break;
                if (one) {
                    mbar_arrive_expect_tx(full + stage.at, S::bytes);
                    for (int p = 0; p < kWidePanels; ++p) load_panel(ring + stage.at * S::bytes + p * kPanelBytes, i & 1 ? &map_v : &map_k, p * kPanel, key_head, low + (i >> 1) * kTile, full + stage.at);
                }
                __syncwarp();
            }
            if (!ok) {              // no copy may be on its way when the block ends
                for (uint32_t u = uses > S::stages ? uses - S::stages : 0; u < uses; ++u) {
                    WaitLimit limit(kWaitNanoseconds, nanoseconds());
                    while (!mbar_try_wait(full + u % S::stages, u / S::stages & 1) && !limit.over(nanoseconds())) {}
                }
                WaitLimit limit(kWaitNanoseconds, nanoseconds());
                while (!mbar_try_wait(own_full, 0) && !limit.over(nanoseconds())) {}
            }
        } else if (warp == 1) {
            const bool one = elect_one();
            const uint32_t score = instruction<T>(kTile, false), sum = instruction<T>((a.width + 15) & ~15, true);
            const int steps = (a.width + 15) / 16;
            Ring<S::stages> stage;
            uint32_t key_slot[2] = {0, 0};
            bool ok = true;
            const auto wait = [&](uint64_t* bar, uint32_t parity) { ok = ok && __all_sync(0xffffffffu, wait_in_line(bar, parity, failed)); };
            // scores of a tile (which 0), or gradients of its weights (1), from the next place of the ring
            const auto product = [&](int which, int j) {
                wait(full + stage.at, stage.round);
                if (!ok) return;
                tmem_fence_after();
                const uint32_t x = along_columns(base + which * S::bytes), y = along_columns(ring_at + stage.at * S::bytes), d = tmem + (which ? 2 * kTile : (j & 1) * kTile);
                if (one) {
                    for (int i = 0; i < steps; ++i) {
                        const uint32_t at = (i >> 2) * kPanelUnits + (i & 3) * 2;
                        multiply(d, x + at, y + at, score, i > 0);
                    }
                    commit(which ? graded : scored + (j & 1));
                    if (which) commit(empty + stage.at);
                }
                __syncwarp();
                if (!which) key_slot[j & 1] = stage.at;
                stage.next();
            };
            wait(own_full, 0);
            if (ok) product(0, 0);
            if (ok) product(1, 0);
            if (ok && n > 1) product(0, 1);
            for (int j = 0; j < n && ok; ++j) {
                wait(changed, j & 1);
                if (!ok) break;
                tmem_fence_after();
                const uint32_t slot = key_slot[j & 1], y = along_rows(ring_at + slot * S::bytes), w = tmem + (j & 1) * kTile;
                const bool added = !whole(j) && (dirty[2 * slot] | dirty[2 * slot + 1]);
                if (one) {
                    #pragma unroll
                    for (int i = 0; i < (added ? 0 : kTile / 16); ++i) multiply_tmem(tmem + 3 * kTile, w + (i >> 2) * 64 + (i & 3) * 8, y + i * (2048 >> 4), sum, j > 0 || i > 0);
                    commit(empty + slot);
                }
                __syncwarp();
                if (j + 1 < n) product(1, j + 1);
                if (ok && j + 2 < n) product(0, j + 2);
            }
            if (one && ok) commit(finished);
            __syncwarp();
        } else {
            Ring<S::stages> stage;
            for (int i = 0; i < 2 * n; ++i, stage.next()) {
                if (!__all_sync(0xffffffffu, wait_in_line(full + stage.at, stage.round, failed))) break;
                const bool found = warp == 2 && !(i & 1) && !whole(i >> 1) && not_finite<T, S::bytes>(ring + stage.at * S::bytes, lane);
                if (lane == 0) {
                    dirty[2 * stage.at + warp - 2] = found;
                    arrive(searched + stage.at);
                    arrive(empty + stage.at);
                }
                __syncwarp();
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int half = (warp >> 2) - 1, quarter = (warp & 3) * 32;
        const int row = min(t.first + quarter + lane, t.end - 1);
        const bool there = t.first + quarter + lane < t.end;
        const uint32_t lanes = uint32_t(quarter) << 16;
        const float scale = a.scale * kLog2e, lift = gradient_lift<T>(b, t.sequence);
        const float* statistics = b.statistics + (head * b.statistics_rows + statistic_base(a, t) + (t.first - t.begin)) * 2 + quarter + lane;
        const float row_sum = there ? statistics[0] : 0.0f, mean = there ? statistics[kStatisticRows] : 0.0f;
        const f32x2 scale2 = pack2(scale, scale), off2 = pack2(-row_sum, -row_sum), mean2 = pack2(-mean, -mean), lift2 = pack2(lift, lift);
        const int row_low = first_seen(a, t.begin, row), row_high = last_seen(a, t.end, row);
        const int middle = min((a.width / 2 + 15) & ~15, a.width);
        uint32_t meetings = 0;
        const auto meet = [&] { return all_meet(met, meetings, lane, failed); };
        bool ok = true;
        for (int j = 0; j < n; ++j) {
            const uint32_t score = tmem + lanes + (j & 1) * kTile + half * 64, grade = tmem + lanes + 2 * kTile + half * 64;
            const int from = row_low - (low + j * kTile), to = row_high - (low + j * kTile);
            const bool masked = !whole(j);
            ok = __all_sync(0xffffffffu, wait_in_line(scored + (j & 1), j >> 1 & 1, failed));
            if (!ok) break;
            tmem_fence_after();
            uint32_t p[64];
            tmem_begin32(score, p);
            tmem_begin32(score + 32, p + 32);
            tmem_loaded();
            #pragma unroll
            for (int c = 0; c < 64; c += 2) {
                const float2 x = unpack2(fma2(pack2(__uint_as_float(p[c]), __uint_as_float(p[c + 1])), scale2, off2));
                p[c] = __float_as_uint(exp2_approx(x.x));
                p[c + 1] = __float_as_uint(exp2_approx(x.y));
            }
            ok = __all_sync(0xffffffffu, wait_in_line(graded, j & 1, failed));
            if (!ok) break;
            tmem_fence_after();
            uint32_t words[32];
            #pragma unroll
            for (int c = 0; c < 64; c += 32) {
                uint32_t g[32];
                tmem_begin32(grade + c, g);
                tmem_loaded();
                #pragma unroll
                for (int k = 0; k < 32; k += 2) {
                    const f32x2 away = add2(pack2(__uint_as_float(g[k]), __uint_as_float(g[k + 1])), mean2), weight = pack2(__uint_as_float(p[c + k]), __uint_as_float(p[c + k + 1]));
                    const float2 ds = unpack2(mul2(std::is_same<T, __half>::value ? mul2(weight, lift2) : weight, away));
                    words[(c + k) / 2] = floats_pair<T>(ds.x, ds.y);
                }
            }
            if (masked) mask_words(words, from - half * 64, to - half * 64);
            tmem_store32(score, words);
            tmem_stored();
            if (masked) {
                const uint32_t at = uint32_t(2 * j) % S::stages, round = uint32_t(2 * j) / S::stages & 1;
                ok = __all_sync(0xffffffffu, wait_in_line(searched + at, round, failed));
                if (!ok) break;
                if (dirty[2 * at] | dirty[2 * at + 1]) {
                    ok = __all_sync(0xffffffffu, wait_in_line(full + at, round, failed)) && meet();             // the other columns' score gradients
                    if (!ok) break;
                    multiply_seen<T>(tmem + lanes + 3 * kTile, half ? middle : 0, half ? a.width : middle, j > 0, tmem + lanes + (j & 1) * kTile, 64, ring + at * S::bytes, from, to);
                }
            }
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) arrive(changed);
        }
        ok = ok && __all_sync(0xffffffffu, wait_in_line(finished, 0, failed));
        if (ok) {
            tmem_fence_after();
            store_sums<T>(tmem + lanes + 3 * kTile, static_cast<T*>(b.grad_q) + (int64_t(row) * a.heads + head) * a.width, half ? middle : 0, half ? a.width : middle, a.scale / lift, there);
        }
        tmem_fence_before();
    }
    __syncthreads();
    if (warp == 1) {
        tmem_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
    if (*failed) {
        nan_rows<T>(b.grad_q, t, a.heads, head, a.width);
        if (threadIdx.x == 0) {
            *reinterpret_cast<volatile unsigned int*>(args.error) = 1;
            __threadfence_system();
        }
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------

// [rows, heads, width] in boxes of so many rows and a panel of one head's columns.
bool make_rows_map(CUtensorMap* map, const void* base, int64_t rows, int heads, int width, int64_t stride, int64_t head_stride, int box_rows = kTile) {
    const cuuint64_t dense = cuuint64_t(width) * 2;                 // a stride that takes no step says nothing
    const cuuint64_t sizes[3] = {cuuint64_t(width), cuuint64_t(heads), cuuint64_t(rows)};
    const cuuint64_t strides[2] = {heads > 1 ? cuuint64_t(head_stride) * 2 : dense, rows > 1 ? cuuint64_t(stride) * 2 : dense * cuuint64_t(heads)};
    const cuuint32_t box[3] = {kPanel, 1, cuuint32_t(box_rows)}, steps[3] = {1, 1, 1};
    const EncodeTiled encode = encode_tiled();
    return encode && encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(base), sizes, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool heads_aligned(const void* p, int64_t rows, int heads, int64_t stride, int64_t head_stride) {
    const auto step = [](int64_t s) { return s > 0 && s % 8 == 0 && s < (int64_t(1) << 38); };
    return aligned(p, 16) && (rows == 1 || step(stride)) && (heads == 1 || step(head_stride));
}

template <typename T, int PANELS, int QUERIES> int launch_forward(const ForwardArgs& args, cudaStream_t stream) {
    using S = ForwardTile<PANELS, QUERIES>;
    const HtgsAttention& a = args.a;
    CUtensorMap q, k, v;
    if (!make_rows_map(&q, a.q, a.rows, a.heads, a.width, a.q_stride, a.q_head_stride) || !make_rows_map(&k, a.k, a.rows, a.key_heads, a.width, a.k_stride, a.k_head_stride) ||
        !make_rows_map(&v, a.v, a.rows, a.key_heads, a.width, a.v_stride, a.v_head_stride))
        return sequence_fail(HTGS_ERR_CUDA, "htgs_attention: the tensor maps cannot be made");
    static PerDeviceOnce once;
    cudaError_t err = once.run([] { return cudaFuncSetAttribute(attention_tiles_kernel<T, PANELS, QUERIES>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::smem); });
    if (err == cudaSuccess) err = launch_after(attention_tiles_kernel<T, PANELS, QUERIES>, dim3(unsigned(sequence_tiles(a, QUERIES * kTile) * a.heads)), S::threads, S::smem, stream, q, k, v, args);
    return err == cudaSuccess ? sequence_status("htgs_attention") : sequence_fail(HTGS_ERR_CUDA, cudaGetErrorString(err));
}
template <typename T> int launch_wide(const BackwardArgs& args, cudaStream_t stream) {
    const HtgsAttention& a = args.a;
    CUtensorMap q, k, v, grad;
    if (!make_rows_map(&q, a.q, a.rows, a.heads, a.width, a.q_stride, a.q_head_stride) || !make_rows_map(&k, a.k, a.rows, a.key_heads, a.width, a.k_stride, a.k_head_stride) ||
        !make_rows_map(&v, a.v, a.rows, a.key_heads, a.width, a.v_stride, a.v_head_stride) || !make_rows_map(&grad, args.b.grad, a.rows, a.heads, a.width, args.b.grad_stride, args.b.grad_head_stride))
        return sequence_fail(HTGS_ERR_CUDA, "htgs_attention_backward: the tensor maps cannot be made");
    static PerDeviceOnce once;
    cudaError_t err = once.run([] {
        const cudaError_t e = cudaFuncSetAttribute(attention_keys_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, KeysTile::smem);
        return e != cudaSuccess ? e : cudaFuncSetAttribute(attention_queries_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, QueriesTile::smem);
    });
    const int64_t tiles = sequence_tiles(a, kTile);
    if (err == cudaSuccess) err = launch_after(attention_keys_kernel<T>, dim3(unsigned(tiles * a.key_heads)), kTilesThreads, KeysTile::smem, stream, q, k, v, grad, args);
    if (err == cudaSuccess) err = launch_after(attention_queries_kernel<T>, dim3(unsigned(tiles * a.heads)), kTilesThreads, QueriesTile::smem, stream, q, k, v, grad, args);
    return err == cudaSuccess ? sequence_status("htgs_attention_backward") : sequence_fail(HTGS_ERR_CUDA, cudaGetErrorString(err));
}
template <typename T> int launch_narrow(const BackwardArgs& args, cudaStream_t stream) {
    const HtgsAttention& a = args.a;
    const auto maps = [&](CUtensorMap (&m)[4], int rows) {          // q, k, v, dout
        return make_rows_map(&m[0], a.q, a.rows, a.heads, a.width, a.q_stride, a.q_head_stride, rows) && make_rows_map(&m[1], a.k, a.rows, a.key_heads, a.width, a.k_stride, a.k_head_stride, rows) &&
               make_rows_map(&m[2], a.v, a.rows, a.key_heads, a.width, a.v_stride, a.v_head_stride, rows) &&
               make_rows_map(&m[3], args.b.grad, a.rows, a.heads, a.width, args.b.grad_stride, args.b.grad_head_stride, rows);
    };
    CUtensorMap own[4], other[4];
    if (!maps(own, kTile) || !maps(other, NarrowTile::other)) return sequence_fail(HTGS_ERR_CUDA, "htgs_attention_backward: the tensor maps cannot be made");
    static PerDeviceOnce once;
    cudaError_t err = once.run([] {
        const cudaError_t e = cudaFuncSetAttribute(attention_narrow_kernel<T, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, NarrowTile::smem);
        return e != cudaSuccess ? e : cudaFuncSetAttribute(attention_narrow_kernel<T, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, NarrowTile::smem);
    });
    const int64_t tiles = sequence_tiles(a, kTile);
    if (err == cudaSuccess) err = launch_after(attention_narrow_kernel<T, true>, dim3(unsigned(tiles * a.key_heads)), kTilesThreads, NarrowTile::smem, stream, own[1], own[2], other[0], other[3], args);
    if (err == cudaSuccess) err = launch_after(attention_narrow_kernel<T, false>, dim3(unsigned(tiles * a.heads)), kTilesThreads, NarrowTile::smem, stream, own[0], own[3], other[1], other[2], args);
    return err == cudaSuccess ? sequence_status("htgs_attention_backward") : sequence_fail(HTGS_ERR_CUDA, cudaGetErrorString(err));
}
template <typename T> int backward_typed(const BackwardArgs& args, cudaStream_t stream) {
    return args.a.width <= kPanel ? launch_narrow<T>(args, stream) : launch_wide<T>(args, stream);
}
template <typename T> int forward_typed(const ForwardArgs& args, cudaStream_t stream) {
    return args.a.width <= kPanel ? launch_forward<T, 1, 1>(args, stream) : launch_forward<T, 2, 2>(args, stream);
}

}  // namespace

bool attention_tiles_take(const HtgsAttention& a, const void* out, const void* rest) {
    return a.type != HTGS_FLOAT32 && a.width % 8 == 0 && aligned(out, 16) && aligned(rest, 16) && heads_aligned(a.q, a.rows, a.heads, a.q_stride, a.q_head_stride) &&
           heads_aligned(a.k, a.rows, a.key_heads, a.k_stride, a.k_head_stride) && heads_aligned(a.v, a.rows, a.key_heads, a.v_stride, a.v_head_stride);
}

bool attention_tiles_take(const HtgsAttention& a, const AttentionBackward& b) {
    return attention_tiles_take(a, b.grad_q, nullptr) && aligned(b.grad_k, 16) && aligned(b.grad_v, 16) && heads_aligned(b.grad, a.rows, a.heads, b.grad_stride, b.grad_head_stride);
}

int attention_tiles_backward(const HtgsAttention& a, const AttentionBackward& b, cudaStream_t stream) {
    unsigned int* error = attention_error_word(current_device());
    if (!error) return sequence_fail(HTGS_ERR_CUDA, "htgs_attention_backward: no host memory for the error word");
    const BackwardArgs args{a, b, error};
    return a.type == HTGS_FLOAT16 ? backward_typed<__half>(args, stream) : backward_typed<__nv_bfloat16>(args, stream);
}

int attention_tiles_forward(const HtgsAttention& a, void* out, void* rest, float* sums, cudaStream_t stream) {
    unsigned int* error = attention_error_word(current_device());
    if (!error) return sequence_fail(HTGS_ERR_CUDA, "htgs_attention: no host memory for the error word");
    const ForwardArgs args{a, out, rest, sums, error};
    return a.type == HTGS_FLOAT16 ? forward_typed<__half>(args, stream) : forward_typed<__nv_bfloat16>(args, stream);
}

}  // namespace htgs
