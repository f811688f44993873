// Gated linear recurrence over long sequences, forward, backward, and one step at a time.
//
//   a = 1 / (1 + exp(-gate));   h_t = a_t h_{t-1} + (1 - a_t) x_t;   h_{-1} = the sequence's initial state
//   backward, from the last row to the first:  D_t = grad_h_t + E_{t+1};   E_t = a_t D_t   (E behind the last row: the last state's gradient)
//       grad_x = (1 - a) D;   grad_gate = D (h_{t-1} - x) a (1 - a);   grad_initial = E at the first row
//
// A step is the map h -> A h + H, and steps compose: (A2, H2) after (A1, H1) is (A1 A2, A2 H1 + H2).  The rows are cut into chunks of 16 to 64.  One
// kernel composes each chunk's rows, one walks from chunk to chunk and leaves the state in front of each, one goes through the
// chunks again from those states and writes h.  The backward pass does the same from the end.  A warp takes a chunk of 64 channels and goes
// through it eight rows at a time, the next on their way into shared memory of its own; warps never wait for one another.  For the backward pass the
// forward one keeps the state in front of every eight rows: h_{t-1} is computed again from there, so it is in 32 bits and neither h nor the rows
// before are read.  A sequence's first row has A = 0 and takes its initial state into H, so packed sequences need no chunks of their own; that zero is
// kept as -0 and tested for, so that a NaN or infinity of one sequence does not reach the next.  States, products and sums are 32-bit; 1 - a is
// exp(-gate) a, which keeps its relative precision where a is close to 1.
//
// Bound by HBM, and x and gate are read twice: a look-back from chunk to chunk in one pass would have to advance a chunk of 64 rows every 15 ns at 128 channels, and one takes
// microseconds.  (Wider rows in longer chunks would give it more time: 120 ns for 256 rows of 512 channels.)  1000000 x 128 in bf16: 86 us first pass (6.0 TB/s), 17 second, 109 third (7.0 TB/s, what L2 still has counted in); 262144 x 512: 91 + 14 + 134 forward,
// 92 + 14 + 221 backward.  Chunks of 64 rows keep every warp of the GPU busy at these sizes; a third pass over rows in registers, without shared memory, took 159 us.
#include "sequence.cuh"

namespace htgs {

namespace {

constexpr int kChannels = 64;                // of a warp, two a lane
constexpr int kBatch = 8;                    // rows that a warp deals with at a time; a state in front of each batch is kept for the backward pass
constexpr int kMostChunk = 64;               // rows
constexpr int kScanWarps = 4, kScanBlock = kScanWarps * 32;
constexpr int kCarryWarps = 32, kCarryChannels = 8, kCarryRun = 16;

struct ScanArgs {
    HtgsScan in;
    int chunk, chunks, channel_tiles;        // rows of a chunk, chunks, and warps side by side
    float2* composed;                        // [chunks, width]
    float* carried;                          // [chunks, width] state in front of each chunk (backward: E behind it); nothing where there is one chunk
    float* states;                           // [ceil(rows / 8), width] state in front of every eight rows, or null
    void* h; int64_t h_stride; float* last;
    const void* grad_h; int64_t grad_h_stride; const float* grad_last;
    void* grad_x; int64_t grad_x_stride; void* grad_gate; int64_t grad_gate_stride; float* grad_initial;
};

// Two channels side by side, in a register pair: one instruction for both.
struct Num {
    f32x2 v;
    __device__ __forceinline__ static Num make(float x, float y) { return {pack2(x, y)}; }
    __device__ __forceinline__ static Num all(float f) { return {pack2(f, f)}; }
    __device__ __forceinline__ float2 get() const { return unpack2(v); }
};
__device__ __forceinline__ Num operator*(Num a, Num b) { return {mul2(a.v, b.v)}; }
__device__ __forceinline__ Num operator+(Num a, Num b) { return {add2(a.v, b.v)}; }
__device__ __forceinline__ Num madd(Num a, Num b, Num c) { return {fma2(a.v, b.v, c.v)}; }

// exp(-g), from the hardware's 2^x (2 units); above exp(80), where a < 2e-35 tells nothing from zero, it stays; a NaN stays one.
__device__ __forceinline__ float exp_negated(float scaled) {        // scaled = -g / ln 2
    float t;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(t) : "f"(scaled), "f"(115.4f));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(t));
    return t;
}
__device__ __forceinline__ float rcp_approx(float x) { float y; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ Num gate_exp(Num g) {
    const float2 scaled = (g * Num::all(-1.4426950408889634f)).get();
    return Num::make(exp_negated(scaled.x), exp_negated(scaled.y));
}
struct Gate { Num a, rest; };                    // a and 1 - a
__device__ __forceinline__ Gate gate_of(Num g) {
    const Num t = gate_exp(g);
    const float2 sum = (t + Num::all(1.0f)).get();
    const Num a = Num::make(rcp_approx(sum.x), rcp_approx(sum.y));
    return {a, t * a};
}

// The map of a sequence's first step takes nothing from the state in front of it: A is -0, which no product of gates is.
constexpr float kCut = -0.0f;
__device__ __forceinline__ bool is_cut(float A) { return __float_as_uint(A) == 0x80000000u; }
__device__ __forceinline__ float follow(float2 m, float state) { return is_cut(m.x) ? m.y : fmaf(m.x, state, m.y); }
__device__ __forceinline__ void compose(float& A, float& H, float2 next) {
    H = follow(next, H);
    A = is_cut(next.x) ? next.x : A * next.x;
}
// Positions p count the rows in the order of the recurrence: row p, or rows - 1 - p in reverse.
// The sequence that holds a position, by its first position and the one behind its last.
struct Span {
    int sequence, begin, end;
    __device__ __forceinline__ void set(const HtgsScan& in) {
        int64_t lo, hi;
        if (in.offsets) { lo = __ldg(in.offsets + sequence); hi = __ldg(in.offsets + sequence + 1); }
        else { const int64_t length = in.n_sequences == 1 ? in.rows : in.rows / in.n_sequences; lo = sequence * length; hi = lo + length; }
        begin = int(in.reverse ? in.rows - hi : lo);
        end = int(in.reverse ? in.rows - lo : hi);
    }
    __device__ __forceinline__ void find(const HtgsScan& in, int p) {
        const int64_t row = in.reverse ? in.rows - 1 - p : p;
        sequence = 0;
        if (in.offsets) {
            int hi = in.n_sequences;
            while (hi - sequence > 1) {
                const int mid = (sequence + hi) >> 1;
                if (__ldg(in.offsets + mid) <= row) sequence = mid; else hi = mid;
            }
        } else if (in.n_sequences > 1) {
            sequence = int(row / (in.rows / in.n_sequences));
        }
        set(in);
    }
    // The next sequence that has rows; forward: behind this one in the order of the recurrence, else in front of it.
    __device__ __forceinline__ void move(const HtgsScan& in, bool forward) {
        const int step = forward != (in.reverse != 0) ? 1 : -1;
        do sequence += step; while (sequence >= 0 && sequence < in.n_sequences && in.offsets && __ldg(in.offsets + sequence + 1) <= __ldg(in.offsets + sequence));
        if (sequence >= 0 && sequence < in.n_sequences) set(in);
        else { sequence = sequence < 0 ? 0 : in.n_sequences - 1; begin = end = -1; }
    }
};

// Where a thread works: two channels side by side, of which `live` exist, positions begin to end - 1.
struct Place {
    int lane, warp, channel0, channel, live, chunk, begin, end;
    __device__ __forceinline__ explicit Place(const ScanArgs& a, bool from_end = false) {
        lane = threadIdx.x & 31; warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0);
        const unsigned int unit = blockIdx.x * kScanWarps + warp, at = unit / unsigned(a.channel_tiles);     // neighbouring channels of a chunk, then the next chunk's
        chunk = from_end ? a.chunks - 1 - int(at) : int(at);
        channel0 = int(unit - at * unsigned(a.channel_tiles)) * kChannels;
        channel = channel0 + lane * 2;
        live = max(0, min(2, a.in.width - channel));
        begin = chunk * a.chunk;
        end = at >= unsigned(a.chunks) ? begin : int(min(int64_t(begin) + a.chunk, a.in.rows));
    }
    __device__ __forceinline__ bool nothing() const { return end <= begin; }
    __device__ __forceinline__ int last_batch() const { return begin + (end - 1 - begin) / kBatch * kBatch; }
    // The thread's channels in row `row` of a matrix of states (null: zeros).
    __device__ __forceinline__ Num load(const float* states, int64_t row, const ScanArgs& a) const {
        const float* p = states + row * a.in.width + channel;
        return Num::make(states && live > 0 ? p[0] : 0.0f, states && live > 1 ? p[1] : 0.0f);
    }
    __device__ __forceinline__ void store(float* states, int64_t row, const ScanArgs& a, Num n) const {
        float* p = states + row * a.in.width + channel;
        const float2 f = n.get();
        if (live > 0) p[0] = f.x;
        if (live > 1) p[1] = f.y;
    }
    __device__ __forceinline__ void leave_map(const ScanArgs& a, Num A, Num H) const {
        float2* p = a.composed + int64_t(chunk) * a.in.width + channel;
        const float2 f = A.get(), h = H.get();
        if (live > 0) p[0] = make_float2(f.x, h.x);
        if (live > 1) p[1] = make_float2(f.y, h.y);
    }
};

// The thread's two values to a matrix; ALIGNED: they begin on a multiple of both, and exist together.
template <typename T, bool ALIGNED> __device__ __forceinline__ void store_pair(T* to, Num n, int live) {
    const float2 f = n.get();
    if (ALIGNED) {
        const float v[2] = {f.x, f.y};
        if (live > 0) store_floats<T, 2>(to, v);
    } else {
        if (live > 0) to[0] = from_float<T>(f.x);
        if (live > 1) to[1] = from_float<T>(f.y);
    }
}

// A matrix's rows at a warp's channels on their way into its shared memory, a batch at a time, 16 bytes at once.  ALIGNED: every row begins on 16 bytes and has a whole
// number of such pieces.  Else the pieces that hold a row are copied, and its values lie up to 15 bytes behind the first one's beginning; what else is in
// those pieces is not looked at (a piece lies in the same 16 bytes of memory as a value that exists, so it can be read).
template <typename T, bool ALIGNED> struct Stream {
    static constexpr int kRow = kChannels * int(sizeof(T)) + (ALIGNED ? 0 : 16);     // bytes
    static constexpr int bytes = kBatch * kRow, kPieces = kRow / 16;
    static constexpr int stages = sizeof(T) == 4 ? 2 : 3;        // batches of a warp in shared memory; with three of 32-bit rows too few warps fit an SM
    const char* first;                        // the channels' first value at position 0
    int64_t step;                             // bytes from position to position
    int valid;                                // bytes of a row that exist
    __device__ __forceinline__ Stream(const void* base, int64_t stride, const ScanArgs& a, const Place& at) {
        first = static_cast<const char*>(base) + ((a.in.reverse ? (a.in.rows - 1) * stride : 0) + at.channel0) * int64_t(sizeof(T));
        step = (a.in.reverse ? -stride : stride) * int64_t(sizeof(T));
        valid = min(kChannels, a.in.width - at.channel0) * int(sizeof(T));
    }
    __device__ __forceinline__ static void piece(uint32_t to, const char* from) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
    }
    __device__ __forceinline__ void copy(unsigned char* to, int p, int count, int lane) const {
        if constexpr (ALIGNED) {
            constexpr int kAtOnce = 32 / kPieces;                 // rows
            const int r = lane / kPieces, c = lane % kPieces * 16;
            const char* from = first + (p + r) * step + c;
            const uint32_t here = smem_u32(to) + uint32_t(r * kRow + c);
            const int there = c < valid ? count - r : 0;
            #pragma unroll
            for (int i = 0; i < kBatch / kAtOnce; ++i, from += kAtOnce * step)
                if (i * kAtOnce < there) piece(here + i * kAtOnce * kRow, from);
        } else {
            #pragma unroll
            for (int i = 0; i < (kBatch * kPieces + 31) / 32; ++i) {
                const int q = lane + 32 * i, r = q / kPieces, w = q % kPieces;
                const char* row = first + (p + r) * step;
                const char* from = row - (reinterpret_cast<uintptr_t>(row) & 15) + 16 * w;
                if (r < count && from < row + valid) piece(smem_u32(to) + uint32_t(r * kRow + 16 * w), from);
            }
        }
    }
    // The thread's channels of row i of a batch that begins at position p.
    __device__ __forceinline__ Num get(const unsigned char* stage, int p, int i, int lane) const {
        const unsigned char* at = stage + i * kRow + lane * 2 * int(sizeof(T));
        float f[2];
        if constexpr (ALIGNED) load_floats<T, 2>(reinterpret_cast<const T*>(at), f);
        else {
            const T* v = reinterpret_cast<const T*>(at + ((uint32_t(reinterpret_cast<uintptr_t>(first)) + uint32_t(p + i) * uint32_t(step)) & 15u));
            f[0] = to_float<T>(v[0]); f[1] = to_float<T>(v[1]);
        }
        return Num::make(f[0], f[1]);
    }
};

// N streams through a ring of stages.  The batches are at positions p, p + kBatch * way, ..., `left` of them.
template <typename S, int N> struct Feed {
    const S (&streams)[N];
    unsigned char* ring;
    int lane, begin, end, p, left, to = 0, from = 0;
    bool back;
    __device__ __forceinline__ void send() {
        if (left > 0) {
            #pragma unroll
            for (int n = 0; n < N; ++n) streams[n].copy(ring + (to * N + n) * S::bytes, p, min(kBatch, end - p), lane);
            p += back ? -kBatch : kBatch;
            --left;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        to = to + 1 == S::stages ? 0 : to + 1;
    }
    __device__ __forceinline__ Feed(const S (&s)[N], unsigned char* memory, int lane_, int begin_, int end_, bool back_)
        : streams(s), ring(memory), lane(lane_), begin(begin_), end(end_), back(back_) {
        left = (end - begin + kBatch - 1) / kBatch;
        p = back ? begin + (left - 1) * kBatch : begin;
        #pragma unroll
        for (int i = 0; i < S::stages - 1; ++i) send();
    }
    // The next batch's place; what was in the stage behind it may be overwritten from here on.
    __device__ __forceinline__ const unsigned char* next() {
        asm volatile("cp.async.wait_group %0;" ::"n"(S::stages - 2) : "memory");
        __syncwarp();
        const unsigned char* stage = ring + from * N * S::bytes;
        from = from + 1 == S::stages ? 0 : from + 1;
        send();
        return stage;
    }
};

template <typename T, bool ALIGNED, int N> constexpr int kFeedBytes = kScanWarps * Stream<T, ALIGNED>::stages * N * Stream<T, ALIGNED>::bytes;

// First pass, forward: the composition of each chunk.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kScanBlock, 10) scan_compose_kernel(const ScanArgs args) {
    extern __shared__ __align__(16) unsigned char memory[];
    using S = Stream<T, ALIGNED>;
    const Place at(args);
    if (at.nothing()) return;
    const S streams[2] = {S(args.in.gate, args.in.gate_stride, args, at), S(args.in.x, args.in.x_stride, args, at)};
    Feed<S, 2> feed(streams, memory + at.warp * S::stages * 2 * S::bytes, at.lane, at.begin, at.end, false);
    Span span;
    span.find(args.in, at.begin);
    Num A = Num::all(1.0f), H = Num::all(0.0f);
    #pragma unroll 1
    for (int p = at.begin; p < at.end; p += kBatch) {
        const unsigned char *g = feed.next(), *x = g + S::bytes;
        if (at.end - p >= kBatch && span.begin < p && span.end >= p + kBatch) {
            #pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const Gate gate = gate_of(streams[0].get(g, p, i, at.lane));
                H = madd(gate.a, H, gate.rest * streams[1].get(x, p, i, at.lane));
                A = A * gate.a;
            }
        } else {
            #pragma unroll 1
            for (int i = 0; i < min(kBatch, at.end - p); ++i) {
                if (p + i == span.end) span.move(args.in, true);
                const Gate gate = gate_of(streams[0].get(g, p, i, at.lane));
                if (p + i == span.begin) {
                    A = Num::all(kCut);
                    H = at.load(args.in.initial, span.sequence, args);
                }
                H = madd(gate.a, H, gate.rest * streams[1].get(x, p, i, at.lane));
                A = A * gate.a;
            }
        }
    }
    at.leave_map(args, A, H);
}

// First pass, backward: E in front of a chunk as a map of E behind it.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kScanBlock, 10) scan_compose_backward_kernel(const ScanArgs args) {
    extern __shared__ __align__(16) unsigned char memory[];
    using S = Stream<T, ALIGNED>;
    const Place at(args);
    if (at.nothing()) return;
    const S streams[2] = {S(args.in.gate, args.in.gate_stride, args, at), S(args.grad_h, args.grad_h_stride, args, at)};
    Feed<S, 2> feed(streams, memory + at.warp * S::stages * 2 * S::bytes, at.lane, at.begin, at.end, true);
    Span span;
    span.find(args.in, at.end - 1);
    Num A = Num::all(1.0f), H = Num::all(0.0f);
    #pragma unroll 1
    for (int p = at.last_batch(); p >= at.begin; p -= kBatch) {
        const unsigned char *g = feed.next(), *d = g + S::bytes;
        if (at.end - p >= kBatch && span.begin <= p && span.end > p + kBatch) {
            #pragma unroll
            for (int i = kBatch - 1; i >= 0; --i) {
                const Num a = gate_of(streams[0].get(g, p, i, at.lane)).a;
                H = a * (H + streams[1].get(d, p, i, at.lane));
                A = A * a;
            }
        } else {
            #pragma unroll 1
            for (int i = min(kBatch, at.end - p) - 1; i >= 0; --i) {
                if (p + i < span.begin) span.move(args.in, false);
                const Num a = gate_of(streams[0].get(g, p, i, at.lane)).a;
                if (p + i + 1 == span.end) {
                    A = Num::all(kCut);
                    H = at.load(args.grad_last, span.sequence, args);
                }
                H = a * (H + streams[1].get(d, p, i, at.lane));
                A = A * a;
            }
        }
    }
    at.leave_map(args, A, H);
}

// Second pass, bound by the latency of its reads: the state at each chunk's beginning (from_end: behind each chunk, walking from the last to the first).  A cluster of `parts` blocks takes eight
// channels.  Each quarter of a warp composes a run of chunks, learns the state in front of it from the quarters, warps and blocks before, and
// goes through its run again.  Up to 16 maps of a run stay in registers, all of them on their way at once; a longer run is read twice.
__global__ void __launch_bounds__(kCarryWarps * 32) scan_carry_kernel(const float2* __restrict__ composed, float* __restrict__ states, int chunks, int width,
                                                                    bool from_end, int parts) {
    constexpr int kQuarters = 32 / kCarryChannels;
    __shared__ float2 shared[kCarryWarps][kCarryChannels];
    __shared__ float2 whole[kCarryChannels];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, at = lane % kCarryChannels, quarter = lane / kCarryChannels;
    const int channel = int(blockIdx.x) / parts * kCarryChannels + at, part = int(blockIdx.x) % parts;
    const bool inside = channel < width;
    grid_dependency();
    const int runs = kCarryWarps * kQuarters * parts, run = (chunks + runs - 1) / runs;
    const int begin = int(min(int64_t((part * kCarryWarps + warp) * kQuarters + quarter) * run, int64_t(chunks))), count = inside ? min(run, chunks - begin) : 0;
    const int64_t first = int64_t(from_end ? chunks - 1 - begin : begin) * width + channel, step = from_end ? -int64_t(width) : width;
    const float2* map = composed + first;
    float* to = states + first;
    float2 maps[kCarryRun];
    float A = 1.0f, H = 0.0f;
    for (int c0 = 0; c0 < run; c0 += kCarryRun) {
        #pragma unroll
        for (int c = 0; c < kCarryRun; ++c, map += step) maps[c] = c0 + c < count ? *map : make_float2(1.0f, 0.0f);
        #pragma unroll
        for (int c = 0; c < kCarryRun; ++c) compose(A, H, maps[c]);
    }
    #pragma unroll
    for (int d = 1; d < kQuarters; d *= 2) {                  // of this quarter and those before
        float P = __shfl_up_sync(0xffffffffu, A, d * kCarryChannels), Q = __shfl_up_sync(0xffffffffu, H, d * kCarryChannels);
        if (quarter >= d) { compose(P, Q, make_float2(A, H)); A = P; H = Q; }
    }
    if (quarter == kQuarters - 1) shared[warp][at] = make_float2(A, H);
    float2 before = make_float2(__shfl_up_sync(0xffffffffu, A, kCarryChannels), __shfl_up_sync(0xffffffffu, H, kCarryChannels));
    if (quarter == 0) before = make_float2(1.0f, 0.0f);
    __syncthreads();
    float state = 0.0f;
    if (parts > 1) {
        if (threadIdx.x < kCarryChannels) {
            float P = 1.0f, Q = 0.0f;
            #pragma unroll
            for (int w = 0; w < kCarryWarps; ++w) compose(P, Q, shared[w][threadIdx.x]);
            whole[threadIdx.x] = make_float2(P, Q);
        }
        cluster_barrier();
        const uint32_t there = smem_u32(&whole[at]);
        for (int p = 0; p < part; ++p) state = follow(make_float2(peer_float(there, p), peer_float(there + 4, p)), state);
        cluster_barrier();               // no block's shared memory goes before the others have read it
    }
    for (int w = 0; w < warp; ++w) state = follow(shared[w][at], state);
    state = follow(before, state);
    map = composed + first;
    for (int c0 = 0; c0 < run; c0 += kCarryRun) {
        if (run > kCarryRun) {
            #pragma unroll
            for (int c = 0; c < kCarryRun; ++c, map += step) maps[c] = c0 + c < count ? *map : make_float2(1.0f, 0.0f);
        }
        #pragma unroll
        for (int c = 0; c < kCarryRun; ++c, to += step) {
            if (c0 + c < count) *to = state;
            state = follow(maps[c], state);
        }
    }
}

// Sequences without rows: their last state is the initial one, and so are the gradients.
__device__ __forceinline__ void pass_empty_sequences(const ScanArgs& args, const float* from, float* to, int chunk, int channel, int v) {
    if (!args.in.offsets || !to) return;
    for (int64_t s = chunk; s < args.in.n_sequences; s += args.chunks)
        if (args.in.offsets[s + 1] <= args.in.offsets[s])
            for (int k = 0; k < v; ++k) to[s * args.in.width + channel + k] = from ? from[s * args.in.width + channel + k] : 0.0f;
}

// Third pass, forward; from the end, where the first pass has left the rows in L2.  Two thirds of the issue slots and the HBM reads are busy.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kScanBlock, 8) scan_apply_kernel(const ScanArgs args) {
    extern __shared__ __align__(16) unsigned char memory[];
    using S = Stream<T, ALIGNED>;
    const Place at(args, true);
    if (at.nothing()) return;
    const S streams[2] = {S(args.in.gate, args.in.gate_stride, args, at), S(args.in.x, args.in.x_stride, args, at)};
    Feed<S, 2> feed(streams, memory + at.warp * S::stages * 2 * S::bytes, at.lane, at.begin, at.end, false);
    grid_dependency();                        // x and gate are older than the first pass, which ended before the second began
    Num h = at.load(args.chunks > 1 ? args.carried : nullptr, at.chunk, args);
    Span span;
    span.find(args.in, at.begin);
    const int64_t step = args.in.reverse ? -args.h_stride : args.h_stride;
    T* to = static_cast<T*>(args.h) + (args.in.reverse ? args.in.rows - 1 - at.begin : at.begin) * args.h_stride + at.channel;
    #pragma unroll 1
    for (int p = at.begin; p < at.end; p += kBatch) {
        const unsigned char *g = feed.next(), *x = g + S::bytes;
        if (args.states) at.store(args.states, p / kBatch, args, h);
        if (at.end - p >= kBatch && span.begin < p && span.end > p + kBatch) {
            #pragma unroll
            for (int i = 0; i < kBatch; ++i, to += step) {
                const Gate gate = gate_of(streams[0].get(g, p, i, at.lane));
                h = madd(gate.a, h, gate.rest * streams[1].get(x, p, i, at.lane));
                store_pair<T, ALIGNED>(to, h, at.live);
            }
        } else {
            #pragma unroll 1
            for (int i = 0; i < min(kBatch, at.end - p); ++i, to += step) {
                if (p + i == span.end) span.move(args.in, true);
                const Gate gate = gate_of(streams[0].get(g, p, i, at.lane));
                if (p + i == span.begin) h = at.load(args.in.initial, span.sequence, args);
                h = madd(gate.a, h, gate.rest * streams[1].get(x, p, i, at.lane));
                store_pair<T, ALIGNED>(to, h, at.live);
                if (p + i + 1 == span.end) at.store(args.last, span.sequence, args, h);
            }
        }
    }
    pass_empty_sequences(args, args.in.initial, args.last, at.chunk, at.channel, at.live);
}

// Third pass, backward: eight rows forward from the state that was kept, then back.  42 instructions a value, 72 % of the issue slots, 5.8 TB/s.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kScanBlock, 5) scan_apply_backward_kernel(const ScanArgs args) {
    extern __shared__ __align__(16) unsigned char memory[];
    using S = Stream<T, ALIGNED>;
    const Place at(args, true);
    if (at.nothing()) return;
    const S streams[3] = {S(args.in.gate, args.in.gate_stride, args, at), S(args.in.x, args.in.x_stride, args, at), S(args.grad_h, args.grad_h_stride, args, at)};
    Feed<S, 3> feed(streams, memory + at.warp * S::stages * 3 * S::bytes, at.lane, at.begin, at.end, true);
    grid_dependency();
    int p = at.last_batch();
    Num kept = at.load(args.states, p / kBatch, args);
    Num E = at.load(args.chunks > 1 ? args.carried : nullptr, at.chunk, args);
    Span span;
    span.find(args.in, at.end - 1);
    const int64_t step_x = args.in.reverse ? -args.grad_x_stride : args.grad_x_stride, step_gate = args.in.reverse ? -args.grad_gate_stride : args.grad_gate_stride;
    const int64_t row = args.in.reverse ? args.in.rows - at.end : at.end - 1;
    T* to_x = static_cast<T*>(args.grad_x) + row * args.grad_x_stride + at.channel;
    T* to_gate = static_cast<T*>(args.grad_gate) + row * args.grad_gate_stride + at.channel;
    const Num minus = Num::all(-1.0f);
    #pragma unroll 1
    for (; p >= at.begin; p -= kBatch) {
        const unsigned char *g = feed.next(), *x = g + S::bytes, *d = x + S::bytes;
        Num h = kept;
        if (p > at.begin) kept = at.load(args.states, p / kBatch - 1, args);
        const int count = min(kBatch, at.end - p);
        Num a[kBatch], rest[kBatch], slope[kBatch];               // slope: (h_{t-1} - x) a (1 - a)
        if (count == kBatch && span.begin < p && span.end > p + kBatch) {
            #pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const Gate gate = gate_of(streams[0].get(g, p, i, at.lane));
                a[i] = gate.a; rest[i] = gate.rest;
                const Num value = streams[1].get(x, p, i, at.lane);
                slope[i] = madd(minus, value, h) * (gate.a * gate.rest);
                h = madd(gate.a, h, gate.rest * value);
            }
            #pragma unroll
            for (int i = kBatch - 1; i >= 0; --i, to_x -= step_x, to_gate -= step_gate) {
                const Num D = streams[2].get(d, p, i, at.lane) + E;
                E = a[i] * D;
                store_pair<T, ALIGNED>(to_x, rest[i] * D, at.live);
                store_pair<T, ALIGNED>(to_gate, slope[i] * D, at.live);
            }
        } else {
            Span ahead;
            ahead.find(args.in, p);
            #pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                if (i >= count) break;
                if (p + i == ahead.end) ahead.move(args.in, true);
                if (p + i == ahead.begin) h = at.load(args.in.initial, ahead.sequence, args);
                const Gate gate = gate_of(streams[0].get(g, p, i, at.lane));
                a[i] = gate.a; rest[i] = gate.rest;
                const Num value = streams[1].get(x, p, i, at.lane);
                slope[i] = madd(minus, value, h) * (gate.a * gate.rest);
                h = madd(gate.a, h, gate.rest * value);
            }
            #pragma unroll
            for (int i = kBatch - 1; i >= 0; --i) {
                if (i >= count) continue;
                if (p + i < span.begin) span.move(args.in, false);
                if (p + i + 1 == span.end) E = at.load(args.grad_last, span.sequence, args);
                const Num D = streams[2].get(d, p, i, at.lane) + E;
                E = a[i] * D;
                store_pair<T, ALIGNED>(to_x, rest[i] * D, at.live);
                store_pair<T, ALIGNED>(to_gate, slope[i] * D, at.live);
                if (p + i == span.begin && args.grad_initial) at.store(args.grad_initial, span.sequence, args, E);
                to_x -= step_x; to_gate -= step_gate;
            }
        }
    }
    pass_empty_sequences(args, args.grad_last, args.grad_initial, at.chunk, at.channel, at.live);
}

// One step for each row, the state updated in place.  Bound by the launch up to some hundred rows (1024 columns in bf16: 64 rows 1.9 us, 256 3.3, 1024 6.0), then by
// instructions, at about half of what HBM gives: 4096 rows 15.8 us, 16384 63.6 (3.7 TB/s).
template <typename T>
__global__ void __launch_bounds__(256) scan_step_kernel(const T* __restrict__ x, int64_t x_stride, const T* __restrict__ gate, int64_t gate_stride, float* state,
                                                       int64_t state_stride, T* h, int64_t h_stride, int64_t rows, int width) {
    const int64_t total = rows * width, step = int64_t(gridDim.x) * 256;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < total; i += step) {
        const int64_t row = i / width, channel = i - row * width;
        const Gate g = gate_of(Num::all(to_float<T>(gate[row * gate_stride + channel])));
        float* s = state + row * state_stride + channel;
        const float next = fmaf(g.a.get().x, *s, g.rest.get().x * to_float<T>(x[row * x_stride + channel]));
        *s = next;
        h[row * h_stride + channel] = from_float<T>(next);
    }
}

size_t align256(size_t n) { return (n + 255) & ~size_t(255); }
int64_t pieces(int64_t rows, int piece) { return (rows + piece - 1) / piece; }

cudaError_t launch_carry(const ScanArgs& args, bool from_end, cudaStream_t stream) {
    int parts = 1;                             // eight chunks in a run, and at most eight blocks
    while (parts < 8 && args.chunks > kCarryWarps * (32 / kCarryChannels) * 8 * parts) parts *= 2;
    cudaLaunchAttribute attributes[2]{};
    attributes[0].id = cudaLaunchAttributeClusterDimension;
    attributes[0].val.clusterDim.x = unsigned(parts); attributes[0].val.clusterDim.y = attributes[0].val.clusterDim.z = 1;
    attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = unsigned((args.in.width + kCarryChannels - 1) / kCarryChannels * parts); config.blockDim = kCarryWarps * 32; config.stream = stream;
    config.attrs = attributes; config.numAttrs = 2;
    return cudaLaunchKernelEx(&config, scan_carry_kernel, static_cast<const float2*>(args.composed), args.carried, args.chunks, int(args.in.width), from_end, parts);
}

// Rows of a chunk: the most, up to 64, that give every SM 32 warps, but at least 16; a few rows are one chunk, whose state needs no walk.
int chunk_rows(int64_t rows, int64_t tiles) {
    if (rows <= kMostChunk) return kMostChunk;
    int chunk = kMostChunk;
    while (chunk > 16 && pieces(rows, chunk) * tiles < 148 * 32) chunk /= 2;
    return chunk;
}
int64_t chunk_count(int64_t rows, int64_t width) { return pieces(rows, chunk_rows(rows, pieces(width, kChannels))); }

// `behind`: close behind the kernel before, for which the kernel waits itself.
template <typename K> cudaError_t launch_chunks(K kernel, PerDeviceOnce& once, const ScanArgs& args, int smem, bool behind, cudaStream_t stream) {
    const cudaError_t err = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
    if (err != cudaSuccess) return err;
    const unsigned int blocks = unsigned(pieces(int64_t(args.chunks) * args.channel_tiles, kScanWarps));
    if (behind) return launch_after(kernel, blocks, kScanBlock, smem, stream, args);
    kernel<<<blocks, kScanBlock, smem, stream>>>(args);
    return cudaSuccess;
}

template <typename T, bool ALIGNED> cudaError_t scan_launch(ScanArgs& args, bool backward, cudaStream_t stream) {
    static PerDeviceOnce compose, apply, compose_backward, apply_backward;
    constexpr int two = kFeedBytes<T, ALIGNED, 2>, three = kFeedBytes<T, ALIGNED, 3>;
    args.channel_tiles = int(pieces(args.in.width, kChannels));
    args.chunk = chunk_rows(args.in.rows, args.channel_tiles);
    args.chunks = int(pieces(args.in.rows, args.chunk));
    cudaError_t err = cudaSuccess;
    if (args.chunks > 1) {
        err = backward ? launch_chunks(scan_compose_backward_kernel<T, ALIGNED>, compose_backward, args, two, false, stream)
                       : launch_chunks(scan_compose_kernel<T, ALIGNED>, compose, args, two, false, stream);
        if (err == cudaSuccess) err = launch_carry(args, backward, stream);
    }
    if (err != cudaSuccess) return err;
    return backward ? launch_chunks(scan_apply_backward_kernel<T, ALIGNED>, apply_backward, args, three, args.chunks > 1, stream)
                    : launch_chunks(scan_apply_kernel<T, ALIGNED>, apply, args, two, args.chunks > 1, stream);
}

template <typename T> int scan_typed(ScanArgs& a, bool backward, cudaStream_t stream) {
    const auto one = [&](const void* p, int64_t stride) { return !p || rows_aligned(p, stride, a.in.rows, sizeof(T), 16); };
    const bool whole = size_t(a.in.width) * sizeof(T) % 16 == 0 && one(a.in.x, a.in.x_stride) && one(a.in.gate, a.in.gate_stride) && one(a.h, a.h_stride) &&
                       one(a.grad_h, a.grad_h_stride) && one(a.grad_x, a.grad_x_stride) && one(a.grad_gate, a.grad_gate_stride);
    const cudaError_t err = whole ? scan_launch<T, true>(a, backward, stream) : scan_launch<T, false>(a, backward, stream);
    return err == cudaSuccess ? sequence_status("htgs_gated_scan") : sequence_fail(HTGS_ERR_CUDA, cudaGetErrorString(err));
}

constexpr int64_t kMostStride = 1 << 22;      // elements: 128 rows of it are within 32 bits' worth of bytes
bool stride_ok(int64_t stride) { return stride >= 0 && stride <= kMostStride; }

int check_scan(const HtgsScan* scan, const char* message) {
    if (!scan || !known_type(scan->type) || scan->rows < 0 || scan->rows > 0x7fffff00 || !stride_ok(scan->x_stride) || !stride_ok(scan->gate_stride) || scan->width < 1 || scan->width > 65536 || scan->n_sequences < 1 ||
        (!scan->offsets && scan->rows % scan->n_sequences != 0) || (scan->rows > 0 && (!scan->x || !scan->gate)))
        return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, message);
    if (pieces(scan->rows, kMostChunk) * ((scan->width + 31) / 32) > 0x7fffffff) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, message);
    return HTGS_OK;
}

int pass_states(const float* from, float* to, const HtgsScan* scan, cudaStream_t stream) {     // no rows at all
    const size_t bytes = size_t(scan->n_sequences) * scan->width * sizeof(float);
    const cudaError_t err = !to ? cudaSuccess : from ? cudaMemcpyAsync(to, from, bytes, cudaMemcpyDeviceToDevice, stream) : cudaMemsetAsync(to, 0, bytes, stream);
    return err == cudaSuccess ? HTGS_OK : sequence_fail(HTGS_ERR_CUDA, cudaGetErrorString(err));
}

}  // namespace

}  // namespace htgs

extern "C" {

size_t htgs_gated_scan_state_bytes(int64_t rows, int32_t width) {
    return rows <= 0 || width <= 0 ? 0 : size_t(htgs::pieces(rows, htgs::kBatch)) * size_t(width) * sizeof(float);
}

size_t htgs_gated_scan_workspace_bytes(int64_t rows, int32_t width) {
    if (rows <= 0 || width <= 0) return 0;
    const size_t values = size_t(htgs::chunk_count(rows, width)) * size_t(width);
    return htgs::align256(values * sizeof(float2)) + htgs::align256(values * sizeof(float));
}

int htgs_gated_scan(const HtgsScan* scan, void* h, int64_t h_stride, float* last, float* states, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace htgs;
    if (check_scan(scan, "htgs_gated_scan: bad type, sizes, sequences or null inputs") != HTGS_OK) return HTGS_ERR_INVALID_ARGUMENT;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (!last) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_gated_scan: last must not be null");
    if (scan->rows == 0) return pass_states(scan->initial, last, scan, s);
    if (!h) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_gated_scan: h must not be null");
    if (!stride_ok(h_stride)) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_gated_scan: row strides are from 0 to 2^22");
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < htgs_gated_scan_workspace_bytes(scan->rows, scan->width))
        return sequence_fail(HTGS_ERR_WORKSPACE_TOO_SMALL, "htgs_gated_scan: workspace too small or not 16-byte aligned");
    ScanArgs a{};
    a.in = *scan;
    a.composed = static_cast<float2*>(workspace);
    a.carried = reinterpret_cast<float*>(static_cast<char*>(workspace) + align256(size_t(chunk_count(scan->rows, scan->width)) * size_t(scan->width) * sizeof(float2)));
    a.states = states;
    a.h = h; a.h_stride = h_stride; a.last = last;
    if (scan->type == HTGS_FLOAT32) return scan_typed<float>(a, false, s);
    if (scan->type == HTGS_FLOAT16) return scan_typed<__half>(a, false, s);
    return scan_typed<__nv_bfloat16>(a, false, s);
}

int htgs_gated_scan_backward(const HtgsScan* scan, const float* states, const void* grad_h, int64_t grad_h_stride, const float* grad_last, void* grad_x,
                             int64_t grad_x_stride, void* grad_gate, int64_t grad_gate_stride, float* grad_initial, void* workspace, size_t workspace_bytes,
                             void* stream) {
    using namespace htgs;
    if (check_scan(scan, "htgs_gated_scan_backward: bad type, sizes, sequences or null inputs") != HTGS_OK) return HTGS_ERR_INVALID_ARGUMENT;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (scan->rows == 0) return pass_states(grad_last, grad_initial, scan, s);
    if (!states || !grad_h || !grad_x || !grad_gate) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_gated_scan_backward: null pointer");
    if (!stride_ok(grad_h_stride) || !stride_ok(grad_x_stride) || !stride_ok(grad_gate_stride))
        return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_gated_scan_backward: row strides are from 0 to 2^22");
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < htgs_gated_scan_workspace_bytes(scan->rows, scan->width))
        return sequence_fail(HTGS_ERR_WORKSPACE_TOO_SMALL, "htgs_gated_scan_backward: workspace too small or not 16-byte aligned");
    ScanArgs a{};
    a.in = *scan;
    a.composed = static_cast<float2*>(workspace);
    a.carried = reinterpret_cast<float*>(static_cast<char*>(workspace) + align256(size_t(chunk_count(scan->rows, scan->width)) * size_t(scan->width) * sizeof(float2)));
    a.states = const_cast<float*>(states);
    a.grad_h = grad_h; a.grad_h_stride = grad_h_stride; a.grad_last = grad_last;
    a.grad_x = grad_x; a.grad_x_stride = grad_x_stride; a.grad_gate = grad_gate; a.grad_gate_stride = grad_gate_stride; a.grad_initial = grad_initial;
    if (scan->type == HTGS_FLOAT32) return scan_typed<float>(a, true, s);
    if (scan->type == HTGS_FLOAT16) return scan_typed<__half>(a, true, s);
    return scan_typed<__nv_bfloat16>(a, true, s);
}

int htgs_gated_scan_step(const void* x, int64_t x_stride, const void* gate, int64_t gate_stride, float* state, int64_t state_stride, void* h,
                         int64_t h_stride, int type, int64_t rows, int32_t width, void* stream) {
    using namespace htgs;
    if (!known_type(type) || rows < 0 || rows > 0x7fffffff || width < 1) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_gated_scan_step: bad type or sizes");
    if (rows == 0) return HTGS_OK;
    if (!x || !gate || !state || !h) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_gated_scan_step: null pointer");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int64_t wanted = (rows * width + 255) / 256;
    const unsigned int blocks = unsigned(wanted < 148 * 8 ? wanted : 148 * 8);
    if (type == HTGS_FLOAT32)
        scan_step_kernel<float><<<blocks, 256, 0, s>>>(static_cast<const float*>(x), x_stride, static_cast<const float*>(gate), gate_stride, state, state_stride,
                                                       static_cast<float*>(h), h_stride, rows, width);
    else if (type == HTGS_FLOAT16)
        scan_step_kernel<__half><<<blocks, 256, 0, s>>>(static_cast<const __half*>(x), x_stride, static_cast<const __half*>(gate), gate_stride, state, state_stride,
                                                        static_cast<__half*>(h), h_stride, rows, width);
    else
        scan_step_kernel<__nv_bfloat16><<<blocks, 256, 0, s>>>(static_cast<const __nv_bfloat16*>(x), x_stride, static_cast<const __nv_bfloat16*>(gate), gate_stride,
                                                               state, state_stride, static_cast<__nv_bfloat16*>(h), h_stride, rows, width);
    return sequence_status("htgs_gated_scan_step");
}

}  // extern "C"
