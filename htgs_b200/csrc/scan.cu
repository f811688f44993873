// Gated linear recurrence over long sequences, forward, backward, and one step at a time.
//
//   a = 1 / (1 + exp(-gate));   h_t = a_t h_{t-1} + (1 - a_t) x_t;   h_{-1} = the sequence's initial state
//   backward, from the last row to the first:  D_t = grad_h_t + E_{t+1};   E_t = a_t D_t   (E behind the last row: the last state's gradient)
//       grad_x = (1 - a) D;   grad_gate = D (h_{t-1} - x) a (1 - a);   grad_initial = E at the first row
//
// A step is the map h -> A h + H, and steps compose: (A2, H2) after (A1, H1) is (A1 A2, A2 H1 + H2).  The rows are cut into chunks of 16 to 64.  One
// kernel composes each chunk's rows, one walks from chunk to chunk and leaves the state in front of each, one goes through the
// chunks again from those states and writes h.  The backward pass does the same from the end.  A warp takes a chunk of 32 or 64 channels and goes
// through it eight rows at a time, the next sixteen on their way into shared memory of its own; warps never wait for one another.  For the backward pass the
// forward one keeps the state in front of every eight rows: h_{t-1} is computed again from there, so it is in 32 bits and neither h nor the rows
// before are read.  A sequence's first row has A = 0 and takes its initial state into H, so packed sequences need no chunks of their own; that zero is
// kept as -0 and tested for, so that a NaN or infinity of one sequence does not reach the next.  States, products and sums are 32-bit; 1 - a is
// exp(-gate) a, which keeps its relative precision where a is close to 1.
//
#include "sequence.cuh"

namespace htgs {

namespace {

constexpr int kBatch = 8;                    // rows that a warp deals with at a time; a state in front of each batch is kept for the backward pass
constexpr int kMostChunk = 64;               // rows
constexpr int kStages = 3;                   // batches of a warp in shared memory
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

// V channels side by side: one float, or two in a register pair (one instruction for both).
template <int V> struct Num;
template <> struct Num<1> {
    float v;
    __device__ __forceinline__ static Num make(const float (&f)[1]) { return {f[0]}; }
    __device__ __forceinline__ static Num all(float f) { return {f}; }
    __device__ __forceinline__ float operator[](int) const { return v; }
};
template <> struct Num<2> {
    f32x2 v;
    __device__ __forceinline__ static Num make(const float (&f)[2]) { return {pack2(f[0], f[1])}; }
    __device__ __forceinline__ static Num all(float f) { return {pack2(f, f)}; }
    __device__ __forceinline__ float operator[](int i) const { const float2 f = unpack2(v); return i ? f.y : f.x; }
};
__device__ __forceinline__ Num<1> operator*(Num<1> a, Num<1> b) { return {a.v * b.v}; }
__device__ __forceinline__ Num<1> operator+(Num<1> a, Num<1> b) { return {a.v + b.v}; }
__device__ __forceinline__ Num<1> madd(Num<1> a, Num<1> b, Num<1> c) { return {fmaf(a.v, b.v, c.v)}; }
__device__ __forceinline__ Num<2> operator*(Num<2> a, Num<2> b) { return {mul2(a.v, b.v)}; }
__device__ __forceinline__ Num<2> operator+(Num<2> a, Num<2> b) { return {add2(a.v, b.v)}; }
__device__ __forceinline__ Num<2> madd(Num<2> a, Num<2> b, Num<2> c) { return {fma2(a.v, b.v, c.v)}; }

// exp(-g), from the hardware's 2^x (2 units); above exp(80), where a < 2e-35 tells nothing from zero, it stays; a NaN stays one.
__device__ __forceinline__ float exp_negated(float scaled) {        // scaled = -g / ln 2
    float t;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(t) : "f"(scaled), "f"(115.4f));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(t));
    return t;
}
__device__ __forceinline__ float rcp_approx(float x) { float y; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
template <int V> __device__ __forceinline__ Num<V> gate_exp(Num<V> g) {
    const Num<V> scaled = g * Num<V>::all(-1.4426950408889634f);
    float t[V];
    #pragma unroll
    for (int k = 0; k < V; ++k) t[k] = exp_negated(scaled[k]);
    return Num<V>::make(t);
}
template <int V> struct Gate { Num<V> a, rest; };                    // a and 1 - a
template <int V> __device__ __forceinline__ Gate<V> gate_of(Num<V> t) {
    const Num<V> sum = t + Num<V>::all(1.0f);
    float a[V];
    #pragma unroll
    for (int k = 0; k < V; ++k) a[k] = rcp_approx(sum[k]);
    const Num<V> A = Num<V>::make(a);
    return {A, t * A};
}
template <typename T, int V> __device__ __forceinline__ Num<V> number(const Pack<T, V>& p) { float f[V]; to_floats<T, V>(p, f); return Num<V>::make(f); }
template <typename T, int V> __device__ __forceinline__ void store_number(T* p, Num<V> n) {
    float f[V];
    #pragma unroll
    for (int k = 0; k < V; ++k) f[k] = n[k];
    store_floats<T, V>(p, f);
}

// The map of a sequence's first step takes nothing from the state in front of it: A is -0, which no product of gates is.
constexpr float kCut = -0.0f;
__device__ __forceinline__ bool is_cut(float A) { return __float_as_uint(A) == 0x80000000u; }
__device__ __forceinline__ float follow(float2 m, float state) { return is_cut(m.x) ? m.y : fmaf(m.x, state, m.y); }
__device__ __forceinline__ void compose(float& A, float& H, float2 next) {
    H = follow(next, H);
    A = is_cut(next.x) ? next.x : A * next.x;
}
template <int V> __device__ __forceinline__ Num<V> follow(const float2* maps, Num<V> state) {
    float f[V];
    #pragma unroll
    for (int k = 0; k < V; ++k) f[k] = follow(maps[k], state[k]);
    return Num<V>::make(f);
}
template <int V> __device__ __forceinline__ void leave_map(float2* to, Num<V> A, Num<V> H) {
    #pragma unroll
    for (int k = 0; k < V; ++k) to[k] = make_float2(A[k], H[k]);
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

template <int V> __device__ __forceinline__ Num<V> load_state(const float* states, int64_t at) {
    float f[V];
    #pragma unroll
    for (int k = 0; k < V; ++k) f[k] = states ? states[at + k] : 0.0f;
    return Num<V>::make(f);
}
template <int V> __device__ __forceinline__ void store_state(float* states, int64_t at, Num<V> n) {
    #pragma unroll
    for (int k = 0; k < V; ++k) states[at + k] = n[k];
}

// Where a thread works: V channels side by side, positions begin to end - 1.
template <int V> struct Place {
    int lane, warp, channel0, channel, chunk, begin, end;
    bool inside;
    __device__ __forceinline__ explicit Place(const ScanArgs& a, bool from_end = false) {
        lane = threadIdx.x & 31; warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0);
        const unsigned int unit = blockIdx.x * kScanWarps + warp, at = unit / unsigned(a.channel_tiles);     // neighbouring channels of a chunk, then the next chunk's
        chunk = from_end ? a.chunks - 1 - int(at) : int(at);
        channel0 = int(unit - at * unsigned(a.channel_tiles)) * 32 * V;
        channel = channel0 + lane * V;
        inside = channel < a.in.width;
        begin = chunk * a.chunk;
        end = at >= unsigned(a.chunks) ? begin : int(min(int64_t(begin) + a.chunk, a.in.rows));
    }
    __device__ __forceinline__ bool nothing() const { return end <= begin; }
    __device__ __forceinline__ int last_batch() const { return begin + (end - 1 - begin) / kBatch * kBatch; }
    __device__ __forceinline__ int64_t state_at(const ScanArgs& a, int sequence) const { return int64_t(sequence) * a.in.width + channel; }
};

// A matrix's rows at a warp's channels on their way into its shared memory, a batch at a time, PIECE bytes at once: 16 where every row of the matrix allows it, or
// 4.  PIECE 2 is for 16-bit rows that begin on 2 bytes: the 4-byte words that hold a row are copied, and its values lie 0 or 2 bytes behind the first.
template <typename T, int V, int PIECE> struct Stream {
    static constexpr int kRow = PIECE == 2 ? 68 : 32 * V * int(sizeof(T));         // bytes
    static constexpr int bytes = kBatch * kRow;
    static constexpr int kPieces = PIECE == 2 ? 17 : kRow / PIECE;
    const char* first;                        // the channels' first value at position 0
    int64_t step;                             // bytes from position to position
    int valid;                                // bytes of a row that exist
    __device__ __forceinline__ Stream(const void* base, int64_t stride, const ScanArgs& a, const Place<V>& at) {
        first = static_cast<const char*>(base) + ((a.in.reverse ? (a.in.rows - 1) * stride : 0) + at.channel0) * int64_t(sizeof(T));
        step = (a.in.reverse ? -stride : stride) * int64_t(sizeof(T));
        valid = min(32 * V, a.in.width - at.channel0) * int(sizeof(T));
    }
    __device__ __forceinline__ void copy(unsigned char* to, int p, int count, int lane) const {
        if constexpr (PIECE == 2) {
            #pragma unroll
            for (int i = 0; i < (kBatch * kPieces + 31) / 32; ++i) {
                const int q = lane + 32 * i, r = q / kPieces, w = q % kPieces;
                const uintptr_t row = reinterpret_cast<uintptr_t>(first + (p + r) * step), word = (row & ~uintptr_t(3)) + 4 * w;
                if (r < count && word < row + valid) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(to + r * kRow + 4 * w)), "l"(word) : "memory");
            }
        } else {
            constexpr int kAtOnce = 32 / kPieces;                 // rows
            const int r = lane / kPieces, c = lane % kPieces * PIECE;
            const char* from = first + (p + r) * step + c;
            const uint32_t here = smem_u32(to) + uint32_t(r * kRow + c);
            const int there = c < valid ? count - r : 0;
            #pragma unroll
            for (int i = 0; i < kBatch / kAtOnce; ++i, from += kAtOnce * step) {
                if (i * kAtOnce >= there) continue;
                if constexpr (PIECE == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(here + i * kAtOnce * kRow), "l"(from) : "memory");
                else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(here + i * kAtOnce * kRow), "l"(from) : "memory");
            }
        }
    }
    // The thread's channels of row i of a batch that begins at position p.
    __device__ __forceinline__ Num<V> get(const unsigned char* stage, int p, int i, int lane) const {
        if constexpr (PIECE == 2) {
            const uint32_t off = uint32_t(reinterpret_cast<uintptr_t>(first)) + uint32_t(p + i) * uint32_t(step) & 2u;
            return number<T, V>(*reinterpret_cast<const Pack<T, V>*>(stage + i * kRow + off + lane * V * int(sizeof(T))));
        } else {
            return number<T, V>(*reinterpret_cast<const Pack<T, V>*>(stage + i * kRow + lane * V * int(sizeof(T))));
        }
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
        to = to + 1 == kStages ? 0 : to + 1;
    }
    __device__ __forceinline__ Feed(const S (&s)[N], unsigned char* memory, int lane_, int begin_, int end_, bool back_)
        : streams(s), ring(memory), lane(lane_), begin(begin_), end(end_), back(back_) {
        left = (end - begin + kBatch - 1) / kBatch;
        p = back ? begin + (left - 1) * kBatch : begin;
        #pragma unroll
        for (int i = 0; i < kStages - 1; ++i) send();
    }
    // The next batch's place; what was in the stage behind it may be overwritten from here on.
    __device__ __forceinline__ const unsigned char* next() {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        __syncwarp();
        const unsigned char* stage = ring + from * N * S::bytes;
        from = from + 1 == kStages ? 0 : from + 1;
        send();
        return stage;
    }
};

template <typename T, int V, int PIECE, int N> constexpr int kFeedBytes = kScanWarps * kStages * N * Stream<T, V, PIECE>::bytes;

// First pass, forward: the composition of each chunk.
template <typename T, int V, int PIECE>
__global__ void __launch_bounds__(kScanBlock, 10) scan_compose_kernel(const ScanArgs args) {
    extern __shared__ __align__(16) unsigned char memory[];
    using S = Stream<T, V, PIECE>;
    const Place<V> at(args);
    if (at.nothing()) return;
    const S streams[2] = {S(args.in.gate, args.in.gate_stride, args, at), S(args.in.x, args.in.x_stride, args, at)};
    Feed<S, 2> feed(streams, memory + at.warp * kStages * 2 * S::bytes, at.lane, at.begin, at.end, false);
    Span span;
    span.find(args.in, at.begin);
    Num<V> A = Num<V>::all(1.0f), H = Num<V>::all(0.0f);
    #pragma unroll 1
    for (int p = at.begin; p < at.end; p += kBatch) {
        const unsigned char *g = feed.next(), *x = g + S::bytes;
        if (at.end - p >= kBatch && span.begin < p && span.end >= p + kBatch) {
            #pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const Gate<V> gate = gate_of<V>(gate_exp<V>(streams[0].get(g, p, i, at.lane)));
                H = madd(gate.a, H, gate.rest * streams[1].get(x, p, i, at.lane));
                A = A * gate.a;
            }
        } else {
            #pragma unroll 1
            for (int i = 0; i < min(kBatch, at.end - p); ++i) {
                if (p + i == span.end) span.move(args.in, true);
                const Gate<V> gate = gate_of<V>(gate_exp<V>(streams[0].get(g, p, i, at.lane)));
                if (p + i == span.begin) {
                    A = Num<V>::all(kCut);
                    H = load_state<V>(at.inside ? args.in.initial : nullptr, at.state_at(args, span.sequence));
                }
                H = madd(gate.a, H, gate.rest * streams[1].get(x, p, i, at.lane));
                A = A * gate.a;
            }
        }
    }
    if (at.inside) leave_map<V>(&args.composed[int64_t(at.chunk) * args.in.width + at.channel], A, H);
}

// First pass, backward: E in front of a chunk as a map of E behind it.
template <typename T, int V, int PIECE>
__global__ void __launch_bounds__(kScanBlock, 10) scan_compose_backward_kernel(const ScanArgs args) {
    extern __shared__ __align__(16) unsigned char memory[];
    using S = Stream<T, V, PIECE>;
    const Place<V> at(args);
    if (at.nothing()) return;
    const S streams[2] = {S(args.in.gate, args.in.gate_stride, args, at), S(args.grad_h, args.grad_h_stride, args, at)};
    Feed<S, 2> feed(streams, memory + at.warp * kStages * 2 * S::bytes, at.lane, at.begin, at.end, true);
    Span span;
    span.find(args.in, at.end - 1);
    Num<V> A = Num<V>::all(1.0f), H = Num<V>::all(0.0f);
    #pragma unroll 1
    for (int p = at.last_batch(); p >= at.begin; p -= kBatch) {
        const unsigned char *g = feed.next(), *d = g + S::bytes;
        if (at.end - p >= kBatch && span.begin <= p && span.end > p + kBatch) {
            #pragma unroll
            for (int i = kBatch - 1; i >= 0; --i) {
                const Num<V> a = gate_of<V>(gate_exp<V>(streams[0].get(g, p, i, at.lane))).a;
                H = a * (H + streams[1].get(d, p, i, at.lane));
                A = A * a;
            }
        } else {
            #pragma unroll 1
            for (int i = min(kBatch, at.end - p) - 1; i >= 0; --i) {
                if (p + i < span.begin) span.move(args.in, false);
                const Num<V> a = gate_of<V>(gate_exp<V>(streams[0].get(g, p, i, at.lane))).a;
                if (p + i + 1 == span.end) {
                    A = Num<V>::all(kCut);
                    H = load_state<V>(at.inside ? args.grad_last : nullptr, at.state_at(args, span.sequence));
                }
                H = a * (H + streams[1].get(d, p, i, at.lane));
                A = A * a;
            }
        }
    }
    if (at.inside) leave_map<V>(&args.composed[int64_t(at.chunk) * args.in.width + at.channel], A, H);
}

// Second pass: the state at each chunk's beginning (from_end: behind each chunk, walking from the last to the first).  A cluster of `parts` blocks takes eight
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

// Third pass, forward; from the end, where the first pass has left the rows in L2.
template <typename T, int V, int PIECE>
__global__ void __launch_bounds__(kScanBlock, 8) scan_apply_kernel(const ScanArgs args) {
    extern __shared__ __align__(16) unsigned char memory[];
    using S = Stream<T, V, PIECE>;
    const Place<V> at(args, true);
    if (at.nothing()) return;
    const S streams[2] = {S(args.in.gate, args.in.gate_stride, args, at), S(args.in.x, args.in.x_stride, args, at)};
    Feed<S, 2> feed(streams, memory + at.warp * kStages * 2 * S::bytes, at.lane, at.begin, at.end, false);
    grid_dependency();                        // x and gate are older than the first pass, which ended before the second began
    Num<V> h = load_state<V>(args.chunks > 1 && at.inside ? args.carried : nullptr, int64_t(at.chunk) * args.in.width + at.channel);
    Span span;
    span.find(args.in, at.begin);
    const int64_t step = args.in.reverse ? -args.h_stride : args.h_stride;
    T* to = static_cast<T*>(args.h) + (args.in.reverse ? args.in.rows - 1 - at.begin : at.begin) * args.h_stride + at.channel;
    #pragma unroll 1
    for (int p = at.begin; p < at.end; p += kBatch) {
        const unsigned char *g = feed.next(), *x = g + S::bytes;
        if (args.states && at.inside) store_state<V>(args.states, int64_t(p / kBatch) * args.in.width + at.channel, h);
        if (at.end - p >= kBatch && span.begin < p && span.end > p + kBatch) {
            #pragma unroll
            for (int i = 0; i < kBatch; ++i, to += step) {
                const Gate<V> gate = gate_of<V>(gate_exp<V>(streams[0].get(g, p, i, at.lane)));
                h = madd(gate.a, h, gate.rest * streams[1].get(x, p, i, at.lane));
                if (at.inside) store_number<T, V>(to, h);
            }
        } else {
            #pragma unroll 1
            for (int i = 0; i < min(kBatch, at.end - p); ++i, to += step) {
                if (p + i == span.end) span.move(args.in, true);
                const Gate<V> gate = gate_of<V>(gate_exp<V>(streams[0].get(g, p, i, at.lane)));
                if (p + i == span.begin) h = load_state<V>(at.inside ? args.in.initial : nullptr, at.state_at(args, span.sequence));
                h = madd(gate.a, h, gate.rest * streams[1].get(x, p, i, at.lane));
                if (at.inside) {
                    store_number<T, V>(to, h);
                    if (p + i + 1 == span.end) store_state<V>(args.last, at.state_at(args, span.sequence), h);
                }
            }
        }
    }
    if (at.inside) pass_empty_sequences(args, args.in.initial, args.last, at.chunk, at.channel, V);
}

// Third pass, backward: eight rows forward from the state that was kept, then back.
template <typename T, int V, int PIECE>
__global__ void __launch_bounds__(kScanBlock, 5) scan_apply_backward_kernel(const ScanArgs args) {
    extern __shared__ __align__(16) unsigned char memory[];
    using S = Stream<T, V, PIECE>;
    const Place<V> at(args, true);
    if (at.nothing()) return;
    const S streams[3] = {S(args.in.gate, args.in.gate_stride, args, at), S(args.in.x, args.in.x_stride, args, at), S(args.grad_h, args.grad_h_stride, args, at)};
    Feed<S, 3> feed(streams, memory + at.warp * kStages * 3 * S::bytes, at.lane, at.begin, at.end, true);
    grid_dependency();
    int p = at.last_batch();
    Num<V> kept = load_state<V>(at.inside ? args.states : nullptr, int64_t(p / kBatch) * args.in.width + at.channel);
    Num<V> E = load_state<V>(args.chunks > 1 && at.inside ? args.carried : nullptr, int64_t(at.chunk) * args.in.width + at.channel);
    Span span;
    span.find(args.in, at.end - 1);
    const int64_t step_x = args.in.reverse ? -args.grad_x_stride : args.grad_x_stride, step_gate = args.in.reverse ? -args.grad_gate_stride : args.grad_gate_stride;
    const int64_t row = args.in.reverse ? args.in.rows - at.end : at.end - 1;
    T* to_x = static_cast<T*>(args.grad_x) + row * args.grad_x_stride + at.channel;
    T* to_gate = static_cast<T*>(args.grad_gate) + row * args.grad_gate_stride + at.channel;
    const Num<V> minus = Num<V>::all(-1.0f);
    #pragma unroll 1
    for (; p >= at.begin; p -= kBatch) {
        const unsigned char *g = feed.next(), *x = g + S::bytes, *d = x + S::bytes;
        Num<V> h = kept;
        if (p > at.begin) kept = load_state<V>(at.inside ? args.states : nullptr, int64_t(p / kBatch - 1) * args.in.width + at.channel);
        const int count = min(kBatch, at.end - p);
        Num<V> a[kBatch], rest[kBatch], slope[kBatch];               // slope: (h_{t-1} - x) a (1 - a)
        if (count == kBatch && span.begin < p && span.end > p + kBatch) {
            #pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const Gate<V> gate = gate_of<V>(gate_exp<V>(streams[0].get(g, p, i, at.lane)));
                a[i] = gate.a; rest[i] = gate.rest;
                const Num<V> value = streams[1].get(x, p, i, at.lane);
                slope[i] = madd(minus, value, h) * (gate.a * gate.rest);
                h = madd(gate.a, h, gate.rest * value);
            }
            #pragma unroll
            for (int i = kBatch - 1; i >= 0; --i, to_x -= step_x, to_gate -= step_gate) {
                const Num<V> D = streams[2].get(d, p, i, at.lane) + E;
                E = a[i] * D;
                if (at.inside) {
                    store_number<T, V>(to_x, rest[i] * D);
                    store_number<T, V>(to_gate, slope[i] * D);
                }
            }
        } else {
            Span ahead;
            ahead.find(args.in, p);
            #pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                if (i >= count) break;
                if (p + i == ahead.end) ahead.move(args.in, true);
                if (p + i == ahead.begin) h = load_state<V>(at.inside ? args.in.initial : nullptr, at.state_at(args, ahead.sequence));
                const Gate<V> gate = gate_of<V>(gate_exp<V>(streams[0].get(g, p, i, at.lane)));
                a[i] = gate.a; rest[i] = gate.rest;
                const Num<V> value = streams[1].get(x, p, i, at.lane);
                slope[i] = madd(minus, value, h) * (gate.a * gate.rest);
                h = madd(gate.a, h, gate.rest * value);
            }
            #pragma unroll
            for (int i = kBatch - 1; i >= 0; --i) {
                if (i >= count) continue;
                if (p + i < span.begin) span.move(args.in, false);
                if (p + i + 1 == span.end) E = load_state<V>(at.inside ? args.grad_last : nullptr, at.state_at(args, span.sequence));
                const Num<V> D = streams[2].get(d, p, i, at.lane) + E;
                E = a[i] * D;
                if (at.inside) {
                    store_number<T, V>(to_x, rest[i] * D);
                    store_number<T, V>(to_gate, slope[i] * D);
                    if (p + i == span.begin && args.grad_initial) store_state<V>(args.grad_initial, at.state_at(args, span.sequence), E);
                }
                to_x -= step_x; to_gate -= step_gate;
            }
        }
    }
    if (at.inside) pass_empty_sequences(args, args.grad_last, args.grad_initial, at.chunk, at.channel, V);
}

// One step for each row, the state updated in place.
template <typename T>
__global__ void __launch_bounds__(256) scan_step_kernel(const T* __restrict__ x, int64_t x_stride, const T* __restrict__ gate, int64_t gate_stride, float* state,
                                                       int64_t state_stride, T* h, int64_t h_stride, int64_t rows, int width) {
    const int64_t total = rows * width, step = int64_t(gridDim.x) * 256;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < total; i += step) {
        const int64_t row = i / width, channel = i - row * width;
        const Gate<1> g = gate_of<1>(gate_exp<1>({to_float<T>(gate[row * gate_stride + channel])}));
        float* s = state + row * state_stride + channel;
        const float next = fmaf(g.a.v, *s, g.rest.v * to_float<T>(x[row * x_stride + channel]));
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
// Over both layouts of the channels: with two a lane there are fewer tiles, and so more chunks.
int64_t most_chunks(int64_t rows, int64_t width) { return pieces(rows, chunk_rows(rows, (width + 63) / 64)); }

// `behind`: close behind the kernel before, for which the kernel waits itself.
template <typename K> cudaError_t launch_chunks(K kernel, PerDeviceOnce& once, const ScanArgs& args, int smem, bool behind, cudaStream_t stream) {
    const cudaError_t err = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
    if (err != cudaSuccess) return err;
    const unsigned int blocks = unsigned(pieces(int64_t(args.chunks) * args.channel_tiles, kScanWarps));
    if (behind) return launch_after(kernel, blocks, kScanBlock, smem, stream, args);
    kernel<<<blocks, kScanBlock, smem, stream>>>(args);
    return cudaSuccess;
}

template <typename T, int V, int PIECE> cudaError_t scan_launch(ScanArgs& args, bool backward, cudaStream_t stream) {
    static PerDeviceOnce compose, apply, compose_backward, apply_backward;
    constexpr int two = kFeedBytes<T, V, PIECE, 2>, three = kFeedBytes<T, V, PIECE, 3>;
    args.channel_tiles = (args.in.width + 32 * V - 1) / (32 * V);
    args.chunk = chunk_rows(args.in.rows, args.channel_tiles);
    args.chunks = int(pieces(args.in.rows, args.chunk));
    cudaError_t err = cudaSuccess;
    if (args.chunks > 1) {
        err = backward ? launch_chunks(scan_compose_backward_kernel<T, V, PIECE>, compose_backward, args, two, false, stream)
                       : launch_chunks(scan_compose_kernel<T, V, PIECE>, compose, args, two, false, stream);
        if (err == cudaSuccess) err = launch_carry(args, backward, stream);
    }
    if (err != cudaSuccess) return err;
    return backward ? launch_chunks(scan_apply_backward_kernel<T, V, PIECE>, apply_backward, args, three, args.chunks > 1, stream)
                    : launch_chunks(scan_apply_kernel<T, V, PIECE>, apply, args, two, args.chunks > 1, stream);
}

// Two channels a lane where every row allows it, in pieces of 16 bytes where they do too.
template <typename T> int scan_typed(ScanArgs& a, bool backward, cudaStream_t stream) {
    const auto allow = [&](size_t bytes) {
        const auto one = [&](const void* p, int64_t stride) { return !p || rows_aligned(p, stride, a.in.rows, sizeof(T), bytes); };
        return size_t(a.in.width) * sizeof(T) % bytes == 0 && one(a.in.x, a.in.x_stride) && one(a.in.gate, a.in.gate_stride) && one(a.h, a.h_stride) &&
               one(a.grad_h, a.grad_h_stride) && one(a.grad_x, a.grad_x_stride) && one(a.grad_gate, a.grad_gate_stride);
    };
    cudaError_t err;
    if (allow(16)) err = scan_launch<T, 2, 16>(a, backward, stream);
    else if constexpr (sizeof(T) == 4) err = scan_launch<T, 1, 4>(a, backward, stream);
    else if (allow(4)) err = scan_launch<T, 2, 4>(a, backward, stream);
    else err = scan_launch<T, 1, 2>(a, backward, stream);
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
    const size_t values = size_t(htgs::most_chunks(rows, width)) * size_t(width);
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
    a.carried = reinterpret_cast<float*>(static_cast<char*>(workspace) + align256(size_t(most_chunks(scan->rows, scan->width)) * size_t(scan->width) * sizeof(float2)));
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
    a.carried = reinterpret_cast<float*>(static_cast<char*>(workspace) + align256(size_t(most_chunks(scan->rows, scan->width)) * size_t(scan->width) * sizeof(float2)));
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
