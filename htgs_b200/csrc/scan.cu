// Gated linear recurrence over long sequences, forward, backward, and one step at a time.
//
//   a = 1 / (1 + exp(-gate));   h_t = a_t h_{t-1} + (1 - a_t) x_t;   h_{-1} = the sequence's initial state
//   backward, from the last row to the first:  D_t = grad_h_t + E_{t+1};   E_t = a_t D_t   (E behind the last row: the last state's gradient)
//       grad_x = (1 - a) D;   grad_gate = D (h_{t-1} - x) a (1 - a);   grad_initial = E at the first row
//
// A step is the map h -> A h + H, and steps compose: (A2, H2) after (A1, H1) is (A1 A2, A2 H1 + H2).  The rows are cut into chunks of
// 128.  One kernel composes each chunk's rows, one walks from chunk to chunk and leaves the state in front of each, one goes through
// the chunks again from those states and writes h.  The backward pass does the same from the end; h_{t-1} is computed again from the
// chunks' states, so it is in 32 bits and h need not be read.  A sequence's first row has A = 0 and takes its initial state into H, so
// packed sequences need no chunks of their own; that zero is kept as
// -0 and tested for, so that a NaN or infinity of one sequence does not reach the next.  States, products and sums are 32-bit; 1 - a is exp(-gate) a, which keeps its relative precision
// where a is close to 1.
#include "sequence.cuh"

namespace htgs {

namespace {

// A block takes a chunk of 32 or 64 channels; each of its warps takes some rows of it.
constexpr int kChunk = 64;                                                       // rows
constexpr int kSteps = 8, kWarps = kChunk / kSteps;                              // rows of a warp
constexpr int kScanBlock = kWarps * 32;
constexpr int kKept = 8;                     // a state for every so many rows is kept for the backward pass
constexpr int kCarryWarps = 32, kCarryChannels = 8, kCarryRun = 16;
static_assert(kSteps == kKept, "a warp keeps one state, and begins with it in the backward pass");

struct ScanArgs {
    HtgsScan in;
    int chunks;
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

// Which of the warp's `STEPS` steps are the first or last of their sequence (bits), and in lane i the sequence of step i.
struct Edges { unsigned int first, last; int sequence; };
template <int STEPS> __device__ __forceinline__ Edges find_edges(const HtgsScan& in, int64_t p0, int lane) {
    const int64_t p = p0 + lane;
    // one sequence: only its first and last position have an edge
    if (!in.offsets && in.n_sequences == 1) {
        const int64_t end = in.rows - 1 - p0;
        return {p0 == 0 ? 1u : 0u, end >= 0 && end < STEPS ? 1u << end : 0u, 0};
    }
    bool first = false, last = false;
    int s = 0;
    if (lane < STEPS && p < in.rows) {
        const int64_t row = in.reverse ? in.rows - 1 - p : p;
        int64_t begin, end;
        if (in.offsets) {
            int hi = in.n_sequences;
            while (hi - s > 1) {
                const int mid = (s + hi) >> 1;
                if (__ldg(in.offsets + mid) <= row) s = mid; else hi = mid;
            }
            begin = __ldg(in.offsets + s); end = __ldg(in.offsets + s + 1);
        } else {
            const int64_t length = in.rows / in.n_sequences;
            s = int(row / length);
            begin = s * length; end = begin + length;
        }
        first = row == begin; last = row + 1 == end;
        if (in.reverse) { const bool swap = first; first = last; last = swap; }
    }
    return {__ballot_sync(0xffffffffu, first), __ballot_sync(0xffffffffu, last), s};
}

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

// Where a thread works: V channels side by side, kSteps rows from position p0 on (positions count rows in the order of the recurrence), `count` of which exist.
constexpr int kGridRows = 32768;              // chunks along the grid's y, the rest along z
template <int V> struct Place {
    int lane, warp, channel0, channel, count, p0, chunk;
    bool inside;
    __device__ __forceinline__ explicit Place(const ScanArgs& a, bool from_end = false) {
        lane = threadIdx.x & 31; warp = threadIdx.x >> 5;
        const int at = int(blockIdx.z * kGridRows + blockIdx.y);
        chunk = from_end ? a.chunks - 1 - at : at;
        channel0 = int(blockIdx.x) * 32 * V;
        channel = channel0 + lane * V;
        inside = channel < a.in.width;
        p0 = chunk * kChunk + warp * kSteps;
        count = max(0, min(kSteps, int(a.in.rows) - p0));
    }
    __device__ __forceinline__ int64_t state_at(const ScanArgs& a, int sequence) const { return int64_t(sequence) * a.in.width + channel; }
};

// A chunk of 32 V channels in shared memory, one row per position, brought and taken away PIECE bytes at a time: 16 where every row of the matrix
// allows it, or 4, or a single 16-bit value.
template <typename T, int V, int PIECE> struct Tile {
    static constexpr int kRow = 32 * V, kElements = PIECE / int(sizeof(T)), kPieces = kRow / kElements, kRowsAtOnce = kScanBlock / kPieces, kTrips = kChunk / kRowsAtOnce;
    static constexpr int bytes = kChunk * kRow * int(sizeof(T));
    T* data;
    __device__ __forceinline__ explicit Tile(unsigned char* at) : data(reinterpret_cast<T*>(at)) {}
    // f(address in the matrix, address here, whether the piece exists), for each of the thread's pieces
    template <typename F> __device__ __forceinline__ void each(const void* base, int64_t stride, const ScanArgs& a, const Place<V>& at, F f) const {
        const int r = int(threadIdx.x) / kPieces, c = int(threadIdx.x) % kPieces * kElements, left = int(a.in.rows) - at.chunk * kChunk;
        const int64_t position = int64_t(at.chunk) * kChunk + r, row = a.in.reverse ? a.in.rows - 1 - position : position;
        const int64_t step = (a.in.reverse ? -stride : stride) * kRowsAtOnce;
        T* there = static_cast<T*>(const_cast<void*>(base)) + row * stride + at.channel0 + c;
        const bool inside = at.channel0 + c < a.in.width;
        T* here = data + r * kRow + c;
        #pragma unroll
        for (int i = 0; i < kTrips; ++i, there += step, here += kRowsAtOnce * kRow) f(there, here, inside && r + i * kRowsAtOnce < left);
    }
    // What does not exist becomes zero.
    __device__ __forceinline__ void load(const void* base, int64_t stride, const ScanArgs& a, const Place<V>& at) const {
        each(base, stride, a, at, [&](T* there, T* here, bool exists) {
            if constexpr (PIECE == 16)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(here)), "l"(exists ? there : base), "r"(exists ? 16 : 0) : "memory");
            else if constexpr (PIECE == 4)
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(here)), "l"(exists ? there : base), "r"(exists ? 4 : 0) : "memory");
            else *here = exists ? *there : from_float<T>(0.0f);
        });
    }
    __device__ __forceinline__ void store(void* base, int64_t stride, const ScanArgs& a, const Place<V>& at) const {
        each(base, stride, a, at, [&](T* there, T* here, bool exists) {
            if (exists) *reinterpret_cast<Pack<T, kElements>*>(there) = *reinterpret_cast<const Pack<T, kElements>*>(here);
        });
    }
    __device__ __forceinline__ T* mine(const Place<V>& at) const { return data + at.warp * kSteps * kRow + at.lane * V; }       // the thread's values: every kRow from here
    __device__ __forceinline__ static Num<V> get(const T* p) { return number<T, V>(*reinterpret_cast<const Pack<T, V>*>(p)); }
    __device__ __forceinline__ static void put(T* p, Num<V> n) { store_number<T, V>(p, n); }
};
__device__ __forceinline__ void tiles_are_here() {
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
}
template <typename T, int V> __device__ __forceinline__ Gate<V> gate_at(const T* p) { return gate_of<V>(gate_exp<V>(number<T, V>(*reinterpret_cast<const Pack<T, V>*>(p)))); }

// First pass, forward: the composition of each chunk.
template <typename T, int V, int PIECE>
__global__ void __launch_bounds__(kScanBlock, 6) scan_compose_kernel(const ScanArgs args) {
    extern __shared__ __align__(16) unsigned char memory[];
    __shared__ float2 shared[kWarps][32 * V];
    using In = Tile<T, V, PIECE>;
    const Place<V> at(args);
    if (at.chunk >= args.chunks) return;
    const In gs(memory), xs(memory + In::bytes);
    gs.load(args.in.gate, args.in.gate_stride, args, at);
    xs.load(args.in.x, args.in.x_stride, args, at);
    const Edges edges = find_edges<kSteps>(args.in, at.p0, at.lane);
    tiles_are_here();
    const T *g = gs.mine(at), *x = xs.mine(at);
    Num<V> A = Num<V>::all(1.0f), H = Num<V>::all(0.0f);
    if (edges.first == 0 && at.count == kSteps) {
        #pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const Gate<V> gate = gate_at<T, V>(g + i * In::kRow);
            H = madd(gate.a, H, gate.rest * In::get(x + i * In::kRow));
            A = A * gate.a;
        }
    } else {
        #pragma unroll 1
        for (int i = 0; i < at.count; ++i) {
            if (edges.first >> i & 1u) {
                const int s = __shfl_sync(0xffffffffu, edges.sequence, i);
                A = Num<V>::all(kCut);
                H = load_state<V>(at.inside ? args.in.initial : nullptr, at.state_at(args, s));
            }
            const Gate<V> gate = gate_at<T, V>(g + i * In::kRow);
            H = madd(gate.a, H, gate.rest * In::get(x + i * In::kRow));
            A = A * gate.a;
        }
    }
    leave_map<V>(&shared[at.warp][at.lane * V], A, H);
    __syncthreads();
    if (threadIdx.x < 32 * V && at.channel0 + int(threadIdx.x) < args.in.width) {
        float P = 1.0f, Q = 0.0f;
        #pragma unroll
        for (int w = 0; w < kWarps; ++w) compose(P, Q, shared[w][threadIdx.x]);
        args.composed[int64_t(at.chunk) * args.in.width + at.channel0 + threadIdx.x] = make_float2(P, Q);
    }
}

// First pass, backward: E in front of a chunk as a map of E behind it.
template <typename T, int V, int PIECE>
__global__ void __launch_bounds__(kScanBlock, 6) scan_compose_backward_kernel(const ScanArgs args) {
    extern __shared__ __align__(16) unsigned char memory[];
    __shared__ float2 shared[kWarps][32 * V];
    using In = Tile<T, V, PIECE>;
    const Place<V> at(args);
    if (at.chunk >= args.chunks) return;
    const In gs(memory), ds(memory + In::bytes);
    gs.load(args.in.gate, args.in.gate_stride, args, at);
    ds.load(args.grad_h, args.grad_h_stride, args, at);
    const Edges edges = find_edges<kSteps>(args.in, at.p0, at.lane);
    tiles_are_here();
    const T *g = gs.mine(at), *d = ds.mine(at);
    Num<V> A = Num<V>::all(1.0f), H = Num<V>::all(0.0f);
    if (edges.last == 0 && at.count == kSteps) {
        #pragma unroll
        for (int i = kSteps - 1; i >= 0; --i) {
            const Num<V> a = gate_at<T, V>(g + i * In::kRow).a;
            H = a * (H + In::get(d + i * In::kRow));
            A = A * a;
        }
    } else {
        #pragma unroll 1
        for (int i = at.count - 1; i >= 0; --i) {
            if (edges.last >> i & 1u) {
                const int s = __shfl_sync(0xffffffffu, edges.sequence, i);
                A = Num<V>::all(kCut);
                H = load_state<V>(at.inside ? args.grad_last : nullptr, at.state_at(args, s));
            }
            const Num<V> a = gate_at<T, V>(g + i * In::kRow).a;
            H = a * (H + In::get(d + i * In::kRow));
            A = A * a;
        }
    }
    leave_map<V>(&shared[at.warp][at.lane * V], A, H);
    __syncthreads();
    if (threadIdx.x < 32 * V && at.channel0 + int(threadIdx.x) < args.in.width) {
        float P = 1.0f, Q = 0.0f;
        #pragma unroll
        for (int w = kWarps - 1; w >= 0; --w) compose(P, Q, shared[w][threadIdx.x]);
        args.composed[int64_t(at.chunk) * args.in.width + at.channel0 + threadIdx.x] = make_float2(P, Q);
    }
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
    const int runs = kCarryWarps * kQuarters * parts, run = (chunks + runs - 1) / runs;
    const int begin = int(min(int64_t((part * kCarryWarps + warp) * kQuarters + quarter) * run, int64_t(chunks))), count = inside ? min(run, chunks - begin) : 0;
    const int64_t first = int64_t(from_end ? chunks - 1 - begin : begin) * width + channel, step = from_end ? -int64_t(width) : width;
    float2 maps[kCarryRun];
    float A = 1.0f, H = 0.0f;
    for (int c0 = 0; c0 < run; c0 += kCarryRun) {
        #pragma unroll
        for (int c = 0; c < kCarryRun; ++c) maps[c] = c0 + c < count ? composed[first + (c0 + c) * step] : make_float2(1.0f, 0.0f);
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
    for (int c0 = 0; c0 < run; c0 += kCarryRun) {
        if (run > kCarryRun) {
            #pragma unroll
            for (int c = 0; c < kCarryRun; ++c) maps[c] = c0 + c < count ? composed[first + (c0 + c) * step] : make_float2(1.0f, 0.0f);
        }
        #pragma unroll
        for (int c = 0; c < kCarryRun; ++c) {
            if (c0 + c < count) states[first + (c0 + c) * step] = state;
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

// Third pass, forward; from the end, where the first pass has left the rows in L2.  h takes the place of x.
template <typename T, int V, int PIECE>
__global__ void __launch_bounds__(kScanBlock, 5) scan_apply_kernel(const ScanArgs args) {
    extern __shared__ __align__(16) unsigned char memory[];
    __shared__ float2 shared[kWarps][32 * V];
    using In = Tile<T, V, PIECE>;
    const Place<V> at(args, true);
    if (at.chunk < 0) return;
    const In gs(memory), xs(memory + In::bytes);
    gs.load(args.in.gate, args.in.gate_stride, args, at);
    xs.load(args.in.x, args.in.x_stride, args, at);
    Num<V> h = load_state<V>(args.chunks > 1 && at.inside ? args.carried : nullptr, int64_t(at.chunk) * args.in.width + at.channel);
    const Edges edges = find_edges<kSteps>(args.in, at.p0, at.lane);
    tiles_are_here();
    const T* g = gs.mine(at);
    T* x = xs.mine(at);
    Num<V> a[kSteps], b[kSteps], A = Num<V>::all(1.0f), H = Num<V>::all(0.0f);
    #pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const Gate<V> gate = gate_at<T, V>(g + i * In::kRow);
        a[i] = gate.a;
        b[i] = gate.rest * In::get(x + i * In::kRow);
    }
    if (edges.first == 0 && at.count == kSteps) {
        #pragma unroll
        for (int i = 0; i < kSteps; ++i) { A = A * a[i]; H = madd(a[i], H, b[i]); }
    } else {
        #pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            if (i >= at.count) break;
            if (edges.first >> i & 1u) {
                const int s = __shfl_sync(0xffffffffu, edges.sequence, i);
                A = Num<V>::all(kCut);
                H = b[i] = madd(a[i], load_state<V>(at.inside ? args.in.initial : nullptr, at.state_at(args, s)), b[i]);
            } else { A = A * a[i]; H = madd(a[i], H, b[i]); }
        }
    }
    leave_map<V>(&shared[at.warp][at.lane * V], A, H);
    __syncthreads();
    for (int w = 0; w < at.warp; ++w) h = follow<V>(&shared[w][at.lane * V], h);
    if (args.states && at.inside && at.count > 0) store_state<V>(args.states, int64_t(at.p0 / kKept) * args.in.width + at.channel, h);
    if ((edges.first | edges.last) == 0) {
        #pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            h = madd(a[i], h, b[i]);
            In::put(x + i * In::kRow, h);
        }
    } else {
        #pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            h = edges.first >> i & 1u ? b[i] : madd(a[i], h, b[i]);
            In::put(x + i * In::kRow, h);
            if (edges.last >> i & 1u) {
                const int s = __shfl_sync(0xffffffffu, edges.sequence, i);
                if (at.inside) store_state<V>(args.last, at.state_at(args, s), h);
            }
        }
    }
    if (at.warp == 0 && at.inside) pass_empty_sequences(args, args.in.initial, args.last, at.chunk, at.channel, V);
    __syncthreads();
    xs.store(args.h, args.h_stride, args, at);
}

// Third pass, backward: each warp goes eight rows forward from the state that was kept, and back from the E that the warps behind it leave.  The gradients
// take the places of x and gate.
template <typename T, int V, int PIECE>
__global__ void __launch_bounds__(kScanBlock, 3) scan_apply_backward_kernel(const ScanArgs args) {
    extern __shared__ __align__(16) unsigned char memory[];
    __shared__ float2 shared[kWarps][32 * V];
    using In = Tile<T, V, PIECE>;
    const Place<V> at(args, true);
    if (at.chunk < 0) return;
    const In gs(memory), xs(memory + In::bytes), ds(memory + 2 * In::bytes);
    gs.load(args.in.gate, args.in.gate_stride, args, at);
    ds.load(args.grad_h, args.grad_h_stride, args, at);
    xs.load(args.in.x, args.in.x_stride, args, at);
    Num<V> h = load_state<V>(at.count > 0 && at.inside ? args.states : nullptr, int64_t(at.p0 / kKept) * args.in.width + at.channel);
    Num<V> E = load_state<V>(args.chunks > 1 && at.inside ? args.carried : nullptr, int64_t(at.chunk) * args.in.width + at.channel);
    const Edges edges = find_edges<kSteps>(args.in, at.p0, at.lane);
    tiles_are_here();
    T *g = gs.mine(at), *x = xs.mine(at);
    const T* d = ds.mine(at);
    const bool plain = (edges.first | edges.last) == 0 && at.count == kSteps;
    Num<V> a[kSteps], rest[kSteps];
    Num<V> P = Num<V>::all(1.0f), Q = Num<V>::all(0.0f);             // E in front of the warp's rows is P E + Q
    #pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const Gate<V> gate = gate_at<T, V>(g + i * In::kRow);
        a[i] = gate.a; rest[i] = gate.rest;
    }
    if (plain) {
        #pragma unroll
        for (int i = kSteps - 1; i >= 0; --i) { Q = a[i] * (Q + In::get(d + i * In::kRow)); P = P * a[i]; }
    } else {
        #pragma unroll
        for (int i = kSteps - 1; i >= 0; --i) {
            if (i >= at.count) continue;
            if (edges.last >> i & 1u) {
                const int s = __shfl_sync(0xffffffffu, edges.sequence, i);
                P = Num<V>::all(kCut);
                Q = load_state<V>(at.inside ? args.grad_last : nullptr, at.state_at(args, s));
            }
            Q = a[i] * (Q + In::get(d + i * In::kRow));
            P = P * a[i];
        }
    }
    leave_map<V>(&shared[at.warp][at.lane * V], P, Q);
    Num<V> slope[kSteps];                     // (h_{t-1} - x) a (1 - a)
    const Num<V> minus = Num<V>::all(-1.0f);
    #pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        if (edges.first && (edges.first >> i & 1u)) {
            const int s = __shfl_sync(0xffffffffu, edges.sequence, i);
            h = load_state<V>(at.inside ? args.in.initial : nullptr, at.state_at(args, s));
        }
        const Num<V> value = In::get(x + i * In::kRow);
        slope[i] = madd(minus, value, h) * (a[i] * rest[i]);
        h = madd(a[i], h, rest[i] * value);
    }
    __syncthreads();
    for (int w = kWarps - 1; w > at.warp; --w) E = follow<V>(&shared[w][at.lane * V], E);
    if (plain) {
        #pragma unroll
        for (int i = kSteps - 1; i >= 0; --i) {
            const Num<V> D = In::get(d + i * In::kRow) + E;
            In::put(x + i * In::kRow, rest[i] * D);
            In::put(g + i * In::kRow, slope[i] * D);
            E = a[i] * D;
        }
    } else {
        #pragma unroll
        for (int i = kSteps - 1; i >= 0; --i) {
            if (i >= at.count) continue;
            const bool first = edges.first >> i & 1u, last = edges.last >> i & 1u;
            int s = 0;
            if (first || last) s = __shfl_sync(0xffffffffu, edges.sequence, i);
            if (last) E = load_state<V>(at.inside ? args.grad_last : nullptr, at.state_at(args, s));
            const Num<V> D = In::get(d + i * In::kRow) + E;
            In::put(x + i * In::kRow, rest[i] * D);
            In::put(g + i * In::kRow, slope[i] * D);
            E = a[i] * D;
            if (first && at.inside && args.grad_initial) store_state<V>(args.grad_initial, at.state_at(args, s), E);
        }
    }
    if (at.warp == 0 && at.inside) pass_empty_sequences(args, args.grad_last, args.grad_initial, at.chunk, at.channel, V);
    __syncthreads();
    xs.store(args.grad_x, args.grad_x_stride, args, at);
    gs.store(args.grad_gate, args.grad_gate_stride, args, at);
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

void launch_carry(const ScanArgs& args, bool from_end, cudaStream_t stream) {
    int parts = 1;                             // eight chunks in a run, and at most eight blocks
    while (parts < 8 && args.chunks > kCarryWarps * (32 / kCarryChannels) * 8 * parts) parts *= 2;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = unsigned(parts); attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = unsigned((args.in.width + kCarryChannels - 1) / kCarryChannels * parts); config.blockDim = kCarryWarps * 32; config.stream = stream;
    config.attrs = &attribute; config.numAttrs = 1;
    cudaLaunchKernelEx(&config, scan_carry_kernel, static_cast<const float2*>(args.composed), args.carried, args.chunks, int(args.in.width), from_end, parts);
}

template <typename K> cudaError_t launch_chunks(K kernel, PerDeviceOnce& once, const ScanArgs& args, int tiles, int smem, cudaStream_t stream) {
    const cudaError_t err = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
    if (err != cudaSuccess) return err;
    const dim3 grid(unsigned(tiles), unsigned(args.chunks < kGridRows ? args.chunks : kGridRows), unsigned((args.chunks + kGridRows - 1) / kGridRows));
    kernel<<<grid, kScanBlock, smem, stream>>>(args);
    return cudaSuccess;
}

template <typename T, int V, int PIECE> cudaError_t scan_launch(ScanArgs& args, bool backward, cudaStream_t stream) {
    static PerDeviceOnce compose, apply, compose_backward, apply_backward;
    constexpr int bytes = Tile<T, V, PIECE>::bytes;
    const int tiles = (args.in.width + 32 * V - 1) / (32 * V);
    args.chunks = int(pieces(args.in.rows, kChunk));
    cudaError_t err = cudaSuccess;
    if (args.chunks > 1) {
        err = backward ? launch_chunks(scan_compose_backward_kernel<T, V, PIECE>, compose_backward, args, tiles, 2 * bytes, stream)
                       : launch_chunks(scan_compose_kernel<T, V, PIECE>, compose, args, tiles, 2 * bytes, stream);
        if (err == cudaSuccess) launch_carry(args, backward, stream);
    }
    if (err != cudaSuccess) return err;
    return backward ? launch_chunks(scan_apply_backward_kernel<T, V, PIECE>, apply_backward, args, tiles, 3 * bytes, stream)
                    : launch_chunks(scan_apply_kernel<T, V, PIECE>, apply, args, tiles, 2 * bytes, stream);
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
    if (pieces(scan->rows, kChunk) * ((scan->width + 31) / 32) > 0x7fffffff) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, message);
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
    return rows <= 0 || width <= 0 ? 0 : size_t(htgs::pieces(rows, htgs::kKept)) * size_t(width) * sizeof(float);
}

size_t htgs_gated_scan_workspace_bytes(int64_t rows, int32_t width) {
    if (rows <= 0 || width <= 0) return 0;
    const size_t values = size_t(htgs::pieces(rows, htgs::kChunk)) * size_t(width);
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
    a.carried = reinterpret_cast<float*>(static_cast<char*>(workspace) + align256(size_t(pieces(scan->rows, kChunk)) * size_t(scan->width) * sizeof(float2)));
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
    a.carried = reinterpret_cast<float*>(static_cast<char*>(workspace) + align256(size_t(pieces(scan->rows, kChunk)) * size_t(scan->width) * sizeof(float2)));
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
