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
constexpr int kComposeSteps = 16, kComposeWarps = kChunk / kComposeSteps;
constexpr int kApplySteps = 8, kApplyWarps = kChunk / kApplySteps;
constexpr int kKept = 8;                     // a state for every so many rows is kept for the backward pass
constexpr int kCarryWarps = 32, kCarryChannels = 8, kCarryRun = 16;
static_assert(kApplySteps == kKept, "a warp keeps one state, and begins with it in the backward pass");

struct ScanArgs {
    HtgsScan in;
    int chunks, channel_tiles;
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

// Where a thread works: V channels side by side, STEPS rows from position p0 on (positions count rows in the order of the recurrence), `count` of which exist.
template <int V, int STEPS, int WARPS> struct Place {
    int lane, warp, channel, count, p0, chunk;
    bool inside;
    __device__ __forceinline__ explicit Place(const ScanArgs& a, bool from_end = false) {
        lane = threadIdx.x & 31; warp = threadIdx.x >> 5;
        const int at = int(blockIdx.x / unsigned(a.channel_tiles));
        chunk = from_end ? a.chunks - 1 - at : at;
        channel = (int(blockIdx.x % unsigned(a.channel_tiles)) * 32 + lane) * V;
        inside = channel < a.in.width;
        p0 = (chunk * WARPS + warp) * STEPS;
        count = max(0, min(STEPS, int(a.in.rows) - p0));
    }
    __device__ __forceinline__ bool whole() const { return count == STEPS && inside; }
    __device__ __forceinline__ int64_t state_at(const ScanArgs& a, int sequence) const { return int64_t(sequence) * a.in.width + channel; }
};

// A matrix's values at a place: the address at position p0, and the bytes to the next position.  Going from row to row by one addition takes
// half the instructions of an address computed for each.
template <typename T, int V> struct Rows {
    char* first;
    int64_t step;
    template <typename P> __device__ __forceinline__ Rows(const void* base, int64_t stride, const HtgsScan& in, const P& at) {
        const int64_t row = in.reverse ? in.rows - 1 - at.p0 : at.p0;
        first = static_cast<char*>(const_cast<void*>(base)) + (row * stride + at.channel) * int64_t(sizeof(T));
        step = (in.reverse ? -stride : stride) * int64_t(sizeof(T));
    }
    template <typename P, int STEPS> __device__ __forceinline__ void load(const P& place, Pack<T, V> (&out)[STEPS]) const {
        const char* p = first;
        if (place.whole()) {
            #pragma unroll
            for (int i = 0; i < STEPS; ++i, p += step) out[i] = *reinterpret_cast<const Pack<T, V>*>(p);
        } else {
            #pragma unroll
            for (int i = 0; i < STEPS; ++i, p += step) {
                if (place.inside && i < place.count) out[i] = *reinterpret_cast<const Pack<T, V>*>(p);
                else {
                    #pragma unroll
                    for (int k = 0; k < V; ++k) out[i].v[k] = from_float<T>(0.0f);
                }
            }
        }
    }
};
template <typename T, int V> __device__ __forceinline__ void store_at(char* p, Num<V> n) { store_number<T, V>(reinterpret_cast<T*>(p), n); }

// The warp's steps as h -> a h + b, and all of them composed (A, H).  The loop for rows in the middle of a sequence asks for nothing else.
template <typename T, int V, int STEPS, typename P>
__device__ __forceinline__ void forward_steps(const ScanArgs& args, const P& at, const Edges& edges, const Pack<T, V> (&x)[STEPS],
                                              const Pack<T, V> (&g)[STEPS], Num<V> (&a)[STEPS], Num<V> (&b)[STEPS], Num<V>& A, Num<V>& H) {
    A = Num<V>::all(1.0f); H = Num<V>::all(0.0f);
    #pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const Gate<V> gate = gate_of<V>(gate_exp<V>(number<T, V>(g[i])));
        a[i] = gate.a;
        b[i] = gate.rest * number<T, V>(x[i]);
    }
    if (edges.first == 0 && at.count == STEPS) {
        #pragma unroll
        for (int i = 0; i < STEPS; ++i) { A = A * a[i]; H = madd(a[i], H, b[i]); }
        return;
    }
    #pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        if (i >= at.count) { a[i] = Num<V>::all(1.0f); b[i] = Num<V>::all(0.0f); }
        if (edges.first >> i & 1u) {
            const int s = __shfl_sync(0xffffffffu, edges.sequence, i);
            b[i] = madd(a[i], load_state<V>(at.inside ? args.in.initial : nullptr, at.state_at(args, s)), b[i]);
            A = a[i] = Num<V>::all(kCut); H = b[i];
        } else { A = A * a[i]; H = madd(a[i], H, b[i]); }
    }
}

// First pass, forward: the composition of each chunk.
template <typename T, int V>
__global__ void __launch_bounds__(kComposeWarps * 32, 8) scan_compose_kernel(const ScanArgs args) {
    constexpr int S = kComposeSteps, W = kComposeWarps;
    __shared__ float2 shared[W][32 * V];
    const Place<V, S, W> at(args);
    Pack<T, V> x[S], g[S];
    Rows<T, V>(args.in.gate, args.in.gate_stride, args.in, at).load(at, g);
    Rows<T, V>(args.in.x, args.in.x_stride, args.in, at).load(at, x);
    const Edges edges = find_edges<S>(args.in, at.p0, at.lane);
    Num<V> A = Num<V>::all(1.0f), H = Num<V>::all(0.0f);
    if (edges.first == 0 && at.count == S) {
        #pragma unroll
        for (int i = 0; i < S; ++i) {
            const Gate<V> gate = gate_of<V>(gate_exp<V>(number<T, V>(g[i])));
            H = madd(gate.a, H, gate.rest * number<T, V>(x[i]));
            A = A * gate.a;
        }
    } else {
        #pragma unroll
        for (int i = 0; i < S; ++i) {
            if (i >= at.count) break;
            if (edges.first >> i & 1u) {
                const int s = __shfl_sync(0xffffffffu, edges.sequence, i);
                A = Num<V>::all(kCut);
                H = load_state<V>(at.inside ? args.in.initial : nullptr, at.state_at(args, s));
            }
            const Gate<V> gate = gate_of<V>(gate_exp<V>(number<T, V>(g[i])));
            H = madd(gate.a, H, gate.rest * number<T, V>(x[i]));
            A = A * gate.a;
        }
    }
    leave_map<V>(&shared[at.warp][at.lane * V], A, H);
    __syncthreads();
    if (at.warp != 0 || !at.inside) return;
    #pragma unroll
    for (int k = 0; k < V; ++k) {
        float P = 1.0f, Q = 0.0f;
        #pragma unroll
        for (int w = 0; w < W; ++w) compose(P, Q, shared[w][at.lane * V + k]);
        args.composed[int64_t(at.chunk) * args.in.width + at.channel + k] = make_float2(P, Q);
    }
}

// First pass, backward: E in front of a chunk as a map of E behind it.
template <typename T, int V>
__global__ void __launch_bounds__(kComposeWarps * 32, 8) scan_compose_backward_kernel(const ScanArgs args) {
    constexpr int S = kComposeSteps, W = kComposeWarps;
    __shared__ float2 shared[W][32 * V];
    const Place<V, S, W> at(args);
    Pack<T, V> d[S], g[S];
    Rows<T, V>(args.in.gate, args.in.gate_stride, args.in, at).load(at, g);
    Rows<T, V>(args.grad_h, args.grad_h_stride, args.in, at).load(at, d);
    const Edges edges = find_edges<S>(args.in, at.p0, at.lane);
    Num<V> A = Num<V>::all(1.0f), H = Num<V>::all(0.0f);
    if (edges.last == 0 && at.count == S) {
        #pragma unroll
        for (int i = S - 1; i >= 0; --i) {
            const Num<V> a = gate_of<V>(gate_exp<V>(number<T, V>(g[i]))).a;
            H = a * (H + number<T, V>(d[i]));
            A = A * a;
        }
    } else {
        #pragma unroll
        for (int i = S - 1; i >= 0; --i) {
            if (i >= at.count) continue;
            if (edges.last >> i & 1u) {
                const int s = __shfl_sync(0xffffffffu, edges.sequence, i);
                A = Num<V>::all(kCut);
                H = load_state<V>(at.inside ? args.grad_last : nullptr, at.state_at(args, s));
            }
            const Num<V> a = gate_of<V>(gate_exp<V>(number<T, V>(g[i]))).a;
            H = a * (H + number<T, V>(d[i]));
            A = A * a;
        }
    }
    leave_map<V>(&shared[at.warp][at.lane * V], A, H);
    __syncthreads();
    if (at.warp != 0 || !at.inside) return;
    #pragma unroll
    for (int k = 0; k < V; ++k) {
        float P = 1.0f, Q = 0.0f;
        #pragma unroll
        for (int w = W - 1; w >= 0; --w) compose(P, Q, shared[w][at.lane * V + k]);
        args.composed[int64_t(at.chunk) * args.in.width + at.channel + k] = make_float2(P, Q);
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

// Third pass, forward; from the end, where the first pass has left the rows in L2.
template <typename T, int V>
__global__ void __launch_bounds__(kApplyWarps * 32, 4) scan_apply_kernel(const ScanArgs args) {
    constexpr int S = kApplySteps, W = kApplyWarps;
    __shared__ float2 shared[W][32 * V];
    const Place<V, S, W> at(args, true);
    Pack<T, V> x[S], g[S];
    Rows<T, V>(args.in.gate, args.in.gate_stride, args.in, at).load(at, g);
    Rows<T, V>(args.in.x, args.in.x_stride, args.in, at).load(at, x);
    Num<V> h = load_state<V>(args.chunks > 1 && at.inside ? args.carried : nullptr, int64_t(at.chunk) * args.in.width + at.channel);
    const Edges edges = find_edges<S>(args.in, at.p0, at.lane);
    Num<V> a[S], b[S], A, H;
    forward_steps<T, V, S>(args, at, edges, x, g, a, b, A, H);
    leave_map<V>(&shared[at.warp][at.lane * V], A, H);
    __syncthreads();
    for (int w = 0; w < at.warp; ++w) h = follow<V>(&shared[w][at.lane * V], h);
    const Rows<T, V> to(args.h, args.h_stride, args.in, at);
    char* p = to.first;
    if (args.states && at.inside && at.count > 0) store_state<V>(args.states, int64_t(at.p0 / kKept) * args.in.width + at.channel, h);
    if ((edges.first | edges.last) == 0 && at.count == S) {
        if (at.inside) {
            #pragma unroll
            for (int i = 0; i < S; ++i, p += to.step) {
                h = madd(a[i], h, b[i]);
                store_at<T, V>(p, h);
            }
        }
    } else {
        #pragma unroll
        for (int i = 0; i < S; ++i, p += to.step) {
            h = edges.first >> i & 1u ? b[i] : madd(a[i], h, b[i]);
            if (at.inside && i < at.count) store_at<T, V>(p, h);
            if (edges.last >> i & 1u) {
                const int s = __shfl_sync(0xffffffffu, edges.sequence, i);
                if (at.inside) store_state<V>(args.last, at.state_at(args, s), h);
            }
        }
    }
    if (at.warp == 0 && at.inside) pass_empty_sequences(args, args.in.initial, args.last, at.chunk, at.channel, V);
}

// Third pass, backward: each warp goes eight rows forward from the state that was kept, and back from the E that the warps behind it leave.
template <typename T, int V>
__global__ void __launch_bounds__(kApplyWarps * 32, 3) scan_apply_backward_kernel(const ScanArgs args) {
    constexpr int S = kApplySteps, W = kApplyWarps;
    __shared__ float2 shared[W][32 * V];
    const Place<V, S, W> at(args, true);
    Pack<T, V> x[S], d[S], g[S];
    Rows<T, V>(args.in.gate, args.in.gate_stride, args.in, at).load(at, g);
    Rows<T, V>(args.grad_h, args.grad_h_stride, args.in, at).load(at, d);
    Rows<T, V>(args.in.x, args.in.x_stride, args.in, at).load(at, x);
    Num<V> h = load_state<V>(at.count > 0 && at.inside ? args.states : nullptr, int64_t(at.p0 / kKept) * args.in.width + at.channel);
    Num<V> E = load_state<V>(args.chunks > 1 && at.inside ? args.carried : nullptr, int64_t(at.chunk) * args.in.width + at.channel);
    const Edges edges = find_edges<S>(args.in, at.p0, at.lane);
    const bool plain = (edges.first | edges.last) == 0 && at.count == S;
    Num<V> a[S], rest[S];
    Num<V> P = Num<V>::all(1.0f), Q = Num<V>::all(0.0f);             // E in front of the warp's rows is P E + Q
    #pragma unroll
    for (int i = 0; i < S; ++i) {
        const Gate<V> gate = gate_of<V>(gate_exp<V>(number<T, V>(g[i])));
        a[i] = gate.a; rest[i] = gate.rest;
    }
    if (plain) {
        #pragma unroll
        for (int i = S - 1; i >= 0; --i) { Q = a[i] * (Q + number<T, V>(d[i])); P = P * a[i]; }
    } else {
        #pragma unroll
        for (int i = S - 1; i >= 0; --i) {
            if (i >= at.count) continue;
            if (edges.last >> i & 1u) {
                const int s = __shfl_sync(0xffffffffu, edges.sequence, i);
                P = Num<V>::all(kCut);
                Q = load_state<V>(at.inside ? args.grad_last : nullptr, at.state_at(args, s));
            }
            Q = a[i] * (Q + number<T, V>(d[i]));
            P = P * a[i];
        }
    }
    leave_map<V>(&shared[at.warp][at.lane * V], P, Q);
    Num<V> slope[S];                          // (h_{t-1} - x) a (1 - a)
    const Num<V> minus = Num<V>::all(-1.0f);
    if (edges.first == 0) {
        #pragma unroll
        for (int i = 0; i < S; ++i) {
            const Num<V> value = number<T, V>(x[i]);
            slope[i] = madd(minus, value, h) * (a[i] * rest[i]);
            h = madd(a[i], h, rest[i] * value);
        }
    } else {
        #pragma unroll
        for (int i = 0; i < S; ++i) {
            if (edges.first >> i & 1u) {
                const int s = __shfl_sync(0xffffffffu, edges.sequence, i);
                h = load_state<V>(at.inside ? args.in.initial : nullptr, at.state_at(args, s));
            }
            const Num<V> value = number<T, V>(x[i]);
            slope[i] = madd(minus, value, h) * (a[i] * rest[i]);
            h = madd(a[i], h, rest[i] * value);
        }
    }
    __syncthreads();
    for (int w = W - 1; w > at.warp; --w) E = follow<V>(&shared[w][at.lane * V], E);
    const Rows<T, V> to_x(args.grad_x, args.grad_x_stride, args.in, at), to_gate(args.grad_gate, args.grad_gate_stride, args.in, at);
    char* px = to_x.first + (S - 1) * to_x.step;
    char* pg = to_gate.first + (S - 1) * to_gate.step;
    if (plain) {
        if (at.inside) {
            #pragma unroll
            for (int i = S - 1; i >= 0; --i, px -= to_x.step, pg -= to_gate.step) {
                const Num<V> D = number<T, V>(d[i]) + E;
                store_at<T, V>(px, rest[i] * D);
                store_at<T, V>(pg, slope[i] * D);
                E = a[i] * D;
            }
        }
    } else {
        #pragma unroll
        for (int i = S - 1; i >= 0; --i, px -= to_x.step, pg -= to_gate.step) {
            if (i >= at.count) continue;
            const bool first = edges.first >> i & 1u, last = edges.last >> i & 1u;
            int s = 0;
            if (first || last) s = __shfl_sync(0xffffffffu, edges.sequence, i);
            if (last) E = load_state<V>(at.inside ? args.grad_last : nullptr, at.state_at(args, s));
            const Num<V> D = number<T, V>(d[i]) + E;
            E = a[i] * D;
            if (at.inside) {
                store_at<T, V>(px, rest[i] * D);
                store_at<T, V>(pg, slope[i] * D);
                if (first && args.grad_initial) store_state<V>(args.grad_initial, at.state_at(args, s), E);
            }
        }
    }
    if (at.warp == 0 && at.inside) pass_empty_sequences(args, args.grad_last, args.grad_initial, at.chunk, at.channel, V);
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

bool pairs_possible(const void* p, int64_t stride, int64_t rows, size_t element) { return !p || rows_aligned(p, stride, rows, element, 2 * element); }

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

template <typename T, int V> void scan_launch(ScanArgs& args, bool backward, cudaStream_t stream) {
    args.channel_tiles = (args.in.width + 32 * V - 1) / (32 * V);
    args.chunks = int(pieces(args.in.rows, kChunk));
    const unsigned int blocks = unsigned(int64_t(args.chunks) * args.channel_tiles);
    if (args.chunks > 1) {
        if (backward) scan_compose_backward_kernel<T, V><<<blocks, kComposeWarps * 32, 0, stream>>>(args);
        else scan_compose_kernel<T, V><<<blocks, kComposeWarps * 32, 0, stream>>>(args);
        launch_carry(args, backward, stream);
    }
    if (backward) scan_apply_backward_kernel<T, V><<<blocks, kApplyWarps * 32, 0, stream>>>(args);
    else scan_apply_kernel<T, V><<<blocks, kApplyWarps * 32, 0, stream>>>(args);
}

// Two channels a lane where every row allows it.
template <typename T> void scan_typed(ScanArgs& a, bool backward, cudaStream_t stream) {
    const int64_t rows = a.in.rows;
    const size_t e = sizeof(T);
    const bool pairs = a.in.width % 2 == 0 && pairs_possible(a.in.x, a.in.x_stride, rows, e) && pairs_possible(a.in.gate, a.in.gate_stride, rows, e) &&
                       pairs_possible(a.h, a.h_stride, rows, e) && pairs_possible(a.grad_h, a.grad_h_stride, rows, e) &&
                       pairs_possible(a.grad_x, a.grad_x_stride, rows, e) && pairs_possible(a.grad_gate, a.grad_gate_stride, rows, e);
    if (pairs) scan_launch<T, 2>(a, backward, stream); else scan_launch<T, 1>(a, backward, stream);
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
    if (scan->type == HTGS_FLOAT32) scan_typed<float>(a, false, s);
    else if (scan->type == HTGS_FLOAT16) scan_typed<__half>(a, false, s);
    else scan_typed<__nv_bfloat16>(a, false, s);
    return sequence_status("htgs_gated_scan");
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
    if (scan->type == HTGS_FLOAT32) scan_typed<float>(a, true, s);
    else if (scan->type == HTGS_FLOAT16) scan_typed<__half>(a, true, s);
    else scan_typed<__nv_bfloat16>(a, true, s);
    return sequence_status("htgs_gated_scan_backward");
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
