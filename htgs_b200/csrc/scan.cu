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

constexpr int kChunk = 128;                  // rows
constexpr int kForwardSteps = 16;            // rows a warp takes, one after the other
constexpr int kBackwardSteps = 8;
constexpr int kCarryWarps = 32;

struct ScanArgs {
    HtgsScan in;
    int64_t chunks;
    int channel_tiles;
    float2* composed;                        // [chunks, width]
    float* states;                           // [chunks, width] state in front of each chunk; the first is not kept
    void* h; int64_t h_stride; float* last;
    const void* grad_h; int64_t grad_h_stride; const float* grad_last;
    void* grad_x; int64_t grad_x_stride; void* grad_gate; int64_t grad_gate_stride; float* grad_initial;
    float* grad_states;                      // [chunks, width] E behind each chunk; that of the last is not kept
};

struct Gate { float a, rest; };              // a and 1 - a
// exp(80) is far from the end of the range, and a below 2e-35 tells nothing from zero.
__device__ __forceinline__ float gate_exp(float g) { return __expf(g < -80.0f ? 80.0f : -g); }
__device__ __forceinline__ Gate gate_of(float t) { const float a = __fdividef(1.0f, 1.0f + t); return {a, t * a}; }

// The map of a sequence's first step takes nothing from the state in front of it: A is -0, which no product of gates is.
constexpr float kCut = -0.0f;
__device__ __forceinline__ bool is_cut(float A) { return __float_as_uint(A) == 0x80000000u; }
__device__ __forceinline__ float follow(float2 m, float state) { return is_cut(m.x) ? m.y : fmaf(m.x, state, m.y); }
__device__ __forceinline__ void compose(float& A, float& H, float2 next) {
    H = follow(next, H);
    A = is_cut(next.x) ? next.x : A * next.x;
}

// Which of the warp's `STEPS` steps are the first or last of their sequence (bits), and in lane i the sequence of step i.
struct Edges { unsigned int first, last; int sequence; };
template <int STEPS> __device__ __forceinline__ Edges find_edges(const HtgsScan& in, int64_t p0, int lane) {
    const int64_t p = p0 + lane;
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

template <int V> __device__ __forceinline__ void load_state(const float* states, int64_t at, float (&v)[V]) {
    #pragma unroll
    for (int k = 0; k < V; ++k) v[k] = states ? states[at + k] : 0.0f;
}

// Where a thread works: V channels side by side, STEPS rows.
template <int V, int STEPS> struct Place {
    int lane, warp, channel;
    int64_t chunk, p0;
    bool inside;
    __device__ __forceinline__ explicit Place(const ScanArgs& a) {
        lane = threadIdx.x & 31; warp = threadIdx.x >> 5;
        chunk = blockIdx.x / unsigned(a.channel_tiles);
        channel = (int(blockIdx.x % unsigned(a.channel_tiles)) * 32 + lane) * V;
        inside = channel < a.in.width;
        p0 = chunk * kChunk + warp * STEPS;
    }
};

template <typename T, int V, int STEPS>
__device__ __forceinline__ void load_rows(const void* base, int64_t stride, const HtgsScan& in, int64_t p0, int channel, bool inside, Pack<T, V> (&out)[STEPS]) {
    #pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const int64_t p = p0 + i;
        if (inside && p < in.rows) {
            const int64_t row = in.reverse ? in.rows - 1 - p : p;
            out[i] = *reinterpret_cast<const Pack<T, V>*>(static_cast<const T*>(base) + row * stride + channel);
        } else {
            #pragma unroll
            for (int k = 0; k < V; ++k) out[i].v[k] = from_float<T>(0.0f);
        }
    }
}

// The warp's steps as (a, b), h -> a h + b, from the loaded rows.
template <typename T, int V, int STEPS>
__device__ __forceinline__ void forward_steps(const ScanArgs& args, const Place<V, STEPS>& at, const Edges& edges, const Pack<T, V> (&x)[STEPS],
                                              const Pack<T, V> (&g)[STEPS], float (&a)[STEPS][V], float (&b)[STEPS][V]) {
    #pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const bool real = at.p0 + i < args.in.rows;
        #pragma unroll
        for (int k = 0; k < V; ++k) {
            const Gate gate = gate_of(gate_exp(to_float<T>(g[i].v[k])));
            a[i][k] = real ? gate.a : 1.0f;
            b[i][k] = real ? gate.rest * to_float<T>(x[i].v[k]) : 0.0f;
        }
        if (edges.first >> i & 1u) {
            const int s = __shfl_sync(0xffffffffu, edges.sequence, i);
            float initial[V];
            load_state<V>(at.inside ? args.in.initial : nullptr, int64_t(s) * args.in.width + at.channel, initial);
            #pragma unroll
            for (int k = 0; k < V; ++k) { b[i][k] = fmaf(a[i][k], initial[k], b[i][k]); a[i][k] = kCut; }
        }
    }
}

// First pass, forward: the composition of each chunk.
template <typename T, int V>
__global__ void __launch_bounds__(kChunk / kForwardSteps * 32) scan_compose_kernel(const ScanArgs args) {
    constexpr int S = kForwardSteps, W = kChunk / S;
    __shared__ float2 shared[W][32 * V];
    const Place<V, S> at(args);
    Pack<T, V> x[S], g[S];
    load_rows<T, V, S>(args.in.x, args.in.x_stride, args.in, at.p0, at.channel, at.inside, x);
    load_rows<T, V, S>(args.in.gate, args.in.gate_stride, args.in, at.p0, at.channel, at.inside, g);
    const Edges edges = find_edges<S>(args.in, at.p0, at.lane);
    float a[S][V], b[S][V];
    forward_steps<T, V, S>(args, at, edges, x, g, a, b);
    #pragma unroll
    for (int k = 0; k < V; ++k) {
        float A = 1.0f, H = 0.0f;
        #pragma unroll
        for (int i = 0; i < S; ++i) {
            if (edges.first >> i & 1u) { A = kCut; H = b[i][k]; }
            else { A *= a[i][k]; H = fmaf(a[i][k], H, b[i][k]); }
        }
        shared[at.warp][at.lane * V + k] = make_float2(A, H);
    }
    __syncthreads();
    if (at.warp != 0 || !at.inside) return;
    #pragma unroll
    for (int k = 0; k < V; ++k) {
        float A = 1.0f, H = 0.0f;
        #pragma unroll
        for (int w = 0; w < W; ++w) compose(A, H, shared[w][at.lane * V + k]);
        args.composed[at.chunk * args.in.width + at.channel + k] = make_float2(A, H);
    }
}

// First pass, backward: E in front of a chunk as a map of E behind it.
template <typename T, int V>
__global__ void __launch_bounds__(kChunk / kForwardSteps * 32) scan_compose_backward_kernel(const ScanArgs args) {
    constexpr int S = kForwardSteps, W = kChunk / S;
    __shared__ float2 shared[W][32 * V];
    const Place<V, S> at(args);
    Pack<T, V> d[S], g[S];
    load_rows<T, V, S>(args.grad_h, args.grad_h_stride, args.in, at.p0, at.channel, at.inside, d);
    load_rows<T, V, S>(args.in.gate, args.in.gate_stride, args.in, at.p0, at.channel, at.inside, g);
    const Edges edges = find_edges<S>(args.in, at.p0, at.lane);
    float A[V], H[V];
    #pragma unroll
    for (int k = 0; k < V; ++k) { A[k] = 1.0f; H[k] = 0.0f; }
    #pragma unroll
    for (int i = S - 1; i >= 0; --i) {
        float behind[V] = {};
        const bool last = edges.last >> i & 1u, real = at.p0 + i < args.in.rows;
        if (last) {
            const int s = __shfl_sync(0xffffffffu, edges.sequence, i);
            load_state<V>(at.inside ? args.grad_last : nullptr, int64_t(s) * args.in.width + at.channel, behind);
        }
        #pragma unroll
        for (int k = 0; k < V; ++k) {
            const float a = gate_of(gate_exp(to_float<T>(g[i].v[k]))).a;
            if (last) { A[k] = kCut; H[k] = behind[k]; }
            if (real) { H[k] = a * (H[k] + to_float<T>(d[i].v[k])); A[k] *= a; }
        }
    }
    #pragma unroll
    for (int k = 0; k < V; ++k) shared[at.warp][at.lane * V + k] = make_float2(A[k], H[k]);
    __syncthreads();
    if (at.warp != 0 || !at.inside) return;
    #pragma unroll
    for (int k = 0; k < V; ++k) {
        float P = 1.0f, Q = 0.0f;
        #pragma unroll
        for (int w = W - 1; w >= 0; --w) compose(P, Q, shared[w][at.lane * V + k]);
        args.composed[at.chunk * args.in.width + at.channel + k] = make_float2(P, Q);
    }
}

// Second pass: the state at each chunk's beginning (from_end: behind each chunk, walking from the last to the first).  A block takes 32
// channels; each of its warps composes a run of chunks, then walks through it again from the state in front of the run.
__global__ void __launch_bounds__(kCarryWarps * 32) scan_carry_kernel(const float2* __restrict__ composed, float* __restrict__ states, int64_t chunks, int width,
                                                                    bool from_end) {
    __shared__ float2 shared[kCarryWarps][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, channel = blockIdx.x * 32 + lane;
    const int64_t run = (chunks + kCarryWarps - 1) / kCarryWarps, begin = min(warp * run, chunks), end = min(begin + run, chunks);
    float A = 1.0f, H = 0.0f;
    if (channel < width) {
        #pragma unroll 8
        for (int64_t c = begin; c < end; ++c) compose(A, H, composed[(from_end ? chunks - 1 - c : c) * width + channel]);
    }
    shared[warp][lane] = make_float2(A, H);
    __syncthreads();
    if (channel >= width) return;
    float state = 0.0f;
    for (int w = 0; w < warp; ++w) state = follow(shared[w][lane], state);
    #pragma unroll 8
    for (int64_t c = begin; c < end; ++c) {
        const int64_t at = (from_end ? chunks - 1 - c : c) * width + channel;
        const float2 m = composed[at];
        states[at] = state;
        state = follow(m, state);
    }
}

// Sequences without rows: their last state is the initial one, and so are the gradients.
__device__ __forceinline__ void pass_empty_sequences(const ScanArgs& args, const float* from, float* to, int64_t chunk, int channel, int v) {
    if (!args.in.offsets || !to) return;
    for (int64_t s = chunk; s < args.in.n_sequences; s += args.chunks)
        if (args.in.offsets[s + 1] <= args.in.offsets[s])
            for (int k = 0; k < v; ++k) to[s * args.in.width + channel + k] = from ? from[s * args.in.width + channel + k] : 0.0f;
}

// Third pass, forward.
template <typename T, int V>
__global__ void __launch_bounds__(kChunk / kForwardSteps * 32) scan_apply_kernel(const ScanArgs args) {
    constexpr int S = kForwardSteps, W = kChunk / S;
    __shared__ float2 shared[W][32 * V];
    const Place<V, S> at(args);
    Pack<T, V> x[S], g[S];
    load_rows<T, V, S>(args.in.x, args.in.x_stride, args.in, at.p0, at.channel, at.inside, x);
    load_rows<T, V, S>(args.in.gate, args.in.gate_stride, args.in, at.p0, at.channel, at.inside, g);
    const Edges edges = find_edges<S>(args.in, at.p0, at.lane);
    float h[V];
    load_state<V>(at.chunk > 0 && at.inside ? args.states : nullptr, at.chunk * args.in.width + at.channel, h);
    float a[S][V], b[S][V];
    forward_steps<T, V, S>(args, at, edges, x, g, a, b);
    #pragma unroll
    for (int k = 0; k < V; ++k) {
        float A = 1.0f, H = 0.0f;
        #pragma unroll
        for (int i = 0; i < S; ++i) {
            if (edges.first >> i & 1u) { A = kCut; H = b[i][k]; }
            else { A *= a[i][k]; H = fmaf(a[i][k], H, b[i][k]); }
        }
        shared[at.warp][at.lane * V + k] = make_float2(A, H);
    }
    __syncthreads();
    for (int w = 0; w < at.warp; ++w) {
        #pragma unroll
        for (int k = 0; k < V; ++k) h[k] = follow(shared[w][at.lane * V + k], h[k]);
    }
    #pragma unroll
    for (int i = 0; i < S; ++i) {
        const int64_t p = at.p0 + i;
        #pragma unroll
        for (int k = 0; k < V; ++k) h[k] = edges.first >> i & 1u ? b[i][k] : fmaf(a[i][k], h[k], b[i][k]);
        if (at.inside && p < args.in.rows) {
            const int64_t row = args.in.reverse ? args.in.rows - 1 - p : p;
            store_floats<T, V>(static_cast<T*>(args.h) + row * args.h_stride + at.channel, h);
        }
        if (edges.last >> i & 1u) {
            const int s = __shfl_sync(0xffffffffu, edges.sequence, i);
            if (at.inside) {
                #pragma unroll
                for (int k = 0; k < V; ++k) args.last[int64_t(s) * args.in.width + at.channel + k] = h[k];
            }
        }
    }
    if (at.warp == 0 && at.inside) pass_empty_sequences(args, args.in.initial, args.last, at.chunk, at.channel, V);
}

// Third pass, backward.
template <typename T, int V>
__global__ void __launch_bounds__(kChunk / kBackwardSteps * 32) scan_apply_backward_kernel(const ScanArgs args) {
    constexpr int S = kBackwardSteps, W = kChunk / S;
    __shared__ float2 ahead[W][32 * V], back[W][32 * V];
    const Place<V, S> at(args);
    Pack<T, V> x[S], g[S], d[S];
    load_rows<T, V, S>(args.in.gate, args.in.gate_stride, args.in, at.p0, at.channel, at.inside, g);
    load_rows<T, V, S>(args.in.x, args.in.x_stride, args.in, at.p0, at.channel, at.inside, x);
    load_rows<T, V, S>(args.grad_h, args.grad_h_stride, args.in, at.p0, at.channel, at.inside, d);
    const Edges edges = find_edges<S>(args.in, at.p0, at.lane);
    float h[V], E[V];
    load_state<V>(at.chunk > 0 && at.inside ? args.states : nullptr, at.chunk * args.in.width + at.channel, h);
    load_state<V>(at.chunk + 1 < args.chunks && at.inside ? args.grad_states : nullptr, at.chunk * args.in.width + at.channel, E);
    float t[S][V];                            // exp(-gate)
    float A[V], H[V], P[V], Q[V];             // h behind the warp's rows is A h + H; E in front of them is P E + Q
    #pragma unroll
    for (int k = 0; k < V; ++k) { A[k] = P[k] = 1.0f; H[k] = Q[k] = 0.0f; }
    bool cut = false;                         // the rows so far hold the end of a sequence
    #pragma unroll
    for (int i = 0; i < S; ++i) {
        const bool real = at.p0 + i < args.in.rows, first = edges.first >> i & 1u, last = edges.last >> i & 1u;
        float initial[V] = {}, behind[V] = {};
        if (first || last) {
            const int64_t s = int64_t(__shfl_sync(0xffffffffu, edges.sequence, i)) * args.in.width + at.channel;
            load_state<V>(first && at.inside ? args.in.initial : nullptr, s, initial);
            load_state<V>(last && at.inside ? args.grad_last : nullptr, s, behind);
        }
        #pragma unroll
        for (int k = 0; k < V; ++k) {
            t[i][k] = gate_exp(to_float<T>(g[i].v[k]));
            if (!real) continue;
            const Gate gate = gate_of(t[i][k]);
            if (first) { A[k] = kCut; H[k] = initial[k]; }
            A[k] *= gate.a;
            H[k] = fmaf(gate.a, H[k], gate.rest * to_float<T>(x[i].v[k]));
            if (cut) continue;
            Q[k] = fmaf(P[k], gate.a * (to_float<T>(d[i].v[k]) + behind[k]), Q[k]);
            P[k] = last ? kCut : P[k] * gate.a;
        }
        cut |= last;
    }
    #pragma unroll
    for (int k = 0; k < V; ++k) {
        ahead[at.warp][at.lane * V + k] = make_float2(A[k], H[k]);
        back[at.warp][at.lane * V + k] = make_float2(P[k], Q[k]);
    }
    __syncthreads();
    for (int w = 0; w < at.warp; ++w) {
        #pragma unroll
        for (int k = 0; k < V; ++k) h[k] = follow(ahead[w][at.lane * V + k], h[k]);
    }
    for (int w = W - 1; w > at.warp; --w) {
        #pragma unroll
        for (int k = 0; k < V; ++k) E[k] = follow(back[w][at.lane * V + k], E[k]);
    }
    float slope[S][V];                        // (h_{t-1} - x) a (1 - a)
    #pragma unroll
    for (int i = 0; i < S; ++i) {
        const bool first = edges.first >> i & 1u;
        if (first) {
            const int s = __shfl_sync(0xffffffffu, edges.sequence, i);
            load_state<V>(at.inside ? args.in.initial : nullptr, int64_t(s) * args.in.width + at.channel, h);
        }
        #pragma unroll
        for (int k = 0; k < V; ++k) {
            const Gate gate = gate_of(t[i][k]);
            const float value = to_float<T>(x[i].v[k]);
            slope[i][k] = (h[k] - value) * gate.a * gate.rest;
            h[k] = fmaf(gate.a, h[k], gate.rest * value);
        }
    }
    #pragma unroll
    for (int i = S - 1; i >= 0; --i) {
        const int64_t p = at.p0 + i;
        const bool first = edges.first >> i & 1u, last = edges.last >> i & 1u, real = p < args.in.rows;
        int s = 0;
        if (first || last) s = __shfl_sync(0xffffffffu, edges.sequence, i);
        if (last) load_state<V>(at.inside ? args.grad_last : nullptr, int64_t(s) * args.in.width + at.channel, E);
        float grad_x[V], grad_gate[V];
        #pragma unroll
        for (int k = 0; k < V; ++k) {
            const Gate gate = gate_of(t[i][k]);
            const float D = to_float<T>(d[i].v[k]) + E[k];
            grad_x[k] = gate.rest * D;
            grad_gate[k] = slope[i][k] * D;
            if (real) E[k] = gate.a * D;
        }
        if (real && at.inside) {
            const int64_t row = args.in.reverse ? args.in.rows - 1 - p : p;
            store_floats<T, V>(static_cast<T*>(args.grad_x) + row * args.grad_x_stride + at.channel, grad_x);
            store_floats<T, V>(static_cast<T*>(args.grad_gate) + row * args.grad_gate_stride + at.channel, grad_gate);
            if (first && args.grad_initial) {
                #pragma unroll
                for (int k = 0; k < V; ++k) args.grad_initial[int64_t(s) * args.in.width + at.channel + k] = E[k];
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
        const Gate g = gate_of(gate_exp(to_float<T>(gate[row * gate_stride + channel])));
        float* s = state + row * state_stride + channel;
        const float next = fmaf(g.a, *s, g.rest * to_float<T>(x[row * x_stride + channel]));
        *s = next;
        h[row * h_stride + channel] = from_float<T>(next);
    }
}

size_t align256(size_t n) { return (n + 255) & ~size_t(255); }
int64_t chunk_count(int64_t rows) { return (rows + kChunk - 1) / kChunk; }

bool pairs_possible(const void* p, int64_t stride, int64_t rows) { return !p || rows_aligned(p, stride, rows, 2, 4); }

template <typename T, int V> void forward_launch(ScanArgs& args, cudaStream_t stream) {
    constexpr int threads = kChunk / kForwardSteps * 32;
    args.channel_tiles = (args.in.width + 32 * V - 1) / (32 * V);
    const unsigned int blocks = unsigned(args.chunks * args.channel_tiles);
    if (args.chunks > 1) {
        scan_compose_kernel<T, V><<<blocks, threads, 0, stream>>>(args);
        scan_carry_kernel<<<(args.in.width + 31) / 32, kCarryWarps * 32, 0, stream>>>(args.composed, args.states, args.chunks, args.in.width, false);
    }
    scan_apply_kernel<T, V><<<blocks, threads, 0, stream>>>(args);
}
template <typename T, int V> void backward_launch(ScanArgs& args, cudaStream_t stream) {
    args.channel_tiles = (args.in.width + 32 * V - 1) / (32 * V);
    const unsigned int blocks = unsigned(args.chunks * args.channel_tiles);
    if (args.chunks > 1) {
        scan_compose_backward_kernel<T, V><<<blocks, kChunk / kForwardSteps * 32, 0, stream>>>(args);
        scan_carry_kernel<<<(args.in.width + 31) / 32, kCarryWarps * 32, 0, stream>>>(args.composed, args.grad_states, args.chunks, args.in.width, true);
    }
    scan_apply_backward_kernel<T, V><<<blocks, kChunk / kBackwardSteps * 32, 0, stream>>>(args);
}

// Two 16-bit channels a lane where every row allows it.
template <typename T> void scan_typed(ScanArgs& a, bool backward, cudaStream_t stream) {
    const int64_t rows = a.in.rows;
    const bool pairs = sizeof(T) == 2 && a.in.width % 2 == 0 && pairs_possible(a.in.x, a.in.x_stride, rows) && pairs_possible(a.in.gate, a.in.gate_stride, rows) &&
                       pairs_possible(a.h, a.h_stride, rows) && pairs_possible(a.grad_h, a.grad_h_stride, rows) &&
                       pairs_possible(a.grad_x, a.grad_x_stride, rows) && pairs_possible(a.grad_gate, a.grad_gate_stride, rows);
    if (pairs) { if (backward) backward_launch<T, 2>(a, stream); else forward_launch<T, 2>(a, stream); }
    else { if (backward) backward_launch<T, 1>(a, stream); else forward_launch<T, 1>(a, stream); }
}

int check_scan(const HtgsScan* scan, const char* message) {
    if (!scan || !known_type(scan->type) || scan->rows < 0 || scan->rows > 0x7fffffff || scan->width < 1 || scan->width > 65536 || scan->n_sequences < 1 ||
        (!scan->offsets && scan->rows % scan->n_sequences != 0) || (scan->rows > 0 && (!scan->x || !scan->gate)))
        return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, message);
    if (chunk_count(scan->rows) * ((scan->width + 31) / 32) > 0x7fffffff) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, message);
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
    return rows <= 0 || width <= 0 ? 0 : size_t(htgs::chunk_count(rows)) * size_t(width) * sizeof(float);
}

size_t htgs_gated_scan_workspace_bytes(int64_t rows, int32_t width) {
    if (rows <= 0 || width <= 0) return 0;
    const size_t values = size_t(htgs::chunk_count(rows)) * size_t(width);
    return htgs::align256(values * sizeof(float2)) + htgs::align256(values * sizeof(float));
}

int htgs_gated_scan(const HtgsScan* scan, void* h, int64_t h_stride, float* last, float* states, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace htgs;
    if (check_scan(scan, "htgs_gated_scan: bad type, sizes, sequences or null inputs") != HTGS_OK) return HTGS_ERR_INVALID_ARGUMENT;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (!last) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_gated_scan: last must not be null");
    if (scan->rows == 0) return pass_states(scan->initial, last, scan, s);
    if (!h) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_gated_scan: h must not be null");
    ScanArgs a{};
    a.in = *scan;
    a.chunks = chunk_count(scan->rows);
    if (a.chunks > 1 && (!workspace || !aligned(workspace, 16) || workspace_bytes < htgs_gated_scan_workspace_bytes(scan->rows, scan->width)))
        return sequence_fail(HTGS_ERR_WORKSPACE_TOO_SMALL, "htgs_gated_scan: workspace too small or not 16-byte aligned");
    const size_t values = size_t(a.chunks) * size_t(scan->width);
    a.composed = static_cast<float2*>(workspace);
    a.states = states ? states : reinterpret_cast<float*>(static_cast<char*>(workspace) + align256(values * sizeof(float2)));
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
    ScanArgs a{};
    a.in = *scan;
    a.chunks = chunk_count(scan->rows);
    if (a.chunks > 1 && (!workspace || !aligned(workspace, 16) || workspace_bytes < htgs_gated_scan_workspace_bytes(scan->rows, scan->width)))
        return sequence_fail(HTGS_ERR_WORKSPACE_TOO_SMALL, "htgs_gated_scan_backward: workspace too small or not 16-byte aligned");
    const size_t values = size_t(a.chunks) * size_t(scan->width);
    a.composed = static_cast<float2*>(workspace);
    a.grad_states = reinterpret_cast<float*>(static_cast<char*>(workspace) + align256(values * sizeof(float2)));
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
