// Rotary positions with several axes: in each head, pair j of the values (a, b) becomes
//
//   (a cos t - b sin t, a sin t + b cos t),   t = position of the row along the pair's axis * base^(-i / n)
//
// for the i-th of the n pairs of that axis.  The gradient is the same with -t.  Positions may be far (10^6 rows): t is reduced in 64 bits, in turns, to an eighth of a turn on either
// side of a quarter, and only then rounded to 32.
#include "sequence.cuh"

#include <cmath>

namespace htgs {

namespace {

constexpr int kRotaryThreads = 256, kMostPairs = 128, kMostRows = 30, kAhead = 2;

struct RotaryArgs {
    HtgsRotary r;
    double turns[kMostPairs];           // per unit of position
    uint8_t axis[kMostPairs];
};

// How pairs lie: first values apart from second ones; side by side; or side by side, but a pair does not begin on a multiple of its size, so that its values come one by one.
enum PairLayout { kHalves, kInterleaved, kInterleavedAnywhere };
// Whether N pairs are one load.
template <typename T, int N, PairLayout LAYOUT> constexpr bool kWholePairs = LAYOUT == kInterleaved && 2 * N * sizeof(T) <= 16;

// N pairs of a head: as they lie in memory, and as first and second values.
template <typename T, int N, PairLayout LAYOUT> struct Pairs {
    static constexpr bool INTERLEAVED = LAYOUT != kHalves, whole = kWholePairs<T, N, LAYOUT>;
    static_assert(LAYOUT != kInterleavedAnywhere || N == 1, "values one by one");
    Pack<T, whole ? 2 * N : N> one, two;
    __device__ __forceinline__ void load(const T* x, int second) {
        one = *reinterpret_cast<const decltype(one)*>(x);
        if (!whole) two = *reinterpret_cast<const decltype(two)*>(x + (INTERLEAVED ? N : second));
    }
    // cosines of a row from the first pair on, then, `pairs` further each time, sines and minus sines
    __device__ __forceinline__ void turn(const float* angles, int pairs, T* y, int second) const {
        float values[2 * N];
        if constexpr (whole) to_floats<T, 2 * N>(one, values);
        else {
            to_floats<T, N>(one, *reinterpret_cast<float (*)[N]>(values));
            to_floats<T, N>(two, *reinterpret_cast<float (*)[N]>(values + N));
        }
        float c[N], d[N], m[N];
        load_floats<float, N>(angles, c);
        load_floats<float, N>(angles + pairs, d);
        load_floats<float, N>(angles + 2 * pairs, m);
        constexpr int kStep = N == 1 ? 1 : 2;
        #pragma unroll
        for (int i = 0; i < N; i += kStep) {
            const int a0 = INTERLEAVED ? 2 * i : i, b0 = INTERLEAVED ? 2 * i + 1 : N + i, a1 = INTERLEAVED ? 2 * i + 2 : i + 1, b1 = INTERLEAVED ? 2 * i + 3 : N + i + 1;
            if constexpr (N == 1) {
                const float a = values[a0], b = values[b0];
                values[a0] = fmaf(b, m[i], a * c[i]);
                values[b0] = fmaf(a, d[i], b * c[i]);
            } else {
                const f32x2 a = pack2(values[a0], values[a1]), b = pack2(values[b0], values[b1]), cosine = pack2(c[i], c[i + 1]);
                const float2 u = unpack2(fma2(b, pack2(m[i], m[i + 1]), mul2(a, cosine))), v = unpack2(fma2(a, pack2(d[i], d[i + 1]), mul2(b, cosine)));
                values[a0] = u.x; values[a1] = u.y;
                values[b0] = v.x; values[b1] = v.y;
            }
        }
        if constexpr (whole) store_floats<T, 2 * N>(y, values);
        else {
            store_floats<T, N>(y, *reinterpret_cast<const float (*)[N]>(values));
            store_floats<T, N>(y + (INTERLEAVED ? N : second), *reinterpret_cast<const float (*)[N]>(values + N));
        }
    }
};

// Sine and cosine of z, |z| at most pi / 4: odd and even polynomials of least maximal error for what lies behind z and 1 - z^2 / 2 (found by linear programming), 2^-24 off at most in 32 bits.
__device__ __forceinline__ void sine_cosine(float z, float& sine, float& cosine) {
    const float w = z * z;
    sine = fmaf(z * w, fmaf(fmaf(-0.0001951528392964974f, w, 0.00833216030150652f), w, -0.16666655242443085f), z);
    cosine = fmaf(fmaf(fmaf(fmaf(2.4438451873720624e-05f, w, -0.001388736767694354f), w, 0.04166664555668831f), w, -0.5f), w, 1.0f);
}

// Bound by HBM: 100000 rows of 10 heads of 64 in bf16 54 us, 4.8 TB/s (52 without angles); as many rows as two loads of a block's threads hold, five blocks on an SM (four 59 us, six 61).
//
// A block has a few rows: their cosines and sines, which all heads share, while the first values are on their way; then all heads of both tensors.  In 64 bits only what multiplies and adds: rounding is by a large
// number, whose low bits then are the quarter, and positions are converted once a row, since conversions and roundings are made by a unit that takes longer than all the rest.
template <typename T, int N, PairLayout LAYOUT> __global__ void __launch_bounds__(kRotaryThreads, 5) rotary_kernel(const __grid_constant__ RotaryArgs args, const int rows_of_block) {
    extern __shared__ __align__(16) float angles[];       // [rows][3][pairs], a row's on 16 bytes
    __shared__ double positions[kMostRows * 4], turns[kMostPairs];
    __shared__ uint8_t axis[kMostPairs];
    grid_dependency();
    const HtgsRotary& r = args.r;
    const int pairs = r.width / 2, heads = r.heads[0] + r.heads[1], chunks = pairs / N, pitch = (3 * pairs + 3) / 4 * 4, of_row = heads * chunks;
    const int64_t first = int64_t(blockIdx.x) * rows_of_block;
    const int rows = int(min(int64_t(rows_of_block), r.rows - first)), count = rows * of_row;
    struct Place { const T* x; T* y; int angle; };
    const auto place = [&](int i) {
        const int row = i / of_row, rest = i - row * of_row, all = rest / chunks, chunk = rest - all * chunks, which = all >= r.heads[0], head = all - (which ? r.heads[0] : 0);
        const int at = LAYOUT == kHalves ? N * chunk : 2 * N * chunk;
        return Place{static_cast<const T*>(r.x[which]) + (first + row) * r.x_stride[which] + head * r.x_head_stride[which] + at,
                     static_cast<T*>(r.y[which]) + ((first + row) * r.heads[which] + head) * r.width + at, row * pitch + N * chunk};
    };
    for (int i = threadIdx.x; i < rows * r.axes; i += kRotaryThreads) {
        const int row = i / r.axes;
        const int64_t at = (first + row) * r.positions_stride + (i - row * r.axes);
        positions[i] = r.positions_type == 0 ? double(static_cast<const float*>(r.positions)[at]) : double(static_cast<const int32_t*>(r.positions)[at]);
    }
    for (int i = threadIdx.x; i < pairs; i += kRotaryThreads) { turns[i] = args.turns[i]; axis[i] = args.axis[i]; }         // arguments are read one address at a time (21 of 70 us)
    Pairs<T, N, LAYOUT> values[kAhead];
    Place places[kAhead];
    #pragma unroll
    for (int k = 0; k < kAhead; ++k) {
        const int i = int(threadIdx.x) + k * kRotaryThreads;
        places[k] = place(i < count ? i : 0);
        if (i < count) values[k].load(places[k].x, pairs);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * pairs; i += kRotaryThreads) {
        const int row = i / pairs, pair = i - row * pairs;
        constexpr double kWhole = 6755399441055744.0;          // 1.5 * 2^52
        const double t = positions[row * r.axes + axis[pair]] * turns[pair], whole = t - ((t + kWhole) - kWhole), quarter = fma(4.0, whole, kWhole);       // whole: -1/2 to 1/2
        float sine, cosine;
        sine_cosine(float(6.283185307179586477 * fma(-0.25, quarter - kWhole, whole)), sine, cosine);
        const int q = __double2loint(quarter);
        float x = q & 1 ? -sine : cosine, y = q & 1 ? cosine : sine;
        if (q & 2) { x = -x; y = -y; }
        if (r.inverse) y = -y;
        float* const to = angles + row * pitch + pair;
        to[0] = x; to[pairs] = y; to[2 * pairs] = -y;
    }
    __syncthreads();
    #pragma unroll
    for (int k = 0; k < kAhead; ++k)
        if (int(threadIdx.x) + k * kRotaryThreads < count) values[k].turn(angles + places[k].angle, pairs, places[k].y, pairs);
    for (int i = threadIdx.x + kAhead * kRotaryThreads; i < count; i += kRotaryThreads) {           // one row of many heads
        const Place p = place(i);
        Pairs<T, N, LAYOUT> v;
        v.load(p.x, pairs);
        v.turn(angles + p.angle, pairs, p.y, pairs);
    }
}

template <typename T, int N, PairLayout LAYOUT> int launch_rotary(const RotaryArgs& args, cudaStream_t stream) {
    // Rows whose values the threads of a block load at once.
    const int items = (args.r.heads[0] + args.r.heads[1]) * (args.r.width / 2 / N), most = kAhead * kRotaryThreads / items, rows = most < 1 ? 1 : most > kMostRows ? kMostRows : most;
    const dim3 grid(unsigned((args.r.rows + rows - 1) / rows));
    const size_t smem = size_t(rows) * ((3 * (args.r.width / 2) + 3) / 4 * 4) * sizeof(float);
    static_assert(kMostRows * 3 * kMostPairs * 4 <= 47 * 1024, "shared memory");
    const cudaError_t err = launch_after(rotary_kernel<T, N, LAYOUT>, grid, kRotaryThreads, smem, stream, args, rows);
    return err == cudaSuccess ? sequence_status("htgs_rotary") : sequence_fail(HTGS_ERR_CUDA, cudaGetErrorString(err));
}

// Pairs that a thread turns: as many as lie side by side in 16 bytes, if all rows and heads begin on such.
template <typename T, int N, PairLayout LAYOUT> bool fits(const HtgsRotary& r) {
    constexpr int unit = kWholePairs<T, N, LAYOUT> ? 2 * N : N;             // values of one load
    bool ok = r.width / 2 % N == 0;
    for (int i = 0; i < 2; ++i)
        if (r.heads[i])
            ok = ok && aligned(r.x[i], unit * sizeof(T)) && aligned(r.y[i], unit * sizeof(T)) && (r.rows == 1 || r.x_stride[i] % unit == 0) && (r.heads[i] == 1 || r.x_head_stride[i] % unit == 0);
    return ok;
}
template <typename T, PairLayout LAYOUT> int rotary_laid_out(const RotaryArgs& args, cudaStream_t stream) {
    if constexpr (sizeof(T) == 2) { if (fits<T, 8, LAYOUT>(args.r)) return launch_rotary<T, 8, LAYOUT>(args, stream); }
    if (fits<T, 4, LAYOUT>(args.r)) return launch_rotary<T, 4, LAYOUT>(args, stream);
    if (fits<T, 2, LAYOUT>(args.r)) return launch_rotary<T, 2, LAYOUT>(args, stream);
    if (fits<T, 1, LAYOUT>(args.r)) return launch_rotary<T, 1, LAYOUT>(args, stream);
    return launch_rotary<T, 1, LAYOUT == kHalves ? kHalves : kInterleavedAnywhere>(args, stream);
}
template <typename T> int rotary_typed(const RotaryArgs& args, cudaStream_t stream) {
    return args.r.interleaved ? rotary_laid_out<T, kInterleaved>(args, stream) : rotary_laid_out<T, kHalves>(args, stream);
}

}  // namespace

}  // namespace htgs

extern "C" {

int htgs_rotary(const HtgsRotary* rotary, void* stream) {
    using namespace htgs;
    if (!rotary || !known_type(rotary->type)) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_rotary: no arguments or unknown element type");
    RotaryArgs args;
    args.r = *rotary;
    const HtgsRotary& r = args.r;
    if (r.rows < 0 || r.rows > 0x7fffff00 || r.heads[0] < 1 || r.heads[1] < 0 || r.heads[0] > 65536 || r.heads[1] > 65536)
        return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_rotary: rows must be below 2^31 - 256, and heads 1 to 65536 (0 of x[1] for none)");
    if (r.width < 2 || r.width > 2 * kMostPairs || r.width % 2) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_rotary: heads must be 2 to 256 values wide, an even number");
    if (r.axes < 1 || r.axes > 4 || (r.positions_type != 0 && r.positions_type != 1) || !(r.base > 0.0 && std::isfinite(r.base)))
        return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_rotary: 1 to 4 axes, positions of type 0 (float) or 1 (int32), a positive base");
    int pairs = 0;
    for (int a = 0; a < r.axes; ++a) {
        const int n = r.sections[a];
        if (n < 0 || n > r.width / 2 - pairs) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_rotary: sections must add up to width / 2");
        const double ratio = n ? std::pow(r.base, -1.0 / n) : 1.0;
        double turns = 0.15915494309189533577;           // 1 / (2 pi)
        for (int i = 0; i < n; ++i, ++pairs, turns *= ratio) {
            args.turns[pairs] = turns;
            args.axis[pairs] = uint8_t(a);
        }
    }
    if (pairs != r.width / 2) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_rotary: sections must add up to width / 2");
    if (r.rows == 0) return HTGS_OK;
    for (int i = 0; i < 2; ++i)
        if (r.heads[i] && (!r.x[i] || !r.y[i] || r.x_stride[i] < 0 || r.x_head_stride[i] < 0)) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_rotary: x and y must not be null, and strides not negative");
    if (!r.positions || r.positions_stride < 0) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_rotary: positions must not be null");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (r.type == HTGS_FLOAT32) return rotary_typed<float>(args, s);
    if (r.type == HTGS_FLOAT16) return rotary_typed<__half>(args, s);
    return rotary_typed<__nv_bfloat16>(args, s);
}

}  // extern "C"
