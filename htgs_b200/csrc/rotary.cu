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

constexpr int kRotaryThreads = 256, kMostPairs = 128, kRotaryRows = 8;

struct RotaryArgs {
    HtgsRotary r;
    double turns[kMostPairs];           // per unit of position
    uint8_t axis[kMostPairs];
};

// N pairs of a head: the first values at `a`, the second ones at `b`, or all of them at `a`, neighbours.
template <typename T, int N, bool INTERLEAVED> __device__ __forceinline__ void turn(const T* x, T* y, int second, const float2* angles) {
    float a[N], b[N];
    if constexpr (INTERLEAVED) {
        float both[2 * N];
        if constexpr (N * 2 * sizeof(T) <= 16) load_floats<T, 2 * N>(x, both);
        else {
            float low[N], high[N];
            load_floats<T, N>(x, low);
            load_floats<T, N>(x + N, high);
            #pragma unroll
            for (int i = 0; i < N; ++i) { both[i] = low[i]; both[N + i] = high[i]; }
        }
        #pragma unroll
        for (int i = 0; i < N; ++i) { a[i] = both[2 * i]; b[i] = both[2 * i + 1]; }
    } else {
        load_floats<T, N>(x, a);
        load_floats<T, N>(x + second, b);
    }
    #pragma unroll
    for (int i = 0; i < N; ++i) {
        const float2 w = angles[i];
        const float u = a[i] * w.x - b[i] * w.y, v = a[i] * w.y + b[i] * w.x;
        a[i] = u;
        b[i] = v;
    }
    if constexpr (INTERLEAVED) {
        float both[2 * N];
        #pragma unroll
        for (int i = 0; i < N; ++i) { both[2 * i] = a[i]; both[2 * i + 1] = b[i]; }
        if constexpr (N * 2 * sizeof(T) <= 16) store_floats<T, 2 * N>(y, both);
        else {
            float low[N], high[N];
            #pragma unroll
            for (int i = 0; i < N; ++i) { low[i] = both[i]; high[i] = both[N + i]; }
            store_floats<T, N>(y, low);
            store_floats<T, N>(y + N, high);
        }
    } else {
        store_floats<T, N>(y, a);
        store_floats<T, N>(y + second, b);
    }
}

// A block has a few rows: their cosines and sines first, which all heads share, then all heads of both tensors.
template <typename T, int N, bool INTERLEAVED> __global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const __grid_constant__ RotaryArgs args) {
    extern __shared__ float2 angles[];                   // [rows][pairs]
    grid_dependency();
    const HtgsRotary& r = args.r;
    const int pairs = r.width / 2, heads = r.heads[0] + r.heads[1], chunks = pairs / N;
    const int64_t first = int64_t(blockIdx.x) * kRotaryRows;
    const int rows = int(min(int64_t(kRotaryRows), r.rows - first));
    for (int i = threadIdx.x; i < rows * pairs; i += kRotaryThreads) {
        const int row = i / pairs, pair = i - row * pairs;
        const int64_t at = (first + row) * r.positions_stride + args.axis[pair];
        const double position = r.positions_type == 0 ? double(static_cast<const float*>(r.positions)[at]) : double(static_cast<const int32_t*>(r.positions)[at]);
        const double t = position * args.turns[pair], whole = t - rint(t), quarter = rint(4.0 * whole);       // whole: -1/2 to 1/2
        float sine, cosine;
        sincospif(float(2.0 * (whole - 0.25 * quarter)), &sine, &cosine);
        const int q = int(quarter) & 3;
        float2 w = q & 1 ? make_float2(-sine, cosine) : make_float2(cosine, sine);
        if (q & 2) w = make_float2(-w.x, -w.y);
        if (r.inverse) w.y = -w.y;
        angles[i] = w;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * heads * chunks; i += kRotaryThreads) {
        const int chunk = i % chunks, rest = i / chunks, row = rest / heads;
        int head = rest - row * heads;
        const int which = head >= r.heads[0];
        if (which) head -= r.heads[0];
        const int at = INTERLEAVED ? 2 * N * chunk : N * chunk;
        const T* x = static_cast<const T*>(r.x[which]) + (first + row) * r.x_stride[which] + head * r.x_head_stride[which] + at;
        T* y = static_cast<T*>(r.y[which]) + ((first + row) * r.heads[which] + head) * r.width + at;
        turn<T, N, INTERLEAVED>(x, y, pairs, angles + row * pairs + N * chunk);
    }
}

template <typename T, int N> int launch_rotary(const RotaryArgs& args, cudaStream_t stream) {
    const dim3 grid(unsigned((args.r.rows + kRotaryRows - 1) / kRotaryRows));
    const size_t smem = size_t(kRotaryRows) * (args.r.width / 2) * sizeof(float2);
    const cudaError_t err = args.r.interleaved ? launch_after(rotary_kernel<T, N, true>, grid, kRotaryThreads, smem, stream, args)
                                               : launch_after(rotary_kernel<T, N, false>, grid, kRotaryThreads, smem, stream, args);
    return err == cudaSuccess ? sequence_status("htgs_rotary") : sequence_fail(HTGS_ERR_CUDA, cudaGetErrorString(err));
}

// Pairs that a thread turns: as many as lie side by side in 16 bytes, if all rows and heads begin on such.
template <typename T> int rotary_typed(const RotaryArgs& args, cudaStream_t stream) {
    const HtgsRotary& r = args.r;
    const auto fits = [&](int n) {
        const int unit = r.interleaved && 2 * n * int(sizeof(T)) <= 16 ? 2 * n : n;      // values of one load
        bool ok = r.width / 2 % n == 0;
        for (int i = 0; i < 2; ++i)
            if (r.heads[i])
                ok = ok && aligned(r.x[i], unit * sizeof(T)) && aligned(r.y[i], unit * sizeof(T)) && (r.rows == 1 || r.x_stride[i] % unit == 0) && (r.heads[i] == 1 || r.x_head_stride[i] % unit == 0);
        return ok;
    };
    if constexpr (sizeof(T) == 2) { if (fits(8)) return launch_rotary<T, 8>(args, stream); }
    if (fits(4)) return launch_rotary<T, 4>(args, stream);
    if (fits(2)) return launch_rotary<T, 2>(args, stream);
    return launch_rotary<T, 1>(args, stream);
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
