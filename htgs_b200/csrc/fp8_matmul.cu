// out = a * b^T for 8-bit matrices with a power-of-two scale for each block of 128 columns (fp8.cu):
//
//   out[m, n] = sum over k of  sa[m, k / 128] sb[n / (1 or 128), k / 128]  a[m, k] b[n, k]
//
// The product of two E4M3 codes is exact in 32 bits, and a scale shifts its exponent, so the only roundings are those of the 32-bit
// sum and the last one to the output's type.
#include "sequence.cuh"

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

template <typename T> int matmul_typed(const MatmulArgs& args, cudaStream_t stream) {
    constexpr int R = 8;
    const dim3 grid(unsigned((args.b.rows + kRowsBlock / 32 - 1) / (kRowsBlock / 32)), unsigned((args.a.rows + R - 1) / R));
    matmul_rows_kernel<T, R><<<grid, kRowsBlock, 0, stream>>>(args);
    return sequence_status("htgs_fp8_matmul");
}

bool matrix_ok(const HtgsFp8Matrix* m) {
    return m && m->rows >= 0 && m->rows <= 0x7fffffff && m->width >= 0 && m->width <= 0x7fffffff && (m->rows_per_scale == 1 || m->rows_per_scale == kScaleBlock) &&
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
        return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_fp8_matmul: matrices need sizes in [0, 2^31), codes on 16 bytes, scales on 4 bytes, rows_per_scale 1 or 128");
    if (a->width != b->width) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_fp8_matmul: a and b must have the same width");
    if (!known_type(out_type)) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_fp8_matmul: unknown element type");
    if (a->rows == 0 || b->rows == 0) return HTGS_OK;
    if (!out || out_stride < b->rows) return sequence_fail(HTGS_ERR_INVALID_ARGUMENT, "htgs_fp8_matmul: out must not be null, and its rows must hold b.rows values");
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
