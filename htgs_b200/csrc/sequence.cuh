// Shared by the sequence operators (norm.cu, fp8.cu, fp8_matmul.cu, scan.cu): element types, vector loads and stores, and the 8-bit
// format: blocks of 128 columns (of 1 or 128 rows) share a scale, a power of two kept as the byte e + 127 (E8M0), and hold codes of
// type E4M3.  With a power of two nothing is rounded by the scale, neither when it is taken out nor when it is put back.
#pragma once

#include "kernels.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace htgs {

constexpr int kScaleBlock = 128;      // columns (and, for weights, rows) that share a scale

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N elements side by side, moved by one load or store (N * sizeof(T) is 2, 4, 8 or 16 bytes, and the address a multiple of that).
template <typename T, int N> struct alignas(N * sizeof(T)) Pack { T v[N]; };

// Two 16-bit values of one 32-bit word as floats, and back: one conversion for both.
template <typename T> __device__ __forceinline__ float2 pair_floats(uint32_t word);
template <> __device__ __forceinline__ float2 pair_floats<__nv_bfloat16>(uint32_t word) { return make_float2(__uint_as_float(word << 16), __uint_as_float(word & 0xffff0000u)); }
template <> __device__ __forceinline__ float2 pair_floats<__half>(uint32_t word) { return __half22float2(*reinterpret_cast<const __half2*>(&word)); }
template <typename T> __device__ __forceinline__ uint32_t floats_pair(float lo, float hi);
template <> __device__ __forceinline__ uint32_t floats_pair<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t floats_pair<__half>(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

template <typename T, int N> __device__ __forceinline__ void to_floats(const Pack<T, N>& pack, float (&out)[N]) {
    if constexpr (sizeof(T) == 2 && N % 2 == 0) {
        const uint32_t* words = reinterpret_cast<const uint32_t*>(&pack);
        #pragma unroll
        for (int i = 0; i < N / 2; ++i) { const float2 f = pair_floats<T>(words[i]); out[2 * i] = f.x; out[2 * i + 1] = f.y; }
    } else {
        #pragma unroll
        for (int i = 0; i < N; ++i) out[i] = to_float<T>(pack.v[i]);
    }
}
template <typename T, int N> __device__ __forceinline__ void load_floats(const T* p, float (&out)[N]) {
    to_floats<T, N>(*reinterpret_cast<const Pack<T, N>*>(p), out);
}
template <typename T, int N> __device__ __forceinline__ void store_floats(T* p, const float (&in)[N]) {
    Pack<T, N> pack;
    if constexpr (sizeof(T) == 2 && N % 2 == 0) {
        uint32_t* words = reinterpret_cast<uint32_t*>(&pack);
        #pragma unroll
        for (int i = 0; i < N / 2; ++i) words[i] = floats_pair<T>(in[2 * i], in[2 * i + 1]);
    } else {
        #pragma unroll
        for (int i = 0; i < N; ++i) pack.v[i] = from_float<T>(in[i]);
    }
    *reinterpret_cast<Pack<T, N>*>(p) = pack;
}

// Magnitude that counts for a block's scale: infinities and NaN do not, their codes are NaN whatever the scale.
__device__ __forceinline__ float finite_magnitude(float v) { const float m = fabsf(v); return m <= FLT_MAX ? m : 0.0f; }

// Least e in [-127, 120] with largest <= 448 * 2^e (448 = 1.75 * 2^8 is the largest finite E4M3 value); 0 for a block of zeros.
__device__ __forceinline__ int scale_exponent(float largest) {
    if (largest == 0.0f) return 0;
    const uint32_t bits = __float_as_uint(largest);
    const int e = int(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return max(e, -127);
}
__device__ __forceinline__ float inverse_scale(int e) { return __uint_as_float(uint32_t(127 - e) << 23); }      // 2^-e
__device__ __forceinline__ float scale_value(uint32_t byte) {                                                     // 2^(byte - 127); 255 is NaN
    return byte == 255u ? __uint_as_float(0x7fffffffu) : byte == 0u ? __uint_as_float(0x400000u) : __uint_as_float(byte << 23);
}
// Two factors whose product is that of two scales: the exponents are added first, so that a sum of codes times one factor and then the other leaves the range of
// 32 bits only where the result does.  (One scale by itself may be up to 2^127, and a sum of 16 products of codes up to 2^22.)
__device__ __forceinline__ float2 scale_factors(uint32_t a, uint32_t b) {
    const uint32_t half = (a + b) >> 1;
    return a == 255u || b == 255u ? make_float2(scale_value(255u), scale_value(255u)) : make_float2(scale_value(half), scale_value(a + b - half));
}

// Codes v * 2^-e to the nearest E4M3 value, ties to even; NaN becomes NaN.  CAREFUL: infinities do too (the conversion takes them for 448).
template <bool CAREFUL> __device__ __forceinline__ uint32_t encode2(float lo, float hi, float inverse) {
    if (CAREFUL) {
        lo = fabsf(lo) <= FLT_MAX ? lo : __uint_as_float(0x7fffffffu);
        hi = fabsf(hi) <= FLT_MAX ? hi : __uint_as_float(0x7fffffffu);
    }
    return __nv_cvt_float2_to_fp8x2(make_float2(lo * inverse, hi * inverse), __NV_SATFINITE, __NV_E4M3);
}
template <bool CAREFUL> __device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, float inverse) {
    return encode2<CAREFUL>(a, b, inverse) | encode2<CAREFUL>(c, d, inverse) << 16;
}
// N codes side by side (N 1, 2, 4 or 8).
template <bool CAREFUL, int N> __device__ __forceinline__ void store_codes(uint8_t* to, const float (&v)[N], float inverse) {
    if constexpr (N == 8) *reinterpret_cast<uint2*>(to) = make_uint2(encode4<CAREFUL>(v[0], v[1], v[2], v[3], inverse), encode4<CAREFUL>(v[4], v[5], v[6], v[7], inverse));
    else if constexpr (N == 4) *reinterpret_cast<uint32_t*>(to) = encode4<CAREFUL>(v[0], v[1], v[2], v[3], inverse);
    else if constexpr (N == 2) *reinterpret_cast<uint16_t*>(to) = uint16_t(encode2<CAREFUL>(v[0], v[1], inverse));
    else *to = uint8_t(encode2<CAREFUL>(v[0], 0.0f, inverse) & 0xffu);
}
// Largest magnitude; a NaN says nothing.  Infinite where one is, which is when the maximum is taken again over finite_magnitude, and CAREFUL codes follow.
template <int N> __device__ __forceinline__ float largest_magnitude(const float (&v)[N], float so_far = 0.0f) {
    #pragma unroll
    for (int i = 0; i < N; ++i) so_far = fmaxf(so_far, fabsf(v[i]));
    return so_far;
}
template <int N> __device__ __forceinline__ float largest_finite(const float (&v)[N], float so_far = 0.0f) {
    #pragma unroll
    for (int i = 0; i < N; ++i) so_far = fmaxf(so_far, finite_magnitude(v[i]));
    return so_far;
}
__device__ __forceinline__ float2 decode2(uint32_t codes) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(codes & 0xffffu), __NV_E4M3);
    return __half22float2(__half2(h));
}

__device__ __forceinline__ float warp_sum(float v) {
    #pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
template <int LANES> __device__ __forceinline__ float lanes_max(float v) {
    #pragma unroll
    for (int d = LANES / 2; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
    return v;
}

// ---- stretches of a row that begin anywhere ----------------------------------------------------------------------------------------
// Where rows do not begin on 16 bytes, a warp brings `count` values of a row into shared memory of its own, and sends some out, in the 16-byte pieces of memory that
// they lie in.  In shared memory they lie as far behind a multiple of 16 as in memory; a slot has 16 bytes more than the values.  What a piece holds beside them is
// copied (it lies in the same 16 bytes as a value that exists) and not looked at.
template <typename T> __device__ __forceinline__ uint32_t misplaced(const T* p) { return uint32_t(reinterpret_cast<uintptr_t>(p)) & 15u; }
template <typename T> __device__ __forceinline__ T* in_slot(unsigned char* slot, const T* at) { return reinterpret_cast<T*>(slot + misplaced(at)); }
template <int MOST, typename T> __device__ __forceinline__ void bring(unsigned char* slot, const T* from, int count, int lane) {        // at most MOST values
    const int m = int(misplaced(from)), left = count > 0 ? m + count * int(sizeof(T)) - 16 * lane : 0;
    const char* at = reinterpret_cast<const char*>(from) + (16 * lane - m);
    const uint32_t to = smem_u32(slot) + 16 * lane;
    #pragma unroll
    for (int i = 0; i < (MOST * int(sizeof(T)) + 15 + 511) / 512; ++i)
        if (512 * i < left) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + 512 * i), "l"(at + 512 * i) : "memory");
}
// Whole pieces, then the values of the first and the last one, a lane for each.
template <int MOST, typename T> __device__ __forceinline__ void send(const unsigned char* slot, T* to, int count, int lane) {
    constexpr int kSize = int(sizeof(T)), kValues = 16 / kSize;
    if (count <= 0) return;
    const int m = int(misplaced(to)), end = m + count * kSize, last = end & ~15;
    char* at = reinterpret_cast<char*>(to) - m;
    const bool early = 16 * lane < m;        // lane 0's first piece is not whole
    #pragma unroll
    for (int i = 0; i < (MOST * kSize + 15 + 511) / 512; ++i)
        if (512 * i < last - 16 * lane && !(i == 0 && early)) *reinterpret_cast<uint4*>(at + 16 * lane + 512 * i) = *reinterpret_cast<const uint4*>(slot + 16 * lane + 512 * i);
    const bool front = lane < kValues;
    const int b = front ? lane * kSize : last + (lane - kValues) * kSize;
    if (b < end && (front ? b >= m && m != 0 : lane < 2 * kValues && (last > 0 || m == 0)))
        *reinterpret_cast<T*>(at + b) = *reinterpret_cast<const T*>(slot + b);
}
__device__ __forceinline__ void copies_begun() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int BEGUN> __device__ __forceinline__ void copies_done() {          // all but the last BEGUN groups, for the whole warp
    asm volatile("cp.async.wait_group %0;" ::"n"(BEGUN) : "memory");
    __syncwarp();
}

// The limit of a wait that polls, in nanoseconds of the time in which it polled: between two polls a hundredth of a second counts at most, so that time in which the
// kernel did not run at all (the GPU was another process's, or the process was suspended) is not held against it.
struct WaitLimit {
    static constexpr uint64_t kMostGap = 10000000;
    uint64_t left, before;
    __host__ __device__ __forceinline__ WaitLimit(uint64_t limit, uint64_t now) : left(limit), before(now) {}
    __host__ __device__ __forceinline__ bool over(uint64_t now) {
        const uint64_t gap = now - before < kMostGap ? now - before : kMostGap;
        before = now;
        if (left <= gap) return true;
        left -= gap;
        return false;
    }
};

// Blocks of a cluster: what block `block` has at this block's shared address `address`, and a barrier of all their threads.  The barrier's instructions are
// of whole warps (.aligned), which have to come back together first if they stand behind a branch or a loop that some lanes took.
__device__ __forceinline__ uint32_t peer_address(uint32_t address, uint32_t block) {
    uint32_t there;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(address), "r"(block));
    return there;
}
__device__ __forceinline__ float peer_float(uint32_t address, uint32_t block) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(peer_address(address, block)) : "memory");
    return v;
}
__device__ __forceinline__ float4 peer_float4(uint32_t address, uint32_t block) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(peer_address(address, block)) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_barrier() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---- host side of the entry points ----------------------------------------------------------------------------------------

inline int sequence_fail(int code, const char* message) { set_last_error(message); return code; }
inline int sequence_status(const char* what) {
    const cudaError_t err = cudaGetLastError();
    if (err == cudaSuccess) return HTGS_OK;
    (void)what;
    return sequence_fail(HTGS_ERR_CUDA, cudaGetErrorString(err));
}
inline bool known_type(int type) { return type == HTGS_FLOAT32 || type == HTGS_FLOAT16 || type == HTGS_BFLOAT16; }
inline size_t type_bytes(int type) { return type == HTGS_FLOAT32 ? 4 : 2; }
inline bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
// A row-major matrix whose rows all begin on a multiple of `bytes`.
inline bool rows_aligned(const void* p, int64_t stride, int64_t rows, size_t element, size_t bytes) {
    return aligned(p, bytes) && (rows <= 1 || (uint64_t(stride) * element) % bytes == 0);
}

}  // namespace htgs
