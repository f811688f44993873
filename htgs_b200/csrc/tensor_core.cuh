// Shared by the kernels on the tensor cores (fp8_matmul.cu, attention_tiles.cu): waits with a time limit, tensor memory, tensor maps.
#pragma once

#include "sequence.cuh"

#include <cuda.h>

#include <cstring>
#include <mutex>

namespace htgs {

constexpr uint64_t kWaitNanoseconds = 2000000000ull;

// Tensor memory (512 columns of an SM) is waited for without a limit, so a block that holds some may not wait for a block that still has to get its own.  The 8-bit product takes its columns ahead of its
// wait for the kernel before, attention behind it; what keeps them apart is shared memory: no block that uses tensor memory has less than kLeastTensorShared, and one that takes columns ahead has so much that
// none of those fits beside it.
constexpr int kSharedOfSm = 228 * 1024, kSharedOfSystem = 1024, kLeastTensorShared = 98 * 1024;         // of system: in each block, beside its own
constexpr bool alone_with_tensor_memory(int smem) { return smem + kLeastTensorShared + 2 * kSharedOfSystem > kSharedOfSm; }

__device__ __forceinline__ uint64_t nanoseconds() { uint64_t t; asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t)); return t; }

__device__ __forceinline__ void arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// False if the time limit ran out or another role has given up.  Out of line: the roles' loops are single threads whose every instruction counts.
static __device__ __noinline__ bool wait_longer(uint32_t bar, uint32_t parity, volatile uint32_t* failed) {
    WaitLimit limit(kWaitNanoseconds, nanoseconds());
    for (;;) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) return true;
        if (*failed) return false;
        if (limit.over(nanoseconds())) { *failed = 1; return false; }
    }
}
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}
// The same in line, for kernels that give registers from one warp to another, which may not call.
__device__ __forceinline__ bool wait_in_line(uint64_t* bar, uint32_t parity, volatile uint32_t* failed) {
    if (mbar_test(bar, parity)) return true;
    WaitLimit limit(kWaitNanoseconds, nanoseconds());
    for (;;) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*failed) return false;
        if (limit.over(nanoseconds())) { *failed = 1; return false; }
    }
}
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, volatile uint32_t* failed) {
    return mbar_try_wait(bar, parity) || wait_longer(smem_u32(bar), parity, failed);
}
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
// A place in a ring of N, and the parity of the round it is in.
template <int N> struct Ring {
    uint32_t at = 0, round = 0;
    __device__ __forceinline__ void next() { if (++at == N) { at = 0; round ^= 1; } }
};

__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tmem_load32(uint32_t address, uint32_t (&v)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
                   "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]),
                   "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(address));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// ---- host ---------------------------------------------------------------------------------------------------------------------

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                 CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiled encode_tiled() {
    static const EncodeTiled found = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult result;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &result) != cudaSuccess || result != cudaDriverEntryPointSuccess) f = nullptr;
        return reinterpret_cast<EncodeTiled>(f);
    }();
    return found;
}

// A word for each device in the host's memory, which a kernel sets when one of its waits runs out.  The next call of its kind on that device reports it, or who asks.
class ErrorWords {
public:
    unsigned int* of(int device) {
        std::call_once(once_, [this] {
            cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;       // the first call may be inside a capture
            cudaThreadExchangeStreamCaptureMode(&mode);
            void* p = nullptr;
            if (cudaHostAlloc(&p, kMostDevices * sizeof(unsigned int), cudaHostAllocPortable | cudaHostAllocMapped) != cudaSuccess) {
                p = nullptr;
                cudaGetLastError();
            }
            cudaThreadExchangeStreamCaptureMode(&mode);
            if (p) std::memset(p, 0, kMostDevices * sizeof(unsigned int));
            words_ = static_cast<unsigned int*>(p);
        });
        return words_ && device >= 0 && device < kMostDevices ? words_ + device : nullptr;
    }
    static constexpr int kMostDevices = 64;

private:
    std::once_flag once_;
    unsigned int* words_ = nullptr;
};
inline int current_device() {
    int device = -1;
    cudaGetDevice(&device);
    return device;
}
// What a word says, once: whoever reads it first clears it.
inline int reported(unsigned int* word, const char* message) {
    if (!word || !__atomic_load_n(word, __ATOMIC_RELAXED) || !__atomic_exchange_n(word, 0u, __ATOMIC_ACQ_REL)) return HTGS_OK;
    return sequence_fail(HTGS_ERR_DEVICE_FLAG, message);
}

}  // namespace htgs
