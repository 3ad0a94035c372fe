// hb_ptx.cuh -- mbarrier and tcgen05 fence wrappers shared by the
// tensor-core kernels.
#pragma once

namespace hb {
namespace tc {

__device__ __forceinline__ unsigned smem_u32(const void *p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(unsigned a, unsigned count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(a), "r"(count));
}
__device__ __forceinline__ void mbar_arrive(unsigned a) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(a) : "memory");
}
__device__ __forceinline__ void mbar_arrive_tx(unsigned a, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(a), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(unsigned a, unsigned parity) {
    unsigned ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(ok)
        : "r"(a), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ unsigned long long gtimer() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
// Bounded wait for the given phase parity.  Gives up after `limit_ns`, or
// at once when another thread of the CTA has given up (*abort set, unless
// abort is null); returns false then, after recording `code` in *err.
__device__ __forceinline__ bool mbar_wait(unsigned a, unsigned parity, volatile int *abort, int *err, int code,
                                          unsigned long long limit_ns) {
    if (mbar_try(a, parity)) return true;
    const unsigned long long t0 = gtimer();
    for (unsigned it = 1;; it++) {
        if (mbar_try(a, parity)) return true;
        if (abort && *abort) return false;
        if ((it & 63) == 0 && gtimer() - t0 > limit_ns) {
            if (abort) *abort = 1;
            atomicOr(err, code);
            return false;
        }
    }
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

}  // namespace tc
}  // namespace hb
