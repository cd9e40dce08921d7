// What the operators on a caller's pages share (paged.cu, prefix.cu).  Interface only.
#pragma once
#include <atomic>

#include "common.cuh"

namespace lcu {

// A kernel's attributes are set once per device: the calls cost as much as a launch.
class OncePerDevice {
    std::atomic<unsigned long long> done_{0};

  public:
    template <class F> int run(F set) {
        int dev = 0;
        LCU_CHECK_CUDA(cudaGetDevice(&dev));
        const unsigned long long bit = 1ull << (dev & 63);
        if (dev < 64 && (done_.load(std::memory_order_acquire) & bit)) return LCU_OK;
        const int rc = set();
        if (rc == LCU_OK && dev < 64) done_.fetch_or(bit, std::memory_order_release);
        return rc;
    }
};

// checks a caller's pages, and copies them with a stride from head to head that may be used where there is one KV head (whose stride nobody reads)
int kv_pages_take(lcu_kv_pages *out, const lcu_kv_pages *p, int nkvh, const char *who);

}  // namespace lcu
