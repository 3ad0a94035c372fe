// hb_error.hpp -- status codes and the message of the last failure at the
// C boundary: every entry point runs its body inside guard(), which turns
// an exception into a negative HB_E* code.
#pragma once
#include <cuda_runtime.h>

#include <new>
#include <stdexcept>
#include <string>

#include "../../include/helrm_b200.h"

namespace hb {

struct HbError : std::runtime_error {
    int code;
    HbError(int c, const std::string &m) : std::runtime_error(m), code(c) {}
};
#define HB_THROW(code, msg) throw hb::HbError(code, msg)

inline void cuda_check(cudaError_t e, const char *what) {
    if (e != cudaSuccess) {
        if (e == cudaErrorMemoryAllocation) HB_THROW(HB_ENOMEM, std::string(what) + ": out of device memory");
        HB_THROW(HB_ECUDA, std::string(what) + ": " + cudaGetErrorString(e));
    }
}

// Keeps the message that helrm_LastError() returns on this thread.
void set_last_error(const char *msg) noexcept;
void call_succeeded() noexcept;

template <class F>
int guard(F &&f) {
    try {
        f();
        call_succeeded();
        return HB_OK;
    } catch (const HbError &e) {
        set_last_error(e.what());
        return e.code;
    } catch (const std::invalid_argument &e) {
        set_last_error(e.what());
        return HB_EINVAL;
    } catch (const std::out_of_range &e) {
        set_last_error(e.what());
        return HB_ENOENT;
    } catch (const std::bad_alloc &e) {
        set_last_error("host allocation failed");
        return HB_ENOMEM;
    } catch (const std::exception &e) {
        set_last_error(e.what());
        return HB_ECUDA;
    }
}

}  // namespace hb

#define HB_API extern "C" __attribute__((visibility("default")))
