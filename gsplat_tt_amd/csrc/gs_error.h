// gs_error.h - the error policy of every C entry point: exceptions inside, a
// status code and a thread-local message outside.
#pragma once

#include <hip/hip_runtime.h>

#include <new>
#include <stdexcept>
#include <string>

#include "../../include/gsplat_hip.h"

namespace gs {

// gs_last_error()'s text of this thread
inline thread_local std::string g_err;

struct GsError : std::runtime_error {
    int code;
    GsError(int c, const std::string& m) : std::runtime_error(m), code(c) {}
};

template <class F>
int guard(F&& f) {
    try {
        f();
        return GS_OK;
    } catch (const GsError& e) {
        g_err = e.what();
        return e.code;
    } catch (const std::exception& e) {
        g_err = e.what();
        return GS_E_DEVICE;
    }
}

}  // namespace gs

#define HIPCHK(x)                                                                            \
    do {                                                                                     \
        hipError_t e_ = (x);                                                                 \
        if (e_ != hipSuccess)                                                                \
            throw gs::GsError(GS_E_DEVICE, std::string(#x) + ": " + hipGetErrorString(e_)); \
    } while (0)

#define REQUIRE(cond, msg)                                   \
    do {                                                     \
        if (!(cond)) throw gs::GsError(GS_E_INVALID, (msg)); \
    } while (0)
