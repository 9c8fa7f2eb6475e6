// fg_host.hpp -- what the library's host sides share: how a failure is reported.
#ifndef FG_HOST_HPP
#define FG_HOST_HPP

#include <hip/hip_runtime.h>

#include <string>

#include "../../include/flashgann.h"

namespace fgk {
// Sets the calling thread's fg_last_error() text and returns `code`.
int fail(int code, const std::string &msg);

// body(), for a C entry point: no C++ exception (a message that found no memory)
// leaves it.
template <class R, class F>
R guarded(F body) noexcept {
    try {
        return body();
    } catch (...) {
        return FG_ENOMEM;
    }
}
}  // namespace fgk

#define FG_HIP(call, what)                                                                          \
    do {                                                                                            \
        hipError_t _e = (call);                                                                     \
        if (_e != hipSuccess) return fgk::fail(FG_EDEVICE, std::string(what) + ": " + hipGetErrorString(_e)); \
    } while (0)

#endif
