#pragma once

// What the translation units of libopworks_ops.so share: the thread-local
// message of the last failed call and the guard that turns exceptions into -1.

#include <exception>
#include <string>

namespace opworks_ops {

std::string &last_error();

template <typename F> int guarded(F &&f) {
    try {
        f();
        return 0;
    } catch (const std::exception &e) {
        last_error() = e.what();
    } catch (...) {
        last_error() = "unknown C++ exception";
    }
    return -1;
}

} // namespace opworks_ops
