// Shared by the files that implement C ABI entry points: the opaque handle
// for synchronous inference and the exception guard.
#pragma once
#include <algorithm>
#include <cstring>
#include <exception>
#include <memory>
#include <string>

#include "engine.hpp"

struct azb_infer {
    std::unique_ptr<azb::Inference> impl;
};

namespace azb {

inline void put_text(char* dst, size_t cap, const std::string& s) {
    if (!dst || cap == 0) return;
    const size_t n = std::min(cap - 1, s.size());
    std::memcpy(dst, s.data(), n);
    dst[n] = '\0';
}

// Runs fn; an exception becomes -1 and `prefix` + its message in err.
template <class Fn>
int guarded(char* err, size_t cap, const char* prefix, Fn fn) {
    try {
        fn();
        return 0;
    } catch (const std::exception& e) {
        put_text(err, cap, std::string(prefix) + e.what());
    } catch (...) {
        put_text(err, cap, std::string(prefix) + "unknown error");
    }
    return -1;
}

}  // namespace azb
