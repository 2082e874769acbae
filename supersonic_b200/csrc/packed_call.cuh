// A C entry's arguments as one run of bytes, each on its natural alignment (Python's struct.Struct of the same types): an entry of 31
// arguments costs a caller 0.9 us so and 3.5 us with one conversion an argument.
#pragma once
#include "common.cuh"
#include <cstring>
#include <tuple>

template <typename... A>
static int ssb_call_packed(int (*f)(A...), const char* bytes) {
    size_t at = 0;
    auto next = [&](auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        at = (at + alignof(T) - 1) / alignof(T) * alignof(T);
        T v;
        memcpy(&v, bytes + at, sizeof(T));
        at += sizeof(T);
        return v;
    };
    return std::apply(f, std::tuple<A...>{next((A*)nullptr)...});      // braces: first argument first
}
#define SSB_PACKED(f_) \
    SSB_API int f_##_packed(const char* bytes) { return ssb_call_packed(f_, bytes); }
