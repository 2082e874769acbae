// What a launch looks up or sets once on every device: a kernel's attributes are the current device's alone.
#pragma once
#include <cuda_runtime.h>

constexpr int SSB_MOST_DEVICES = 64;

template <typename T>
struct SsbPerDevice {
    T of[SSB_MOST_DEVICES];
    // The current device's (zero at first); null where there is none.
    T* here() {
        int d = -1;
        return cudaGetDevice(&d) == cudaSuccess && d >= 0 && d < SSB_MOST_DEVICES ? of + d : nullptr;
    }
};
