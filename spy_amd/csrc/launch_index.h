// Which entries of an array the threads of a launch take where all of them share it.  Plain C++: a test on the host walks the same functions.
#pragma once

#include <cstdint>

// Entry `first`, then every `step`-th.  A launch has up to 2^32 - 1 threads, so that neither fits an int, and the sum of both no 32 bits.
constexpr int64_t launch_first(uint32_t block, uint32_t threads, uint32_t thread) { return (int64_t)block * threads + thread; }
constexpr int64_t launch_step(uint32_t blocks, uint32_t threads) { return (int64_t)blocks * threads; }
