// Division by a number that the host knows: n / by as the upper half of n * ceil(2^32 / by), which is exact while n * by < 2^32.
#pragma once
#include "common.cuh"

struct FrDivide {
    unsigned by, magic;                   // magic 0: divide the ordinary way
    // most: the greatest number that is divided
    FrDivide(long long n = 1, long long most = 1)
        : by((unsigned)n), magic(n > 1 && most * n < (1ll << 32) ? (unsigned)(((1ull << 32) + n - 1) / n) : 0) {}
    // where the host has made sure that most * n < 2^32
    __device__ __forceinline__ int quick(int n) const { return by == 1 ? n : (int)__umulhi((unsigned)n, magic); }
    __device__ __forceinline__ int operator()(int n) const {
        return by == 1 ? n : magic != 0 ? (int)__umulhi((unsigned)n, magic) : (int)((unsigned)n / by);
    }
};
