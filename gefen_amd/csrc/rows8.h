// Eight consecutive elements as float32, at any alignment and at the end of a row.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"

namespace gefen {

template <typename T>
struct Eight {
    T v[8];
    // the first n of them exist
    __device__ __forceinline__ void load(const T* p, int n) {
        if (n >= 8) {
            constexpr int W = 16 / sizeof(T);
            using R = typename RawAny<16, sizeof(T)>::type;
#pragma unroll
            for (int i = 0; i < 8 / W; ++i) {
                const typename RawVec<16>::type r = reinterpret_cast<const R*>(p)[i];
                __builtin_memcpy(v + W * i, &r, 16);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : T{};
        }
    }
    __device__ __forceinline__ void store(T* p, int n) const {
        if (n >= 8) {
            constexpr int W = 16 / sizeof(T);
            using R = typename RawAny<16, sizeof(T)>::type;
#pragma unroll
            for (int i = 0; i < 8 / W; ++i) {
                typename RawVec<16>::type r;
                __builtin_memcpy(&r, v + W * i, 16);
                reinterpret_cast<R*>(p)[i] = r;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < n) p[i] = v[i];
        }
    }
    __device__ __forceinline__ float operator[](int i) const { return to_f32(v[i]); }
    __device__ __forceinline__ void set(int i, float x) { v[i] = from_f32<T>(x); }
};

}  // namespace gefen
