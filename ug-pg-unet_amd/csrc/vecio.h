// Vector access to values stored in fp32 or bf16, shared by the group-norm and the
// distillation kernels.
#pragma once
#include "common.h"

namespace ugpg {

template <int N> struct RawBytes;
template <> struct RawBytes<2> { typedef uint16_t t; };
template <> struct RawBytes<4> { typedef uint32_t t; };
template <> struct RawBytes<8> { typedef uint2 t; };
template <> struct RawBytes<16> { typedef uint4 t; };
template <> struct RawBytes<32> { struct t { uint4 a, b; }; };

// V consecutive values of T as loaded (bf16 stays packed: half the registers)
template <typename T, int V> struct Pack {
    union {
        typename RawBytes<sizeof(T) * V>::t raw;
        uint32_t w[sizeof(T) * V >= 4 ? sizeof(T) * V / 4 : 1];
        uint16_t h[sizeof(T) * V / 2];
    };
    __device__ __forceinline__ Pack() {}
    __device__ __forceinline__ void load(const T* p) {
        raw = *reinterpret_cast<const typename RawBytes<sizeof(T) * V>::t*>(p);
    }
    __device__ __forceinline__ float get(int e) const {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(w[e]);
        } else if constexpr (V == 1) {
            return __uint_as_float((uint32_t)h[0] << 16);
        } else {
            return __uint_as_float((e & 1) ? (w[e / 2] & 0xffff0000u) : (w[e / 2] << 16));
        }
    }
    __device__ __forceinline__ void set(int e, float v) {
        if constexpr (sizeof(T) == 4) {
            w[e] = __float_as_uint(v);
        } else {
            union { __bf16 b; uint16_t u; } c;
            c.b = (__bf16)v;  // round to nearest even: half a bf16 step, once, at the store
            h[e] = c.u;
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        *reinterpret_cast<typename RawBytes<sizeof(T) * V>::t*>(p) = raw;
    }
};

}  // namespace ugpg
