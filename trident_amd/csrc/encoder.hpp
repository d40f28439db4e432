// Shared by the encoder's kernels (embedding.hip, layernorm.hip, adamw.hip, fp8mm.hip): element
// types, 16-byte loads and stores through float, wave reductions, and the C entry points' errors.
//
// Every sum is held in float32 and every result is rounded to its type once.  Rows may start at any
// element: gfx950 takes 16-byte accesses at any element's address, so one vector form serves every
// row pitch, and a row's last vector is shifted back to end with the row (it overlaps the one before).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/trident_hip.h"
#include "common.hpp"

namespace trident {

// Records the calling thread's last error (trident_last_error) and returns `code`; never throws.
int capi_fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int capi_check_launch(const char* what);

using f16_t = _Float16;
using bf16_t = __bf16;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);  // elements of one 16-byte access

inline bool dtype_ok(int32_t t) { return t == TRIDENT_F32 || t == TRIDENT_F16 || t == TRIDENT_BF16; }

// Calls f with std::true_type or std::false_type.
template <typename F>
inline void with_bool(bool b, F&& f) {
    if (b) f(std::true_type{});
    else f(std::false_type{});
}

// Calls f with a value of the element type that `t` names.
template <typename F>
inline void with_dtype(int32_t t, F&& f) {
    if (t == TRIDENT_F32) f(float{});
    else if (t == TRIDENT_F16) f(f16_t{});
    else f(bf16_t{});
}

// A result larger than the card's L2 (eight times 4 MB) is written past it: nothing of it would be left
// for the next kernel, and the rows that this one reads again stay (131,072 embedding rows of 960
// bfloat16 from a table of 126 MB: 78 us through L2, 47 past it).  Reading past it pays where nothing is
// read twice (AdamW on 62M elements: 314 to 300 us) and not where the next pass reads the same again
// (layer norm's rows, forward and backward: 193 to 196 us).
constexpr int64_t kL2Bytes = 32 << 20;

// `WORDS`, 4 to 16 bytes, from any element's address.
template <bool PAST_L2, typename WORDS>
__device__ __forceinline__ WORDS load_words(const void* p) {
    typedef WORDS any __attribute__((aligned(2), may_alias));
    if constexpr (PAST_L2) return __builtin_nontemporal_load(reinterpret_cast<const any*>(p));
    else return *reinterpret_cast<const any*>(p);
}

// N elements from any element's address, held as they are stored: one element, or whole 16-byte
// accesses.
template <typename T, int N>
struct Vec {
    static constexpr int kWords = N == 1 ? 1 : N / kVec<T>;
    u32x4 raw[kWords];
    T one;
    __device__ __forceinline__ void load(const T* __restrict__ p) {
        if constexpr (N == 1) {
            one = *p;
        } else {
            static_assert(N % kVec<T> == 0, "whole 16-byte accesses");
#pragma unroll
            for (int k = 0; k < kWords; ++k) raw[k] = load_words<false, u32x4>(p + k * kVec<T>);
        }
    }
    __device__ __forceinline__ void get(float (&f)[N]) const {
        if constexpr (N == 1) {
            f[0] = (float)one;
        } else {
#pragma unroll
            for (int k = 0; k < kWords; ++k) {
                if constexpr (sizeof(T) == 4) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) f[4 * k + i] = __uint_as_float(raw[k][i]);
                } else if constexpr (std::is_same<T, bf16_t>::value) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        f[8 * k + 2 * i] = __uint_as_float(raw[k][i] << 16);
                        f[8 * k + 2 * i + 1] = __uint_as_float(raw[k][i] & 0xffff0000u);
                    }
                } else {
                    typedef f16_t h8 __attribute__((ext_vector_type(8)));
                    const h8 h = __builtin_bit_cast(h8, raw[k]);
#pragma unroll
                    for (int i = 0; i < 8; ++i) f[8 * k + i] = (float)h[i];
                }
            }
        }
    }
};

template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* __restrict__ p, float (&f)[N]) {
    Vec<T, N> v;
    v.load(p);
    v.get(f);
}

template <typename T, int N>
__device__ __forceinline__ void store_vec(T* __restrict__ p, const float (&f)[N]) {
    if constexpr (N == 1) {
        p[0] = (T)f[0];
    } else {
        typedef T tv __attribute__((ext_vector_type(N)));
        tv t;
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = (T)f[i];
        __builtin_memcpy(p, &t, sizeof(t));
    }
}

// A template argument: of two stores under a condition the compiler makes one, an ordinary one.
template <bool PAST_L2, typename T, int N>
__device__ __forceinline__ void put_vec(T* __restrict__ p, const float (&f)[N]) {
    if constexpr (N == 1 || !PAST_L2) {
        store_vec(p, f);
    } else {
        typedef T tv __attribute__((ext_vector_type(N)));
        typedef uint32_t words __attribute__((ext_vector_type(N * sizeof(T) / 4)));
        typedef words any __attribute__((aligned(2)));
        tv t;
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = (T)f[i];
        __builtin_nontemporal_store(__builtin_bit_cast(words, t), reinterpret_cast<any*>(p));
    }
}

// Sum over the 64 lanes of a wave, the same in every lane: each step adds a neighbour's partial sum in
// the vector unit itself (no trip through LDS), 16 lanes, then the rows of 16; lane 63 ends with all.
template <int CTRL>
__device__ __forceinline__ float add_from(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float wave_sum(float v) {
    v = add_from<0x111>(v);  // one lane down
    v = add_from<0x112>(v);  // two
    v = add_from<0x114>(v);
    v = add_from<0x118>(v);
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x142, 0xa, 0xf, true));  // row 0 to 1, 2 to 3
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x143, 0xc, 0xf, true));  // rows 0, 1 to 2, 3
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), kWave - 1));
}

}  // namespace trident
