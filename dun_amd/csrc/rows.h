// Rows of fp32 / bf16 / fp16 elements as the layer norm and checkpoint kernels walk them, and the 8-bit checkpoint format.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "common.h"

namespace dun {

typedef unsigned int u32;
typedef unsigned short u16;

// ---- vectors of one lane -------------------------------------------------------------------------------------------------
// 16 bytes per lane and load.  The vector types carry the alignment of ONE element: global memory takes 16-byte accesses
// at any element address on this hardware, so odd widths and strides run the same loads as aligned ones.
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef u16 u16x8_any __attribute__((ext_vector_type(8), aligned(2)));
typedef u32 u32x2_t __attribute__((ext_vector_type(2)));

struct bf16_t { u16 bits; };
struct fp16_t { u16 bits; };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16_t v) { return __builtin_bit_cast(float, (u32)v.bits << 16); }
__device__ __forceinline__ float to_f32(fp16_t v) { return (float)__builtin_bit_cast(_Float16, v.bits); }
// one rounding, to nearest even
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16_t from_f32<bf16_t>(float v) {
    return bf16_t{__builtin_bit_cast(u16, (__bf16)v)};
}
template <> __device__ __forceinline__ fp16_t from_f32<fp16_t>(float v) {
    return fp16_t{__builtin_bit_cast(u16, (_Float16)v)};
}

template <typename T> struct Row { static constexpr int E = 8; };
template <> struct Row<float> { static constexpr int E = 4; };

__device__ __forceinline__ void load_vec(const float* p, float* v) {
    const f32x4_any q = *reinterpret_cast<const f32x4_any*>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = q[e];
}
template <typename T>
__device__ __forceinline__ void load_vec(const T* p, float* v) {
    const u16x8_any q = *reinterpret_cast<const u16x8_any*>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = to_f32(T{q[e]});
}
__device__ __forceinline__ void store_vec(float* p, const float* v) {
    f32x4_any q;
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] = v[e];
    *reinterpret_cast<f32x4_any*>(p) = q;
}
template <typename T>
__device__ __forceinline__ void store_vec(T* p, const float* v) {
    u16x8_any q;
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = from_f32<T>(v[e]).bits;
    *reinterpret_cast<u16x8_any*>(p) = q;
}
// E elements of a row from column i0 on; columns from `cols` on read as `fill` and are not written
template <typename T>
__device__ __forceinline__ void load_part(const T* row, int i0, int cols, float* v, float fill = 0.f) {
    constexpr int E = Row<T>::E;
    if (i0 + E <= cols) {
        load_vec(row + i0, v);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = i0 + e < cols ? to_f32(row[i0 + e]) : fill;
    }
}
template <typename T>
__device__ __forceinline__ void store_part(T* row, int i0, int cols, const float* v) {
    constexpr int E = Row<T>::E;
    if (i0 + E <= cols) {
        store_vec(row + i0, v);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (i0 + e < cols) row[i0 + e] = from_f32<T>(v[e]);
    }
}
// E fp32 elements (weights, statistics) at column i0, for lanes that hold E elements of another type
template <int E>
__device__ __forceinline__ void load_f32(const float* row, int i0, int cols, float* v) {
    if (i0 + E <= cols) {
#pragma unroll
        for (int e = 0; e < E; e += 4) load_vec(row + i0 + e, v + e);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = i0 + e < cols ? row[i0 + e] : 0.f;
    }
}

// max(v, 0) that keeps NaN
__device__ __forceinline__ float rectify(float v) { return v <= 0.f ? 0.f : v; }

// ---- the 8-bit checkpoint --------------------------------------------------------------------------------------------------
// codes [rows][32 G] and biased exponents [rows][G], G = ceil(cols / 32): value = (code - zero) 2^(byte - 127), zero = 128
// (signed) or 0 (rectified input, >= 0).  2^e is the smallest power of two, not below 2^-126, for which the group's
// largest magnitude rounds to at most 127 (255): with amax = m 2^k, m in [1, 2), that is e = k - 6 (k - 7), one more
// where m 64 (m 128) rounds up past the limit, m >= 127.5 / 64 (255.5 / 128) -- a comparison of the mantissa's bits, so the
// choice involves no rounding.  A power of two keeps the scaling exact and the value representable in bf16 (at most 8
// significant bits), which is what lets a product with checkpointed values run on the bf16 matrix cores unrounded.
// A positive rectified element keeps code >= 1 (value > 0 is ReLU's mask).  A group with an infinity or a NaN, or whose
// largest magnitude would round to 2^128, has byte 255 and code = zero throughout: 0 * inf, NaN, for every element, so that a
// diverged forward shows in the backward.
constexpr int ACT8_GROUP = 32;
constexpr u32 ACT8_NONFINITE = 255;

__device__ __forceinline__ u32 act8_byte(u32 amax_bits, bool rectified) {
    const int k = (int)(amax_bits >> 23);
    const u32 m = amax_bits & 0x7fffffu;
    const int up = m >= (rectified ? 0x7f8000u : 0x7f0000u);
    if (k + up >= 255) return ACT8_NONFINITE;
    const int byte = k + up - (rectified ? 7 : 6);
    return (u32)(byte < 1 ? 1 : byte);
}
__device__ __forceinline__ float act8_scale(u32 byte) { return __builtin_bit_cast(float, byte << 23); }

template <int CTRL>
__device__ __forceinline__ u32 dpp_move_u32(u32 v) {
    return (u32)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
}
// largest |v| of the 32 / E lanes that hold a group, as bits: unsigned order is the order of magnitudes, NaN above infinity
template <int E>
__device__ __forceinline__ u32 act8_group_max(const float* v) {
    u32 m = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const u32 b = __builtin_bit_cast(u32, v[e]) & 0x7fffffffu;
        m = b > m ? b : m;
    }
    u32 o = dpp_move_u32<DPP_QUAD_XOR1>(m);
    m = o > m ? o : m;
    o = dpp_move_u32<DPP_QUAD_XOR2>(m);
    m = o > m ? o : m;
    if (E == 4) {
        o = dpp_move_u32<DPP_ROW_HALF_MIRROR>(m);
        m = o > m ? o : m;
    }
    return m;
}
// Packs E elements of a lane; the lanes of a group call together (32 / E consecutive lanes, the first a multiple of that).
// v must be 0 in columns from the row's end on.  Returns the group's byte; w holds the codes, four to a word.
template <int E>
__device__ __forceinline__ u32 act8_pack(const float* v, bool rectified, u32* w) {
    const u32 byte = act8_byte(act8_group_max<E>(v), rectified);
    const bool ok = byte != ACT8_NONFINITE;
    const float inv = act8_scale(254u - (ok ? byte : 127u));
    const int zero = rectified ? 0 : 128, least = rectified ? 1 : -127;
#pragma unroll
    for (int q = 0; q < E / 4; ++q) {
        u32 word = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float x = v[4 * q + j];
            int c = ok ? (int)rintf(x * inv) : 0;
            if (rectified && x > 0.f && ok) c = c < least ? least : c;
            word |= (u32)(c + zero) << (8 * j);
        }
        w[q] = word;
    }
    return byte;
}
// E values from codes; zs = zero * scale (0 * inf is NaN, as wanted)
template <int E>
__device__ __forceinline__ void act8_values(const u32* w, u32 byte, float zero, float* v) {
    const float s = act8_scale(byte);
#pragma unroll
    for (int q = 0; q < E / 4; ++q)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * q + j] = ((float)((w[q] >> (8 * j)) & 0xffu) - zero) * s;
}
template <int E>
__device__ __forceinline__ void act8_load_words(const uint8_t* p, u32* w) {
    if (E == 4) {
        w[0] = *reinterpret_cast<const u32*>(p);
    } else {
        const u32x2_t q = *reinterpret_cast<const u32x2_t*>(p);
        w[0] = q[0];
        w[E / 4 - 1] = q[1];
    }
}
template <int E>
__device__ __forceinline__ void act8_store_words(uint8_t* p, const u32* w) {
    if (E == 4) {
        *reinterpret_cast<u32*>(p) = w[0];
    } else {
        u32x2_t q;
        q[0] = w[0];
        q[1] = w[E / 4 - 1];
        *reinterpret_cast<u32x2_t*>(p) = q;
    }
}

}  // namespace dun
