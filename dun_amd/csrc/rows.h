// Rows of fp32 / bf16 / fp16 elements as the layer norm and checkpoint kernels walk them, and the 8-bit checkpoint format.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "common.h"

namespace dun {

typedef unsigned int u32;
typedef unsigned short u16;
typedef unsigned long long u64;

// ---- vectors of one lane -------------------------------------------------------------------------------------------------
// Four elements per lane and load.  The vector types carry the alignment of ONE element: global memory takes vector accesses
// at any element address on this hardware, so odd widths and strides run the same loads as aligned ones.
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef u16 u16x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef u32 u32x2_t __attribute__((ext_vector_type(2)));
typedef u32 u32x4_t __attribute__((ext_vector_type(4)));

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

constexpr int E = 4;

__device__ __forceinline__ void load_vec(const float* p, float* v) {
    const f32x4_any q = *reinterpret_cast<const f32x4_any*>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = q[e];
}
template <typename T>
__device__ __forceinline__ void load_vec(const T* p, float* v) {
    const u16x4_any q = *reinterpret_cast<const u16x4_any*>(p);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = to_f32(T{q[e]});
}
__device__ __forceinline__ void store_vec(float* p, const float* v) {
    f32x4_any q;
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] = v[e];
    *reinterpret_cast<f32x4_any*>(p) = q;
}
template <typename T>
__device__ __forceinline__ void store_vec(T* p, const float* v) {
    u16x4_any q;
#pragma unroll
    for (int e = 0; e < E; ++e) q[e] = from_f32<T>(v[e]).bits;
    *reinterpret_cast<u16x4_any*>(p) = q;
}
// Four elements of a row from column i0 on, as they lie in memory: kernels hold many of them, and 16-bit ones in half the registers.
// Columns from `cols` on read as 0.  No branches around the loads, which would keep a row's loads from overlapping: a vector that passes the
// row's end is loaded from where it ends with the row and moved down.  (Rows of fewer than four elements are read one by one.)
__device__ __forceinline__ int clamp_vec(int i0, int cols) { return i0 < cols - E ? i0 : cols - E; }
template <typename T> struct RawVec {
    static constexpr int W = 2;
    u32 w[W];
    __device__ __forceinline__ void load(const T* row, int i0) {
        const u16x4_any q = *reinterpret_cast<const u16x4_any*>(row + i0);
        w[0] = (u32)q[0] | (u32)q[1] << 16;
        w[1] = (u32)q[2] | (u32)q[3] << 16;
    }
    __device__ __forceinline__ void load_end(const T* row, int i0, int cols) {
        if (cols < E) {  // (the same for all lanes)
            w[0] = w[1] = 0;
            for (int e = 0; e < E; ++e)
                if (i0 + e < cols) w[e >> 1] |= (u32)row[i0 + e].bits << (16 * (e & 1));
            return;
        }
        load(row, clamp_vec(i0, cols));
        const int past = i0 - (cols - E);  // elements to move down by: 1 .. 3, or all where i0 >= cols
        const u64 q = (u64)w[1] << 32 | w[0];
        const u64 m = past <= 0 ? q : past >= E ? 0 : q >> (16 * past);
        w[0] = (u32)m;
        w[1] = (u32)(m >> 32);
    }
    __device__ __forceinline__ float operator[](int e) const { return to_f32(T{(u16)(w[e >> 1] >> (16 * (e & 1)))}); }
    // what was converted before this point is converted again behind it instead of being kept as twice as many registers
    __device__ __forceinline__ void forget() { asm volatile("" : "+v"(w[0]), "+v"(w[1])); }
};
template <> struct RawVec<float> {
    static constexpr int W = 4;
    u32 w[W];
    __device__ __forceinline__ void load(const float* row, int i0) {
        float v[E];
        load_vec(row + i0, v);
#pragma unroll
        for (int e = 0; e < E; ++e) w[e] = __builtin_bit_cast(u32, v[e]);
    }
    __device__ __forceinline__ void load_end(const float* row, int i0, int cols) {
        if (cols < E) {
#pragma unroll
            for (int e = 0; e < E; ++e) w[e] = i0 + e < cols ? __builtin_bit_cast(u32, row[i0 + e]) : 0u;
            return;
        }
        load(row, clamp_vec(i0, cols));
        const int past = i0 - (cols - E);
        if (past > 0) {
            if (past & 1) { w[0] = w[1]; w[1] = w[2]; w[2] = w[3]; w[3] = 0; }
            if (past & 2) { w[0] = w[2]; w[1] = w[3]; w[2] = w[3] = 0; }
            if (past >= E) { w[0] = w[1] = w[2] = w[3] = 0; }
        }
    }
    __device__ __forceinline__ float operator[](int e) const { return __builtin_bit_cast(float, w[e]); }
    __device__ __forceinline__ void forget() {}
};
// the same as floats, wherever it lies
template <typename T>
__device__ __forceinline__ void load_part(const T* row, int i0, int cols, float* v) {
    RawVec<T> q;
    q.load_end(row, i0, cols);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = q[e];
}
template <typename T>
__device__ __forceinline__ void store_part(T* row, int i0, int cols, const float* v) {
    if (i0 + E <= cols) {
        store_vec(row + i0, v);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (i0 + e < cols) row[i0 + e] = from_f32<T>(v[e]);
    }
}
// max(v, floor) that keeps NaN: floor 0 rectifies, minus infinity leaves v as it is
__device__ __forceinline__ float max_nan(float v, float floor) { return __builtin_elementwise_maximum(v, floor); }
__device__ __forceinline__ float rectify(float v) { return max_nan(v, 0.f); }

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
// largest |v| of the 8 lanes that hold a group, as bits: unsigned order is the order of magnitudes, NaN above infinity
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
    o = dpp_move_u32<DPP_ROW_HALF_MIRROR>(m);
    return o > m ? o : m;
}
// Packs the four elements of a lane into a word; the 8 lanes of a group call together (the first a multiple of 8).
// v must be 0 in columns from the row's end on.
__device__ __forceinline__ u32 act8_pack(const float* v, bool rectified, u32* byte) {
    *byte = act8_byte(act8_group_max(v), rectified);
    const bool ok = *byte != ACT8_NONFINITE;
    const float inv = act8_scale(254u - (ok ? *byte : 127u));
    u32 word = 0;
#pragma unroll
    for (int j = 0; j < E; ++j) {
        int c = ok ? (int)rintf(v[j] * inv) : 0;
        if (rectified && v[j] > 0.f && ok) c = c < 1 ? 1 : c;
        word |= (u32)(c + (rectified ? 0 : 128)) << (8 * j);
    }
    return word;
}
// (0 * inf is NaN, as wanted)
__device__ __forceinline__ void act8_values(u32 word, u32 byte, float zero, float* v) {
    const float s = act8_scale(byte);
#pragma unroll
    for (int j = 0; j < E; ++j) v[j] = ((float)((word >> (8 * j)) & 0xffu) - zero) * s;
}
// a lane's word of column i0 on, and the group's byte from the group's first lane
__device__ __forceinline__ void act8_store(uint8_t* codes, uint8_t* exps, size_t row, int groups, int i0, u32 word, u32 byte) {
    if (i0 < groups * ACT8_GROUP) {
        *reinterpret_cast<u32*>(codes + row * groups * ACT8_GROUP + i0) = word;
        if (i0 % ACT8_GROUP == 0) exps[row * groups + i0 / ACT8_GROUP] = (uint8_t)byte;
    }
}

// ---- sums over partial results ---------------------------------------------------------------------------------------------
// out[i] = sum_r part[r][i], i < n: C columns x SL slices of the rows per workgroup; a slice adds its rows four chains at a time, the
// slices are added in order.  Always the same order, so the same bits.  Elements from n1 on go to out2.
template <int SL>
__global__ __launch_bounds__(32 * SL) void sum_rows_kernel(const float* part, int P, size_t n, float* out, size_t n1, float* out2) {
    __shared__ float lds[SL][32];
    const int c = threadIdx.x & 31, s = threadIdx.x >> 5;
    const size_t i = (size_t)blockIdx.x * 32 + c;
    float a[4] = {0.f, 0.f, 0.f, 0.f};
    if (i < n) {
        int r = s;
        for (; r + 3 * SL < P; r += 4 * SL) {
#pragma unroll
            for (int k = 0; k < 4; ++k) a[k] += part[(size_t)(r + k * SL) * n + i];
        }
        for (int k = 0; r < P; r += SL, ++k) a[k & 3] += part[(size_t)r * n + i];
    }
    lds[s][c] = (a[0] + a[1]) + (a[2] + a[3]);
    __syncthreads();
    if (s == 0 && i < n) {
        float t = lds[0][c];
#pragma unroll
        for (int j = 1; j < SL; ++j) t += lds[j][c];
        if (i < n1)
            out[i] = t;
        else
            out2[i - n1] = t;
    }
}
// few partial rows: four elements a thread, no LDS
static __global__ __launch_bounds__(256) void sum_few_rows_kernel(const float* part, int P, size_t n, float* out, size_t n1, float* out2) {
    const size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= n) return;
    if (i + 4 <= n1) {
        float a[4] = {0.f, 0.f, 0.f, 0.f}, v[4];
#pragma unroll 4
        for (int r = 0; r < P; ++r) {
            load_vec(part + (size_t)r * n + i, v);
#pragma unroll
            for (int e = 0; e < 4; ++e) a[e] += v[e];
        }
        store_vec(out + i, a);
        return;
    }
    for (size_t j = i; j < n && j < i + 4; ++j) {
        float a = 0.f;
        for (int r = 0; r < P; ++r) a += part[(size_t)r * n + j];
        if (j < n1)
            out[j] = a;
        else
            out2[j - n1] = a;
    }
}
static inline void launch_sum_rows(const float* part, size_t P, size_t n, float* out, size_t n1, float* out2, hipStream_t s) {
    // rows x elements, us: 8 x 10100 one thread an element 5.7, 8 slices 2.7; 4 x 4.2 M 15 and 32; 128 x 20480 45 and 11
    if (P <= 8 && n >= (size_t)1 << 18)
        hipLaunchKernelGGL(sum_few_rows_kernel, dim3((unsigned)((n + 1023) / 1024)), dim3(256), 0, s, part, (int)P, n, out, n1, out2);
    else if (P <= 64)
        hipLaunchKernelGGL((sum_rows_kernel<8>), dim3((unsigned)((n + 31) / 32)), dim3(256), 0, s, part, (int)P, n, out, n1, out2);
    else
        hipLaunchKernelGGL((sum_rows_kernel<32>), dim3((unsigned)((n + 31) / 32)), dim3(1024), 0, s, part, (int)P, n, out, n1, out2);
}
static __global__ __launch_bounds__(256) void zero_floats_kernel(float* p, size_t n) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) p[i] = 0.f;
}
static inline void launch_zero_floats(float* p, size_t n, hipStream_t s) {
    const size_t need = (n + 255) / 256;
    hipLaunchKernelGGL(zero_floats_kernel, dim3((unsigned)(need < 4096 ? need : 4096)), dim3(256), 0, s, p, n);
}

}  // namespace dun
