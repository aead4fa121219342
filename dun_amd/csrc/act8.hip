// 8-bit activation checkpoints: pack, unpack, and a Linear layer's weight gradient taken from one.
//
//   dw[o, i] = sum_r dy[r, o] value(r, i),  value = (code - zero) 2^(byte - 127),  db[o] = sum_r dy[r, o]
//
// A value has at most 8 significant bits and a power-of-two scale: it IS a bf16 number.  An fp32 dy is the exact sum of
// three bf16 numbers (its significand's upper, middle and lower 8 bits, cut off and not rounded: every remainder is exact), an
// fp16 one of two, a bf16 one of itself.  So the product runs as three (two, one) bf16 MFMAs per tile, accumulating in
// fp32, with no bit of the operands lost -- at a third of the bf16 matrix rate, five times the fp32 one.
//
// The reduction index is the ROW of both operands, while an MFMA wants 8 consecutive reduction indices in a lane: a
// lane therefore loads 8 rows (4 of the codes) of a few columns and hands the columns on as they lie in its registers; the
// transposition costs no instruction.
#include "rows.h"

namespace dun {

typedef u32 u32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef u32 u32_any __attribute__((aligned(2)));
typedef u32 u32x2_any __attribute__((ext_vector_type(2), aligned(4)));

// ---- pack / unpack: elementwise streams -----------------------------------------------------------------------------------------
// One vector of E columns per lane; a row is G * 32 / E vectors (padded groups included), so the lanes of a group are neighbours.
template <typename T>
__global__ __launch_bounds__(256) void act8_pack_kernel(const T* x, size_t ldx, uint8_t* codes, uint8_t* exps, size_t vecs,
                                                        u32 vpr, int cols, int relu) {
    constexpr int E = Row<T>::E, GV = ACT8_GROUP / E;
    for (size_t v0 = (size_t)blockIdx.x * 256; v0 < vecs; v0 += (size_t)gridDim.x * 256) {
        const size_t i = v0 + threadIdx.x;
        if (i >= vecs) break;  // (vecs is a multiple of GV: the lanes of a group stay together)
        size_t row;
        u32 vec;
        if (vecs <= 0xffffffffu) {
            row = (u32)i / vpr;
            vec = (u32)i - (u32)row * vpr;
        } else {
            row = i / vpr;
            vec = (u32)(i - row * vpr);
        }
        float v[E];
        load_part(x + row * ldx, (int)vec * E, cols, v);
        if (relu) {
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = rectify(v[e]);
        }
        u32 w[E / 4];
        const u32 byte = act8_pack<E>(v, relu, w);
        act8_store_words<E>(codes + i * E, w);
        if (vec % GV == 0) exps[i / GV] = (uint8_t)byte;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void act8_unpack_kernel(const uint8_t* codes, const uint8_t* exps, T* out, size_t ldo,
                                                          size_t vecs, u32 vpr, int cols, float zero) {
    constexpr int E = Row<T>::E, GV = ACT8_GROUP / E;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < vecs; i += (size_t)gridDim.x * 256) {
        size_t row;
        u32 vec;
        if (vecs <= 0xffffffffu) {
            row = (u32)i / vpr;
            vec = (u32)i - (u32)row * vpr;
        } else {
            row = i / vpr;
            vec = (u32)(i - row * vpr);
        }
        u32 w[E / 4];
        float v[E];
        act8_load_words<E>(codes + i * E, w);
        act8_values<E>(w, exps[i / GV], zero, v);
        store_part(out + row * ldo, (int)vec * E, cols, v);
    }
}

// ---- weight gradient ------------------------------------------------------------------------------------------------------------------
struct WgradP {
    const void* dy;
    const uint8_t* codes;
    const uint8_t* exps;
    float* dw;  // [S][O][I]
    float* db;  // [S][O] or null
    size_t lddy, rows;
    size_t rows_per;  // rows of one split, a multiple of 32
    int O, I, groups, pitch;
    int tiles_m, tiles_n, splits;
    float zero;
};

template <typename T> struct Terms { static constexpr int N = 1; };
template <> struct Terms<float> { static constexpr int N = 3; };
template <> struct Terms<fp16_t> { static constexpr int N = 2; };

__device__ __forceinline__ u32 top_halves(float hi, float lo) {
    return __builtin_amdgcn_perm(__builtin_bit_cast(u32, hi), __builtin_bit_cast(u32, lo), 0x07060302u);
}
__device__ __forceinline__ float cut_bf16(float v) {
    return __builtin_bit_cast(float, __builtin_bit_cast(u32, v) & 0xffff0000u);
}
// eight fp32 numbers -> N packed bf16x8, whose sum they are (N = 3; 16 bits of them for N = 2)
template <int N>
__device__ __forceinline__ void split_terms(const float* x, u32x4_t* out) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        float a = x[2 * q], b = x[2 * q + 1];
#pragma unroll
        for (int t = 0; t < N; ++t) {
            out[t][q] = top_halves(b, a);
            if (t + 1 < N) {
                a -= cut_bf16(a);
                b -= cut_bf16(b);
            }
        }
    }
}
// (code - zero first: zero * scale overflows where a group's largest magnitude is 2^127 or more)
__device__ __forceinline__ float code_value(u32 word, int j, float s, float zero) {
    return ((float)((word >> (8 * j)) & 0xffu) - zero) * s;
}

// Simplest form: one wave per 32 x 32 tile of dw and split, operands from global memory straight into MFMA registers.
// v_mfma_f32_32x32x16_bf16: lane l holds row / column l % 32 and reduction indices 8 (l / 32) .. + 7.
template <typename T>
__global__ __launch_bounds__(64) void act8_wgrad_simple_kernel(const WgradP p) {
    constexpr int N = Terms<T>::N;
    const int lane = threadIdx.x, c = lane & 31, kc = lane >> 5;
    int id = blockIdx.x;
    const int tn = id % p.tiles_n;
    id /= p.tiles_n;
    const int tm = id % p.tiles_m, split = id / p.tiles_m;
    const int o = tm * 32 + c, i = tn * 32 + c;
    const size_t r_begin = (size_t)split * p.rows_per;
    const size_t r_end = r_begin + p.rows_per < p.rows ? r_begin + p.rows_per : p.rows;
    const T* dy = (const T*)p.dy;
    f32x16 acc;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.f;
    float bias = 0.f;
    for (size_t r0 = r_begin; r0 < r_end; r0 += 16) {
        float a[8], b[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const size_t r = r0 + kc * 8 + j;
            const bool in = r < r_end;
            a[j] = in && o < p.O ? to_f32(dy[r * p.lddy + o]) : 0.f;
            const bool inb = in && i < p.pitch;
            const u32 code = inb ? p.codes[r * p.pitch + i] : 0u;
            const float s = inb ? act8_scale(p.exps[r * p.groups + i / ACT8_GROUP]) : 0.f;
            b[j] = code_value(code, 0, s, inb ? p.zero : 0.f);
            bias += a[j];
        }
        u32x4_t at[N], bt[1];
        split_terms<N>(a, at);
        split_terms<1>(b, bt);
#pragma unroll
        for (int t = 0; t < N; ++t)
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, at[t]), __builtin_bit_cast(bf16x8_t, bt[0]), acc, 0, 0, 0);
    }
    float* dw = p.dw + (size_t)split * p.O * p.I;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const int m = tm * 32 + (e & 3) + 8 * (e >> 2) + 4 * kc;
        if (m < p.O && i < p.I) dw[(size_t)m * p.I + i] = acc[e];
    }
    if (p.db && tn == 0) {
        bias += __shfl_xor(bias, 32, 64);
        if (kc == 0 && o < p.O) p.db[(size_t)split * p.O + o] = bias;
    }
}

// out[i] = sum over splits, in order
__global__ __launch_bounds__(256) void act8_sum_splits_kernel(const float* part, int S, size_t n, size_t stride, float* out) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        float a = 0.f;
        for (int s = 0; s < S; ++s) a += part[(size_t)s * stride + i];
        out[i] = a;
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------------------
struct WgradPlan {
    int tiles_m, tiles_n, splits;
    size_t rows_per;
};

static WgradPlan wgrad_plan(size_t rows, int O, int I) {
    WgradPlan q;
    q.tiles_m = ceil_div(O, 32);
    q.tiles_n = ceil_div(I, 32);
    const size_t tiles = (size_t)q.tiles_m * q.tiles_n;
    size_t s = (4096 + tiles - 1) / tiles;
    const size_t most = (rows + 127) / 128;
    s = s < 1 ? 1 : s > most ? most : s;
    if (s > 64) s = 64;
    q.rows_per = ((rows + s - 1) / s + 31) / 32 * 32;
    q.splits = (int)((rows + q.rows_per - 1) / q.rows_per);
    return q;
}

template <typename T>
static void wgrad_launch(const WgradP& p, hipStream_t s) {
    const unsigned grid = (unsigned)p.tiles_m * p.tiles_n * p.splits;
    hipLaunchKernelGGL((act8_wgrad_simple_kernel<T>), dim3(grid), dim3(64), 0, s, p);
}

static unsigned stream_grid(size_t vecs) {
    const size_t need = (vecs + 255) / 256;
    return (unsigned)(need < (1u << 20) ? need : (1u << 20));
}

}  // namespace dun

using namespace dun;

extern "C" int dun_act8_pack(const void* x, int64_t ldx, uint8_t* codes, uint8_t* exps, int64_t rows, int cols, int dtype,
                             int relu, dun_stream_t stream) {
    DUN_REQUIRE(dtype == DUN_F32 || dtype == DUN_BF16 || dtype == DUN_F16, "dun_act8_pack: dtype %d", dtype);
    DUN_REQUIRE(rows >= 0 && cols > 0 && cols <= INT32_MAX - 65536, "dun_act8_pack: rows %lld, cols %d", (long long)rows, cols);
    if (rows == 0) return DUN_OK;
    DUN_REQUIRE(x && codes && exps, "dun_act8_pack: null tensor");
    DUN_REQUIRE(ldx >= cols, "dun_act8_pack: row stride %lld below %d columns", (long long)ldx, cols);
    DUN_REQUIRE(((uintptr_t)codes & 7) == 0, "dun_act8_pack: codes need 8-byte alignment");
    const int groups = ceil_div(cols, ACT8_GROUP), E = dtype == DUN_F32 ? 4 : 8;
    const u32 vpr = (u32)groups * (ACT8_GROUP / E);
    const size_t vecs = (size_t)rows * vpr;
    const dim3 grid(stream_grid(vecs));
    hipStream_t s = (hipStream_t)stream;
    if (dtype == DUN_F32)
        hipLaunchKernelGGL((act8_pack_kernel<float>), grid, dim3(256), 0, s, (const float*)x, (size_t)ldx, codes, exps, vecs, vpr, cols, relu != 0);
    else if (dtype == DUN_BF16)
        hipLaunchKernelGGL((act8_pack_kernel<bf16_t>), grid, dim3(256), 0, s, (const bf16_t*)x, (size_t)ldx, codes, exps, vecs, vpr, cols, relu != 0);
    else
        hipLaunchKernelGGL((act8_pack_kernel<fp16_t>), grid, dim3(256), 0, s, (const fp16_t*)x, (size_t)ldx, codes, exps, vecs, vpr, cols, relu != 0);
    DUN_LAUNCH_CHECK();
    return DUN_OK;
}

extern "C" int dun_act8_unpack(const uint8_t* codes, const uint8_t* exps, void* out, int64_t ldo, int64_t rows, int cols,
                               int dtype, int relu, dun_stream_t stream) {
    DUN_REQUIRE(dtype == DUN_F32 || dtype == DUN_BF16 || dtype == DUN_F16, "dun_act8_unpack: dtype %d", dtype);
    DUN_REQUIRE(rows >= 0 && cols > 0 && cols <= INT32_MAX - 65536, "dun_act8_unpack: rows %lld, cols %d", (long long)rows, cols);
    if (rows == 0) return DUN_OK;
    DUN_REQUIRE(out && codes && exps, "dun_act8_unpack: null tensor");
    DUN_REQUIRE(ldo >= cols, "dun_act8_unpack: row stride %lld below %d columns", (long long)ldo, cols);
    DUN_REQUIRE(((uintptr_t)codes & 7) == 0, "dun_act8_unpack: codes need 8-byte alignment");
    const int groups = ceil_div(cols, ACT8_GROUP), E = dtype == DUN_F32 ? 4 : 8;
    const u32 vpr = (u32)groups * (ACT8_GROUP / E);
    const size_t vecs = (size_t)rows * vpr;
    const dim3 grid(stream_grid(vecs));
    const float zero = relu ? 0.f : 128.f;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == DUN_F32)
        hipLaunchKernelGGL((act8_unpack_kernel<float>), grid, dim3(256), 0, s, codes, exps, (float*)out, (size_t)ldo, vecs, vpr, cols, zero);
    else if (dtype == DUN_BF16)
        hipLaunchKernelGGL((act8_unpack_kernel<bf16_t>), grid, dim3(256), 0, s, codes, exps, (bf16_t*)out, (size_t)ldo, vecs, vpr, cols, zero);
    else
        hipLaunchKernelGGL((act8_unpack_kernel<fp16_t>), grid, dim3(256), 0, s, codes, exps, (fp16_t*)out, (size_t)ldo, vecs, vpr, cols, zero);
    DUN_LAUNCH_CHECK();
    return DUN_OK;
}

extern "C" size_t dun_act8_weight_grad_workspace_floats(int64_t rows, int outs, int cols, int dtype) {
    (void)dtype;
    if (rows <= 0 || outs <= 0 || cols <= 0) return 0;
    const WgradPlan q = wgrad_plan((size_t)rows, outs, cols);
    return q.splits > 1 ? (size_t)q.splits * ((size_t)outs * cols + outs) : 0;
}

extern "C" int dun_act8_weight_grad(const void* dy, int64_t lddy, const uint8_t* codes, const uint8_t* exps, float* dw, float* db,
                                    float* ws, size_t ws_floats, int64_t rows, int outs, int cols, int dtype, int relu,
                                    dun_stream_t stream) {
    DUN_REQUIRE(dtype == DUN_F32 || dtype == DUN_BF16 || dtype == DUN_F16, "dun_act8_weight_grad: dtype %d", dtype);
    DUN_REQUIRE(rows >= 0 && outs > 0 && cols > 0 && cols <= INT32_MAX - 65536 && outs <= INT32_MAX - 65536,
                "dun_act8_weight_grad: rows %lld, outs %d, cols %d", (long long)rows, outs, cols);
    DUN_REQUIRE(dw, "dun_act8_weight_grad: null dw");
    hipStream_t s = (hipStream_t)stream;
    const size_t n = (size_t)outs * cols;
    if (rows == 0) {  // (no splits to add up: zeros)
        hipLaunchKernelGGL(act8_sum_splits_kernel, dim3(stream_grid(n)), dim3(256), 0, s, (const float*)nullptr, 0, n, n, dw);
        if (db) hipLaunchKernelGGL(act8_sum_splits_kernel, dim3(stream_grid(outs)), dim3(256), 0, s, (const float*)nullptr, 0, (size_t)outs, (size_t)outs, db);
        DUN_LAUNCH_CHECK();
        return DUN_OK;
    }
    DUN_REQUIRE(dy && codes && exps, "dun_act8_weight_grad: null tensor");
    DUN_REQUIRE(lddy >= outs, "dun_act8_weight_grad: row stride %lld below %d columns", (long long)lddy, outs);
    DUN_REQUIRE(((uintptr_t)codes & 7) == 0, "dun_act8_weight_grad: codes need 8-byte alignment");
    const WgradPlan q = wgrad_plan((size_t)rows, outs, cols);
    DUN_REQUIRE((size_t)q.tiles_m * q.tiles_n * q.splits <= 0x7fffffffu, "dun_act8_weight_grad: %d x %d is too large a gradient", outs, cols);
    const size_t need = dun_act8_weight_grad_workspace_floats(rows, outs, cols, dtype);
    DUN_REQUIRE(need == 0 || (ws && ws_floats >= need), "dun_act8_weight_grad: workspace of %zu floats, %zu needed", ws_floats, need);
    WgradP p;
    memset(&p, 0, sizeof(p));
    p.dy = dy;
    p.codes = codes;
    p.exps = exps;
    p.dw = need ? ws : dw;
    p.db = !db ? nullptr : need ? ws + q.splits * n : db;
    p.lddy = (size_t)lddy;
    p.rows = (size_t)rows;
    p.rows_per = q.rows_per;
    p.O = outs;
    p.I = cols;
    p.groups = ceil_div(cols, ACT8_GROUP);
    p.pitch = p.groups * ACT8_GROUP;
    p.tiles_m = q.tiles_m;
    p.tiles_n = q.tiles_n;
    p.splits = q.splits;
    p.zero = relu ? 0.f : 128.f;
    if (dtype == DUN_F32)
        wgrad_launch<float>(p, s);
    else if (dtype == DUN_BF16)
        wgrad_launch<bf16_t>(p, s);
    else
        wgrad_launch<fp16_t>(p, s);
    DUN_LAUNCH_CHECK();
    if (need) {
        hipLaunchKernelGGL(act8_sum_splits_kernel, dim3(stream_grid(n)), dim3(256), 0, s, (const float*)ws, q.splits, n, n, dw);
        if (db)
            hipLaunchKernelGGL(act8_sum_splits_kernel, dim3(stream_grid(outs)), dim3(256), 0, s, (const float*)(ws + q.splits * n), q.splits,
                               (size_t)outs, (size_t)outs, db);
        DUN_LAUNCH_CHECK();
    }
    return DUN_OK;
}
