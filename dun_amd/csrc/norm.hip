// Layer normalisation over rows, forward and backward, with the residual block's extras: rectified input, residual add,
// 8-bit checkpoints of the normalised input and of the output, backward from the checkpoint.
//
//   z = x or max(x, 0) ; mean = sum z / n ; rstd = 1 / sqrt(sum (z - mean)^2 / n + eps)
//   y = [res +] (z - mean) rstd w + b
//   g = dy w ; xhat = (z - mean) rstd ; dx = rstd (g - mean(g) - xhat mean(g xhat)) [where z > 0]
//   dw = sum_rows dy xhat ; db = sum_rows dy ; [ds = sum_rows dx, the bias gradient of the Linear that made x]
//
// Both directions move bytes: forward reads x (and res) once and writes y, backward reads x or its codes and dy and
// writes dx.  So a row stays in the registers of the lanes that loaded it -- a TEAM of 8 to 64 lanes of a wave for rows of
// up to 1024 elements, a workgroup for up to 8192 -- and the statistics are taken there in two passes over registers
// (mean first, then squares of differences: no cancellation for rows far from zero), all in fp32.  Longer rows are walked in
// memory.  The column sums dw, db, ds are kept per lane over all rows that a team visits (a lane always
// sees the same columns), added up over a workgroup in LDS in a fixed order, and over workgroups by a second small
// kernel: no atomics, the same bits every time.
//
// 65536 x 2048 fp32 (a copy of 1 GiB: 5.2 TB/s): forward 231 - 248 us by itself, 205 us in turn with a backward (4.5, 5.2 TB/s), backward 292 -
// 300 us (5.4); the residual block with its checkpoint 300 us and, from the codes, 216 - 220 us (5.8, 5.6 TB/s), with its output packed
// as well 356 us.  bf16, half the bytes: forward 166 - 187 us, backward 176 us, block 256 - 264 us and 176 us: 3.1 and 4.6 TB/s, four elements
// a load whatever the type.  16391 x 1031 bf16, where rows start anywhere: 25 and 28 us (2.7, 3.6 TB/s): too few bytes in flight, a
// row of 2 KB on two waves.  Small ones are launches: 512 x 100 fp32 3.6 + 4.2 + 2.7 us.
#include "rows.h"

namespace dun {

constexpr int LN_LONG_THREADS = 1024;

struct LnFwdP {
    const void* x;
    const void* res;
    const float* w;
    const float* b;
    void* y;
    float* mean;
    float* rstd;
    uint8_t *xc, *xe, *yc, *ye;
    size_t ldx, ldr, ldy;
    size_t rows;
    int cols, groups, relu;
    float eps;
};

struct LnBwdP {
    const void* dy;
    const void* x;
    const uint8_t *xc, *xe;
    const float* w;
    const float* mean;
    const float* rstd;
    void* dx;
    float* part;  // [gridDim.x][K][cols]
    size_t lddy, ldx, lddx;
    size_t rows;
    int cols, groups, relu, K;
};

// Sum over a team; every lane of the team gets it.  Teams wider than a wave go through LDS: two slots used in turn, so one
// barrier per sum is enough (a slot is written again only behind the barrier of the sum in between).
template <int TEAM>
struct TeamSum {
    float* red;
    int turn;
    __device__ __forceinline__ explicit TeamSum(float* lds) : red(lds), turn(0) {}
    __device__ __forceinline__ float operator()(float v) {
        if (TEAM == 64) return wave_allsum(v);
        if (TEAM < 64) {
            v += dpp_move<DPP_QUAD_XOR1>(v);
            v += dpp_move<DPP_QUAD_XOR2>(v);
            v += dpp_move<DPP_ROW_HALF_MIRROR>(v);
            if (TEAM >= 16) v += dpp_move<DPP_ROW_MIRROR>(v);
            if (TEAM >= 32) v += __shfl_xor(v, 16, 64);
            return v;
        }
        constexpr int NW = TEAM / 64;
        v = wave_allsum(v);
        float* slot = red + turn * NW;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
        __syncthreads();
        float s = slot[0];
#pragma unroll
        for (int i = 1; i < NW; ++i) s += slot[i];
        return s;
    }
};

struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };

template <int TEAM> constexpr int ln_block() { return TEAM > 64 ? TEAM : 256; }

// Chunks of a lane that lie inside the row whatever its length, by the choice of the team (ln_team): the last chunk may end early, of
// 256 x 4 the last two
template <int TEAM, int CH> constexpr int ln_whole() { return TEAM == 256 && CH == 4 ? 2 : CH - 1; }

template <typename T, int TEAM, int CH>
__device__ __forceinline__ void ln_load_row(const T* row, int t, int cols, RawVec<T>* v) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int i0 = (c * TEAM + t) * E;
        if (c < ln_whole<TEAM, CH>())
            v[c].load(row, i0);
        else
            v[c].load_end(row, i0, cols);
    }
}

template <typename T, int TEAM, int CH>
__global__ __launch_bounds__(ln_block<TEAM>()) void ln_forward_kernel(const LnFwdP p) {
    constexpr int TPB = ln_block<TEAM>() / TEAM;
    __shared__ float red[TEAM > 64 ? 2 * (TEAM / 64) : 1];
    TeamSum<TEAM> sum(red);
    const int t = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    const float n = (float)p.cols, floor_ = p.relu ? 0.f : -INFINITY;
    for (size_t row = (size_t)blockIdx.x * TPB + team; row < p.rows; row += (size_t)gridDim.x * TPB) {
        RawVec<T> xv[CH], rv[CH];
        ln_load_row<T, TEAM, CH>((const T*)p.x + row * p.ldx, t, p.cols, xv);
        if (p.res) {
            ln_load_row<T, TEAM, CH>((const T*)p.res + row * p.ldr, t, p.cols, rv);
        } else {
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int e = 0; e < RawVec<T>::W; ++e) rv[c].w[e] = 0;
        }
        auto z = [&](int c, int e) { return max_nan(xv[c][e], floor_); };
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int e = 0; e < E; ++e) s += z(c, e);
        const float mean = sum(s) / n;
        s = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) xv[c].forget();
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int i0 = (c * TEAM + t) * E;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float d = c < ln_whole<TEAM, CH>() || i0 + e < p.cols ? z(c, e) - mean : 0.f;
                s += d * d;
            }
        }
        const float rstd = 1.f / sqrtf(sum(s) / n + p.eps);
        if (p.mean && t == 0) {
            p.mean[row] = mean;
            p.rstd[row] = rstd;
        }
        T* y = (T*)p.y + row * p.ldy;
#pragma unroll
        for (int c = 0; c < CH; ++c) xv[c].forget();
        // (the choices are the same for every row; made once here, not once per chunk)
        auto finish = [&](auto affine, auto keep_x, auto keep_y) {
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int i0 = (c * TEAM + t) * E;
                constexpr bool any = !decltype(affine)::value;
                RawVec<float> w, b;
                if (!any || p.w) {
                    if (c < ln_whole<TEAM, CH>()) w.load(p.w, i0); else w.load_end(p.w, i0, p.cols);
                }
                if (!any || p.b) {
                    if (c < ln_whole<TEAM, CH>()) b.load(p.b, i0); else b.load_end(p.b, i0, p.cols);
                }
                if (keep_x.value && (!any || p.xc)) {
                    float v[E];
                    u32 byte;
#pragma unroll
                    for (int e = 0; e < E; ++e) v[e] = z(c, e);
                    const u32 word = act8_pack(v, p.relu, &byte);
                    act8_store(p.xc, p.xe, row, p.groups, i0, word, byte);
                }
                float o[E];
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    float h = (z(c, e) - mean) * rstd;
                    if (!any || p.w) h *= w[e];
                    if (!any || p.b) h += b[e];
                    o[e] = h + rv[c][e];
                }
                store_part(y, i0, p.cols, o);
                if (keep_y.value && (!any || p.yc)) {
                    // the checkpoint holds what the next layer reads: the output as it is stored
                    u32 byte;
#pragma unroll
                    for (int e = 0; e < E; ++e) o[e] = i0 + e < p.cols ? to_f32(from_f32<T>(o[e])) : 0.f;
                    const u32 word = act8_pack(o, false, &byte);
                    act8_store(p.yc, p.ye, row, p.groups, i0, word, byte);
                }
            }
        };
        if (p.w && p.b && !p.xc && !p.yc)
            finish(Yes(), No(), No());
        else if (p.w && p.b && p.xc && !p.yc)
            finish(Yes(), Yes(), No());
        else
            finish(No(), Yes(), Yes());
    }
}

// z of a lane's chunk in backward: x (rectified), or the checkpoint's word and its group's byte
template <typename T>
__device__ __forceinline__ void ln_fetch_codes(const LnBwdP& p, size_t row, int i0, RawVec<T>& raw) {
    const int last = p.groups * ACT8_GROUP - E;
    const int i = i0 < last ? i0 : last;
    const u32 word = *reinterpret_cast<const u32*>(p.xc + row * p.groups * ACT8_GROUP + i);
    const u32 byte = p.xe[row * p.groups + i / ACT8_GROUP];
    // (past the row's groups: a code that stands for a number)
    raw.w[0] = i0 <= last ? word : 0u;
    raw.w[1] = i0 <= last ? byte : 0u;
}
template <typename T>
__device__ __forceinline__ void ln_bwd_z(const LnBwdP& p, size_t row, int i0, float* v) {
    RawVec<T> raw;
    if (p.xc) {
        ln_fetch_codes(p, row, i0, raw);
        act8_values(raw.w[0], raw.w[1], p.relu ? 0.f : 128.f, v);
    } else {
        const float floor_ = p.relu ? 0.f : -INFINITY;
        raw.load_end((const T*)p.x + row * p.ldx, i0, p.cols);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = max_nan(raw[e], floor_);
    }
}

// a * b rounded by itself: as fma(a, b, -mean) it would leave its rounding error where g - mean(g) is 0, in rows of one element
__device__ __forceinline__ float product(float a, float b) {
#pragma clang fp contract(off)
    return a * b;
}

// K: column sums wanted (0, 2 or 3).  MASK: rows may be rectified (p.relu), so z itself is kept for ReLU's mask and xhat is worked out a
// second time, two operations per element against six for a mask of bits.
template <typename T, int TEAM, int CH, int K, bool MASK>
__global__ __launch_bounds__(ln_block<TEAM>()) void ln_backward_kernel(const LnBwdP p) {
    constexpr int BLOCK = ln_block<TEAM>(), TPB = BLOCK / TEAM;
    constexpr int SPAN = TEAM * E * CH;  // columns that a team covers
    __shared__ float red[TEAM > 64 ? 2 * (TEAM / 64) : 1];
    __shared__ float acc_lds[TEAM > 64 ? 1 : (K > 0 ? K : 1) * SPAN];
    TeamSum<TEAM> sum(red);
    const int t = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    const float n = (float)p.cols, floor_ = MASK && p.relu ? 0.f : -INFINITY;
    const float dead = MASK && p.relu ? 0.f : NAN;  // z <= dead has no gradient; without ReLU none, -inf not either
    float acc[K > 0 ? K : 1][CH][E];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int e = 0; e < E; ++e) acc[k][c][e] = 0.f;
    // A lane sees the same columns in every row.  Weights that stay in registers spare each row a wait for the cache:
    // with them in 16-bit rows 16391 x 1031 takes 29 us and not 38, in fp32 rows with 8-bit codes 65536 x 2048 takes
    // 218 us and not 237.  Plain fp32 rows are bound by memory and want the waves instead: 310 us at 65536 x 2048 with
    // the weights read row by row, 338 with them kept.  The MASK forms serve codes and x alike and keep them for both: fp32 rows
    // read from x take 320 - 324 us there (rectified, with the sums of dx, or dx alone) where the plain form takes 292.
    constexpr bool KEEP_W = MASK || sizeof(T) < 4;
    RawVec<float> w[CH];
    auto weights = [&] {
        if (p.w) {
            ln_load_row<float, TEAM, CH>(p.w, t, p.cols, w);
        } else {
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int e = 0; e < E; ++e) w[c].w[e] = 0x3f800000u;  // 1.0
        }
    };
    if (KEEP_W) weights();
    for (size_t row = (size_t)blockIdx.x * TPB + team; row < p.rows; row += (size_t)gridDim.x * TPB) {
        RawVec<T> dv[CH], zv[CH];
        float h[CH][E], g[CH][E];
        ln_load_row<T, TEAM, CH>((const T*)p.dy + row * p.lddy, t, p.cols, dv);
        if (p.xc) {
#pragma unroll
            for (int c = 0; c < CH; ++c) ln_fetch_codes(p, row, (c * TEAM + t) * E, zv[c]);
        } else {
            ln_load_row<T, TEAM, CH>((const T*)p.x + row * p.ldx, t, p.cols, zv);
        }
        const float mean = p.mean[row], rstd = p.rstd[row];
        if (p.xc) {
#pragma unroll
            for (int c = 0; c < CH; ++c) act8_values(zv[c].w[0], zv[c].w[1], p.relu ? 0.f : 128.f, h[c]);
        } else {
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int e = 0; e < E; ++e) h[c][e] = MASK ? max_nan(zv[c][e], floor_) : zv[c][e];
        }
        float s1 = 0.f, s2 = 0.f;
        if (!KEEP_W) weights();
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                // (columns past the row's end hold dy = 0: they add nothing to any sum)
                const float xhat = (h[c][e] - mean) * rstd;
                if (!MASK) h[c][e] = xhat;
                const float d = dv[c][e];
                if (K > 0) {
                    acc[0][c][e] += d * xhat;
                    acc[1][c][e] += d;
                }
                g[c][e] = product(d, w[c][e]);
                s1 += g[c][e];
                s2 += g[c][e] * xhat;
            }
        s1 = sum(s1) / n;
        s2 = sum(s2) / n;
        T* dx = (T*)p.dx + row * p.lddx;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int i0 = (c * TEAM + t) * E;
            float o[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float xhat = MASK ? (h[c][e] - mean) * rstd : h[c][e];
                o[e] = rstd * (g[c][e] - s1 - xhat * s2);
                if (MASK) o[e] = h[c][e] <= dead ? 0.f : o[e];
                if (K > 2) acc[K > 2 ? 2 : 0][c][e] += c < ln_whole<TEAM, CH>() || i0 + e < p.cols ? o[e] : 0.f;
            }
            store_part(dx, i0, p.cols, o);
        }
    }
    if (K == 0) return;
    float* part = p.part + (size_t)blockIdx.x * K * p.cols;
    if (TEAM > 64) {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int i = (c * TEAM + t) * E + e;
                    if (i < p.cols) part[(size_t)k * p.cols + i] = acc[k][c][e];
                }
        return;
    }
    // teams of a wave first (they hold the same columns), then the waves of the workgroup in order
#pragma unroll
    for (int off = TEAM; off < 64; off <<= 1)
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int e = 0; e < E; ++e) acc[k][c][e] += __shfl_xor(acc[k][c][e], off, 64);
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    for (int w = 0; w < BLOCK / 64; ++w) {
        if (wid == w && lane < TEAM) {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int c = 0; c < CH; ++c)
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        float* a = acc_lds + k * SPAN + (c * TEAM + t) * E + e;
                        *a = w ? *a + acc[k][c][e] : acc[k][c][e];
                    }
        }
        __syncthreads();
    }
    for (int k = 0; k < K; ++k)
        for (int i = threadIdx.x; i < p.cols; i += BLOCK) part[(size_t)k * p.cols + i] = acc_lds[k * SPAN + i];
}

// ---- rows longer than 1024 lanes hold: the same sums, the row read again instead of kept ------------------------------------
template <typename T>
__global__ __launch_bounds__(LN_LONG_THREADS) void ln_forward_long_kernel(const LnFwdP p) {
    constexpr int STEP = LN_LONG_THREADS * E;
    __shared__ float red[2 * (LN_LONG_THREADS / 64)];
    TeamSum<LN_LONG_THREADS> sum(red);
    const float n = (float)p.cols;
    const int t0 = threadIdx.x * E;
    for (size_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = (const T*)p.x + row * p.ldx;
        const T* res = p.res ? (const T*)p.res + row * p.ldr : nullptr;
        T* y = (T*)p.y + row * p.ldy;
        float v[E], s = 0.f;
        for (int i0 = t0; i0 < p.cols; i0 += STEP) {
            load_part(x, i0, p.cols, v);
#pragma unroll
            for (int e = 0; e < E; ++e) s += p.relu ? rectify(v[e]) : v[e];
        }
        const float mean = sum(s) / n;
        s = 0.f;
        for (int i0 = t0; i0 < p.cols; i0 += STEP) {
            load_part(x, i0, p.cols, v);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float d = i0 + e < p.cols ? (p.relu ? rectify(v[e]) : v[e]) - mean : 0.f;
                s += d * d;
            }
        }
        const float rstd = 1.f / sqrtf(sum(s) / n + p.eps);
        if (p.mean && threadIdx.x == 0) {
            p.mean[row] = mean;
            p.rstd[row] = rstd;
        }
        // (whole groups enter: the lanes of a group leave the loop together, and the codes past the row's end are written)
        for (int i0 = t0; i0 < p.groups * ACT8_GROUP; i0 += STEP) {
            float r[E], w[E], b[E], o[E];
            load_part(x, i0, p.cols, v);
            if (res) load_part(res, i0, p.cols, r);
            if (p.w) load_part(p.w, i0, p.cols, w);
            if (p.b) load_part(p.b, i0, p.cols, b);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (p.relu) v[e] = rectify(v[e]);
                float h = (v[e] - mean) * rstd;
                if (p.w) h *= w[e];
                if (p.b) h += b[e];
                o[e] = res ? h + r[e] : h;
            }
            if (p.xc) {
                u32 byte;
                const u32 word = act8_pack(v, p.relu, &byte);
                act8_store(p.xc, p.xe, row, p.groups, i0, word, byte);
            }
            store_part(y, i0, p.cols, o);
            if (p.yc) {
                u32 byte;
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] = i0 + e < p.cols ? to_f32(from_f32<T>(o[e])) : 0.f;
                const u32 word = act8_pack(o, false, &byte);
                act8_store(p.yc, p.ye, row, p.groups, i0, word, byte);
            }
        }
    }
}

template <typename T>
__global__ __launch_bounds__(LN_LONG_THREADS) void ln_backward_long_kernel(const LnBwdP p) {
    constexpr int STEP = LN_LONG_THREADS * E;
    __shared__ float red[2 * (LN_LONG_THREADS / 64)];
    TeamSum<LN_LONG_THREADS> sum(red);
    const float n = (float)p.cols;
    const int t0 = threadIdx.x * E;
    float* part = p.part ? p.part + (size_t)blockIdx.x * p.K * p.cols : nullptr;
    bool first = true;
    for (size_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* dy = (const T*)p.dy + row * p.lddy;
        T* dx = (T*)p.dx + row * p.lddx;
        const float mean = p.mean[row], rstd = p.rstd[row];
        float s1 = 0.f, s2 = 0.f, h[E], g[E], w[E];
        for (int i0 = t0; i0 < p.cols; i0 += STEP) {
            load_part(dy, i0, p.cols, g);
            ln_bwd_z<T>(p, row, i0, h);
            if (p.w) load_part(p.w, i0, p.cols, w);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float q = p.w ? g[e] * w[e] : g[e];
                s1 += q;
                s2 += q * ((h[e] - mean) * rstd);
            }
        }
        s1 = sum(s1) / n;
        s2 = sum(s2) / n;
        for (int i0 = t0; i0 < p.cols; i0 += STEP) {
            float o[E];
            load_part(dy, i0, p.cols, g);
            ln_bwd_z<T>(p, row, i0, h);
            if (p.w) load_part(p.w, i0, p.cols, w);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const bool dead = p.relu && h[e] <= 0.f;
                const float xh = (h[e] - mean) * rstd, q = p.w ? g[e] * w[e] : g[e];
                o[e] = dead ? 0.f : rstd * (q - s1 - xh * s2);
                if (part && i0 + e < p.cols) {  // this workgroup's own partial row: columns belong to threads
                    float* a = part + i0 + e;
                    a[0] = (first ? 0.f : a[0]) + g[e] * xh;
                    a[p.cols] = (first ? 0.f : a[p.cols]) + g[e];
                    if (p.K > 2) a[2 * (size_t)p.cols] = (first ? 0.f : a[2 * (size_t)p.cols]) + o[e];
                }
            }
            store_part(dx, i0, p.cols, o);
        }
        first = false;
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------------------
// Teams and vectors of four elements per lane, by the elements that a team holds: the fewest lanes up to a wave, then more vectors per
// lane, then more waves.  What decides is the bytes in flight: few registers per row for many rows at a time, but no idle lanes.
// 65536 x 2048 fp32, forward / backward in turn: 64 x 8 237 / 330 us, 256 x 2 200 / 297 us (a plain copy of as many bytes: 208 / 312);
// 16391 x 1031 bf16: 256 x 2, half of its lanes idle, 34 / 60 us, 128 x 3 26 / 38 us (since: 25 / 28).  512 x 8 for rows of up to 16384 elements spills: 2000 x
// 16384 fp32 96 / 163 us, walked in memory 75 / 235 us (since: 71 / 223).  Idle lanes show between the teams: 16384 rows of 3000, 4100 and 6000
// fp32 elements take 101 / 137, 228 / 200 and 239 / 245 us (copies of as many bytes: 76 / 114, 104 / 156, 152 / 228).
#define DUN_LN_TEAMS(X) X(8, 1) X(16, 1) X(32, 1) X(64, 1) X(64, 2) X(64, 3) X(64, 4) X(128, 3) X(256, 2) X(256, 4) X(1024, 2)

static int ln_team(int cols, int* ch) {
    const int vecs = ceil_div(cols, E);
#define DUN_LN_PICK(TEAM, CH) \
    if (vecs <= TEAM * CH) {  \
        *ch = CH;             \
        return TEAM;          \
    }
    DUN_LN_TEAMS(DUN_LN_PICK)
#undef DUN_LN_PICK
    *ch = 0;
    return 0;  // too long for registers
}

// Workgroups of a backward pass, each with a partial row of sums: as many as 256 CUs hold at once (by the registers of the team's rows; a second
// round costs as much as it brings: 65536 x 2048 fp32 from the checkpoint: 512 272 us, 1024 230 us (218 since), 1536 256 us), and two rows a team
// before more workgroups (4099 x 517: 1025 15.7 us, 513 11.7 us)
static size_t ln_backward_blocks(size_t rows, int cols) {
    int ch;
    const int team = ln_team(cols, &ch);
    if (team == 0) return rows < 256 ? rows : 256;
    const size_t tpb = team <= 64 ? 256 / team : 1;
    const size_t need = (rows + tpb - 1) / tpb;
    const size_t most = team == 1024 ? 256 : team == 256 ? (ch == 2 ? 1024 : 512) : team == 128 ? 1536 : ch <= 2 ? 1024 : ch == 3 ? 768 : 512;
    if (need <= 4) return 1;  // one workgroup's sums need no second launch
    const size_t half = need <= 512 ? need : need <= 1024 ? 512 : (need + 1) / 2;
    return half < most ? half : most;
}

template <typename T>
static void ln_launch_forward(const LnFwdP& p, hipStream_t s) {
    int ch;
    const int team = ln_team(p.cols, &ch);
    const size_t tpb = team && team <= 64 ? 256 / team : 1;
    const size_t need = (p.rows + tpb - 1) / tpb;
    const dim3 grid((unsigned)(need < (1u << 20) ? need : (1u << 20)));
#define DUN_LN_FWD(TEAM, CH)                                                                               \
    if (team == TEAM && ch == CH) {                                                                        \
        hipLaunchKernelGGL((ln_forward_kernel<T, TEAM, CH>), grid, dim3(ln_block<TEAM>()), 0, s, p);       \
        return;                                                                                            \
    }
    DUN_LN_TEAMS(DUN_LN_FWD)
    hipLaunchKernelGGL((ln_forward_long_kernel<T>), dim3((unsigned)(p.rows < 65536 ? p.rows : 65536)), dim3(LN_LONG_THREADS), 0, s, p);
#undef DUN_LN_FWD
}

template <typename T, int K, bool MASK>
static void ln_launch_backward_k(const LnBwdP& p, unsigned blocks, hipStream_t s) {
    int ch;
    const int team = ln_team(p.cols, &ch);
#define DUN_LN_BWD(TEAM, CH)                                                                                     \
    if (team == TEAM && ch == CH) {                                                                              \
        hipLaunchKernelGGL((ln_backward_kernel<T, TEAM, CH, K, MASK>), dim3(blocks), dim3(ln_block<TEAM>()), 0, s, p); \
        return;                                                                                                  \
    }
    DUN_LN_TEAMS(DUN_LN_BWD)
#undef DUN_LN_BWD
    hipLaunchKernelGGL((ln_backward_long_kernel<T>), dim3(blocks), dim3(LN_LONG_THREADS), 0, s, p);
}

template <typename T>
static void ln_launch_backward(const LnBwdP& p, unsigned blocks, hipStream_t s) {
    if (p.K == 0)
        ln_launch_backward_k<T, 0, true>(p, blocks, s);
    else if (p.K == 3)
        ln_launch_backward_k<T, 3, true>(p, blocks, s);
    else if (p.relu)
        ln_launch_backward_k<T, 2, true>(p, blocks, s);
    else
        ln_launch_backward_k<T, 2, false>(p, blocks, s);
}

}  // namespace dun

using namespace dun;

extern "C" size_t dun_layer_norm_backward_workspace_floats(int64_t rows, int cols, int dtype, int sums) {
    if (rows <= 0 || cols <= 0 || sums < 2) return 0;
    const size_t blocks = ln_backward_blocks((size_t)rows, cols);
    return blocks > 1 ? blocks * (size_t)sums * cols : 0;
}

extern "C" int dun_layer_norm_forward(const void* x, int64_t ldx, const void* res, int64_t ldr, const float* w, const float* b,
                                      void* y, int64_t ldy, float* stats, uint8_t* x_codes, uint8_t* x_exps, uint8_t* y_codes,
                                      uint8_t* y_exps, int64_t rows, int cols, int dtype, float eps, int relu,
                                      dun_stream_t stream) {
    DUN_REQUIRE(dtype == DUN_F32 || dtype == DUN_BF16 || dtype == DUN_F16, "dun_layer_norm_forward: dtype %d", dtype);
    DUN_REQUIRE(rows >= 0 && cols > 0, "dun_layer_norm_forward: rows %lld, cols %d", (long long)rows, cols);
    if (rows == 0) return DUN_OK;
    DUN_REQUIRE(x && y, "dun_layer_norm_forward: null tensor");
    DUN_REQUIRE(cols <= INT32_MAX - 65536, "dun_layer_norm_forward: %d columns", cols);
    DUN_REQUIRE(ldx >= cols && ldy >= cols && (!res || ldr >= cols), "dun_layer_norm_forward: a row stride is below %d columns", cols);
    DUN_REQUIRE(!x_codes == !x_exps && !y_codes == !y_exps, "dun_layer_norm_forward: codes and exponents come together");
    DUN_REQUIRE(((uintptr_t)x_codes & 7) == 0 && ((uintptr_t)y_codes & 7) == 0, "dun_layer_norm_forward: codes need 8-byte alignment");
    LnFwdP p;
    memset(&p, 0, sizeof(p));
    p.x = x;
    p.res = res;
    p.w = w;
    p.b = b;
    p.y = y;
    p.mean = stats;
    p.rstd = stats ? stats + rows : nullptr;
    p.xc = x_codes;
    p.xe = x_exps;
    p.yc = y_codes;
    p.ye = y_exps;
    p.ldx = (size_t)ldx;
    p.ldr = (size_t)ldr;
    p.ldy = (size_t)ldy;
    p.rows = (size_t)rows;
    p.cols = cols;
    p.groups = ceil_div(cols, ACT8_GROUP);
    p.relu = relu != 0;
    p.eps = eps;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == DUN_F32)
        ln_launch_forward<float>(p, s);
    else if (dtype == DUN_BF16)
        ln_launch_forward<bf16_t>(p, s);
    else
        ln_launch_forward<fp16_t>(p, s);
    DUN_LAUNCH_CHECK();
    return DUN_OK;
}

extern "C" int dun_layer_norm_backward(const void* dy, int64_t lddy, const void* x, int64_t ldx, const uint8_t* x_codes,
                                       const uint8_t* x_exps, const float* w, const float* stats, void* dx, int64_t lddx,
                                       float* sums_out, int sums, float* ws, size_t ws_floats, int64_t rows, int cols,
                                       int dtype, int relu, dun_stream_t stream) {
    DUN_REQUIRE(dtype == DUN_F32 || dtype == DUN_BF16 || dtype == DUN_F16, "dun_layer_norm_backward: dtype %d", dtype);
    DUN_REQUIRE(rows >= 0 && cols > 0, "dun_layer_norm_backward: rows %lld, cols %d", (long long)rows, cols);
    DUN_REQUIRE(cols <= INT32_MAX - 65536, "dun_layer_norm_backward: %d columns", cols);
    DUN_REQUIRE(sums == 0 || sums == 2 || sums == 3, "dun_layer_norm_backward: sums is 0, 2 or 3, got %d", sums);
    DUN_REQUIRE(sums == 0 || sums_out, "dun_layer_norm_backward: null sums_out");
    hipStream_t s = (hipStream_t)stream;
    if (rows == 0) {
        if (sums) {
            launch_zero_floats(sums_out, (size_t)sums * cols, s);
            DUN_LAUNCH_CHECK();
        }
        return DUN_OK;
    }
    DUN_REQUIRE(dy && dx && stats, "dun_layer_norm_backward: null tensor");
    DUN_REQUIRE(!x != !x_codes && !x_codes == !x_exps, "dun_layer_norm_backward: either x or its codes and exponents");
    DUN_REQUIRE(((uintptr_t)x_codes & 7) == 0, "dun_layer_norm_backward: codes need 8-byte alignment");
    DUN_REQUIRE(lddy >= cols && lddx >= cols && (!x || ldx >= cols), "dun_layer_norm_backward: a row stride is below %d columns", cols);
    const size_t blocks = ln_backward_blocks((size_t)rows, cols);
    const size_t need = dun_layer_norm_backward_workspace_floats(rows, cols, dtype, sums);
    DUN_REQUIRE(need == 0 || (ws && ws_floats >= need), "dun_layer_norm_backward: workspace of %zu floats, %zu needed", ws_floats, need);
    LnBwdP p;
    memset(&p, 0, sizeof(p));
    p.dy = dy;
    p.x = x;
    p.xc = x_codes;
    p.xe = x_exps;
    p.w = w;
    p.mean = stats;
    p.rstd = stats + rows;
    p.dx = dx;
    p.part = sums == 0 ? nullptr : (need ? ws : sums_out);
    p.lddy = (size_t)lddy;
    p.ldx = (size_t)ldx;
    p.lddx = (size_t)lddx;
    p.rows = (size_t)rows;
    p.cols = cols;
    p.groups = ceil_div(cols, ACT8_GROUP);
    p.relu = relu != 0;
    p.K = sums;
    if (dtype == DUN_F32)
        ln_launch_backward<float>(p, (unsigned)blocks, s);
    else if (dtype == DUN_BF16)
        ln_launch_backward<bf16_t>(p, (unsigned)blocks, s);
    else
        ln_launch_backward<fp16_t>(p, (unsigned)blocks, s);
    DUN_LAUNCH_CHECK();
    if (need) {
        const size_t n = (size_t)sums * cols;
        launch_sum_rows(ws, blocks, n, sums_out, n, nullptr, s);
        DUN_LAUNCH_CHECK();
    }
    return DUN_OK;
}
