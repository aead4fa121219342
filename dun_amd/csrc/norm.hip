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
// up to 2048 elements, a workgroup for longer ones -- and the statistics are taken there in two passes over registers
// (mean first, then squares of differences: no cancellation for rows far from zero), all in fp32.  Rows longer than what 1024
// lanes hold are walked in memory.  The column sums dw, db, ds are kept per lane over all rows that a team visits (a lane always
// sees the same columns), added up over a workgroup in LDS in a fixed order, and over workgroups by a second small
// kernel: no atomics, the same bits every time.
#include "rows.h"

namespace dun {

constexpr int LN_MAX_PER_LANE = 32;   // elements of a row that a lane holds
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

template <int TEAM> constexpr int ln_block() { return TEAM > 256 ? TEAM : 256; }

template <typename T, int TEAM, int CH>
__global__ __launch_bounds__(ln_block<TEAM>()) void ln_forward_kernel(const LnFwdP p) {
    constexpr int E = Row<T>::E, TPB = ln_block<TEAM>() / TEAM;
    __shared__ float red[TEAM > 64 ? 2 * (TEAM / 64) : 1];
    TeamSum<TEAM> sum(red);
    const int t = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    const float n = (float)p.cols;
    for (size_t row = (size_t)blockIdx.x * TPB + team; row < p.rows; row += (size_t)gridDim.x * TPB) {
        const T* x = (const T*)p.x + row * p.ldx;
        float v[CH][E], r[CH][E];
#pragma unroll
        for (int c = 0; c < CH; ++c) load_part(x, (c * TEAM + t) * E, p.cols, v[c]);
        if (p.res) {
            const T* res = (const T*)p.res + row * p.ldr;
#pragma unroll
            for (int c = 0; c < CH; ++c) load_part(res, (c * TEAM + t) * E, p.cols, r[c]);
        } else {
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int e = 0; e < E; ++e) r[c][e] = 0.f;
        }
        if (p.relu) {
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int e = 0; e < E; ++e) v[c][e] = rectify(v[c][e]);
        }
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int e = 0; e < E; ++e) s += v[c][e];
        const float mean = sum(s) / n;
        s = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int i0 = (c * TEAM + t) * E;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float d = i0 + e < p.cols ? v[c][e] - mean : 0.f;
                s += d * d;
            }
        }
        const float rstd = 1.f / sqrtf(sum(s) / n + p.eps);
        if (p.mean && t == 0) {
            p.mean[row] = mean;
            p.rstd[row] = rstd;
        }
        if (p.xc) {
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int i0 = (c * TEAM + t) * E;
                u32 w[E / 4];
                const u32 byte = act8_pack<E>(v[c], p.relu, w);
                if (i0 < p.groups * ACT8_GROUP) {
                    act8_store_words<E>(p.xc + (row * p.groups) * ACT8_GROUP + i0, w);
                    if (i0 % ACT8_GROUP == 0) p.xe[row * p.groups + i0 / ACT8_GROUP] = (uint8_t)byte;
                }
            }
        }
        T* y = (T*)p.y + row * p.ldy;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int i0 = (c * TEAM + t) * E;
            float o[E], w[E], b[E];
            if (p.w) load_f32<E>(p.w, i0, p.cols, w);
            if (p.b) load_f32<E>(p.b, i0, p.cols, b);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                float h = (v[c][e] - mean) * rstd;
                if (p.w) h *= w[e];
                if (p.b) h += b[e];
                o[e] = h + r[c][e];
            }
            store_part(y, i0, p.cols, o);
            if (p.yc) {
                // the checkpoint holds what the next layer reads: the output as it is stored
                u32 q[E / 4];
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] = i0 + e < p.cols ? to_f32(from_f32<T>(o[e])) : 0.f;
                const u32 byte = act8_pack<E>(o, false, q);
                if (i0 < p.groups * ACT8_GROUP) {
                    act8_store_words<E>(p.yc + (row * p.groups) * ACT8_GROUP + i0, q);
                    if (i0 % ACT8_GROUP == 0) p.ye[row * p.groups + i0 / ACT8_GROUP] = (uint8_t)byte;
                }
            }
        }
    }
}

// z of a lane's chunk in backward: the checkpoint's values, or x itself (rectified)
template <typename T>
__device__ __forceinline__ void ln_bwd_z(const LnBwdP& p, size_t row, int i0, float* v) {
    constexpr int E = Row<T>::E;
    if (p.xc) {
        if (i0 < p.groups * ACT8_GROUP) {
            u32 w[E / 4];
            act8_load_words<E>(p.xc + (row * p.groups) * ACT8_GROUP + i0, w);
            act8_values<E>(w, p.xe[row * p.groups + i0 / ACT8_GROUP], p.relu ? 0.f : 128.f, v);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = 0.f;
        }
    } else {
        load_part((const T*)p.x + row * p.ldx, i0, p.cols, v);
        if (p.relu) {
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = rectify(v[e]);
        }
    }
}

template <typename T, int TEAM, int CH, int K>
__global__ __launch_bounds__(ln_block<TEAM>()) void ln_backward_kernel(const LnBwdP p) {
    constexpr int E = Row<T>::E, BLOCK = ln_block<TEAM>(), TPB = BLOCK / TEAM;
    constexpr int SPAN = TEAM * E * CH;  // columns that a team covers
    __shared__ float red[TEAM > 64 ? 2 * (TEAM / 64) : 1];
    __shared__ float acc_lds[TEAM > 64 ? 1 : (K > 0 ? K : 1) * SPAN];
    TeamSum<TEAM> sum(red);
    const int t = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    const float n = (float)p.cols;
    float acc[K > 0 ? K : 1][CH][E];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int e = 0; e < E; ++e) acc[k][c][e] = 0.f;
    for (size_t row = (size_t)blockIdx.x * TPB + team; row < p.rows; row += (size_t)gridDim.x * TPB) {
        const T* dy = (const T*)p.dy + row * p.lddy;
        float h[CH][E], g[CH][E];
#pragma unroll
        for (int c = 0; c < CH; ++c) load_part(dy, (c * TEAM + t) * E, p.cols, g[c]);
#pragma unroll
        for (int c = 0; c < CH; ++c) ln_bwd_z<T>(p, row, (c * TEAM + t) * E, h[c]);
        const float mean = p.mean[row], rstd = p.rstd[row];
        u32 live = ~0u;  // bit c * E + e: z > 0, or NaN (CH * E <= 32)
        if (p.relu) {
            live = 0;
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int e = 0; e < E; ++e) live |= (u32)!(h[c][e] <= 0.f) << (c * E + e);
        }
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int i0 = (c * TEAM + t) * E;
            float w[E];
            if (p.w) load_f32<E>(p.w, i0, p.cols, w);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                // (columns past the row's end hold dy = 0: they add nothing to any sum, whatever h is there, as long as it is finite)
                h[c][e] = (h[c][e] - mean) * rstd;
                if (K > 0) {
                    acc[0][c][e] += g[c][e] * h[c][e];
                    acc[1][c][e] += g[c][e];
                }
                if (p.w) g[c][e] *= w[e];
                s1 += g[c][e];
                s2 += g[c][e] * h[c][e];
            }
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
                o[e] = rstd * (g[c][e] - s1 - h[c][e] * s2);
                if (!((live >> (c * E + e)) & 1u)) o[e] = 0.f;
                if (K > 2) acc[K > 2 ? 2 : 0][c][e] += i0 + e < p.cols ? o[e] : 0.f;
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
    constexpr int E = Row<T>::E, STEP = LN_LONG_THREADS * E;
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
            if (p.w) load_f32<E>(p.w, i0, p.cols, w);
            if (p.b) load_f32<E>(p.b, i0, p.cols, b);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (p.relu) v[e] = rectify(v[e]);
                float h = (v[e] - mean) * rstd;
                if (p.w) h *= w[e];
                if (p.b) h += b[e];
                o[e] = res ? h + r[e] : h;
            }
            if (p.xc) {
                u32 q[E / 4];
                const u32 byte = act8_pack<E>(v, p.relu, q);
                act8_store_words<E>(p.xc + (row * p.groups) * ACT8_GROUP + i0, q);
                if (i0 % ACT8_GROUP == 0) p.xe[row * p.groups + i0 / ACT8_GROUP] = (uint8_t)byte;
            }
            store_part(y, i0, p.cols, o);
            if (p.yc) {
                u32 q[E / 4];
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] = i0 + e < p.cols ? to_f32(from_f32<T>(o[e])) : 0.f;
                const u32 byte = act8_pack<E>(o, false, q);
                act8_store_words<E>(p.yc + (row * p.groups) * ACT8_GROUP + i0, q);
                if (i0 % ACT8_GROUP == 0) p.ye[row * p.groups + i0 / ACT8_GROUP] = (uint8_t)byte;
            }
        }
    }
}

template <typename T>
__global__ __launch_bounds__(LN_LONG_THREADS) void ln_backward_long_kernel(const LnBwdP p) {
    constexpr int E = Row<T>::E, STEP = LN_LONG_THREADS * E;
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
            if (p.w) load_f32<E>(p.w, i0, p.cols, w);
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
            if (p.w) load_f32<E>(p.w, i0, p.cols, w);
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

// out[i] = sum over the workgroups' partial rows: 32 columns x 8 slices of the rows per workgroup, slices added in order
__global__ __launch_bounds__(256) void ln_reduce_kernel(const float* part, size_t P, size_t n, float* out) {
    __shared__ float lds[8][32];
    const int c = threadIdx.x & 31, s = threadIdx.x >> 5;
    const size_t i = (size_t)blockIdx.x * 32 + c;
    float a = 0.f;
    if (i < n) {
        size_t r = s;
        float a1 = 0.f, a2 = 0.f, a3 = 0.f;
        for (; r + 24 < P; r += 32) {
            a += part[r * n + i];
            a1 += part[(r + 8) * n + i];
            a2 += part[(r + 16) * n + i];
            a3 += part[(r + 24) * n + i];
        }
        for (; r < P; r += 8) a += part[r * n + i];
        a = (a + a1) + (a2 + a3);
    }
    lds[s][c] = a;
    __syncthreads();
    if (s == 0 && i < n) {
#pragma unroll
        for (int j = 1; j < 8; ++j) a += lds[j][c];
        out[i] = a;
    }
}

__global__ __launch_bounds__(256) void ln_zero_kernel(float* p, size_t n) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) p[i] = 0.f;
}

// ---- host side ---------------------------------------------------------------------------------------------------------------
// The team for rows of `cols` elements: the fewest lanes that hold a row at 16 bytes each up to a wave, then more vectors per
// lane up to 32 elements, then more lanes.  0: too long for registers.
static int ln_team(int cols, int E, int* ch) {
    const int vecs = ceil_div(cols, E);
    *ch = 1;
    for (int team = 8; team <= 64; team *= 2)
        if (vecs <= team) return team;
    const int most = LN_MAX_PER_LANE / E;
    for (int team = 64; team <= 1024; team *= 4)
        for (int c = 2; c <= most; c *= 2)
            if (vecs <= team * c && (team == 64 || c == most)) {
                *ch = c;
                return team;
            }
    return 0;
}

// Workgroups of a backward pass: enough to fill 256 CUs at the registers that the row takes, no more than there are rows
static size_t ln_backward_blocks(size_t rows, int cols, int E) {
    int ch;
    const int team = ln_team(cols, E, &ch);
    if (team == 0) return rows < 256 ? rows : 256;
    const size_t tpb = team < 256 ? 256 / team : 1;
    const size_t need = (rows + tpb - 1) / tpb, most = ch == 1 ? 1024 : 512;
    return need < most ? need : most;
}

template <typename T>
static void ln_launch_forward(const LnFwdP& p, hipStream_t s) {
    int ch;
    const int team = ln_team(p.cols, Row<T>::E, &ch);
    const size_t tpb = team && team < 256 ? 256 / team : 1;
    const size_t need = (p.rows + tpb - 1) / tpb;
    const dim3 grid((unsigned)(need < (1u << 20) ? need : (1u << 20)));
#define DUN_LN_FWD(TEAM, CH)                                                                               \
    if (team == TEAM && ch == CH) {                                                                        \
        hipLaunchKernelGGL((ln_forward_kernel<T, TEAM, CH>), grid, dim3(ln_block<TEAM>()), 0, s, p);       \
        return;                                                                                            \
    }
    constexpr int M = LN_MAX_PER_LANE / Row<T>::E;
    DUN_LN_FWD(8, 1)
    DUN_LN_FWD(16, 1)
    DUN_LN_FWD(32, 1)
    DUN_LN_FWD(64, 1)
    DUN_LN_FWD(64, 2)
    DUN_LN_FWD(64, 4)
    if constexpr (M == 8) DUN_LN_FWD(64, M)
    DUN_LN_FWD(256, M)
    DUN_LN_FWD(1024, M)
    hipLaunchKernelGGL((ln_forward_long_kernel<T>), dim3((unsigned)(p.rows < 65536 ? p.rows : 65536)), dim3(LN_LONG_THREADS), 0, s, p);
#undef DUN_LN_FWD
}

template <typename T, int K>
static void ln_launch_backward_k(const LnBwdP& p, unsigned blocks, hipStream_t s) {
    int ch;
    const int team = ln_team(p.cols, Row<T>::E, &ch);
#define DUN_LN_BWD(TEAM, CH)                                                                               \
    if (team == TEAM && ch == CH) {                                                                        \
        hipLaunchKernelGGL((ln_backward_kernel<T, TEAM, CH, K>), dim3(blocks), dim3(ln_block<TEAM>()), 0, s, p); \
        return;                                                                                            \
    }
    constexpr int M = LN_MAX_PER_LANE / Row<T>::E;
    DUN_LN_BWD(8, 1)
    DUN_LN_BWD(16, 1)
    DUN_LN_BWD(32, 1)
    DUN_LN_BWD(64, 1)
    DUN_LN_BWD(64, 2)
    DUN_LN_BWD(64, 4)
    if constexpr (M == 8) DUN_LN_BWD(64, M)
    DUN_LN_BWD(256, M)
    DUN_LN_BWD(1024, M)
    hipLaunchKernelGGL((ln_backward_long_kernel<T>), dim3(blocks), dim3(LN_LONG_THREADS), 0, s, p);
#undef DUN_LN_BWD
}

template <typename T>
static void ln_launch_backward(const LnBwdP& p, unsigned blocks, hipStream_t s) {
    if (p.K == 0) return ln_launch_backward_k<T, 0>(p, blocks, s);
    if (p.K == 2) return ln_launch_backward_k<T, 2>(p, blocks, s);
    ln_launch_backward_k<T, 3>(p, blocks, s);
}

}  // namespace dun

using namespace dun;

extern "C" size_t dun_layer_norm_backward_workspace_floats(int64_t rows, int cols, int dtype, int sums) {
    if (rows <= 0 || cols <= 0 || sums < 2) return 0;
    const size_t blocks = ln_backward_blocks((size_t)rows, cols, dtype == DUN_F32 ? 4 : 8);
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
            const size_t n = (size_t)sums * cols;
            hipLaunchKernelGGL(ln_zero_kernel, dim3((unsigned)(n < (1u << 18) ? (n + 255) / 256 : 1024)), dim3(256), 0, s, sums_out, n);
            DUN_LAUNCH_CHECK();
        }
        return DUN_OK;
    }
    DUN_REQUIRE(dy && dx && stats, "dun_layer_norm_backward: null tensor");
    DUN_REQUIRE(!x != !x_codes && !x_codes == !x_exps, "dun_layer_norm_backward: either x or its codes and exponents");
    DUN_REQUIRE(((uintptr_t)x_codes & 7) == 0, "dun_layer_norm_backward: codes need 8-byte alignment");
    DUN_REQUIRE(lddy >= cols && lddx >= cols && (!x || ldx >= cols), "dun_layer_norm_backward: a row stride is below %d columns", cols);
    const size_t blocks = ln_backward_blocks((size_t)rows, cols, dtype == DUN_F32 ? 4 : 8);
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
        hipLaunchKernelGGL(ln_reduce_kernel, dim3((unsigned)((n + 31) / 32)), dim3(256), 0, s, ws, blocks, n, sums_out);
        DUN_LAUNCH_CHECK();
    }
    return DUN_OK;
}
