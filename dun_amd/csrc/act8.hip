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

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef u32 u32x4_any __attribute__((ext_vector_type(4), aligned(8)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

// ---- pack / unpack: elementwise streams -----------------------------------------------------------------------------------------
// 65536 x 2048 fp32: pack 147 us, unpack 128 - 144 us (4.6, 4.7 - 5.3 TB/s); bf16 125 and 103 us (3.2, 3.9 TB/s).
// One vector of E columns per lane; a row is G * 32 / E vectors (padded groups included), so the lanes of a group are neighbours.
template <typename T>
__global__ __launch_bounds__(256) void act8_pack_kernel(const T* x, size_t ldx, uint8_t* codes, uint8_t* exps, size_t vecs,
                                                        u32 vpr, int cols, int relu) {
    constexpr int GV = ACT8_GROUP / E;
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
        u32 byte;
        const u32 word = act8_pack(v, relu, &byte);
        *reinterpret_cast<u32*>(codes + i * E) = word;
        if (vec % GV == 0) exps[i / GV] = (uint8_t)byte;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void act8_unpack_kernel(const uint8_t* codes, const uint8_t* exps, T* out, size_t ldo,
                                                          size_t vecs, u32 vpr, int cols, float zero) {
    constexpr int GV = ACT8_GROUP / E;
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
        float v[E];
        act8_values(*reinterpret_cast<const u32*>(codes + i * E), exps[i / GV], zero, v);
        store_part(out + row * ldo, (int)vec * E, cols, v);
    }
}

// ---- weight gradient ------------------------------------------------------------------------------------------------------------------
struct WgradP {
    const void* dy;
    const uint8_t* codes;
    const uint8_t* exps;
    float* dw;  // [S][O][I], `stride` apart
    float* db;  // [S][O], `stride` apart, or null
    size_t lddy, rows, stride;
    size_t rows_per;  // rows of one split, a multiple of 32
    int O, I, groups, pitch;
    int tiles_m, tiles_n, splits;
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
// value of byte j of a word of codes: unsigned, or signed (stored + 128; `word` has been turned into signed bytes by code_word)
template <bool SIGNED>
__device__ __forceinline__ u32 code_word(u32 word) { return SIGNED ? word ^ 0x80808080u : word; }
template <bool SIGNED>
__device__ __forceinline__ float code_value(u32 word, int j, float s) {
    return SIGNED ? (float)(signed char)(word >> (8 * j)) * s : (float)((word >> (8 * j)) & 0xffu) * s;
}

// What a thread holds of dy between its load and the matrix cores: AC neighbouring columns of 8 rows.  `up`: the pair was loaded one column
// early, because it passed the last one; its first column is the second that was loaded.
template <typename T, int AC> struct DyRegs {
    f32x2_t v[8];
    __device__ __forceinline__ void get(int j, __amdgpu_buffer_rsrc_t r, u32 lane, u32 row) {
        if constexpr (AC == 2)
            v[j] = __builtin_bit_cast(f32x2_t, __builtin_amdgcn_raw_buffer_load_b64(r, lane, row, 0));
        else
            v[j][0] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, lane, row, 0));
    }
    __device__ __forceinline__ void keep(int j, bool yes) { v[j] = yes ? v[j] : f32x2_t{0.f, 0.f}; }
    __device__ __forceinline__ void align(bool up) {
        if constexpr (AC == 2) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j][0] = up ? v[j][1] : v[j][0];
        }
    }
    __device__ __forceinline__ float value(int j, int c) const { return v[j][c]; }
    __device__ __forceinline__ void terms(int c, u32x4_t* out) const {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = v[j][c];
        split_terms<3>(x, out);
    }
};
template <typename T, int AC> struct DyRegs16 {
    u32 v[8];  // AC = 2: both columns in a word
    __device__ __forceinline__ void get(int j, __amdgpu_buffer_rsrc_t r, u32 lane, u32 row) {
        if constexpr (AC == 2)
            v[j] = __builtin_amdgcn_raw_buffer_load_b32(r, lane, row, 0);
        else
            v[j] = (u16)__builtin_amdgcn_raw_buffer_load_b16(r, lane, row, 0);
    }
    __device__ __forceinline__ void keep(int j, bool yes) { v[j] = yes ? v[j] : 0u; }
    __device__ __forceinline__ void align(bool up) {
        if constexpr (AC == 2) {
            const int by = up ? 16 : 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] >>= by;
        }
    }
    __device__ __forceinline__ float value(int j, int c) const { return to_f32(T{(u16)(v[j] >> (16 * c))}); }
};
template <int AC> struct DyRegs<bf16_t, AC> : DyRegs16<bf16_t, AC> {
    __device__ __forceinline__ void terms(int c, u32x4_t* out) const {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            out[0][q] = __builtin_amdgcn_perm(this->v[2 * q + 1], this->v[2 * q], c ? 0x07060302u : 0x05040100u);
    }
};
template <int AC> struct DyRegs<fp16_t, AC> : DyRegs16<fp16_t, AC> {
    __device__ __forceinline__ void terms(int c, u32x4_t* out) const {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = this->value(j, c);
        split_terms<2>(x, out);
    }
};

// Barrier for data in LDS only: loads from global memory stay in flight across it
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// A buffer of `bytes` from p on (0x00027000: raw 32-bit data)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_buffer(const void* p, u32 bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00027000);
}

// A workgroup owns a BM x BN tile of dw over one range of rows and walks it 32 rows at a time through two LDS buffers of
// bf16 operands: [column][32 rows], 64 bytes a column, N such planes for dy and one for the values.  While the matrix
// cores work on one buffer, the rows two steps ahead are on their way into registers and those one step ahead are taken
// apart into the other buffer.  Waves own WM x WN sub-tiles; dy has N planes, so WM < WN keeps the LDS reads of a wave, N WM + WN
// columns per step, low.
// 65536 x 2048 x 2048 fp32: 1.31 ms, 1.26 PFLOP/s of bf16 products (an 8192^3 bf16 product of the installed library: 1.20), the matrix pipe busy
// for 66 % of the cycles at a clock that falls to 1.6 GHz under it.  On the way: loads under branches, waited for where they were
// issued, 1.54 ms (49 %); an fp32 product of the library 4.2 ms.  fp16 dy 0.93 ms (1.18 PFLOP/s), bf16 dy 0.61 ms (0.90): one MFMA a tile,
// the staging shows.
// A column's four 16-byte chunks (8 rows each) and the column's place among its neighbours are permuted by its
// index so that the writes (columns 1, 2 or 4 apart, one chunk) and the reads (columns in a row, one chunk) spread over the banks.
__device__ __forceinline__ int lds_chunk(int col, int kc) {
    const int g = col >> 2;
    return ((col & ~3) | ((col ^ g) & 3)) * 4 + (kc ^ (-g & 3) ^ ((g >> 2) & 3));
}

template <typename T, bool SIGNED, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64, (BM / WM) * (BN / WN) >= 8 ? 2 : 1) void act8_wgrad_tile_kernel(const WgradP p) {
    constexpr int N = Terms<T>::N, NT = (BM / WM) * (BN / WN) * 64;
    constexpr int AC = 4 * BM / NT, BC = 8 * BN / NT;
    constexpr int MT = WM / 32, CT = WN / 32;
    constexpr int PLANE_A = BM * 4, PLANE_B = BN * 4;  // 16-byte chunks
    constexpr int BUF = N * PLANE_A + PLANE_B;
    __shared__ u32x4_t lds[2 * BUF];

    // workgroups go round-robin over the 8 XCDs: each takes a contiguous range of (split, tile row, tile column), so that the
    // tiles that read the same rows of dy and codes meet in one L2
    int id = blockIdx.x;
    {
        const int nwg = gridDim.x, q = nwg >> 3, r = nwg & 7, xcd = id & 7, idx = id >> 3;
        id = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + idx;
    }
    const int tn = id % p.tiles_n;
    id /= p.tiles_n;
    const int tm = id % p.tiles_m, split = id / p.tiles_m;
    const int m0 = tm * BM, n0 = tn * BN;
    const size_t r_begin = (size_t)split * p.rows_per;
    const size_t r_end = r_begin + p.rows_per < p.rows ? r_begin + p.rows_per : p.rows;
    const int steps = (int)((r_end - r_begin + 31) / 32);

    const int tid = threadIdx.x;
    // Loads: 8 rows x AC columns of dy, 4 rows x BC columns of codes (one group).  No branches around them and nothing done with what
    // they bring before it is staged, or they would be waited for where they are issued.  Columns past the last are read from inside
    // the row: they make rows or columns of dw that nobody stores.  The last step of a range takes the range's last 32 rows, and counts
    // the ones it has seen before as zeros.  Through buffer descriptors that start at the step's first row: an offset of the lane
    // that never changes plus one of the row.
    const int a_cg = tid % (BM / AC), a_kc = tid / (BM / AC);
    const int a_col = m0 + a_cg * AC, a_most = p.O - AC;  // (O > 32 here)
    const bool up = a_col > a_most;
    const u32 a_row = (u32)p.lddy * (u32)sizeof(T);
    const u32 a_off = (u32)a_kc * 8 * a_row + (u32)(up ? a_most : a_col) * (u32)sizeof(T);
    // (neighbouring lanes take the two halves of a chunk: 32 lanes write all of 256 bytes)
    const int b_cg = (tid >> 1) % (BN / BC), b_kq = (tid & 1) + 2 * (tid / (2 * BN / BC));
    int b_col = n0 + b_cg * BC;
    b_col = b_col < p.pitch ? b_col : p.pitch - BC;
    const u32 b_off = (u32)(b_kq * 4) * (u32)p.pitch + (u32)b_col;
    const u32 e_off = (u32)(b_kq * 4) * (u32)p.groups + (u32)(b_col / ACT8_GROUP);

    DyRegs<T, AC> ra;
    u32 rb[4][(BC + 3) / 4], re[4];
    const int rest = (int)(r_end - r_begin) - 32 * (steps - 1);  // rows of the last step
    const bool few = r_end < 32;                                 // (no 32 rows to take: only step 0 of all there is)
    auto load = [&](int step) {
        const size_t r = step + 1 < steps ? r_begin + (size_t)step * 32 : r_end - 32;
        const __amdgpu_buffer_rsrc_t da = rows_buffer((const char*)p.dy + r * a_row, 31 * a_row + (u32)p.O * (u32)sizeof(T));
        const __amdgpu_buffer_rsrc_t db = rows_buffer(p.codes + r * p.pitch, 32 * (u32)p.pitch);
        const __amdgpu_buffer_rsrc_t de = rows_buffer(p.exps + r * p.groups, 32 * (u32)p.groups);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const u32 at = (u32)j * (u32)p.pitch;
            if constexpr (BC == 2) {
                rb[j][0] = (u16)__builtin_amdgcn_raw_buffer_load_b16(db, b_off, at, 0);
            } else if constexpr (BC == 4) {
                rb[j][0] = __builtin_amdgcn_raw_buffer_load_b32(db, b_off, at, 0);
            } else {
                const u32x2_t q = __builtin_amdgcn_raw_buffer_load_b64(db, b_off, at, 0);
                rb[j][0] = q[0];
                rb[j][(BC + 3) / 4 - 1] = q[1];
            }
            re[j] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(de, e_off, (u32)j * (u32)p.groups, 0);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) ra.get(j, da, a_off, (u32)j * a_row);
    };
    auto load_few = [&] {  // rows past the last are read from the last, and count as zeros
        const int last = (int)r_end - 1;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = b_kq * 4 + j < last ? b_kq * 4 + j : last;
#pragma unroll
            for (int k = 0; k < (BC + 3) / 4; ++k) {
                const uint8_t* q = p.codes + (size_t)r * p.pitch + b_col + 4 * k;
                rb[j][k] = BC == 2 ? (u32)*reinterpret_cast<const u16*>(q) : *reinterpret_cast<const u32*>(q);
            }
            re[j] = p.exps[(size_t)r * p.groups + b_col / ACT8_GROUP];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int r = a_kc * 8 + j < last ? a_kc * 8 + j : last;
            ra.get(j, rows_buffer(p.dy, (u32)last * a_row + (u32)p.O * (u32)sizeof(T)), a_off - (u32)a_kc * 8 * a_row + (u32)r * a_row, 0);
        }
    };

    const bool want_db = p.db && tn == 0;
    double bias[AC];
#pragma unroll
    for (int c = 0; c < AC; ++c) bias[c] = 0.0;
    auto stage = [&](int buf, int step) {
        if (step + 1 == steps && (rest < 32)) {  // (the same for the whole workgroup) zeros in both operands: a value there could be a NaN
            const int lo = few ? 0 : 32 - rest, hi = few ? rest : 32;
#pragma unroll
            for (int j = 0; j < 8; ++j) ra.keep(j, a_kc * 8 + j >= lo && a_kc * 8 + j < hi);
#pragma unroll
            for (int j = 0; j < 4; ++j) re[j] = b_kq * 4 + j >= lo && b_kq * 4 + j < hi ? re[j] : 0u;
        }
        u32x4_t* A = lds + buf * BUF;
        u32x4_t* B = A + N * PLANE_A;
        if (m0 + BM > p.O) ra.align(up);  // (the same for the whole workgroup)
#pragma unroll
        for (int c = 0; c < AC; ++c) {
            u32x4_t t[N];
            ra.terms(c, t);
            const int at = lds_chunk(a_cg * AC + c, a_kc);
#pragma unroll
            for (int k = 0; k < N; ++k) A[k * PLANE_A + at] = t[k];
        }
        if (want_db) {
#pragma unroll
            for (int c = 0; c < AC; ++c) {
                const float s0 = ra.value(0, c) + ra.value(1, c), s1 = ra.value(2, c) + ra.value(3, c);
                const float s2 = ra.value(4, c) + ra.value(5, c), s3 = ra.value(6, c) + ra.value(7, c);
                bias[c] += (double)((s0 + s1) + (s2 + s3));
            }
        }
        float s[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            s[j] = act8_scale(re[j]);
#pragma unroll
            for (int k = 0; k < (BC + 3) / 4; ++k) rb[j][k] = code_word<SIGNED>(rb[j][k]);
        }
#pragma unroll
        for (int c = 0; c < BC; ++c) {
            u32x2_t w;
            w[0] = top_halves(code_value<SIGNED>(rb[1][c / 4], c % 4, s[1]), code_value<SIGNED>(rb[0][c / 4], c % 4, s[0]));
            w[1] = top_halves(code_value<SIGNED>(rb[3][c / 4], c % 4, s[3]), code_value<SIGNED>(rb[2][c / 4], c % 4, s[2]));
            reinterpret_cast<u32x2_t*>(B)[lds_chunk(b_cg * BC + c, b_kq >> 1) * 2 + (b_kq & 1)] = w;
        }
    };

    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = (wave / (BN / WN)) * WM, wn = (wave % (BN / WN)) * WN;
    const int fc = lane & 31, fk = lane >> 5;
    f32x16 acc[MT][CT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < CT; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    // A wave alone has to keep the matrix pipe busy for as long as its partner stages: the operands of the next 32 rows of dw are read
    // from LDS before the products of these are issued.
    auto compute = [&](int buf) {
        const u32x4_t* A = lds + buf * BUF;
        const u32x4_t* B = A + N * PLANE_A;
        u32x4_t a[2][N], b[2][CT];
        auto read_a = [&](int g) {
            const int at = lds_chunk(wm + 32 * (g % MT) + fc, 2 * (g / MT) + fk);
#pragma unroll
            for (int t = 0; t < N; ++t) a[g & 1][t] = A[t * PLANE_A + at];
        };
        auto read_b = [&](int ks) {
#pragma unroll
            for (int j = 0; j < CT; ++j) b[ks][j] = B[lds_chunk(wn + 32 * j + fc, 2 * ks + fk)];
        };
        read_b(0);
        read_a(0);
#pragma unroll
        for (int g = 0; g < 2 * MT; ++g) {
            if (g + 1 < 2 * MT) {
                if ((g + 1) % MT == 0) read_b(1);
                read_a(g + 1);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int t = 0; t < N; ++t)
#pragma unroll
                for (int j = 0; j < CT; ++j)
                    acc[g % MT][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a[g & 1][t]), __builtin_bit_cast(bf16x8_t, b[g / MT][j]),
                                                                             acc[g % MT][j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    // Two waves share a SIMD in the large tile: one of each pair takes its rows apart before its matrix products, the other after them, so
    // that the vector and the matrix pipe both have work all the time.  Between two barriers the early waves stage step k + 1 and
    // multiply step k, the late ones multiply k and stage k + 1; with the loop turned by half a step for the late ones both do it in
    // the same place of the code: stage, [late: barrier], multiply, [early: barrier].
    const bool early = NT < 512 || wave < NT / 128;
    if (few)
        load_few();
    else
        load(0);
    stage(0, 0);
    if (steps > 1) load(1);
    lds_barrier();
    for (int k = 0; k < steps; ++k) {
        const int s = early ? k + 1 : k;
        if (s >= 1 && s < steps) {
            stage(s & 1, s);
            load(s + 1 < steps ? s + 1 : s);
        }
        if (!early && k >= 1) lds_barrier();
        compute(k & 1);
        if (early) lds_barrier();
    }
    if (!early) lds_barrier();

    float* dw = p.dw + split * p.stride;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < CT; ++j) {
            const int n = n0 + wn + 32 * j + fc;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int m = m0 + wm + 32 * i + (e & 3) + 8 * (e >> 2) + 4 * fk;
                if (m < p.O && n < p.I) dw[(size_t)m * p.I + n] = acc[i][j][e];
            }
        }
    if (want_db) {  // (uniform; the last barrier above closed the buffers)
        double* sum = reinterpret_cast<double*>(lds);
#pragma unroll
        for (int c = 0; c < AC; ++c) sum[a_kc * BM + a_cg * AC + c] = bias[c];
        __syncthreads();
        for (int m = tid; m < BM; m += NT)
            if (m0 + m < p.O) p.db[split * p.stride + m0 + m] = (float)((sum[m] + sum[BM + m]) + (sum[2 * BM + m] + sum[3 * BM + m]));
    }
}

// Few outputs (up to 16 G): nothing to share between waves, and the codes are the whole traffic.  A wave owns 256 columns and a range of
// rows and takes both operands from global memory straight into the MFMA's registers, no LDS: v_mfma_f32_16x16x32_bf16 wants rows
// 8 (l / 16) .. + 7 of column l % 16 in lane l, and WHICH column of dw that is, is free: with the lane's 16 codes per row (one
// load) being columns 16 (l % 16) + t, tile t = 0 .. 15 takes byte t of every load.  49152 x 10 x 2048: 31 us, 3.4 TB/s (without the loads of the
// next rows under way 46 us): 48 ranges of rows x 8 column tiles are 384 workgroups on 256 CUs, and a wave has eight steps whose load
// latency shows.  65536 x 32 x 2048, two groups: 48 us, 3.0 TB/s.
template <typename T, bool SIGNED, int G>
__global__ __launch_bounds__(256, 2) void act8_wgrad_narrow_kernel(const WgradP p) {
    constexpr int N = Terms<T>::N;
    __shared__ float lds[G * 16 * 256];
    __shared__ double lds_db[4][G * 16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c = lane & 15, k8 = lane >> 4;
    const int tn = blockIdx.x % p.tiles_n, split = blockIdx.x / p.tiles_n;
    const int n0 = tn * 256;
    const size_t r_begin = (size_t)split * p.rows_per;
    const size_t r_end = r_begin + p.rows_per < p.rows ? r_begin + p.rows_per : p.rows;
    int col = n0 + 16 * c;
    col = col < p.pitch ? col : p.pitch - 16;  // (columns that nobody stores)
    f32x4 acc[G][16];
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int t = 0; t < 16; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[g][t][e] = 0.f;
    double bias[G];
    int off[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        bias[g] = 0.0;
        off[g] = 16 * g + c < p.O ? 16 * g + c : p.O - 1;
    }
    const T* dy = (const T*)p.dy;
    // the next 32 rows are on their way while these are worked on (two groups of outputs leave no registers for that)
    constexpr bool AHEAD = G == 1;
    u32x4_t qn[8];
    u32 en[8];
    T an[G][8];
    auto fetch = [&](size_t r0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const size_t r = r0 + 8 * k8 + j, rr = r < r_end ? r : r_end - 1;
            qn[j] = *reinterpret_cast<const u32x4_any*>(p.codes + rr * p.pitch + col);
            en[j] = p.exps[rr * p.groups + col / ACT8_GROUP];
#pragma unroll
            for (int g = 0; g < G; ++g) an[g][j] = dy[rr * p.lddy + off[g]];
        }
    };
    size_t r0 = r_begin + 32 * wave;
    if (AHEAD && r0 < r_end) fetch(r0);
    for (; r0 < r_end; r0 += 128) {
        if (!AHEAD) fetch(r0);
        u32x4_t q[8];
        float s[8], a[G][8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool in = r0 + 8 * k8 + j < r_end;  // rows past the last are zeros in both operands
#pragma unroll
            for (int k = 0; k < 4; ++k) q[j][k] = code_word<SIGNED>(qn[j][k]);
            s[j] = in ? act8_scale(en[j]) : 0.f;
#pragma unroll
            for (int g = 0; g < G; ++g) a[g][j] = in ? to_f32(an[g][j]) : 0.f;
        }
        if (AHEAD && r0 + 128 < r_end) fetch(r0 + 128);
        u32x4_t at[G][N];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            split_terms<N>(a[g], at[g]);
            bias[g] += (double)(((a[g][0] + a[g][1]) + (a[g][2] + a[g][3])) + ((a[g][4] + a[g][5]) + (a[g][6] + a[g][7])));
        }
#pragma unroll
        for (int t = 0; t < 16; ++t) {
            u32x4_t b;
#pragma unroll
            for (int h = 0; h < 4; ++h)
                b[h] = top_halves(code_value<SIGNED>(q[2 * h + 1][t >> 2], t & 3, s[2 * h + 1]), code_value<SIGNED>(q[2 * h][t >> 2], t & 3, s[2 * h]));
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int k = 0; k < N; ++k)
                    acc[g][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, at[g][k]), __builtin_bit_cast(bf16x8_t, b),
                                                                        acc[g][t], 0, 0, 0);
        }
    }
    // the four waves in order; lane l holds rows 4 (l / 16) + e of dw's tile and its column l % 16
    for (int w = 0; w < 4; ++w) {
        if (wave == w) {
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int t = 0; t < 16; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float* at = lds + (g * 16 + 4 * k8 + e) * 256 + 16 * t + c;
                        *at = w ? *at + acc[g][t][e] : acc[g][t][e];
                    }
        }
        __syncthreads();
    }
    float* dw = p.dw + split * p.stride;
    const int rows_out = p.O < 16 * G ? p.O : 16 * G;
    for (int i = threadIdx.x; i < rows_out * 256; i += 256) {
        const int o = i >> 8, n = i & 255;  // column n: lane n / 16, tile n % 16
        if (n0 + n < p.I) dw[(size_t)o * p.I + n0 + n] = lds[o * 256 + 16 * (n & 15) + (n >> 4)];
    }
    if (p.db && tn == 0) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
            bias[g] += __shfl_xor(bias[g], 16, 64);
            bias[g] += __shfl_xor(bias[g], 32, 64);
            if (k8 == 0) lds_db[wave][16 * g + c] = bias[g];
        }
        __syncthreads();
        if (threadIdx.x < rows_out)
            p.db[split * p.stride + threadIdx.x] =
                (float)((lds_db[0][threadIdx.x] + lds_db[1][threadIdx.x]) + (lds_db[2][threadIdx.x] + lds_db[3][threadIdx.x]));
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------------------
enum WgradKind { WGRAD_64, WGRAD_64x256, WGRAD_128, WGRAD_256, WGRAD_NARROW1, WGRAD_NARROW2 };
constexpr int WGRAD_MOST = 1 << 24;
struct WgradPlan {
    WgradKind kind;
    int tiles_m, tiles_n, splits;
    size_t rows_per;
};

// `s` ranges of whole 32-row steps, of at least 64 rows
static void wgrad_split(WgradPlan* q, size_t rows, size_t s) {
    const size_t most = (rows + 63) / 64;
    s = s < 1 ? 1 : s > most ? most : s;
    q->rows_per = ((rows + s - 1) / s + 31) / 32 * 32;
    q->splits = (int)((rows + q->rows_per - 1) / q->rows_per);
}

// Tile and number of row ranges with the least estimated time: steps of 32 rows times what a step of that tile takes with 1, 2 or 4
// workgroups on each of 256 CUs (measured with fp32 dy, us, and taken for 16-bit ones too, whose steps are shorter), times the rounds,
// plus the partial results, written and read, and the launch that
// adds them up.  Over 24 shapes from 512 x 40 x 40 to 65536 x 2048 x 100 the choice is within 9 % of the best of all tiles and splits,
// 1.5 % on average; the large tile alone would be 1.6 times slower on the small ones (512 x 100 x 100: 17.2 us against 10.8), the
// small one 1.5 times on the large (65536 x 100 x 2048: 202 us against 125).
static WgradPlan wgrad_plan(size_t rows, int O, int I) {
    WgradPlan q;
    if (O <= 32) {  // the codes are the traffic: enough ranges for every CU, more only while each wave has 8 steps of its own
        q.kind = O <= 16 ? WGRAD_NARROW1 : WGRAD_NARROW2;
        q.tiles_m = 1;
        q.tiles_n = ceil_div(I, 256);
        const size_t one = ceil_div(256, q.tiles_n), two = ceil_div(512, q.tiles_n);
        // (512 rows: one range 6 us, eight and the launch that adds them up 5 us and another 4 on the host)
        const size_t s = rows <= 512 ? 1 : rows / 1024 > one ? (rows / 1024 < two ? rows / 1024 : two) : one;
        wgrad_split(&q, rows, s);
        return q;
    }
    static const struct {
        WgradKind kind;
        int bm, bn;
        double first;    // us before the first and after the last step
        double step[3];  // us a step with 1, 2, 4 workgroups on a CU (0: they do not fit)
    } tiles[] = {{WGRAD_64, 64, 64, 3., {.75, .88, 1.55}},
                 {WGRAD_64x256, 64, 256, 5., {1.3, 2.0, 0.}},
                 {WGRAD_128, 128, 128, 5., {1.45, 2.05, 0.}},
                 {WGRAD_256, 256, 256, 8., {2.65, 0., 0.}}};
    double best = 1e300;
    for (const auto& t : tiles) {
        WgradPlan c;
        c.kind = t.kind;
        c.tiles_m = ceil_div(O, t.bm);
        c.tiles_n = ceil_div(I, t.bn);
        const size_t n = (size_t)c.tiles_m * c.tiles_n;
        for (int want = 128; want <= 1024; want *= 2) {
            wgrad_split(&c, rows, want / n);
            const size_t wgs = n * c.splits;
            int k = 0;
            while (k < 2 && t.step[k + 1] > 0. && wgs > (256u << k)) ++k;
            const double rounds = (double)((wgs + (256u << k) - 1) / (256u << k));
            const double us = t.first + rounds * (double)(c.rows_per / 32) * t.step[k] +
                              (c.splits > 1 ? 5. + (double)c.splits * O * I * 8. / 4e6 : 0.);
            if (us < best) {
                best = us;
                q = c;
            }
        }
    }
    return q;
}

template <typename T, bool SIGNED>
static void wgrad_launch_as(WgradKind kind, const WgradP& p, hipStream_t s) {
    const unsigned grid = (unsigned)p.tiles_m * p.tiles_n * p.splits;
    switch (kind) {
        case WGRAD_NARROW1: hipLaunchKernelGGL((act8_wgrad_narrow_kernel<T, SIGNED, 1>), dim3(grid), dim3(256), 0, s, p); break;
        case WGRAD_NARROW2: hipLaunchKernelGGL((act8_wgrad_narrow_kernel<T, SIGNED, 2>), dim3(grid), dim3(256), 0, s, p); break;
        case WGRAD_64: hipLaunchKernelGGL((act8_wgrad_tile_kernel<T, SIGNED, 64, 64, 32, 32>), dim3(grid), dim3(256), 0, s, p); break;
        case WGRAD_64x256: hipLaunchKernelGGL((act8_wgrad_tile_kernel<T, SIGNED, 64, 256, 32, 128>), dim3(grid), dim3(256), 0, s, p); break;
        case WGRAD_128: hipLaunchKernelGGL((act8_wgrad_tile_kernel<T, SIGNED, 128, 128, 64, 64>), dim3(grid), dim3(256), 0, s, p); break;
        case WGRAD_256: hipLaunchKernelGGL((act8_wgrad_tile_kernel<T, SIGNED, 256, 256, 64, 128>), dim3(grid), dim3(512), 0, s, p); break;
    }
}

template <typename T>
static void wgrad_launch(WgradKind kind, bool rectified, const WgradP& p, hipStream_t s) {
    if (rectified)
        wgrad_launch_as<T, false>(kind, p, s);
    else
        wgrad_launch_as<T, true>(kind, p, s);
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
    const int groups = ceil_div(cols, ACT8_GROUP);
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
    const int groups = ceil_div(cols, ACT8_GROUP);
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
        launch_zero_floats(dw, n, s);
        if (db) launch_zero_floats(db, outs, s);
        DUN_LAUNCH_CHECK();
        return DUN_OK;
    }
    DUN_REQUIRE(dy && codes && exps, "dun_act8_weight_grad: null tensor");
    DUN_REQUIRE(lddy >= outs, "dun_act8_weight_grad: row stride %lld below %d columns", (long long)lddy, outs);
    DUN_REQUIRE(((uintptr_t)codes & 7) == 0, "dun_act8_weight_grad: codes need 8-byte alignment");
    // (offsets inside 32 rows are 32-bit numbers in the kernels)
    DUN_REQUIRE(lddy <= WGRAD_MOST && cols <= WGRAD_MOST, "dun_act8_weight_grad: row stride %lld or %d columns above %d", (long long)lddy, cols, WGRAD_MOST);
    const WgradPlan q = wgrad_plan((size_t)rows, outs, cols);
    DUN_REQUIRE((size_t)q.tiles_m * q.tiles_n * q.splits <= 0x7fffffffu, "dun_act8_weight_grad: %d x %d is too large a gradient", outs, cols);
    const size_t need = dun_act8_weight_grad_workspace_floats(rows, outs, cols, dtype);
    DUN_REQUIRE(need == 0 || (ws && ws_floats >= need), "dun_act8_weight_grad: workspace of %zu floats, %zu needed", ws_floats, need);
    WgradP p;
    memset(&p, 0, sizeof(p));
    p.dy = dy;
    p.codes = codes;
    p.exps = exps;
    p.stride = db ? n + outs : n;  // a split's dw and db lie one behind the other: one launch adds both up
    p.dw = need ? ws : dw;
    p.db = !db ? nullptr : need ? ws + n : db;
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
    if (dtype == DUN_F32)
        wgrad_launch<float>(q.kind, relu != 0, p, s);
    else if (dtype == DUN_BF16)
        wgrad_launch<bf16_t>(q.kind, relu != 0, p, s);
    else
        wgrad_launch<fp16_t>(q.kind, relu != 0, p, s);
    DUN_LAUNCH_CHECK();
    if (need) {
        launch_sum_rows(ws, q.splits, p.stride, dw, n, db, s);
        DUN_LAUNCH_CHECK();
    }
    return DUN_OK;
}
