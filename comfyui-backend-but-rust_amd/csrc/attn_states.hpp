// Attention of query rows to stored states: the kernel that cross_attn.hip (16-bit keys and values) and kv8_attn.hip (pages of 8-bit
// codes) share.  What differs is where a tile of keys and values comes from: a Source.
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = 2^(x_j - base),   x_j = c s_j + bias_j (in units of log2),   s_j = q . k_j
//
// One pass over the keys with a running base (the maximum so far, moved only when a row outgrows it by 2^kLag) and sum, both in fp32.
//
// The rows of a problem are the query tokens times the query heads that share a key-value head: row r is token r / group, head
// r % group.  A wave holds 32 of them, one per lane and half wave.  Keys ride in src0 and queries in src1 of
// v_mfma_f32_32x32x16, so a lane ends up with 16 of every 32 scores of ONE row: maxima and sums are in-lane plus one exchange with
// lane ^ 32, and the scores are, in order, what the lane has to supply as src1 of the product with V if that product counts its keys as
// key_of() does.  Probabilities never cross lanes.  V is read from LDS with the transposing 16-bit read, which turns four keys times
// 16 channels, so it is staged as it lies in memory.
//
// A workgroup is QW waves of 32 rows on the same keys, or KW waves on the same 32 rows and different keys, whose results meet in LDS.
// With SPLIT several workgroups share a row's keys and leave numerators, denominators and bases in the workspace.
#pragma once
#include "common.hpp"

#include <math.h>

namespace states {

typedef float f16acc __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// Rows may outgrow their base by 2^kLag before numerator and denominator are rescaled: far from the ends of fp32, and of the f16 that
// probabilities are rounded to (2^15.99).
constexpr float kLag = 6.f;
constexpr float kLog2e = 1.4426950408889634f;

template <int DT> __device__ __forceinline__ f16acc mfma(u32x4 a, u32x4 b, f16acc c) {
    if constexpr (DT == DT_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <int DT> __device__ __forceinline__ uint32_t pack2(float a, float b) { return DT == DT_BF16 ? pack_bf16x2(a, b) : pack_f16x2(a, b); }
// The larger / the sum of this lane's value and lane ^ 32's.
__device__ __forceinline__ float half_max(float v) {
    const auto s = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
    return fmaxf(u2f(s[0]), u2f(s[1]));
}
__device__ __forceinline__ float half_sum(float v) {
    const auto s = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
    return u2f(s[0]) + u2f(s[1]);
}
// Key, within a block of 32, of accumulator register i in the half wave g.
__device__ __forceinline__ constexpr int key_of(int i, int g) { return (i & 3) + 8 * (i >> 2) + 4 * g; }

// Byte position of an 8-element chunk of a staged row, rows of DP 16-bit elements.  K rows are read 16 bytes a lane, 16 rows at a time:
// the XOR spreads one chunk of 16 rows over all banks.  V rows are read by the transposing read, four rows of 64 bytes at a time.
template <int DP> __device__ __forceinline__ int k_place(int row, int chunk) {
    return row * (2 * DP) + 16 * (chunk ^ (DP == 64 ? (row >> 1) & 7 : row & 15));
}
template <int DP> __device__ __forceinline__ int v_place(int row, int chunk) {
    return row * (2 * DP) + 16 * (chunk ^ (DP == 64 ? ((row >> 1) & 1) << 2 : (row & 3) << 2));
}

// Eight signed bytes as f16, exactly: 0x6400 | u is 1024 + u in f16, and codes are u - 128.
__device__ __forceinline__ u32x4 bytes_to_f16(uint32_t lo, uint32_t hi) {
    const f16x2 off = {(_Float16)-1152.f, (_Float16)-1152.f};
    const auto two = [&](uint32_t w, uint32_t sel) { return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, sel)) + off); };
    lo ^= 0x80808080u;
    hi ^= 0x80808080u;
    return u32x4{two(lo, 0x04010400u), two(lo, 0x04030402u), two(hi, 0x04010400u), two(hi, 0x04030402u)};
}

// The rows of a workgroup, as a Source names them.
struct Problem {
    int64_t q_at, o_at;      // element offsets of token 0 at the key-value head's first query head
    int tokens;              // query tokens
    int keys;                // keys that any row may see
    int limit0;              // row of token t sees keys below min(keys, limit0 + t)
};

struct Common {
    const void* q;
    void* o;
    int64_t q_rs, q_hs, o_rs, o_hs;    // element strides of tokens and heads
    int hk, group, d, q_dt;
    int row_tiles, problems, splits;   // grid: row_tiles * problems (batch x hk) * splits
    int aligned;                       // q rows start on 16 bytes (bit 0), o rows on 8 (bit 1)
    float c;                           // scale * log2 e, its sign in `negate`
    int negate;
    float* part;                       // [splits][problems][rows padded to tiles][DP + 2] where splits > 1
    int rows_padded;
};

__device__ __forceinline__ u32x4 load8(const uint16_t* p, bool aligned) {
    if (aligned) return *reinterpret_cast<const u32x4*>(p);
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = (uint32_t)p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
    return r;
}
__device__ __forceinline__ float elem(u32x4 u, int i, int dt) {
    const uint32_t w = u[i >> 1];
    if (dt == DT_BF16) return (i & 1) ? u2f(w & 0xffff0000u) : u2f(w << 16);
    return f16_to_f((uint16_t)((i & 1) ? w >> 16 : w));
}

// grid: one workgroup per (split, problem, row tile), renumbered so that the workgroups of one XCD (every eighth) share keys.
__device__ __forceinline__ int xcd_contiguous(int b, int n) {
    const int base = n >> 3, rem = n & 7, xcd = b & 7, idx = b >> 3;
    return xcd * base + (xcd < rem ? xcd : rem) + idx;
}

template <class Src, int DP, int QW, int KW, int TK>
__global__ __launch_bounds__(64 * QW * KW, DP == 256 ? 1 : 2) void rows_kernel(const Common a, const typename Src::Args sa) {
    constexpr int DT = Src::DT, NB = TK / 32, KS = DP / 16, DB = DP / 32, NBUF = QW > 1 ? 2 : 1, TILE = TK * DP * 2;
    static_assert(QW == 1 || KW == 1, "waves share keys or rows");
    static_assert(KW == 1 || TK >= 32, "the results of KW waves meet in the tiles' place");
    __shared__ __align__(16) uint8_t lds[KW * NBUF * 2 * TILE];
    __shared__ float stat[KW > 1 ? KW * 64 : 1];
    __shared__ __align__(16) float bias[Src::kBias ? KW * NBUF * TK : 4];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, col = lane & 31, g = lane >> 5;
    const int kw = KW > 1 ? wave : 0, qw = KW > 1 ? 0 : wave, tid = KW > 1 ? lane : (int)threadIdx.x;

    int id = xcd_contiguous(blockIdx.x, gridDim.x);
    const int row_tile = id % a.row_tiles;
    id /= a.row_tiles;
    const int split = id % a.splits, problem = id / a.splits;
    const Problem pr = Src::problem(sa, a, problem);
    const int rows = pr.tokens * a.group, r0 = row_tile * 32 * QW;
    if (r0 >= rows) return;     // the whole workgroup: rows of a shorter sequence
    const int row = r0 + qw * 32 + col, token = (row < rows ? row : rows - 1) / a.group, head = (row < rows ? row : rows - 1) - token * a.group;
    const int last_token = (min(rows, r0 + 32 * QW) - 1) / a.group;
    const int limit = min(pr.keys, pr.limit0 + token);              // this lane's row
    const int end = min(pr.keys, pr.limit0 + last_token);           // the workgroup's last key + 1
    const int wave_first = min(rows - 1, r0 + qw * 32) / a.group;
    const int all_see = min(pr.keys, pr.limit0 + wave_first);       // every row of the wave sees the keys below

    // the wave's share of the key tiles
    int t0 = 0, t1 = end > 0 ? (end + TK - 1) / TK : 0;
    if (a.splits > 1) {
        const int share = (t1 + a.splits - 1) / a.splits;
        t0 = min(t1, split * share);
        t1 = min(t1, t0 + share);
    }
    if (KW > 1) {
        const int share = (t1 - t0 + KW - 1) / KW;
        t0 = min(t1, t0 + kw * share);
        t1 = min(t1, t0 + share);
    }

    // q: the lane's row in the order of the products' channels.  The 8-bit source multiplies f16: rows are scaled by a power of two there.
    u32x4 qf[KS];
    float c = a.c;
    {
        const uint16_t* qp = (const uint16_t*)a.q + pr.q_at + token * a.q_rs + head * a.q_hs;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int at = 16 * s + 8 * g;
            qf[s] = at < a.d ? load8(qp + at, a.aligned & 1) : u32x4{0, 0, 0, 0};
        }
        const uint32_t flip = a.negate ? 0x80008000u : 0u;
        if constexpr (Src::kNormalize) {
            float m = 0.f;
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(elem(qf[s], i, a.q_dt)));
            m = half_max(m);
            const int e = m > 0.f && m < INFINITY ? ilogbf(m) : 0;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                u32x4 f;
#pragma unroll
                for (int i = 0; i < 4; ++i) f[i] = pack_f16x2(ldexpf(elem(qf[s], 2 * i, a.q_dt), -e), ldexpf(elem(qf[s], 2 * i + 1, a.q_dt), -e)) ^ flip;
                qf[s] = f;
            }
            c = ldexpf(c, e);
        } else {
#pragma unroll
            for (int s = 0; s < KS; ++s) qf[s] ^= flip;
        }
    }

    f16acc acc[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i) acc[i] = f16acc{};
    float base = -INFINITY, sum = 0.f;

    typename Src::template Stage<DP, TK, 64 * QW> st(sa, a, problem, pr, tid);
    uint8_t* const mine = lds + kw * (NBUF * 2 * TILE);
    float* const my_bias = bias + (Src::kBias ? kw * (NBUF * TK) : 0);
    const auto sync = [] {
        if (QW > 1) __syncthreads();
        else {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    };
    if (t0 < t1) st.load(t0);
    if (NBUF == 2 && t0 < t1) {
        st.write(mine, mine + TILE, my_bias);
        if (t0 + 1 < t1) st.load(t0 + 1);
        sync();
    }
    for (int t = t0; t < t1; ++t) {
        uint8_t* const kb = mine + (NBUF == 2 ? ((t - t0) & 1) * 2 * TILE : 0);
        uint8_t* const vb = kb + TILE;
        float* const tb = my_bias + (Src::kBias && NBUF == 2 ? ((t - t0) & 1) * TK : 0);
        const auto scales = st.scales(NBUF == 2 && t + 1 < t1);
        if (NBUF == 1) {
            sync();
            st.write(kb, vb, tb);
            if (t + 1 < t1) st.load(t + 1);
            sync();
        }
        f16acc s[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) s[b] = f16acc{};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int b = 0; b < NB; ++b) s[b] = mfma<DT>(*reinterpret_cast<const u32x4*>(kb + k_place<DP>(32 * b + col, 2 * ks + g)), qf[ks], s[b]);

        // x = c s (+ bias), and the largest of the tile
        const int k0 = t * TK;
        float top = -INFINITY;
        const bool plain = !Src::kBias && k0 + TK <= all_see;
        if (plain) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float m = s[b][8 * h];
#pragma unroll
                    for (int i = 1; i < 8; ++i) m = fmaxf(m, s[b][8 * h + i]);
                    top = fmaxf(top, fmaf(m, c * scales.k(2 * b + h), scales.lv(2 * b + h)));
                }
        } else {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int key = 32 * b + key_of(i, g);
                    const float add = Src::kBias ? tb[key] : 0.f;
                    const float x = fmaf(s[b][i], c * scales.k(2 * b + (i >> 3)), add);
                    s[b][i] = k0 + key < limit && add != -INFINITY ? x : -INFINITY;
                    top = fmaxf(top, s[b][i] + scales.lv(2 * b + (i >> 3)));
                }
        }
        top = half_max(top);
        if (__any(top > base + kLag)) {
            const float nb = fmaxf(base, top), f = base == -INFINITY ? 0.f : exp2f(base - nb);
            base = nb;
            sum *= f;
#pragma unroll
            for (int i = 0; i < DB; ++i) acc[i] *= f;
        }
        const float from = base == -INFINITY ? 0.f : base;

        uint32_t p[NB][8];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float kc = plain ? c * scales.k(2 * b + h) : 1.f, off = scales.lv(2 * b + h) - from;
                float part = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const float x0 = s[b][8 * h + i], x1 = s[b][8 * h + i + 1];
                    const float p0 = __builtin_amdgcn_exp2f(plain ? fmaf(x0, kc, off) : x0 + off), p1 = __builtin_amdgcn_exp2f(plain ? fmaf(x1, kc, off) : x1 + off);
                    part += p0 + p1;
                    p[b][4 * h + i / 2] = pack2<DT>(p0, p1);
                }
                sum = fmaf(part, scales.iv(2 * b + h), sum);
            }
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const u32x4 pf = {p[b][4 * h], p[b][4 * h + 1], p[b][4 * h + 2], p[b][4 * h + 3]};
#pragma unroll
                for (int i = 0; i < DB; ++i) {
                    u32x2 half[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int r = 32 * b + 16 * h + 8 * j + 4 * g + ((lane & 15) >> 2), chunk = 4 * i + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
                        half[j] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) s16x4*)(vb + v_place<DP>(r, chunk) + 8 * (lane & 1))));
                    }
                    acc[i] = mfma<DT>(u32x4{half[0][0], half[0][1], half[1][0], half[1][1]}, pf, acc[i]);
                }
            }
        if (NBUF == 2) {
            if (t + 1 < t1) {
                uint8_t* const nk = mine + ((t + 1 - t0) & 1) * 2 * TILE;
                st.write(nk, nk + TILE, my_bias + (Src::kBias ? ((t + 1 - t0) & 1) * TK : 0));
                if (t + 2 < t1) st.load(t + 2);
            }
            sync();
        }
    }
    sum = half_sum(sum);

    // Channels of register j of block i: 32 i + key_of(j, g).
    const int64_t part_at = ((int64_t)split * a.problems + problem) * a.rows_padded;
    if constexpr (KW > 1) {
        __syncthreads();
        float* const mo = reinterpret_cast<float*>(lds) + kw * 32 * DP;
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) mo[(32 * i + key_of(j, g)) * 32 + col] = acc[i][j];
        if (g == 0) {
            stat[kw * 64 + col] = base;
            stat[kw * 64 + 32 + col] = sum;
        }
        __syncthreads();
        // every wave adds a part of the channels: DP / KW of them for its lane's row
        float nb = -INFINITY, w[KW];
#pragma unroll
        for (int k = 0; k < KW; ++k) nb = fmaxf(nb, stat[k * 64 + col]);
        float l = 0.f;
#pragma unroll
        for (int k = 0; k < KW; ++k) {
            const float b = stat[k * 64 + col];
            w[k] = b == -INFINITY ? 0.f : exp2f(b - nb);
            l = fmaf(stat[k * 64 + 32 + col], w[k], l);
        }
        if (row >= rows) return;
        constexpr int EACH = DP / KW / 2;      // channels of a lane
        const int d0 = kw * (DP / KW) + g * EACH;
        const float inv = l == 0.f ? 0.f : Src::kOut / l;
        uint16_t* const op = (uint16_t*)a.o + pr.o_at + token * a.o_rs + head * a.o_hs;
        float* const pp = a.part + (part_at + row) * (DP + 2);
#pragma unroll
        for (int j = 0; j < EACH; j += 4) {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = 0.f;
#pragma unroll
                for (int k = 0; k < KW; ++k) v[e] = fmaf(reinterpret_cast<const float*>(lds)[(k * DP + d0 + j + e) * 32 + col], w[k], v[e]);
            }
            if (a.splits > 1) {
#pragma unroll
                for (int e = 0; e < 4; ++e) pp[d0 + j + e] = v[e];
            } else if (d0 + j < a.d) {
#pragma unroll
                for (int e = 0; e < 4; ++e) op[d0 + j + e] = a.q_dt == DT_BF16 ? f_to_bf16(v[e] * inv) : f_to_f16(v[e] * inv);
            }
        }
        if (a.splits > 1 && kw == 0 && g == 0) {
            pp[DP] = nb;
            pp[DP + 1] = l;
        }
    } else {
        if (row >= rows) return;
        if (a.splits > 1) {
            float* const pp = a.part + (part_at + row) * (DP + 2);
#pragma unroll
            for (int i = 0; i < DB; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) pp[32 * i + key_of(j, g)] = acc[i][j];
            if (g == 0) {
                pp[DP] = base;
                pp[DP + 1] = sum;
            }
        } else {
            const float inv = sum == 0.f ? 0.f : Src::kOut / sum;
            uint16_t* const op = (uint16_t*)a.o + pr.o_at + token * a.o_rs + head * a.o_hs;
#pragma unroll
            for (int i = 0; i < DB; ++i)
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    const int at = 32 * i + key_of(j, g);
                    if (at >= a.d) continue;
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = acc[i][j + e] * inv;
                    const u32x2 u = a.q_dt == DT_BF16 ? u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])} : u32x2{pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3])};
                    if (a.aligned & 2) *reinterpret_cast<u32x2*>(op + at) = u;
                    else
#pragma unroll
                        for (int e = 0; e < 4; ++e) op[at + e] = (uint16_t)(u[e >> 1] >> 16 * (e & 1));
                }
        }
    }
}

// The parts of rows whose keys several workgroups shared, added in the order of the keys: one workgroup of DP threads per row.
template <class Src, int DP>
__global__ __launch_bounds__(DP) void join_kernel(const Common a, const typename Src::Args sa) {
    const int row = blockIdx.x % a.rows_padded, problem = blockIdx.x / a.rows_padded;
    const Problem pr = Src::problem(sa, a, problem);
    if (row >= pr.tokens * a.group) return;
    const int token = row / a.group, head = row - token * a.group, ch = threadIdx.x;
    const float* const p = a.part + ((int64_t)problem * a.rows_padded + row) * (DP + 2);
    const int64_t step = (int64_t)a.problems * a.rows_padded * (DP + 2);
    float nb = -INFINITY;
    for (int s = 0; s < a.splits; ++s) nb = fmaxf(nb, p[s * step + DP]);
    float v = 0.f, l = 0.f;
    for (int s = 0; s < a.splits; ++s) {
        const float b = p[s * step + DP], w = b == -INFINITY ? 0.f : exp2f(b - nb);
        v = fmaf(p[s * step + ch], w, v);
        l = fmaf(p[s * step + DP + 1], w, l);
    }
    if (ch >= a.d) return;
    const float r = l == 0.f ? 0.f : v * (Src::kOut / l);
    uint16_t* const op = (uint16_t*)a.o + pr.o_at + token * a.o_rs + head * a.o_hs + ch;
    *op = a.q_dt == DT_BF16 ? f_to_bf16(r) : f_to_f16(r);
}

// How a call runs: rows of 32 with the keys over a workgroup's waves, or tiles of more rows; and over how many workgroups the keys of a row go.
struct Plan {
    int few, rows, row_tiles, splits;
    int64_t bytes;     // workspace
};
inline int padded_dim(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }
inline Plan make_plan(int64_t rows, int64_t problems, int64_t keys, int d) {
    Plan p;
    const int dp = padded_dim(d);
    p.few = rows <= 32;
    p.rows = p.few ? 32 : 128;
    p.row_tiles = (int)((rows + p.rows - 1) / p.rows);
    const int64_t groups = p.row_tiles * problems, want = 2 * (int64_t)device_cu_count();
    const int64_t least = p.few ? 256 : 512;       // keys that are worth a workgroup
    int64_t s = groups >= want ? 1 : (want + groups - 1) / (groups > 0 ? groups : 1);
    const int64_t most = keys / least > 1 ? keys / least : 1;
    p.splits = (int)(s < most ? s : most);
    p.bytes = p.splits > 1 ? 4 * p.splits * problems * p.row_tiles * p.rows * (dp + 2) : 0;
    return p;
}

template <class Src, int DP> inline int launch(const Plan& p, Common& a, const typename Src::Args& sa, hipStream_t stream) {
    const int64_t grid = (int64_t)p.row_tiles * a.problems * p.splits;
    if (grid > 0x7fffffff) return -1;
    if (p.few) rows_kernel<Src, DP, 1, DP == 256 ? 2 : 4, 32><<<(int)grid, DP == 256 ? 128 : 256, 0, stream>>>(a, sa);
    else rows_kernel<Src, DP, 4, 1, DP == 256 ? 32 : 64><<<(int)grid, 256, 0, stream>>>(a, sa);
    KCHECK();
    if (p.splits > 1) {
        join_kernel<Src, DP><<<a.problems * a.rows_padded, DP, 0, stream>>>(a, sa);
        KCHECK();
    }
    return 0;
}
template <class Src> inline int launch_dim(const Plan& p, Common& a, const typename Src::Args& sa, hipStream_t stream) {
    switch (padded_dim(a.d)) {
        case 64: return launch<Src, 64>(p, a, sa, stream);
        case 128: return launch<Src, 128>(p, a, sa, stream);
        default: return launch<Src, 256>(p, a, sa, stream);
    }
}

}  // namespace states
