// Attention of query rows to stored states: the kernel that cross_attn.hip (16-bit keys and values) and kv8_attn.hip (pages of 8-bit
// codes) share.  What differs is where a tile of keys and values comes from: a Source.
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = 2^(x_j - base),   x_j = c s_j (in units of log2),   s_j = q . k_j + bias_j / scale
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
// A workgroup is waves with rows of their own on the same keys (tiles_kernel), or four waves on the same 16 or 32 rows and different keys,
// whose results meet in LDS (few_kernel).  Where that leaves CUs idle, several workgroups share a row's keys and leave numerators,
// denominators and bases in the workspace.
#pragma once
#include "common.hpp"

#include <math.h>

namespace states {

typedef float f16acc __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// Rows may outgrow their base by 2^kLag before numerator and denominator are rescaled: far from the ends of fp32, and of the f16 that
// probabilities are rounded to (2^15.99).
constexpr float kLag = 6.f;
// Where probabilities are f16 they are 2^kShift times as large, up to 2^15: below 2^-23 of the base they are subnormal, and rounded by 2^-34 of it.
template <int DT> constexpr float kShift = DT == DT_F16 ? 9.f : 0.f;
// The least log2 of a value block's A that a row's base counts (8-bit codes).
constexpr float kLeast = -90.f;
constexpr float kLog2e = 1.4426950408889634f;

template <int DT> __device__ __forceinline__ f16acc mfma(u32x4 a, u32x4 b, f16acc c) {
    if constexpr (DT == DT_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <int DT> __device__ __forceinline__ uint32_t pack2(float a, float b) { return DT == DT_BF16 ? pack_bf16x2(a, b) : pack_f16x2(a, b); }
// a plus the two values of a pair: the denominator adds the probabilities as they are rounded for the product with V.
template <int DT> __device__ __forceinline__ float add2(uint32_t two, float a) {
    if constexpr (DT == DT_BF16) return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, two), bf16x2{(__bf16)1.f, (__bf16)1.f}, a, false);
    else return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, two), f16x2{(_Float16)1.f, (_Float16)1.f}, a, false);
}
// The larger / the sum of this lane's value and lane ^ 32's.
__device__ __forceinline__ float half_max(float v) {
    const auto s = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
    return fmaxf(u2f(s[0]), u2f(s[1]));
}
__device__ __forceinline__ float half_sum(float v) {
    const auto s = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
    return u2f(s[0]) + u2f(s[1]);
}
// Sixteen times the sum of 2^(x - from), x = kc s, of N scores from `at` on: by their own largest, so that nothing leaves fp32 which counts.
template <int N, class Scores> __device__ __forceinline__ float sum_of(const Scores& s, int at, float kc, float from) {
    float m = s[at], sum = 0.f;
#pragma unroll
    for (int i = 1; i < N; ++i) m = fmaxf(m, s[at + i]);
    m = fmaxf(m * kc, -3e38f);      // (-inf of all: each is 0)
#pragma unroll
    for (int i = 0; i < N; ++i) sum += __builtin_amdgcn_exp2f(fmaf(s[at + i], kc, -m));
    const float e = fmaxf(m - from + 4.f, -200.f), whole = floorf(e);
    return sum * ldexpf(__builtin_amdgcn_exp2f(e - whole), (int)whole);
}
// What sums and numerators take when their base gives way to a new one: 2^d, d = base - now.  With 8-bit codes bases of the same scores differ as
// far as the A of values do, and sums of a small base are large: 2^d alone would leave fp32, so they take 2^(d / 2) twice.
template <class Src> struct Rebase {
    float f;
    __device__ __forceinline__ Rebase(float base, float now) {
        const float d = base == -INFINITY ? -INFINITY : base - now;     // no keys yet: nothing
        f = exp2f(Src::kNormalize ? 0.5f * d : d);
    }
    __device__ __forceinline__ float whole() const { return Src::kNormalize ? f * f : f; }
    __device__ __forceinline__ float add(float to, float sum) const { return fmaf(Src::kNormalize ? sum * f : sum, f, to); }
};
// Key, within a block of 32, of accumulator register i in the half wave g.
__device__ __forceinline__ constexpr int key_of(int i, int g) { return (i & 3) + 8 * (i >> 2) + 4 * g; }

// A staged tile's rows of DP 16-bit elements, and byte positions in it.  K rows are read 16 bytes a lane, 16 rows at a time: 16 bytes behind
// each row spread one chunk of 16 rows over all banks.  V rows are read by the transposing read, 64 bytes of four rows at a time: 64 bytes
// behind each row, 128 where 64 would end on the first bank again.  (An XOR of the chunk does the same without the room, but costs an instruction a read where a constant offset is free.)
template <int DP> constexpr int kRowK = 2 * DP + 16;
template <int DP> constexpr int kRowV = DP == 96 ? 320 : 2 * DP + 64;
template <int DP> __device__ __forceinline__ int k_place(int row, int chunk) { return row * kRowK<DP> + 16 * chunk; }
template <int DP> __device__ __forceinline__ int v_place(int row, int chunk) { return row * kRowV<DP> + 16 * chunk; }

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
    int aligned;                       // rows start on 16 bytes: q's (bit 0), o's (bit 1)
    float c;                           // |scale| log2 e; 1 where that is 0
    uint32_t q_and, q_xor;             // what q's words take: a negative scale flips their signs, a scale of 0 makes them 0
    float* part;                       // [splits][problems][rows padded to tiles][DP + 2] where splits > 1
    int rows_padded;
};

// A |scale| log2 e below `least` counts as 0.
inline void set_scale(Common& c, float scale, float least) {
    c.c = fabsf(scale) * kLog2e < least ? 0.f : fabsf(scale) * kLog2e;
    c.q_and = 0xffffffffu;
    c.q_xor = scale < 0.f ? 0x80008000u : 0u;
    if (c.c == 0.f) {
        c.c = 1.f;
        c.q_and = c.q_xor = 0u;
    }
}

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

// The rows of a wave: which they are, their queries, and what they have so far.
template <class Src, int DP, int RW> struct Lanes {
    static constexpr int KS = DP / 16, DB = DP / 32, DT = Src::DT;
    int limit[RW];                                   // the lane's rows see keys below
    int all_see;                                     // every row of the wave sees the keys below
    u32x4 qf[RW][KS];                                // in the order of the products' channels
    float c[RW], base[RW], sum[RW];
    f16acc acc[RW][DB];

    // rows from r0 on, of `rows`
    __device__ __forceinline__ void start(const Common& a, const Problem& pr, int r0, int rows, int lane) {
        const int col = lane & 31, g = lane >> 5;
        all_see = min(pr.keys, pr.limit0 + min(rows - 1, r0) / a.group);
#pragma unroll
        for (int w = 0; w < RW; ++w) {
            const int r = min(r0 + 32 * w + col, rows - 1), token = r / a.group, head = r - token * a.group;
            limit[w] = min(pr.keys, pr.limit0 + token);
            c[w] = a.c;
            const uint16_t* qp = (const uint16_t*)a.q + pr.q_at + token * a.q_rs + head * a.q_hs;
            if (a.aligned & 1) {
#pragma unroll
                for (int s = 0; s < KS; ++s) qf[w][s] = 16 * s + 8 * g < a.d ? load8(qp + 16 * s + 8 * g, true) : u32x4{0, 0, 0, 0};
            } else {
#pragma unroll
                for (int s = 0; s < KS; ++s) qf[w][s] = 16 * s + 8 * g < a.d ? load8(qp + 16 * s + 8 * g, false) : u32x4{0, 0, 0, 0};
            }
        }
#pragma unroll
        for (int w = 0; w < RW; ++w) {
            // The 8-bit source multiplies f16: rows are scaled by a power of two there.
            if constexpr (Src::kNormalize) {
                float m = 0.f;
#pragma unroll
                for (int s = 0; s < KS; ++s)
#pragma unroll
                    for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(elem(qf[w][s], i, a.q_dt)));
                m = half_max(m);
                const int e = m > 0.f && m < INFINITY ? ilogbf(m) : 0;
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    u32x4 f;
#pragma unroll
                    for (int i = 0; i < 4; ++i) f[i] = pack_f16x2(ldexpf(elem(qf[w][s], 2 * i, a.q_dt), -e), ldexpf(elem(qf[w][s], 2 * i + 1, a.q_dt), -e)) & a.q_and ^ a.q_xor;
                    qf[w][s] = f;
                }
                c[w] = ldexpf(c[w], e);
            } else {
#pragma unroll
                for (int s = 0; s < KS; ++s) qf[w][s] = qf[w][s] & a.q_and ^ a.q_xor;
            }
            base[w] = -INFINITY;
            sum[w] = 0.f;
#pragma unroll
            for (int i = 0; i < DB; ++i) acc[w][i] = f16acc{};
        }
    }

    // Scores of NB blocks of 32 keys; `k`: the lane's first chunk in LDS.  A key's bias is what its score starts with, in units of the score:
    // -inf for one that is out or past the end, whose K is numbers.
    template <int NB> __device__ __forceinline__ void scores(f16acc (&s)[NB][RW], const uint8_t* k, const float* bias, int g) const {
        f16acc from[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            from[b] = f16acc{};
            if constexpr (Src::kBias)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const f32x4 add = *reinterpret_cast<const f32x4*>(bias + 32 * b + key_of(i, g));
#pragma unroll
                    for (int e = 0; e < 4; ++e) from[b][i + e] = add[e];
                }
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const u32x4 kf = *reinterpret_cast<const u32x4*>(k + 32 * b * kRowK<DP> + 32 * ks);
#pragma unroll
                for (int w = 0; w < RW; ++w) s[b][w] = mfma<DT>(kf, qf[w][ks], ks == 0 ? from[b] : s[b][w]);
            }
    }
    // The largest x of NB blocks of 32 keys from key0, and the base moved where a row outgrew it.  kc: what a score is multiplied with, of
    // each 16 keys; from: what is taken off that.  plain: every row of the wave sees every key, and every block is numbers.  even: no A is
    // below 2^kLeast.
    template <int NB, class Scales>
    __device__ __forceinline__ void raise(f16acc (&s)[NB][RW], float (&kc)[RW][2 * NB], float (&from)[RW], const Scales& sc, int key0, bool plain, bool even, int g) {
        if (!Src::kBias && !plain) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int w = 0; w < RW; ++w)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        if (Src::kNormalize && sc.k(2 * b + (i >> 3)) != sc.k(2 * b + (i >> 3))) s[b][w][i] = NAN;      // a block without numbers
                        if (key0 + 32 * b + key_of(i, g) >= limit[w]) s[b][w][i] = -INFINITY;
                    }
        }
#pragma unroll
        for (int w = 0; w < RW; ++w) {
            float tops[2 * NB];
#pragma unroll
            for (int h = 0; h < 2 * NB; ++h) {
                // never 0, so that -inf stays that (a block of zeros has scores of 0)
                const float k = c[w] * sc.k(h);
                kc[w][h] = k > 1.17549435e-38f ? k : 1.17549435e-38f;
                const f16acc& x = s[h >> 1][w];
                const int i = 8 * (h & 1);
                const float m = fmaxf(fmaxf(fmaxf(fmaxf(x[i], x[i + 1]), x[i + 2]), fmaxf(fmaxf(x[i + 3], x[i + 4]), x[i + 5])), fmaxf(x[i + 6], x[i + 7]));
                tops[h] = fmaf(m, kc[w][h], sc.lv(h));
            }
            float top = tops[0];
#pragma unroll
            for (int h = 1; h < 2 * NB; ++h) top = fmaxf(top, tops[h]);
            if (Src::kNormalize && __builtin_expect(!even, 0))
#pragma unroll
                for (int h = 0; h < 2 * NB; ++h)
#pragma unroll
                    for (int i = 0; i < 8; ++i) top = fmaxf(top, fmaf(s[h >> 1][w][8 * (h & 1) + i], kc[w][h], kLeast));
            top = half_max(top);
            if (__any(top > base[w] + kLag)) {
                const float nb = fmaxf(base[w], top);
                const Rebase<Src> by(base[w], nb);
                const float f = by.whole();
                base[w] = nb;
                sum[w] = by.add(0.f, sum[w]);
#pragma unroll
                for (int i = 0; i < DB; ++i) acc[w][i] *= f;
            }
            from[w] = base[w] == -INFINITY ? 0.f : base[w] - kShift<DT>;
            // far out (a bias like the type's lowest value) a fused c s - base would show how base was rounded: the rounded product does not
            if (Src::kBias && __any(fabsf(from[w]) > 262144.f)) {
#pragma unroll
                for (int h = 0; h < 2 * NB; ++h) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) s[h >> 1][w][8 * (h & 1) + i] = s[h >> 1][w][8 * (h & 1) + i] * kc[w][h] - from[w];
                    kc[w][h] = 1.f;
                }
                from[w] = 0.f;
            }
        }
    }
    // The sum of NB blocks where probs() adds none of it, their A being uneven: what is subnormal or nothing beside the largest p' may be a
    // large probability of a small A.
    template <int NB> __device__ __forceinline__ void add_sum(const f16acc (&s)[NB][RW], const float (&kc)[RW][2 * NB], const float (&from)[RW]) {
#pragma unroll
        for (int w = 0; w < RW; ++w)
#pragma unroll
            for (int h = 0; h < 2 * NB; ++h) sum[w] += sum_of<8>(s[h >> 1][w], 8 * (h & 1), kc[w][h], from[w]);
    }
    // Probabilities of 16 of the keys (h), rounded and in pairs, and their sum.  The product with V takes 16-bit operands, so they are rounded to V's type
    // (codes: f16), each by 2^-8 (bf16) or 2^-11 of itself at most; the sum is of them as rounded, which takes half the
    // instructions and leaves out what all keys lose alike.
    template <int NB, class Scales>
    __device__ __forceinline__ void probs(u32x4 (&p)[RW], const f16acc (&s)[NB][RW], const float (&kc)[RW][2 * NB], const float (&from)[RW], const Scales& sc, int h) {
#pragma unroll
        for (int w = 0; w < RW; ++w) {
            const float off = sc.lv(h) - from[w];
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = __builtin_amdgcn_exp2f(fmaf(s[h >> 1][w][8 * (h & 1) + i], kc[w][h], off));
#pragma unroll
            for (int i = 0; i < 8; i += 2) p[w][i / 2] = pack2<DT>(e[i], e[i + 1]);
            float part = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) part = add2<DT>(p[w][i], part);
            sum[w] = fmaf(part, sc.iv(h), sum[w]);
        }
    }
    // acc += V^T p for those 16 keys; `v`: the lane's place in the first of their rows.
    __device__ __forceinline__ void values(const u32x4 (&p)[RW], const uint8_t* v) {
#pragma unroll
        for (int i = 0; i < DB; ++i) {
            u32x2 half[2];
#pragma unroll
            for (int j = 0; j < 2; ++j)
                half[j] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(v + 64 * i + 8 * j * kRowV<DP>)));
            const u32x4 vf = {half[0][0], half[0][1], half[1][0], half[1][1]};
#pragma unroll
            for (int w = 0; w < RW; ++w) acc[w][i] = mfma<DT>(vf, p[w], acc[w][i]);
        }
    }
    template <class Stage> __device__ __forceinline__ void finish(const Stage& st, int key0, int key1) {
#pragma unroll
        for (int w = 0; w < RW; ++w) {
            sum[w] = half_sum(sum[w]);
            if (Src::kBias && base[w] == -INFINITY && sum[w] != sum[w] && !st.any_key(key0, key1)) {     // q is no number, and saw nothing
                sum[w] = 0.f;
#pragma unroll
                for (int i = 0; i < DB; ++i) acc[w][i] = f16acc{};
            }
        }
    }
};
// The lane's places in a staged tile: chunk g of row col of K; of V the four rows and 16 channels that it turns.
template <int DP> __device__ __forceinline__ int lane_k(int lane) { return k_place<DP>(lane & 31, lane >> 5); }
template <int DP> __device__ __forceinline__ int lane_v(int lane) {
    return v_place<DP>(4 * (lane >> 5) + ((lane & 15) >> 2), 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) + 8 * (lane & 1);
}

// The scales of a tile from block h0 on.
template <class Scales> struct Part {
    const Scales& all;
    const int h0;
    __device__ __forceinline__ float k(int h) const { return all.k(h0 + h); }
    __device__ __forceinline__ float lv(int h) const { return all.lv(h0 + h); }
    __device__ __forceinline__ float iv(int h) const { return all.iv(h0 + h); }
};
template <class Scales> __device__ __forceinline__ Part<Scales> part_of(const Scales& all, int h0) { return {all, h0}; }

// Which tiles of TK keys a workgroup takes.
__device__ __forceinline__ void share_of(int end, int tk, int splits, int split, int& t0, int& t1) {
    t0 = 0;
    t1 = end > 0 ? (end + tk - 1) / tk : 0;
    if (splits > 1) {
        const int share = (t1 + splits - 1) / splits;
        t0 = min(t1, split * share);
        t1 = min(t1, t0 + share);
    }
}

// Many rows: QW waves of 32 RW rows on the same keys, 32 NB at a time in two buffers: a tile is on its way into registers while the one
// before goes into LDS and the one before that is multiplied, SB blocks of 32 keys per step of the softmax.
//
// 4 * d operations a pair on the matrix pipes, one exponential a pair beside them.  2 x 1024 new tokens of 32 heads behind 7168 stored ones
// (223 GFLOP) take 274 us, 0.81 PFLOP/s where an 8192-cubed product of the vendor's library reaches 1.23; matrix pipes 41 % and vector
// pipes 51 % busy at 1.7 GHz under the power limit, and the two hardly overlap: a probe shows a product of another wave keeping vector
// instructions from issue for 11 of its 32 cycles (v_dot2 for all of them).  Head dim 64 (frame of 2025 tokens to 16200, f16, 16 heads):
// vector pipes 78 % busy, 189 us.
// Eight waves on a tile spend half the instructions on staging, conversion to f16 above all, that four do (289 us against 325), but few rows
// do not fill them; 64 keys per softmax step with one branch 285 against 289; sums of rounded pairs (v_dot2) against additions 270 and
// 284.  Not kept: scores of the next keys between the exponentials, left to the compiler (292) or held there by sched_barrier (310); two
// groups of waves half a tile apart (288 at best, 312); two row blocks a wave, which halve the reads of LDS but leave one wave a SIMD at head
// dim 128 (440) or fewer at 64 (252 against 210).
template <class Src, int DP, int RW, int QW, int NB, int SB, int OCC>
__global__ __launch_bounds__(64 * QW, OCC) void tiles_kernel(const Common a, const typename Src::Args sa) {
    constexpr int TK = 32 * NB, WR = 32 * RW, TILE_K = TK * kRowK<DP>, TILE_V = TK * kRowV<DP>;
    __shared__ __align__(16) uint8_t lds[2 * (TILE_K + TILE_V)];
    __shared__ __align__(16) float bias[Src::kBias ? 2 * TK : 4];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 5;
    int id = xcd_contiguous(blockIdx.x, gridDim.x);
    const int row_tile = id % a.row_tiles;
    id /= a.row_tiles;
    const int split = id % a.splits, problem = id / a.splits;
    const Problem pr = Src::problem(sa, a, problem);
    const int rows = pr.tokens * a.group, r0 = row_tile * (QW * WR);
    if (r0 >= rows) return;     // the whole workgroup: rows of a shorter sequence
    int t0, t1;
    share_of(min(pr.keys, pr.limit0 + (min(rows, r0 + QW * WR) - 1) / a.group), TK, a.splits, split, t0, t1);
    typename Src::template Stage<DP, TK, 64 * QW> st(sa, a, problem, pr, threadIdx.x);
    if (t0 < t1) {
        st.load_k(t0 * TK);
        st.load_v(t0 * TK);
    }
    Lanes<Src, DP, RW> L;
    L.start(a, pr, r0 + wave * WR, rows, lane);

    uint8_t *kb = lds, *vb = lds + 2 * TILE_K;                       // the tile that is multiplied
    uint8_t *kn = lds + TILE_K, *vn = lds + 2 * TILE_K + TILE_V;     // and the one behind it
    float *tb = bias, *tn = bias + (Src::kBias ? TK : 0);
    const int at_k = lane_k<DP>(lane), at_v = lane_v<DP>(lane);
    if (t0 < t1) {
        st.write_k(kb, tb);
        st.write_v(vb);
        if (t0 + 1 < t1) {
            st.load_k(t0 * TK + TK);
            st.load_v(t0 * TK + TK);
        }
        __syncthreads();
    }
    for (int t = t0; t < t1; ++t) {
        const auto all = st.scales(t * TK);
        const bool plain = st.numbers() && (t + 1) * TK <= L.all_see;
#pragma unroll
        for (int b = 0; b < NB; b += SB) {
            const auto sc = part_of(all, 2 * b);
            f16acc s[SB][RW];
            float kc[RW][2 * SB], from[RW];
            L.scores(s, kb + at_k + 32 * b * kRowK<DP>, tb + 32 * b, g);
            L.raise(s, kc, from, sc, t * TK + 32 * b, plain, st.even(), g);
            if (Src::kNormalize && __builtin_expect(!st.even(), 0)) L.add_sum(s, kc, from);
#pragma unroll
            for (int h = 0; h < 2 * SB; ++h) {
                u32x4 p[RW];
                L.probs(p, s, kc, from, sc, h);
                L.values(p, vb + at_v + (32 * b + 16 * h) * kRowV<DP>);
            }
        }
        // (behind the last tile the registers hold it still, and nothing reads where it goes)
        st.write_k(kn, tn);
        st.write_v(vn);
        if (t + 2 < t1) {
            st.load_k((t + 2) * TK);
            st.load_v((t + 2) * TK);
        }
        __syncthreads();
        uint8_t* const k = kb; kb = kn; kn = k;
        uint8_t* const v = vb; vb = vn; vn = v;
        float* const f = tb; tb = tn; tn = f;
    }
    L.finish(st, t0 * TK, min(t1 * TK, pr.keys));

    // Channels of register j of block i: 32 i + key_of(j, g).
    const int64_t part_at = ((int64_t)split * a.problems + problem) * a.rows_padded;
#pragma unroll
    for (int w = 0; w < RW; ++w) {
        const int row = r0 + wave * WR + 32 * w + (lane & 31), token = row / a.group, head = row - token * a.group;
        if (row >= rows) continue;
        if (a.splits > 1) {
            float* const pp = a.part + (part_at + row) * (DP + 2);
#pragma unroll
            for (int i = 0; i < DP / 32; ++i)
#pragma unroll
                for (int j = 0; j < 16; j += 2) *reinterpret_cast<f32x2*>(pp + 32 * i + key_of(j, g)) = f32x2{L.acc[w][i][j], L.acc[w][i][j + 1]};
            if (g == 0) *reinterpret_cast<f32x2*>(pp + DP) = f32x2{L.base[w], L.sum[w]};
            continue;
        }
        const float inv = L.sum[w] == 0.f ? 0.f : Src::kOut / L.sum[w];
        uint16_t* const op = (uint16_t*)a.o + pr.o_at + token * a.o_rs + head * a.o_hs;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i)
#pragma unroll
            for (int j = 0; j < 16; j += 8) {
                if (32 * i + 2 * j >= a.d) continue;
                uint32_t u[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = L.acc[w][i][j + 2 * e] * inv, y = L.acc[w][i][j + 2 * e + 1] * inv;
                    u[e] = a.q_dt == DT_BF16 ? pack_bf16x2(x, y) : pack_f16x2(x, y);
                }
                // of 16 channels a half wave has 0 .. 3 and 8 .. 11, or the others: each takes half from the other and has 8 in a row
                const auto s0 = __builtin_amdgcn_permlane32_swap(u[0], u[2], false, false), s1 = __builtin_amdgcn_permlane32_swap(u[1], u[3], false, false);
                const u32x4 eight = {s0[0], s1[0], s0[1], s1[1]};
                const int at = 32 * i + 2 * j + 8 * g;
                if (at >= a.d) continue;
                if (a.aligned & 2) *reinterpret_cast<u32x4*>(op + at) = eight;
                else
#pragma unroll
                    for (int e = 0; e < 8; ++e) op[at + e] = (uint16_t)(eight[e >> 1] >> 16 * (e & 1));
            }
    }
}

// Few rows, the form for single tokens: KW waves on the same 16 RT rows, each with 32 keys of its own at a time and no barrier until their
// results meet.  What counts is the keys' way in: K goes from memory straight into the fragments of v_mfma_f32_16x16x32 (lane: key
// lane % 16, channels in the order of Source::q_chunk), V through the wave's own piece of LDS, where it is turned.  Lanes hold row lane % 16 and
// keys 4 (lane / 16) .. + 3 of each 16, which is, in order, what the product with V takes, if that counts its keys so.
// 12 tokens to 16 to 32 thousand keys of 8 heads of 128 codes each: 130 us with the joining, 4.8 TB/s, where a copy reaches 5.2; in the 32 x 32 x 16
// form with K through LDS, twice the registers and half the waves, 203.  One token to 613 keys: 10 us, of which 3.5 are the second launch.
template <int DT> __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (DT == DT_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// The largest / the sum of the four lanes of a row.
__device__ __forceinline__ float quarter_max(float v) {
    const auto s = __builtin_amdgcn_permlane16_swap(f2u(v), f2u(v), false, false);
    return half_max(fmaxf(u2f(s[0]), u2f(s[1])));
}
__device__ __forceinline__ float quarter_sum(float v) {
    const auto s = __builtin_amdgcn_permlane16_swap(f2u(v), f2u(v), false, false);
    return half_sum(u2f(s[0]) + u2f(s[1]));
}

template <class Src, int DP, int KW, int RT, int OCC>
__global__ __launch_bounds__(64 * KW, OCC) void few_kernel(const Common a, const typename Src::Args sa) {
    constexpr int TK = 32, TILE = TK * kRowV<DP>, KS = DP / 32, DB = DP / 16, R = 16 * RT, DT = Src::DT;
    constexpr int MEET = R * DP * 4;      // a wave's numerators
    __shared__ __align__(16) uint8_t lds[KW * (TILE > MEET ? TILE : MEET)];
    __shared__ __align__(16) float bias[Src::kBias ? KW * TK : 4];
    __shared__ float stat[KW * 2 * R];
    const int kw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, gg = lane >> 4;
    int id = xcd_contiguous(blockIdx.x, gridDim.x);
    const int row_tile = id % a.row_tiles;
    id /= a.row_tiles;
    const int split = id % a.splits, problem = id / a.splits;
    const Problem pr = Src::problem(sa, a, problem);
    const int rows = pr.tokens * a.group, r0 = row_tile * R;
    if (r0 >= rows) return;
    int t0, t1;
    share_of(min(pr.keys, pr.limit0 + (min(rows, r0 + R) - 1) / a.group), TK, a.splits, split, t0, t1);
    {
        const int share = (t1 - t0 + KW - 1) / KW;
        t0 = min(t1, t0 + kw * share);
        t1 = min(t1, t0 + share);
    }
    typename Src::template Stage<DP, TK, 64> st(sa, a, problem, pr, lane);
    if (t0 < t1) {
        st.load_fragments(t0 * TK);
        st.load_v(t0 * TK);
    }

    int row[RT], token[RT], head[RT], limit[RT];
    u32x4 qf[RT][KS];
    float c[RT], base[RT], sum[RT];
    f32x4 acc[RT][DB];
#pragma unroll
    for (int w = 0; w < RT; ++w) {
        row[w] = r0 + 16 * w + col;
        const int r = row[w] < rows ? row[w] : rows - 1;
        token[w] = r / a.group;
        head[w] = r - token[w] * a.group;
        limit[w] = min(pr.keys, pr.limit0 + token[w]);
        c[w] = a.c;
        const uint16_t* qp = (const uint16_t*)a.q + pr.q_at + token[w] * a.q_rs + head[w] * a.q_hs;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int at = 8 * Src::q_chunk(s, gg);
            qf[w][s] = at < a.d ? load8(qp + at, a.aligned & 1) : u32x4{0, 0, 0, 0};
        }
    }
    const int all_see = min(pr.keys, pr.limit0 + min(rows - 1, r0) / a.group);
#pragma unroll
    for (int w = 0; w < RT; ++w) {
        if constexpr (Src::kNormalize) {
            float m = 0.f;
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(elem(qf[w][s], i, a.q_dt)));
            m = quarter_max(m);
            const int e = m > 0.f && m < INFINITY ? ilogbf(m) : 0;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                u32x4 f;
#pragma unroll
                for (int i = 0; i < 4; ++i) f[i] = pack_f16x2(ldexpf(elem(qf[w][s], 2 * i, a.q_dt), -e), ldexpf(elem(qf[w][s], 2 * i + 1, a.q_dt), -e)) & a.q_and ^ a.q_xor;
                qf[w][s] = f;
            }
            c[w] = ldexpf(c[w], e);
        } else {
#pragma unroll
            for (int s = 0; s < KS; ++s) qf[w][s] = qf[w][s] & a.q_and ^ a.q_xor;
        }
        base[w] = -INFINITY;
        sum[w] = 0.f;
#pragma unroll
        for (int i = 0; i < DB; ++i) acc[w][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    uint8_t* const mine = lds + kw * TILE;
    float* const my_bias = bias + (Src::kBias ? kw * TK : 0);
    const auto fence = [] {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
    const int at_v = v_place<DP>(4 * gg + (col >> 2), (col & 3) >> 1) + 8 * (col & 1);
    for (int t = t0; t < t1; ++t) {
        const auto sc = st.scales(t * TK);
        fence();
        st.write_v(mine);
        st.write_bias(my_bias);
        if (t + 1 < t1) st.load_v((t + 1) * TK);
        fence();
        f32x4 s[RT][2];
#pragma unroll
        for (int w = 0; w < RT; ++w)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                if constexpr (Src::kBias) s[w][b] = *reinterpret_cast<const f32x4*>(my_bias + 16 * b + 4 * gg);
                else s[w][b] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const u32x4 kf = st.fragment(b, ks);
#pragma unroll
                for (int w = 0; w < RT; ++w) s[w][b] = mfma16<DT>(kf, qf[w][ks], s[w][b]);
            }
        if (t + 1 < t1) st.load_fragments((t + 1) * TK);
        const bool plain = st.numbers() && (t + 1) * TK <= all_see;
        u32x4 p[RT];
#pragma unroll
        for (int w = 0; w < RT; ++w) {
            float kc[2], top = -INFINITY;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                if (!Src::kBias && !plain) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (Src::kNormalize && sc.k(b) != sc.k(b)) s[w][b][i] = NAN;
                        if (t * TK + 16 * b + 4 * gg + i >= limit[w]) s[w][b][i] = -INFINITY;
                    }
                }
                const float k = c[w] * sc.k(b);
                kc[b] = k > 1.17549435e-38f ? k : 1.17549435e-38f;
                const float m = fmaxf(fmaxf(s[w][b][0], s[w][b][1]), fmaxf(s[w][b][2], s[w][b][3]));
                top = fmaxf(top, fmaf(m, kc[b], sc.lv(b)));
                if (Src::kNormalize && __builtin_expect(!st.even(), 0)) top = fmaxf(top, fmaf(m, kc[b], kLeast));
            }
            top = quarter_max(top);
            if (__any(top > base[w] + kLag)) {
                const float nb = fmaxf(base[w], top);
                const Rebase<Src> by(base[w], nb);
                const float f = by.whole();
                base[w] = nb;
                sum[w] = by.add(0.f, sum[w]);
#pragma unroll
                for (int i = 0; i < DB; ++i) acc[w][i] *= f;
            }
            float from = base[w] == -INFINITY ? 0.f : base[w] - kShift<DT>;
            if (Src::kBias && __any(fabsf(from) > 262144.f)) {      // as in Lanes::raise
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    s[w][b] = s[w][b] * kc[b] - from;
                    kc[b] = 1.f;
                }
                from = 0.f;
            }
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                if (Src::kNormalize && __builtin_expect(!st.even(), 0)) sum[w] += sum_of<4>(s[w][b], 0, kc[b], from);      // as in Lanes::add_sum
                const float off = sc.lv(b) - from;
                float e[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) e[i] = __builtin_amdgcn_exp2f(fmaf(s[w][b][i], kc[b], off));
                p[w][2 * b] = pack2<DT>(e[0], e[1]);
                p[w][2 * b + 1] = pack2<DT>(e[2], e[3]);
                sum[w] = fmaf(Src::kNormalize ? (e[0] + e[1]) + (e[2] + e[3]) : add2<DT>(p[w][2 * b + 1], add2<DT>(p[w][2 * b], 0.f)), sc.iv(b), sum[w]);
            }
        }
#pragma unroll
        for (int i = 0; i < DB; ++i) {
            u32x2 half[2];
#pragma unroll
            for (int j = 0; j < 2; ++j)
                half[j] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(mine + at_v + 16 * j * kRowV<DP> + 32 * i)));
            const u32x4 vf = {half[0][0], half[0][1], half[1][0], half[1][1]};
#pragma unroll
            for (int w = 0; w < RT; ++w) acc[w][i] = mfma16<DT>(vf, p[w], acc[w][i]);
        }
    }
#pragma unroll
    for (int w = 0; w < RT; ++w) {
        sum[w] = quarter_sum(sum[w]);
        if (Src::kBias && base[w] == -INFINITY && sum[w] != sum[w] && !st.any_key(t0 * TK, min(t1 * TK, pr.keys))) {     // q is no number, and saw nothing
            sum[w] = 0.f;
#pragma unroll
            for (int i = 0; i < DB; ++i) acc[w][i] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }

    // register j of block i: channel 16 i + 4 gg + j
    __syncthreads();
    float* const mo = reinterpret_cast<float*>(lds + kw * MEET);
#pragma unroll
    for (int w = 0; w < RT; ++w) {
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) mo[(16 * i + 4 * gg + j) * R + 16 * w + col] = acc[w][i][j];
        if (gg == 0) {
            stat[kw * 2 * R + 16 * w + col] = base[w];
            stat[kw * 2 * R + R + 16 * w + col] = sum[w];
        }
    }
    __syncthreads();
    // a thread per row and piece of four channels
    const int64_t part_at = ((int64_t)split * a.problems + problem) * a.rows_padded;
    for (int i = threadIdx.x; i < R * (DP / 4); i += 64 * KW) {
        const int ch = 4 * (i % (DP / 4)), rr = i / (DP / 4), r = r0 + rr;
        if (r >= rows) break;
        float nb = -INFINITY, wt[KW], l = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KW; ++k) nb = fmaxf(nb, stat[k * 2 * R + rr]);
#pragma unroll
        for (int k = 0; k < KW; ++k) {
            const Rebase<Src> by(stat[k * 2 * R + rr], nb);
            wt[k] = by.whole();
            l = by.add(l, stat[k * 2 * R + R + rr]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int k = 0; k < KW; ++k) v[e] = fmaf(reinterpret_cast<const float*>(lds + k * MEET)[(ch + e) * R + rr], wt[k], v[e]);
        if (a.splits > 1) {
            float* const pp = a.part + (part_at + r) * (DP + 2);
            *reinterpret_cast<f32x2*>(pp + ch) = f32x2{v[0], v[1]};
            *reinterpret_cast<f32x2*>(pp + ch + 2) = f32x2{v[2], v[3]};
            if (ch == 0) *reinterpret_cast<f32x2*>(pp + DP) = f32x2{nb, l};
        } else if (ch < a.d) {
            const float inv = l == 0.f ? 0.f : Src::kOut / l;
            const int tk = r / a.group;
            uint16_t* const op = (uint16_t*)a.o + pr.o_at + tk * a.o_rs + (r - tk * a.group) * a.o_hs + ch;
#pragma unroll
            for (int e = 0; e < 4; ++e) op[e] = a.q_dt == DT_BF16 ? f_to_bf16(v[e] * inv) : f_to_f16(v[e] * inv);
        }
    }
}

// The parts of rows whose keys several workgroups shared, added in the order of the keys, so every call gives the same bits: a wave per row,
// first a lane per part, then DP / 64 channels a lane.  Two trips to memory: 3.5 us for a few rows, 13.7 for 4 parts of 32400 rows of 64.
template <class Src, int DP>
__global__ __launch_bounds__(256) void join_kernel(const Common a, const typename Src::Args sa, int rows_most) {
    constexpr int E = (DP + 63) / 64;      // channels of a lane
    typedef float fe __attribute__((ext_vector_type(E)));
    const int lane = threadIdx.x & 63, id = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)), problem = id / rows_most, row = id - problem * rows_most;
    if (problem >= a.problems) return;
    const Problem pr = Src::problem(sa, a, problem);
    if (row >= pr.tokens * a.group) return;
    const float* const p = a.part + ((int64_t)problem * a.rows_padded + row) * (DP + 2);
    const int64_t step = (int64_t)a.problems * a.rows_padded * (DP + 2);
    const f32x2 s = lane < a.splits ? *reinterpret_cast<const f32x2*>(p + lane * step + DP) : f32x2{-INFINITY, 0.f};
    fe x[8];      // eight parts on their way at once, the first before the weights are known
    const auto load = [&](int i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[j] = fe{};
            if (i + j < a.splits && (DP % 64 == 0 || E * lane < DP))
#pragma unroll
                for (int e = 0; e < E; ++e) x[j][e] = p[(i + j) * step + E * lane + e];
        }
    };
    load(0);
    const Rebase<Src> by(s[0], wave_max_f32(s[0]));
    const float w = by.whole(), l = (float)wave_sum_f64((double)by.add(0.f, s[1])), inv = l == 0.f ? 0.f : Src::kOut / l;
    fe v{};
    for (int i = 0; i < a.splits; i += 8) {
        if (i) load(i);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float wj = u2f(__builtin_amdgcn_readlane(f2u(w), (i + j) & 63));      // 0 behind the last part
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = fmaf(x[j][e], wj, v[e]);
        }
    }
    const int token = row / a.group, head = row - token * a.group;
    uint16_t* const op = (uint16_t*)a.o + pr.o_at + token * a.o_rs + head * a.o_hs + E * lane;
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (E * lane + e < a.d) {
            const float r = inv == 0.f ? 0.f : v[e] * inv;
            op[e] = a.q_dt == DT_BF16 ? f_to_bf16(r) : f_to_f16(r);
        }
}

// How a call runs: 16 or 32 rows with the keys over a workgroup's waves, or tiles of 128 or 256 rows; and over how many workgroups the keys of a
// row go.
struct Plan {
    int rows, row_tiles, splits;
    int blocks = 1;    // of 32 keys that a tile of 128 rows of head dims to 64 takes at a time
    int64_t bytes;     // workspace
};
// Kernels are built for these.  192 and 256 rows of 256 keep two waves a SIMD, 128 rows
// of 256 cannot (2 x 4096 x 4096 x 16 heads of 160: 444 us against 703 in those, 8 of 256: 278 against 366); 96 keeps three
// with tiles of 128 rows (2 x 4096 x 77 x 10 heads of 80: 13.7 us against 19.2 padded to 128; 2 x 4096 x 4096 x 8: 113 against 125).
inline int padded_dim(int d, int64_t rows) { return d <= 64 ? 64 : d <= 96 && rows > 32 ? 96 : d <= 128 ? 128 : d <= 192 ? 192 : 256; }
inline Plan plan_of(int tile, int splits, int64_t rows, int64_t problems, int dp) {
    Plan p;
    p.rows = tile;
    p.row_tiles = (int)((rows + tile - 1) / tile);
    p.splits = splits;
    p.bytes = splits > 1 ? 4 * splits * problems * p.row_tiles * tile * (dp + 2) : 0;
    return p;
}
// Query tokens and keys of a problem: a position some tiles past the last key, and the sum of two, stay 32-bit numbers.
constexpr int kMostLength = 1 << 30;
// A launch has fewer than 2^32 threads: workgroups of 512 at most, and rows that the join can take, four in 256.
constexpr int64_t kMostGroups = 0xffffffff / 512, kMostJoined = 0xffffffff / 256 * 4;
// bytes: of a key's or value's element.
inline Plan make_plan(int64_t rows, int64_t problems, int64_t keys, int d, int bytes) {
    const int dp = padded_dim(d, rows);
    const int64_t cus = device_cu_count();
    const auto can = [&](int64_t groups, int s) { return s == 1 || (groups * s <= kMostGroups && rows * problems <= kMostJoined); };
    if (rows <= 32) {
        // In microseconds: a workgroup starts and ends in 4; 32 keys of a wave take 1.65 at least (1 x 1369 keys x 64 heads of 72 channels in one
        // part 22.6 in all), and longer where the waves of a CU together ask for more than its share of the copy rate, 20 KB a microsecond,
        // of which CUs with few waves reach less (12 x 32749 keys x 8 heads of 128 codes: 3 parts 183, 5 parts 138, 8 parts, which are one
        // full round, 130, 16 parts 136); a wave beside others on its CU takes a little more; joining 3.  per_cu is the workgroups that share a CU in
        // this reckoning, and what registers and LDS allow but for head dims to 64, where 4 or 5 would fit (3 with 32 rows): not measured there.
        const int tile = rows <= 16 || dp >= 192 ? 16 : 32, per_cu = dp == 256 || (bytes > 1 && dp == 192) ? 1 : tile == 32 || dp == 192 || (bytes > 1 && dp == 128) ? 2 : 3;
        const int64_t slots = cus * per_cu, tiles = (keys + 31) / 32, groups = problems * ((rows + tile - 1) / tile);
        const double full = per_cu * 4 * 32. * d * 2 * bytes / 20e3;
        int best = 1;
        double least = 0.;
        for (int s = 1; s <= 64 && (s == 1 || s <= tiles) && can(groups, s); ++s) {
            const int64_t rounds = (groups * s + slots - 1) / slots, each = ((tiles + s - 1) / s + 3) / 4;
            const double busy = groups * s >= slots ? 1. : (double)(groups * s) / slots, shared = full * busy / (0.85 + 0.15 * busy), step = shared > 1.65 ? shared : 1.65;
            const int64_t in_one = (tiles + s - 1) / s;
            const double us = rounds * (4. + each * step + 0.25 * (in_one < 4 ? in_one : 4)) + (s == 1 ? 0. : 3. + 0.02 * s + 4e-6 * (dp + 2) * rows * problems * s / 2.);
            if (s == 1 || us < least) {
                least = us;
                best = s;
            }
        }
        return plan_of(tile, best, rows, problems, dp);
    }
    // In microseconds: a workgroup's start and end; 64 keys of it alone on its CU (4 x 150 x 584, 6 heads of 128: 20 in all; 2 x 512 x 800, 8 heads: 24)
    // or among as many as fit; and the joining of parts, which at 128 keys a part still pays where most CUs would idle (100 new tokens of 8 heads behind
    // 800: 16 us in parts, 31 in one; 4 x 83 x 524, 20 heads of 168: 28 and 45).
    Plan best{};
    double least = 0.;
    for (int tile = 128; tile <= (rows <= 128 ? 128 : 256); tile *= 2) {
        const bool small = tile == 128;
        const int fit = small ? (dp == 64 ? 4 : dp == 96 ? 3 : dp == 256 ? 1 : 2) : dp == 64 ? 2 : 1;
        const int64_t slots = cus * fit, groups = (rows + tile - 1) / tile * problems, tiles = (keys + 63) / 64;
        if (small && rows > 128 && groups > kMostGroups) continue;
        const double start = (small ? 7. : 13.) + (dp == 256 ? 6. : 0.);
        // (of head dims to 64, where a CU has one, with 64 keys at a time)
        const double alone = dp == 256 ? (small ? 3.7 : 4.2) : dp == 192 ? (small ? 4.2 : 3.3) : !small ? (dp == 64 ? 1.55 : dp == 96 ? 1.6 : bytes > 1 ? 1.9 : 2.2) : dp == 64 ? 1.7 : dp == 96 ? 2.1 : bytes > 1 ? 1.3 : 1.75;
        const double full = dp >= 192 || (dp > 64 && !small) ? alone : small ? 2.6 : 2.4;
        for (int s = 1; s <= 16 && (s == 1 || keys >= (int64_t)s * 128) && can(groups, s); ++s) {
            const int64_t rounds = (groups * s + slots - 1) / slots, on_one = rounds > 1 ? fit : (groups * s + cus - 1) / cus;
            const double share = full * on_one / fit, each = dp == 64 && small && on_one == 1 ? 1.2 : share > alone ? share : alone;
            const double us = rounds * (start + each * ((tiles + s - 1) / s)) + (s == 1 ? 0. : 5. + 1e-6 * 4. * (dp + 2) * rows * problems * (2 * s) / 4.);
            if (best.rows == 0 || us < least) {
                least = us;
                best = plan_of(tile, s, rows, problems, dp);
                // Two where no CU has more than one: 16 x 2048 rows, 512 keys 15.6 us against 18.5; with four on a CU the smaller tile's
                // are ahead, 120 x 8 heads of 120 rows and 1024 keys 66 against 70.
                best.blocks = groups * s <= cus && keys > 64 ? 2 : 1;
            }
        }
    }
    return best;
}

// Waves a SIMD (the last argument) are what the registers of a form allow, spilling a few at most (codes at 256 with 256 rows 40, and
// ahead all the same: 2025 rows of 8 heads of 240 to 8100, 173 us against 247 with 128 rows); blocks of 32 keys a tile follow: one where
// two would cost a workgroup its place (head dims to 64 and 96 with 128 rows: 4 and 3 on a CU; 192), two elsewhere.  At 256 with 128 rows, one wave a SIMD
// either way: 16-bit keys one at a time (4 x 638 x 6, 72 heads: 84 us against 98 with two), codes two (the last 1024 of 2 x 4096 tokens, 16 over 4 heads: 235 against 251).
template <class Src, int DP> inline int launch(const Plan& p, int64_t rows, Common& a, const typename Src::Args& sa, hipStream_t stream) {
    const int64_t grid = (int64_t)p.row_tiles * a.problems * p.splits;
    if (grid > kMostGroups) return -1;
    if constexpr (DP == 96) {
        if (p.rows == 128) tiles_kernel<Src, DP, 1, 4, 1, 1, 3><<<(int)grid, 256, 0, stream>>>(a, sa);
        else tiles_kernel<Src, DP, 1, 8, 2, 2, 2><<<(int)grid, 512, 0, stream>>>(a, sa);
    } else if (p.rows == 16) few_kernel<Src, DP, 4, 1, DP == 256 ? 1 : DP == 192 ? (Src::kNormalize ? 2 : 1) : Src::kNormalize || DP == 64 ? 3 : 2><<<(int)grid, 256, 0, stream>>>(a, sa);
    else if constexpr (DP == 256) {
        if (p.rows == 128) tiles_kernel<Src, DP, 1, 4, Src::kNormalize ? 2 : 1, 1, 1><<<(int)grid, 256, 0, stream>>>(a, sa);
        else tiles_kernel<Src, DP, 1, 8, 1, 1, 2><<<(int)grid, 512, 0, stream>>>(a, sa);
    }
    else if constexpr (DP == 192) {
        if (p.rows == 128) tiles_kernel<Src, DP, 1, 4, 1, 1, 2><<<(int)grid, 256, 0, stream>>>(a, sa);
        else tiles_kernel<Src, DP, 1, 8, 2, 1, 2><<<(int)grid, 512, 0, stream>>>(a, sa);
    } else if (p.rows == 32) few_kernel<Src, DP, 4, 2, 2><<<(int)grid, 256, 0, stream>>>(a, sa);
    else if constexpr (DP == 128) {
        if (p.rows == 128) tiles_kernel<Src, DP, 1, 4, 2, 2, 2><<<(int)grid, 256, 0, stream>>>(a, sa);
        else tiles_kernel<Src, DP, 1, 8, 2, 2, 2><<<(int)grid, 512, 0, stream>>>(a, sa);
    } else {
        if (p.rows == 128 && p.blocks == 1) tiles_kernel<Src, DP, 1, 4, 1, 1, 4><<<(int)grid, 256, 0, stream>>>(a, sa);
        else if (p.rows == 128) tiles_kernel<Src, DP, 1, 4, 2, 2, 3><<<(int)grid, 256, 0, stream>>>(a, sa);
        else tiles_kernel<Src, DP, 1, 8, 2, 1, 4><<<(int)grid, 512, 0, stream>>>(a, sa);
    }
    KCHECK();
    if (p.splits > 1) {
        join_kernel<Src, DP><<<(int)((a.problems * rows + 3) / 4), 256, 0, stream>>>(a, sa, (int)rows);
        KCHECK();
    }
    return 0;
}
template <class Src> inline int launch_dim(const Plan& p, int64_t rows, Common& a, const typename Src::Args& sa, hipStream_t stream) {
    switch (padded_dim(a.d, rows)) {
        case 64: return launch<Src, 64>(p, rows, a, sa, stream);
        case 96: return launch<Src, 96>(p, rows, a, sa, stream);
        case 128: return launch<Src, 128>(p, rows, a, sa, stream);
        case 192: return launch<Src, 192>(p, rows, a, sa, stream);
        default: return launch<Src, 256>(p, rows, a, sa, stream);
    }
}

}  // namespace states
