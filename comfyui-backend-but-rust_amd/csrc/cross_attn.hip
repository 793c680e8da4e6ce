// Cross attention to an encoder's states: 16-bit keys and values of another length, named per batch item, with a mask or a bias per key.
#include "attn_states.hpp"

#include <float.h>
#include <string.h>

namespace {

using namespace states;

struct CrossArgs {
    const uint16_t *k, *v;
    int64_t q_bs, o_bs, k_bs, k_rs, k_hs, v_bs, v_rs, v_hs;
    int lq, lk, aligned;
    uint32_t near_bits;     // (this and far_step stand where the block has room: with 12 bytes more of it 4 x 16 single queries took 12.8 us for 12.5)
    const int32_t* k_lens;
    const void* mask;
    int mask_kind;          // 1: bytes, 0 = out; 2: f32, added to the logits
    uint32_t far_step;
    int64_t mask_bs;
    float per_score, near;  // a bias in units of the score, and the magnitude there from which on (a bias of near_bits) a step of its bits is
                            // far_step / 2^32 of a score's
};

// What a key's mask holds, and what that adds to its score: -inf takes the key out.  A finite bias stays finite, so that the type's lowest
// value is what it is in the formula: a logit like any other.  Biases too large for units of the score, or for units of log2 afterwards, keep their
// order: those from `near` on, a quarter of what has room, share that in steps of their bits.  Any two logits of that size that are
// not the same lie further apart than exp reaches, so what is left to tell is which is the larger.
__device__ __forceinline__ uint32_t mask_word(const CrossArgs& a, const void* mask, int key) {
    return a.mask_kind == 1 ? ((const uint8_t*)mask)[key] : ((const uint32_t*)mask)[key];
}
__device__ __forceinline__ bool is_out(const CrossArgs& a, uint32_t w) { return w == (a.mask_kind == 1 ? 0u : 0xff800000u); }
__device__ __forceinline__ float key_bias(const CrossArgs& a, uint32_t w) {
    if (a.mask_kind == 1) return w ? 0.f : -INFINITY;
    const float b = u2f(w), x = b * a.per_score;
    if (fabsf(x) < a.near || !(fabsf(b) < INFINITY)) return x;
    const uint32_t bits = f2u(fabsf(b)), above = bits > a.near_bits ? bits - a.near_bits : 0u;
    return copysignf(u2f(f2u(a.near) + __umulhi(above, a.far_step)), b);
}

template <int DTYPE, bool BIAS> struct Dense {
    typedef CrossArgs Args;
    static constexpr int DT = DTYPE;
    static constexpr bool kBias = BIAS, kNormalize = false;
    static constexpr float kOut = 1.f;
    struct Scales {
        __device__ float k(int) const { return 1.f; }
        __device__ float lv(int) const { return 0.f; }
        __device__ float iv(int) const { return 1.f; }
    };
    static __device__ __forceinline__ Problem problem(const Args& a, const Common& c, int id) {
        const int b = id / c.hk, head = id - b * c.hk;
        Problem p;
        p.q_at = b * a.q_bs + head * c.group * c.q_hs;
        p.o_at = b * a.o_bs + head * c.group * c.o_hs;
        p.tokens = a.lq;
        p.keys = a.k_lens ? min(max(a.k_lens[b], 0), a.lk) : a.lk;
        p.limit0 = p.keys;
        return p;
    }
    // the chunk of 8 channels that step s of the product of few rows takes from lanes 16 gg ..
    static __device__ __forceinline__ int q_chunk(int s, int gg) { return 4 * s + gg; }
    template <int DP, int TK, int NT> struct Stage {
        static constexpr int ROW = DP == 192 ? 32 : DP == 96 ? 16 : DP / 8, CH = (TK * ROW + NT - 1) / NT;      // a power of two threads to a row
        static constexpr bool kAll = TK * ROW % NT == 0;      // every thread has a piece of every load
        static_assert(kAll || (CH == 1 && TK <= NT), "some threads are without a piece");
        __device__ __forceinline__ bool mine() const { return kAll || tid < TK * ROW; }
        const Args& a;
        const uint16_t *k, *v;
        const void* mask;
        int tid, keys, d;
        u32x4 kr[CH], vr[CH];      // (for few rows kr are the fragments, [16 keys][step])
        uint32_t k_mask[BIAS ? CH : 1], v_mask[BIAS ? CH : 1], row_mask;     // as they lie in memory: looked at when they have arrived
        int row_key;
        __device__ Stage(const Args& a_, const Common& c, int id, const Problem& p, int tid_) : a(a_), tid(tid_), keys(p.keys), d(c.d) {
            const int b = id / c.hk, head = id - b * c.hk;
            k = a.k + b * a.k_bs + head * a.k_hs;
            v = a.v + b * a.v_bs + head * a.v_hs;
#pragma unroll
            for (int j = 0; j < CH; ++j) kr[j] = vr[j] = u32x4{0, 0, 0, 0};
            mask = a.mask_kind == 1 ? (const void*)((const uint8_t*)a.mask + b * a.mask_bs) : (const void*)((const float*)a.mask + b * a.mask_bs);
        }
        // rows from key0 on into registers, and what their keys' masks say; past the end zeros
        __device__ __forceinline__ void rows(u32x4 (&x)[CH], const uint16_t* p, int64_t rs, int key0) {
            if (!mine()) return;
            static_assert(NT % ROW == 0, "a thread's pieces are of one chunk");
            if (a.aligned && key0 + TK <= keys) {     // 16-byte pieces: a scalar base and 32-bit offsets; behind the head dim they stay 0
                const char* const at = (const char*)(p + (int64_t)key0 * rs);
                if (8 * (tid % ROW) < d)
#pragma unroll
                for (int j = 0; j < CH; ++j) {
                    const int i = tid + j * NT;
                    x[j] = *reinterpret_cast<const u32x4*>(at + (uint32_t)(2 * (i / ROW * (int)rs + 8 * (i % ROW))));
                }
            } else {
#pragma unroll
                for (int j = 0; j < CH; ++j) {
                    const int i = tid + j * NT, key = key0 + i / ROW, ch = i % ROW;
                    x[j] = key < keys && 8 * ch < d ? load8(p + key * rs + 8 * ch, a.aligned) : u32x4{0, 0, 0, 0};
                }
            }
        }
        __device__ __forceinline__ void load_k(int key0) {
            rows(kr, k, a.k_rs, key0);
            if (BIAS && mine())
#pragma unroll
                for (int j = 0; j < CH; ++j) {
                    const int key = key0 + (tid + j * NT) / ROW;
                    k_mask[j] = key < keys ? mask_word(a, mask, key) : 1u;
                }
            if (BIAS && tid < TK) {
                row_key = key0 + tid;
                row_mask = row_key < keys ? mask_word(a, mask, row_key) : 1u;
            }
        }
        __device__ __forceinline__ void load_fragments(int key0) {
            static_assert(NT != 64 || CH >= 2 * (DP / 32), "32 keys of a wave");
            const int col = tid & 15, gg = tid >> 4;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int key = key0 + 16 * b + col;
                const uint16_t* const at = k + (key < keys ? key : 0) * a.k_rs + 8 * gg;
                if (a.aligned) {
#pragma unroll
                    for (int s = 0; s < DP / 32; ++s)
                        if (32 * s + 8 * gg < d) kr[b * (DP / 32) + s] = load8(at + 32 * s, true);
                } else {
#pragma unroll
                    for (int s = 0; s < DP / 32; ++s) if (32 * s + 8 * gg < d) kr[b * (DP / 32) + s] = load8(at + 32 * s, false);
                }
                if (BIAS) k_mask[b] = key < keys ? mask_word(a, mask, key) : a.mask_kind == 1 ? 0u : 0xff800000u;     // past the end: out
            }
            if (BIAS && tid < TK) {
                row_key = key0 + tid;
                row_mask = row_key < keys ? mask_word(a, mask, row_key) : 1u;
            }
        }
        __device__ __forceinline__ u32x4 fragment(int b, int s) const { return BIAS && is_out(a, k_mask[b]) ? u32x4{0, 0, 0, 0} : kr[b * (DP / 32) + s]; }
        __device__ __forceinline__ void write_bias(float* bias) {
            if (BIAS && tid < TK) bias[tid] = row_key < keys ? key_bias(a, row_mask) : -INFINITY;
        }
        __device__ __forceinline__ void load_v(int key0) {
            rows(vr, v, a.v_rs, key0);
            if (BIAS) {
                if (mine())
#pragma unroll
                for (int j = 0; j < CH; ++j) {
                    const int key = key0 + (tid + j * NT) / ROW;
                    v_mask[j] = key < keys ? mask_word(a, mask, key) : 1u;
                }
            }
        }
        // a key that is out has probability 0, and its value must be a number for the product to leave it out, its score for the bias to
        __device__ __forceinline__ void write_k(uint8_t* kb, float* bias) {
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const int i = tid + j * NT;
                if (mine() && i % ROW < DP / 8) *reinterpret_cast<u32x4*>(kb + k_place<DP>(i / ROW, i % ROW)) = BIAS && is_out(a, k_mask[j]) ? u32x4{0, 0, 0, 0} : kr[j];
            }
            if (BIAS && tid < TK) bias[tid] = row_key < keys ? key_bias(a, row_mask) : -INFINITY;
        }
        __device__ __forceinline__ void write_v(uint8_t* vb) {
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const int i = tid + j * NT;
                if (mine() && i % ROW < DP / 8) *reinterpret_cast<u32x4*>(vb + v_place<DP>(i / ROW, i % ROW)) = BIAS && is_out(a, v_mask[j]) ? u32x4{0, 0, 0, 0} : vr[j];
            }
        }
        __device__ __forceinline__ bool any_key(int from, int to) const {
            for (int i = from; i < to; ++i)
                if (!is_out(a, mask_word(a, mask, i))) return true;
            return false;
        }
        __device__ __forceinline__ bool numbers() const { return true; }
        __device__ __forceinline__ bool even() const { return true; }
        __device__ __forceinline__ Scales scales(int) const { return {}; }
    };
};

}  // namespace

GPU_API int64_t gpu_cross_attn_workspace(int b, int lq, int lk, int h, int hk, int head_dim) {
    if (b <= 0 || lq <= 0 || lk <= 0 || h <= 0 || hk <= 0 || h % hk != 0 || head_dim <= 0 || head_dim > 256) return 0;
    return make_plan((int64_t)lq * (h / hk), (int64_t)b * hk, lk, head_dim, 2).bytes;
}

GPU_API int gpu_cross_attn(int dtype, const void* q, const void* k, const void* v, void* o, void* ws, int b, int lq, int lk, int h, int hk,
                           int head_dim, int64_t q_bs, int64_t q_rs, int64_t q_hs, int64_t k_bs, int64_t k_rs, int64_t k_hs, int64_t v_bs,
                           int64_t v_rs, int64_t v_hs, int64_t o_bs, int64_t o_rs, int64_t o_hs, float scale, const int32_t* k_lens,
                           const void* mask, int mask_kind, int64_t mask_bs, void* stream) {
    if (dtype != DT_F16 && dtype != DT_BF16) return -4;
    if (b < 0 || lq < 0 || lk < 0 || h <= 0 || hk <= 0 || h % hk != 0 || head_dim <= 0 || head_dim > 256 || head_dim % 8 != 0) return -1;
    if (lq > kMostLength || lk > kMostLength) return -1;
    if (mask_kind < 0 || mask_kind > 2 || (mask_kind != 0 && !mask && lk > 0) || !(fabsf(scale) < INFINITY)) return -1;
    if (b == 0 || lq == 0) return 0;
    if ((int64_t)lq * (h / hk) > 0x7ffff000 || (int64_t)b * hk > 0x7fffffff || !q || !o || (lk > 0 && (!k || !v))) return -1;
    const Plan p = make_plan((int64_t)lq * (h / hk), (int64_t)b * hk, lk, head_dim, 2);
    if (p.bytes && (!ws || (uintptr_t)ws % 16 != 0)) return -1;
    const auto sixteen = [](const void* at, int64_t s0, int64_t s1, int64_t s2) { return (uintptr_t)at % 16 == 0 && (s0 | s1 | s2) % 8 == 0; };
    Common c{};
    c.q = q; c.o = o; c.q_rs = q_rs; c.q_hs = q_hs; c.o_rs = o_rs; c.o_hs = o_hs;
    c.hk = hk; c.group = h / hk; c.d = head_dim; c.q_dt = dtype;
    c.row_tiles = p.row_tiles; c.problems = b * hk; c.splits = p.splits; c.rows_padded = p.row_tiles * p.rows;
    c.aligned = (sixteen(q, q_bs, q_rs, q_hs) ? 1 : 0) | (sixteen(o, o_bs, o_rs, o_hs) ? 2 : 0);
    // with a bias, which is counted in units of the score, scales from which it would leave fp32 are none
    set_scale(c, scale, mask_kind == 2 ? 1e-30f : 1.17549435e-38f);
    c.part = (float*)ws;
    CrossArgs s{};
    s.per_score = (float)(1.4426950408889634 / c.c);
    const float most = 3e38f / (c.c > 1.f ? c.c : 1.f);
    s.near = 0.25f * most;
    const auto bits = [](float x) { uint32_t u; memcpy(&u, &x, 4); return u; };
    s.near_bits = bits(s.near / s.per_score);
    s.far_step = (uint32_t)(((uint64_t)(bits(most) - bits(s.near)) << 32) / (bits(FLT_MAX) - s.near_bits));
    s.k = (const uint16_t*)k; s.v = (const uint16_t*)v;
    s.q_bs = q_bs; s.o_bs = o_bs; s.k_bs = k_bs; s.k_rs = k_rs; s.k_hs = k_hs; s.v_bs = v_bs; s.v_rs = v_rs; s.v_hs = v_hs;
    // (and rows of a tile within 32-bit offsets of its first)
    const bool near = k_rs < (1 << 23) && v_rs < (1 << 23) && k_rs >= 0 && v_rs >= 0;
    s.lq = lq; s.lk = lk; s.aligned = near && sixteen(k, k_bs, k_rs, k_hs) && sixteen(v, v_bs, v_rs, v_hs);
    s.k_lens = k_lens; s.mask = mask; s.mask_kind = mask_kind; s.mask_bs = mask_bs;
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == DT_BF16) return mask_kind ? launch_dim<Dense<DT_BF16, true>>(p, (int64_t)lq * (h / hk), c, s, st) : launch_dim<Dense<DT_BF16, false>>(p, (int64_t)lq * (h / hk), c, s, st);
    return mask_kind ? launch_dim<Dense<DT_F16, true>>(p, (int64_t)lq * (h / hk), c, s, st) : launch_dim<Dense<DT_F16, false>>(p, (int64_t)lq * (h / hk), c, s, st);
}

GPU_API int gpu_internal_states_plan(int64_t rows, int64_t problems, int64_t keys, int head_dim, int bytes, int32_t* out) {
    if (rows <= 0 || problems <= 0 || keys < 0 || head_dim <= 0 || head_dim > 256 || (bytes != 1 && bytes != 2) || !out || (bytes == 2 && keys > kMostLength)) return -1;
    const Plan p = make_plan(rows, problems, keys, head_dim, bytes);
    if (p.row_tiles * problems * p.splits > kMostGroups) return -1;
    out[0] = p.rows;
    out[1] = p.splits;
    out[2] = padded_dim(head_dim, rows) == 64 && p.rows == 128 ? p.blocks : 0;
    return 0;
}
