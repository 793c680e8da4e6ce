// Attention over whole prompts, packed one behind the other: 16-bit queries, keys and values, causal or not, query heads that share key-value
// heads.  The arithmetic is attn_states.hpp's: one pass over the keys with a running base and sum, 32 rows a wave, products of 32 x 32 x 16.
#include "attn_states.hpp"

namespace {

using namespace states;

struct PackedArgs {
    const uint16_t *k, *v;
    int64_t k_rs, k_hs, v_rs, v_hs;
    const int32_t* starts;
    int n, tokens, aligned, causal;
};

template <int DTYPE> struct Packed {
    typedef PackedArgs Args;
    static constexpr int DT = DTYPE;
    static constexpr bool kBias = false, kNormalize = false;
    static constexpr float kOut = 1.f;
    struct Scales {
        __device__ float k(int) const { return 1.f; }
        __device__ float lv(int) const { return 0.f; }
        __device__ float iv(int) const { return 1.f; }
    };
    // Keys and values of a prompt's key-value head, TK rows at a time through NT threads' registers into LDS.
    template <int DP, int TK, int NT> struct Stage {
        static constexpr int ROW = DP == 192 ? 32 : DP == 96 ? 16 : DP / 8, CH = (TK * ROW + NT - 1) / NT;      // a power of two threads to a row
        static constexpr bool kAll = TK * ROW % NT == 0;
        static_assert(NT % ROW == 0 && (kAll || CH == 1), "a thread's pieces are of one chunk");
        const uint16_t *k, *v;
        int64_t k_rs, v_rs;
        int tid, keys, d;
        bool aligned;
        u32x4 kr[CH], vr[CH];
        __device__ Stage(const Args& a, int d_, int64_t first, int head, int keys_, int tid_)
            : k(a.k + first * a.k_rs + head * a.k_hs), v(a.v + first * a.v_rs + head * a.v_hs), k_rs(a.k_rs), v_rs(a.v_rs), tid(tid_), keys(keys_), d(d_), aligned(a.aligned) {
#pragma unroll
            for (int j = 0; j < CH; ++j) kr[j] = vr[j] = u32x4{0, 0, 0, 0};
        }
        __device__ __forceinline__ bool mine() const { return kAll || tid < TK * ROW; }
        // rows from key0 on; past the end and behind the head dim zeros
        __device__ __forceinline__ void rows(u32x4 (&x)[CH], const uint16_t* p, int64_t rs, int key0) {
            if (!mine()) return;
            if (aligned && key0 + TK <= keys) {     // a scalar base and 32-bit offsets
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
                    x[j] = key < keys && 8 * ch < d ? load8(p + key * rs + 8 * ch, aligned) : u32x4{0, 0, 0, 0};
                }
            }
        }
        __device__ __forceinline__ void load(int key0) {
            rows(kr, k, k_rs, key0);
            rows(vr, v, v_rs, key0);
        }
        // What some row does not see must be a number in V, or 0 times it would be none: `edge` tiles take 0 for those that are not, and the
        // end of the kernel puts NaN where they count.
        __device__ __forceinline__ bool clean() {
            constexpr uint32_t E = DT == DT_BF16 ? 0x7f80u : 0x7c00u;
            bool found = false;
#pragma unroll
            for (int j = 0; j < CH; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t w = vr[j][e];
                    const bool lo = (w & E) == E, hi = (w >> 16 & E) == E;
                    found |= lo | hi;
                    vr[j][e] = w & ((lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u));
                }
            return found;
        }
        __device__ __forceinline__ void write(uint8_t* kb, uint8_t* vb) {
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const int i = tid + j * NT;
                if (!mine() || i % ROW >= DP / 8) continue;
                *reinterpret_cast<u32x4*>(kb + k_place<DP>(i / ROW, i % ROW)) = kr[j];
                *reinterpret_cast<u32x4*>(vb + v_place<DP>(i / ROW, i % ROW)) = vr[j];
            }
        }
        __device__ bool any_key(int, int) const { return true; }
    };
};

// Which prompt the tile `slot` of a key-value head's row tiles lies in: a wave counts the tiles of 64 prompts at a time.  `starts` is device data
// that the host has not seen: everything from it is brought into 0 .. tokens.
struct Place {
    int first, count, tile;      // the prompt's tokens; its row tile, the last one first: those have the most keys
};
__device__ __forceinline__ bool find(const PackedArgs& a, int group, int tile_rows, int slot, Place& p) {
    const int lane = threadIdx.x & 63;
    for (int s0 = 0; s0 < a.n; s0 += 64) {
        const int s = s0 + lane;
        int first = 0, count = 0;
        if (s < a.n) {
            first = min(max(a.starts[s], 0), a.tokens);
            count = min(max(a.starts[s + 1], first), a.tokens) - first;
        }
        const int tiles = (count * group + tile_rows - 1) / tile_rows;
        int upto = tiles;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int o = __shfl_up(upto, d);
            if (lane >= d) upto += o;
        }
        const uint64_t behind = __ballot(upto > slot);
        if (behind) {
            const int l = __builtin_amdgcn_readfirstlane(__builtin_ctzll(behind));
            p.first = __builtin_amdgcn_readlane(first, l);
            p.count = __builtin_amdgcn_readlane(count, l);
            p.tile = __builtin_amdgcn_readlane(upto, l) - slot - 1;
            return true;
        }
        slot -= __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// QW waves of 32 rows on the same keys, 32 NB at a time in two LDS buffers: a tile is on its way into registers while the one before goes into
// LDS and the one before that is multiplied, SB blocks of 32 keys per step of the softmax.
template <class Src, int DP, int QW, int NB, int SB, int OCC>
__global__ __launch_bounds__(64 * QW, OCC) void prompt_kernel(const Common a, const PackedArgs sa) {
    constexpr int TK = 32 * NB, TILE_K = TK * kRowK<DP>, TILE_V = TK * kRowV<DP>;
    __shared__ __align__(16) uint8_t lds[2 * (TILE_K + TILE_V)];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 5;
    // workgroups are dealt to the XCDs in turn: each has its own heads where their number allows, and as many long tiles as the others
    const int slot = blockIdx.x / a.hk, head = blockIdx.x - slot * a.hk;
    Place at;
    if (!find(sa, a.group, 32 * QW, slot, at)) return;
    Problem pr;
    pr.q_at = at.first * a.q_rs + head * a.group * a.q_hs;
    pr.o_at = at.first * a.o_rs + head * a.group * a.o_hs;
    pr.tokens = pr.keys = at.count;
    pr.limit0 = sa.causal ? 1 : at.count;
    const int rows = pr.tokens * a.group, r0 = at.tile * 32 * QW, wr = r0 + 32 * wave;
    const int end = min(pr.keys, pr.limit0 + (min(rows, r0 + 32 * QW) - 1) / a.group), t1 = (end + TK - 1) / TK;
    const int sees = min(pr.keys, pr.limit0 + (min(rows, wr + 32) - 1) / a.group), t_mine = wr < rows ? (sees + TK - 1) / TK : 0;      // of this wave's rows
    typename Src::template Stage<DP, TK, 64 * QW> st(sa, a.d, at.first, head, pr.keys, threadIdx.x);
    st.load(0);
    Lanes<Src, DP, 1> L;
    L.start(a, pr, wr, rows, lane);
    uint8_t *kb = lds, *vb = lds + 2 * TILE_K;                       // the tile that is multiplied
    uint8_t *kn = lds + TILE_K, *vn = lds + 2 * TILE_K + TILE_V;     // and the one behind it
    const int at_k = lane_k<DP>(lane), at_v = lane_v<DP>(lane);
    const int edge = min(pr.keys, pr.limit0 + r0 / a.group) / TK;      // tiles before this one are seen whole by every row
    bool found = false;
    if (edge == 0) found |= st.clean();
    st.write(kb, vb);
    if (1 < t1) st.load(TK);
    __syncthreads();
    const typename Src::Scales sc{};
    const auto next = [&](int t) {
        // (behind the last tile the registers hold it still, and nothing reads where it goes)
        if (t + 1 >= edge) found |= st.clean();
        st.write(kn, vn);
        if (t + 2 < t1) st.load((t + 2) * TK);
        __syncthreads();
        uint8_t* const k = kb; kb = kn; kn = k;
        uint8_t* const v = vb; vb = vn; vn = v;
    };
    for (int t = 0; t < t_mine; ++t) {
        const bool plain = (t + 1) * TK <= L.all_see;
#pragma unroll
        for (int b = 0; b < NB; b += SB) {
            f16acc s[SB][1];
            float kc[1][2 * SB], from[1];
            L.scores(s, kb + at_k + 32 * b * kRowK<DP>, (const float*)nullptr, g);
            L.raise(s, kc, from, sc, t * TK + 32 * b, plain, true, g);
#pragma unroll
            for (int h = 0; h < 2 * SB; ++h) {
                u32x4 p[1];
                L.probs(p, s, kc, from, sc, h);
                L.values(p, vb + at_v + (32 * b + 16 * h) * kRowV<DP>);
            }
        }
        next(t);
    }
    for (int t = t_mine; t < t1; ++t) next(t);      // tiles that only other waves' rows see (in a loop of its own: a branch around the products costs registers)
    L.finish(st, 0, end);

    // Channels of register j of block i: 32 i + key_of(j, g).
    const int row = wr + (lane & 31), token = row / a.group, h = row - token * a.group;
    uint16_t* const op = (uint16_t*)a.o + pr.o_at + token * a.o_rs + h * a.o_hs;
    if (row < rows) {
        const float inv = L.sum[0] == 0.f ? 0.f : 1.f / L.sum[0];
#pragma unroll
        for (int i = 0; i < DP / 32; ++i)
#pragma unroll
            for (int j = 0; j < 16; j += 8) {
                if (32 * i + 2 * j >= a.d) continue;
                uint32_t u[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = L.acc[0][i][j + 2 * e] * inv, y = L.acc[0][i][j + 2 * e + 1] * inv;
                    u[e] = Src::DT == DT_BF16 ? pack_bf16x2(x, y) : pack_f16x2(x, y);
                }
                // of 16 channels a half wave has 0 .. 3 and 8 .. 11, or the others: each takes half from the other and has 8 in a row
                const auto s0 = __builtin_amdgcn_permlane32_swap(u[0], u[2], false, false), s1 = __builtin_amdgcn_permlane32_swap(u[1], u[3], false, false);
                const u32x4 eight = {s0[0], s1[0], s0[1], s1[1]};
                const int c = 32 * i + 2 * j + 8 * g;
                if (c >= a.d) continue;
                if (a.aligned & 2) *reinterpret_cast<u32x4*>(op + c) = eight;
                else
#pragma unroll
                    for (int e = 0; e < 8; ++e) op[c + e] = (uint16_t)(eight[e >> 1] >> 16 * (e & 1));
            }
    }
    if (__syncthreads_or(found)) {
        __threadfence();
        if (row < rows)
#pragma unroll 1
            for (int key = edge * TK; key < L.limit[0]; ++key)
#pragma unroll 1
                for (int c = g; c < a.d; c += 2)
                    if (!(fabsf(elem(u32x4{st.v[key * st.v_rs + c], 0, 0, 0}, 0, Src::DT)) < INFINITY)) op[c] = 0x7fff;      // (NaN in both types)
    }
}

// Rows of a workgroup.  (Row tiles of a head: all rows' and a partial one for each prompt.)
inline int64_t tiles_of(int64_t rows, int n, int tile) { return rows / tile + n; }

template <class Src, int DP> int launch(Common& a, const PackedArgs& sa, int tile, hipStream_t st) {
    const int64_t grid = tiles_of((int64_t)sa.tokens * a.group, sa.n, tile) * a.hk;
    if (grid > kMostGroups) return -1;
    if (tile == 256) {
        if constexpr (DP == 64) prompt_kernel<Src, DP, 8, 2, 1, 4><<<(int)grid, 512, 0, st>>>(a, sa);
        else if constexpr (DP == 192) prompt_kernel<Src, DP, 8, 2, 1, 2><<<(int)grid, 512, 0, st>>>(a, sa);
        else if constexpr (DP == 256) prompt_kernel<Src, DP, 8, 1, 1, 2><<<(int)grid, 512, 0, st>>>(a, sa);
        else prompt_kernel<Src, DP, 8, 2, 2, 2><<<(int)grid, 512, 0, st>>>(a, sa);
    } else {
        if constexpr (DP == 64) prompt_kernel<Src, DP, 4, 1, 1, 4><<<(int)grid, 256, 0, st>>>(a, sa);
        else if constexpr (DP == 96) prompt_kernel<Src, DP, 4, 1, 1, 3><<<(int)grid, 256, 0, st>>>(a, sa);
        else if constexpr (DP == 128) prompt_kernel<Src, DP, 4, 2, 2, 2><<<(int)grid, 256, 0, st>>>(a, sa);
        else if constexpr (DP == 192) prompt_kernel<Src, DP, 4, 1, 1, 2><<<(int)grid, 256, 0, st>>>(a, sa);
        else prompt_kernel<Src, DP, 4, 1, 1, 1><<<(int)grid, 256, 0, st>>>(a, sa);
    }
    KCHECK();
    return 0;
}
template <class Src> int launch_dim(Common& a, const PackedArgs& sa, hipStream_t st) {
    const int tile = tiles_of((int64_t)sa.tokens * a.group, sa.n, 256) * a.hk >= 2 * device_cu_count() ? 256 : 128;
    switch (padded_dim(a.d, 64)) {
        case 64: return launch<Src, 64>(a, sa, tile, st);
        case 96: return launch<Src, 96>(a, sa, tile, st);
        case 128: return launch<Src, 128>(a, sa, tile, st);
        case 192: return launch<Src, 192>(a, sa, tile, st);
        default: return launch<Src, 256>(a, sa, tile, st);
    }
}

}  // namespace

GPU_API int gpu_prompt_attn(int dtype, const void* q, int64_t q_rs, int64_t q_hs, const void* k, int64_t k_rs, int64_t k_hs, const void* v,
                            int64_t v_rs, int64_t v_hs, void* o, int64_t o_rs, int64_t o_hs, const int32_t* starts, int n, int tokens, int h,
                            int hk, int head_dim, float scale, int causal, void* stream) {
    if (dtype != DT_F16 && dtype != DT_BF16) return -4;
    if (n < 0 || tokens < 0 || tokens > kMostLength || h <= 0 || hk <= 0 || h % hk != 0 || head_dim <= 0 || head_dim > 256 || head_dim % 8 != 0 || !(fabsf(scale) < INFINITY)) return -1;
    if (n == 0 || tokens == 0) return 0;
    if (!q || !k || !v || !o || !starts || (uintptr_t)starts % 4 != 0 || (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o) & 1)) return -1;
    if ((int64_t)tokens * (h / hk) > 0x7ffff000) return -1;
    const auto sixteen = [](const void* at, int64_t s0, int64_t s1) { return (uintptr_t)at % 16 == 0 && (s0 | s1) % 8 == 0; };
    Common c{};
    c.q = q; c.o = o; c.q_rs = q_rs; c.q_hs = q_hs; c.o_rs = o_rs; c.o_hs = o_hs;
    c.hk = hk; c.group = h / hk; c.d = head_dim; c.q_dt = dtype;
    c.aligned = (sixteen(q, q_rs, q_hs) ? 1 : 0) | (sixteen(o, o_rs, o_hs) ? 2 : 0);
    set_scale(c, scale, 1.17549435e-38f);
    PackedArgs s{};
    s.k = (const uint16_t*)k; s.v = (const uint16_t*)v;
    s.k_rs = k_rs; s.k_hs = k_hs; s.v_rs = v_rs; s.v_hs = v_hs;
    // (and rows of a tile within 32-bit offsets of its first)
    const bool near = k_rs >= 0 && v_rs >= 0 && k_rs < (1 << 23) && v_rs < (1 << 23);
    s.starts = starts; s.n = n; s.tokens = tokens; s.causal = causal != 0;
    s.aligned = near && sixteen(k, k_rs, k_hs) && sixteen(v, v_rs, v_hs);
    return dtype == DT_BF16 ? launch_dim<Packed<DT_BF16>>(c, s, (hipStream_t)stream) : launch_dim<Packed<DT_F16>>(c, s, (hipStream_t)stream);
}
