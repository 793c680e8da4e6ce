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
// that the host has not seen: everything from it is brought into 0 .. tokens, and one that is below an earlier one counts as that one, so that no
// row belongs to two prompts, whose workgroups would both write it, and the tiles are no more than the launch has.
struct Place {
    int first, count, tile;      // the prompt's tokens; its row tile, the last one first: those have the most keys
};
__device__ __forceinline__ bool find(const PackedArgs& a, int group, int tile_rows, int slot, Place& p) {
    const int lane = threadIdx.x & 63;
    int high = 0;      // the largest of the starts before
    for (int s0 = 0; s0 < a.n; s0 += 64) {
        const int s = s0 + lane;
        int first = 0, end = 0;
        if (s < a.n) {
            first = min(max(a.starts[s], 0), a.tokens);
            end = min(max(a.starts[s + 1], 0), a.tokens);
        }
        if (__any(s < a.n && (first < high || end < first))) {
            first = max(first, high);
#pragma unroll
            for (int d = 1; d < 64; d *= 2) first = max(first, __shfl_up(first, d));      // (a lane below d gets its own)
            end = max(end, first);
        }
        high = __builtin_amdgcn_readlane(end, 63);      // (read where another 64 follow)
        const int count = end - first;
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

// A wave's rows out, and NaN where a value that is no number counts: `found` says that some were taken out of the tiles from key first_edge on.
template <class Src, int DP, class L_, class Stage>
__device__ __forceinline__ void store_rows(const Common& a, const PackedArgs& sa, const Problem& pr, const L_& L, const Stage& st, int first_edge, bool found, int wr, int rows, int lane) {
    const int g = lane >> 5;
    // Channels of register j of block i: 32 i + key_of(j, g).
    const int row = wr + (lane & 31), token = row / a.group, h = row - token * a.group;
    uint16_t* const op = (uint16_t*)a.o + pr.o_at + token * a.o_rs + h * a.o_hs;
    if (row < rows) {
        const float inv = 1.f / L.sum[0];      // (a row sees its own key at least: 0 is the sum of scores of -inf alone, and makes it NaN)
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
            for (int key = first_edge; key < L.limit[0]; ++key)
#pragma unroll 1
                for (int c = g; c < a.d; c += 2)
                    if (!(fabsf(elem(u32x4{st.v[key * st.v_rs + c], 0, 0, 0}, 0, Src::DT)) < INFINITY)) op[c] = 0x7fff;      // (NaN in both types)
    }
}

// The waves of the same rows: the first takes the others' numerators, sums and bases, in their order, through LDS that is idle.
template <int DB, int KG, int RG> constexpr int kJoinBytes = (KG - 1) * RG * (DB * 16 + 2) * 256;
template <class Src, int DB, int KG, int RG, class L_> __device__ __forceinline__ void join_waves(L_& L, uint8_t* lds, int kg, int rg, int lane) {
    __syncthreads();
    float* const out = reinterpret_cast<float*>(lds) + ((kg - 1) * RG + rg) * (DB * 16 + 2) * 64 + lane;
    if (kg > 0) {
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) out[(16 * i + j) * 64] = L.acc[0][i][j];
        out[DB * 16 * 64] = L.base[0];
        out[(DB * 16 + 1) * 64] = L.sum[0];
    }
    __syncthreads();
    if (kg == 0)
#pragma unroll 1
        for (int k = 1; k < KG; ++k) {
            const float* const in = reinterpret_cast<const float*>(lds) + ((k - 1) * RG + rg) * (DB * 16 + 2) * 64 + lane;
            const float base = in[DB * 16 * 64], nb = fmaxf(L.base[0], base);
            const Rebase<Src> mine_by(L.base[0], nb), its(base, nb);
            L.base[0] = nb;
            L.sum[0] = fmaf(in[(DB * 16 + 1) * 64], its.f, L.sum[0] * mine_by.f);
#pragma unroll
            for (int i = 0; i < DB; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) L.acc[0][i][j] = fmaf(in[(16 * i + j) * 64], its.f, L.acc[0][i][j] * mine_by.f);
        }
}

// QW waves of 32 rows on the same keys, or QW / KG of which KG waves each share the keys, 32 NB at a time in two LDS buffers: a tile is on its way into registers while the one before goes into
// LDS and the one before that is multiplied, SB blocks of 32 keys per step of the softmax.
template <class Src, int DP, int QW, int NB, int SB, int OCC, int KG = 1>
__global__ __launch_bounds__(64 * QW, OCC) void prompt_kernel(const Common a, const PackedArgs sa) {
    constexpr int TK = 32 * NB, TILE_K = TK * kRowK<DP>, TILE_V = TK * kRowV<DP>, RG = QW / KG, MB = NB / KG;      // (MB: blocks of a wave)
    static_assert(MB % SB == 0 && (KG == 1 || kJoinBytes<DP / 32, KG, RG> <= 2 * (TILE_K + TILE_V)), "whole steps, and room to join in");
    __shared__ __align__(16) uint8_t lds[2 * (TILE_K + TILE_V)];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 5, rg = KG == 1 ? wave : wave % RG, kg = KG == 1 ? 0 : wave / RG, mine = 32 * MB * kg;
    // workgroups are dealt to the XCDs in turn: each has its own heads where their number allows, and as many long tiles as the others
    const int slot = blockIdx.x / a.hk, head = blockIdx.x - slot * a.hk;
    Place at;
    if (!find(sa, a.group, 32 * RG, slot, at)) return;
    Problem pr;
    pr.q_at = at.first * a.q_rs + head * a.group * a.q_hs;
    pr.o_at = at.first * a.o_rs + head * a.group * a.o_hs;
    pr.tokens = pr.keys = at.count;
    pr.limit0 = sa.causal ? 1 : at.count;
    const int rows = pr.tokens * a.group, r0 = at.tile * 32 * RG, wr = r0 + 32 * rg;
    const int end = min(pr.keys, pr.limit0 + (min(rows, r0 + 32 * RG) - 1) / a.group), t1 = (end + TK - 1) / TK;
    const int sees = min(pr.keys, pr.limit0 + (min(rows, wr + 32) - 1) / a.group), t_mine = wr < rows ? max(0, sees - mine + TK - 1) / TK : 0;      // of this wave's rows and keys
    typename Src::template Stage<DP, TK, 64 * QW> st(sa, a.d, at.first, head, pr.keys, threadIdx.x);
    st.load(0);
    Lanes<Src, DP, 1> L;
    L.start(a, pr, wr, rows, lane);
    uint8_t *kb = lds, *vb = lds + 2 * TILE_K;                       // the tile that is multiplied
    uint8_t *kn = lds + TILE_K, *vn = lds + 2 * TILE_K + TILE_V;     // and the one behind it
    const int at_k = lane_k<DP>(lane) + mine * kRowK<DP>, at_v = lane_v<DP>(lane) + mine * kRowV<DP>;
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
        const bool plain = t * TK + mine + 32 * MB <= L.all_see;
#pragma unroll
        for (int b = 0; b < MB; b += SB) {
            f16acc s[SB][1];
            float kc[1][2 * SB], from[1];
            L.scores(s, kb + at_k + 32 * b * kRowK<DP>, (const float*)nullptr, g);
            L.raise(s, kc, from, sc, t * TK + mine + 32 * b, plain, true, g);
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
    if constexpr (KG > 1) join_waves<Src, DP / 32, KG, RG>(L, lds, kg, rg, lane);
    store_rows<Src, DP>(a, sa, pr, L, st, edge * TK, found, wr, kg == 0 ? rows : 0, lane);
}

// ---- head dims to 64 and to 128: products of the next tile under the softmax of this one -------------------------------------------

__device__ __forceinline__ void dma16(uint32_t lds_dst, uint32_t lane_off, const void* base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_dst), "v"(lane_off), "s"(base) : "memory", "m0");
}
template <int N> __device__ __forceinline__ void wait_vmcnt() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
template <int V> struct ic { static constexpr int value = V; };
#define SCHED_FENCE() __builtin_amdgcn_sched_barrier(0)

// A staged tile's rows are 2 DP bytes, one behind the other, as the DMA writes them; chunk c of 16 bytes of row r lies at slot c ^ turn(r).  K is read
// 16 rows at one chunk at a time, V 8 rows at four chunks: both then touch every bank once.
template <int DP> __device__ __forceinline__ int turn(int r) { return DP == 64 ? (r & 2) << 1 | (r >> 2 & 3) : (r & 3) << 2 | (r >> 2 & 3); }
template <int DP> __device__ __forceinline__ int slot_of(int r, int c) { return r * 2 * DP + ((c ^ turn<DP>(r)) << 4); }

// A row's sum takes the probabilities as they are rounded, as in Lanes::probs, which says why.  Here that is bf16 by v_dot2, and f16, which
// v_fma_mix reads as fp32, as lo + hi: the other way 16384 tokens take 1009 us for 998 (bf16; 967 with the sum of what is not rounded yet) and 1077 for 1036 (f16; 1083).
template <int DT> __device__ __forceinline__ float add_two(uint32_t a, uint32_t b, float sum) {
    if constexpr (DT == DT_BF16) return add2<DT>(a, add2<DT>(b, sum));
    else {
        float one = 1.f;
        asm("" : "+s"(one));      // (a factor that the compiler does not see, or it would convert both and add)
        const auto pair = [&](uint32_t two) {
            float lo, hi;
            unpack_f16x2(two, lo, hi);
            return fmaf(lo, one, hi);
        };
        return sum + (pair(a) + pair(b));
    }
}

// A workgroup's 8 waves (WHOLE: the head dim is DP): 8 / KG groups of 32 rows, which each KG waves share, every one with 64 keys of a tile of 64 KG; what they have of a row
// meets in LDS at the end.
//
// In iteration t a wave has the scores of tile t in registers.  Sixteen keys at a time it makes probabilities of them, and between those instructions run
// the products of the sixteen keys before with V and a quarter of the next tile's scores: every slot of the matrix pipe's 8 products (256
// cycles) has about as many cycles of vector instructions beside it.  K is a tile ahead of V.  Tiles travel by DMA into two LDS stages.  That holds
// for tiles that every row of the workgroup sees whole; the others, at the diagonal and at the prompt's end, follow in a loop that masks, with
// their rows through registers, where values that are no numbers are taken out.  16384 tokens of 16 over 4 heads of 128, causal: 990 to 1040 us, 1.06 to 1.11 PFLOP/s, where
// a library's large product reaches 1.35; matrix pipes 54 %, vector issue 42 % busy.
template <class Src, int DP, int KG, bool WHOLE>
__global__ __launch_bounds__(512, 2) void prompt_pipe_kernel(const Common a, const PackedArgs sa) {
    constexpr int QW = 8, RG = QW / KG, NS = 2, TK = 64 * KG, TILE = TK * 2 * DP, KS = DP / 16, DB = DP / 32, DT = Src::DT, ND = TILE / 1024 / QW;
    constexpr int QH = KS / 4, VH = DB / 2;      // products of half a slot
    static_assert(NS * TILE <= 65536, "a tensor's stages within the reach of a read's offset");
    extern __shared__ __align__(16) uint8_t lds[];      // K's stages, then V's
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rg = wave % RG, kg = wave / RG, lane = threadIdx.x & 63, g = lane >> 5, col = lane & 31;
    const int slot = blockIdx.x / a.hk, head = blockIdx.x - slot * a.hk;
    Place at;
    if (!find(sa, a.group, 32 * RG, slot, at)) return;
    Problem pr;
    pr.q_at = at.first * a.q_rs + head * a.group * a.q_hs;
    pr.o_at = at.first * a.o_rs + head * a.group * a.o_hs;
    pr.tokens = pr.keys = at.count;
    pr.limit0 = sa.causal ? 1 : at.count;
    const int rows = pr.tokens * a.group, r0 = at.tile * 32 * RG, wr = r0 + 32 * rg, mine = 64 * kg;      // this wave's rows, and its keys within a tile
    const int end = min(pr.keys, pr.limit0 + (min(rows, r0 + 32 * RG) - 1) / a.group), t1 = (end + TK - 1) / TK;
    const int edge = min(pr.keys, pr.limit0 + r0 / a.group) / TK;      // tiles before this one are seen whole by every row
    const int sees = min(pr.keys, pr.limit0 + (min(rows, wr + 32) - 1) / a.group), t_mine = wr < rows ? max(0, sees - mine + TK - 1) / TK : 0;
    const int piped = sa.aligned ? edge / NS * NS : 0;
    const uint16_t *const k0 = sa.k + at.first * sa.k_rs + head * sa.k_hs, *const v0 = sa.v + at.first * sa.v_rs + head * sa.v_hs;
    const uint32_t lds_base = (uint32_t)(uintptr_t)lds;

    // DMA: a kilobyte an instruction, rows RPI (wave + 8 j) .. of the tile
    constexpr int CPR = DP / 8, RPI = 64 / CPR;
    const int drow = RPI * wave + lane / CPR;
    // (the same for j: 8 RPI is a multiple of 16.  Behind the head dim V has its last chunk again, since those channels are not stored; K has zeros, which
    // no DMA writes over, since q is 0 there and 0 times an infinite key would be none)
    const int chunk = (lane % CPR) ^ turn<DP>(drow);
    const uint32_t dchunk = 16 * min(chunk, a.d / 8 - 1);
    const bool channels = chunk < a.d / 8;
    const uint32_t k_off = 2 * drow * (int)sa.k_rs + dchunk, v_off = 2 * drow * (int)sa.v_rs + dchunk;
    const auto fetch_k = [&](int t, auto stage) {
        if (WHOLE || channels)
#pragma unroll
            for (int j = 0; j < ND; ++j) dma16(lds_base + decltype(stage)::value * TILE + (wave + 8 * j) * 1024, k_off, k0 + (int64_t)(t * TK + 8 * RPI * j) * sa.k_rs);
    };
    const auto fetch_v = [&](int t, auto stage) {
#pragma unroll
        for (int j = 0; j < ND; ++j) dma16(lds_base + (NS + decltype(stage)::value) * TILE + (wave + 8 * j) * 1024, v_off, v0 + (int64_t)(t * TK + 8 * RPI * j) * sa.v_rs);
    };
    if (!WHOLE && piped && !channels)
#pragma unroll
        for (int j = 0; j < NS * ND; ++j) *reinterpret_cast<u32x4*>(lds + (wave + 8 * j) * 1024 + 16 * lane) = u32x4{0, 0, 0, 0};
    if (piped) {      // K of tiles 0 .. NS - 1, V of 0 .. NS - 2
        fetch_k(0, ic<0>{});
        fetch_v(0, ic<0>{});
        fetch_k(NS - 1, ic<NS - 1>{});
    }
    Lanes<Src, DP, 1> L;
    L.start(a, pr, wr, rows, lane);
    const typename Src::Scales sc{};

    // a lane's places in a stage: K row col, chunk 2 ks + g; V rows 16 h + 8 j + 4 g + r', its two chunks' half of block i
    int at_k[KS], at_v[2][DB];
#pragma unroll
    for (int s = 0; s < KS; ++s) at_k[s] = slot_of<DP>(mine + col, 2 * s + g);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < DB; ++i)
            at_v[j][i] = slot_of<DP>(mine + 8 * j + 4 * g + ((lane & 15) >> 2), 4 * i + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) + 8 * (lane & 1);
    const auto read_k = [&](int stage_at, int b, int s) { return *reinterpret_cast<const u32x4*>(lds + at_k[s] + stage_at + 32 * b * 2 * DP); };
    const auto read_v = [&](int stage_at, int h, int i) {
        u32x2 half[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
            half[j] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds + at_v[j][i] + stage_at + 16 * h * 2 * DP)));
        return u32x4{half[0][0], half[0][1], half[1][0], half[1][1]};
    };
    const auto meet = [] {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // (read: what was read from may be fetched into)
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    const auto largest = [&](const f16acc& x) {
        float m = fmaxf(x[0], x[1]);
#pragma unroll
        for (int i = 2; i < 16; i += 2) m = fmaxf(fmaxf(m, x[i]), x[i + 1]);
        return m;
    };
    // the base moved where a row outgrew it; `top`: the row's largest score in this lane
    const auto rebase = [&](float top) {
        top = half_max(top) * L.c[0];
        if (__any(top > L.base[0] + kLag)) {
            const float nb = fmaxf(L.base[0], top);
            const Rebase<Src> by(L.base[0], nb);
            L.base[0] = nb;
            L.sum[0] *= by.f;
#pragma unroll
            for (int i = 0; i < DB; ++i) L.acc[0][i] *= by.f;
        }
    };
    // probabilities of eight of sixteen keys (four of this lane's), rounded and in pairs
    const auto probs = [&](const f16acc (&s)[2], float from, int h, int half, u32x4& p) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = __builtin_amdgcn_exp2f(fmaf(s[h >> 1][8 * (h & 1) + 4 * half + i], L.c[0], -from));
        p[2 * half] = pack2<DT>(e[0], e[1]);
        p[2 * half + 1] = pack2<DT>(e[2], e[3]);
    };
    // their sum, while they are multiplied, so that nothing waits for it: behind the other instructions of half a slot for bf16 of 128 channels (16384 tokens 989 us, among
    // them 996), among them else (16384 of f16 1018 and 1034, 8192 of 20 heads of 64 224 and 228)
    constexpr bool kSumLast = DT == DT_BF16 && DP == 128;
    const auto sum = [&](const u32x4& p, int half) { L.sum[0] = add_two<DT>(p[2 * half], p[2 * half + 1], L.sum[0]); };

    if (piped) {
        wait_vmcnt<(NS - 2) * 2 * ND>();      // K and V of tile 0 at least
        meet();
        f16acc s[2][2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            s[0][b] = f16acc{};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) s[0][b] = mfma<DT>(read_k(0, b, ks), L.qf[0][ks], s[0][b]);
        }
        rebase(fmaxf(largest(s[0][0]), largest(s[0][1])));
        wait_vmcnt<(NS - 2) * 2 * ND>();
        meet();
        // tile t, whose number is `st` modulo NS: V of it and K of the next have landed
        const auto tile = [&](int t, auto st_tag) {
            constexpr int ST = decltype(st_tag)::value, KN = (ST + 1) % NS * TILE, VT = (NS + ST) * TILE;
            // into the stages that were read last in the iteration before: K of tile t + NS, V of tile t + NS - 1
            fetch_k(min(t + NS, edge - 1), ic<ST>{});
            fetch_v(min(t + NS - 1, edge - 1), ic<(ST + NS - 1) % NS>{});
            f16acc(&now)[2] = s[ST & 1];
            f16acc(&next)[2] = s[(ST & 1) ^ 1];
            const float from = L.base[0] == -INFINITY ? 0.f : L.base[0] - kShift<DT>;
            u32x4 p[2], kf[2][QH], vf[2][VH];
            const auto read = [&](int u) {      // the operands of half a slot: of the scores from 2 u QH products on, of V half the blocks
#pragma unroll
                for (int i = 0; i < QH; ++i) kf[u & 1][i] = read_k(KN, u >> 2, (u & 3) * QH + i);
#pragma unroll
                for (int i = 0; i < VH; ++i) vf[u & 1][i] = read_v(VT, u >> 1, (u & 1) * VH + i);
            };
            read(0);
            probs(now, from, 0, 0, p[0]);
            probs(now, from, 0, 1, p[0]);
            SCHED_FENCE();
            float top = -INFINITY;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int h = u >> 1;
                if (u < 7) read(u + 1);
                if (h < 3) probs(now, from, h + 1, u & 1, p[(h + 1) & 1]);
                if (!kSumLast) sum(p[h & 1], u & 1);
                if (u == 6) top = largest(next[0]);
#pragma unroll
                for (int i = 0; i < QH; ++i) next[u >> 2] = mfma<DT>(kf[u & 1][i], L.qf[0][(u & 3) * QH + i], i == 0 && (u & 3) == 0 ? f16acc{} : next[u >> 2]);
#pragma unroll
                for (int i = 0; i < VH; ++i) L.acc[0][(u & 1) * VH + i] = mfma<DT>(vf[u & 1][i], p[h & 1], L.acc[0][(u & 1) * VH + i]);
                // the reads, the products in a run, then the vector instructions (one by one between them: 988 us for 980)
                __builtin_amdgcn_sched_group_barrier(0x100, QH + 2 * VH, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, QH + VH, 0);
                __builtin_amdgcn_sched_group_barrier(0x402, 24, 0);
                SCHED_FENCE();
                if (kSumLast) {
                    sum(p[h & 1], u & 1);
                    SCHED_FENCE();
                }
            }
            rebase(fmaxf(top, largest(next[1])));
            wait_vmcnt<(NS - 2) * 2 * ND>();
            meet();
        };
        for (int t = 0; t < piped; t += NS) {
            tile(t, ic<0>{});
            tile(t + 1, ic<1>{});
        }
        wait_vmcnt<0>();
        meet();
    }

    // the other tiles, in two buffers: a tile is on its way into registers while the one before goes into LDS and the one before that is multiplied
    bool found = false;
    typename Src::template Stage<DP, TK, 64 * QW> st(sa, a.d, at.first, head, pr.keys, threadIdx.x);
    if (piped < t1) {
        int now = 0, then = TILE;
        const auto write = [&](int to, int t) {
            if (t >= edge) found |= st.clean();
            constexpr int CH = decltype(st)::CH;
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const int i = threadIdx.x + j * 64 * QW, place = slot_of<DP>(i / CPR, i % CPR);
                *reinterpret_cast<u32x4*>(lds + to + place) = st.kr[j];
                *reinterpret_cast<u32x4*>(lds + NS * TILE + to + place) = st.vr[j];
            }
        };
        const auto next = [&](int t) {
            // (behind the last tile the registers hold it still, and nothing reads where it goes)
            write(then, t + 1);
            if (t + 2 < t1) st.load((t + 2) * TK);
            __syncthreads();
            const int x = now; now = then; then = x;
        };
        st.load(piped * TK);
        write(now, piped);
        if (piped + 1 < t1) st.load((piped + 1) * TK);
        __syncthreads();
        for (int t = piped; t < t_mine; ++t) {
            const bool plain = t * TK + mine + 64 <= L.all_see;
            f16acc s[2][1];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                s[b][0] = f16acc{};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) s[b][0] = mfma<DT>(read_k(now, b, ks), L.qf[0][ks], s[b][0]);
            }
            float kc[1][4], from[1];
            L.raise(s, kc, from, sc, t * TK + mine, plain, true, g);
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                u32x4 p[1];
                L.probs(p, s, kc, from, sc, h);
#pragma unroll
                for (int i = 0; i < DB; ++i) L.acc[0][i] = mfma<DT>(read_v(NS * TILE + now, h, i), p[0], L.acc[0][i]);
            }
            next(t);
        }
        for (int t = max(piped, t_mine); t < t1; ++t) next(t);      // tiles that only other waves' rows see (in a loop of its own: a branch around the products costs registers)
    }
    L.finish(st, 0, end);
    if constexpr (KG > 1) join_waves<Src, DB, KG, RG>(L, lds, kg, rg, lane);
    store_rows<Src, DP>(a, sa, pr, L, st, edge * TK, found, wr, kg == 0 ? rows : 0, lane);
}

// Row tiles of a head: all rows' and a partial one for each prompt.
inline int64_t tiles_of(int64_t rows, int n, int tile) { return rows / tile + n; }

// How a call runs: tiles of `rows` rows, of whose keys `keys` waves each take a part, or 0: one wave has them all, in
// prompt_kernel.  Head dims to 64 and to 128 run in prompt_pipe_kernel where `keys` is not 0, the others always in prompt_kernel, 32 `blocks` keys at a time where there is a choice.
// Head dims to 64 and to 128.  Where tiles of 256 rows fill the CUs: the pipelined kernel, but for prompts that are short in the mean, which are
// mostly tiles with an edge, and of which prompt_kernel has two workgroups on a CU (us, bf16: 48 prompts to 231 tokens of 20 heads of 64 40.8 and
// 28.7; 12 to 800, mean 480, 43 and 37, 39 with 128 rows; 4 to 2500 67 and 84; of 16 heads of 128 24 to 400, mean 240, 45 and 37; 8 to 1300, mean 780, 58
// and 58; 4 to 2500 78 and 93).  Of 128 channels below 160 tokens 32 keys at a time and not 64, which have three workgroups on a CU (64 prompts to 77 tokens, 16 over 4
// heads 15.1 and 16.8; 48 to 160 29.3 and 30.8; 32 to 320, mean 192, 38.4 and 37.1).  Where they do not fill them: the keys of a row over two or four waves, and tiles of 128 or
// 64 rows (one prompt of 2000 tokens, 8 over 2 heads of 128 54 us in one, 42 in two; 20 heads of 64 45 and 30; 8 over 2 heads of 64 41, 28 and in four 24; 1000
// tokens of 20 heads of 64, 80 tiles, 27, 20 and 22), but for prompts of less than 128 tokens (one of 77 of 16 heads of 64 9.1 in tiles of 128 rows, 11.0 so, of 128 11.5 and 12.7;
// one of 231 13.3 and 12.1, 16.1 and 15.6).
// Many prompts of fewer rows than half such a tile in tiles of 64 (64 prompts to 20 tokens of 16 heads: of 64 channels 9.1 for 10.6, of 96 10.9 for 13.7, of 128 10.7 for 14.4, of 256
// 28.4 for 37.7; to 77 tokens, 46 rows, of 64 13.4 for 13.0, and of 20 heads 14.8 for 16.6; of 96 22.8 for 21.0; of 192 never: 34 for 21).
// The other head dims, 256 rows or 128 (of 96 128: 48 prompts to 160 tokens 33.7 and 26.1, 8 to 2500 142 and 131): of 192 24 to 600, mean 360, 119
// and 111, 12 to 1200 145 and 157; of 256 24 to 600 174 and 177, 8 to 2500 416 and 522.
// And where there are few tiles a row's keys over two waves: of 192 in tiles of 128 rows (one prompt of 300 tokens of 16 heads 21 us, 26 with one wave to a row, of 700 36 and 56, of 8000 of
// 8 over 4 heads 315 and 577; 16 to 300 24 and 33; one of 77 15.3 and 14.9; 24 to 600 of 16 over 4 heads, 820 tiles, 93 and 75), of 256 in tiles of 64, since eight waves' registers do not
// hold it (16 heads 300 27 and 29, 700 45 and 58, 2500, 640 tiles, 178 and 176; of 8 over 4 heads 2500 116 and 175, 16 to 300, mean 165, 41 and 35).
struct Form {
    int rows, keys, blocks;
};
inline Form form_of(int64_t tokens, int n, int group, int hk, int dp) {
    const int64_t cus = device_cu_count(), rows = tokens * group, mean = tokens / n, each = rows / n;      // of a prompt, in the mean
    Form f{0, 0, 0};
    const int64_t wide = tiles_of(rows, n, 256) * hk;
    if (dp == 64 || dp == 128) {
        if (wide <= cus) f.keys = mean < 128 ? 0 : dp == 64 && 4 * wide <= cus ? 4 : 2;
        else f.keys = mean >= (dp == 64 ? 800 : 500) ? 1 : 0;
        f.rows = f.keys ? 256 / f.keys : wide > cus && each < (dp == 64 ? 48 : 32) ? 64 : dp == 64 && mean >= 400 ? 256 : 128;
        if (dp == 128 && f.rows == 128) f.blocks = mean >= 160 ? 2 : 1;
        return f;
    }
    const bool long_enough = dp == 192 ? mean >= 500 : each >= 32;
    f.rows = dp != 96 && wide >= 2 * cus && long_enough ? 256 : dp != 192 && each < 32 ? 64 : 128;
    if (f.rows == 128 && dp == 192 && mean >= 128 && tiles_of(rows, n, 128) * hk <= 2 * cus) f.keys = 2;
    if (f.rows == 128 && dp == 256 && mean >= 200 && tiles_of(rows, n, 64) * hk <= 2 * cus) f.keys = 2, f.rows = 64;
    return f;
}

// The channels that a call is padded to.  Of 72 to 96 there are 128 in the pipelined kernel, where few tiles leave CUs idle (one prompt of 2500 tokens of 16 heads of 96 52 us, 114 in
// 96; three to 700 of 16 over 4 heads 23 and 35), and for long prompts (10 to 2500, mean 1500, 169 and 187; 16 to 1200 of 16 over 4 heads, mean 680, 69 and 65).
inline int dim_of(int head_dim, int64_t tokens, int n, int group, int hk) {
    const int dp = padded_dim(head_dim, 64);
    if (dp != 96) return dp;
    return tokens / n >= (tiles_of(tokens * group, n, 256) * hk <= device_cu_count() ? 128 : 1000) ? 128 : 96;
}

template <class Src, int DP, int KG, bool WHOLE> int launch_pipe_as(Common& a, const PackedArgs& sa, int64_t grid, hipStream_t st) {
    constexpr int LDS = 2 * 2 * 64 * KG * 2 * DP;
    const auto kern = prompt_pipe_kernel<Src, DP, KG, WHOLE>;
    static PerDeviceOnce once;
    if (const int e = allow_dynamic_lds((const void*)kern, LDS, once)) return e;
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(512), LDS, st, a, sa);
    KCHECK();
    return 0;
}
// (a kernel of its own where no channels are padded: the condition at K's loads costs 16384 tokens 996 us for 987, in f16 1045 for 1019, five prompts of 32 heads 329 for 323; where it is
// needed, ten prompts to 2500 of 16 heads of 96 take 167 for 164)
template <class Src, int DP, int KG> int launch_pipe(Common& a, const PackedArgs& sa, int64_t grid, hipStream_t st) {
    return a.d == DP ? launch_pipe_as<Src, DP, KG, true>(a, sa, grid, st) : launch_pipe_as<Src, DP, KG, false>(a, sa, grid, st);
}
template <class Src, int DP> int launch(Common& a, const PackedArgs& sa, hipStream_t st) {
    const Form f = form_of(sa.tokens, sa.n, a.group, a.hk, DP);
    const int64_t grid = tiles_of((int64_t)sa.tokens * a.group, sa.n, f.rows) * a.hk;
    if (grid > kMostGroups) return -1;
    if constexpr (DP == 64 || DP == 128) {
        if (f.keys == 1) return launch_pipe<Src, DP, 1>(a, sa, grid, st);
        if (f.keys == 2) return launch_pipe<Src, DP, 2>(a, sa, grid, st);
        if constexpr (DP == 64)
            if (f.keys == 4) return launch_pipe<Src, DP, 4>(a, sa, grid, st);
    }
    if (f.rows == 256) {
        if constexpr (DP == 64) prompt_kernel<Src, DP, 8, 2, 1, 4><<<(int)grid, 512, 0, st>>>(a, sa);
        else if constexpr (DP == 192) prompt_kernel<Src, DP, 8, 2, 1, 2><<<(int)grid, 512, 0, st>>>(a, sa);
        else if constexpr (DP == 256) prompt_kernel<Src, DP, 8, 1, 1, 2><<<(int)grid, 512, 0, st>>>(a, sa);
    } else if (f.rows == 64) {
        if constexpr (DP == 256) {
            if (f.keys == 2) prompt_kernel<Src, DP, 4, 2, 1, 1, 2><<<(int)grid, 256, 0, st>>>(a, sa);
            else prompt_kernel<Src, DP, 2, 1, 1, 1><<<(int)grid, 128, 0, st>>>(a, sa);
        } else if constexpr (DP != 192) prompt_kernel<Src, DP, 2, 1, 1, DP == 64 ? 4 : 2><<<(int)grid, 128, 0, st>>>(a, sa);
    } else {
        if constexpr (DP == 64) prompt_kernel<Src, DP, 4, 1, 1, 4><<<(int)grid, 256, 0, st>>>(a, sa);
        else if constexpr (DP == 96) prompt_kernel<Src, DP, 4, 1, 1, 3><<<(int)grid, 256, 0, st>>>(a, sa);
        else if constexpr (DP == 128) {
            if (f.blocks == 1) prompt_kernel<Src, DP, 4, 1, 1, 2><<<(int)grid, 256, 0, st>>>(a, sa);
            else prompt_kernel<Src, DP, 4, 2, 2, 2><<<(int)grid, 256, 0, st>>>(a, sa);
        } else if constexpr (DP == 192) {
            if (f.keys == 2) prompt_kernel<Src, DP, 8, 2, 1, 2, 2><<<(int)grid, 512, 0, st>>>(a, sa);
            else prompt_kernel<Src, DP, 4, 1, 1, 2><<<(int)grid, 256, 0, st>>>(a, sa);
        }
        else prompt_kernel<Src, DP, 4, 1, 1, 1><<<(int)grid, 256, 0, st>>>(a, sa);
    }
    KCHECK();
    return 0;
}
template <class Src> int launch_dim(Common& a, const PackedArgs& sa, hipStream_t st) {
    switch (dim_of(a.d, sa.tokens, sa.n, a.group, a.hk)) {
        case 64: return launch<Src, 64>(a, sa, st);
        case 96: return launch<Src, 96>(a, sa, st);
        case 128: return launch<Src, 128>(a, sa, st);
        case 192: return launch<Src, 192>(a, sa, st);
        default: return launch<Src, 256>(a, sa, st);
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
    const bool near = k_rs >= 0 && v_rs >= 0 && k_rs < (1 << 21) && v_rs < (1 << 21);
    s.starts = starts; s.n = n; s.tokens = tokens; s.causal = causal != 0;
    s.aligned = near && sixteen(k, k_rs, k_hs) && sixteen(v, v_rs, v_hs);
    return dtype == DT_BF16 ? launch_dim<Packed<DT_BF16>>(c, s, (hipStream_t)stream) : launch_dim<Packed<DT_F16>>(c, s, (hipStream_t)stream);
}

GPU_API int gpu_internal_prompt_attn_form(int tokens, int n, int h, int hk, int head_dim, int32_t* out) {
    if (tokens <= 0 || n <= 0 || h <= 0 || hk <= 0 || h % hk != 0 || head_dim <= 0 || head_dim > 256 || !out) return -1;
    const Form f = form_of(tokens, n, h / hk, hk, dim_of(head_dim, tokens, n, h / hk, hk));
    out[0] = f.rows;
    out[1] = f.keys;
    return 0;
}
