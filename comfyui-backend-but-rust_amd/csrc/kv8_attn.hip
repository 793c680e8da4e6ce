// Attention over pages of keys and values held in 8 bits, with a scale for each 16 tokens of a head.
#include "attn_states.hpp"
#include "kv8.hpp"

namespace {

using namespace states;

static_assert(kMostTokens <= kMostLength, "positions stay 32-bit numbers");

struct CacheArgs {
    const int8_t *k, *v;
    const float *ks, *vs;
    const int32_t *starts, *lens, *table;
    int rows, most, n_pages, page_shift, table_cols, causal;
};

// Codes are exact in f16, so the products take f16 operands whatever q is: a row of q is scaled by a power of two, after which bf16 values
// are f16 values but for those 2^14 below the row's largest, which round like a 32-bit sum would.  The key's scale multiplies the score.  The
// value's scale A becomes part of the probability, p' = p A <= 2^kLag, by its log2 in the exponent, and the denominator takes the block's
// sum of p' divided by A again: nothing per element.  That holds where the A of 64 blocks are within 1/16 of the largest so far, and not below
// kLeast; elsewhere p' may vanish beside a p that does not, and the denominator is summed from p itself (Lanes::add_sum).
struct Codes {
    typedef CacheArgs Args;
    static constexpr int DT = DT_F16;
    static constexpr bool kBias = false, kNormalize = true;
    // iv is 16 / A, so that sums of both ends of A's range, 2^kLeast and 2^128, stay ordinary numbers; a row's base counts a smaller A as
    // 2^kLeast, so that p, which is 2^-kLeast of the base then, does so too
    static constexpr float kOut = 16.f / 127.f;
    template <int N> struct Scales {
        float ks[N], lvs[N], ivs[N];
        __device__ float k(int h) const { return ks[h]; }
        __device__ float lv(int h) const { return lvs[h]; }
        __device__ float iv(int h) const { return ivs[h]; }
    };
    static __device__ __forceinline__ Problem problem(const Args& a, const Common& c, int id) {
        const int s = id / c.hk, head = id - s * c.hk;
        const Span sp = span(a.starts, a.lens, s, a.rows, a.most);
        Problem p;
        p.q_at = sp.first * c.q_rs + head * c.group * c.q_hs;
        p.o_at = sp.first * c.o_rs + head * c.group * c.o_hs;
        p.tokens = sp.count;
        // tokens past the table are one block of no page: they make the rows that see them NaN
        const int64_t held = ((int64_t)a.table_cols << a.page_shift) + kBlock;
        p.keys = (int)min((int64_t)sp.len, held);
        p.limit0 = a.causal ? sp.len - sp.count + 1 : p.keys;
        return p;
    }
    // the chunk of 8 channels that step s of the product of few rows takes from lanes 16 gg ..: half of the 16 codes of a load
    static __device__ __forceinline__ int q_chunk(int s, int gg) { return 8 * (s >> 1) + 2 * gg + (s & 1); }
    template <int DP, int TK, int NT> struct Stage {
        static constexpr int ROW = DP == 192 ? 16 : DP == 96 ? 8 : DP / 16, CH = (TK * ROW + NT - 1) / NT;      // a power of two threads to a row
        static constexpr bool kAll = TK * ROW % NT == 0;      // every thread has a piece of every load
        static_assert(kAll || (CH == 1 && TK * ROW % 64 == 0), "whole waves are without a piece");
        __device__ __forceinline__ bool mine() const { return kAll || tid < TK * ROW; }
        const Args& a;
        const int32_t* table;
        int tid, lane, keys, d, hk, head;
        int window = -1, s_window = -1;
        int pages;                       // of block 64 * window + lane
        float ks, lv, iv, top = 0.f;     // its scales
        bool all_numbers, all_even;      // of the window: no block without numbers; iv in use
        u32x4 kr[CH], vr[CH];
        __device__ Stage(const Args& a_, const Common& c, int id, const Problem& p, int tid_)
            : a(a_), tid(tid_), lane(threadIdx.x & 63), keys(p.keys), d(c.d), hk(c.hk) {
            const int s = id / c.hk;
            head = id - s * c.hk;
            table = a.table + (int64_t)s * a.table_cols;
#pragma unroll
            for (int j = 0; j < CH; ++j) kr[j] = vr[j] = u32x4{0, 0, 0, 0};     // behind the head dim they stay 0
        }
        // the page of a block, 0 for one that none holds: what is read there counts for nothing, or for NaN
        __device__ __forceinline__ int page(int block) const {
            const int p = page_of(table, a.table_cols, a.n_pages, a.page_shift, block);
            return p < 0 ? 0 : p;
        }
        __device__ __forceinline__ void look(int w) {
            s_window = w;
            const int block = 64 * w + lane, p = page_of(table, a.table_cols, a.n_pages, a.page_shift, block);
            const bool there = block < (keys + kBlock - 1) / kBlock, ok = p >= 0;
            const int64_t i = scale_at(there && ok ? p : 0, hk, head, a.page_shift, block);
            // a block of no page, or whose values are no numbers, makes the scores NaN: rows that do not see it put -inf there
            const float A = there && ok ? a.vs[i] : 0.f;
            const bool good = A >= 0.f && A < INFINITY;
            ks = !there ? 0.f : ok && good ? a.ks[i] * (1.f / 127.f) : NAN;
            // the A of p' and of the sum's division: any will do where all values are 0
            top = fmaxf(top, wave_max_f32(good ? A : 0.f));
            const float u = top == 0.f ? 1.f : A > 0.f && good ? A : top;
            all_numbers = !__any(ks != ks);
            lv = u < 0x1p-64f ? __builtin_amdgcn_logf(u * 0x1p64f) - 64.f : __builtin_amdgcn_logf(u);      // the instruction takes ordinary numbers
            all_even = !__any(u < fmaxf(top * 0x1p-4f, 0x1p-90f));
            static_assert(kLeast == -90.f, "which is where iv ends");
            iv = all_even ? 16.f / u : 0.f;
        }
        // TK rows from key0, a multiple of 32
        __device__ __forceinline__ void rows(u32x4 (&x)[CH], const int8_t* codes, int key0) {
            if (!mine()) return;
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const int i = tid + j * NT, token = key0 + i / ROW, ch = i % ROW;
                // the rows that a wave loads at once lie in one block: a scalar base and 32-bit offsets
                const int block = __builtin_amdgcn_readfirstlane(token >> 4);
                if (block >> 6 != window) {
                    window = block >> 6;
                    pages = page(64 * window + lane);
                }
                const int64_t at = codes_at(__builtin_amdgcn_readlane(pages, block & 63), hk, head, a.page_shift, block, d);
                const uint32_t in = (token & (kBlock - 1)) * d + 16 * ch;
                if (16 * ch < d) x[j] = *reinterpret_cast<const u32x4*>(codes + at + in);
            }
        }
        __device__ __forceinline__ void load_k(int key0) { rows(kr, a.k, key0); }
        __device__ __forceinline__ void load_v(int key0) { rows(vr, a.v, key0); }
        __device__ __forceinline__ void load_fragments(int key0) {
            static_assert(NT != 64 || CH >= 2 * (DP / 64), "32 keys of a wave");
            const int col = tid & 15, gg = tid >> 4;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int block = __builtin_amdgcn_readfirstlane(key0 >> 4) + b;
                if (block >> 6 != window) {
                    window = block >> 6;
                    pages = page(64 * window + lane);
                }
                const int8_t* const at = a.k + codes_at(__builtin_amdgcn_readlane(pages, block & 63), hk, head, a.page_shift, block, d);
#pragma unroll
                for (int i = 0; i < DP / 64; ++i)
                    if (64 * i + 16 * gg < d) kr[b * (DP / 64) + i] = *reinterpret_cast<const u32x4*>(at + (uint32_t)(col * d + 64 * i + 16 * gg));
            }
        }
        __device__ __forceinline__ u32x4 fragment(int b, int s) const {
            const u32x4 c = kr[b * (DP / 64) + s / 2];
            return bytes_to_f16(c[2 * (s & 1)], c[2 * (s & 1) + 1]);
        }
        __device__ __forceinline__ void write_bias(float*) {}
        __device__ __forceinline__ void write_k(uint8_t* kb, float*) {
            if (!mine()) return;
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const int i = tid + j * NT;
                if (i % ROW >= DP / 16) continue;
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    *reinterpret_cast<u32x4*>(kb + k_place<DP>(i / ROW, 2 * (i % ROW) + e)) = bytes_to_f16(kr[j][2 * e], kr[j][2 * e + 1]);
            }
        }
        __device__ __forceinline__ void write_v(uint8_t* vb) {
            if (!mine()) return;
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const int i = tid + j * NT;
                if (i % ROW >= DP / 16) continue;
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    *reinterpret_cast<u32x4*>(vb + v_place<DP>(i / ROW, 2 * (i % ROW) + e)) = bytes_to_f16(vr[j][2 * e], vr[j][2 * e + 1]);
            }
        }
        __device__ bool any_key(int, int) const { return true; }
        __device__ __forceinline__ bool numbers() const { return all_numbers; }
        __device__ __forceinline__ bool even() const { return all_even; }
        // of the TK keys from key0
        __device__ __forceinline__ Scales<TK / kBlock> scales(int key0) {
            const int block = __builtin_amdgcn_readfirstlane(key0 >> 4);
            if (block >> 6 != s_window) look(block >> 6);
            Scales<TK / kBlock> r;
#pragma unroll
            for (int h = 0; h < TK / kBlock; ++h) {
                r.ks[h] = u2f(__builtin_amdgcn_readlane(f2u(ks), (block + h) & 63));
                r.lvs[h] = u2f(__builtin_amdgcn_readlane(f2u(lv), (block + h) & 63));
                r.ivs[h] = u2f(__builtin_amdgcn_readlane(f2u(iv), (block + h) & 63));
            }
            return r;
        }
    };
};

}  // namespace

GPU_API int64_t gpu_kv8_attn_workspace(int n, int most, int h, int hk, int head_dim, int page, int table_cols) {
    if (n <= 0 || most <= 0 || h <= 0 || hk <= 0 || h % hk != 0 || head_dim <= 0 || head_dim > 256 || table_cols <= 0 || page <= 0) return 0;
    return make_plan((int64_t)most * (h / hk), (int64_t)n * hk, (int64_t)table_cols * page, head_dim, 1).bytes;
}

GPU_API int gpu_kv8_attn(int dtype, const void* q, int64_t q_rs, int64_t q_hs, void* o, int64_t o_rs, int64_t o_hs, void* ws, const int8_t* k,
                         const int8_t* v, const float* k_scale, const float* v_scale, int n_pages, int page, const int32_t* starts,
                         const int32_t* lens, const int32_t* table, int table_cols, int n, int rows, int most, int h, int hk, int head_dim,
                         float scale, int causal, void* stream) {
    if (dtype != DT_F16 && dtype != DT_BF16) return -4;
    if (!cache_ok(k, v, k_scale, v_scale, n_pages, page, hk, head_dim) || h <= 0 || h % hk != 0 || !(fabsf(scale) < INFINITY)) return -1;
    if (!rows_ok(starts, lens, table, table_cols, n, rows, most)) return -1;
    if (n == 0 || rows == 0 || most == 0) return 0;
    if (!q || !o || most > kMostLength || (int64_t)most * (h / hk) > 0x7ffff000 || (int64_t)n * hk > 0x7fffffff) return -1;
    const Plan p = make_plan((int64_t)most * (h / hk), (int64_t)n * hk, (int64_t)table_cols * page, head_dim, 1);
    if (p.bytes && (!ws || (uintptr_t)ws % 16 != 0)) return -1;
    Common c{};
    c.q = q; c.o = o; c.q_rs = q_rs; c.q_hs = q_hs; c.o_rs = o_rs; c.o_hs = o_hs;
    c.hk = hk; c.group = h / hk; c.d = head_dim; c.q_dt = dtype;
    c.row_tiles = p.row_tiles; c.problems = n * hk; c.splits = p.splits; c.rows_padded = p.row_tiles * p.rows;
    c.aligned = ((uintptr_t)q % 16 == 0 && (q_rs | q_hs) % 8 == 0 ? 1 : 0) | ((uintptr_t)o % 16 == 0 && (o_rs | o_hs) % 8 == 0 ? 2 : 0);
    set_scale(c, scale, 1.17549435e-38f);
    c.part = (float*)ws;
    CacheArgs s{k, v, k_scale, v_scale, starts, lens, table, rows, most, n_pages, __builtin_ctz(page), table_cols, causal != 0};
    return launch_dim<Codes>(p, (int64_t)most * (h / hk), c, s, (hipStream_t)stream);
}
