// Attention over pages of keys and values held in 8 bits, with a scale for each 16 tokens of a head.
#include "attn_states.hpp"
#include "kv8.hpp"

namespace {

using namespace states;

struct CacheArgs {
    const int8_t *k, *v;
    const float *ks, *vs;
    const int32_t *starts, *lens, *table;
    int rows, most, n_pages, page_shift, table_cols, causal;
};

// Codes are exact in f16, so the products take f16 operands whatever q is: a row of q is scaled by a power of two, after which bf16 values
// are f16 values but for those 2^14 below the row's largest, which round like a 32-bit sum would.  The key's scale multiplies the score.  The
// value's scale A becomes part of the probability, p' = p A <= 2^kLag, by its log2 in the exponent, and the denominator takes the block's
// sum of p' divided by A again: nothing per element.
struct Codes {
    typedef CacheArgs Args;
    static constexpr int DT = DT_F16;
    static constexpr bool kBias = false, kNormalize = true;
    // iv is 2^16 / A, so that sums of both ends of A's range, 2^-90 and 2^128, stay ordinary numbers; a smaller A counts as 2^-90, and as
    // 2^-60 of the largest so far, so that p' does not leave fp32
    static constexpr float kOut = 65536.f / 127.f;
    template <int N> struct Scales {
        float ks[N], lvs[N], ivs[N];
        __device__ float k(int i) const { return ks[i]; }
        __device__ float lv(int i) const { return lvs[i]; }
        __device__ float iv(int i) const { return ivs[i]; }
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
    template <int DP, int TK, int NT> struct Stage {
        static constexpr int ROW = DP / 16, CH = TK * ROW / NT, NS = TK / kBlock;
        const Args& a;
        const int32_t* table;
        int tid, lane, keys, d, hk, head, window = -1;
        int pid;                         // of block 64 * window + lane, and its scales
        float ks, lv, iv, top = 0.f;
        u32x4 kr[CH], vr[CH];
        Scales<NS> now, next;
        __device__ Stage(const Args& a_, const Common& c, int id, const Problem& p, int tid_)
            : a(a_), tid(tid_), lane(threadIdx.x & 63), keys(p.keys), d(c.d), hk(c.hk) {
            const int s = id / c.hk;
            head = id - s * c.hk;
            table = a.table + (int64_t)s * a.table_cols;
        }
        __device__ __forceinline__ void look(int w) {
            window = w;
            const int block = 64 * w + lane, page = page_of(table, a.table_cols, a.n_pages, a.page_shift, block);
            const bool there = block < (keys + kBlock - 1) / kBlock, ok = page >= 0;
            pid = there && ok ? page : 0;
            const int64_t i = scale_at(pid, hk, head, a.page_shift, block);
            // a block of no page, or whose values are no numbers, makes the scores NaN: rows that do not see it put -inf there
            const float A = there && ok ? a.vs[i] : 0.f;
            const bool good = A >= 0.f && A < INFINITY;
            ks = !there ? 0.f : ok && good ? a.ks[i] * (1.f / 127.f) : NAN;
            // the A of p' and of the sum's division: any will do where all values are 0
            top = fmaxf(top, wave_max_f32(good ? A : 0.f));
            const float u = top == 0.f ? 1.f : A > 0.f && good ? fmaxf(A, fmaxf(top * 0x1p-60f, 0x1p-90f)) : top;
            lv = __builtin_amdgcn_logf(u);
            iv = 65536.f / u;
        }
        __device__ __forceinline__ void load(int t) {
            const int b0 = t * NS;
            if (b0 >> 6 != window) look(b0 >> 6);
            now = next;
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                next.ks[i] = u2f(__builtin_amdgcn_readlane(f2u(ks), (b0 + i) & 63));
                next.lvs[i] = u2f(__builtin_amdgcn_readlane(f2u(lv), (b0 + i) & 63));
                next.ivs[i] = u2f(__builtin_amdgcn_readlane(f2u(iv), (b0 + i) & 63));
            }
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const int i = tid + j * NT, r = i / ROW, ch = i % ROW, token = t * TK + r;
                const int page = __builtin_amdgcn_readlane(pid, __builtin_amdgcn_readfirstlane(token >> 4) & 63);
                const int64_t at = ((((int64_t)page * hk + head) << a.page_shift) + (token & ((1 << a.page_shift) - 1))) * d + 16 * ch;
                const bool there = 16 * ch < d;
                kr[j] = there ? *reinterpret_cast<const u32x4*>(a.k + at) : u32x4{0, 0, 0, 0};
                vr[j] = there ? *reinterpret_cast<const u32x4*>(a.v + at) : u32x4{0, 0, 0, 0};
            }
        }
        __device__ __forceinline__ void write(uint8_t* kb, uint8_t* vb, float*) {
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const int i = tid + j * NT, r = i / ROW, ch = i % ROW;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    *reinterpret_cast<u32x4*>(kb + k_place<DP>(r, 2 * ch + e)) = bytes_to_f16(kr[j][2 * e], kr[j][2 * e + 1]);
                    *reinterpret_cast<u32x4*>(vb + v_place<DP>(r, 2 * ch + e)) = bytes_to_f16(vr[j][2 * e], vr[j][2 * e + 1]);
                }
            }
        }
        // of the tile that is multiplied next; `ahead`: the one behind it has been asked for already
        __device__ __forceinline__ Scales<NS> scales(bool ahead) const { return ahead ? now : next; }
    };
};

}  // namespace

GPU_API int64_t gpu_kv8_attn_workspace(int n, int most, int h, int hk, int head_dim, int page, int table_cols) {
    if (n <= 0 || most <= 0 || h <= 0 || hk <= 0 || h % hk != 0 || head_dim <= 0 || head_dim > 256 || table_cols <= 0 || page <= 0) return 0;
    return make_plan((int64_t)most * (h / hk), (int64_t)n * hk, (int64_t)table_cols * page, head_dim).bytes;
}

GPU_API int gpu_kv8_attn(int dtype, const void* q, int64_t q_rs, int64_t q_hs, void* o, int64_t o_rs, int64_t o_hs, void* ws, const int8_t* k,
                         const int8_t* v, const float* k_scale, const float* v_scale, int n_pages, int page, const int32_t* starts,
                         const int32_t* lens, const int32_t* table, int table_cols, int n, int rows, int most, int h, int hk, int head_dim,
                         float scale, int causal, void* stream) {
    if (dtype != DT_F16 && dtype != DT_BF16) return -4;
    if (!cache_ok(k, v, k_scale, v_scale, n_pages, page, hk, head_dim) || h <= 0 || h % hk != 0 || !(fabsf(scale) < INFINITY)) return -1;
    if (!rows_ok(starts, lens, table, table_cols, n, rows, most)) return -1;
    if (n == 0 || rows == 0 || most == 0) return 0;
    if (!q || !o || (int64_t)most * (h / hk) > 0x7fffff00 || (int64_t)n * hk > 0x7fffffff) return -1;
    const Plan p = make_plan((int64_t)most * (h / hk), (int64_t)n * hk, (int64_t)table_cols * page, head_dim);
    if (p.bytes && (!ws || (uintptr_t)ws % 16 != 0)) return -1;
    Common c{};
    c.q = q; c.o = o; c.q_rs = q_rs; c.q_hs = q_hs; c.o_rs = o_rs; c.o_hs = o_hs;
    c.hk = hk; c.group = h / hk; c.d = head_dim; c.q_dt = dtype;
    c.row_tiles = p.row_tiles; c.problems = n * hk; c.splits = p.splits; c.rows_padded = p.row_tiles * p.rows;
    c.aligned = ((uintptr_t)q % 16 == 0 && (q_rs | q_hs) % 8 == 0 ? 1 : 0) | ((uintptr_t)o % 8 == 0 && (o_rs | o_hs) % 4 == 0 ? 2 : 0);
    c.c = fabsf(scale) * kLog2e; c.negate = scale < 0.f; c.part = (float*)ws;
    CacheArgs s{k, v, k_scale, v_scale, starts, lens, table, rows, most, n_pages, __builtin_ctz(page), table_cols, causal != 0};
    return launch_dim<Codes>(p, c, s, (hipStream_t)stream);
}
