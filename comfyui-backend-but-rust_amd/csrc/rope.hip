// Rotary positions of queries and keys, with an optional RMS norm of each head before them.
//
// Of every head the first `rot` channels are pairs, (j, j + rot / 2) or (2j, 2j + 1), and pair j of a token at position p turns by the angle
// p f_j:  (a, b) -> factor (a cos - b sin, a sin + b cos).  The others stay, or are normed.  p f_j / 2 pi is taken in 64 bits and brought to
// half a turn there, so that far positions are as exact as near ones; the sine and cosine of what is left are fp32, and everything is
// rounded once.
//
// Bound by memory: 2 + 2 bytes a channel of 16 bits (16384 tokens of 40 heads of 128 59 us, 5.7 TB/s, a little of it from the last-level cache).  A workgroup has a few tokens: their sines and cosines go into LDS once, for all heads.
#include "common.hpp"

namespace {

struct Side {
    const void* x;
    void* o;
    int64_t x_rs, x_hs, o_rs, o_hs;     // element strides of tokens and heads
    const float* norm;                  // weight [d], or null
};
struct Rope {
    Side q, k;
    const int32_t* positions;
    const double* freqs;
    int T, h, hk, d, rot, tokens;       // tokens of a workgroup
    float factor, eps;
    int wide;                           // pieces start on multiples of their size
};

// N consecutive elements, as one access where they lie on a multiple of their size (two of 16 bytes for eight floats).
template <int DT, int N, bool PAST> __device__ __forceinline__ void load_n(const void* p, int64_t at, bool wide, float (&v)[N]) {
    constexpr int WORDS = N * dt_size<DT>::value / 4;
    if (!wide) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = ld_dt<DT>(p, at + i);
        return;
    }
    typedef uint32_t piece __attribute__((ext_vector_type(WORDS < 4 ? WORDS : 4)));
    constexpr int PER = WORDS < 4 ? WORDS : 4;
    uint32_t w[WORDS];
    const piece* const src = reinterpret_cast<const piece*>((const char*)p + at * dt_size<DT>::value);
#pragma unroll
    for (int i = 0; i < WORDS / PER; ++i) {
        const piece x = PAST ? __builtin_nontemporal_load(src + i) : src[i];
#pragma unroll
        for (int j = 0; j < PER; ++j) w[i * PER + j] = x[j];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (DT == DT_F32) v[i] = u2f(w[i]);
        else if (DT == DT_BF16) v[i] = u2f(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
        else v[i] = f16_to_f((uint16_t)(w[i >> 1] >> 16 * (i & 1)));
    }
}
template <int DT, int N> __device__ __forceinline__ void store_n(void* p, int64_t at, bool wide, const float (&v)[N]) {
    constexpr int WORDS = N * dt_size<DT>::value / 4, PER = WORDS < 4 ? WORDS : 4;
    if (!wide) {
#pragma unroll
        for (int i = 0; i < N; ++i) st_dt<DT>(p, at + i, v[i]);
        return;
    }
    uint32_t w[WORDS];
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = DT == DT_F32 ? f2u(v[i]) : DT == DT_BF16 ? pack_bf16x2(v[2 * i < N ? 2 * i : 0], v[2 * i + 1 < N ? 2 * i + 1 : 0]) : pack_f16x2(v[2 * i < N ? 2 * i : 0], v[2 * i + 1 < N ? 2 * i + 1 : 0]);
    typedef uint32_t piece __attribute__((ext_vector_type(PER)));
    piece* const to = reinterpret_cast<piece*>((char*)p + at * dt_size<DT>::value);
#pragma unroll
    for (int i = 0; i < WORDS / PER; ++i) {
        piece x;
#pragma unroll
        for (int j = 0; j < PER; ++j) x[j] = w[i * PER + j];
        to[i] = x;
    }
}

constexpr int kMostTokens = 4;

// A lane has V pairs of a head at a time, or 2 V of the channels that stay; a head's lanes are a power of two side by side.
template <int DT, int V, bool INTER, bool NORM, bool PAST>
__global__ __launch_bounds__(256) void rope_kernel(const Rope a) {
    __shared__ f32x2 turn[kMostTokens * 128];
    const int pairs = a.rot / 2, t0 = blockIdx.x * a.tokens, tokens = min(a.tokens, a.T - t0);
    const int turned = pairs / V, units = a.d / (2 * V), heads = a.h + a.hk;
    const int lanes_log = units <= 1 ? 0 : 32 - __builtin_clz(units - 1), unit = threadIdx.x & ((1 << lanes_log) - 1), step = 256 >> lanes_log;
    // The two pieces of V channels.  Halves: one in each half of what turns, or of the rest.  Neighbours, where a piece has its pairs whole: one in
    // each half of the head, so that lanes side by side have whole lines.
    const bool rotates = INTER ? true : unit < turned, some = unit < units;
    const int c0 = INTER || rotates ? V * unit : a.rot + V * (unit - turned), c1 = c0 + (INTER ? a.d / 2 : rotates ? pairs : (a.d - a.rot) / 2);
    const int end = tokens * heads;
    const auto head_of = [&](int i, int& token, int& head) {      // -> whether it is one of q's
        token = i / heads;
        head = i - token * heads;
        const bool is_q = head < a.h;
        if (!is_q) head -= a.h;
        return is_q;
    };
    float x[2][V];
    const auto load = [&](int i) {
        int token, head;
        const Side& s = head_of(i, token, head) ? a.q : a.k;
        const int64_t from = (t0 + token) * s.x_rs + head * s.x_hs;
        if (!some) return;
        load_n<DT, V, PAST>(s.x, from + c0, a.wide, x[0]);
        load_n<DT, V, PAST>(s.x, from + c1, a.wide, x[1]);
    };
    int i = threadIdx.x >> lanes_log;
    if (i < end) load(i);      // on its way while the sines are made
    for (int j = threadIdx.x; j < tokens * pairs; j += 256) {
        const int token = j / pairs;
        const double at = (double)a.positions[t0 + token] * (a.freqs[j - token * pairs] * 0.15915494309189533577), left = at - rint(at);
        float s, c;
        sincospif(2.f * (float)left, &s, &c);
        turn[j] = f32x2{a.factor * c, a.factor * s};
    }
    __syncthreads();
    for (; i < end; i += step) {
        int token, head;
        const Side& s = head_of(i, token, head) ? a.q : a.k;
        const int64_t to = (t0 + token) * s.o_rs + head * s.o_hs;
        if constexpr (NORM) {
            float sum = 0.f;
            if (some)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < V; ++e) sum = fmaf(x[j][e], x[j][e], sum);
            for (int m = 1; m < 1 << lanes_log; m *= 2) sum += __shfl_xor(sum, m);
            if (some && s.norm) {
                const float r = 1.f / sqrtf(sum / (float)a.d + a.eps);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < V; ++e) x[j][e] = x[j][e] * r * s.norm[(j ? c1 : c0) + e];
            }
        }
        float y[2][V];
#pragma unroll
        for (int e = 0; e < V; ++e) y[0][e] = x[0][e], y[1][e] = x[1][e];
        if (i + step < end) load(i + step);
        if (!some) continue;
        if (rotates) {
            const f32x2* const cs = turn + token * pairs;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int half = INTER ? 2 * e / V : 0, k = INTER ? 2 * e % V : e;      // the pair's first channel
                if (INTER && (half ? c1 : c0) >= a.rot) continue;
                const f32x2 t = cs[INTER ? (half ? c1 : c0) / 2 + e % (V / 2) : c0 + e];
                float& p = y[half][k];
                float& q = INTER ? y[half][k + 1] : y[1][e];
                const float u = fmaf(p, t[0], -(q * t[1]));
                q = fmaf(p, t[1], q * t[0]);
                p = u;
            }
        }
        store_n<DT, V>(s.o, to + c0, a.wide, y[0]);
        store_n<DT, V>(s.o, to + c1, a.wide, y[1]);
    }
}

template <int DT, int V, bool PAST> int launch_loads(const Rope& a, bool interleaved, hipStream_t st) {
    const int grid = (int)(((int64_t)a.T + a.tokens - 1) / a.tokens);
    const bool norm = a.q.norm || a.k.norm;
    if (interleaved) {
        if (norm) rope_kernel<DT, V, true, true, PAST><<<grid, 256, 0, st>>>(a);
        else rope_kernel<DT, V, true, false, PAST><<<grid, 256, 0, st>>>(a);
    } else {
        if (norm) rope_kernel<DT, V, false, true, PAST><<<grid, 256, 0, st>>>(a);
        else rope_kernel<DT, V, false, false, PAST><<<grid, 256, 0, st>>>(a);
    }
    KCHECK();
    return 0;
}
// Calls of 128 MB or more load past the caches (32768 tokens of 40 heads of 128: 131 us without, 124 with; 2048 tokens, which stay in the last-level
// cache, 10.8 and 12.4).  A token to a workgroup, more where its heads do not fill one (16384 x 40 heads of 128: 75 us with one, 78 with four; 2048 tokens 10.7 and 12.7).
template <int DT, int V> int launch(Rope a, bool interleaved, hipStream_t st) {
    int lanes = 1;
    while (lanes < a.d / (2 * V)) lanes *= 2;
    const int fit = 256 / (lanes * (a.h + a.hk));
    a.tokens = a.T < 4 * device_cu_count() || fit < 1 ? 1 : fit < kMostTokens ? fit : kMostTokens;
    if (((int64_t)a.T + a.tokens - 1) / a.tokens > 0xffffffffll / 256) return -1;
    const int64_t bytes = (int64_t)dt_size<DT>::value * 2 * a.T * (a.h + a.hk) * a.d;
    return bytes >= (int64_t)128 << 20 ? launch_loads<DT, V, true>(a, interleaved, st) : launch_loads<DT, V, false>(a, interleaved, st);
}
template <int DT> int launch_width(Rope a, bool interleaved, hipStream_t st) {
    // the widest pieces that cut both parts of a head into whole ones
    const auto cuts = [&](int v) { return interleaved ? a.d % (2 * v) == 0 && a.rot % v == 0 : a.rot % (2 * v) == 0 && (a.d - a.rot) % (2 * v) == 0; };
    const int v = cuts(8) ? 8 : cuts(4) ? 4 : 2;
    const int size = dt_size<DT>::value, bytes = v * size < 16 ? v * size : 16;
    const auto on = [&](const Side& s) {
        return (uintptr_t)s.x % bytes == 0 && (uintptr_t)s.o % bytes == 0 && (s.x_rs * size) % bytes == 0 && (s.x_hs * size) % bytes == 0 && (s.o_rs * size) % bytes == 0 && (s.o_hs * size) % bytes == 0;
    };
    a.wide = on(a.q) && (a.hk == 0 || on(a.k));
    return v == 8 ? launch<DT, 8>(a, interleaved, st) : v == 4 ? launch<DT, 4>(a, interleaved, st) : launch<DT, 2>(a, interleaved, st);
}

}  // namespace

GPU_API int gpu_rope(int dtype, const void* q, int64_t q_rs, int64_t q_hs, void* q_out, int64_t qo_rs, int64_t qo_hs, int h, const void* k,
                     int64_t k_rs, int64_t k_hs, void* k_out, int64_t ko_rs, int64_t ko_hs, int hk, const int32_t* positions,
                     const double* freqs, int rot, int interleaved, float factor, const float* q_norm, const float* k_norm, float eps, int T,
                     int head_dim, void* stream) {
    if (dtype != DT_BF16 && dtype != DT_F16 && dtype != DT_F32) return -4;
    if (T < 0 || h < 0 || hk < 0 || head_dim <= 0 || head_dim > 256 || head_dim % 4 != 0 || rot <= 0 || rot > head_dim || rot % 4 != 0) return -1;
    if (h > 65536 || hk > 65536 || !(fabsf(factor) < INFINITY) || ((q_norm || k_norm) && !(eps >= 0.f && eps < INFINITY))) return -1;
    if (T == 0 || h + hk == 0) return 0;
    const int size = dtype == DT_F32 ? 4 : 2;
    if ((h && (!q || !q_out)) || (hk && (!k || !k_out)) || !positions || !freqs || (uintptr_t)freqs % 8 != 0 || (uintptr_t)positions % 4 != 0) return -1;
    if (((uintptr_t)q | (uintptr_t)q_out | (uintptr_t)k | (uintptr_t)k_out) % size != 0 || ((uintptr_t)q_norm | (uintptr_t)k_norm) % 4 != 0) return -1;
    Rope a{};
    a.q = {q, q_out, q_rs, q_hs, qo_rs, qo_hs, q_norm};
    a.k = {k, k_out, k_rs, k_hs, ko_rs, ko_hs, k_norm};
    a.positions = positions; a.freqs = freqs;
    a.T = T; a.h = h; a.hk = hk; a.d = head_dim; a.rot = rot; a.factor = factor; a.eps = eps;
    const hipStream_t st = (hipStream_t)stream;
    return dtype == DT_BF16 ? launch_width<DT_BF16>(a, interleaved != 0, st) : dtype == DT_F16 ? launch_width<DT_F16>(a, interleaved != 0, st) : launch_width<DT_F32>(a, interleaved != 0, st);
}
