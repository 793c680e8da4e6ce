// The paged cache of keys and values in 8 bits: new tokens into it, tokens back out of it, pages from one place to another.
#include "common.hpp"
#include "kv8.hpp"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct Pages {
    int8_t *k, *v;
    float *ks, *vs;
    const int32_t *starts, *lens, *table;
    int n_pages, page_shift, table_cols, hk, d, rows, most;
};

// The codes of 16 values x (or of codes to be scaled again): rne(n / A), n = 127 x or code * old A, exactly.  n has at most 18 significant
// bits and A 11, so n / A is either a tie, which a division gives exactly, or further from one than its rounding to 24 bits moves it.  A
// multiplication by the rounded f / A is off by less than 2^-15 of a code, so only quotients that near to a tie are divided.
__device__ __forceinline__ u32x4 codes_of(const float (&n)[16], float f, float A) {
    const float r = f / A;
    u32x4 w = {0, 0, 0, 0};
    bool near = false;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float t = n[i] * r, q = rintf(t);
        near |= fabsf(t - q) > 0.5f - 0x1p-14f;
        w[i >> 2] |= (uint32_t)((int)q & 255) << 8 * (i & 3);
    }
    if (near) {
        w = u32x4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i >> 2] |= (uint32_t)((int)rintf(n[i] * f / A) & 255) << 8 * (i & 3);
    }
    return w;
}
// The power of two that both sides take first where 127 x would leave fp32, or A its ordinary numbers.
__device__ __forceinline__ float shifted(float A) { return A > 1e30f ? 0x1p-100f : A < 1e-25f ? 0x1p+60f : 1.f; }

template <int DT> __device__ __forceinline__ void widen(const u32x4 (&x)[2], float (&f)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const uint16_t h = (uint16_t)(x[i >> 3][(i >> 1) & 3] >> 16 * (i & 1));
        f[i] = DT == DT_BF16 ? bf16_to_f(h) : f16_to_f(h);
    }
}

// grid: blocks of 16 tokens that a sequence's rows can touch, keys and values of the heads (a wave each, those of a block side by side, as
// their rows lie in memory); sequences.
// A wave quantizes one block of one head, keys or values: its 16 rows of d in registers, 16 values of a row at a time, the largest magnitude
// over the wave.  Codes of earlier tokens in the block are scaled again where A grew.  Bound by memory: 8187 tokens of 8 heads of 128
// channels, keys and values, 50 MB in 14.5 us (3.5 TB/s; one wave's trips for row descriptors, page, rows are 4 us of that, what a
// single token takes); with a division per value, eight values a lane and a head's blocks side by side 18.
template <int DT, int DP>
__global__ __launch_bounds__(256) void store_kernel(const Pages a, const uint16_t* k, int64_t k_rs, int64_t k_hs, const uint16_t* v, int64_t v_rs,
                                                    int64_t v_hs, int aligned) {
    constexpr int ROW = DP / 16, CH = kBlock * ROW / 64;
    const int lane = threadIdx.x & 63, groups = (2 * a.hk + 3) / 4, blk = blockIdx.x / groups, line = __builtin_amdgcn_readfirstlane((blockIdx.x - blk * groups) * 4 + (threadIdx.x >> 6)), head = line >> 1, which = line & 1, s = blockIdx.y;
    if (head >= a.hk) return;
    const Span sp = span(a.starts, a.lens, s, a.rows, a.most);
    const int first = sp.len - sp.count;                   // position of the first new token
    const int b = (first > 0 ? first : 0) / kBlock + blk, t0 = b * kBlock;
    if (sp.count == 0 || t0 >= sp.len) return;
    const int page = page_of(a.table + (int64_t)s * a.table_cols, a.table_cols, a.n_pages, a.page_shift, b);
    if (page < 0) return;
    int8_t* const codes = (which ? a.v : a.k) + codes_at(page, a.hk, head, a.page_shift, b, a.d);
    float* const scale = (which ? a.vs : a.ks) + scale_at(page, a.hk, head, a.page_shift, b);
    const uint16_t* const x = which ? v + head * v_hs : k + head * k_hs;
    const int64_t rs = which ? v_rs : k_rs;
    const int begun = first > t0 ? first - t0 : 0;         // earlier tokens in the block
    const float old = begun ? *scale : 0.f;

    u32x4 xr[CH][2];
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        const int i = lane + 64 * j, r = i / ROW, ch = i % ROW, t = t0 + r;
        xr[j][0] = xr[j][1] = u32x4{0, 0, 0, 0};
        if (r >= begun && t < sp.len && 16 * ch < a.d) {
            const uint16_t* const p = x + (int64_t)(sp.first + t - first) * rs + 16 * ch;
            if (aligned) {
                xr[j][0] = *reinterpret_cast<const u32x4*>(p);
                xr[j][1] = *reinterpret_cast<const u32x4*>(p + 8);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) xr[j][e >> 2][e & 3] = (uint32_t)p[2 * e] | (uint32_t)p[2 * e + 1] << 16;
            }
        }
    }
    float A = 0.f;
    bool odd = false;      // a value that is no number
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        float f[16];
        widen<DT>(xr[j], f);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            odd |= !(fabsf(f[i]) < INFINITY);
            A = fmaxf(A, fabsf(f[i]));
        }
    }
    A = wave_max_f32(A);
    odd = __any(odd) || !(old < INFINITY);
    A = fmaxf(A, old);
    const float by = shifted(A), div = A > 0.f ? A * by : 1.f;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        const int i = lane + 64 * j, r = i / ROW, ch = i % ROW, t = t0 + r;
        if (t >= sp.len || 16 * ch >= a.d || (r < begun && A == old && !odd)) continue;
        u32x4* const to = reinterpret_cast<u32x4*>(codes + r * a.d + 16 * ch);
        float n[16], f = 127.f;
        if (r < begun) {
            const u32x4 c = *to;
#pragma unroll
            for (int e = 0; e < 16; ++e) n[e] = (float)(int8_t)(c[e >> 2] >> 8 * (e & 3));
            f = old * by;
        } else {
            widen<DT>(xr[j], n);
#pragma unroll
            for (int e = 0; e < 16; ++e) n[e] *= by;
        }
        *to = odd ? u32x4{0, 0, 0, 0} : codes_of(n, f, div);
    }
    if (lane == 0) *scale = odd ? NAN : A;
}

// Tokens back out: a wave per block of a head, keys or values, 16 values of a row at a time.  The same 50 MB the other way: 11.4 us, 4.4 TB/s.
template <int DT, int DP>
__global__ __launch_bounds__(256) void read_kernel(const Pages a, void* k, int64_t k_rs, int64_t k_hs, void* v, int64_t v_rs, int64_t v_hs, int aligned) {
    constexpr int ROW = DP / 16, CH = kBlock * ROW / 64;
    const int lane = threadIdx.x & 63, groups = (2 * a.hk + 3) / 4, blk = blockIdx.x / groups, line = __builtin_amdgcn_readfirstlane((blockIdx.x - blk * groups) * 4 + (threadIdx.x >> 6)), head = line >> 1, which = line & 1, s = blockIdx.y;
    if (head >= a.hk) return;
    const Span sp = span(a.starts, a.lens, s, a.rows, a.most);
    const int first = sp.len - sp.count;
    const int b = (first >= 0 ? first : first - (kBlock - 1)) / kBlock + blk, t0 = b * kBlock;
    if (sp.count == 0 || t0 >= sp.len) return;
    const int page = page_of(a.table + (int64_t)s * a.table_cols, a.table_cols, a.n_pages, a.page_shift, b);
    const bool there = page >= 0;
    const int8_t* const codes = (which ? a.v : a.k) + codes_at(there ? page : 0, a.hk, head, a.page_shift, b, a.d);
    void* const out = which ? v : k;
    const int64_t rs = which ? v_rs : k_rs, base = head * (which ? v_hs : k_hs);
    u32x4 c[CH];
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        const int i = lane + 64 * j;
        c[j] = there && 16 * (i % ROW) < a.d ? *reinterpret_cast<const u32x4*>(codes + i / ROW * a.d + 16 * (i % ROW)) : u32x4{0, 0, 0, 0};
    }
    const float A = there ? (which ? a.vs : a.ks)[scale_at(page, a.hk, head, a.page_shift, b)] * (1.f / 127.f) : NAN;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        const int i = lane + 64 * j, r = i / ROW, ch = i % ROW, t = t0 + r;
        if (t < first || t >= sp.len || 16 * ch >= a.d) continue;
        const int64_t to = base + (int64_t)(sp.first + t - first) * rs + 16 * ch;
        float f[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) f[e] = (float)(int8_t)(c[j][e >> 2] >> 8 * (e & 3)) * A;
        if (DT != DT_F32 && aligned) {
            u32x4 u[2];
#pragma unroll
            for (int e = 0; e < 16; e += 2) u[e >> 3][(e >> 1) & 3] = DT == DT_BF16 ? pack_bf16x2(f[e], f[e + 1]) : pack_f16x2(f[e], f[e + 1]);
            u32x4* const p = reinterpret_cast<u32x4*>((uint16_t*)out + to);
            p[0] = u[0];
            p[1] = u[1];
        } else {
#pragma unroll
            for (int e = 0; e < 16; e += 4) store4<DT>(out, to + e, f + e);
        }
    }
}

// Pages src[i] -> dst[i] of every layer: a workgroup per piece of 16 KB of one page's keys or values, four loads of a thread in flight; the
// first piece takes the scales along.  160 pages of 28 layers, 1.18 GB in and out: 230 us, 5.1 TB/s, the rate of a large copy.
constexpr int kPiece = 16384;
__global__ __launch_bounds__(256) void copy_kernel(int8_t* k, int8_t* v, float* ks, float* vs, int n_pages, int64_t page_bytes, int page_scales,
                                                   const int32_t* src, const int32_t* dst, int pieces) {
    const int piece = blockIdx.x % pieces, which = blockIdx.x / pieces, i = blockIdx.y;
    const int from = src[i], to = dst[i];
    if ((unsigned)from >= (unsigned)n_pages || (unsigned)to >= (unsigned)n_pages || from == to) return;
    const int64_t layer = (int64_t)blockIdx.z * n_pages;
    int8_t* const c = which ? v : k;
    const u32x4* const a = reinterpret_cast<const u32x4*>(c + (layer + from) * page_bytes + (int64_t)piece * kPiece);
    u32x4* const b = reinterpret_cast<u32x4*>(c + (layer + to) * page_bytes + (int64_t)piece * kPiece);
    const int64_t left = page_bytes - (int64_t)piece * kPiece;
    const int n = (int)(left < kPiece ? left : kPiece) / 16;
    u32x4 r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if ((int)threadIdx.x + 256 * j < n) r[j] = a[threadIdx.x + 256 * j];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if ((int)threadIdx.x + 256 * j < n) b[threadIdx.x + 256 * j] = r[j];
    if (piece == 0) {
        float* const sc = which ? vs : ks;
        for (int j = threadIdx.x; j < page_scales; j += 256) sc[(layer + to) * page_scales + j] = sc[(layer + from) * page_scales + j];
    }
}

template <int DP> void launch_store(int dtype, const Pages& a, dim3 grid, const void* k, int64_t k_rs, int64_t k_hs, const void* v, int64_t v_rs, int64_t v_hs,
                                    int aligned, hipStream_t st) {
    if (dtype == DT_BF16) store_kernel<DT_BF16, DP><<<grid, 256, 0, st>>>(a, (const uint16_t*)k, k_rs, k_hs, (const uint16_t*)v, v_rs, v_hs, aligned);
    else store_kernel<DT_F16, DP><<<grid, 256, 0, st>>>(a, (const uint16_t*)k, k_rs, k_hs, (const uint16_t*)v, v_rs, v_hs, aligned);
}

template <int DT> void launch_read(const Pages& a, dim3 grid, void* k, int64_t k_rs, int64_t k_hs, void* v, int64_t v_rs, int64_t v_hs, int aligned, hipStream_t st) {
    if (a.d <= 64) read_kernel<DT, 64><<<grid, 256, 0, st>>>(a, k, k_rs, k_hs, v, v_rs, v_hs, aligned);
    else if (a.d <= 128) read_kernel<DT, 128><<<grid, 256, 0, st>>>(a, k, k_rs, k_hs, v, v_rs, v_hs, aligned);
    else read_kernel<DT, 256><<<grid, 256, 0, st>>>(a, k, k_rs, k_hs, v, v_rs, v_hs, aligned);
}

}  // namespace

GPU_API int gpu_kv8_store(int dtype, const void* k, int64_t k_rs, int64_t k_hs, const void* v, int64_t v_rs, int64_t v_hs, int8_t* ck, int8_t* cv,
                          float* k_scale, float* v_scale, int n_pages, int page, const int32_t* starts, const int32_t* lens, const int32_t* table,
                          int table_cols, int n, int rows, int most, int hk, int head_dim, void* stream) {
    if (dtype != DT_F16 && dtype != DT_BF16) return -4;
    if (!cache_ok(ck, cv, k_scale, v_scale, n_pages, page, hk, head_dim) || !rows_ok(starts, lens, table, table_cols, n, rows, most)) return -1;
    if (n == 0 || rows == 0 || most == 0) return 0;
    if (!k || !v || n > 65535) return -1;
    const int blocks = (int)(((int64_t)most + 2 * kBlock - 2) / kBlock);     // that `most` tokens can touch
    const int64_t grid = (int64_t)blocks * ((2 * (int64_t)hk + 3) / 4);
    if (grid > 0xffffff) return -1;      // 2^32 threads
    const Pages a{ck, cv, k_scale, v_scale, starts, lens, table, n_pages, __builtin_ctz(page), table_cols, hk, head_dim, rows, most};
    const int aligned = (uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0 && (k_rs | k_hs | v_rs | v_hs) % 8 == 0;
    const dim3 g((unsigned)grid, n);
    const hipStream_t st = (hipStream_t)stream;
    if (head_dim <= 64) launch_store<64>(dtype, a, g, k, k_rs, k_hs, v, v_rs, v_hs, aligned, st);
    else if (head_dim <= 128) launch_store<128>(dtype, a, g, k, k_rs, k_hs, v, v_rs, v_hs, aligned, st);
    else launch_store<256>(dtype, a, g, k, k_rs, k_hs, v, v_rs, v_hs, aligned, st);
    KCHECK();
    return 0;
}

GPU_API int gpu_kv8_read(int dtype, void* k, int64_t k_rs, int64_t k_hs, void* v, int64_t v_rs, int64_t v_hs, const int8_t* ck, const int8_t* cv,
                         const float* k_scale, const float* v_scale, int n_pages, int page, const int32_t* starts, const int32_t* lens,
                         const int32_t* table, int table_cols, int n, int rows, int most, int hk, int head_dim, void* stream) {
    if (dtype != DT_F32 && dtype != DT_F16 && dtype != DT_BF16) return -4;
    if (!cache_ok(ck, cv, k_scale, v_scale, n_pages, page, hk, head_dim) || !rows_ok(starts, lens, table, table_cols, n, rows, most)) return -1;
    if (n == 0 || rows == 0 || most == 0) return 0;
    const int four = dtype == DT_F32 ? 16 : 8;
    if (!k || !v || n > 65535 || (uintptr_t)k % four != 0 || (uintptr_t)v % four != 0 || (k_rs | k_hs | v_rs | v_hs) % 4 != 0) return -1;
    const int blocks = (int)(((int64_t)most + 2 * kBlock - 2) / kBlock);
    const int64_t grid = (int64_t)blocks * ((2 * (int64_t)hk + 3) / 4);
    if (grid > 0xffffff) return -1;      // 2^32 threads
    const Pages a{(int8_t*)ck, (int8_t*)cv, (float*)k_scale, (float*)v_scale, starts, lens, table, n_pages, __builtin_ctz(page), table_cols, hk, head_dim, rows, most};
    const dim3 g((unsigned)grid, n);
    const hipStream_t st = (hipStream_t)stream;
    const int aligned = (uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0 && (k_rs | k_hs | v_rs | v_hs) % 8 == 0;
    if (dtype == DT_BF16) launch_read<DT_BF16>(a, g, k, k_rs, k_hs, v, v_rs, v_hs, aligned, st);
    else if (dtype == DT_F16) launch_read<DT_F16>(a, g, k, k_rs, k_hs, v, v_rs, v_hs, aligned, st);
    else launch_read<DT_F32>(a, g, k, k_rs, k_hs, v, v_rs, v_hs, aligned, st);
    KCHECK();
    return 0;
}

GPU_API int gpu_kv8_copy_pages(int8_t* k, int8_t* v, float* k_scale, float* v_scale, int layers, int n_pages, int page, int hk, int head_dim,
                               const int32_t* src, const int32_t* dst, int n, void* stream) {
    if (!cache_ok(k, v, k_scale, v_scale, n_pages, page, hk, head_dim) || layers < 0 || n < 0) return -1;
    if (layers == 0 || n == 0) return 0;
    if (!src || !dst || layers > 65535 || n > 65535) return -1;
    const int64_t bytes = (int64_t)hk * page * head_dim, scales = (int64_t)hk * (page / kBlock);
    const int64_t pieces = (bytes + kPiece - 1) / kPiece;
    if (pieces > 0x7fffff || scales > 0x7fffffff) return -1;
    copy_kernel<<<dim3((unsigned)(2 * pieces), n, layers), 256, 0, (hipStream_t)stream>>>(k, v, k_scale, v_scale, n_pages, bytes, (int)scales, src, dst, (int)pieces);
    KCHECK();
    return 0;
}
