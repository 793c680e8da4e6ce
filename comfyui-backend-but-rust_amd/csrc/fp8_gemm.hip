// e4m3 x e4m3 products with a scale for each row and group of 128 columns of A and for each block of 128 x 128 of W:
//
//   D[m, n] = Out( sum_g xs[g, m] ws[n / 128, g] ( sum_{k in group g} A[m, k] W[n, k] ) + bias[n] )
//
// One v_mfma_f32_16x16x128_f8f6f4 takes a whole group: its 16 x 16 sums start at 0, and a lane folds its four into fp32 accumulators with one
// fma each.  W rides in src0 and A in src1, so a lane has one row m and four consecutive n, and one scale xs ws for all of them: a block of ws
// is never less than a wave tile wide.
//
// That instruction adds the products of each eight k (0 .. 7, 8 .. 15, ...) in units of 2^-13 of the largest's power of two and cuts off what lies
// below; everything else in it is fp32.  On normally distributed operands that is 1.5e-5 of the result, a hundredth of bf16's rounding and a
// twentieth of f16's, and it is what twice the rate costs.  For 32-bit outputs the codes become f16, which they are exactly, and four
// v_mfma_f32_16x16x32_f16 take the group, which add in fp32 (1e-8).
#include "common.hpp"

namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

#define SCHED_FENCE() __builtin_amdgcn_sched_barrier(0)

constexpr int kGroup = 128;
constexpr int64_t kMostGroups = 0xffffffff / 512;      // a launch has fewer than 2^32 threads

struct Fp8Gemm {
    const uint8_t *A, *W;
    const float *xs, *ws;
    const void* bias;
    void* D;
    int64_t xs_rs;
    int M, N, K, groups;
    int tiles_m, tiles_n;
    int rows_ok;      // rows of D start on 16 bytes
    int slices;       // workgroups that share an output's K
    float* planes;    // [slices][M][N] where those are several
};
// Groups g0 .. g1 of slice `s`.
__device__ __forceinline__ void slice_of(int groups, int slices, int s, int& g0, int& g1) {
    const int share = (groups + slices - 1) / slices;
    g0 = min(groups, s * share);
    g1 = min(groups, g0 + share);
}

// Both operands in the instruction's lane order: row lane % 16, and of its 128 bytes the 16-byte chunks lane / 16 and 4 + lane / 16.  (Which
// k a lane holds does not matter as long as both operands agree.)
__device__ __forceinline__ v8i two(v4i a, v4i b) { return v8i{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}; }
__device__ __forceinline__ v4f mfma(v8i w, v8i a, v4f c) { return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, c, 0, 0, 0, 0, 0, 0); }
// Eight codes as f16.
__device__ __forceinline__ v8h widen(int lo, int hi) {
    const auto pair = [](auto h) { return __builtin_bit_cast(uint32_t, h); };
    return __builtin_bit_cast(v8h, v4i{(int)pair(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false)), (int)pair(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true)),
                                       (int)pair(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false)), (int)pair(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true))});
}
// A group's sums for outputs of a type.
template <int OUT_DT> __device__ __forceinline__ v4f product(v8i w, v8i a) {
    v4f d = {0.f, 0.f, 0.f, 0.f};
    if constexpr (OUT_DT == DT_F32) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen(w[e], w[e + 1]), widen(a[e], a[e + 1]), d, 0, 0, 0);
        return d;
    } else return mfma(w, a, d);
}
// Chunk c of row r at slot c ^ ((r >> 1) & 7): 16 rows at one chunk lie on 16 of the 64 banks' 16-byte groups.
__device__ __forceinline__ int place(int row, int chunk) { return row * kGroup + ((chunk ^ ((row >> 1) & 7)) << 4); }

template <int OUT_DT> __device__ __forceinline__ void store_four(const Fp8Gemm& p, int m, int n, v4f v) {
    if (m >= p.M || n >= p.N) return;
    if (p.bias)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n + j < p.N) v[j] += ld_dt<OUT_DT>(p.bias, n + j);
    const int64_t at = (int64_t)m * p.N + n;
    if (p.rows_ok && n + 4 <= p.N) {
        const float f[4] = {v[0], v[1], v[2], v[3]};
        store4<OUT_DT>(p.D, at, f);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n + j < p.N) st_dt<OUT_DT>(p.D, at + j, v[j]);
    }
}

__device__ __forceinline__ void store_plane(const Fp8Gemm& p, int slice, int m, int n, v4f v) {
    if (m >= p.M || n >= p.N) return;
    float* const to = p.planes + ((int64_t)slice * p.M + m) * p.N + n;
    if (p.N % 4 == 0) *reinterpret_cast<v4f*>(to) = v;
    else
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n + j < p.N) to[j] = v[j];
}

// K below 128 or from 2^23 on: tiles of 128 x 128, four waves of 64 x 64, a group at a time through registers into one of two LDS stages.
template <int OUT_DT>
__global__ void __launch_bounds__(256, 2) fp8_gemm_kernel(const Fp8Gemm p) {
    constexpr int STAGE = 128 * kGroup;
    __shared__ __align__(16) uint8_t lds[4 * STAGE];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64, row = lane & 15, part = lane >> 4;
    int tm, tn;
    tile_of_block((int)blockIdx.x, (int)gridDim.x, p.tiles_m, p.tiles_n, tm, tn);
    const int m0 = tm * 128, n0 = tn * 128;
    v4i ra[4], rw[4];
    const auto load = [&](int g) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = tid + 256 * j, r = i >> 3, c = i & 7, k = g * kGroup + 16 * c;
            const bool in = k < p.K;
            ra[j] = rw[j] = v4i{0, 0, 0, 0};
            if (in) {
                ra[j] = *reinterpret_cast<const v4i*>(p.A + (int64_t)min(m0 + r, p.M - 1) * p.K + k);
                rw[j] = *reinterpret_cast<const v4i*>(p.W + (int64_t)min(n0 + r, p.N - 1) * p.K + k);
            }
        }
    };
    const auto write = [&](int stage) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = tid + 256 * j, at = place(i >> 3, i & 7);
            *reinterpret_cast<v4i*>(lds + stage * STAGE + at) = ra[j];
            *reinterpret_cast<v4i*>(lds + (2 + stage) * STAGE + at) = rw[j];
        }
    };
    const auto fragment = [&](const uint8_t* s, int r) {
        return two(*reinterpret_cast<const v4i*>(s + place(r, part)), *reinterpret_cast<const v4i*>(s + place(r, 4 + part)));
    };
    v4f acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
    load(0);
    write(0);
    __syncthreads();
    for (int g = 0; g < p.groups; ++g) {
        if (g + 1 < p.groups) load(g + 1);
        const float ws = p.ws[(int64_t)tn * p.groups + g];
        float s[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = p.xs[g * p.xs_rs + min(m0 + wm + 16 * i + row, p.M - 1)] * ws;
        const uint8_t *sa = lds + (g & 1) * STAGE, *sw = lds + (2 + (g & 1)) * STAGE;
        v8i fa[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) fa[i] = fragment(sa, wm + 16 * i + row);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const v8i fw = fragment(sw, wn + 16 * j + row);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const v4f d = product<OUT_DT>(fw, fa[i]);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(d[e], s[i], acc[i][j][e]);
            }
        }
        if (g + 1 < p.groups) write((g + 1) & 1);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) store_four<OUT_DT>(p, m0 + wm + 16 * i + row, n0 + wn + 16 * j + 4 * part, acc[i][j]);
}

// ---- tiles by DMA ----------------------------------------------------------------------------------------------------------------

__device__ __forceinline__ void dma16(uint32_t lds_dst, uint32_t lane_off, const void* base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_dst), "v"(lane_off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void dma4(uint32_t lds_dst, uint32_t lane_off, const void* base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds_dst), "v"(lane_off), "s"(base) : "memory", "m0");
}
template <int N> __device__ __forceinline__ void wait_vmcnt() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ int lane_now() { return (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)); }

// The scales of a column block's groups from g0 on, for loops that read LDS: a scalar load would have them wait for all of it, so a lane holds a
// group's, of 64 and of the next 64.  (1024 x 4096 -> 4096 in tiles of 128 x 128: 39.9 us with a scalar load a group, 28.9 without.)
struct BlockScales {
    const float* from;
    int lane, last, at = 0;      // the groups that there are; groups done
    float now, next;
    __device__ __forceinline__ BlockScales(const float* ws, int g0, int end, int lane_) : from(ws + g0), lane(lane_), last(end - g0 - 1) {
        now = from[min(lane, last)];
        next = from[min(lane + 64, last)];
    }
    __device__ __forceinline__ float take() {
        const float s = u2f(__builtin_amdgcn_readlane(f2u(now), at & 63));
        if ((++at & 63) == 0) {
            now = next;
            next = from[min(at + 64 + lane, last)];
        }
        return s;
    }
};

// A wave's FM x FN tiles, first row mw, first column nb: rounded, passed 32 rows at a time through `wl`, LDS of its own (32 rows of its columns;
// 16-byte chunks swizzled by row), and stored in whole row segments, 16 bytes a lane.
template <int OUT_DT, int FM, int FN>
__device__ __forceinline__ void store_wave_tile(const Fp8Gemm& p, uint8_t* wl, const v4f (&acc)[FN][FM], int mw, int nb, int lane) {
    static_assert(OUT_DT != DT_F32, "16-bit outputs");
    const int row = lane & 15, part = lane >> 4;
    if (!p.rows_ok) {
#pragma unroll
        for (int in = 0; in < FN; ++in)
#pragma unroll
            for (int im = 0; im < FM; ++im) store_four<OUT_DT>(p, mw + 16 * im + row, nb + 16 * in + 4 * part, acc[in][im]);
        return;
    }
    constexpr int CPR = 2 * FN, RPI = 64 / CPR;      // 16-byte chunks of a row, rows of a store instruction
    float bv[FN][4];
#pragma unroll
    for (int in = 0; in < FN; ++in)
#pragma unroll
        for (int c = 0; c < 4; ++c) bv[in][c] = p.bias && nb + 16 * in + 4 * part + c < p.N ? ld_dt<OUT_DT>(p.bias, nb + 16 * in + 4 * part + c) : 0.f;
#pragma unroll
    for (int ip = 0; ip < FM / 2; ++ip) {
#pragma unroll
        for (int hm = 0; hm < 2; ++hm) {
            const int r = 16 * hm + row;
#pragma unroll
            for (int in = 0; in < FN; ++in) {
                const v4f x = acc[in][2 * ip + hm];
                float v[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) v[c] = x[c] + bv[in][c];
                uint8_t* const to = wl + r * (16 * CPR) + (((2 * in + (part >> 1)) ^ (r & (CPR - 1))) << 4) + 8 * (part & 1);
                *reinterpret_cast<uint2*>(to) = OUT_DT == DT_BF16 ? make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])) : make_uint2(pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]));
            }
        }
        asm volatile("" ::: "memory");      // a wave's LDS accesses stay in order
#pragma unroll
        for (int t = 0; t < 32 / RPI; ++t) {
            const int r = t * RPI + lane / CPR, c = lane % CPR, m = mw + 32 * ip + r, n = nb + 8 * c;
            const uint4 v = *reinterpret_cast<const uint4*>(wl + r * (16 * CPR) + ((c ^ (r & (CPR - 1))) << 4));
            if (m < p.M && n < p.N) *reinterpret_cast<uint4*>((uint16_t*)p.D + (int64_t)m * p.N + n) = v;
        }
        asm volatile("" ::: "memory");
    }
}

// A fragment of the group that is not a whole one, straight from memory: 0 behind K.
__device__ __forceinline__ v8i tail_fragment(const uint8_t* x, int row, int limit, int K, int k0, int part) {
    const uint8_t* const at = x + (int64_t)min(row, limit - 1) * K + k0;
    v4i a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
    if (k0 + 16 * part < K) a = *reinterpret_cast<const v4i*>(at + 16 * part);
    if (k0 + 64 + 16 * part < K) b = *reinterpret_cast<const v4i*>(at + 64 + 16 * part);
    return two(a, b);
}

// Large sizes: tiles of 256 x 256, eight waves of 128 x 64, two LDS stages: group g + 1 travels while group g is multiplied, one barrier a group.
// Bound by power: 8192 x 4096 -> 24576 710 to 745 us by the box, 2.2 to 2.3 PFLOP/s, matrix pipes 58 % busy at 1.73 GHz (a library product with one scale, which has no folds, 2.98
// PFLOP/s on 8192 cubed; this 2.48).  Not faster: products of 32 x 32 x 64 (730), waves that take turns at multiplying and fetching (862), the next group's
// first fragments under the last products (727: its rows have to land earlier for that).
constexpr int BIG = 256, BIG_STAGE = BIG * kGroup, BIG_S = 4 * BIG_STAGE, BIG_LDS = BIG_S + 2 * BIG * 4;

template <int OUT_DT>
__global__ void __launch_bounds__(512, 1) fp8_gemm_big_kernel(const Fp8Gemm p) {
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 2, wn = wave & 3;
    int tm, tn;
    tile_of_block((int)blockIdx.x, (int)gridDim.x, p.tiles_m, p.tiles_n, tm, tn);
    const int m0 = tm * BIG, n0 = tn * BIG, full = p.K / kGroup;
    const uint32_t lds_base = (uint32_t)(uintptr_t)smem;
    constexpr int FM = 8, FN = 4;

    // The lower waves fetch: 8-row blocks wn + 4 j of W and of A, the swizzle on the memory's side, and the scales of rows 64 wn ..
    const uint32_t lrow = (uint32_t)lane >> 3, K = (uint32_t)p.K;
    const uint32_t chunk = ((lane & 7) ^ (((wn & 1) << 2) | (lrow >> 1))) * 16, drow = wn * 8 + lrow;
    const uint32_t w_last = (uint32_t)min(BIG - 1, p.N - 1 - n0), a_last = (uint32_t)min(BIG - 1, p.M - 1 - m0);
    const uint32_t s_off = 4u * min((uint32_t)(64 * wn + lane), a_last);
    const uint8_t *const a_base = p.A + (int64_t)m0 * p.K, *const w_base = p.W + (int64_t)n0 * p.K;
    const float* const s_base = p.xs + m0;
    constexpr int NDMA = 17;
    const auto dma = [&](int g, int j) {      // groups past the end fetch the last one again, which nothing reads
        const int gc = g < full ? g : full - 1, stage = g & 1;
        if (j < 8) dma16(lds_base + (2 + stage) * BIG_STAGE + (wn + 4 * j) * 1024, __umul24(min(drow + 32 * j, w_last), K) + chunk, w_base + (int64_t)gc * kGroup);
        else if (j < 16) dma16(lds_base + stage * BIG_STAGE + (wn + 4 * (j - 8)) * 1024, __umul24(min(drow + 32 * (j - 8), a_last), K) + chunk, a_base + (int64_t)gc * kGroup);
        else dma4(lds_base + BIG_S + stage * (BIG * 4) + wn * 256, s_off, s_base + gc * p.xs_rs);
    };
    const int frow = lane & 15, part = lane >> 4;
    const int fsw = (part ^ ((frow >> 1) & 7)) << 4, aoff = (wm * 128 + frow) * kGroup + fsw, woff = (wn * 64 + frow) * kGroup + fsw;
    // (waves whose columns lie behind N take any block's scales)
    const float* const ws = p.ws + (int64_t)min((n0 + wn * 64) / kGroup, (p.N - 1) / kGroup) * p.groups;

    v4f sums[2][FN], acc[FN][FM];      // a group's sums of a row tile and of the one before
    float s[2];
#pragma unroll
    for (int in = 0; in < FN; ++in) {
        sums[1][in] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int im = 0; im < FM; ++im) acc[in][im] = v4f{0.f, 0.f, 0.f, 0.f};
    }
    s[1] = 0.f;
    const auto fold = [&](int buf, int in, int im) {
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[in][im][c] = fmaf(sums[buf][in][c], s[buf], acc[in][im][c]);
    };
    // No branch inside: the compiler would move the folds behind it.
    const auto loop = [&](auto fetches_tag) {
        constexpr bool fetches = decltype(fetches_tag)::value;
        if constexpr (fetches) {
#pragma unroll
            for (int j = 0; j < NDMA; ++j) dma(0, j);
            wait_vmcnt<0>();
        }
        __syncthreads();
        BlockScales scales(ws, 0, full, lane);
        for (int g = 0; g < full; ++g) {
            const uint8_t *sa = smem + (g & 1) * BIG_STAGE, *sw = smem + (2 + (g & 1)) * BIG_STAGE;
            const float* const sx = reinterpret_cast<const float*>(smem + BIG_S + (g & 1) * (BIG * 4)) + wm * 128 + frow;
            const float wg = scales.take();
            v8i fw[FN], fa[2];
            const auto read = [&](const uint8_t* from, int off) { return two(*reinterpret_cast<const v4i*>(from + off), *reinterpret_cast<const v4i*>(from + (off ^ 64))); };
            fa[0] = read(sa, aoff);
#pragma unroll
            for (int in = 0; in < FN; ++in) fw[in] = read(sw, woff + in * 16 * kGroup);
            SCHED_FENCE();
#pragma unroll
            for (int in = 0; in < FN; ++in) fold(1, in, FM - 1);      // the last row tile of the group before, under the first reads of this one
            SCHED_FENCE();
#pragma unroll
            for (int im = 0; im < FM; ++im) {
                if (im + 1 < FM) fa[(im + 1) & 1] = read(sa, aoff + (im + 1) * 16 * kGroup);
                s[im & 1] = sx[16 * im] * wg;
#pragma unroll
                for (int in = 0; in < FN; ++in) sums[im & 1][in] = mfma(fw[in], fa[im & 1], v4f{0.f, 0.f, 0.f, 0.f});
                SCHED_FENCE();
#pragma unroll
                for (int in = 0; in < FN; ++in) {
                    const int j = im * 3 + in;
                    if (im > 0) fold((im - 1) & 1, in, im - 1);
                    SCHED_FENCE();
                    if (fetches && in < 3 && j < NDMA) dma(g + 1, j);      // the stage last read before the previous barrier
                    SCHED_FENCE();
                }
            }
            if constexpr (fetches) wait_vmcnt<0>();
            __syncthreads();
        }
    };
    if (wm == 0) loop(std::true_type{});
    else loop(std::false_type{});
#pragma unroll
    for (int in = 0; in < FN; ++in) fold(1, in, FM - 1);
    if (p.K > full * kGroup) {
        const int k0 = full * kGroup, r = lane_now() & 15, c = lane_now() >> 4;
        v8i fw[FN];
#pragma unroll
        for (int in = 0; in < FN; ++in) fw[in] = tail_fragment(p.W, n0 + wn * 64 + 16 * in + r, p.N, p.K, k0, c);
#pragma unroll
        for (int im = 0; im < FM; ++im) {
            const int m = m0 + wm * 128 + 16 * im + r;
            const v8i fa = tail_fragment(p.A, m, p.M, p.K, k0, c);
            s[0] = p.xs[full * p.xs_rs + min(m, p.M - 1)] * ws[full];
#pragma unroll
            for (int in = 0; in < FN; ++in) sums[0][in] = mfma(fw[in], fa, v4f{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int in = 0; in < FN; ++in) fold(0, in, im);
        }
    }
    // (the stages are idle; the lane number is taken anew so that the loop does not keep it)
    store_wave_tile<OUT_DT, FM, FN>(p, smem + wave * 4096, acc, m0 + wm * 128, n0 + wn * 64, lane_now());
}

template <int OUT_DT> int launch_big(Fp8Gemm p, hipStream_t st) {
    const auto kern = fp8_gemm_big_kernel<OUT_DT>;
    p.tiles_m = (p.M + BIG - 1) / BIG;
    p.tiles_n = (p.N + BIG - 1) / BIG;
    if ((int64_t)p.tiles_m * p.tiles_n > kMostGroups) return -1;
    static PerDeviceOnce once;
    if (const int e = allow_dynamic_lds((const void*)kern, BIG_LDS, once)) return e;
    hipLaunchKernelGGL(kern, dim3((unsigned)(p.tiles_m * p.tiles_n)), dim3(512), BIG_LDS, st, p);
    KCHECK();
    return 0;
}

// Few tiles: 64 or 128 rows by 128 columns, four waves that multiply (2 x 2 of BM / 2 x 64) and four that do nothing but fetch, into a ring of LDS
// stages; K in slices over workgroups where the tiles are fewer than CUs.  At the barrier before group g the groups up to g + 1 have landed, so
// that the first fragments of the next group are read behind the last products of this one; the stage of group g - 1 is fetched into.
template <int BM> struct Mid {
    static constexpr int BN = 128, STAGE = (BM + BN) * kGroup, SCALES = 128 * 4, NS = BM == 128 ? 4 : 6, LDS = NS * (STAGE + SCALES);
    static constexpr int FM = BM / 32, FN = 4, NDMA = (BM + BN) / 32 + 1;      // of a fetching wave and group
};

template <int BM, int OUT_DT>
__global__ void __launch_bounds__(512, 1) fp8_gemm_mid_kernel(const Fp8Gemm p) {
    using C = Mid<BM>;
    constexpr int FM = C::FM, FN = C::FN;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles = p.tiles_m * p.tiles_n, slice = blockIdx.x / tiles;
    int tm, tn;
    tile_of_block((int)blockIdx.x - slice * tiles, tiles, p.tiles_m, p.tiles_n, tm, tn);
    const int m0 = tm * BM, n0 = tn * C::BN;
    int g0, g1;
    slice_of(p.groups, p.slices, slice, g0, g1);
    const bool tail = g1 == p.groups && g0 < g1 && p.K % kGroup != 0;
    const int end = tail ? g1 - 1 : g1, n = end - g0;      // whole groups
    const auto meet = [] {
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    if (wave >= 4) {
        if (n <= 0) return;      // (no barrier is waited for then)
        // 8-row blocks w + 4 j, of A and then of W; the swizzle on the memory's side.  The scales of the rows 64 (w % 2) .., by two waves alike.
        const int w = wave - 4;
        const uint32_t lds_base = (uint32_t)(uintptr_t)smem, lrow = (uint32_t)lane >> 3, K = (uint32_t)p.K;
        const uint32_t chunk = ((lane & 7) ^ (((w & 1) << 2) | (lrow >> 1))) * 16, drow = w * 8 + lrow;
        const uint32_t w_last = (uint32_t)min(C::BN - 1, p.N - 1 - n0), a_last = (uint32_t)min(BM - 1, p.M - 1 - m0);
        uint32_t off[C::NDMA - 1];
#pragma unroll
        for (int j = 0; j < C::NDMA - 1; ++j) off[j] = (j < BM / 32 ? min(drow + 32 * j, a_last) : min(drow + 32 * (j - BM / 32), w_last)) * K + chunk;
        const uint32_t s_off = 4u * min((uint32_t)(64 * (w & 1) + lane), a_last);
        const uint8_t *const a_base = p.A + (int64_t)m0 * p.K, *const w_base = p.W + (int64_t)n0 * p.K;
        const float* const s_base = p.xs + m0;
        int put = 0;
        const auto fetch = [&](int g) {      // groups past the end fetch the last one again, which nothing reads
            const int gc = g < end ? g : end - 1;
            const uint32_t to = lds_base + put * C::STAGE + w * 1024;
#pragma unroll
            for (int j = 0; j < C::NDMA - 1; ++j) dma16(to + j * 4096, off[j], (j < BM / 32 ? a_base : w_base) + (int64_t)gc * kGroup);
            dma4(lds_base + C::NS * C::STAGE + put * C::SCALES + (w & 1) * 256, s_off, s_base + gc * p.xs_rs);
            put = put == C::NS - 1 ? 0 : put + 1;
        };
#pragma unroll
        for (int i = 0; i < C::NS - 1; ++i) fetch(g0 + i);
        for (int i = 0; i < n; ++i) {
            wait_vmcnt<(C::NS - 3) * C::NDMA>();
            meet();
            if (i + 1 < n) fetch(g0 + i + C::NS - 1);
        }
        wait_vmcnt<0>();      // nothing may still be writing this workgroup's LDS when it retires, or is stored through
        meet();
        return;
    }
    const int wm = wave >> 1, wn = wave & 1, frow = lane & 15, part = lane >> 4;
    const int fsw = (part ^ ((frow >> 1) & 7)) << 4, aoff = (wm * (BM / 2) + frow) * kGroup + fsw, woff = (BM + wn * 64 + frow) * kGroup + fsw;
    const float* const ws = p.ws + (int64_t)tn * p.groups;
    v4f acc[FN][FM], sums[2][FN];
    float last = 0.f;      // the scale of the row tile that is not folded yet
#pragma unroll
    for (int in = 0; in < FN; ++in) {
        sums[(FM - 1) & 1][in] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int im = 0; im < FM; ++im) acc[in][im] = v4f{0.f, 0.f, 0.f, 0.f};
    }
    const auto fold = [&](int buf, int in, int im, float s) {
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[in][im][c] = fmaf(sums[buf][in][c], s, acc[in][im][c]);
    };
    struct First {      // what a group begins with
        v8i w[FN], a;
        float s[FM], ws;
    };
    int get = 0;
    const auto read = [&](const uint8_t* at, int o) { return two(*reinterpret_cast<const v4i*>(at + o), *reinterpret_cast<const v4i*>(at + (o ^ 64))); };
    const auto begin = [&](First& f) {      // of the stage `get`
        const uint8_t* const at = smem + get * C::STAGE;
        const float* const sx = reinterpret_cast<const float*>(smem + C::NS * C::STAGE + get * C::SCALES) + wm * (BM / 2) + frow;
        f.a = read(at, aoff);
#pragma unroll
        for (int in = 0; in < FN; ++in) f.w[in] = read(at, woff + in * 16 * kGroup);
#pragma unroll
        for (int im = 0; im < FM; ++im) f.s[im] = sx[16 * im];
    };
    // A group's products; what the next one begins with is read a piece under each row tile (all of it under the last one: 1024 x 16384 -> 4096 84 us
    // for 76, since the four waves then wait for LDS at once).
    const auto group = [&](First& f, First& next) {
        const uint8_t* const at = smem + get * C::STAGE;
        get = get == C::NS - 1 ? 0 : get + 1;
        const uint8_t* const nx = smem + get * C::STAGE;
        const float* const sx = reinterpret_cast<const float*>(smem + C::NS * C::STAGE + get * C::SCALES) + wm * (BM / 2) + frow;
        v8i fa[2];
        fa[0] = f.a;
#pragma unroll
        for (int im = 0; im < FM; ++im) {
            if (im + 1 < FM) fa[(im + 1) & 1] = read(at, aoff + (im + 1) * 16 * kGroup);
            else {
                next.a = read(nx, aoff);
#pragma unroll
                for (int i = 0; i < FM; ++i) next.s[i] = sx[16 * i];
            }
#pragma unroll
            for (int in = im * FN / FM; in < (im + 1) * FN / FM; ++in) next.w[in] = read(nx, woff + in * 16 * kGroup);
            SCHED_FENCE();
            const int done = im ? im - 1 : FM - 1;
            const float s = im ? f.s[im - 1] * f.ws : last;
            // the products of this row tile, and the fold of the one before between them
#pragma unroll
            for (int in = 0; in < FN; ++in) {
                const v4f d = mfma(f.w[in], fa[im & 1], v4f{0.f, 0.f, 0.f, 0.f});
                fold(done & 1, in, done, s);
                sums[im & 1][in] = d;
                SCHED_FENCE();
            }
        }
        last = f.s[FM - 1] * f.ws;
    };
    static_assert(FM % 2 == 0, "row tiles alternate between two sets of sums");
    if (n > 0) {
        BlockScales scales(ws, g0, end, lane);
        First f[2];
        meet();
        begin(f[0]);
        f[0].ws = scales.take();
        int g = g0;
        if (n & 1) {      // (so that the loop has no way out in its middle, for which the compiler would move all sums)
            f[1].ws = scales.take();
            group(f[0], f[1]);
            meet();
            f[0] = f[1];
            ++g;
        }
        for (; g < end; g += 2) {
            f[1].ws = scales.take();      // (here and not among the products: it has a branch, behind which the compiler would move the folds)
            group(f[0], f[1]);
            meet();                       // (behind the last group: the fetching waves' last)
            f[0].ws = scales.take();
            group(f[1], f[0]);
            meet();
        }
#pragma unroll
        for (int in = 0; in < FN; ++in) fold((FM - 1) & 1, in, FM - 1, last);
    }
    if (tail) {
        const int k0 = end * kGroup;
        v8i fw[FN];
#pragma unroll
        for (int in = 0; in < FN; ++in) fw[in] = tail_fragment(p.W, n0 + wn * 64 + 16 * in + frow, p.N, p.K, k0, part);
#pragma unroll
        for (int im = 0; im < FM; ++im) {
            const int m = m0 + wm * (BM / 2) + 16 * im + frow;
            const v8i fa = tail_fragment(p.A, m, p.M, p.K, k0, part);
            const float s = p.xs[end * p.xs_rs + min(m, p.M - 1)] * ws[end];
#pragma unroll
            for (int in = 0; in < FN; ++in) {
                const v4f d = product<OUT_DT>(fw[in], fa);
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[in][im][c] = fmaf(d[c], s, acc[in][im][c]);
            }
        }
    }
    if (p.slices > 1) {      // (16 bytes a lane, 64 in a row)
#pragma unroll
        for (int in = 0; in < FN; ++in)
#pragma unroll
            for (int im = 0; im < FM; ++im) {
                const int m = m0 + wm * (BM / 2) + 16 * im + frow, n = n0 + wn * 64 + 16 * in + 4 * part;
                store_plane(p, slice, m, n, acc[in][im]);
            }
    } else store_wave_tile<OUT_DT, FM, FN>(p, smem + wave * 4096, acc, m0 + wm * (BM / 2), n0 + wn * 64, lane);      // (the stages are idle)
}

// One to two tiles a CU, and 32-bit outputs: tiles of 64 or 128 rows by 128 columns, eight waves of BM / 2 x 32 that all fetch and multiply, so that one's
// conversions to f16 run beside another's products, in two or three LDS stages, so that a CU has two workgroups (2048 x 4096 -> 4096, 32-bit: 76 us; 88 with four stages and one).
// With 32-bit outputs bound by vector issue (52 %) and the matrix pipes (38 %), which hardly overlap; 32 x 32 x 16 products are no faster (78).
template <int BM> struct Wide {
    static constexpr int BN = 128, STAGE = (BM + BN) * kGroup, SCALES = 128 * 4, NS = BM == 128 ? 2 : 3, LDS = NS * (STAGE + SCALES);
    static constexpr int FM = BM / 32, FN = 2, NDMA = (BM + BN) / 64 + 1;      // of a wave and group
};

template <int BM, int OUT_DT>
__global__ void __launch_bounds__(512, 2) fp8_gemm_wide_kernel(const Fp8Gemm p) {
    using C = Wide<BM>;
    constexpr int FM = C::FM, FN = C::FN;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 2, wn = wave & 3;
    const int tiles = p.tiles_m * p.tiles_n, slice = blockIdx.x / tiles;
    int tm, tn;
    tile_of_block((int)blockIdx.x - slice * tiles, tiles, p.tiles_m, p.tiles_n, tm, tn);
    const int m0 = tm * BM, n0 = tn * C::BN;
    int g0, g1;
    slice_of(p.groups, p.slices, slice, g0, g1);
    const bool tail = g1 == p.groups && g0 < g1 && p.K % kGroup != 0;
    const int end = tail ? g1 - 1 : g1, n = end - g0;      // whole groups

    // DMA: 8-row blocks wave + 8 j, of A and then of W; the swizzle on the memory's side.  The scales of the rows 64 (wave % 2) .., by four waves alike.
    const uint32_t lds_base = (uint32_t)(uintptr_t)smem, lrow = (uint32_t)lane >> 3, K = (uint32_t)p.K;
    const uint32_t chunk = ((lane & 7) ^ (((wave & 1) << 2) | (lrow >> 1))) * 16, drow = wave * 8 + lrow;
    const uint32_t w_last = (uint32_t)min(C::BN - 1, p.N - 1 - n0), a_last = (uint32_t)min(BM - 1, p.M - 1 - m0);
    uint32_t off[C::NDMA - 1];
#pragma unroll
    for (int j = 0; j < C::NDMA - 1; ++j) off[j] = (j < BM / 64 ? min(drow + 64 * j, a_last) : min(drow + 64 * (j - BM / 64), w_last)) * K + chunk;
    const uint32_t s_off = 4u * min((uint32_t)(64 * (wave & 1) + lane), a_last);
    const uint8_t *const a_base = p.A + (int64_t)m0 * p.K, *const w_base = p.W + (int64_t)n0 * p.K;
    const float* const s_base = p.xs + m0;
    int put = 0;
    const auto fetch = [&](int g) {      // groups past the end fetch the last one again, which nothing reads
        const int gc = g < end ? g : end - 1;
        const uint32_t to = lds_base + put * C::STAGE + wave * 1024;
#pragma unroll
        for (int j = 0; j < C::NDMA - 1; ++j) dma16(to + j * 8192, off[j], (j < BM / 64 ? a_base : w_base) + (int64_t)gc * kGroup);
        dma4(lds_base + C::NS * C::STAGE + put * C::SCALES + (wave & 1) * 256, s_off, s_base + gc * p.xs_rs);
        put = put == C::NS - 1 ? 0 : put + 1;
    };
    const int frow = lane & 15, part = lane >> 4;
    const int fsw = (part ^ ((frow >> 1) & 7)) << 4, aoff = (wm * (BM / 2) + frow) * kGroup + fsw, woff = (BM + wn * 32 + frow) * kGroup + fsw;
    const float* const ws = p.ws + (int64_t)tn * p.groups;
    v4f acc[FN][FM];
#pragma unroll
    for (int in = 0; in < FN; ++in)
#pragma unroll
        for (int im = 0; im < FM; ++im) acc[in][im] = v4f{0.f, 0.f, 0.f, 0.f};
    const auto read = [&](const uint8_t* at, int o) { return two(*reinterpret_cast<const v4i*>(at + o), *reinterpret_cast<const v4i*>(at + (o ^ 64))); };
    if (n > 0) {
        BlockScales scales(ws, g0, end, lane);
        asm volatile("" : "+v"(scales.now), "+v"(scales.next));      // (here, or the compiler waits for them, and so for all rows on their way, in every group)
#pragma unroll
        for (int i = 0; i < C::NS - 1; ++i) fetch(g0 + i);
        int get = 0;
        for (int g = g0; g < end; ++g) {
            const float wg = scales.take();
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // (what was read from is fetched into next)
            wait_vmcnt<(C::NS - 2) * C::NDMA>();
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            fetch(g + C::NS - 1);
            const uint8_t* const at = smem + get * C::STAGE;
            const float* const sx = reinterpret_cast<const float*>(smem + C::NS * C::STAGE + get * C::SCALES) + wm * (BM / 2) + frow;
            get = get == C::NS - 1 ? 0 : get + 1;
            v8i fw[FN], fa[FM];
            float s[FM];
#pragma unroll
            for (int in = 0; in < FN; ++in) fw[in] = read(at, woff + in * 16 * kGroup);
#pragma unroll
            for (int im = 0; im < FM; ++im) fa[im] = read(at, aoff + im * 16 * kGroup);
#pragma unroll
            for (int im = 0; im < FM; ++im) s[im] = sx[16 * im] * wg;
#pragma unroll
            for (int i2 = 0; i2 < FM; i2 += 2) {
                v4f d[2][FN];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int in = 0; in < FN; ++in) {
                        d[i][in] = v4f{0.f, 0.f, 0.f, 0.f};
                        if constexpr (OUT_DT != DT_F32) d[i][in] = mfma(fw[in], fa[i2 + i], d[i][in]);
                    }
                if constexpr (OUT_DT == DT_F32)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        v8h w[FN];
#pragma unroll
                        for (int in = 0; in < FN; ++in) w[in] = widen(fw[in][2 * e], fw[in][2 * e + 1]);
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const v8h x = widen(fa[i2 + i][2 * e], fa[i2 + i][2 * e + 1]);
#pragma unroll
                            for (int in = 0; in < FN; ++in) d[i][in] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[in], x, d[i][in], 0, 0, 0);
                        }
                    }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int in = 0; in < FN; ++in)
#pragma unroll
                        for (int c = 0; c < 4; ++c) acc[in][i2 + i][c] = fmaf(d[i][in][c], s[i2 + i], acc[in][i2 + i][c]);
            }
        }
        wait_vmcnt<0>();      // nothing may still be writing this workgroup's LDS when it retires
    }
    if (tail) {
        const int k0 = end * kGroup;
        v8i fw[FN];
#pragma unroll
        for (int in = 0; in < FN; ++in) fw[in] = tail_fragment(p.W, n0 + wn * 32 + 16 * in + frow, p.N, p.K, k0, part);
#pragma unroll
        for (int im = 0; im < FM; ++im) {
            const int m = m0 + wm * (BM / 2) + 16 * im + frow;
            const v8i fa = tail_fragment(p.A, m, p.M, p.K, k0, part);
            const float s = p.xs[end * p.xs_rs + min(m, p.M - 1)] * ws[end];
#pragma unroll
            for (int in = 0; in < FN; ++in) {
                const v4f d = product<OUT_DT>(fw[in], fa);
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[in][im][c] = fmaf(d[c], s, acc[in][im][c]);
            }
        }
    }
    if constexpr (OUT_DT != DT_F32) {
        __syncthreads();      // (the stages are idle)
        store_wave_tile<OUT_DT, FM, FN>(p, smem + wave * 4096, acc, m0 + wm * (BM / 2), n0 + wn * 32, lane);
    } else
#pragma unroll
        for (int in = 0; in < FN; ++in)
#pragma unroll
            for (int im = 0; im < FM; ++im) {      // (16 bytes a lane, 64 in a row)
                const int m = m0 + wm * (BM / 2) + 16 * im + frow, c = n0 + wn * 32 + 16 * in + 4 * part;
                if (p.slices > 1) store_plane(p, slice, m, c, acc[in][im]);
                else store_four<OUT_DT>(p, m, c, acc[in][im]);
            }
}

// Few rows: the weights' way in is what counts.  They go from memory straight into the operand of the matrix instruction, as do the rows of A (from
// the caches): eight waves on the same 16 MT rows and 16 CT columns, each with every eighth group of K, two on their way; the waves' sums meet in
// LDS and are added in their order.  Bound by memory: 5 x 4096 -> 24576 21 us, 4.8 TB/s.
template <int MT, int CT, int OUT_DT>
__global__ void __launch_bounds__(512) fp8_gemm_few_kernel(const Fp8Gemm p) {
    constexpr int TILES = MT * CT;
    __shared__ __align__(16) float meet[8 * TILES * 256];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = lane & 15, part = lane >> 4;
    const int slice = blockIdx.x / p.tiles_n, n0 = (blockIdx.x - slice * p.tiles_n) * 16 * CT;
    int g0, g1;
    slice_of(p.groups, p.slices, slice, g0, g1);
    const uint8_t *wp[CT], *ap[MT];
    const float* sp[MT];
#pragma unroll
    for (int c = 0; c < CT; ++c) wp[c] = p.W + (int64_t)min(n0 + 16 * c + row, p.N - 1) * p.K + 16 * part;
#pragma unroll
    for (int m = 0; m < MT; ++m) ap[m] = p.A + (int64_t)min(16 * m + row, p.M - 1) * p.K + 16 * part, sp[m] = p.xs + min(16 * m + row, p.M - 1);
    const float* const ws = p.ws + (int64_t)(n0 / kGroup) * p.groups;
    struct Group {
        v8i w[CT], a[MT];
        float s[MT], ws;
    };
    const auto load = [&](Group& x, int g) {
        const int k0 = g * kGroup;
        const auto at = [&](const uint8_t* q) {
            if (k0 + kGroup <= p.K) return two(*reinterpret_cast<const v4i*>(q + k0), *reinterpret_cast<const v4i*>(q + k0 + 64));
            v4i a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
            if (k0 + 16 * part < p.K) a = *reinterpret_cast<const v4i*>(q + k0);
            if (k0 + 64 + 16 * part < p.K) b = *reinterpret_cast<const v4i*>(q + k0 + 64);
            return two(a, b);
        };
#pragma unroll
        for (int c = 0; c < CT; ++c) x.w[c] = at(wp[c]);
#pragma unroll
        for (int m = 0; m < MT; ++m) x.a[m] = at(ap[m]), x.s[m] = sp[m][g * p.xs_rs];
        x.ws = ws[g];
    };
    v4f acc[CT][MT];
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[c][m] = v4f{0.f, 0.f, 0.f, 0.f};
    const auto multiply = [&](const Group& x) {
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const v4f d = product<OUT_DT>(x.w[c], x.a[m]);
                const float s = x.s[m] * x.ws;
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[c][m][e] = fmaf(d[e], s, acc[c][m][e]);
            }
    };
    Group x[2];
    int g = g0 + wave;
    if (g < g1) load(x[0], g);
    if (g + 8 < g1) load(x[1], g + 8);
    for (; g < g1; g += 16) {
        multiply(x[0]);
        if (g + 16 < g1) load(x[0], g + 16);
        if (g + 8 < g1) multiply(x[1]);
        if (g + 24 < g1) load(x[1], g + 24);
    }
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int m = 0; m < MT; ++m) *reinterpret_cast<v4f*>(meet + ((wave * CT + c) * MT + m) * 256 + 4 * lane) = acc[c][m];
    __syncthreads();
    for (int i = threadIdx.x; i < TILES * 64; i += 512) {      // four outputs of a row
        const int tile = i >> 6, l = i & 63, m = 16 * (tile % MT) + (l & 15), n = n0 + 16 * (tile / MT) + 4 * (l >> 4);
        v4f v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 8; ++w) v += *reinterpret_cast<const v4f*>(meet + (w * TILES + tile) * 256 + 4 * l);
        if (p.slices > 1) store_plane(p, slice, m, n, v);
        else store_four<OUT_DT>(p, m, n, v);
    }
}

// The planes of a K in slices, added in their order.
template <int OUT_DT> __global__ void __launch_bounds__(256) fp8_gemm_join_kernel(const Fp8Gemm p) {
    const int64_t size = (int64_t)p.M * p.N;
    for (int64_t i = 4 * ((int64_t)blockIdx.x * 256 + threadIdx.x); i < size; i += 4 * 256 * (int64_t)gridDim.x) {
        if (p.N % 4 == 0) {
            v4f v = *reinterpret_cast<const v4f*>(p.planes + i);
            for (int s = 1; s < p.slices; ++s) v += *reinterpret_cast<const v4f*>(p.planes + s * size + i);
            const int m = (int)(i / p.N);
            store_four<OUT_DT>(p, m, (int)(i - (int64_t)m * p.N), v);
        } else
            for (int e = 0; e < 4 && i + e < size; ++e) {
                float v = p.planes[i + e];
                for (int s = 1; s < p.slices; ++s) v += p.planes[s * size + i + e];
                const int n = (int)((i + e) % p.N);
                st_dt<OUT_DT>(p.D, i + e, p.bias ? v + ld_dt<OUT_DT>(p.bias, n) : v);
            }
    }
}

// How a call runs.
enum Form { kAny, kBig, kMid128, kMid64, kFew, kWide };
struct Plan {
    int form, slices, ct;
};
std::atomic<int> g_force{-1};      // test hook: 100 * form + slices

// Slices of a few rows' K where there are fewer workgroups than CUs: the eight waves of one share 24 groups at least, or the joining costs more than
// it saves (16 x 4096 -> 1024: 6.3 us in one slice, 6.9 in two; 8 x 12288 -> 512: 11.2 in one, 7.6 in four).  Two column tiles a wave where that
// leaves two workgroups a CU.
// Else the smallest sum of rounds of one workgroup a CU, in us: a fixed time, and one for every group of 128, which grows from `alone` with the share of
// the CUs that are busy (the caches' and the memory's rates) to `full`; slices are joined for 3 us, 0.35 for each, and their planes' way out and
// in.  Fitted to 117 sizes of 33 to 3000 rows in up to 14 forms each, weights from memory: 0.25 % slower than the best of them in the mean, 7 % at most.
// 64 rows: 4.2 + 0.36 .. 0.45 (64 x 4096 -> 24576 29 us), 128 rows: 4.5 + 0.50 .. 0.62 (1024 x 4096 -> 4096 23 us; 35 with 64 rows), 256 x 256: 6 + 1.3 ..
// 1.65 (2048 x 4096 -> 24576 185 us; 270 with 128 rows).  128 rows with two workgroups on a CU where there are so many, for which the fixed time comes once: 5.5 + 0.48
// .. 1.19 for both's groups (2048 x 4096 -> 4096 43 us; 46 with one at a time, 52 in tiles of 256 x 256; 700 x 1024 -> 6144 13, 16 and 16).
// 32-bit outputs: two workgroups run on a CU but no faster than one behind the other, so a fixed time of 5 us and 0.62 (64 rows) or 1.02 (128) for every group and workgroup of a CU
// (2048 x 4096 -> 4096 72 us in 128 rows, 85 in 64; 1024 x 4096 -> 1024 26 in one slice of 64 rows, 22 in four).  Of 72 sizes of 33 to 4096 rows 1 % slower than the best in the mean.
Plan plan_of(int64_t M, int64_t N, int64_t K, int out_dt) {
    const int64_t cus = device_cu_count(), groups = (K + kGroup - 1) / kGroup;
    Plan p{kAny, 1, (N + 31) / 32 >= 2 * cus ? 2 : 1};
    const bool fits = K >= kGroup && K < (1 << 23);
    // (as many as have groups: slices of ceil(groups / s) may use them up before the last, which would begin behind the scales)
    const auto at_most = [&](int64_t s) {
        s = s < 1 ? 1 : s > groups ? groups : s > 32 ? 32 : s;
        const int64_t share = (groups + s - 1) / s;
        return (int)((groups + share - 1) / share);
    };
    const int force = g_force.load(std::memory_order_relaxed);
    if (force >= 0) {
        p.form = force / 100;
        p.slices = at_most(force % 100);
        if ((p.form == kFew && M > 32) || (p.form != kFew && !fits) || ((p.form == kBig || p.form == kWide) && out_dt == DT_F32)) p.form = kAny;
        if (p.form == kAny || p.form == kBig || p.form == kWide) p.slices = 1;
        return p;
    }
    const int64_t tiles = (N + 16 * p.ct - 1) / (16 * p.ct);
    if (M <= 32 && tiles <= kMostGroups) {
        p.form = kFew;
        p.slices = at_most(groups / 24 < cus / tiles ? groups / 24 : cus / tiles);
        return p;
    }
    if (!fits) return p;
    static const struct {
        Form form;
        int bm, bn;
        double start, alone, full;
    } halves[] = {{kMid64, 64, 128, 4.2, 0.36, 0.45}, {kMid128, 128, 128, 4.5, 0.50, 0.62}, {kBig, 256, 256, 6.0, 1.3, 1.65}, {kWide, 128, 128, 5.5, 0.48, 1.19}},
      wide[] = {{kMid64, 64, 128, 5.0, 0.62, 0.62}, {kMid128, 128, 128, 5.0, 1.02, 1.02}};
    const bool words = out_dt == DT_F32;
    const int most = at_most(groups);
    double least = 0.;
    for (int i = 0; i < (words ? 2 : 4); ++i) {
        const auto& f = words ? wide[i] : halves[i];
        const int64_t tiles = ((M + f.bm - 1) / f.bm) * ((N + f.bn - 1) / f.bn);
        for (int s = 1; s == 1 || (f.form != kBig && f.form != kWide && s <= most && tiles * s <= 2 * cus); ++s) {
            const int64_t slots = f.form == kWide ? 2 * cus : cus, whole = tiles * s / slots, left = tiles * s % slots, steps = (groups + s - 1) / s;
            if ((s - 1) * steps >= groups || tiles * s > kMostGroups) continue;      // (larger tiles where a launch does not hold so many; where it holds none of them, the form for any size)
            const double part = left ? f.alone + (f.full - f.alone) * left / slots : 0.;      // of the last round's groups
            const double us = (f.form == kWide ? f.start + (whole * f.full + part) * steps
                               : words         ? f.start + (whole + (left != 0)) * f.full * steps
                                               : whole * (f.start + f.full * steps) + (left ? f.start + part * steps : 0.)) +
                              (s > 1 ? 3.0 + 0.35 * s + 1.44e-6 * s * M * N : 0.);
            if (p.form == kAny || us < least) {
                least = us;
                p.form = f.form;
                p.slices = s;
            }
        }
    }
    return p;
}
int64_t planes_of(const Plan& p, int64_t M, int64_t N) { return p.slices > 1 ? 4 * p.slices * M * N : 0; }

template <int OUT_DT> int launch_join(const Fp8Gemm& p, hipStream_t st) {
    const int64_t blocks = ((int64_t)p.M * p.N + 1023) / 1024, most = 8 * (int64_t)device_cu_count();
    fp8_gemm_join_kernel<OUT_DT><<<(int)(blocks < most ? blocks : most), 256, 0, st>>>(p);
    KCHECK();
    return 0;
}
template <int BM, int OUT_DT, bool WIDE> constexpr auto mid_kernel() {
    if constexpr (WIDE) return fp8_gemm_wide_kernel<BM, OUT_DT>;
    else return fp8_gemm_mid_kernel<BM, OUT_DT>;
}
template <int BM, int OUT_DT, bool WIDE = OUT_DT == DT_F32> int launch_mid(Fp8Gemm p, hipStream_t st) {
    const auto kern = mid_kernel<BM, OUT_DT, WIDE>();
    constexpr int LDS = WIDE ? Wide<BM>::LDS : Mid<BM>::LDS;
    p.tiles_m = (p.M + BM - 1) / BM;
    p.tiles_n = (p.N + 127) / 128;
    const int64_t grid = (int64_t)p.tiles_m * p.tiles_n * p.slices;
    if (grid > kMostGroups) return -1;
    static PerDeviceOnce once;
    if (const int e = allow_dynamic_lds((const void*)kern, LDS, once)) return e;
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(512), LDS, st, p);
    KCHECK();
    return p.slices > 1 ? launch_join<OUT_DT>(p, st) : 0;
}
template <int MT, int CT, int OUT_DT> int launch_few(Fp8Gemm p, hipStream_t st) {
    p.tiles_n = (p.N + 16 * CT - 1) / (16 * CT);
    const int64_t grid = (int64_t)p.tiles_n * p.slices;
    if (grid > kMostGroups) return -1;
    fp8_gemm_few_kernel<MT, CT, OUT_DT><<<(int)grid, 512, 0, st>>>(p);
    KCHECK();
    return p.slices > 1 ? launch_join<OUT_DT>(p, st) : 0;
}

template <int OUT_DT> int launch(Fp8Gemm p, const Plan& plan, hipStream_t st) {
    p.slices = plan.slices;
    if (plan.form == kFew) {
        if (p.M <= 16) return plan.ct == 2 ? launch_few<1, 2, OUT_DT>(p, st) : launch_few<1, 1, OUT_DT>(p, st);
        return plan.ct == 2 ? launch_few<2, 2, OUT_DT>(p, st) : launch_few<2, 1, OUT_DT>(p, st);
    }
    if (plan.form == kMid64) return launch_mid<64, OUT_DT>(p, st);
    if (plan.form == kMid128) return launch_mid<128, OUT_DT>(p, st);
    if constexpr (OUT_DT != DT_F32) {
        if (plan.form == kBig) return launch_big<OUT_DT>(p, st);
        if (plan.form == kWide) return launch_mid<128, OUT_DT, true>(p, st);
    }
    p.tiles_m = (p.M + 127) / 128;
    p.tiles_n = (p.N + 127) / 128;
    if ((int64_t)p.tiles_m * p.tiles_n > 0xffffffffll / 256) return -1;
    fp8_gemm_kernel<OUT_DT><<<p.tiles_m * p.tiles_n, 256, 0, st>>>(p);
    KCHECK();
    return 0;
}

}  // namespace

GPU_API int64_t gpu_fp8_gemm_workspace(int64_t M, int64_t N, int64_t K, int out_dt) {
    if (M <= 0 || N <= 0 || K <= 0 || M > 0x7fffff00 || N > 0x7fffff00 || K > 0x7fffff00) return 0;
    return planes_of(plan_of(M, N, K, out_dt), M, N);
}

GPU_API int gpu_fp8_gemm(const void* A, const void* W, const float* xs, int64_t xs_stride, const float* ws, const void* bias, void* D,
                         void* work, int64_t M, int64_t N, int64_t K, int out_dt, void* stream) {
    if (out_dt != DT_BF16 && out_dt != DT_F16 && out_dt != DT_F32) return -4;
    if (M < 0 || N < 0 || K <= 0 || K % 16 != 0 || M > 0x7fffff00 || N > 0x7fffff00 || K > 0x7fffff00 || xs_stride < M) return -1;
    if (M == 0 || N == 0) return 0;
    const int size = out_dt == DT_F32 ? 4 : 2;
    if (!A || !W || !xs || !ws || !D || (uintptr_t)A % 16 != 0 || (uintptr_t)W % 16 != 0 || (uintptr_t)xs % 4 != 0 || (uintptr_t)ws % 4 != 0 || (uintptr_t)D % size != 0 ||
        (uintptr_t)bias % size != 0) return -1;
    const Plan plan = plan_of(M, N, K, out_dt);
    if (plan.slices > 1 && (!work || (uintptr_t)work % 16 != 0)) return -1;
    Fp8Gemm p{};
    p.A = (const uint8_t*)A; p.W = (const uint8_t*)W; p.xs = xs; p.ws = ws; p.bias = bias; p.D = D; p.xs_rs = xs_stride; p.planes = (float*)work;
    p.M = (int)M; p.N = (int)N; p.K = (int)K; p.groups = (int)((K + kGroup - 1) / kGroup);
    p.rows_ok = (uintptr_t)D % 16 == 0 && N * size % 16 == 0;
    const hipStream_t st = (hipStream_t)stream;
    return out_dt == DT_BF16 ? launch<DT_BF16>(p, plan, st) : out_dt == DT_F16 ? launch<DT_F16>(p, plan, st) : launch<DT_F32>(p, plan, st);
}

GPU_API int gpu_internal_fp8_gemm_plan(int64_t M, int64_t N, int64_t K, int out_dt, int32_t* out) {
    if (M <= 0 || N <= 0 || K <= 0 || !out) return -1;
    const Plan p = plan_of(M, N, K, out_dt);
    out[0] = p.form;
    out[1] = p.slices;
    return 0;
}
GPU_API int gpu_internal_fp8_gemm_force(int form_and_slices) {
    g_force.store(form_and_slices, std::memory_order_relaxed);
    return 0;
}
