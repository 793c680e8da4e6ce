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

struct Fp8Gemm {
    const uint8_t *A, *W;
    const float *xs, *ws;
    const void* bias;
    void* D;
    int64_t xs_rs;
    int M, N, K, groups;
    int tiles_m, tiles_n;
    int rows_ok;      // rows of D start on 16 bytes
};

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

// Any sizes: tiles of 128 x 128, four waves of 64 x 64, a group at a time through registers into one of two LDS stages.
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
                v4f d = {0.f, 0.f, 0.f, 0.f};
                if constexpr (OUT_DT == DT_F32) {
#pragma unroll
                    for (int e = 0; e < 8; e += 2) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen(fw[e], fw[e + 1]), widen(fa[i][e], fa[i][e + 1]), d, 0, 0, 0);
                } else d = mfma(fw, fa[i], d);
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

template <int OUT_DT> int launch(Fp8Gemm p, hipStream_t st) {
    p.tiles_m = (p.M + 127) / 128;
    p.tiles_n = (p.N + 127) / 128;
    if ((int64_t)p.tiles_m * p.tiles_n > 0xffffffffll / 256) return -1;
    fp8_gemm_kernel<OUT_DT><<<p.tiles_m * p.tiles_n, 256, 0, st>>>(p);
    KCHECK();
    return 0;
}

}  // namespace

GPU_API int gpu_fp8_gemm(const void* A, const void* W, const float* xs, int64_t xs_stride, const float* ws, const void* bias, void* D,
                         int64_t M, int64_t N, int64_t K, int out_dt, void* stream) {
    if (out_dt != DT_BF16 && out_dt != DT_F16 && out_dt != DT_F32) return -4;
    if (M < 0 || N < 0 || K <= 0 || K % 16 != 0 || M > 0x7fffff00 || N > 0x7fffff00 || K > 0x7fffff00 || xs_stride < M) return -1;
    if (M == 0 || N == 0) return 0;
    const int size = out_dt == DT_F32 ? 4 : 2;
    if (!A || !W || !xs || !ws || !D || (uintptr_t)A % 16 != 0 || (uintptr_t)W % 16 != 0 || (uintptr_t)xs % 4 != 0 || (uintptr_t)ws % 4 != 0 || (uintptr_t)D % size != 0 ||
        (uintptr_t)bias % size != 0) return -1;
    Fp8Gemm p{};
    p.A = (const uint8_t*)A; p.W = (const uint8_t*)W; p.xs = xs; p.ws = ws; p.bias = bias; p.D = D; p.xs_rs = xs_stride;
    p.M = (int)M; p.N = (int)N; p.K = (int)K; p.groups = (int)((K + kGroup - 1) / kGroup);
    p.rows_ok = (uintptr_t)D % 16 == 0 && N * size % 16 == 0;
    const hipStream_t st = (hipStream_t)stream;
    return out_dt == DT_BF16 ? launch<DT_BF16>(p, st) : out_dt == DT_F16 ? launch<DT_F16>(p, st) : launch<DT_F32>(p, st);
}
