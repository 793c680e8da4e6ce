// Rows -> e4m3 codes with a scale for each group of 128 columns, the operands of fp8_gemm.hip: plain rows, rows behind a residual's addition
// and an RMS norm, and the gate of an MLP.
//
//   s = T(x + resid)          where there is a residual; stored
//   n = s                     PRO_PLAIN
//   n = s r w,  r = 1 / sqrt(mean(s^2) + eps)      PRO_RMS, over the row
//   n = x / (1 + e^-x) up     PRO_SWIGLU
//   A = max(largest |n| of the group, 2^-100),  scale = A / 448,  code = e4m3(n (448 / A))
//
// All of n in 32 bits, rounded once, to the code.  448 is the largest e4m3 value, and n (448 / A) exceeds it by two roundings at most, which
// the conversion takes back.  A value that is not finite makes its group's A, and so what the codes stand for, NaN or infinite: magnitudes are
// compared as whole numbers, where NaN is the largest.
#include "common.hpp"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct Fp8Rows {
    const void *x, *resid;
    void* sum;
    int64_t x_rs, resid_rs, sum_rs, up_offset;
    const float* norm_w;
    float eps;
    uint8_t* q;
    float* scales;
    int64_t scales_rs;
    int M, K, wpr, wide;      // waves of a row; pieces start on whole 16 bytes: x (bit 0), resid (1), sum (2), the half at up_offset (3), norm_w (4)
};

constexpr int kPiece = 8;           // columns of a lane at a time: 16 lanes to a group of 128
constexpr float kLeastA = 0x1p-100f, kTop = 448.f;

// PAST: rows that are read once and do not fit the last-level cache leave what is in it alone.
template <bool PAST, class V> __device__ __forceinline__ V fetch(const V* p) { return PAST ? __builtin_nontemporal_load(p) : *p; }
template <int DT, bool PAST> __device__ __forceinline__ void load_piece(const void* base, int64_t at, bool wide, float (&v)[kPiece]) {
    if constexpr (DT == DT_F32) {
        const float* const p = (const float*)base + at;
        if (wide) {
            const f32x4 a = fetch<PAST>(reinterpret_cast<const f32x4*>(p)), b = fetch<PAST>(reinterpret_cast<const f32x4*>(p + 4));
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
        } else {
#pragma unroll
            for (int i = 0; i < kPiece; ++i) v[i] = p[i];
        }
    } else {
        const uint16_t* const p = (const uint16_t*)base + at;
        u32x4 w;
        if (wide) w = fetch<PAST>(reinterpret_cast<const u32x4*>(p));
        else
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = (uint32_t)p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (DT == DT_BF16) v[2 * i] = u2f(w[i] << 16), v[2 * i + 1] = u2f(w[i] & 0xffff0000u);
            else unpack_f16x2(w[i], v[2 * i], v[2 * i + 1]);
        }
    }
}
// v rounded to T, in memory and in v.
template <int DT> __device__ __forceinline__ void round_store(void* base, int64_t at, bool wide, float (&v)[kPiece]) {
    if constexpr (DT == DT_F32) {
        float* const p = (float*)base + at;
        if (wide) {
            *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
            *reinterpret_cast<f32x4*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
        } else {
#pragma unroll
            for (int i = 0; i < kPiece; ++i) p[i] = v[i];
        }
    } else {
        uint16_t* const p = (uint16_t*)base + at;
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = DT == DT_BF16 ? pack_bf16x2(v[2 * i], v[2 * i + 1]) : pack_f16x2(v[2 * i], v[2 * i + 1]);
            if (DT == DT_BF16) v[2 * i] = u2f(w[i] << 16), v[2 * i + 1] = u2f(w[i] & 0xffff0000u);
            else unpack_f16x2(w[i], v[2 * i], v[2 * i + 1]);
        }
        if (wide) *reinterpret_cast<u32x4*>(p) = w;
        else
#pragma unroll
            for (int i = 0; i < kPiece; ++i) p[i] = (uint16_t)(w[i >> 1] >> 16 * (i & 1));
    }
}

__device__ __forceinline__ float wave_sum_f32(float v) {
    const auto mv = [](float x, auto ctrl) { return __builtin_bit_cast(float, dpp_int<decltype(ctrl)::value>(__builtin_bit_cast(int, x))); };
    v += mv(v, std::integral_constant<int, 0xB1>{});
    v += mv(v, std::integral_constant<int, 0x4E>{});
    v += mv(v, std::integral_constant<int, 0x141>{});
    v += mv(v, std::integral_constant<int, 0x140>{});
    auto s = __builtin_amdgcn_permlane16_swap(f2u(v), f2u(v), false, false);
    v = u2f(s[0]) + u2f(s[1]);
    s = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
    return u2f(s[0]) + u2f(s[1]);
}
// The largest of a row of 16 lanes, as whole numbers.
__device__ __forceinline__ uint32_t row_max_u32(uint32_t v) {
    const auto mv = [](uint32_t x, auto ctrl) { return (uint32_t)dpp_int<decltype(ctrl)::value>((int)x); };
    v = max(v, mv(v, std::integral_constant<int, 0xB1>{}));
    v = max(v, mv(v, std::integral_constant<int, 0x4E>{}));
    v = max(v, mv(v, std::integral_constant<int, 0x141>{}));
    return max(v, mv(v, std::integral_constant<int, 0x140>{}));
}
// x / (1 + e^-x) by the hardware's exp2 and reciprocal: off by three units of fp32 and |x| / 3, where half a step of a code is 2^20 of them.  (The rounding of
// the exponent put back and a Newton step on the reciprocal make that one unit, and the kernel bound by its vector instructions: 4099 x
// 12288 from f16 48.7 -> 56.4 us.)
__device__ __forceinline__ float silu(float x) {
    return x * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * -1.44269504088896340736f));
}

// A row is a.wpr waves of C pieces a lane, piece i of lane l at columns 8 (64 (wave + wpr i) + l) ..; a workgroup has rows side by side.
template <int DT, int PRO, int C, bool PAST>
__global__ __launch_bounds__(512) void fp8_rows_kernel(const Fp8Rows a) {
    __shared__ float part[8];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int rows = waves / a.wpr, mine = wave / a.wpr, part_of_row = wave - mine * a.wpr;
    // neighbouring rows on one XCD: their scales are neighbours in memory
    const int n = gridDim.x, base = n >> 3, rem = n & 7, xcd = blockIdx.x & 7;
    const int row = (xcd * base + (xcd < rem ? xcd : rem) + (blockIdx.x >> 3)) * rows + mine;
    const bool there = row < a.M;
    float v[C][kPiece], up[PRO == PRO_SWIGLU ? C : 1][kPiece], w[PRO == PRO_RMS ? C : 1][kPiece];
    if (there) {
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int col = kPiece * (64 * (part_of_row + a.wpr * i) + lane);
#pragma unroll
            for (int j = 0; j < kPiece; ++j) v[i][j] = 0.f;
            if (col >= a.K) continue;
            load_piece<DT, PAST>(a.x, row * a.x_rs + col, a.wide & 1, v[i]);
            if (PRO == PRO_SWIGLU) load_piece<DT, PAST>(a.x, row * a.x_rs + a.up_offset + col, a.wide & 8, up[i]);
            if (PRO == PRO_RMS) load_piece<DT_F32, false>(a.norm_w, col, a.wide & 16, w[i]);
        }
        if (PRO != PRO_SWIGLU && a.resid) {
#pragma unroll
            for (int i = 0; i < C; ++i) {
                const int col = kPiece * (64 * (part_of_row + a.wpr * i) + lane);
                if (col >= a.K) continue;
                float r[kPiece];
                load_piece<DT, PAST>(a.resid, row * a.resid_rs + col, a.wide & 2, r);
#pragma unroll
                for (int j = 0; j < kPiece; ++j) v[i][j] += r[j];
                round_store<DT>(a.sum, row * a.sum_rs + col, a.wide & 4, v[i]);
            }
        }
    }
    if constexpr (PRO == PRO_RMS) {
        float ss = 0.f;
        if (there)
#pragma unroll
            for (int i = 0; i < C; ++i)
#pragma unroll
                for (int j = 0; j < kPiece; ++j) ss = fmaf(v[i][j], v[i][j], ss);
        ss = wave_sum_f32(ss);
        if (a.wpr > 1) {
            if (lane == 0) part[wave] = ss;
            __syncthreads();
            ss = 0.f;
            for (int i = 0; i < a.wpr; ++i) ss += part[mine * a.wpr + i];
        }
        const float r = 1.f / sqrtf(ss / (float)a.K + a.eps);
        if (there)
#pragma unroll
            for (int i = 0; i < C; ++i)
#pragma unroll
                for (int j = 0; j < kPiece; ++j) v[i][j] = v[i][j] * r * w[i][j];
    }
    if (!there) return;
#pragma unroll
    for (int i = 0; i < C; ++i) {
        const int col = kPiece * (64 * (part_of_row + a.wpr * i) + lane);
        const bool some = col < a.K;
        uint32_t top = 0;
        if (some)
#pragma unroll
            for (int j = 0; j < kPiece; ++j) {
                if (PRO == PRO_SWIGLU) v[i][j] = silu(v[i][j]) * up[i][j];
                top = max(top, f2u(v[i][j]) & 0x7fffffffu);
            }
        const float A = u2f(max(row_max_u32(top), f2u(kLeastA)));
        if (!some) continue;
        const float r = kTop / A;
        int c[2] = {0, 0};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            c[h] = __builtin_amdgcn_cvt_pk_fp8_f32(v[i][4 * h] * r, v[i][4 * h + 1] * r, c[h], false);
            c[h] = __builtin_amdgcn_cvt_pk_fp8_f32(v[i][4 * h + 2] * r, v[i][4 * h + 3] * r, c[h], true);
        }
        uint8_t* const to = a.q + (int64_t)row * a.K + col;
        *reinterpret_cast<u32x2*>(to) = u32x2{(uint32_t)c[0], (uint32_t)c[1]};
        if ((lane & 15) == 0) a.scales[(col >> 7) * a.scales_rs + row] = A / kTop;
    }
}

// A row's waves have a piece each up to 4096 columns, more of them beyond (RMS at 8192 x 4096, bf16, with a residual, 235 MB: 44.7 us, 5.25 TB/s, as
// one large copy; 46.9 with two pieces, 49.0 with four).  Calls of 64 MB or more load past the caches: 8192 x 4096 44.7 us, 49.7 without, 16384 x
// 1024 23.7 and 25.2; 1024 x 5120, which stay in the last-level cache, 11.5 and 11.0.
template <int DT, int PRO, bool PAST> int launch(Fp8Rows a, hipStream_t st) {
    const int pieces = (a.K + 64 * kPiece - 1) / (64 * kPiece);      // of 512 columns
    int wpr = 1;
    while (wpr < 8 && pieces > wpr) wpr *= 2;
    a.wpr = wpr;
    const int waves = wpr < 4 ? 4 : wpr, rows = waves / wpr, c = (pieces + wpr - 1) / wpr;
    if (((int64_t)a.M + rows - 1) / rows > 0xffffffffll / (64 * waves)) return -1;      // a launch has fewer than 2^32 threads
    const int grid = (int)(((int64_t)a.M + rows - 1) / rows);
    if (c <= 1) fp8_rows_kernel<DT, PRO, 1, PAST><<<grid, 64 * waves, 0, st>>>(a);
    else if (c <= 2) fp8_rows_kernel<DT, PRO, 2, PAST><<<grid, 64 * waves, 0, st>>>(a);
    else if (c <= 4) fp8_rows_kernel<DT, PRO, 4, PAST><<<grid, 64 * waves, 0, st>>>(a);
    else fp8_rows_kernel<DT, PRO, 8, PAST><<<grid, 64 * waves, 0, st>>>(a);
    KCHECK();
    return 0;
}
template <int DT, int PRO> int launch(const Fp8Rows& a, hipStream_t st) {
    const int64_t each = dt_size<DT>::value * (PRO == PRO_SWIGLU ? 2 : a.resid ? 3 : 1) + 1;
    return each * a.M * a.K >= (int64_t)64 << 20 ? launch<DT, PRO, true>(a, st) : launch<DT, PRO, false>(a, st);
}
template <int DT> int launch_pro(int prologue, const Fp8Rows& a, hipStream_t st) {
    switch (prologue) {
        case PRO_PLAIN: return launch<DT, PRO_PLAIN>(a, st);
        case PRO_RMS: return launch<DT, PRO_RMS>(a, st);
        default: return launch<DT, PRO_SWIGLU>(a, st);
    }
}

}  // namespace

GPU_API int gpu_fp8_quant_rows(int dtype, int prologue, const void* x, int64_t x_stride, const void* resid, int64_t resid_stride, void* sum,
                               int64_t sum_stride, int64_t up_offset, const float* norm_w, float eps, void* q, float* scales,
                               int64_t scales_stride, int M, int K, void* stream) {
    if (dtype != DT_BF16 && dtype != DT_F16 && dtype != DT_F32) return -4;
    if (prologue != PRO_PLAIN && prologue != PRO_RMS && prologue != PRO_SWIGLU) return -3;
    if (M < 0 || K <= 0 || K % 16 != 0 || scales_stride < M) return -1;
    if (K > 32768) return -2;
    if ((resid != nullptr) != (sum != nullptr) || (resid && prologue == PRO_SWIGLU) || (prologue == PRO_RMS && (!norm_w || !(eps >= 0.f && eps < INFINITY)))) return -1;
    if (M == 0) return 0;
    const int size = dtype == DT_F32 ? 4 : 2;
    if (!x || !q || !scales || (uintptr_t)q % 8 != 0 || (uintptr_t)scales % 4 != 0 || (uintptr_t)x % size != 0 || (uintptr_t)resid % size != 0 || (uintptr_t)sum % size != 0 ||
        (uintptr_t)norm_w % 4 != 0) return -1;
    const auto wide = [&](const void* p, int64_t at, int64_t rs) { return ((uintptr_t)p + (uintptr_t)(at * size)) % 16 == 0 && rs * size % 16 == 0; };
    Fp8Rows a{};
    a.x = x; a.resid = resid; a.sum = sum;
    a.x_rs = x_stride; a.resid_rs = resid_stride; a.sum_rs = sum_stride; a.up_offset = up_offset;
    a.norm_w = norm_w; a.eps = eps; a.q = (uint8_t*)q; a.scales = scales; a.scales_rs = scales_stride; a.M = M; a.K = K;
    a.wide = (wide(x, 0, x_stride) ? 1 : 0) | (wide(resid, 0, resid_stride) ? 2 : 0) | (wide(sum, 0, sum_stride) ? 4 : 0) | (wide(x, up_offset, x_stride) ? 8 : 0) |
             ((uintptr_t)norm_w % 16 == 0 ? 16 : 0);
    const hipStream_t st = (hipStream_t)stream;
    return dtype == DT_BF16 ? launch_pro<DT_BF16>(prologue, a, st) : dtype == DT_F16 ? launch_pro<DT_F16>(prologue, a, st) : launch_pro<DT_F32>(prologue, a, st);
}
