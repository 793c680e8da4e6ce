//! Generated by rust/gen_sys.py from include/gpu_api.h and include/gpu_blas_api.h.  Do not edit: change the
//! header and run the generator.  Argument meaning, alignment rules and return codes are documented at the
//! prototypes in the headers.
#![allow(clippy::too_many_arguments)]

use std::ffi::c_void;
use std::os::raw::c_char;

/// a device (or, where the header says so, host) address that the callee only reads
pub type P = *const c_void;
/// an address the callee writes, and the `hipStream_t` every call takes last
pub type PM = *mut c_void;

// libgpu_kernels: linked by build.rs
extern "C" {
    pub fn gpu_quant_rows(dtype: i32, prologue: i32, x: P, x_stride: i64, g: P, g_stride: i64, up_offset: i64,
        norm_w: P, eps: f32, mod_scale: P, mod_shift: P, q: PM, scales: PM, m: i32, k: i32, rotate: i32, stream: PM) -> i32;
    pub fn gpu_quant_rows_b(dtype: i32, prologue: i32, x: P, x_stride: i64, norm_w: P, norm_b: P, eps: f32,
        mod_scale: P, mod_shift: P, q: PM, scales: PM, m: i32, k: i32, rotate: i32, stream: PM) -> i32;
    pub fn gpu_rotate_rows_f32(prologue: i32, x: P, x_stride: i64, up_offset: i64, norm_w: P, eps: f32, out: PM,
        m: i32, k: i32, stream: PM) -> i32;
    pub fn gpu_prologue_rows(dtype: i32, prologue: i32, x: P, x_stride: i64, g: P, g_stride: i64, up_offset: i64,
        norm_w: P, eps: f32, mod_scale: P, mod_shift: P, out: PM, out_stride: i64, m: i32, k: i32, stream: PM) -> i32;
    pub fn gpu_prologue_rows_b(dtype: i32, prologue: i32, x: P, x_stride: i64, norm_w: P, norm_b: P, eps: f32,
        mod_scale: P, mod_shift: P, out: PM, out_stride: i64, m: i32, k: i32, stream: PM) -> i32;
    pub fn gpu_sd_quant_rows(x: P, x_stride: i64, q: PM, scales: PM, m: i32, k: i32, rotate: i32, stream: PM) -> i32;
    pub fn gpu_sd_ln_quant_rows(x: P, x_stride: i64, w: P, b: P, eps: f32, q: PM, scales: PM, m: i32, k: i32,
        rotate: i32, stream: PM) -> i32;
    pub fn gpu_sd_geglu_quant_rows(in_: P, q: PM, scales: PM, m: i32, i: i32, rotate: i32, stream: PM) -> i32;
    pub fn gpu_sd_unpad_quant_rows(src: P, q: PM, scales: PM, m: i32, h: i32, d: i32, dp: i32, rotate: i32,
        stream: PM) -> i32;
    pub fn gpu_sd_group_norm_quant_rows(x: P, w: P, b: P, sums: PM, n: i32, p: i64, c: i32, g: i32, eps: f32,
        q: PM, scales: PM, rotate: i32, stream: PM) -> i32;
    pub fn gpu_dequant_i8(q: P, s: P, out: PM, n: i64, k: i64, stream: PM) -> i32;
    pub fn gpu_embed_dequant(q: P, s: P, out: PM, m: i32, k: i32, rotate: i32, stream: PM) -> i32;
    pub fn gpu_convrot_dequant(dtype: i32, q: P, s: P, out: PM, n: i64, k: i32, stream: PM) -> i32;
    pub fn gpu_convrot_requant(dtype: i32, x: P, q: PM, s: PM, n: i64, k: i32, seed: u64, stream: PM) -> i32;
    pub fn gpu_w6_requant(weight: P, packed: PM, s_rel: PM, s_channel: PM, n: i64, k: i32, seed: u64, stream: PM) -> i32;
    pub fn gpu_internal_w6_requant_rows(n: i64, k: i32) -> i32;
    pub fn gpu_int8_attn_workspace_d(b: i32, h: i32, hk: i32, lq: i32, lk: i32, head_dim: i32) -> i64;
    pub fn gpu_int8_attn_workspace(b: i32, h: i32, hk: i32, lq: i32, lk: i32) -> i64;
    pub fn gpu_int8_attn_d(q: P, k: P, v: P, o: PM, ws: PM, b: i32, lq: i32, lk: i32, h: i32, hk: i32,
        head_dim: i32, q_bs: i64, q_rs: i64, q_hs: i64, k_bs: i64, k_rs: i64, k_hs: i64, v_bs: i64, v_rs: i64,
        v_hs: i64, o_bs: i64, o_rs: i64, o_hs: i64, scale: f32, stream: PM) -> i32;
    pub fn gpu_int8_attn_f16(q: P, k: P, v: P, o: PM, ws: PM, b: i32, lq: i32, lk: i32, h: i32, hk: i32,
        head_dim: i32, q_bs: i64, q_rs: i64, q_hs: i64, k_bs: i64, k_rs: i64, k_hs: i64, v_bs: i64, v_rs: i64,
        v_hs: i64, o_bs: i64, o_rs: i64, o_hs: i64, scale: f32, stream: PM) -> i32;
    pub fn gpu_int8_attn(q: P, k: P, v: P, o: PM, ws: PM, b: i32, lq: i32, lk: i32, h: i32, hk: i32, q_bs: i64,
        q_rs: i64, q_hs: i64, k_bs: i64, k_rs: i64, k_hs: i64, v_bs: i64, v_rs: i64, v_hs: i64, o_bs: i64,
        o_rs: i64, o_hs: i64, scale: f32, stream: PM) -> i32;
    pub fn gpu_int8_attn_sink(q: P, k: P, v: P, o: PM, ws: PM, b: i32, lq: i32, lk: i32, h: i32, hk: i32,
        q_bs: i64, q_rs: i64, q_hs: i64, k_bs: i64, k_rs: i64, k_hs: i64, v_bs: i64, v_rs: i64, v_hs: i64,
        o_bs: i64, o_rs: i64, o_hs: i64, scale: f32, sink: f32, qw: P, eps: f32, stream: PM) -> i32;
    pub fn gpu_int8_attn_norm_rope(q: P, k: P, v: P, o: PM, ws: PM, b: i32, lq: i32, lk: i32, h: i32, hk: i32,
        q_bs: i64, q_rs: i64, q_hs: i64, k_bs: i64, k_rs: i64, k_hs: i64, v_bs: i64, v_rs: i64, v_hs: i64,
        o_bs: i64, o_rs: i64, o_hs: i64, scale: f32, qw: P, kw: P, eps: f32, rope: P, rope_mode: i32, stream: PM) -> i32;
    pub fn gpu_int8_attn_key_bias_workspace(b: i32, h: i32, hk: i32, lq: i32, lk: i32) -> i64;
    pub fn gpu_int8_attn_key_bias(q: P, k: P, v: P, o: PM, ws: PM, b: i32, lq: i32, lk: i32, h: i32, hk: i32,
        q_bs: i64, q_rs: i64, q_hs: i64, k_bs: i64, k_rs: i64, k_hs: i64, v_bs: i64, v_rs: i64, v_hs: i64,
        o_bs: i64, o_rs: i64, o_hs: i64, scale: f32, bias: P, stream: PM) -> i32;
    pub fn gpu_internal_act_probe(which: i32, in_: P, out: PM, n: i32, stream: PM) -> i32;
    pub fn gpu_internal_geglu_form(m: i32, k: i32) -> i32;
    pub fn gpu_internal_cvt_pk_u8_probe(x: P, y: PM, n: i32, stream: PM) -> i32;
    pub fn gpu_internal_w6a8_group_gemm_ablate(ablate: i32, a: P, wp: P, xs: P, sw: P, d: PM, m: i64, n: i64,
        k: i64, stream: PM) -> i32;
    pub fn gpu_internal_w6a8_group_gemm_mode(mode: i32) -> i32;
    pub fn gpu_internal_attn_sumsq_probe(x: P, out: PM, rows: i32, split: i32, stream: PM) -> i32;
    pub fn gpu_internal_attn_layout(b: i32, h: i32, hk: i32, lq: i32, lk: i32, out: PM) -> i32;
    pub fn gpu_internal_attn_layout_d(b: i32, h: i32, hk: i32, lq: i32, lk: i32, head_dim: i32, out: PM) -> i32;
    pub fn gpu_int8_gemm(a: P, w: P, xs: P, ws: P, bias: P, d: PM, m: i64, n: i64, k: i64, out_dt: i32, stream: PM) -> i32;
    pub fn gpu_int8_gemm_residual(a: P, w: P, xs: P, ws: P, bias: P, rscale: P, resid: P, d: PM, m: i64, n: i64,
        k: i64, out_dt: i32, stream: PM) -> i32;
    pub fn gpu_w6_decode(q: P, s_rel: P, out: PM, n: i64, k: i32, g: i32, stream: PM) -> i32;
    pub fn gpu_act_tables_init() -> i32;
    pub fn gpu_int8_gemm_acc(a: P, w: P, acc: PM, m: i64, n: i64, k: i64, stream: PM) -> i32;
    pub fn gpu_int8_gemm_static(a: P, w: P, xs: P, ws: P, bias: P, d: PM, m: i64, n: i64, k: i64, out_dt: i32,
        stream: PM) -> i32;
    pub fn gpu_int8_gemm_static_limit() -> i64;
    pub fn gpu_linear_w8a8(dtype: i32, x: P, x_stride: i64, w: P, ws: P, bias: P, d: PM, scratch: PM, m: i64,
        n: i64, k: i64, rotate: i32, out_dt: i32, stream: PM) -> i32;
    pub fn gpu_w6a8_gemm(a: P, wq: P, s_rel: P, g: i32, xs: P, s_channel: P, bias: P, d: PM, m: i64, n: i64,
        k: i64, out_dt: i32, stream: PM) -> i32;
    pub fn gpu_w6a8_gemm_ws(a: P, wq: P, s_rel: P, g: i32, xs: P, s_channel: P, bias: P, d: PM, scratch: PM,
        m: i64, n: i64, k: i64, out_dt: i32, stream: PM) -> i32;
    pub fn gpu_w6a8_group_gemm(a: P, wp: P, xs: P, sw: P, bias: P, d: PM, partials: PM, m: i64, n: i64, k: i64,
        out_dt: i32, stream: PM) -> i32;
    pub fn gpu_w6a8_group_gemm_ws(a: P, wp: P, xs: P, sw: P, bias: P, d: PM, partials: PM, scratch: PM, m: i64,
        n: i64, k: i64, out_dt: i32, stream: PM) -> i32;
    pub fn gpu_w6a8_group_gemm_scratch(wp: P, m: i64, n: i64, k: i64) -> i64;
    pub fn gpu_cross_attn_workspace(b: i32, lq: i32, lk: i32, h: i32, hk: i32, head_dim: i32) -> i64;
    pub fn gpu_cross_attn(dtype: i32, q: P, k: P, v: P, o: PM, ws: PM, b: i32, lq: i32, lk: i32, h: i32, hk: i32,
        head_dim: i32, q_bs: i64, q_rs: i64, q_hs: i64, k_bs: i64, k_rs: i64, k_hs: i64, v_bs: i64, v_rs: i64,
        v_hs: i64, o_bs: i64, o_rs: i64, o_hs: i64, scale: f32, k_lens: P, mask: P, mask_kind: i32, mask_bs: i64,
        stream: PM) -> i32;
    pub fn gpu_kv8_store(dtype: i32, k: P, k_rs: i64, k_hs: i64, v: P, v_rs: i64, v_hs: i64, ck: PM, cv: PM,
        k_scale: PM, v_scale: PM, n_pages: i32, page: i32, starts: P, lens: P, table: P, table_cols: i32, n: i32,
        rows: i32, most: i32, hk: i32, head_dim: i32, stream: PM) -> i32;
    pub fn gpu_kv8_read(dtype: i32, k: PM, k_rs: i64, k_hs: i64, v: PM, v_rs: i64, v_hs: i64, ck: P, cv: P,
        k_scale: P, v_scale: P, n_pages: i32, page: i32, starts: P, lens: P, table: P, table_cols: i32, n: i32,
        rows: i32, most: i32, hk: i32, head_dim: i32, stream: PM) -> i32;
    pub fn gpu_kv8_attn_workspace(n: i32, most: i32, h: i32, hk: i32, head_dim: i32, page: i32, table_cols: i32) -> i64;
    pub fn gpu_kv8_attn(dtype: i32, q: P, q_rs: i64, q_hs: i64, o: PM, o_rs: i64, o_hs: i64, ws: PM, ck: P, cv: P,
        k_scale: P, v_scale: P, n_pages: i32, page: i32, starts: P, lens: P, table: P, table_cols: i32, n: i32,
        rows: i32, most: i32, h: i32, hk: i32, head_dim: i32, scale: f32, causal: i32, stream: PM) -> i32;
    pub fn gpu_kv8_copy_pages(ck: PM, cv: PM, k_scale: PM, v_scale: PM, layers: i32, n_pages: i32, page: i32,
        hk: i32, head_dim: i32, src: P, dst: P, n: i32, stream: PM) -> i32;
    pub fn gpu_internal_states_plan(rows: i64, problems: i64, keys: i64, head_dim: i32, bytes: i32, out: PM) -> i32;
    pub fn gpu_int8_gemm_force_config(cfg: i32) -> i32;
    pub fn gpu_internal_int8_gemm_plan(m: i64, n: i64, k: i64, start: i32, aligned: i32, out: PM) -> i32;
    pub fn gpu_mfma_layout_probe(out: PM, stream: PM) -> i32;
    pub fn gpu_mfma_ceiling_probe(iters: i32, random_bits: i32, cycles: PM, sink: PM, stream: PM) -> i32;
    pub fn gpu_kernels_build_info() -> *const c_char;
}

// libgpu_blas: linked by build.rs
extern "C" {
    pub fn gpu_blas_init(workspace_bytes: usize) -> i32;
    pub fn gpu_gemm(a: P, lda: i64, b: P, ldb: i64, d: PM, ldd: i64, bias: P, m: i64, n: i64, k: i64, transb: i32,
        in_dt: i32, out_dt: i32, alpha: f32, beta: f32, stream: PM) -> i32;
}
