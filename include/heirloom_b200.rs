// Generated by include/make_rust_shim.py from include/heirloom_b200.h; do not edit by hand.
// Rust side of the C ABI of libheirloom_b200.so, for heirloom-kernels (the only crate of the reference that
// contains unsafe code).  Not compiled in this repository: the image it is built in has no Rust toolchain.
#![allow(non_camel_case_types, dead_code)]
use std::os::raw::{c_char, c_void};
use super::cuda::{AdamWParams, CausalAttentionDims, CudaError, CudaResult};

pub const HL_OK: i32 = 0;
pub const HL_ERR_INVALID: i32 = -1;
pub const HL_ERR_CUDA: i32 = -2;
pub const HL_ERR_DEVICE: i32 = -3;
pub const HL_ERR_NCCL: i32 = -4;
pub const HL_F32: i32 = 0;
pub const HL_BF16: i32 = 1;
pub const HL_F64: i32 = 2;
pub const HL_I64: i32 = 3;
pub const HL_U8: i32 = 4;
pub const HL_PROF_GEMM: i32 = 0;
pub const HL_PROF_ATTENTION_FWD: i32 = 1;
pub const HL_PROF_ATTENTION_BWD: i32 = 2;
pub const HL_PROF_LAYER_NORM: i32 = 3;
pub const HL_PROF_LOSS: i32 = 4;
pub const HL_PROF_OPTIMIZER: i32 = 5;
pub const HL_PROF_BIAS_GRAD: i32 = 6;
pub const HL_PROF_EMBEDDING: i32 = 7;
pub const HL_PROF_OTHER: i32 = 8;
pub const HL_PROF_CATEGORIES: i32 = 9;
pub const HL_ADD: i32 = 0;
pub const HL_SUB: i32 = 1;
pub const HL_MUL: i32 = 2;
pub const HL_DIV: i32 = 3;
pub const HL_SPLIT_HI_MID_LO: i32 = 0;
pub const HL_SPLIT_HI_HI_LO: i32 = 1;
pub const HL_SPLIT_HI_LO: i32 = 2;
pub const HL_SPLIT_STACK_ROWS: i32 = 4;
pub const HL_K_MAJOR: i32 = 0;
pub const HL_MN_MAJOR: i32 = 1;
pub const HL_EPI_NONE: i32 = 0;
pub const HL_EPI_BIAS: i32 = 1;
pub const HL_EPI_BIAS_GELU: i32 = 2;
pub const HL_EPI_BIAS_RESIDUAL: i32 = 3;
pub const HL_EPI_DGELU: i32 = 4;
pub const HL_PRECISION_F32: i32 = 0;
pub const HL_PRECISION_AMP_BF16: i32 = 1;
pub const HL_MEMORY_UPDATE_FULL: i32 = 0;
pub const HL_MEMORY_UPDATE_MEMORY_ONLY: i32 = 1;
pub const HL_MEMORY_UPDATE_SPARSE_ROWS: i32 = 2;
pub const HL_MEMORY_UPDATE_FROZEN: i32 = 3;
pub const HL_MEMORY_UPDATE_DENSE_PLUS_SPARSE_VALUES: i32 = 4;

pub enum HlCtx {}
pub enum HlBuffer {}
pub enum HlAdamwPlan {}
pub enum HlDecoder {}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct HlDeviceInfo {
    pub sm_major: i32,
    pub sm_minor: i32,
    pub sm_count: i32,
    pub total_bytes: usize,
    pub free_bytes: usize,
    pub supports_tcgen05: i32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct HlCounters {
    pub launches: u64,
    pub gemm_tcgen05_launches: u64,
    pub attention_launches: u64,
    pub h2d_bytes: u64,
    pub d2h_bytes: u64,
    pub allocations: u64,
    pub allocated_bytes: u64,
    pub nccl_calls: u64,
    pub nccl_bytes: u64,
    pub gemm_pair_launches: u64,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct HlProfile {
    pub ms: [f64; 9],
    pub work: [f64; 9],
    pub scopes: [u64; 9],
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct HlAdamwParams {
    pub lr: f32,
    pub beta1: f32,
    pub beta2: f32,
    pub eps: f32,
    pub weight_decay: f32,
    pub clip_scale: f32,
    pub bias_correction1: f32,
    pub bias_correction2: f32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct HlAdamwTensor {
    pub param: *mut f32,
    pub grad: *const f32,
    pub m: *mut f32,
    pub v: *mut f32,
    pub shadow_bf16: *mut c_void,
    pub n: u64,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct HlMatrixLayout {
    pub rows: i64,
    pub cols: i64,
    pub row_stride: i64,
    pub col_stride: i64,
    pub offset: i64,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct HlGemmDesc {
    pub m: i32,
    pub n: i32,
    pub k: i32,
    pub a_layout: i32,
    pub b_layout: i32,
    pub lda: i64,
    pub ldb: i64,
    pub ldc: i64,
    pub epilogue: i32,
    pub out_dtype: i32,
    pub split_k: i32,
    pub ld_aux_in: i64,
    pub ld_aux_out: i64,
    pub a_k_period: i32,
    pub b_k_period: i32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct HlPagedCache {
    pub k_pages: *mut c_void,
    pub v_pages: *mut c_void,
    pub dtype: i32,
    pub pages: i32,
    pub page_size: i32,
    pub kv_heads: i32,
    pub head_dim: i32,
    pub page_stride: i64,
    pub position_stride: i64,
    pub head_stride: i64,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct HlPagedBatch {
    pub page_table: *const i32,
    pub lengths: *const i32,
    pub first: *const i32,
    pub ld_table: i64,
    pub table_width: i32,
    pub sequences: i32,
    pub tokens: i32,
    pub max_new: i32,
    pub max_length: i32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct HlDecoderConfig {
    pub vocab: i32,
    pub d_model: i32,
    pub n_layers: i32,
    pub n_heads: i32,
    pub d_ff: i32,
    pub context: i32,
    pub batch: i32,
    pub precision: i32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct HlAdamwConfig {
    pub lr: f32,
    pub beta1: f32,
    pub beta2: f32,
    pub eps: f32,
    pub weight_decay: f32,
    pub clip_norm: f32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct HlMemoryConfig {
    pub n_memory_layers: i32,
    pub memory_layers: [i32; 16],
    pub slots: i32,
    pub key_dim: i32,
    pub value_dim: i32,
    pub top_k: i32,
    pub memory_heads: i32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct HlSamplingOptions {
    pub temperature: f64,
    pub top_p: f64,
    pub repetition_penalty: f64,
    pub frequency_penalty: f64,
    pub presence_penalty: f64,
    pub top_k: i64,
}

#[link(name = "heirloom_b200")]
extern "C" {
    pub fn hl_ctx_create(device_ordinal: i32, out: *mut *mut HlCtx) -> i32;
    pub fn hl_ctx_destroy(ctx: *mut HlCtx);
    pub fn hl_ctx_sync(ctx: *mut HlCtx) -> i32;
    pub fn hl_ctx_set_test_hooks(ctx: *mut HlCtx, wait_limit_ns: u64, gemm_skip_kblock: i32) -> i32;
    pub fn hl_ctx_stream(ctx: *mut HlCtx) -> *mut c_void;
    pub fn hl_last_error() -> *const c_char;
    pub fn hl_fnv1a64(data: *const c_void, bytes: usize, seed: u64) -> u64;
    pub fn hl_device_info(ctx: *mut HlCtx, out: *mut HlDeviceInfo) -> i32;
    pub fn hl_counters_get(ctx: *mut HlCtx, out: *mut HlCounters) -> i32;
    pub fn hl_counters_reset(ctx: *mut HlCtx) -> i32;
    pub fn hl_profile_enable(ctx: *mut HlCtx, on: i32) -> i32;
    pub fn hl_profile_read(ctx: *mut HlCtx, out: *mut HlProfile) -> i32;
    pub fn hl_buffer_alloc(ctx: *mut HlCtx, bytes: usize, out: *mut *mut HlBuffer) -> i32;
    pub fn hl_buffer_retain(buf: *mut HlBuffer) -> i32;
    pub fn hl_buffer_release(buf: *mut HlBuffer) -> i32;
    pub fn hl_buffer_ptr(buf: *mut HlBuffer) -> *mut c_void;
    pub fn hl_buffer_bytes(buf: *mut HlBuffer) -> usize;
    pub fn hl_memcpy_h2d(ctx: *mut HlCtx, dst_dev: *mut c_void, src_host: *const c_void, bytes: usize) -> i32;
    pub fn hl_memcpy_d2h(ctx: *mut HlCtx, dst_host: *mut c_void, src_dev: *const c_void, bytes: usize) -> i32;
    pub fn hl_memset_zero(ctx: *mut HlCtx, dst_dev: *mut c_void, bytes: usize) -> i32;
    pub fn hl_binary_f32(ctx: *mut HlCtx, op: i32, a: *const f32, b: *const f32, out: *mut f32, n: usize) -> i32;
    pub fn hl_scale_f32(ctx: *mut HlCtx, a: *const f32, s: f32, out: *mut f32, n: usize) -> i32;
    pub fn hl_fill_f32(ctx: *mut HlCtx, out: *mut f32, value: f32, n: usize) -> i32;
    pub fn hl_sgd_update_f32(ctx: *mut HlCtx, param: *mut f32, grad: *const f32, lr: f32, n: usize) -> i32;
    pub fn hl_arange_i64(ctx: *mut HlCtx, out: *mut i64, n: usize) -> i32;
    pub fn hl_concat_i64(ctx: *mut HlCtx, inputs: *const *const i64, lengths: *const usize, count: i32, out: *mut i64, out_capacity: usize) -> i32;
    pub fn hl_relu_f32(ctx: *mut HlCtx, x: *const f32, out: *mut f32, n: usize) -> i32;
    pub fn hl_relu_backward_f32(ctx: *mut HlCtx, x: *const f32, grad_out: *const f32, grad_in: *mut f32, n: usize) -> i32;
    pub fn hl_cast(ctx: *mut HlCtx, src: *const c_void, src_dtype: i32, dst: *mut c_void, dst_dtype: i32, n: usize) -> i32;
    pub fn hl_split_bf16_f32(ctx: *mut HlCtx, src: *const f32, dst: *mut c_void, rows: i64, cols: i32, mode: i32) -> i32;
    pub fn hl_gelu(ctx: *mut HlCtx, x: *const c_void, out: *mut c_void, dtype: i32, n: usize) -> i32;
    pub fn hl_gelu_backward(ctx: *mut HlCtx, x: *const c_void, grad_out: *const c_void, grad_in: *mut c_void, dtype: i32, n: usize) -> i32;
    pub fn hl_bias_add_f32(ctx: *mut HlCtx, x: *const f32, bias: *const f32, out: *mut f32, rows: i32, cols: i32) -> i32;
    pub fn hl_bias_grad(ctx: *mut HlCtx, grad_out: *const c_void, dtype: i32, grad_bias: *mut f32, rows: i32, cols: i32) -> i32;
    pub fn hl_sum_f32(ctx: *mut HlCtx, x: *const f32, n: usize, out_dev: *mut f32) -> i32;
    pub fn hl_mean_f32(ctx: *mut HlCtx, x: *const f32, n: usize, out_dev: *mut f32) -> i32;
    pub fn hl_sum_squares_f32(ctx: *mut HlCtx, x: *const f32, n: usize, out_dev: *mut f32) -> i32;
    pub fn hl_layer_norm_forward(ctx: *mut HlCtx, x: *const c_void, x_dtype: i32, gamma: *const f32, beta: *const f32, y: *mut c_void, y_dtype: i32, mean: *mut f32, rstd: *mut f32, rows: i32, features: i32, eps: f32) -> i32;
    pub fn hl_layer_norm_backward(ctx: *mut HlCtx, x: *const c_void, x_dtype: i32, gamma: *const f32, dy: *const f32, mean: *const f32, rstd: *const f32, residual_grad: *const f32, dx_f32: *mut f32, dx_bf16: *mut c_void, dgamma: *mut f32, dbeta: *mut f32, dx_colsum: *mut f32, rows: i32, features: i32) -> i32;
    pub fn hl_embedding_forward(ctx: *mut HlCtx, table: *const f32, table_rows: i32, idx: *const i64, pos_table: *const f32, period: i32, out: *mut c_void, out_dtype: i32, n: i32, dim: i32) -> i32;
    pub fn hl_embedding_backward(ctx: *mut HlCtx, grad_out: *const f32, idx: *const i64, grad_table: *mut f32, table_rows: i32, pos_grad: *mut f32, period: i32, n: i32, dim: i32) -> i32;
    pub fn hl_cross_entropy(ctx: *mut HlCtx, logits: *const f32, ld: i64, targets: *const i64, rows: i32, classes: i32, grad_scale: f32, loss_dev: *mut f32, row_loss: *mut f32, dlogits: *mut c_void, dlogits_dtype: i32, ld_dlogits: i64) -> i32;
    pub fn hl_adamw_f32(ctx: *mut HlCtx, param: *mut f32, grad: *const f32, m: *mut f32, v: *mut f32, n: usize, hp: *const HlAdamwParams) -> i32;
    pub fn hl_adamw_multi(ctx: *mut HlCtx, tensors_host: *const HlAdamwTensor, count: i32, hp: *const HlAdamwParams) -> i32;
    pub fn hl_adamw_plan_create(ctx: *mut HlCtx, tensors_host: *const HlAdamwTensor, count: i32, out: *mut *mut HlAdamwPlan) -> i32;
    pub fn hl_adamw_plan_step(ctx: *mut HlCtx, plan: *mut HlAdamwPlan, hp: *const HlAdamwParams) -> i32;
    pub fn hl_adamw_plan_destroy(plan: *mut HlAdamwPlan);
    pub fn hl_matmul_f32_strided(ctx: *mut HlCtx, a: *const f32, la: *const HlMatrixLayout, b: *const f32, lb: *const HlMatrixLayout, out: *mut f32, lo: *const HlMatrixLayout, accumulate: i32) -> i32;
    pub fn hl_causal_attention_f32_forward(ctx: *mut HlCtx, q: *const f32, k: *const f32, v: *const f32, out: *mut f32, probs: *mut f32, batch: i32, time: i32, channels: i32, n_heads: i32) -> i32;
    pub fn hl_causal_attention_f32_backward(ctx: *mut HlCtx, q: *const f32, k: *const f32, v: *const f32, probs: *const f32, grad_out: *const f32, dq: *mut f32, dk: *mut f32, dv: *mut f32, batch: i32, time: i32, channels: i32, n_heads: i32) -> i32;
    pub fn hl_gemm_bf16(ctx: *mut HlCtx, desc: *const HlGemmDesc, a: *const c_void, b: *const c_void, c: *mut c_void, bias: *const f32, aux_in: *const c_void, aux_out: *mut c_void) -> i32;
    pub fn hl_gemm_bf16_plan(ctx: *mut HlCtx, desc: *const HlGemmDesc, splits: *mut i32, dealt_tiles: *mut i32, scratch_bytes: *mut usize) -> i32;
    pub fn hl_gemm_bf16_static_scratch(ctx: *mut HlCtx, desc: *const HlGemmDesc, a: *const c_void, b: *const c_void, c: *mut c_void, bias: *const f32, aux_in: *const c_void, aux_out: *mut c_void) -> i32;
    pub fn hl_flash_attention_forward(ctx: *mut HlCtx, q: *const c_void, k: *const c_void, v: *const c_void, ld_qkv: i64, out: *mut c_void, ld_out: i64, lse: *mut f32, batch: i32, time: i32, n_heads: i32, head_dim: i32) -> i32;
    pub fn hl_flash_attention_backward(ctx: *mut HlCtx, q: *const c_void, k: *const c_void, v: *const c_void, ld_qkv: i64, out: *const c_void, ld_out: i64, dout: *const c_void, ld_dout: i64, lse: *const f32, dq: *mut c_void, dk: *mut c_void, dv: *mut c_void, ld_dqkv: i64, batch: i32, time: i32, n_heads: i32, head_dim: i32) -> i32;
    pub fn hl_paged_append(ctx: *mut HlCtx, cache: *const HlPagedCache, batch: *const HlPagedBatch, q: *const c_void, ld_q: i64, q_out: *mut c_void, ld_q_out: i64, heads: i32, k: *const c_void, ld_k: i64, v: *const c_void, ld_v: i64, frequencies: *const f32, rotary_dim: i32, interleaved: i32) -> i32;
    pub fn hl_paged_attention(ctx: *mut HlCtx, cache: *const HlPagedCache, batch: *const HlPagedBatch, q: *const c_void, ld_q: i64, out: *mut c_void, ld_out: i64, lse: *mut f32, heads: i32, scale: f32, workspace: *mut c_void, workspace_bytes: usize) -> i32;
    pub fn hl_paged_attention_workspace(ctx: *mut HlCtx, dtype: i32, heads: i32, kv_heads: i32, head_dim: i32, bytes: *mut usize) -> i32;
    pub fn hl_topk_rows_f32(ctx: *mut HlCtx, scores: *const f32, out: *mut i64, rows: i32, cols: i32, k: i32) -> i32;
    pub fn hl_product_key_side_scores_f32(ctx: *mut HlCtx, query: *const f32, ld_query: i64, left_keys: *const f32, right_keys: *const f32, left_scores: *mut f32, right_scores: *mut f32, tokens: i32, side: i32, key_dim: i32) -> i32;
    pub fn hl_product_key_topk_from_side_scores(ctx: *mut HlCtx, left_scores: *const f32, right_scores: *const f32, out: *mut i64, tokens: i32, side: i32, top_k: i32, beam: i32) -> i32;
    pub fn hl_product_key_lookup(ctx: *mut HlCtx, query: *const f32, left_keys: *const f32, right_keys: *const f32, pieces: *mut c_void, query_pieces: *mut c_void, left_approx: *mut f32, right_approx: *mut f32, out: *mut i64, tokens: i32, side: i32, key_dim: i32, top_k: i32, beam: i32) -> i32;
    pub fn hl_product_key_split_rows(ctx: *mut HlCtx, rows: *const i64, left: *mut i64, right: *mut i64, n: i64, side: i32) -> i32;
    pub fn hl_memory_selected_scores_forward(ctx: *mut HlCtx, indices: *const i64, query: *const f32, ld_query: i64, left_or_keys: *const f32, right_keys: *const f32, scores: *mut f32, tokens: i32, top_k: i32, side: i32, key_dim: i32, slots: i32) -> i32;
    pub fn hl_memory_selected_scores_backward(ctx: *mut HlCtx, indices: *const i64, query: *const f32, ld_query: i64, left_or_keys: *const f32, right_keys: *const f32, grad_scores: *const f32, grad_query: *mut f32, ld_grad_query: i64, grad_left_or_keys: *mut f32, grad_right_keys: *mut f32, tokens: i32, top_k: i32, side: i32, key_dim: i32, slots: i32) -> i32;
    pub fn hl_softmax_rows_f32(ctx: *mut HlCtx, x: *const f32, y: *mut f32, rows: i32, cols: i32) -> i32;
    pub fn hl_softmax_rows_backward_f32(ctx: *mut HlCtx, y: *const f32, grad_y: *const f32, grad_x: *mut f32, rows: i32, cols: i32) -> i32;
    pub fn hl_memory_weighted_value_forward(ctx: *mut HlCtx, indices: *const i64, weights: *const f32, values: *const f32, out: *mut f32, tokens: i32, top_k: i32, rows: i32, dim: i32) -> i32;
    pub fn hl_memory_weighted_value_backward(ctx: *mut HlCtx, indices: *const i64, weights: *const f32, values: *const f32, grad_out: *const f32, grad_weights: *mut f32, grad_values: *mut f32, tokens: i32, top_k: i32, rows: i32, dim: i32) -> i32;
    pub fn hl_mark_rows_u8(ctx: *mut HlCtx, selected_rows: *const i64, n_selected: i64, row_mask: *const u8, flags: *mut u8, rows: i32) -> i32;
    pub fn hl_mask_to_indices_u8(ctx: *mut HlCtx, mask: *const u8, rows: i32, out_indices: *mut i64, count_dev: *mut i32) -> i32;
    pub fn hl_gather_rows_f32(ctx: *mut HlCtx, src: *const f32, indices: *const i64, n: i32, dim: i32, dst: *mut f32) -> i32;
    pub fn hl_scatter_rows_f32(ctx: *mut HlCtx, src: *const f32, indices: *const i64, n: i32, dim: i32, dst: *mut f32) -> i32;
    pub fn hl_sparse_rows_sum_squares_f32(ctx: *mut HlCtx, grad: *const f32, selected_rows: *const i64, n_selected: i64, row_mask: *const u8, row_flags: *mut u8, rows: i32, row_dim: i32, sum_dev: *mut f64) -> i32;
    pub fn hl_sparse_adamw_rows_f32(ctx: *mut HlCtx, param: *mut f32, grad: *mut f32, m: *mut f32, v: *mut f32, selected_rows: *const i64, n_selected: i64, row_mask: *const u8, row_flags: *mut u8, rows: i32, row_dim: i32, hp: *const HlAdamwParams, zero_grad_rows: i32) -> i32;
    pub fn hl_nccl_version(out: *mut i32) -> i32;
    pub fn hl_nccl_unique_id(out: *mut u8) -> i32;
    pub fn hl_nccl_init(ctx: *mut HlCtx, rank: i32, world: i32, id: *const u8) -> i32;
    pub fn hl_nccl_allreduce_f32(ctx: *mut HlCtx, buf_dev: *mut f32, count: usize) -> i32;
    pub fn hl_nccl_allreduce_max_u8(ctx: *mut HlCtx, buf_dev: *mut u8, count: usize) -> i32;
    pub fn hl_nccl_abort(ctx: *mut HlCtx) -> i32;
    pub fn hl_nccl_destroy(ctx: *mut HlCtx) -> i32;
    pub fn hl_ddp_bucket_count(arena_elems: i64, bucket_elems: i64) -> i64;
    pub fn hl_ddp_ready_buckets(arena_elems: i64, bucket_elems: i64, next_bucket: i64, done_elems: i64, starts: *mut i64, counts: *mut i64, capacity: i32) -> i32;
    pub fn hl_decoder_create(ctx: *mut HlCtx, cfg: *const HlDecoderConfig, out: *mut *mut HlDecoder) -> i32;
    pub fn hl_memory_decoder_create(ctx: *mut HlCtx, cfg: *const HlDecoderConfig, mem: *const HlMemoryConfig, out: *mut *mut HlDecoder) -> i32;
    pub fn hl_decoder_optimizer_step_sparse_rows(model: *mut HlDecoder) -> i32;
    pub fn hl_decoder_optimizer_step_policy(model: *mut HlDecoder, policy: i32) -> i32;
    pub fn hl_memory_access_count_rows_i64_u64(ctx: *mut HlCtx, selected_rows: *const i64, n_selected: i64, slots: i32, counts: *mut u64) -> i32;
    pub fn hl_decoder_memory_access_counts(model: *mut HlDecoder, counts_dev: *mut u64) -> i32;
    pub fn hl_decoder_set_smft_masks(model: *mut HlDecoder, value_mask_host: *const u8, left_mask_host: *const u8, right_mask_host: *const u8) -> i32;
    pub fn hl_decoder_selected_indices(model: *mut HlDecoder, layer: i32, host: *mut i64, count: i64) -> i32;
    pub fn hl_decoder_destroy(model: *mut HlDecoder);
    pub fn hl_decoder_param_count(model: *mut HlDecoder) -> i32;
    pub fn hl_decoder_param_info(model: *mut HlDecoder, index: i32, name_out: *mut c_char, name_cap: usize, numel: *mut i64, rank: *mut i32, shape_out: *mut i64) -> i32;
    pub fn hl_decoder_set_param(model: *mut HlDecoder, index: i32, host: *const f32, numel: i64) -> i32;
    pub fn hl_decoder_get_param(model: *mut HlDecoder, index: i32, host: *mut f32, numel: i64) -> i32;
    pub fn hl_decoder_get_grad(model: *mut HlDecoder, index: i32, host: *mut f32, numel: i64) -> i32;
    pub fn hl_decoder_get_moments(model: *mut HlDecoder, index: i32, m_host: *mut f32, v_host: *mut f32, numel: i64) -> i32;
    pub fn hl_decoder_set_optimizer(model: *mut HlDecoder, opt: *const HlAdamwConfig) -> i32;
    pub fn hl_decoder_optimizer_steps(model: *mut HlDecoder) -> i64;
    pub fn hl_decoder_set_moments(model: *mut HlDecoder, index: i32, m_host: *const f32, v_host: *const f32, numel: i64) -> i32;
    pub fn hl_decoder_set_optimizer_steps(model: *mut HlDecoder, steps: i64) -> i32;
    pub fn hl_decoder_eval_loss(model: *mut HlDecoder, tokens_dev: *const i64, targets_dev: *const i64, sequences: i32, loss_host: *mut f32) -> i32;
    pub fn hl_decoder_next_token_logits(model: *mut HlDecoder, window_dev: *const i64, window_len: i32, logits_host: *mut f32) -> i32;
    pub fn hl_decoder_prefill(model: *mut HlDecoder, window_host: *const i64, window_len: i32, logits_host: *mut f32) -> i32;
    pub fn hl_decoder_decode_next(model: *mut HlDecoder, token: i64, logits_host: *mut f32) -> i32;
    pub fn hl_decoder_cached_positions(model: *mut HlDecoder) -> i32;
    pub fn hl_decoder_forward_backward(model: *mut HlDecoder, tokens_dev: *const i64, targets_dev: *const i64) -> i32;
    pub fn hl_decoder_optimizer_step(model: *mut HlDecoder) -> i32;
    pub fn hl_decoder_train_step_device(model: *mut HlDecoder, tokens_dev: *const i64, targets_dev: *const i64) -> i32;
    pub fn hl_decoder_train_step(model: *mut HlDecoder, tokens_host: *const i64, targets_host: *const i64, loss_host: *mut f32) -> i32;
    pub fn hl_decoder_loss(model: *mut HlDecoder, loss_host: *mut f32) -> i32;
    pub fn hl_decoder_launches_last_step(model: *mut HlDecoder) -> u64;
    pub fn hl_decoder_comm_exposed_ms(model: *mut HlDecoder, total_ms: *mut f32, waits: *mut i32) -> i32;
    pub fn hl_sample_token(logits: *const c_void, dtype: i32, vocab: i64, context: *const i64, n_context: i64, options: *const HlSamplingOptions, draw: f64, token: *mut i64, probability: *mut f64, log_probability: *mut f64) -> i32;
    pub fn hl_sample_rows(ctx: *mut HlCtx, logits: *const c_void, dtype: i32, ld: i64, rows: i32, vocab: i32, temperature: *const f32, top_k: *const i32, top_p: *const f32, min_p: *const f32, draws: *const f64, tokens: *mut i64, probabilities: *mut f32) -> i32;
    pub fn hl_decoder_generate_token(model: *mut HlDecoder, tokens: *const i64, length: i64, appended: i32, options: *const HlSamplingOptions, draw: f64, token: *mut i64, probability: *mut f64, log_probability: *mut f64) -> i32;
}

// ---------------------------------------------------------------------------------------------------------------
// Safe layer: the names and meaning of today's `heirloom_kernels::cuda::*` wrappers (file:line in the Heirloom tree).
// `CudaBuffer`, `CudaResult`, `CudaError` are the crate's own types (cuda.rs:259-280, :652-656); a buffer here is a
// reference-counted `hl_buffer` plus the element bookkeeping the crate already keeps.
// ---------------------------------------------------------------------------------------------------------------
use std::cell::RefCell;
use std::collections::HashMap;
use std::rc::Rc;

thread_local! {
    // one context per (thread, device), as the reference caches one stream per context per thread (cuda.rs:7653-7681)
    static CONTEXTS: RefCell<HashMap<i32, *mut HlCtx>> = RefCell::new(HashMap::new());
}

fn check(rc: i32) -> CudaResult<()> {
    if rc == HL_OK {
        return Ok(());
    }
    let msg = unsafe { std::ffi::CStr::from_ptr(hl_last_error()) }.to_string_lossy().into_owned();
    Err(CudaError::new(msg))
}

fn ctx_for(device_ordinal: i32) -> CudaResult<*mut HlCtx> {
    CONTEXTS.with(|map| {
        if let Some(ctx) = map.borrow().get(&device_ordinal) {
            return Ok(*ctx);
        }
        let mut ctx: *mut HlCtx = std::ptr::null_mut();
        check(unsafe { hl_ctx_create(device_ordinal, &mut ctx) })?;
        map.borrow_mut().insert(device_ordinal, ctx);
        Ok(ctx)
    })
}

struct Allocation {
    handle: *mut HlBuffer,
    device_ordinal: i32,
}
impl Drop for Allocation {
    fn drop(&mut self) {
        // the library frees in stream order, like the pending-release list of cuda.rs:7870-7922
        unsafe { hl_buffer_release(self.handle) };
    }
}

#[derive(Clone)]
pub struct CudaBuffer {
    inner: Rc<Allocation>,
    len: usize,
    element_size: usize,
}

impl CudaBuffer {
    pub fn uninit_bytes(device_ordinal: i32, len: usize, element_size: usize) -> CudaResult<Self> {
        let bytes = len.checked_mul(element_size).ok_or_else(|| CudaError::new("CUDA buffer byte length overflow"))?;
        let ctx = ctx_for(device_ordinal)?;
        let mut handle: *mut HlBuffer = std::ptr::null_mut();
        check(unsafe { hl_buffer_alloc(ctx, bytes.max(1), &mut handle) })?;
        Ok(Self { inner: Rc::new(Allocation { handle, device_ordinal }), len, element_size })
    }
    fn from_slice<T: Copy>(device_ordinal: i32, values: &[T]) -> CudaResult<Self> {
        let out = Self::uninit_bytes(device_ordinal, values.len(), std::mem::size_of::<T>())?;
        check(unsafe {
            hl_memcpy_h2d(ctx_for(device_ordinal)?, out.ptr(), values.as_ptr() as *const c_void, out.byte_len())
        })?;
        Ok(out)
    }
    fn to_vec<T: Copy + Default>(&self) -> CudaResult<Vec<T>> {
        let mut host = vec![T::default(); self.len];
        // waits for the compute stream first, as the reference's device-to-host copies do (cuda.rs:836)
        check(unsafe {
            hl_memcpy_d2h(ctx_for(self.device_ordinal())?, host.as_mut_ptr() as *mut c_void, self.ptr(), self.byte_len())
        })?;
        Ok(host)
    }
    pub fn from_f32(device_ordinal: i32, values: &[f32]) -> CudaResult<Self> { Self::from_slice(device_ordinal, values) }
    pub fn from_i64(device_ordinal: i32, values: &[i64]) -> CudaResult<Self> { Self::from_slice(device_ordinal, values) }
    pub fn from_u16(device_ordinal: i32, values: &[u16]) -> CudaResult<Self> { Self::from_slice(device_ordinal, values) }
    pub fn from_u8(device_ordinal: i32, values: &[u8]) -> CudaResult<Self> { Self::from_slice(device_ordinal, values) }
    pub fn to_f32(&self) -> CudaResult<Vec<f32>> { self.to_vec() }
    pub fn to_i64(&self) -> CudaResult<Vec<i64>> { self.to_vec() }
    pub fn to_u16(&self) -> CudaResult<Vec<u16>> { self.to_vec() }
    pub fn len(&self) -> usize { self.len }
    pub fn is_empty(&self) -> bool { self.len == 0 }
    pub fn element_size(&self) -> usize { self.element_size }
    pub fn byte_len(&self) -> usize { self.len * self.element_size }
    pub fn device_ordinal(&self) -> i32 { self.inner.device_ordinal }
    fn ptr(&self) -> *mut c_void { unsafe { hl_buffer_ptr(self.inner.handle) } }
}

fn ensure(buffer: &CudaBuffer, element_size: usize, label: &str) -> CudaResult<()> {
    if buffer.element_size() != element_size {
        return Err(CudaError::new(format!("{label} expects {element_size}-byte elements, got {}", buffer.element_size())));
    }
    Ok(())
}

fn dim(value: usize, label: &str) -> CudaResult<i32> {
    i32::try_from(value).map_err(|_| CudaError::new(format!("{label} exceeds the launch limit")))
}

/// cuda.rs add/sub/mul/div_f32_buffers (kernels.ptx:6-141)
fn binary(op: i32, lhs: &CudaBuffer, rhs: &CudaBuffer, label: &str) -> CudaResult<CudaBuffer> {
    ensure(lhs, 4, label)?;
    ensure(rhs, 4, label)?;
    if lhs.len() != rhs.len() || lhs.device_ordinal() != rhs.device_ordinal() {
        return Err(CudaError::new(format!("{label} expects equal lengths on one device")));
    }
    let out = CudaBuffer::uninit_bytes(lhs.device_ordinal(), lhs.len(), 4)?;
    check(unsafe {
        hl_binary_f32(ctx_for(lhs.device_ordinal())?, op, lhs.ptr() as *const f32, rhs.ptr() as *const f32,
                      out.ptr() as *mut f32, lhs.len())
    })?;
    Ok(out)
}
pub fn add_f32_buffers(lhs: &CudaBuffer, rhs: &CudaBuffer) -> CudaResult<CudaBuffer> { binary(HL_ADD, lhs, rhs, "add_f32_buffers") }
pub fn sub_f32_buffers(lhs: &CudaBuffer, rhs: &CudaBuffer) -> CudaResult<CudaBuffer> { binary(HL_SUB, lhs, rhs, "sub_f32_buffers") }
pub fn mul_f32_buffers(lhs: &CudaBuffer, rhs: &CudaBuffer) -> CudaResult<CudaBuffer> { binary(HL_MUL, lhs, rhs, "mul_f32_buffers") }
pub fn div_f32_buffers(lhs: &CudaBuffer, rhs: &CudaBuffer) -> CudaResult<CudaBuffer> { binary(HL_DIV, lhs, rhs, "div_f32_buffers") }

/// cuda.rs gelu_f32_buffer / gelu_backward_f32_buffers (kernels.ptx:4786-4907)
pub fn gelu_f32_buffer(input: &CudaBuffer) -> CudaResult<CudaBuffer> {
    ensure(input, 4, "gelu_f32_buffer")?;
    let out = CudaBuffer::uninit_bytes(input.device_ordinal(), input.len(), 4)?;
    check(unsafe { hl_gelu(ctx_for(input.device_ordinal())?, input.ptr(), out.ptr(), HL_F32, input.len()) })?;
    Ok(out)
}
pub fn gelu_backward_f32_buffers(input: &CudaBuffer, grad_out: &CudaBuffer) -> CudaResult<CudaBuffer> {
    ensure(input, 4, "gelu_backward_f32_buffers")?;
    let out = CudaBuffer::uninit_bytes(input.device_ordinal(), input.len(), 4)?;
    check(unsafe {
        hl_gelu_backward(ctx_for(input.device_ordinal())?, input.ptr(), grad_out.ptr(), out.ptr(), HL_F32, input.len())
    })?;
    Ok(out)
}

/// cuda.rs f32_to_bf16_bits_buffer / bf16_bits_to_f32_buffer (kernels.ptx:174-237; storage.rs:440-449)
pub fn f32_to_bf16_bits_buffer(input: &CudaBuffer) -> CudaResult<CudaBuffer> {
    ensure(input, 4, "f32_to_bf16_bits_buffer")?;
    let out = CudaBuffer::uninit_bytes(input.device_ordinal(), input.len(), 2)?;
    check(unsafe { hl_cast(ctx_for(input.device_ordinal())?, input.ptr(), HL_F32, out.ptr(), HL_BF16, input.len()) })?;
    Ok(out)
}
pub fn bf16_bits_to_f32_buffer(input: &CudaBuffer) -> CudaResult<CudaBuffer> {
    ensure(input, 2, "bf16_bits_to_f32_buffer")?;
    let out = CudaBuffer::uninit_bytes(input.device_ordinal(), input.len(), 4)?;
    check(unsafe { hl_cast(ctx_for(input.device_ordinal())?, input.ptr(), HL_BF16, out.ptr(), HL_F32, input.len()) })?;
    Ok(out)
}

/// cuda.rs layer_norm_forward_f32_buffers (kernels.ptx:3260-3384)
pub fn layer_norm_forward_f32_buffers(x: &CudaBuffer, gamma: &CudaBuffer, beta: &CudaBuffer, rows: usize,
                                      features: usize, eps: f32) -> CudaResult<CudaBuffer> {
    ensure(x, 4, "layer_norm_forward_f32_buffers")?;
    let out = CudaBuffer::uninit_bytes(x.device_ordinal(), rows * features, 4)?;
    check(unsafe {
        hl_layer_norm_forward(ctx_for(x.device_ordinal())?, x.ptr(), HL_F32, gamma.ptr() as *const f32,
                              beta.ptr() as *const f32, out.ptr(), HL_F32, std::ptr::null_mut(), std::ptr::null_mut(),
                              dim(rows, "layer norm rows")?, dim(features, "layer norm features")?, eps)
    })?;
    Ok(out)
}

/// cuda.rs embedding_f32_i64_buffers (kernels.ptx:1660-1713); rows that are out of range are reported by the next sync
pub fn embedding_f32_i64_buffers(weight: &CudaBuffer, indices: &CudaBuffer, vocab: usize, dim_: usize) -> CudaResult<CudaBuffer> {
    ensure(weight, 4, "embedding_f32_i64_buffers weight")?;
    ensure(indices, 8, "embedding_f32_i64_buffers indices")?;
    let out = CudaBuffer::uninit_bytes(weight.device_ordinal(), indices.len() * dim_, 4)?;
    let ctx = ctx_for(weight.device_ordinal())?;
    check(unsafe {
        hl_embedding_forward(ctx, weight.ptr() as *const f32, dim(vocab, "vocab")?, indices.ptr() as *const i64,
                             std::ptr::null(), 0, out.ptr(), HL_F32, dim(indices.len(), "tokens")?, dim(dim_, "dim")?)
    })?;
    check(unsafe { hl_ctx_sync(ctx) })?; // the reference reads its status word after the launch (cuda.rs:7184-7193)
    Ok(out)
}

/// cuda.rs matmul_bf16_tensor_core_rhs_transposed_f32_buffers (cuda.rs:4215-4386): C[m,n] = A[m,k] · B[n,k]ᵀ,
/// bf16 operands, f32 result; pad / crop / transpose kernels are gone, ragged edges are handled by the tile loads
pub fn matmul_bf16_tensor_core_rhs_transposed_f32_buffers(lhs_bf16: &CudaBuffer, rhs_bf16: &CudaBuffer, m: usize,
                                                          n: usize, k: usize) -> CudaResult<CudaBuffer> {
    ensure(lhs_bf16, 2, "matmul_bf16_tensor_core lhs")?;
    ensure(rhs_bf16, 2, "matmul_bf16_tensor_core rhs")?;
    let out = CudaBuffer::uninit_bytes(lhs_bf16.device_ordinal(), m * n, 4)?;
    let desc = HlGemmDesc { m: dim(m, "m")?, n: dim(n, "n")?, k: dim(k, "k")?, a_layout: HL_K_MAJOR, b_layout: HL_K_MAJOR,
                            lda: k as i64, ldb: k as i64, ldc: n as i64, epilogue: HL_EPI_NONE, out_dtype: HL_F32,
                            split_k: 0, ld_aux_in: 0, ld_aux_out: 0, a_k_period: 0, b_k_period: 0 };
    check(unsafe {
        hl_gemm_bf16(ctx_for(lhs_bf16.device_ordinal())?, &desc, lhs_bf16.ptr(), rhs_bf16.ptr(), out.ptr(),
                     std::ptr::null(), std::ptr::null(), std::ptr::null_mut())
    })?;
    Ok(out)
}

/// cuda.rs causal_attention_bf16_flash_tensor_core_forward_f32_buffers (cuda.rs:5283-5420): returns (output, lse)
pub fn causal_attention_bf16_flash_forward_buffers(q: &CudaBuffer, k: &CudaBuffer, v: &CudaBuffer,
                                                   dims: CausalAttentionDims) -> CudaResult<(CudaBuffer, CudaBuffer)> {
    let channels = dims.channels;  // heads interleaved along the channel dimension (src/tensor.rs:5156-5177)
    let head_dim = channels / dims.n_heads;
    let out = CudaBuffer::uninit_bytes(q.device_ordinal(), dims.batch * dims.time * channels, 2)?;
    let lse = CudaBuffer::uninit_bytes(q.device_ordinal(), dims.batch * dims.n_heads * dims.time, 4)?;
    check(unsafe {
        hl_flash_attention_forward(ctx_for(q.device_ordinal())?, q.ptr(), k.ptr(), v.ptr(), channels as i64, out.ptr(),
                                   channels as i64, lse.ptr() as *mut f32, dim(dims.batch, "batch")?,
                                   dim(dims.time, "time")?, dim(dims.n_heads, "heads")?, dim(head_dim, "head_dim")?)
    })?;
    Ok((out, lse))
}

/// cuda.rs sgd_update_f32_buffer (cuda.rs:6280-6303)
pub fn sgd_update_f32_buffer(param: &CudaBuffer, grad: &CudaBuffer, lr: f32) -> CudaResult<()> {
    ensure(param, 4, "sgd_update_f32_buffer param")?;
    ensure(grad, 4, "sgd_update_f32_buffer grad")?;
    check(unsafe {
        hl_sgd_update_f32(ctx_for(param.device_ordinal())?, param.ptr() as *mut f32, grad.ptr() as *const f32, lr, param.len())
    })
}

/// cuda.rs adamw_update_f32_buffers (cuda.rs:6305-6334; kernels.ptx:390-468): same operation order as the reference kernel
pub fn adamw_update_f32_buffers(param: &CudaBuffer, grad: &CudaBuffer, m: &CudaBuffer, v: &CudaBuffer,
                                params: AdamWParams) -> CudaResult<()> {
    let hp = HlAdamwParams { lr: params.lr, beta1: params.beta1, beta2: params.beta2, eps: params.eps,
                             weight_decay: params.weight_decay, clip_scale: params.clip_scale,
                             bias_correction1: params.bias_correction1, bias_correction2: params.bias_correction2 };
    check(unsafe {
        hl_adamw_f32(ctx_for(param.device_ordinal())?, param.ptr() as *mut f32, grad.ptr() as *const f32,
                     m.ptr() as *mut f32, v.ptr() as *mut f32, param.len(), &hp)
    })
}

/// cuda.rs i64_arange_buffer (cuda.rs:2090-2103)
pub fn i64_arange_buffer(device_ordinal: i32, len: usize) -> CudaResult<CudaBuffer> {
    let out = CudaBuffer::uninit_bytes(device_ordinal, len, 8)?;
    check(unsafe { hl_arange_i64(ctx_for(device_ordinal)?, out.ptr() as *mut i64, len) })?;
    Ok(out)
}

/// cuda.rs concat_i64_buffers (cuda.rs:6437-6490)
pub fn concat_i64_buffers(inputs: &[CudaBuffer]) -> CudaResult<CudaBuffer> {
    let first = inputs.first().ok_or_else(|| CudaError::new("concat_i64_buffers requires at least one input buffer"))?;
    let total: usize = inputs.iter().map(|b| b.len()).sum();
    let out = CudaBuffer::uninit_bytes(first.device_ordinal(), total, 8)?;
    let ptrs: Vec<*const i64> = inputs.iter().map(|b| b.ptr() as *const i64).collect();
    let lens: Vec<usize> = inputs.iter().map(|b| b.len()).collect();
    check(unsafe {
        hl_concat_i64(ctx_for(first.device_ordinal())?, ptrs.as_ptr(), lens.as_ptr(), dim(inputs.len(), "inputs")?,
                      out.ptr() as *mut i64, total)
    })?;
    Ok(out)
}

/// cuda.rs memory_product_key_topk_from_side_scores (kernels.ptx product-key family): i64 slots [tokens, top_k]
pub fn product_key_topk_from_side_scores_buffers(left: &CudaBuffer, right: &CudaBuffer, tokens: usize, side: usize,
                                                 top_k: usize, beam: usize) -> CudaResult<CudaBuffer> {
    let out = CudaBuffer::uninit_bytes(left.device_ordinal(), tokens * top_k, 8)?;
    check(unsafe {
        hl_product_key_topk_from_side_scores(ctx_for(left.device_ordinal())?, left.ptr() as *const f32,
                                             right.ptr() as *const f32, out.ptr() as *mut i64, dim(tokens, "tokens")?,
                                             dim(side, "side")?, dim(top_k, "top_k")?, dim(beam, "beam")?)
    })?;
    Ok(out)
}

/// NcclCommunicator::all_reduce_sum_in_place_f32 (cuda.rs:8049-8233) on the context's collective stream
pub fn nccl_all_reduce_sum_in_place_f32(buffer: &CudaBuffer) -> CudaResult<()> {
    ensure(buffer, 4, "all_reduce_sum_in_place_f32")?;
    check(unsafe { hl_nccl_allreduce_f32(ctx_for(buffer.device_ordinal())?, buffer.ptr() as *mut f32, buffer.len()) })
}

/// The loop body of `train-lm` (src/bin/heirloom/commands/training.rs:125-167) as one call: host token ids in, loss out.
pub struct B200Decoder {
    handle: *mut HlDecoder,
}
impl B200Decoder {
    pub fn new(device_ordinal: i32, config: HlDecoderConfig) -> CudaResult<Self> {
        let mut handle: *mut HlDecoder = std::ptr::null_mut();
        check(unsafe { hl_decoder_create(ctx_for(device_ordinal)?, &config, &mut handle) })?;
        Ok(Self { handle })
    }
    pub fn set_parameter(&mut self, state_dict_index: usize, values: &[f32]) -> CudaResult<()> {
        check(unsafe { hl_decoder_set_param(self.handle, dim(state_dict_index, "index")?, values.as_ptr(), values.len() as i64) })
    }
    pub fn set_optimizer(&mut self, config: HlAdamwConfig) -> CudaResult<()> {
        check(unsafe { hl_decoder_set_optimizer(self.handle, &config) })
    }
    pub fn train_step(&mut self, tokens: &[i64], targets: &[i64]) -> CudaResult<f32> {
        let mut loss = 0f32;
        check(unsafe { hl_decoder_train_step(self.handle, tokens.as_ptr(), targets.as_ptr(), &mut loss) })?;
        Ok(loss)
    }
}
impl Drop for B200Decoder {
    fn drop(&mut self) {
        unsafe { hl_decoder_destroy(self.handle) };
    }
}

