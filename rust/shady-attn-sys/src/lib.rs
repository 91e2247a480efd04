//! Raw bindings of `libshady_attn` (the C ABI in `include/shady_attn.h`): the CUDA backend of
//! shady-thinker's attention hot path for B200 (sm_100a).
//!
//! GENERATED by `gen_bindings.py` from the header; do not edit by hand.  This crate has not been
//! compiled where it was written (no Rust toolchain there); the same ABI is exercised from C++ and
//! Python by the repository's tests.
#![allow(non_camel_case_types, clippy::too_many_arguments)]
use std::os::raw::{c_char, c_int, c_void};

pub const SHADY_OK: c_int = 0;
pub const SHADY_ERR_BAD_ARG: c_int = 1;
pub const SHADY_ERR_UNSUPPORTED: c_int = 2;
pub const SHADY_ERR_CUDA: c_int = 3;
pub const SHADY_ERR_WORKSPACE: c_int = 4;
pub const SHADY_ERR_TIMEOUT: c_int = 5;
pub const SHADY_F32: u32 = 0;
pub const SHADY_F16: u32 = 1;
pub const SHADY_BF16: u32 = 2;
pub const SHADY_F8E4M3: u32 = 3;
pub const SHADY_F8E5M2: u32 = 4;

/// Opaque `shady_ctx`.
#[repr(C)]
pub struct ShadyCtx { _private: [u8; 0] }

/// `shady_kv_cache` — same fields, same order.
#[repr(C)]
#[derive(Clone, Copy)]
pub struct ShadyKvCache {
    pub d_k_base: *mut c_void,
    pub d_v_base: *mut c_void,
    pub seq_stride: u64,
    pub d_k_ptrs: *const *mut c_void,
    pub d_v_ptrs: *const *mut c_void,
    pub dtype: u32,
    pub page_rows: u32,
    pub d_page_table: *const u32,
    pub max_pages_per_seq: u32,
    pub k_scale: f32,
    pub v_scale: f32,
    pub _pad: u32,
}

/// `shady_append_params` — same fields, same order.
#[repr(C)]
#[derive(Clone, Copy)]
pub struct ShadyAppendParams {
    pub num_heads: u32,
    pub num_kv_heads: u32,
    pub head_dim: u32,
    pub eps: f32,
    pub rope_theta: f32,
    pub rotary_dim: u32,
    pub s1_limit: u32,
    pub s2_limit: u32,
    pub interleaved: u32,
    pub num_seqs: u32,
    pub tokens_per_seq: u32,
    pub in_dtype: u32,
    pub q_dtype: u32,
    pub has_gate: u32,
    pub write_k_back: u32,
    pub _pad: u32,
}

/// `shady_decode_params` — same fields, same order.
#[repr(C)]
#[derive(Clone, Copy)]
pub struct ShadyDecodeParams {
    pub head_dim: u32,
    pub num_kv_heads: u32,
    pub num_q_heads: u32,
    pub heads_per_kv: u32,
    pub num_splits: u32,
    pub num_seqs: u32,
    pub q_dtype: u32,
    pub out_dtype: u32,
}

/// `shady_prefill_params` — same fields, same order.
#[repr(C)]
#[derive(Clone, Copy)]
pub struct ShadyPrefillParams {
    pub head_dim: u32,
    pub num_kv_heads: u32,
    pub num_q_heads: u32,
    pub num_seqs: u32,
    pub seq_len: u32,
    pub dtype: u32,
}

/// `shady_prefill_batch` — same fields, same order.
#[repr(C)]
#[derive(Clone, Copy)]
pub struct ShadyPrefillBatch {
    pub h_seq_lens: *const u32,
    pub h_k_ptrs: *const *const c_void,
    pub h_v_ptrs: *const *const c_void,
}

/// `shady_gptq_weight` — same fields, same order.
#[repr(C)]
#[derive(Clone, Copy)]
pub struct ShadyGptqWeight {
    pub d_qweight: *const u32,
    pub d_scales: *const u32,
    pub K: u32,
    pub N: u32,
    pub group_size: u32,
    pub _pad: u32,
}

/// `shady_rowq_cache` — same fields, same order.
#[repr(C)]
#[derive(Clone, Copy)]
pub struct ShadyRowqCache {
    pub d_k_codes: *mut c_void,
    pub d_v_codes: *mut c_void,
    pub d_k_scales: *mut f32,
    pub d_v_scales: *mut f32,
    pub seq_rows: u64,
    pub d_page_table: *const u32,
    pub page_rows: u32,
    pub max_pages_per_seq: u32,
    pub num_pages: u32,
    pub _pad: u32,
}

/// `shady_score_rule` — same fields, same order.
#[repr(C)]
#[derive(Clone, Copy)]
pub struct ShadyScoreRule {
    pub scale: f32,
    pub cap: f32,
    pub window: u32,
    pub _pad: u32,
    pub d_slopes: *const f32,
    pub d_prefix_lens: *const u32,
    pub d_doc_start: *const u32,
}

extern "C" {
    pub fn shady_ctx_create(device: c_int, stream: *mut c_void, out: *mut *mut ShadyCtx) -> c_int;
    pub fn shady_ctx_destroy(ctx: *mut ShadyCtx) -> c_int;
    pub fn shady_last_error(ctx: *const ShadyCtx) -> *const c_char;
    pub fn shady_ctx_stream(ctx: *const ShadyCtx) -> *mut c_void;
    pub fn shady_ctx_launch_count(ctx: *const ShadyCtx) -> u64;
    pub fn shady_ctx_set_wait_limits(ctx: *mut ShadyCtx, grid_polls: u32, peer_polls: u32, mbarrier_polls: u32) -> c_int;
    pub fn shady_buffer_create(ctx: *mut ShadyCtx, bytes: usize, d_out: *mut *mut c_void) -> c_int;
    pub fn shady_buffer_free(ctx: *mut ShadyCtx, d_buf: *mut c_void) -> c_int;
    pub fn shady_buffer_write(ctx: *mut ShadyCtx, d_buf: *mut c_void, offset: usize, src: *const c_void, bytes: usize) -> c_int;
    pub fn shady_buffer_read(ctx: *mut ShadyCtx, d_buf: *const c_void, offset: usize, dst: *mut c_void, bytes: usize) -> c_int;
    pub fn shady_buffer_copy(ctx: *mut ShadyCtx, d_src: *const c_void, d_dst: *mut c_void, bytes: usize) -> c_int;
    pub fn shady_host_device_ptr(ctx: *mut ShadyCtx, host_ptr: *const c_void, d_ptr: *mut *mut c_void) -> c_int;
    pub fn shady_flush(ctx: *mut ShadyCtx) -> c_int;
    pub fn shady_synchronize(ctx: *mut ShadyCtx) -> c_int;
    pub fn shady_kv_append_rope(ctx: *mut ShadyCtx, p: *const ShadyAppendParams, d_q_proj_full: *const c_void, d_k_proj: *mut c_void, d_v_proj: *const c_void, d_q_out: *mut c_void, d_q_gate: *mut f32, cache: *const ShadyKvCache, d_qk_norm_bf16: *const u16, d_pos_start: *const u32, d_pos_h: *const u32, d_pos_w: *const u32) -> c_int;
    pub fn shady_decode_workspace_size(p: *const ShadyDecodeParams, bytes: *mut usize) -> c_int;
    pub fn shady_decode_workspace_init(ctx: *mut ShadyCtx, p: *const ShadyDecodeParams, d_workspace: *mut c_void, workspace_bytes: usize) -> c_int;
    pub fn shady_attn_decode(ctx: *mut ShadyCtx, p: *const ShadyDecodeParams, d_q: *const c_void, cache: *const ShadyKvCache, d_seq_lens: *const u32, seq_lens_host: *const u32, d_out: *mut c_void, d_lse: *mut f32, d_gate: *const f32, d_workspace: *mut c_void, workspace_bytes: usize) -> c_int;
    pub fn shady_attn_decode_append(ctx: *mut ShadyCtx, ap: *const ShadyAppendParams, p: *const ShadyDecodeParams, d_q_proj_full: *const c_void, d_k_proj: *const c_void, d_v_proj: *const c_void, d_qk_norm_bf16: *const u16, cache: *const ShadyKvCache, d_seq_lens: *const u32, seq_lens_host: *const u32, d_out: *mut c_void, d_lse: *mut f32, d_workspace: *mut c_void, workspace_bytes: usize) -> c_int;
    pub fn shady_attn_decode_shard(ctx: *mut ShadyCtx, p: *const ShadyDecodeParams, d_q: *const c_void, cache: *const ShadyKvCache, d_seq_lens: *const u32, seq_lens_host: *const u32, d_records: *mut f32, d_workspace: *mut c_void, workspace_bytes: usize) -> c_int;
    pub fn shady_ipc_export(ctx: *mut ShadyCtx, d_buf: *mut c_void, handle: *mut u8) -> c_int;
    pub fn shady_ipc_open(ctx: *mut ShadyCtx, handle: *const u8, d_peer: *mut *mut c_void) -> c_int;
    pub fn shady_ipc_close(ctx: *mut ShadyCtx, d_peer: *mut c_void) -> c_int;
    pub fn shady_combine_p2p_buffer_size(world: u32, num_heads: u32, head_dim: u32, bytes: *mut usize) -> c_int;
    pub fn shady_attn_combine_p2p(ctx: *mut ShadyCtx, world: u32, rank: u32, num_heads: u32, head_dim: u32, epoch: u32, d_peer_table: *const *mut c_void, d_records: *const f32, d_out: *mut c_void, out_dtype: u32, d_gate: *const f32) -> c_int;
    pub fn shady_attn_decode_shard_p2p(ctx: *mut ShadyCtx, p: *const ShadyDecodeParams, d_q: *const c_void, cache: *const ShadyKvCache, d_seq_lens: *const u32, seq_lens_host: *const u32, world: u32, rank: u32, epoch: u32, d_peer_table: *const *mut c_void, d_records: *mut f32, d_out: *mut c_void, out_dtype: u32, d_gate: *const f32, d_workspace: *mut c_void, workspace_bytes: usize) -> c_int;
    pub fn shady_attn_decode_static(ctx: *mut ShadyCtx, p: *const ShadyDecodeParams, d_q: *const c_void, cache: *const ShadyKvCache, d_seq_lens: *const u32, seq_lens_host: *const u32, d_out: *mut c_void, d_lse: *mut f32, d_gate: *const f32) -> c_int;
    pub fn shady_attn_decode_partials(ctx: *mut ShadyCtx, p: *const ShadyDecodeParams, d_q: *const c_void, cache: *const ShadyKvCache, d_seq_lens: *const u32, d_partials: *mut f32) -> c_int;
    pub fn shady_attn_reduce(ctx: *mut ShadyCtx, head_dim: u32, num_splits: u32, num_heads: u32, split_stride: u64, head_stride: u64, d_partials: *const f32, d_out: *mut c_void, out_dtype: u32, d_gate: *const f32) -> c_int;
    pub fn shady_attn_prefill(ctx: *mut ShadyCtx, p: *const ShadyPrefillParams, d_q: *const c_void, cache: *const ShadyKvCache, d_out: *mut c_void) -> c_int;
    pub fn shady_prefill_workspace_size(p: *const ShadyPrefillParams, bytes: *mut usize) -> c_int;
    pub fn shady_attn_prefill_append(ctx: *mut ShadyCtx, ap: *const ShadyAppendParams, p: *const ShadyPrefillParams, d_q_proj_full: *const c_void, d_k_proj: *const c_void, d_v_proj: *const c_void, d_qk_norm_bf16: *const u16, cache: *const ShadyKvCache, d_out: *mut c_void, d_workspace: *mut c_void, workspace_bytes: usize) -> c_int;
    pub fn shady_prefill_ragged_workspace_size(p: *const ShadyPrefillParams, h_seq_lens: *const u32, with_append: c_int, bytes: *mut usize) -> c_int;
    pub fn shady_attn_prefill_ragged(ctx: *mut ShadyCtx, p: *const ShadyPrefillParams, batch: *const ShadyPrefillBatch, d_q: *const c_void, cache: *const ShadyKvCache, d_out: *mut c_void, d_workspace: *mut c_void, workspace_bytes: usize) -> c_int;
    pub fn shady_attn_prefill_append_ragged(ctx: *mut ShadyCtx, ap: *const ShadyAppendParams, p: *const ShadyPrefillParams, batch: *const ShadyPrefillBatch, d_q_proj_full: *const c_void, d_k_proj: *const c_void, d_v_proj: *const c_void, d_qk_norm_bf16: *const u16, cache: *const ShadyKvCache, d_out: *mut c_void, d_workspace: *mut c_void, workspace_bytes: usize) -> c_int;
    pub fn shady_sigmoid_mul(ctx: *mut ShadyCtx, d_x: *mut f32, d_gate: *const f32, n: u32) -> c_int;
    pub fn shady_gptq_matvec(ctx: *mut ShadyCtx, w: *const ShadyGptqWeight, d_x: *const f32, d_y: *mut f32, num_vecs: u32) -> c_int;
    pub fn shady_qkv_proj_append(ctx: *mut ShadyCtx, p: *const ShadyAppendParams, wq: *const ShadyGptqWeight, wk: *const ShadyGptqWeight, wv: *const ShadyGptqWeight, d_x: *const f32, d_q_out: *mut c_void, d_q_gate: *mut f32, cache: *const ShadyKvCache, d_qk_norm_bf16: *const u16, d_pos_start: *const u32, d_pos_h: *const u32, d_pos_w: *const u32) -> c_int;
    pub fn shady_kv_append_rowq(ctx: *mut ShadyCtx, p: *const ShadyAppendParams, d_q_proj_full: *const c_void, d_k_proj: *const c_void, d_v_proj: *const c_void, d_q_out: *mut c_void, d_q_gate: *mut f32, d_k_out: *mut c_void, d_v_out: *mut c_void, cache: *const ShadyRowqCache, d_qk_norm_bf16: *const u16, d_pos_start: *const u32, d_pos_h: *const u32, d_pos_w: *const u32, d_tok_start: *const u32, total_tokens: u32) -> c_int;
    pub fn shady_kv_read_rowq(ctx: *mut ShadyCtx, cache: *const ShadyRowqCache, num_kv_heads: u32, head_dim: u32, num_seqs: u32, d_row_start: *const u32, d_out_start: *const u32, total_rows: u32, d_k_out: *mut c_void, d_v_out: *mut c_void, out_dtype: u32) -> c_int;
    pub fn shady_decode_rule_workspace_size(ctx: *mut ShadyCtx, p: *const ShadyDecodeParams, bytes: *mut usize) -> c_int;
    pub fn shady_decode_rule_workspace_init(ctx: *mut ShadyCtx, p: *const ShadyDecodeParams, d_workspace: *mut c_void, workspace_bytes: usize) -> c_int;
    pub fn shady_attn_decode_rule(ctx: *mut ShadyCtx, p: *const ShadyDecodeParams, rule: *const ShadyScoreRule, d_q: *const c_void, cache: *const ShadyKvCache, rowq: *const ShadyRowqCache, d_seq_lens: *const u32, d_out: *mut c_void, d_lse: *mut f32, d_workspace: *mut c_void, workspace_bytes: usize) -> c_int;
    pub fn shady_attn_prefill_rule(ctx: *mut ShadyCtx, p: *const ShadyPrefillParams, rule: *const ShadyScoreRule, d_q: *const c_void, cache: *const ShadyKvCache, cache_rows: u64, d_q_starts: *const u32, total_q: u32, d_kv_starts: *const u32, d_kv_lens: *const u32, d_out: *mut c_void, d_lse: *mut f32) -> c_int;
    pub fn shady_fill_randn(ctx: *mut ShadyCtx, d_dst: *mut c_void, n: u64, dtype: u32, seed: u64, tensor_id: u64, first_idx: u64) -> c_int;
}
