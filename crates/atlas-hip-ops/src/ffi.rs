// Generated by crates/atlas-hip-ops/gen_ffi.py from include/atlas_hip_ops.h and
// include/atlas_gguf.h; do not edit by hand.  Raw declarations of
// libatlas_hip_ops.so: every pointer is a device pointer unless the header
// says otherwise (the atlas_ops_* host-slice entry points take host memory).
#![allow(non_camel_case_types, dead_code)]

use std::os::raw::{c_char, c_int, c_void};

#[repr(C)]
pub struct AtlasHipCtx {
    _private: [u8; 0],
}

#[repr(C)]
pub struct AtlasGguf {
    _private: [u8; 0],
}

/// atlas_dispatch_timing (DispatchTiming, crates/atlas-metal/src/lib.rs:81-88).
#[repr(C)]
#[derive(Debug, Default, Clone, Copy)]
pub struct AtlasDispatchTiming {
    pub wall_ms: f64,
    pub gpu_ms: f64,
}

/// atlas_hip_telemetry (RuntimeTelemetry, crates/atlas-metal/src/lib.rs:91-193).
#[repr(C)]
#[derive(Debug, Default, Clone, Copy)]
pub struct AtlasHipTelemetry {
    pub dispatches: u64,
    pub syncs: u64,
    pub upload_bytes: u64,
    pub readback_bytes: u64,
    pub allocations: u64,
    pub resident_bytes: u64,
    pub peak_resident_bytes: u64,
}

/// atlas_gguf_tensor (GgufTensor, crates/atlas-core/src/gguf.rs:80-87).
#[repr(C)]
#[derive(Debug, Clone, Copy)]
pub struct AtlasGgufTensor {
    pub name: *const c_char,
    pub name_len: u64,
    pub n_dims: u32,
    pub dims: [u64; 4],
    pub type_: u32,
    pub offset: u64,
    pub bytes: u64,
}

pub const ATLAS_OK: c_int = 0;
pub const ATLAS_ERR_NO_DEVICE: c_int = -1;
pub const ATLAS_ERR_INVALID_INPUT: c_int = -2;
pub const ATLAS_ERR_COMMAND_FAILED: c_int = -3;
pub const ATLAS_ERR_OUT_OF_MEMORY: c_int = -4;

pub const ATLAS_REDUCTION_SEQUENTIAL: c_int = 0;
pub const ATLAS_REDUCTION_WIDE: c_int = 1;
pub const ATLAS_REDUCTION_AUTO: c_int = 2;

pub const ATLAS_GGUF_F32: u32 = 0;
pub const ATLAS_GGUF_F16: u32 = 1;
pub const ATLAS_GGUF_Q4_0: u32 = 2;
pub const ATLAS_GGUF_Q8_0: u32 = 8;
pub const ATLAS_GGUF_Q6_K: u32 = 14;

#[link(name = "atlas_hip_ops")]
extern "C" {
    // include/atlas_hip_ops.h
    pub fn atlas_hip_device_count(count: *mut c_int) -> c_int;
    pub fn atlas_hip_init(device: c_int, out: *mut *mut AtlasHipCtx) -> c_int;
    pub fn atlas_hip_destroy(ctx: *mut AtlasHipCtx);
    pub fn atlas_hip_sync(ctx: *mut AtlasHipCtx) -> c_int;
    pub fn atlas_hip_set_stream(ctx: *mut AtlasHipCtx, hip_stream: *mut c_void) -> c_int;
    pub fn atlas_hip_get_stream(ctx: *mut AtlasHipCtx) -> *mut c_void;
    pub fn atlas_hip_set_reduction(ctx: *mut AtlasHipCtx, reduction: c_int) -> c_int;
    pub fn atlas_hip_last_error(ctx: *const AtlasHipCtx) -> *const c_char;
    pub fn atlas_hip_get_telemetry(ctx: *const AtlasHipCtx, out: *mut AtlasHipTelemetry) -> c_int;
    pub fn atlas_hip_malloc(ctx: *mut AtlasHipCtx, bytes: usize, device_ptr: *mut *mut c_void) -> c_int;
    pub fn atlas_hip_free(ctx: *mut AtlasHipCtx, device_ptr: *mut c_void) -> c_int;
    pub fn atlas_hip_upload(ctx: *mut AtlasHipCtx, device_dst: *mut c_void, host_src: *const c_void, bytes: usize) -> c_int;
    pub fn atlas_hip_download(ctx: *mut AtlasHipCtx, host_dst: *mut c_void, device_src: *const c_void, bytes: usize) -> c_int;
    pub fn atlas_hip_memset(ctx: *mut AtlasHipCtx, device_dst: *mut c_void, value: c_int, bytes: usize) -> c_int;
    pub fn atlas_hip_copy_d2d(ctx: *mut AtlasHipCtx, device_dst: *mut c_void, device_src: *const c_void, bytes: usize) -> c_int;
    pub fn atlas_hip_event_create(ctx: *mut AtlasHipCtx, event: *mut *mut c_void) -> c_int;
    pub fn atlas_hip_event_record(ctx: *mut AtlasHipCtx, event: *mut c_void) -> c_int;
    pub fn atlas_hip_event_elapsed_ms(ctx: *mut AtlasHipCtx, start: *mut c_void, stop: *mut c_void, ms: *mut f32) -> c_int;
    pub fn atlas_hip_event_destroy(ctx: *mut AtlasHipCtx, event: *mut c_void) -> c_int;
    pub fn atlas_hip_graph_begin(ctx: *mut AtlasHipCtx) -> c_int;
    pub fn atlas_hip_graph_end(ctx: *mut AtlasHipCtx, graph: *mut *mut c_void) -> c_int;
    pub fn atlas_hip_graph_launch(ctx: *mut AtlasHipCtx, graph: *mut c_void) -> c_int;
    pub fn atlas_hip_graph_destroy(ctx: *mut AtlasHipCtx, graph: *mut c_void) -> c_int;
    pub fn atlas_hip_rms_norm_f32(ctx: *mut AtlasHipCtx, input: *const f32, weight: *const f32, output: *mut f32, rows: u32, hidden: u32, epsilon: f32) -> c_int;
    pub fn atlas_hip_rms_norm_residual_f32(ctx: *mut AtlasHipCtx, input: *const f32, weight: *const f32, residual: *const f32, normalized: *mut f32, output: *mut f32, rows: u32, hidden: u32, epsilon: f32) -> c_int;
    pub fn atlas_hip_add_rms_norm_f32(ctx: *mut AtlasHipCtx, input: *const f32, residual: *const f32, weight: *const f32, residual_out: *mut f32, output: *mut f32, rows: u32, hidden: u32, epsilon: f32) -> c_int;
    pub fn atlas_hip_rms_norm_add_scale_f32(ctx: *mut AtlasHipCtx, input: *const f32, weight: *const f32, state: *mut f32, scale: *const f32, rows: u32, hidden: u32, epsilon: f32) -> c_int;
    pub fn atlas_hip_rms_norm_groups_stable_f32(ctx: *mut AtlasHipCtx, values: *mut f32, weight: *const f32, width: u32, groups: u32, epsilon: f32) -> c_int;
    pub fn atlas_hip_rms_norm_f16(ctx: *mut AtlasHipCtx, input: *const u16, weight: *const u16, output: *mut u16, rows: u32, hidden: u32, epsilon: f32) -> c_int;
    pub fn atlas_hip_add_rms_norm_f16(ctx: *mut AtlasHipCtx, input: *const u16, residual: *const u16, weight: *const u16, residual_out: *mut u16, output: *mut u16, rows: u32, hidden: u32, epsilon: f32) -> c_int;
    pub fn atlas_hip_qk_norm_rope_f32(ctx: *mut AtlasHipCtx, q: *const f32, k: *const f32, q_weight: *const f32, k_weight: *const f32, cosine: *const f32, sine: *const f32, q_out: *mut f32, k_out: *mut f32, tokens: u32, q_heads: u32, has_key: u32, head_dim: u32, rope_stride: u32, epsilon: f32) -> c_int;
    pub fn atlas_hip_rope_half_f32(ctx: *mut AtlasHipCtx, input: *const f32, cosine: *const f32, sine: *const f32, output: *mut f32, tokens: u32, heads: u32, head_dim: u32, rope_stride: u32) -> c_int;
    pub fn atlas_hip_rope_half_f16(ctx: *mut AtlasHipCtx, input: *const u16, cosine: *const f32, sine: *const f32, output: *mut u16, tokens: u32, heads: u32, head_dim: u32, rope_stride: u32) -> c_int;
    pub fn atlas_hip_rope_half_qk_f32(ctx: *mut AtlasHipCtx, q: *const f32, k: *const f32, cosine: *const f32, sine: *const f32, q_out: *mut f32, k_out: *mut f32, tokens: u32, q_heads: u32, k_heads: u32, head_dim: u32, rope_stride: u32) -> c_int;
    pub fn atlas_hip_rope_half_qk_f16(ctx: *mut AtlasHipCtx, q: *const u16, k: *const u16, cosine: *const f32, sine: *const f32, q_out: *mut u16, k_out: *mut u16, tokens: u32, q_heads: u32, k_heads: u32, head_dim: u32, rope_stride: u32) -> c_int;
    pub fn atlas_hip_rope_interleaved_f32(ctx: *mut AtlasHipCtx, input: *const f32, cosine: *const f32, sine: *const f32, output: *mut f32, rows: u32, hidden: u32) -> c_int;
    pub fn atlas_rope_tables_gemma4(positions: *const u32, tokens: usize, rope_pairs: usize, rotary: usize, theta: f32, frequency_factors: *const f32, cos_out: *mut f32, sin_out: *mut f32) -> c_int;
    pub fn atlas_rope_tables_llama(positions: *const u32, tokens: usize, head_dim: usize, theta: f32, cos_out: *mut f32, sin_out: *mut f32) -> c_int;
    pub fn atlas_hip_swiglu_f32(ctx: *mut AtlasHipCtx, gate: *const f32, up: *const f32, output: *mut f32, count: u64) -> c_int;
    pub fn atlas_hip_swiglu_f16(ctx: *mut AtlasHipCtx, gate: *const u16, up: *const u16, output: *mut u16, count: u64) -> c_int;
    pub fn atlas_hip_geglu_f32(ctx: *mut AtlasHipCtx, gate: *const f32, up: *const f32, output: *mut f32, count: u64) -> c_int;
    pub fn atlas_hip_geglu_offset_f32(ctx: *mut AtlasHipCtx, gate: *const f32, ple: *const f32, output: *mut f32, ple_offset: u32, ple_row_stride: u32, width: u32, rows: u32) -> c_int;
    pub fn atlas_hip_silu_f32(ctx: *mut AtlasHipCtx, input: *const f32, output: *mut f32, count: u64) -> c_int;
    pub fn atlas_hip_gelu_f32(ctx: *mut AtlasHipCtx, input: *const f32, output: *mut f32, count: u64) -> c_int;
    pub fn atlas_hip_add_f32(ctx: *mut AtlasHipCtx, lhs: *const f32, rhs: *const f32, output: *mut f32, count: u64) -> c_int;
    pub fn atlas_hip_multiply_f32(ctx: *mut AtlasHipCtx, lhs: *const f32, rhs: *const f32, output: *mut f32, count: u64) -> c_int;
    pub fn atlas_hip_scale_f32(ctx: *mut AtlasHipCtx, input: *const f32, scalar: f32, output: *mut f32, count: u64) -> c_int;
    pub fn atlas_hip_embed_f32(ctx: *mut AtlasHipCtx, table: *const f32, ids: *const u32, output: *mut f32, vocab: u32, hidden: u32, tokens: u32, scale: f32) -> c_int;
    pub fn atlas_hip_embed_q4_0(ctx: *mut AtlasHipCtx, table: *const u8, ids: *const u32, output: *mut f32, vocab: u32, hidden: u32, tokens: u32, scale: f32) -> c_int;
    pub fn atlas_hip_embed_q6_k(ctx: *mut AtlasHipCtx, table: *const u8, ids: *const u32, output: *mut f32, vocab: u32, hidden: u32, tokens: u32, scale: f32) -> c_int;
    pub fn atlas_hip_embed_q8_0(ctx: *mut AtlasHipCtx, table: *const u8, ids: *const u32, output: *mut f32, vocab: u32, hidden: u32, tokens: u32, scale: f32) -> c_int;
    pub fn atlas_hip_ple_q4_0(ctx: *mut AtlasHipCtx, table: *const u8, ids: *const u32, projection: *const f32, output: *mut f32, vocab: u32, layers: u32, width: u32, tokens: u32, embedding_scale: f32, output_scale: f32) -> c_int;
    pub fn atlas_hip_ple_q6_k(ctx: *mut AtlasHipCtx, table: *const u8, ids: *const u32, projection: *const f32, output: *mut f32, vocab: u32, layers: u32, width: u32, tokens: u32, embedding_scale: f32, output_scale: f32) -> c_int;
    pub fn atlas_hip_matvec_q4_0_rms_f32(ctx: *mut AtlasHipCtx, input: *const f32, weights: *const u8, output: *mut f32, input_width: u32, output_width: u32, rms_weight: *const f32, epsilon: f32) -> c_int;
    pub fn atlas_hip_matmul_q4_0_qkv_rms_f32(ctx: *mut AtlasHipCtx, input: *const f32, q_weights: *const u8, k_weights: *const u8, v_weights: *const u8, q_output: *mut f32, k_output: *mut f32, v_output: *mut f32, input_width: u32, q_width: u32, kv_width: u32, rms_weight: *const f32, epsilon: f32) -> c_int;
    pub fn atlas_hip_matmul_q4_0_gate_up_rms_f32(ctx: *mut AtlasHipCtx, input: *const f32, gate_weights: *const u8, up_weights: *const u8, gate_output: *mut f32, up_output: *mut f32, input_width: u32, output_width: u32, rms_weight: *const f32, epsilon: f32) -> c_int;
    pub fn atlas_hip_ple_gate_gelu_f32(ctx: *mut AtlasHipCtx, input: *const f32, weights: *const u8, ple: *const f32, ple_offset: u32, output: *mut f32, input_width: u32, output_width: u32) -> c_int;
    pub fn atlas_hip_ple_projection_f16(ctx: *mut AtlasHipCtx, input: *const f32, weights: *const u16, norm_weight: *const f32, output: *mut f32, hidden: u32, width: u32, groups: u32, scale: f32, epsilon: f32) -> c_int;
    pub fn atlas_hip_kv_append_f32(ctx: *mut AtlasHipCtx, key: *const f32, value: *const f32, cache: *mut f32, kv_width: u32, capacity: u32, positions: *const u32, tokens: u32, vnorm: c_int, epsilon: f32) -> c_int;
    pub fn atlas_hip_kv_append_q8_0(ctx: *mut AtlasHipCtx, key: *const f32, value: *const f32, cache: *mut u8, kv_width: u32, capacity: u32, positions: *const u32, tokens: u32, vnorm: c_int, epsilon: f32) -> c_int;
    pub fn atlas_hip_kv_append_q4_0(ctx: *mut AtlasHipCtx, key: *const f32, value: *const f32, cache: *mut u8, kv_width: u32, capacity: u32, positions: *const u32, tokens: u32, vnorm: c_int, epsilon: f32) -> c_int;
    pub fn atlas_hip_prefix_attention_workspace(ctx: *mut AtlasHipCtx, format: c_int, sequences: u32, tokens: u32, q_heads: u32, kv_heads: u32, head_dim: u32, prefix_length: u32, capacity: u32, weights: c_int, bytes: *mut u64) -> c_int;
    pub fn atlas_hip_prefix_attention_f32(ctx: *mut AtlasHipCtx, q: *const f32, prefix: *const f32, prefix_length: u32, prefix_capacity: u32, cache: *const f32, lengths: *const u32, capacity: u32, output: *mut f32, weights_in: *const f32, weights_out: *mut f32, sequences: u32, tokens: u32, q_heads: u32, kv_heads: u32, head_dim: u32, scale: f32, workspace: *mut c_void, workspace_bytes: u64) -> c_int;
    pub fn atlas_hip_prefix_attention_q8_0(ctx: *mut AtlasHipCtx, q: *const f32, prefix: *const u8, prefix_length: u32, prefix_capacity: u32, cache: *const u8, lengths: *const u32, capacity: u32, output: *mut f32, weights_in: *const f32, weights_out: *mut f32, sequences: u32, tokens: u32, q_heads: u32, kv_heads: u32, head_dim: u32, scale: f32, workspace: *mut c_void, workspace_bytes: u64) -> c_int;
    pub fn atlas_hip_prefix_attention_q4_0(ctx: *mut AtlasHipCtx, q: *const f32, prefix: *const u8, prefix_length: u32, prefix_capacity: u32, cache: *const u8, lengths: *const u32, capacity: u32, output: *mut f32, weights_in: *const f32, weights_out: *mut f32, sequences: u32, tokens: u32, q_heads: u32, kv_heads: u32, head_dim: u32, scale: f32, workspace: *mut c_void, workspace_bytes: u64) -> c_int;
    pub fn atlas_hip_kv_evict_f32(ctx: *mut AtlasHipCtx, cache: *const f32, cache_out: *mut f32, weights: *const f32, weights_out: *mut f32, lengths: *const u32, lengths_out: *mut u32, kept: *mut u32, sequences: u32, capacity: u32, kv_width: u32, budget: u32, recent: u32) -> c_int;
    pub fn atlas_hip_kv_evict_q8_0(ctx: *mut AtlasHipCtx, cache: *const u8, cache_out: *mut u8, weights: *const f32, weights_out: *mut f32, lengths: *const u32, lengths_out: *mut u32, kept: *mut u32, sequences: u32, capacity: u32, kv_width: u32, budget: u32, recent: u32) -> c_int;
    pub fn atlas_hip_kv_evict_q4_0(ctx: *mut AtlasHipCtx, cache: *const u8, cache_out: *mut u8, weights: *const f32, weights_out: *mut f32, lengths: *const u32, lengths_out: *mut u32, kept: *mut u32, sequences: u32, capacity: u32, kv_width: u32, budget: u32, recent: u32) -> c_int;
    pub fn atlas_hip_softcap_f32(ctx: *mut AtlasHipCtx, input: *const f32, output: *mut f32, count: u64, cap: f32) -> c_int;
    pub fn atlas_hip_argmax_f32(ctx: *mut AtlasHipCtx, values: *const f32, selected: *mut u32, rows: u32, count: u32) -> c_int;
    pub fn atlas_hip_softcap_argmax_f32(ctx: *mut AtlasHipCtx, logits: *const f32, capped: *mut f32, selected: *mut u32, rows: u32, count: u32, cap: f32) -> c_int;
    pub fn atlas_hip_softcap_argmax_f32_noalloc(ctx: *mut AtlasHipCtx, logits: *const f32, capped: *mut f32, selected: *mut u32, rows: u32, count: u32, cap: f32) -> c_int;
    pub fn atlas_hip_verify_draft_workspace(ctx: *mut AtlasHipCtx, sequences: u32, drafts: u32, vocab: u32, bytes: *mut u64) -> c_int;
    pub fn atlas_hip_verify_draft_f32(ctx: *mut AtlasHipCtx, target_logits: *const f32, draft_logits: *const f32, draft_tokens: *const u32, draft_lengths: *const u32, accept_uniform: *const f32, sample_uniform: *const f32, accepted: *mut u32, tokens: *mut u32, sequences: u32, drafts: u32, vocab: u32, inv_temperature: f64, workspace: *mut c_void, workspace_bytes: u64) -> c_int;
    pub fn atlas_ops_embedding(ctx: *mut AtlasHipCtx, table: *const f32, table_len: usize, vocabulary: usize, hidden: usize, token_ids: *const u32, token_count: usize, output: *mut f32, output_len: usize, timing: *mut AtlasDispatchTiming) -> c_int;
    pub fn atlas_ops_embedding_q6_k(ctx: *mut AtlasHipCtx, weights: *const u8, weights_len: usize, vocabulary: usize, hidden: usize, token_ids: *const u32, token_count: usize, output: *mut f32, output_len: usize, timing: *mut AtlasDispatchTiming) -> c_int;
    pub fn atlas_ops_add(ctx: *mut AtlasHipCtx, lhs: *const f32, lhs_len: usize, rhs: *const f32, rhs_len: usize, output: *mut f32, output_len: usize, timing: *mut AtlasDispatchTiming) -> c_int;
    pub fn atlas_ops_multiply(ctx: *mut AtlasHipCtx, lhs: *const f32, lhs_len: usize, rhs: *const f32, rhs_len: usize, output: *mut f32, output_len: usize, timing: *mut AtlasDispatchTiming) -> c_int;
    pub fn atlas_ops_scalar_multiply(ctx: *mut AtlasHipCtx, input: *const f32, input_len: usize, scalar: f32, output: *mut f32, output_len: usize, timing: *mut AtlasDispatchTiming) -> c_int;
    pub fn atlas_ops_silu(ctx: *mut AtlasHipCtx, input: *const f32, input_len: usize, output: *mut f32, output_len: usize, timing: *mut AtlasDispatchTiming) -> c_int;
    pub fn atlas_ops_gelu(ctx: *mut AtlasHipCtx, input: *const f32, input_len: usize, output: *mut f32, output_len: usize, timing: *mut AtlasDispatchTiming) -> c_int;
    pub fn atlas_ops_rms_norm(ctx: *mut AtlasHipCtx, input: *const f32, input_len: usize, rows: usize, hidden: usize, weight: *const f32, weight_len: usize, epsilon: f32, output: *mut f32, output_len: usize, timing: *mut AtlasDispatchTiming) -> c_int;
    pub fn atlas_ops_rope(ctx: *mut AtlasHipCtx, input: *const f32, input_len: usize, rows: usize, hidden: usize, cosine: *const f32, cosine_len: usize, sine: *const f32, sine_len: usize, output: *mut f32, output_len: usize, timing: *mut AtlasDispatchTiming) -> c_int;
    // include/atlas_gguf.h
    pub fn atlas_gguf_open(path: *const c_char, out: *mut *mut AtlasGguf, error: *mut c_char, error_len: usize) -> c_int;
    pub fn atlas_gguf_from_bytes(data: *const c_void, bytes: usize, out: *mut *mut AtlasGguf, error: *mut c_char, error_len: usize) -> c_int;
    pub fn atlas_gguf_close(model: *mut AtlasGguf);
    pub fn atlas_gguf_tensor_count(model: *const AtlasGguf) -> u64;
    pub fn atlas_gguf_tensor_info(model: *const AtlasGguf, index: u64, out: *mut AtlasGgufTensor) -> c_int;
    pub fn atlas_gguf_find_tensor(model: *const AtlasGguf, name: *const c_char) -> i64;
    pub fn atlas_gguf_tensor_data(model: *const AtlasGguf, index: u64, data: *mut *const c_void, bytes: *mut u64) -> c_int;
    pub fn atlas_gguf_upload_tensor(ctx: *mut AtlasHipCtx, model: *const AtlasGguf, index: u64, device_dst: *mut c_void) -> c_int;
    pub fn atlas_gguf_metadata_count(model: *const AtlasGguf) -> u64;
    pub fn atlas_gguf_metadata_entry(model: *const AtlasGguf, index: u64, key: *mut *const c_char, key_len: *mut u64, value: *mut *const c_char, value_len: *mut u64) -> c_int;
    pub fn atlas_gguf_metadata_get(model: *const AtlasGguf, key: *const c_char) -> *const c_char;
    pub fn atlas_gguf_metadata_array_count(model: *const AtlasGguf) -> u64;
    pub fn atlas_gguf_metadata_array_entry(model: *const AtlasGguf, index: u64, key: *mut *const c_char, key_len: *mut u64, element_type: *mut u32, count: *mut u64, values: *mut *const c_void) -> c_int;
    pub fn atlas_gguf_metadata_array_string(model: *const AtlasGguf, index: u64, element: u64, text: *mut *const c_char, text_len: *mut u64) -> c_int;
    pub fn atlas_gguf_find_metadata_array(model: *const AtlasGguf, key: *const c_char) -> i64;
}
