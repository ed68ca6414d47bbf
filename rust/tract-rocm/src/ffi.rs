// Raw binding of include/tract_rocm.h.  GENERATED by include/gen_rust_ffi.py --write: do not edit by hand.
// Error convention (the reverse of api/ffi/src/lib.rs:18-62): every call returns 0 = OK or 1 = KO, and the
// message of the last KO on the calling thread is read with trocm_last_error().
#![allow(non_camel_case_types, clippy::too_many_arguments)]
use std::os::raw::{c_char, c_int, c_void};

#[repr(C)]
pub struct trocm_kivi_cache {
    _private: [u8; 0],
}
#[repr(C)]
pub struct trocm_kv_cache {
    _private: [u8; 0],
}
#[repr(C)]
pub struct trocm_kv_pool {
    _private: [u8; 0],
}
#[repr(C)]
pub struct trocm_q4_weights {
    _private: [u8; 0],
}

pub const TROCM_F32: c_int = 0;
pub const TROCM_F16: c_int = 1;
pub const TROCM_Q8_0: c_int = 2;
pub const TROCM_Q4_0: c_int = 3;
pub const TROCM_KIVI_PER_TOKEN: c_int = 0;
pub const TROCM_KIVI_BLOCK_CHANNEL: c_int = 1;
pub const TROCM_KIVI_RUNNING_CHANNEL: c_int = 2;
pub const TROCM_KIVI_PART_SINK: c_int = 0;
pub const TROCM_KIVI_PART_CODES: c_int = 1;
pub const TROCM_KIVI_PART_LO: c_int = 2;
pub const TROCM_KIVI_PART_SCALE: c_int = 3;
pub const TROCM_KIVI_PART_RESIDUAL: c_int = 4;

extern "C" {
    pub fn trocm_init(device: c_int) -> c_int;
    pub fn trocm_last_error() -> *const c_char;
    pub fn trocm_device_info(compute_units: *mut c_int, hbm_bytes: *mut usize, name: *mut c_char, name_len: usize) -> c_int;
    pub fn trocm_malloc(ptr: *mut *mut c_void, bytes: usize) -> c_int;
    pub fn trocm_free(ptr: *mut c_void) -> c_int;
    pub fn trocm_h2d(dst_device: *mut c_void, src_host: *const c_void, bytes: usize, stream: *mut c_void) -> c_int;
    pub fn trocm_d2h(dst_host: *mut c_void, src_device: *const c_void, bytes: usize, stream: *mut c_void) -> c_int;
    pub fn trocm_memset(dst_device: *mut c_void, byte_value: c_int, bytes: usize, stream: *mut c_void) -> c_int;
    pub fn trocm_stream_create(stream: *mut *mut c_void) -> c_int;
    pub fn trocm_stream_destroy(stream: *mut c_void) -> c_int;
    pub fn trocm_stream_sync(stream: *mut c_void) -> c_int;
    pub fn trocm_device_sync() -> c_int;
    pub fn trocm_event_create(event: *mut *mut c_void) -> c_int;
    pub fn trocm_event_destroy(event: *mut c_void) -> c_int;
    pub fn trocm_event_record(event: *mut c_void, stream: *mut c_void) -> c_int;
    pub fn trocm_event_elapsed_ms(start: *mut c_void, stop: *mut c_void, ms: *mut f32) -> c_int;
    pub fn trocm_copy_nd(dst: *mut c_void, dst_offset_bytes: usize, dst_strides: *const i64, src: *const c_void, src_offset_bytes: usize, src_strides: *const i64, shape: *const i64, rank: c_int, elem_size: c_int, stream: *mut c_void) -> c_int;
    pub fn trocm_kv_pool_create(out: *mut *mut trocm_kv_pool, bytes: usize) -> c_int;
    pub fn trocm_kv_pool_destroy(pool: *mut trocm_kv_pool) -> c_int;
    pub fn trocm_kv_pool_stats(pool: *mut trocm_kv_pool, bytes_total: *mut usize, bytes_in_use: *mut usize, largest_free: *mut usize, base: *mut *mut c_void) -> c_int;
    pub fn trocm_kv_cache_create(out: *mut *mut trocm_kv_cache, storage_format: c_int, batch: i64, kv_heads: i64, head_dim: i64) -> c_int;
    pub fn trocm_kv_cache_create_in_pool(out: *mut *mut trocm_kv_cache, pool: *mut trocm_kv_pool, storage_format: c_int, batch: i64, kv_heads: i64, head_dim: i64) -> c_int;
    pub fn trocm_kv_cache_create_window(out: *mut *mut trocm_kv_cache, storage_format: c_int, batch: i64, kv_heads: i64, head_dim: i64, window: i64) -> c_int;
    pub fn trocm_kv_cache_window(cache: *const trocm_kv_cache, window: *mut i64, cursor: *mut i64) -> c_int;
    pub fn trocm_kv_cache_destroy(cache: *mut trocm_kv_cache) -> c_int;
    pub fn trocm_kv_cache_len(cache: *const trocm_kv_cache, len: *mut i64) -> c_int;
    pub fn trocm_kv_cache_capacity(cache: *const trocm_kv_cache, capacity: *mut i64) -> c_int;
    pub fn trocm_kv_cache_reallocs(cache: *const trocm_kv_cache, reallocs: *mut i64) -> c_int;
    pub fn trocm_kv_cache_reserve(cache: *mut trocm_kv_cache, capacity: i64, stream: *mut c_void) -> c_int;
    pub fn trocm_kv_append(cache: *mut trocm_kv_cache, src: *const c_void, src_dtype: c_int, src_strides: *const i64, n_new: i64, stream: *mut c_void) -> c_int;
    pub fn trocm_kv_append_pair(k_cache: *mut trocm_kv_cache, v_cache: *mut trocm_kv_cache, k_src: *const c_void, v_src: *const c_void, src_dtype: c_int, src_strides: *const i64, n_new: i64, stream: *mut c_void) -> c_int;
    pub fn trocm_kv_cache_truncate(cache: *mut trocm_kv_cache, len: i64) -> c_int;
    pub fn trocm_kv_export(cache: *const trocm_kv_cache, dst_device: *mut c_void, stream: *mut c_void) -> c_int;
    pub fn trocm_kv_row_bytes(cache: *const trocm_kv_cache, bytes: *mut usize) -> c_int;
    pub fn trocm_kv_cache_clone(cache: *const trocm_kv_cache, out: *mut *mut trocm_kv_cache, stream: *mut c_void) -> c_int;
    pub fn trocm_kv_cache_raw(cache: *const trocm_kv_cache, data: *mut *mut c_void, scales: *mut *mut c_void, pitch: *mut i64) -> c_int;
    pub fn trocm_kv_import_blocks(cache: *mut trocm_kv_cache, blocks_device: *const c_void, n_tokens: i64, stream: *mut c_void) -> c_int;
    pub fn trocm_dat_header_write(dst128: *mut c_void, item: c_int, rank: c_int, dims: *const i64, data_bytes: usize) -> c_int;
    pub fn trocm_dat_header_read(src128: *const c_void, item: *mut c_int, rank: *mut c_int, dims8: *mut i64, data_bytes: *mut usize, flags: *mut c_int) -> c_int;
    pub fn trocm_dat_q4_0_legacy_to_gguf(blocks: *mut c_void, bytes: usize) -> c_int;
    pub fn trocm_q8_1_to_q8_0(src_36: *const c_void, dst_34: *mut c_void, n_blocks: usize) -> c_int;
    pub fn trocm_q8_0_to_q8_1(src_34: *const c_void, dst_36: *mut c_void, n_blocks: usize) -> c_int;
    pub fn trocm_block_quant(format: c_int, src: *const c_void, src_dtype: c_int, n_elems: usize, dst_blocks: *mut c_void, stream: *mut c_void) -> c_int;
    pub fn trocm_block_dequant(format: c_int, src_blocks: *const c_void, n_elems: usize, dst: *mut c_void, dst_dtype: c_int, stream: *mut c_void) -> c_int;
    pub fn trocm_block_simulate_precision_loss(format: c_int, src: *const c_void, dst: *mut c_void, dtype: c_int, n_elems: usize, stream: *mut c_void) -> c_int;
    pub fn trocm_q4_0_weights_create(out: *mut *mut trocm_q4_weights, blocks_device: *const c_void, batch: i64, n: i64, k: i64, stream: *mut c_void) -> c_int;
    pub fn trocm_q4_0_weights_destroy(weights: *mut trocm_q4_weights) -> c_int;
    pub fn trocm_q4_0_weights_shape(weights: *const trocm_q4_weights, batch: *mut i64, n: *mut i64, k: *mut i64) -> c_int;
    pub fn trocm_q4_0_weights_export(weights: *const trocm_q4_weights, dst_blocks_device: *mut c_void, stream: *mut c_void) -> c_int;
    pub fn trocm_q4_0_matvec(weights: *const trocm_q4_weights, act: *const c_void, act_dtype: c_int, act_batch: i64, m: i64, out: *mut c_void, stream: *mut c_void) -> c_int;
    pub fn trocm_release_unused(wait: c_int) -> c_int;
    pub fn trocm_launch_floor(kind: c_int, src: *const c_void, bytes: usize, workgroups: c_int, threads: c_int, sink: *mut c_void, stream: *mut c_void) -> c_int;
    pub fn trocm_cast(src: *const c_void, src_dtype: c_int, dst: *mut c_void, dst_dtype: c_int, n_elems: usize, stream: *mut c_void) -> c_int;
    pub fn trocm_apply_rope(input: *const c_void, cos: *const c_void, sin: *const c_void, out: *mut c_void, dtype: c_int, rank: c_int, shape: *const i64, in_strides: *const i64, cos_sin_strides: *const i64, out_strides: *const i64, stream: *mut c_void) -> c_int;
    pub fn trocm_rotate_half(input: *const c_void, out: *mut c_void, dtype: c_int, rank: c_int, shape: *const i64, in_strides: *const i64, out_strides: *const i64, stream: *mut c_void) -> c_int;
    pub fn trocm_sdpa_workspace_bytes(batch: i64, q_heads: i64, q_len: i64, head_dim: i64, bytes: *mut usize) -> c_int;
    pub fn trocm_sdpa_workspace_init(workspace: *mut c_void, bytes: usize, stream: *mut c_void) -> c_int;
    pub fn trocm_sdpa(q: *const c_void, k: *const c_void, v: *const c_void, mask: *const c_void, out: *mut c_void, dtype: c_int, batch: i64, q_heads: i64, kv_heads: i64, q_len: i64, kv_len: i64, head_dim: i64, kv_strides: *const i64, mask_batch: i64, mask_heads: i64, scale: f32, causal: c_int, workspace: *mut c_void, workspace_bytes: usize, stream: *mut c_void) -> c_int;
    pub fn trocm_sdpa_cached(q: *const c_void, q_dtype: c_int, q_heads: i64, q_len: i64, k_cache: *const trocm_kv_cache, v_cache: *const trocm_kv_cache, out: *mut c_void, scale: f32, causal: c_int, workspace: *mut c_void, workspace_bytes: usize, stream: *mut c_void) -> c_int;
    pub fn trocm_sdpa_cached_noalloc(q: *const c_void, q_dtype: c_int, q_heads: i64, q_len: i64, k_cache: *const trocm_kv_cache, v_cache: *const trocm_kv_cache, out: *mut c_void, scale: f32, causal: c_int, stream: *mut c_void) -> c_int;
    pub fn trocm_inplace_kv_sdpa_eval(q: *const c_void, k_new: *const c_void, v_new: *const c_void, dtype: c_int, q_heads: i64, n_new: i64, kv_new_strides: *const i64, k_cache: *mut trocm_kv_cache, v_cache: *mut trocm_kv_cache, out: *mut c_void, scale: f32, causal: c_int, workspace: *mut c_void, workspace_bytes: usize, stream: *mut c_void) -> c_int;
    pub fn trocm_inplace_kv_sdpa_eval_rope(q: *const c_void, k_new: *const c_void, v_new: *const c_void, cos: *const c_void, sin: *const c_void, cos_sin_batch_stride: i64, dtype: c_int, q_heads: i64, n_new: i64, k_cache: *mut trocm_kv_cache, v_cache: *mut trocm_kv_cache, out: *mut c_void, scale: f32, causal: c_int, workspace: *mut c_void, workspace_bytes: usize, rot_scratch: *mut c_void, rot_scratch_bytes: usize, stream: *mut c_void) -> c_int;
    pub fn trocm_window_kv_sdpa_eval(q: *const c_void, k_new: *const c_void, v_new: *const c_void, dtype: c_int, q_heads: i64, n_new: i64, kv_new_strides: *const i64, k_cache: *mut trocm_kv_cache, v_cache: *mut trocm_kv_cache, out: *mut c_void, scale: f32, workspace: *mut c_void, workspace_bytes: usize, stream: *mut c_void) -> c_int;
    pub fn trocm_sdpa_decode_ragged(q: *const c_void, q_dtype: c_int, q_heads: i64, n_seq: i64, k_caches: *const *mut trocm_kv_cache, v_caches: *const *mut trocm_kv_cache, out: *mut c_void, scale: f32, workspace: *mut c_void, workspace_bytes: usize, stream: *mut c_void) -> c_int;
    pub fn trocm_inplace_kv_sdpa_eval_ragged(q: *const c_void, k_new: *const c_void, v_new: *const c_void, dtype: c_int, q_heads: i64, n_seq: i64, k_caches: *const *mut trocm_kv_cache, v_caches: *const *mut trocm_kv_cache, out: *mut c_void, scale: f32, workspace: *mut c_void, workspace_bytes: usize, stream: *mut c_void) -> c_int;
    pub fn trocm_inplace_kv_sdpa_eval_ragged_rope(q: *const c_void, k_new: *const c_void, v_new: *const c_void, cos: *const c_void, sin: *const c_void, dtype: c_int, q_heads: i64, n_seq: i64, k_caches: *const *mut trocm_kv_cache, v_caches: *const *mut trocm_kv_cache, out: *mut c_void, scale: f32, workspace: *mut c_void, workspace_bytes: usize, rot_scratch: *mut c_void, rot_scratch_bytes: usize, stream: *mut c_void) -> c_int;
    pub fn trocm_kivi_cache_create(out: *mut *mut trocm_kivi_cache, layout: c_int, bits: c_int, sink_tokens: i64, batch: i64, heads: i64, head_dim: i64) -> c_int;
    pub fn trocm_kivi_cache_destroy(cache: *mut trocm_kivi_cache) -> c_int;
    pub fn trocm_kivi_cache_reset(cache: *mut trocm_kivi_cache, stream: *mut c_void) -> c_int;
    pub fn trocm_kivi_cache_len(cache: *const trocm_kivi_cache, len: *mut i64) -> c_int;
    pub fn trocm_kivi_cache_counts(cache: *const trocm_kivi_cache, n_sink: *mut i64, n_rows: *mut i64, n_res: *mut i64, row_bytes: *mut i64) -> c_int;
    pub fn trocm_kivi_cache_memory_bytes(cache: *const trocm_kivi_cache, bytes: *mut usize) -> c_int;
    pub fn trocm_kivi_cache_append(cache: *mut trocm_kivi_cache, src: *const c_void, src_dtype: c_int, n_new: i64, stream: *mut c_void) -> c_int;
    pub fn trocm_kivi_cache_dequantize(cache: *const trocm_kivi_cache, dst: *mut c_void, dst_dtype: c_int, stream: *mut c_void) -> c_int;
    pub fn trocm_kivi_cache_export(cache: *const trocm_kivi_cache, part: c_int, dst_device: *mut c_void, bytes: *mut usize, stream: *mut c_void) -> c_int;
    pub fn trocm_kivi_cache_clone(cache: *const trocm_kivi_cache, out: *mut *mut trocm_kivi_cache, stream: *mut c_void) -> c_int;
    pub fn trocm_quantized_kv_sdpa_eval(q: *const c_void, k_new: *const c_void, v_new: *const c_void, dtype: c_int, q_heads: i64, n_new: i64, k_cache: *mut trocm_kivi_cache, v_cache: *mut trocm_kivi_cache, out: *mut c_void, scale: f32, workspace: *mut c_void, workspace_bytes: usize, stream: *mut c_void) -> c_int;
    pub fn trocm_qk_norm_rope(q: *const c_void, k: *const c_void, q_weight: *const c_void, k_weight: *const c_void, eps: f32, cos: *const c_void, sin: *const c_void, cos_sin_batch_stride: i64, dtype: c_int, batch: i64, q_heads: i64, kv_heads: i64, n: i64, head_dim: i64, q_strides: *const i64, k_strides: *const i64, q_out: *mut c_void, k_out: *mut c_void, stream: *mut c_void) -> c_int;
    pub fn trocm_inplace_kv_sdpa_eval_norm_rope(q: *const c_void, k_new: *const c_void, v_new: *const c_void, q_weight: *const c_void, k_weight: *const c_void, eps: f32, cos: *const c_void, sin: *const c_void, cos_sin_batch_stride: i64, dtype: c_int, q_heads: i64, n_new: i64, q_strides: *const i64, k_strides: *const i64, v_strides: *const i64, k_cache: *mut trocm_kv_cache, v_cache: *mut trocm_kv_cache, out: *mut c_void, scale: f32, causal: c_int, workspace: *mut c_void, workspace_bytes: usize, rot_scratch: *mut c_void, rot_scratch_bytes: usize, stream: *mut c_void) -> c_int;
    pub fn trocm_sdpa_shared_workspace_bytes(n_seq: i64, q_heads: i64, q_len: i64, head_dim: i64, bytes: *mut usize) -> c_int;
    pub fn trocm_sdpa_shared_prefix(q: *const c_void, dtype: c_int, n_seq: i64, q_heads: i64, kv_heads: i64, q_len: i64, head_dim: i64, prefix_k: *const c_void, prefix_v: *const c_void, prefix_len: i64, prefix_strides: *const i64, k: *const c_void, v: *const c_void, kv_strides: *const i64, lens: *const i64, out: *mut c_void, scale: f32, causal: c_int, workspace: *mut c_void, workspace_bytes: usize, stream: *mut c_void) -> c_int;
    pub fn trocm_inplace_kv_sdpa_eval_shared(q: *const c_void, k_new: *const c_void, v_new: *const c_void, dtype: c_int, q_heads: i64, n_seq: i64, n_new: i64, prefix_k_cache: *const trocm_kv_cache, prefix_v_cache: *const trocm_kv_cache, k_caches: *const *mut trocm_kv_cache, v_caches: *const *mut trocm_kv_cache, out: *mut c_void, scale: f32, causal: c_int, workspace: *mut c_void, workspace_bytes: usize, stream: *mut c_void) -> c_int;
    pub fn trocm_sdpa_scored(q: *const c_void, k: *const c_void, v: *const c_void, out: *mut c_void, dtype: c_int, batch: i64, q_heads: i64, kv_heads: i64, q_len: i64, kv_len: i64, head_dim: i64, kv_strides: *const i64, scale: f32, softcap: f32, slopes: *const f32, documents: *const i32, prefix_lens: *const i32, causal: c_int, workspace: *mut c_void, workspace_bytes: usize, stream: *mut c_void) -> c_int;
    pub fn trocm_sdpa_cached_scored(q: *const c_void, q_dtype: c_int, q_heads: i64, q_len: i64, k_cache: *const trocm_kv_cache, v_cache: *const trocm_kv_cache, out: *mut c_void, scale: f32, softcap: f32, slopes: *const f32, documents: *const i32, prefix_lens: *const i32, causal: c_int, workspace: *mut c_void, workspace_bytes: usize, stream: *mut c_void) -> c_int;
}

/// KO -> an error that carries the library's message.
pub fn check(rc: c_int) -> tract_core::internal::TractResult<()> {
    if rc == 0 {
        return Ok(());
    }
    let msg = unsafe { std::ffi::CStr::from_ptr(trocm_last_error()) }.to_string_lossy().into_owned();
    tract_core::internal::bail!("tract-rocm: {msg}")
}
