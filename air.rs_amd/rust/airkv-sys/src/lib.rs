// Generated by air.rs_amd/rust/gen_sys.py from include/air_kv.h -- do not edit.
//
// Raw bindings of libairkv.so, the C ABI of the MI355X paged KV-cache path.
// This crate is source for Air.rs maintainers; it is not compiled in this
// repository (no Rust toolchain here).  See the safe wrapper in ../airkv.
#![allow(non_camel_case_types, non_upper_case_globals, clippy::all)]

use core::ffi::{c_char, c_int, c_void};

pub const AIR_KV_OK: c_int = 0;
pub const AIR_KV_E_INVALID_ARG: c_int = -1;
pub const AIR_KV_E_OOM: c_int = -2;
pub const AIR_KV_E_NOT_FOUND: c_int = -3;
pub const AIR_KV_E_HIP: c_int = -4;
pub const AIR_KV_E_STATE: c_int = -5;
pub const AIR_KV_F32: c_int = 0;
pub const AIR_KV_BF16: c_int = 1;
pub const AIR_KV_INT8: c_int = 2;
pub const AIR_KV_FP8: c_int = 3;
pub const AIR_KV_LAYOUT_HEAD_MAJOR: c_int = 0;
pub const AIR_KV_LAYOUT_TOKEN_MAJOR: c_int = 1;
pub const AIR_KV_NOALLOC_SCRATCH_BYTES: usize = 32 << 20;

#[repr(C)]
pub struct air_block_allocator {
    _private: [u8; 0],
}

#[repr(C)]
pub struct air_kv_pool {
    _private: [u8; 0],
}

#[repr(C)]
pub struct air_kv_session {
    _private: [u8; 0],
}

#[repr(C)]
pub struct air_kv_swap {
    _private: [u8; 0],
}

#[repr(C)]
pub struct air_seq_manager {
    _private: [u8; 0],
}

#[repr(C)]
#[derive(Clone, Copy, Debug, Default)]
pub struct air_kv_pool_desc {
    pub num_blocks: i64,
    pub block_size: i32,
    pub n_kv_heads: i32,
    pub head_dim: i32,
    pub dtype: i32,
    pub scale_group: i32,
}

pub type air_kv_block_read_fn = Option<unsafe extern "C" fn(*mut c_void, u32, *mut u8, usize) -> c_int>;
pub type air_kv_block_write_fn = Option<unsafe extern "C" fn(*mut c_void, u32, *const u8, usize) -> c_int>;

#[link(name = "airkv")]
extern "C" {
    pub fn air_kv_last_error(buf: *mut c_char, cap: usize) -> c_int;
    pub fn air_block_allocator_create(capacity: i64, block_size: i32, free_order: *const u32, out: *mut *mut air_block_allocator) -> c_int;
    pub fn air_block_allocator_destroy(a: *mut air_block_allocator) -> c_int;
    pub fn air_block_allocator_allocate(a: *mut air_block_allocator, block: *mut u32) -> c_int;
    pub fn air_block_allocator_share(a: *mut air_block_allocator, block: u32) -> c_int;
    pub fn air_block_allocator_release(a: *mut air_block_allocator, block: u32) -> c_int;
    pub fn air_block_allocator_ref_count(a: *const air_block_allocator, block: u32, rc: *mut u32) -> c_int;
    pub fn air_block_allocator_num_free(a: *const air_block_allocator) -> i64;
    pub fn air_block_allocator_num_used(a: *const air_block_allocator) -> i64;
    pub fn air_block_allocator_cow_write(a: *mut air_block_allocator, block: u32, out: *mut u32) -> c_int;
    pub fn air_block_allocator_append_token(a: *mut air_block_allocator, block: u32, is_full: *mut i32) -> c_int;
    pub fn air_block_allocator_block_info(a: *const air_block_allocator, block: u32, num_tokens: *mut i32, is_full: *mut i32) -> c_int;
    pub fn air_block_allocator_can_allocate(a: *const air_block_allocator, n: i64) -> c_int;
    pub fn air_block_allocator_utilization(a: *const air_block_allocator) -> f32;
    pub fn air_num_blocks_for_tokens(n_tokens: i64, block_size: i32) -> i64;
    pub fn air_seq_manager_create(capacity: i64, block_size: i32, free_order: *const u32, out: *mut *mut air_seq_manager) -> c_int;
    pub fn air_seq_manager_destroy(m: *mut air_seq_manager) -> c_int;
    pub fn air_seq_manager_allocator(m: *mut air_seq_manager) -> *mut air_block_allocator;
    pub fn air_seq_create(m: *mut air_seq_manager, seq: *mut u32) -> c_int;
    pub fn air_seq_append_token(m: *mut air_seq_manager, seq: u32, block: *mut u32) -> c_int;
    pub fn air_seq_append_slots(m: *mut air_seq_manager, seq: u32, n: i32, slots: *mut i64, n_done: *mut i32) -> c_int;
    pub fn air_seq_fork(m: *mut air_seq_manager, parent: u32, child: *mut u32) -> c_int;
    pub fn air_seq_free(m: *mut air_seq_manager, seq: u32) -> c_int;
    pub fn air_seq_cow_last_block(m: *mut air_seq_manager, seq: u32, old_block: *mut u32, new_block: *mut u32) -> c_int;
    pub fn air_seq_truncate(m: *mut air_seq_manager, seq: u32, n_tokens: i64) -> c_int;
    pub fn air_seq_cow_block(m: *mut air_seq_manager, seq: u32, index: i64, old_block: *mut u32, new_block: *mut u32) -> c_int;
    pub fn air_seq_table(m: *const air_seq_manager, seq: u32, blocks: *mut u32, cap: i32, n_blocks: *mut i32, n_tokens: *mut i64) -> c_int;
    pub fn air_seq_export_tables(m: *const air_seq_manager, seqs: *const u32, n: i32, max_blocks: i32, tables: *mut i32, seq_lens: *mut i32) -> c_int;
    pub fn air_seq_num_sequences(m: *const air_seq_manager) -> i64;
    pub fn air_seq_can_schedule(m: *const air_seq_manager) -> c_int;
    pub fn air_seq_swap_out(m: *mut air_seq_manager, seq: u32, blocks: *mut u32, cap: i32, n_blocks: *mut i32) -> c_int;
    pub fn air_seq_swap_in(m: *mut air_seq_manager, seq: u32, n_blocks: i32, blocks: *mut u32) -> c_int;
    pub fn air_kv_swap_create(capacity: i64, block_size: i32, block_bytes: usize, out: *mut *mut air_kv_swap) -> c_int;
    pub fn air_kv_swap_destroy(s: *mut air_kv_swap) -> c_int;
    pub fn air_kv_swap_seq_manager(s: *mut air_kv_swap) -> *mut air_seq_manager;
    pub fn air_kv_swap_evict(s: *mut air_kv_swap, seq: u32, read: air_kv_block_read_fn, ctx: *mut c_void, released: *mut u32, cap: i32, n_released: *mut i32) -> c_int;
    pub fn air_kv_swap_restore(s: *mut air_kv_swap, seq: u32, write: air_kv_block_write_fn, ctx: *mut c_void, blocks: *mut u32, cap: i32, n_blocks: *mut i32) -> c_int;
    pub fn air_kv_swap_is_evicted(s: *const air_kv_swap, seq: u32) -> c_int;
    pub fn air_kv_swap_evicted_count(s: *const air_kv_swap) -> i64;
    pub fn air_kv_swap_cpu_bytes_used(s: *const air_kv_swap) -> i64;
    pub fn air_kv_swap_maybe_evict(s: *mut air_kv_swap, seq: u32, free_threshold: i64, read: air_kv_block_read_fn, ctx: *mut c_void, evicted: *mut i32) -> c_int;
    pub fn air_kv_pool_create(desc: *const air_kv_pool_desc, out: *mut *mut air_kv_pool) -> c_int;
    pub fn air_kv_pool_destroy(pool: *mut air_kv_pool) -> c_int;
    pub fn air_kv_pool_info(pool: *const air_kv_pool, desc: *mut air_kv_pool_desc, k_pages: *mut *mut c_void, v_pages: *mut *mut c_void, k_scales: *mut *mut c_void, v_scales: *mut *mut c_void, block_bytes: *mut usize) -> c_int;
    pub fn air_kv_append(pool: *mut air_kv_pool, stream: *mut c_void, k: *const f32, v: *const f32, slot_mapping: *const i64, n_tokens: i32) -> c_int;
    pub fn air_kv_gather(pool: *mut air_kv_pool, stream: *mut c_void, block_tables: *const i32, seq_lens: *const i32, out_offsets: *const i64, batch: i32, max_blocks: i32, out_k: *mut c_void, out_v: *mut c_void, out_dtype: i32, out_layout: i32) -> c_int;
    pub fn air_paged_decode_workspace_size(pool: *const air_kv_pool, n_q_heads: i32, batch: i32, max_blocks: i32, max_splits: i32, bytes: *mut usize) -> c_int;
    pub fn air_paged_decode(pool: *mut air_kv_pool, stream: *mut c_void, q: *const c_void, q_dtype: i32, n_q_heads: i32, block_tables: *const i32, seq_lens: *const i32, batch: i32, max_blocks: i32, scale: f32, max_splits: i32, workspace: *mut c_void, ws_bytes: usize, out: *mut c_void, out_dtype: i32) -> c_int;
    pub fn air_paged_decode_append(pool: *mut air_kv_pool, stream: *mut c_void, q: *const c_void, q_dtype: i32, n_q_heads: i32, k_new: *const f32, v_new: *const f32, block_tables: *const i32, seq_lens: *const i32, batch: i32, max_blocks: i32, scale: f32, max_splits: i32, workspace: *mut c_void, ws_bytes: usize, out: *mut c_void, out_dtype: i32) -> c_int;
    pub fn air_paged_decode_noalloc(pool: *mut air_kv_pool, stream: *mut c_void, q: *const c_void, q_dtype: i32, n_q_heads: i32, block_tables: *const i32, seq_lens: *const i32, batch: i32, max_blocks: i32, scale: f32, max_splits: i32, out: *mut c_void, out_dtype: i32) -> c_int;
    pub fn air_paged_prefill(pool: *mut air_kv_pool, stream: *mut c_void, q: *const c_void, q_dtype: i32, n_q_heads: i32, cu_q: *const i32, total_q: i32, max_q_len: i32, block_tables: *const i32, seq_lens: *const i32, batch: i32, max_blocks: i32, scale: f32, workspace: *mut c_void, ws_bytes: usize, out: *mut c_void, out_dtype: i32) -> c_int;
    pub fn air_paged_prefill_workspace_size(pool: *const air_kv_pool, n_q_heads: i32, batch: i32, max_q_len: i32, bytes: *mut usize) -> c_int;
    pub fn air_paged_diff_decode_workspace_size(pool: *const air_kv_pool, n_q_heads: i32, batch: i32, max_blocks: i32, max_splits: i32, bytes: *mut usize) -> c_int;
    pub fn air_paged_diff_decode(pool: *mut air_kv_pool, stream: *mut c_void, q: *const c_void, q_dtype: i32, n_q_heads: i32, lambda: *const f32, lambda_per_row: i32, block_tables: *const i32, seq_lens: *const i32, batch: i32, max_blocks: i32, scale: f32, max_splits: i32, norm_weight: *const f32, norm_eps: f32, out_scale: f32, workspace: *mut c_void, ws_bytes: usize, out: *mut c_void, out_dtype: i32) -> c_int;
    pub fn air_paged_diff_prefill_workspace_size(pool: *const air_kv_pool, n_q_heads: i32, batch: i32, max_q_len: i32, bytes: *mut usize) -> c_int;
    pub fn air_paged_diff_prefill(pool: *mut air_kv_pool, stream: *mut c_void, q: *const c_void, q_dtype: i32, n_q_heads: i32, lambda: *const f32, lambda_per_row: i32, cu_q: *const i32, total_q: i32, max_q_len: i32, block_tables: *const i32, seq_lens: *const i32, batch: i32, max_blocks: i32, scale: f32, norm_weight: *const f32, norm_eps: f32, out_scale: f32, workspace: *mut c_void, ws_bytes: usize, out: *mut c_void, out_dtype: i32) -> c_int;
    pub fn air_kv_session_create(mgr: *mut air_seq_manager, layer_pools: *const *mut air_kv_pool, n_layers: i32, out: *mut *mut air_kv_session) -> c_int;
    pub fn air_kv_session_destroy(s: *mut air_kv_session) -> c_int;
    pub fn air_kv_session_fork(parent: *mut air_kv_session, out: *mut *mut air_kv_session) -> c_int;
    pub fn air_kv_session_seq_id(s: *const air_kv_session, seq: *mut u32) -> c_int;
    pub fn air_kv_session_seq_len(s: *const air_kv_session, layer: i32, len: *mut i64) -> c_int;
    pub fn air_kv_session_append(s: *mut air_kv_session, stream: *mut c_void, layer: i32, k: *const f32, v: *const f32, n_new: i64) -> c_int;
    pub fn air_kv_session_save(s: *mut air_kv_session, stream: *mut c_void, layer: i32, k: *const f32, v: *const f32, n_tokens: i64) -> c_int;
    pub fn air_kv_session_load(s: *mut air_kv_session, stream: *mut c_void, layer: i32, out_k: *mut c_void, out_v: *mut c_void, out_dtype: i32) -> c_int;
    pub fn air_kv_session_clear(s: *mut air_kv_session) -> c_int;
    pub fn air_kv_session_truncate_to(s: *mut air_kv_session, pos: i64) -> c_int;
    pub fn air_kv_session_compact(s: *mut air_kv_session, stream: *mut c_void, keep: *const i64, n_keep: i64) -> c_int;
    pub fn air_kv_session_memory_usage(s: *const air_kv_session, bytes: *mut usize) -> c_int;
    pub fn air_kv_block_wire_bytes(pool: *const air_kv_pool, bytes: *mut usize) -> c_int;
    pub fn air_kv_pack_blocks(pool: *mut air_kv_pool, stream: *mut c_void, ids: *const i32, n: i32, out: *mut c_void) -> c_int;
    pub fn air_kv_unpack_blocks(pool: *mut air_kv_pool, stream: *mut c_void, ids: *const i32, n: i32, in_: *const c_void) -> c_int;
    pub fn air_kv_wire_int8_quantize(stream: *mut c_void, wire: *const c_void, n_blocks: i32, elems_per_block: usize, codes: *mut i8, scales: *mut f32) -> c_int;
    pub fn air_kv_pack_blocks_int8(pool: *mut air_kv_pool, stream: *mut c_void, ids: *const i32, n: i32, codes: *mut i8, scales: *mut f32) -> c_int;
    pub fn air_kv_block_frame_bytes(data_len: usize) -> usize;
    pub fn air_kv_block_serialise(block_id: u32, layer_idx: u16, data: *const c_void, data_len: usize, out: *mut c_void, cap: usize, written: *mut usize) -> c_int;
    pub fn air_kv_block_deserialise(buf: *const c_void, len: usize, block_id: *mut u32, layer_idx: *mut u16, data: *mut *const c_void, data_len: *mut usize) -> c_int;
    pub fn air_kv_block_serialise_n(block_ids: *const u32, layer_idx: u16, data: *const c_void, block_bytes: usize, n: i32, out: *mut c_void) -> c_int;
    pub fn air_kv_int8_payload_bytes(n_codes: usize) -> usize;
    pub fn air_kv_int8_payload_serialise(block_id: u32, layer_idx: u16, scale: f32, codes: *const i8, n_codes: usize, out: *mut c_void, cap: usize, written: *mut usize) -> c_int;
    pub fn air_kv_int8_payload_deserialise(buf: *const c_void, len: usize, block_id: *mut u32, layer_idx: *mut u16, scale: *mut f32, codes: *mut *const i8, n_codes: *mut usize) -> c_int;
    pub fn air_kv_int8_payload_serialise_n(block_ids: *const u32, layer_idx: u16, scales: *const f32, codes: *const i8, codes_per_block: usize, n: i32, out: *mut c_void) -> c_int;
    pub fn air_kv_key_compress(stream: *mut c_void, rows: *const c_void, rows_dtype: i32, n_rows: i64, dim: i32, bits: *mut u64, magnitude: *mut f32, mean: *mut f32) -> c_int;
    pub fn air_kv_key_decompress(stream: *mut c_void, bits: *const u64, magnitude: *const f32, mean: *const f32, n_rows: i64, dim: i32, out: *mut f32) -> c_int;
    pub fn air_kv_value_compress(stream: *mut c_void, rows: *const c_void, rows_dtype: i32, n_rows: i64, dim: i32, codes: *mut u8, scale: *mut f32, min_val: *mut f32) -> c_int;
    pub fn air_kv_value_decompress(stream: *mut c_void, codes: *const u8, scale: *const f32, min_val: *const f32, n_rows: i64, dim: i32, out: *mut f32) -> c_int;
    pub fn air_kv_qjl_compress(stream: *mut c_void, rows: *const c_void, rows_dtype: i32, n_rows: i64, dim: i32, proj: *const f32, proj_dim: i32, bits: *mut u64, magnitude: *mut f32) -> c_int;
    pub fn air_kv_qjl_scores(stream: *mut c_void, key_bits: *const u64, key_magnitude: *const f32, n_keys: i64, proj_dim: i32, query_bits: *const u64, query_magnitude: f32, cos_sim: *mut f32, dot: *mut f32) -> c_int;
    pub fn air_kv_compress_blocks(pool: *mut air_kv_pool, stream: *mut c_void, ids: *const i32, n: i32, key_bits: *mut u64, key_magnitude: *mut f32, key_mean: *mut f32, value_codes: *mut u8, value_scale: *mut f32, value_min: *mut f32) -> c_int;
    pub fn air_kv_qjl_compress_blocks(pool: *mut air_kv_pool, stream: *mut c_void, ids: *const i32, n: i32, proj: *const f32, proj_dim: i32, bits: *mut u64, magnitude: *mut f32) -> c_int;
    pub fn air_kv_copy_blocks(pool: *mut air_kv_pool, stream: *mut c_void, src_blocks: *const i32, dst_blocks: *const i32, n: i32) -> c_int;
    pub fn air_kv_compact(pool: *mut air_kv_pool, stream: *mut c_void, block_tables: *const i32, seq_lens: *const i32, batch: i32, max_blocks: i32, keep: *const i32, cu_keep: *const i32, total_keep: i32) -> c_int;
    pub fn air_kv_read_blocks(pool: *mut air_kv_pool, stream: *mut c_void, ids: *const i32, n: i32, host_dst: *mut c_void) -> c_int;
    pub fn air_kv_write_blocks(pool: *mut air_kv_pool, stream: *mut c_void, ids: *const i32, n: i32, host_src: *const c_void) -> c_int;
    pub fn air_kv_pool_read_cb(ctx: *mut c_void, block: u32, dst: *mut u8, bytes: usize) -> c_int;
    pub fn air_kv_pool_write_cb(ctx: *mut c_void, block: u32, src: *const u8, bytes: usize) -> c_int;
    pub fn air_kv_pool_error_count(pool: *mut air_kv_pool, stream: *mut c_void, count: *mut i64, reset: i32) -> c_int;
}
