//! Raw FFI declarations of libhearth_b200.so (include/hb200.h): the B200 implementation of Hearth's quantized
//! matrix-product path.  Generated by bindings/generate.py from the header; do not edit by hand.
#![allow(non_camel_case_types)]

use core::ffi::{c_char, c_int, c_void};

#[repr(C)]
pub struct hb200_weight {
    _private: [u8; 0],
}
#[repr(C)]
pub struct hb200_act {
    _private: [u8; 0],
}
#[repr(C)]
pub struct hb200_batch {
    _private: [u8; 0],
}
#[repr(C)]
pub struct hb200_gguf {
    _private: [u8; 0],
}
#[repr(C)]
pub struct hb200_weight_i8 {
    _private: [u8; 0],
}
#[repr(C)]
pub struct hb200_act_i8 {
    _private: [u8; 0],
}

pub const HB200_OK: c_int = 0;
pub const HB200_ERR_NOT_INITIALIZED: c_int = -1;
pub const HB200_ERR_NO_DEVICE: c_int = -2;
pub const HB200_ERR_BAD_DTYPE: c_int = -3;
pub const HB200_ERR_BAD_SHAPE: c_int = -4;
pub const HB200_ERR_NULL: c_int = -5;
pub const HB200_ERR_CUDA: c_int = -6;
pub const HB200_ERR_UNSUPPORTED: c_int = -7;
pub const HB200_ERR_TOO_LARGE: c_int = -8;
pub const HB200_ERR_TIMEOUT: c_int = -9;
pub const HB200_ERR_IO: c_int = -10;
pub const HB200_ERR_BAD_FORMAT: c_int = -11;
pub const HB200_ERR_NOT_FOUND: c_int = -12;
pub const HB200_Q8_0: c_int = 8;
pub const HB200_Q4_K: c_int = 12;
pub const HB200_Q6_K: c_int = 14;
pub const HB200_Q1_0_G128_LEGACY: c_int = 39;
pub const HB200_Q1_0: c_int = 41;
pub const HB200_Q2_0: c_int = 42;
pub const HB200_Q1_0_G128: c_int = 43;
pub const HB200_PQ2_0: c_int = 142;
pub const HB200_PTQ1_0: c_int = 143;
pub const HB200_MAX_SEQ_LEN: usize = 65535;
pub const HB200_NOALLOC_MAX_TOKENS: usize = 4;
pub const HB200_NOALLOC_MAX_COLS: usize = 32768;
pub const HB200_I8_MAX_COLS: usize = 65536;
pub const HB200_I8_MAX_ROWS: usize = 8388480;
pub const HB200_PEER_HANDLE_BYTES: usize = 64;
pub const HB200_MAX_PEERS: usize = 8;

#[link(name = "hearth_b200")]
extern "C" {
    pub fn hb200_init(device: c_int) -> c_int;
    pub fn hb200_init_multi(n_devices: c_int) -> c_int;
    pub fn hb200_init_slots(devices: *const c_int, n_slots: c_int) -> c_int;
    pub fn hb200_set_slot(slot: c_int) -> c_int;
    pub fn hb200_slot_count() -> c_int;
    pub fn hb200_shutdown() -> c_int;
    pub fn hb200_last_error() -> *const c_char;
    pub fn hb200_sm_count() -> c_int;
    pub fn hb200_measure_i8_peak(tops: *mut f64) -> c_int;
    pub fn hb200_bounds_checked() -> c_int;
    pub fn hb200_bounds_selftest() -> c_int;
    pub fn hb200_plan_chunks(cost: *const c_int, n_items: usize, grid: c_int, chunks: *mut c_int) -> c_int;
    pub fn hb200_plan_rounds(op: *const c_int, panel: *const c_int, rounds: *const c_int, n_items: usize, grid: c_int, seg_begin: *mut c_int, segs: *mut c_int, seg_cap: usize, n_segs: *mut usize) -> c_int;
    pub fn hb200_block_size(dtype: c_int) -> usize;
    pub fn hb200_block_bytes(dtype: c_int) -> usize;
    pub fn hb200_byte_size(dtype: c_int, n_cols: usize) -> usize;
    pub fn hb200_selected_kernel(dtype: c_int, seq_len: usize) -> *const c_char;
    pub fn hb200_dispatch_report(dtypes: *const c_int, n_dtypes: usize, json: *mut c_char, cap: usize, needed: *mut usize) -> c_int;
    pub fn hb200_dispatch_banner(dtypes: *const c_int, n_dtypes: usize, text: *mut c_char, cap: usize, needed: *mut usize) -> c_int;
    pub fn hb200_weight_upload(dtype: c_int, n_rows: usize, n_cols: usize, packed: *const u8, bytes: usize, out: *mut *mut hb200_weight) -> c_int;
    pub fn hb200_weight_upload_dev(dtype: c_int, n_rows: usize, n_cols: usize, packed_dev: *const u8, bytes: usize, stream: *mut c_void, out: *mut *mut hb200_weight) -> c_int;
    pub fn hb200_weight_upload_rows(dtype: c_int, n_rows: usize, n_cols: usize, packed: *const u8, bytes: usize, row_begin: usize, row_end: usize, out: *mut *mut hb200_weight) -> c_int;
    pub fn hb200_weight_free(w: *mut hb200_weight) -> c_int;
    pub fn hb200_weight_info(w: *mut hb200_weight, dtype: *mut c_int, n_rows: *mut usize, n_cols: *mut usize, resident_bytes: *mut usize) -> c_int;
    pub fn hb200_act_create(max_seq_len: usize, n_cols: usize, out: *mut *mut hb200_act) -> c_int;
    pub fn hb200_act_free(a: *mut hb200_act) -> c_int;
    pub fn hb200_act_f32_ptr(a: *mut hb200_act, dev_ptr: *mut *mut f32) -> c_int;
    pub fn hb200_act_q8_planes(a: *mut hb200_act, q: *mut *mut i8, d: *mut *mut f32, sums: *mut *mut f32, ld_q: *mut usize, ld_b: *mut usize) -> c_int;
    pub fn hb200_act_quantize_dev(a: *mut hb200_act, x_dev: *const f32, seq_len: usize, stream: *mut c_void) -> c_int;
    pub fn hb200_act_load_q8_0_dev(a: *mut hb200_act, q8_dev: *const u8, seq_len: usize, q8_stride: usize, stream: *mut c_void) -> c_int;
    pub fn hb200_act_store_q8_0_dev(a: *mut hb200_act, q8_dev: *mut u8, seq_len: usize, q8_stride: usize, stream: *mut c_void) -> c_int;
    pub fn hb200_act_rms_norm_q8_dev(a: *mut hb200_act, x_dev: *const f32, weight_dev: *const f32, eps: f32, seq_len: usize, stream: *mut c_void) -> c_int;
    pub fn hb200_act_silu_mul_q8_dev(a: *mut hb200_act, gate_dev: *const f32, up_dev: *const f32, seq_len: usize, stream: *mut c_void) -> c_int;
    pub fn hb200_act_hadamard_quantize_dev(a: *mut hb200_act, x_dev: *const f32, signs_dev: *const f32, block_size: usize, seq_len: usize, rotated_dev: *mut f32, stream: *mut c_void) -> c_int;
    pub fn hb200_matmul_f32act_dev(w: *mut hb200_weight, x_dev: *const f32, seq_len: usize, out_dev: *mut f32, ld_out: usize, accumulate: c_int, stream: *mut c_void) -> c_int;
    pub fn hb200_matmul_f32act(w: *mut hb200_weight, x: *const f32, seq_len: usize, out: *mut f32, accumulate: c_int) -> c_int;
    pub fn hb200_argmax_f32_dev(x_dev: *const f32, n: usize, index_out: *mut u32, stream: *mut c_void) -> c_int;
    pub fn hb200_argmax_f32_dev_async(x_dev: *const f32, n: usize, index_dev: *mut u32, stream: *mut c_void) -> c_int;
    pub fn hb200_quantize_q8_0(x: *const f32, seq_len: usize, dim: usize, q8_out: *mut u8) -> c_int;
    pub fn hb200_rms_norm_q8(x: *const f32, weight: *const f32, eps: f32, q8_out: *mut u8, seq_len: usize, dim: usize) -> c_int;
    pub fn hb200_silu_mul_q8(gate: *const f32, up: *const f32, q8_out: *mut u8, seq_len: usize, dim: usize) -> c_int;
    pub fn hb200_hadamard_quantize_q8_0(x: *const f32, signs: *const f32, block_size: usize, q8_out: *mut u8, rotated_out: *mut f32, seq_len: usize, dim: usize) -> c_int;
    pub fn hb200_dot_rows(w: *mut hb200_weight, a_q8: *const u8, out: *mut f32) -> c_int;
    pub fn hb200_dot_rows_batched(w: *mut hb200_weight, a_q8: *const u8, seq_len: usize, q8_stride: usize, out: *mut f32) -> c_int;
    pub fn hb200_matmul_f32(w: *mut hb200_weight, x: *const f32, seq_len: usize, out: *mut f32) -> c_int;
    pub fn hb200_matmul_f32_fused(ws: *mut *mut hb200_weight, n_weights: usize, x: *const f32, seq_len: usize, outs: *const *mut f32) -> c_int;
    pub fn hb200_block_dots_i32(w: *mut hb200_weight, a_q8: *const u8, seq_len: usize, q8_stride: usize, out: *mut i32) -> c_int;
    pub fn hb200_dot_rows_dev(w: *mut hb200_weight, a: *mut hb200_act, seq_len: usize, out_dev: *mut f32, ld_out: usize, stream: *mut c_void) -> c_int;
    pub fn hb200_matmul_f32_dev(w: *mut hb200_weight, a: *mut hb200_act, seq_len: usize, out_dev: *mut f32, ld_out: usize, stream: *mut c_void) -> c_int;
    pub fn hb200_matmul_f32_noalloc(w: *mut hb200_weight, x_dev: *const f32, seq_len: usize, out_dev: *mut f32, ld_out: usize, stream: *mut c_void) -> c_int;
    pub fn hb200_weight_i8_upload(n_rows: usize, n_cols: usize, q: *const i8, scales: *const f32, out: *mut *mut hb200_weight_i8) -> c_int;
    pub fn hb200_weight_i8_upload_rows(n_rows: usize, n_cols: usize, q: *const i8, scales: *const f32, row_begin: usize, row_end: usize, out: *mut *mut hb200_weight_i8) -> c_int;
    pub fn hb200_weight_i8_upload_dev(n_rows: usize, n_cols: usize, q_dev: *const i8, ld_q: usize, scales_dev: *const f32, stream: *mut c_void, out: *mut *mut hb200_weight_i8) -> c_int;
    pub fn hb200_weight_i8_quantize_dev(n_rows: usize, n_cols: usize, w_dev: *const f32, ld_w: usize, stream: *mut c_void, out: *mut *mut hb200_weight_i8) -> c_int;
    pub fn hb200_weight_i8_store_dev(w: *mut hb200_weight_i8, q_dev: *mut i8, ld_q: usize, scales_dev: *mut f32, stream: *mut c_void) -> c_int;
    pub fn hb200_weight_i8_free(w: *mut hb200_weight_i8) -> c_int;
    pub fn hb200_weight_i8_info(w: *mut hb200_weight_i8, n_rows: *mut usize, n_cols: *mut usize, resident_bytes: *mut usize, device: *mut c_int) -> c_int;
    pub fn hb200_act_i8_create(max_seq_len: usize, n_cols: usize, out: *mut *mut hb200_act_i8) -> c_int;
    pub fn hb200_act_i8_free(a: *mut hb200_act_i8) -> c_int;
    pub fn hb200_act_i8_info(a: *mut hb200_act_i8, max_seq_len: *mut usize, n_cols: *mut usize, device: *mut c_int) -> c_int;
    pub fn hb200_act_i8_quantize_dev(a: *mut hb200_act_i8, x_dev: *const f32, ld_x: usize, seq_len: usize, stream: *mut c_void) -> c_int;
    pub fn hb200_act_i8_add_rms_norm_dev(a: *mut hb200_act_i8, x_dev: *const f32, residual_dev: *const f32, ld_x: usize, weight_dev: *const f32, eps: f32, seq_len: usize, sum_dev: *mut f32, ld_sum: usize, stream: *mut c_void) -> c_int;
    pub fn hb200_act_i8_silu_mul_dev(a: *mut hb200_act_i8, gate_dev: *const f32, up_dev: *const f32, ld: usize, seq_len: usize, stream: *mut c_void) -> c_int;
    pub fn hb200_act_i8_load_dev(a: *mut hb200_act_i8, q_dev: *const i8, ld_q: usize, scales_dev: *const f32, seq_len: usize, stream: *mut c_void) -> c_int;
    pub fn hb200_act_i8_store_dev(a: *mut hb200_act_i8, q_dev: *mut i8, ld_q: usize, scales_dev: *mut f32, seq_len: usize, stream: *mut c_void) -> c_int;
    pub fn hb200_act_i8_dequantize_dev(a: *mut hb200_act_i8, out_dev: *mut f32, ld_out: usize, seq_len: usize, stream: *mut c_void) -> c_int;
    pub fn hb200_matmul_i8_dev(w: *mut hb200_weight_i8, a: *mut hb200_act_i8, seq_len: usize, out_dev: *mut f32, ld_out: usize, accumulate: c_int, stream: *mut c_void) -> c_int;
    pub fn hb200_matmul_i8(w: *mut hb200_weight_i8, x: *const f32, seq_len: usize, out: *mut f32) -> c_int;
    pub fn hb200_matmul_i8_kernel(n_rows: usize, n_cols: usize, seq_len: usize) -> *const c_char;
    pub fn hb200_batch_create(out: *mut *mut hb200_batch) -> c_int;
    pub fn hb200_batch_add(b: *mut hb200_batch, w: *mut hb200_weight, a: *mut hb200_act, seq_len: usize, out_dev: *mut f32, ld_out: usize) -> c_int;
    pub fn hb200_batch_seal(b: *mut hb200_batch) -> c_int;
    pub fn hb200_batch_launch(b: *mut hb200_batch, stream: *mut c_void) -> c_int;
    pub fn hb200_batch_free(b: *mut hb200_batch) -> c_int;
    pub fn hb200_multi_batch_launch(batches: *mut *mut hb200_batch, n: c_int, streams: *const *mut c_void) -> c_int;
    pub fn hb200_batch_launch_count(b: *mut hb200_batch) -> c_int;
    pub fn hb200_batch_run_host(b: *mut hb200_batch, x_host: *const f32, out_dev_base: *const f32, out_floats: usize, out_host: *mut f32) -> c_int;
    pub fn hb200_batch_input_floats(b: *mut hb200_batch) -> usize;
    pub fn hb200_batch_run_dev(b: *mut hb200_batch, x_dev: *const f32, x_stream: *mut c_void, out_dev_base: *const f32, out_floats: usize, out_host: *mut f32) -> c_int;
    pub fn hb200_peer_alloc(bytes: usize, data_dev: *mut *mut c_void, handle: *mut u8) -> c_int;
    pub fn hb200_peer_free(data_dev: *mut c_void) -> c_int;
    pub fn hb200_peer_open(handle: *const u8, data_dev: *mut *mut c_void) -> c_int;
    pub fn hb200_peer_close(data_dev: *mut c_void) -> c_int;
    pub fn hb200_batch_set_peers(b: *mut hb200_batch, n_ranks: c_int, my_rank: c_int, data: *const *mut c_void, area_bytes: usize, wait: c_int) -> c_int;
    pub fn hb200_batch_peer_area(b: *mut hb200_batch) -> c_int;
    pub fn hb200_check_status() -> c_int;
    pub fn hb200_stream_synchronize(stream: *mut c_void) -> c_int;
    pub fn hb200_gguf_open(path: *const c_char, out: *mut *mut hb200_gguf) -> c_int;
    pub fn hb200_gguf_close(g: *mut hb200_gguf) -> c_int;
    pub fn hb200_gguf_version(g: *mut hb200_gguf) -> u32;
    pub fn hb200_gguf_data_offset(g: *mut hb200_gguf) -> u64;
    pub fn hb200_gguf_tensor_count(g: *mut hb200_gguf) -> usize;
    pub fn hb200_gguf_tensor_info(g: *mut hb200_gguf, index: usize, name: *mut *const c_char, dtype_id: *mut c_int, n_dims: *mut usize, shape: *mut u64, offset: *mut u64, bytes: *mut usize) -> c_int;
    pub fn hb200_gguf_find_tensor(g: *mut hb200_gguf, name: *const c_char, index: *mut usize) -> c_int;
    pub fn hb200_gguf_tensor_data(g: *mut hb200_gguf, index: usize, data: *mut *const u8, bytes: *mut usize) -> c_int;
    pub fn hb200_gguf_upload_tensor(g: *mut hb200_gguf, index: usize, out: *mut *mut hb200_weight) -> c_int;
    pub fn hb200_gguf_meta_u64(g: *mut hb200_gguf, key: *const c_char, out: *mut u64) -> c_int;
    pub fn hb200_gguf_meta_f64(g: *mut hb200_gguf, key: *const c_char, out: *mut f64) -> c_int;
    pub fn hb200_gguf_meta_str(g: *mut hb200_gguf, key: *const c_char, out: *mut *const c_char, len: *mut usize) -> c_int;
    pub fn hb200_gguf_meta_array_f32(g: *mut hb200_gguf, key: *const c_char, out: *mut f32, capacity: usize, count: *mut usize) -> c_int;
}
