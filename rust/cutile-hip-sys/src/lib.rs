//! Raw FFI declarations of `libcutile_hip.so` — one item per declaration of `include/cutile_hip.h`, in the
//! header's order.  This is the crate that takes the place of `cuda-bindings` / the driver half of `cuda-core`
//! (cuda-bindings/src/lib.rs:16, cuda-core/src/cudarc_shim.rs:28-807) under the reference's host crates.
//!
//! GENERATED by `gen_bindings.py` from the header; do not edit.  NOT COMPILED in the environment this was
//! written in (it has no Rust toolchain): `tests/test_rust_bindings.py` compares every declaration here with
//! the header instead (names, argument count, pointer / integer / float class and width per position, record
//! field order and sizes, constant values).
#![allow(non_camel_case_types, non_upper_case_globals, unused_imports)]
#![no_std]

use core::ffi::{c_char, c_int, c_uint, c_void};

pub const CUTILE_MAX_RANK: usize = 4;
pub const CUTILE_MAP_OWNED: i32 = 0;

pub type cutile_status_t = i32;

pub const CUTILE_SUCCESS: i32 = 0;
pub const CUTILE_ERR_LIBRARY_INIT: i32 = -1;
pub const CUTILE_ERR_INVALID_ARGUMENT: i32 = -2;
pub const CUTILE_ERR_KERNEL_NOT_FOUND: i32 = -3;
pub const CUTILE_ERR_KERNEL_LAUNCH: i32 = -4;
pub const CUTILE_ERR_TENSOR: i32 = -5;
pub const CUTILE_ERR_STATE: i32 = -6;
pub const CUTILE_ERR_OUT_OF_SLOTS: i32 = -7;

#[repr(C)]
pub struct cutile_device {
    _private: [u8; 0],
}
pub type cutile_device_t = *mut cutile_device;

pub type cutile_stream_t = *mut c_void;

pub type cutile_event_t = *mut c_void;

#[repr(C)]
pub struct cutile_module {
    _private: [u8; 0],
}
pub type cutile_module_t = *mut cutile_module;

pub type cutile_function_t = *mut c_void;

pub type cutile_mempool_t = *mut c_void;

pub type cutile_graph_t = *mut c_void;

pub type cutile_graph_exec_t = *mut c_void;

#[repr(C)]
#[derive(Clone, Copy)]
pub struct cutile_device_props_t {
    pub compute_units: i32,
    pub clock_khz: i32,
    pub memory_clock_khz: i32,
    pub memory_bus_bits: i32,
    pub l2_bytes: i32,
    pub lds_bytes_per_block: i32,
    pub wavefront_size: i32,
    pub reserved: i32,
    pub total_memory_bytes: u64,
}

pub type cutile_host_fn_t = Option<unsafe extern "C" fn(user: *mut c_void)>;

#[repr(C)]
#[derive(Clone, Copy)]
pub struct cutile_pool_mem_stats_t {
    pub reserved_current: u64,
    pub reserved_high: u64,
    pub used_current: u64,
    pub used_high: u64,
}

#[repr(C)]
pub struct cutile_rng {
    _private: [u8; 0],
}
pub type cutile_rng_t = *mut cutile_rng;

#[repr(C)]
#[derive(Clone, Copy)]
pub struct cutile_kernel_info_t {
    pub function: cutile_function_t,
    pub symbol: *const c_char,
    pub variant: *const c_char,
    pub block: [u32; 3],
    pub lds_bytes: u32,
    pub tile: [i32; 4],
}

#[repr(C)]
pub struct cutile_launch {
    _private: [u8; 0],
}
pub type cutile_launch_t = *mut cutile_launch;

pub type cutile_dtype_t = c_int;
pub const CUTILE_DTYPE_F32: cutile_dtype_t = 0;
pub const CUTILE_DTYPE_F64: cutile_dtype_t = 1;
pub const CUTILE_DTYPE_F16: cutile_dtype_t = 2;
pub const CUTILE_DTYPE_BF16: cutile_dtype_t = 3;
pub const CUTILE_DTYPE_I8: cutile_dtype_t = 4;
pub const CUTILE_DTYPE_I16: cutile_dtype_t = 5;
pub const CUTILE_DTYPE_I32: cutile_dtype_t = 6;
pub const CUTILE_DTYPE_I64: cutile_dtype_t = 7;
pub const CUTILE_DTYPE_U8: cutile_dtype_t = 8;
pub const CUTILE_DTYPE_U16: cutile_dtype_t = 9;
pub const CUTILE_DTYPE_U32: cutile_dtype_t = 10;
pub const CUTILE_DTYPE_U64: cutile_dtype_t = 11;
pub const CUTILE_DTYPE_BOOL: cutile_dtype_t = 12;
pub const CUTILE_DTYPE_F8E4M3FN: cutile_dtype_t = 13;
pub const CUTILE_DTYPE_F8E5M2: cutile_dtype_t = 14;
pub const CUTILE_DTYPE_F8E8M0FNU: cutile_dtype_t = 15;
pub const CUTILE_DTYPE_F4E2M1FNX2: cutile_dtype_t = 16;
pub const CUTILE_DTYPE_COUNT: cutile_dtype_t = 17;

#[repr(C)]
#[derive(Clone, Copy)]
pub struct cutile_tensor_arg_t {
    pub ptr: *mut c_void,
    pub dtype: cutile_dtype_t,
    pub rank: i32,
    pub shape: [i32; CUTILE_MAX_RANK],
    pub strides: [i32; CUTILE_MAX_RANK],
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct cutile_partition_arg_t {
    pub tensor: cutile_tensor_arg_t,
    pub partition_shape: [i32; CUTILE_MAX_RANK],
    pub partition_strides: [i32; CUTILE_MAX_RANK],
    pub prefix_coverage: i32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct cutile_launch_opts_t {
    pub grid: [u32; 3],
    pub generics: *const *const c_char,
    pub n_generics: i32,
    pub variant: *const c_char,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct cutile_mapped_partition_arg_t {
    pub partition: cutile_partition_arg_t,
    pub map_rank: i32,
    pub map_shape: [i32; 3],
    pub num_tile_blocks: u32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct cutile_spec_bits_t {
    pub shape_div: [i32; CUTILE_MAX_RANK],
    pub stride_div: [i32; CUTILE_MAX_RANK],
    pub stride_one: [i32; CUTILE_MAX_RANK],
    pub base_ptr_div: i32,
    pub elements_disjoint: i32,
}

pub const CUTILE_KVBM_STACKED_NHD: i32 = 0;
pub const CUTILE_KVBM_STACKED_HND: i32 = 1;

pub const CUTILE_KVBM_OPERATIONAL_NHD: i32 = 0;
pub const CUTILE_KVBM_OPERATIONAL_HND: i32 = 1;
pub const CUTILE_KVBM_UNIVERSAL: i32 = 2;

pub type cutile_policy_kind_t = c_int;
pub const CUTILE_POLICY_ROUND_ROBIN: cutile_policy_kind_t = 0;
pub const CUTILE_POLICY_SINGLE_STREAM: cutile_policy_kind_t = 1;

pub type cutile_waker_fn_t = Option<unsafe extern "C" fn(user: *mut c_void)>;

#[link(name = "cutile_hip")]
extern "C" {
    pub fn cutile_last_error_message() -> *const c_char;
    pub fn cutile_status_name(status: cutile_status_t) -> *const c_char;
    pub fn cutile_version() -> *const c_char;
    pub fn cutile_init() -> cutile_status_t;
    pub fn cutile_device_count(count: *mut i32) -> cutile_status_t;
    pub fn cutile_device_get(ordinal: i32, device: *mut cutile_device_t) -> cutile_status_t;
    pub fn cutile_device_name(device: cutile_device_t, buf: *mut c_char, buf_len: usize) -> cutile_status_t;
    pub fn cutile_device_arch(device: cutile_device_t, buf: *mut c_char, buf_len: usize) -> cutile_status_t;
    pub fn cutile_device_bind_to_thread(device: cutile_device_t) -> cutile_status_t;
    pub fn cutile_device_synchronize(device: cutile_device_t) -> cutile_status_t;
    pub fn cutile_device_l2_cache_size(device: cutile_device_t, bytes: *mut usize) -> cutile_status_t;
    pub fn cutile_device_props(device: cutile_device_t, props: *mut cutile_device_props_t) -> cutile_status_t;
    pub fn cutile_stream_create(device: cutile_device_t, stream: *mut cutile_stream_t) -> cutile_status_t;
    pub fn cutile_stream_release(device: cutile_device_t, stream: cutile_stream_t) -> cutile_status_t;
    pub fn cutile_stream_synchronize(stream: cutile_stream_t) -> cutile_status_t;
    pub fn cutile_stream_query(stream: cutile_stream_t, done: *mut i32) -> cutile_status_t;
    pub fn cutile_stream_launch_host_func(stream: cutile_stream_t, r#fn: cutile_host_fn_t, user: *mut c_void) -> cutile_status_t;
    pub fn cutile_stream_begin_capture(stream: cutile_stream_t) -> cutile_status_t;
    pub fn cutile_stream_end_capture(stream: cutile_stream_t, graph: *mut cutile_graph_t) -> cutile_status_t;
    pub fn cutile_stream_write_value32(stream: cutile_stream_t, device_ptr: *mut c_void, value: u32) -> cutile_status_t;
    pub fn cutile_event_create(event: *mut cutile_event_t) -> cutile_status_t;
    pub fn cutile_event_record(event: cutile_event_t, stream: cutile_stream_t) -> cutile_status_t;
    pub fn cutile_event_synchronize(event: cutile_event_t) -> cutile_status_t;
    pub fn cutile_event_elapsed_ms(start: cutile_event_t, end: cutile_event_t, ms: *mut f32) -> cutile_status_t;
    pub fn cutile_event_destroy(event: cutile_event_t) -> cutile_status_t;
    pub fn cutile_module_load_data(device: cutile_device_t, image: *const c_void, size: usize, module: *mut cutile_module_t) -> cutile_status_t;
    pub fn cutile_module_unload(module: cutile_module_t) -> cutile_status_t;
    pub fn cutile_module_get_function(module: cutile_module_t, name: *const c_char, function: *mut cutile_function_t) -> cutile_status_t;
    pub fn cutile_launch_kernel(function: cutile_function_t, grid: *const u32, block: *const u32, shared_mem_bytes: u32, stream: cutile_stream_t, kernel_params: *mut *mut c_void) -> cutile_status_t;
    pub fn cutile_malloc_async(bytes: usize, stream: cutile_stream_t, device_ptr: *mut *mut c_void) -> cutile_status_t;
    pub fn cutile_malloc_from_pool_async(bytes: usize, pool: cutile_mempool_t, stream: cutile_stream_t, device_ptr: *mut *mut c_void) -> cutile_status_t;
    pub fn cutile_free_async(device_ptr: *mut c_void, stream: cutile_stream_t) -> cutile_status_t;
    pub fn cutile_memset_d8_async(device_ptr: *mut c_void, value: u8, bytes: usize, stream: cutile_stream_t) -> cutile_status_t;
    pub fn cutile_memcpy_htod_async(dst: *mut c_void, src: *const c_void, bytes: usize, stream: cutile_stream_t) -> cutile_status_t;
    pub fn cutile_memcpy_dtoh_async(dst: *mut c_void, src: *const c_void, bytes: usize, stream: cutile_stream_t) -> cutile_status_t;
    pub fn cutile_memcpy_dtod_async(dst: *mut c_void, src: *const c_void, bytes: usize, stream: cutile_stream_t) -> cutile_status_t;
    pub fn cutile_host_alloc_mapped(bytes: usize, host_ptr: *mut *mut c_void, device_ptr: *mut *mut c_void) -> cutile_status_t;
    pub fn cutile_host_free(host_ptr: *mut c_void) -> cutile_status_t;
    pub fn cutile_mempool_create(device: cutile_device_t, pool: *mut cutile_mempool_t) -> cutile_status_t;
    pub fn cutile_mempool_default(device: cutile_device_t, pool: *mut cutile_mempool_t) -> cutile_status_t;
    pub fn cutile_mempool_destroy(pool: cutile_mempool_t) -> cutile_status_t;
    pub fn cutile_mempool_set_release_threshold(pool: cutile_mempool_t, bytes: u64) -> cutile_status_t;
    pub fn cutile_mempool_stats(pool: cutile_mempool_t, stats: *mut cutile_pool_mem_stats_t) -> cutile_status_t;
    pub fn cutile_mempool_reset_used_high(pool: cutile_mempool_t) -> cutile_status_t;
    pub fn cutile_mempool_reset_reserved_high(pool: cutile_mempool_t) -> cutile_status_t;
    pub fn cutile_graph_instantiate(graph: cutile_graph_t, exec: *mut cutile_graph_exec_t) -> cutile_status_t;
    pub fn cutile_graph_upload(exec: cutile_graph_exec_t, stream: cutile_stream_t) -> cutile_status_t;
    pub fn cutile_graph_launch(exec: cutile_graph_exec_t, stream: cutile_stream_t) -> cutile_status_t;
    pub fn cutile_graph_exec_destroy(exec: cutile_graph_exec_t) -> cutile_status_t;
    pub fn cutile_graph_destroy(graph: cutile_graph_t) -> cutile_status_t;
    pub fn cutile_rng_create(rng: *mut cutile_rng_t) -> cutile_status_t;
    pub fn cutile_rng_set_seed(rng: cutile_rng_t, seed: u64) -> cutile_status_t;
    pub fn cutile_rng_set_offset(rng: cutile_rng_t, offset: u64) -> cutile_status_t;
    pub fn cutile_rng_get_offset(rng: cutile_rng_t, offset: *mut u64) -> cutile_status_t;
    pub fn cutile_rng_normal_f32(rng: cutile_rng_t, device_ptr: *mut c_void, num_elements: usize, mean: f32, std: f32, stream: cutile_stream_t) -> cutile_status_t;
    pub fn cutile_rng_normal_f64(rng: cutile_rng_t, device_ptr: *mut c_void, num_elements: usize, mean: f64, std: f64, stream: cutile_stream_t) -> cutile_status_t;
    pub fn cutile_rng_uniform_f32(rng: cutile_rng_t, device_ptr: *mut c_void, num_elements: usize, stream: cutile_stream_t) -> cutile_status_t;
    pub fn cutile_rng_uniform_f64(rng: cutile_rng_t, device_ptr: *mut c_void, num_elements: usize, stream: cutile_stream_t) -> cutile_status_t;
    pub fn cutile_rng_destroy(rng: cutile_rng_t) -> cutile_status_t;
    pub fn cutile_kernel_lookup(device: cutile_device_t, function: *const c_char, generics: *const *const c_char, n_generics: i32, variant: *const c_char, info: *mut cutile_kernel_info_t) -> cutile_status_t;
    pub fn cutile_module_load_count() -> u64;
    pub fn cutile_kernel_list(names: *mut *const c_char, cap: i32) -> i32;
    pub fn cutile_kernel_set_preferred_variant(function: *const c_char, variant: *const c_char) -> cutile_status_t;
    pub fn cutile_kernel_set_preferred_variant_for(function: *const c_char, bucket: *const c_char, variant: *const c_char) -> cutile_status_t;
    pub fn cutile_tuning_reload(directory: *const c_char) -> cutile_status_t;
    pub fn cutile_tuning_report() -> *const c_char;
    pub fn cutile_tuning_applied_count() -> i32;
    pub fn cutile_last_resolved_source() -> *const c_char;
    pub fn cutile_last_resolved_bucket() -> *const c_char;
    pub fn cutile_library_version() -> *const c_char;
    pub fn cutile_toolchain_fingerprint() -> *const c_char;
    pub fn cutile_target_arch() -> *const c_char;
    pub fn cutile_kernel_fingerprint(function: *const c_char, variant: *const c_char, out: *mut c_char) -> cutile_status_t;
    pub fn cutile_launch_create(function: cutile_function_t, launch: *mut cutile_launch_t) -> cutile_status_t;
    pub fn cutile_launch_destroy(launch: cutile_launch_t) -> cutile_status_t;
    pub fn cutile_launch_push_arg(launch: cutile_launch_t, value: *const c_void, size: usize, align: usize) -> cutile_status_t;
    pub fn cutile_launch_push_device_ptr(launch: cutile_launch_t, device_ptr: *mut c_void) -> cutile_status_t;
    pub fn cutile_launch_set_config(launch: cutile_launch_t, grid: *const u32, block: *const u32, shared_mem_bytes: u32) -> cutile_status_t;
    pub fn cutile_launch_execute(launch: cutile_launch_t, stream: cutile_stream_t) -> cutile_status_t;
    pub fn cutile_dtype_name(dtype: cutile_dtype_t) -> *const c_char;
    pub fn cutile_dtype_size(dtype: cutile_dtype_t) -> usize;
    pub fn cutile_dtype_from_name(name: *const c_char) -> cutile_dtype_t;
    pub fn cutile_set_launch_mode(mode: i32) -> cutile_status_t;
    pub fn cutile_get_launch_mode(mode: *mut i32) -> cutile_status_t;
    pub fn cutile_last_resolved_kernel(function: *mut *const c_char, info: *mut cutile_kernel_info_t) -> cutile_status_t;
    pub fn cutile_partition_grid(p: *const cutile_partition_arg_t, grid: *mut u32) -> cutile_status_t;
    pub fn cutile_infer_launch_grid(explicit_grid: *const u32, partitions: *const *const cutile_partition_arg_t, n_partitions: i32, grid: *mut u32) -> cutile_status_t;
    pub fn cutile_mapped_partition_grid(p: *const cutile_mapped_partition_arg_t, grid: *mut u32) -> cutile_status_t;
    pub fn cutile_mapped_partition_index(p: *const cutile_mapped_partition_arg_t, item: u32, index: *mut u32, n_items: *mut u32) -> cutile_status_t;
    pub fn cutile_mapped_partition_index_within(p: *const cutile_mapped_partition_arg_t, ranges: *const i32, item: u32, index: *mut u32, n_items: *mut u32) -> cutile_status_t;
    pub fn cutile_launch_mapped_tile_index_within(stream: cutile_stream_t, z: *const cutile_mapped_partition_arg_t, ranges: *const i32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_mapped_partitions_shared(a: *const cutile_mapped_partition_arg_t, b: *const cutile_mapped_partition_arg_t) -> cutile_status_t;
    pub fn cutile_launch_mapped_shared_cache_update_f32(stream: cutile_stream_t, k_cache: *const cutile_mapped_partition_arg_t, v_cache: *const cutile_mapped_partition_arg_t, new_k: *const cutile_tensor_arg_t, source_seq_major: i32, position: *const cutile_tensor_arg_t, start_tile: i32, n_tiles: i32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_gemm_persistent(stream: cutile_stream_t, z: *const cutile_mapped_partition_arg_t, x: *const cutile_tensor_arg_t, y: *const cutile_tensor_arg_t, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_mapped_tile_index(stream: cutile_stream_t, z: *const cutile_mapped_partition_arg_t, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_compute_spec(t: *const cutile_tensor_arg_t, spec: *mut cutile_spec_bits_t) -> cutile_status_t;
    pub fn cutile_launch_saxpy(stream: cutile_stream_t, y: *const cutile_partition_arg_t, a: f64, x: *const cutile_tensor_arg_t, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_axpy(stream: cutile_stream_t, z: *const cutile_partition_arg_t, a: f64, x: *const cutile_tensor_arg_t, y: *const cutile_tensor_arg_t, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_add(stream: cutile_stream_t, z: *const cutile_partition_arg_t, x: *const cutile_tensor_arg_t, y: *const cutile_tensor_arg_t, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_full(stream: cutile_stream_t, value: f64, int_value: i64, t: *const cutile_partition_arg_t, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_arange(stream: cutile_stream_t, t: *const cutile_partition_arg_t, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_linspace(stream: cutile_stream_t, t: *const cutile_partition_arg_t, start: f32, step: f32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_eye(stream: cutile_stream_t, t: *const cutile_partition_arg_t, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_relu(stream: cutile_stream_t, input_output: *const cutile_partition_arg_t, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_dropout(stream: cutile_stream_t, p: f32, x: *const cutile_tensor_arg_t, x_keep: *const cutile_tensor_arg_t, out: *const cutile_partition_arg_t, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_scale_ptr(stream: cutile_stream_t, out_ptr: *mut c_void, in_ptr: *const c_void, scale: f32, len: i32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_matvec(stream: cutile_stream_t, z: *const cutile_partition_arg_t, x: *const cutile_tensor_arg_t, y: *const cutile_tensor_arg_t, k: i32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_convert(stream: cutile_stream_t, src: *const cutile_tensor_arg_t, dst: *const cutile_partition_arg_t, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_rms_norm_f16(stream: cutile_stream_t, x: *const cutile_tensor_arg_t, w: *const cutile_tensor_arg_t, out: *const cutile_partition_arg_t, eps: f32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_rms_norm_f32(stream: cutile_stream_t, x: *const cutile_tensor_arg_t, w: *const cutile_tensor_arg_t, out: *const cutile_partition_arg_t, eps: f32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_softmax(stream: cutile_stream_t, x: *const cutile_tensor_arg_t, y: *const cutile_partition_arg_t, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_rms_norm_all_f16(stream: cutile_stream_t, x: *const cutile_tensor_arg_t, w: *const cutile_tensor_arg_t, out: *const cutile_partition_arg_t, eps: f32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_softmax_all_f16(stream: cutile_stream_t, x: *const cutile_tensor_arg_t, y: *const cutile_partition_arg_t, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_add_rms_norm_f16(stream: cutile_stream_t, residual: *const cutile_tensor_arg_t, x: *const cutile_tensor_arg_t, w: *const cutile_tensor_arg_t, out: *const cutile_partition_arg_t, residual_out: *const cutile_partition_arg_t, eps: f32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_qk_norm_f16(stream: cutile_stream_t, q: *const cutile_tensor_arg_t, k: *const cutile_tensor_arg_t, q_weight: *const cutile_tensor_arg_t, k_weight: *const cutile_tensor_arg_t, out: *const cutile_partition_arg_t, eps: f32, num_q_rows: i32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_add_2d_f16(stream: cutile_stream_t, out: *const cutile_partition_arg_t, lhs: *const cutile_tensor_arg_t, rhs: *const cutile_tensor_arg_t, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_silu_mul_2d_f16(stream: cutile_stream_t, out: *const cutile_partition_arg_t, gate: *const cutile_tensor_arg_t, up: *const cutile_tensor_arg_t, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_rope_f16(stream: cutile_stream_t, q: *const cutile_tensor_arg_t, k: *const cutile_tensor_arg_t, inv_freq: *const cutile_tensor_arg_t, position_start_dev: *const cutile_tensor_arg_t, position_start: i32, out: *const cutile_partition_arg_t, num_q_heads: i32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_kv_cache_update_f16(stream: cutile_stream_t, new_k: *const cutile_tensor_arg_t, new_v: *const cutile_tensor_arg_t, k_cache: *const cutile_partition_arg_t, v_cache: *const cutile_partition_arg_t, position_start_dev: *const cutile_tensor_arg_t, position_start: i32, seq_len: i32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_fmha_decode_gqa_split(stream: cutile_stream_t, q: *const cutile_tensor_arg_t, k: *const cutile_tensor_arg_t, v: *const cutile_tensor_arg_t, att_out: *const cutile_partition_arg_t, lse_out: *const cutile_partition_arg_t, qk_scale: f32, position_start: *const cutile_tensor_arg_t, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_attention_decode_kernel_grouped_f16(stream: cutile_stream_t, q: *const c_void, q_shape: *const i32, q_strides: *const i32, k: *const c_void, k_shape: *const i32, k_strides: *const i32, v: *const c_void, v_shape: *const i32, v_strides: *const i32, att: *mut c_void, att_shape: *const i32, att_strides: *const i32, lse: *mut c_void, lse_shape: *const i32, lse_strides: *const i32, softmax_scale: f32, s_kv: *const c_void, tile_n: i32, kv_len_per_split: i32, query_group_tile_size: i32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_splitk_reduce_merge(stream: cutile_stream_t, att_partial: *const cutile_tensor_arg_t, lse_partial: *const cutile_tensor_arg_t, out: *const cutile_partition_arg_t, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_fmha_decode_gqa_noalloc(stream: cutile_stream_t, q: *const cutile_tensor_arg_t, k: *const cutile_tensor_arg_t, v: *const cutile_tensor_arg_t, out: *const cutile_partition_arg_t, qk_scale: f32, position_start: *const cutile_tensor_arg_t, num_kv_splits: i32, bn: i32) -> cutile_status_t;
    pub fn cutile_fmha_decode_gqa_noalloc_prepare(q: *const cutile_tensor_arg_t, k: *const cutile_tensor_arg_t, v: *const cutile_tensor_arg_t, out: *const cutile_partition_arg_t, position_start: *const cutile_tensor_arg_t, num_kv_splits: i32, bn: i32) -> cutile_status_t;
    pub fn cutile_scratch_capacity(bytes: *mut usize) -> cutile_status_t;
    pub fn cutile_launch_gemm(stream: cutile_stream_t, z: *const cutile_partition_arg_t, x: *const cutile_tensor_arg_t, y: *const cutile_tensor_arg_t, k: i32, accumulate: i32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_batch_matmul(stream: cutile_stream_t, c: *const cutile_partition_arg_t, a: *const cutile_tensor_arg_t, b: *const cutile_tensor_arg_t, k: i32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_copy_stacked_to_contiguous_f16(stream: cutile_stream_t, stacked_layout: i32, contiguous_layout: i32, num_blocks: i32, stacked_tensors: *const cutile_tensor_arg_t, contiguous_tensors: *const cutile_tensor_arg_t, nh: i32, nl: i32, no: i32, nt: i32, hd: i32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_copy_contiguous_to_stacked_f16(stream: cutile_stream_t, stacked_layout: i32, contiguous_layout: i32, num_blocks: i32, stacked_tensors: *const cutile_tensor_arg_t, contiguous_tensors: *const cutile_tensor_arg_t, nh: i32, nl: i32, no: i32, nt: i32, hd: i32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_add_rms_norm_decode_raw_f16(stream: cutile_stream_t, residual: *const c_void, x: *const c_void, w: *const c_void, out: *mut c_void, residual_out: *mut c_void, eps: f32, n: i32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_qk_norm_rope_kv_prefill_raw_f16(stream: cutile_stream_t, q: *const c_void, k: *const c_void, v: *const c_void, q_weight: *const c_void, k_weight: *const c_void, inv_freq: *const c_void, q_out: *mut c_void, k_cache: *mut c_void, v_cache: *mut c_void, eps: f32, position_start: i32, seq_len: i32, num_q_heads: i32, num_kv_heads: i32, d: i32, max_seq: i32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_qk_norm_rope_kv_decode_raw_f16(stream: cutile_stream_t, qkv: *const c_void, q_weight: *const c_void, k_weight: *const c_void, inv_freq: *const c_void, q_out: *mut c_void, k_cache: *mut c_void, v_cache: *mut c_void, position_start: *const cutile_tensor_arg_t, eps: f32, num_q_heads: i32, num_kv_heads: i32, d: i32, max_seq: i32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_group_gemm_f16_nt_desc(stream: cutile_stream_t, a_ptrs: *const cutile_tensor_arg_t, b_ptrs: *const cutile_tensor_arg_t, c_ptrs: *const cutile_tensor_arg_t, a_metas: *const cutile_tensor_arg_t, b_metas: *const cutile_tensor_arg_t, c_metas: *const cutile_tensor_arg_t, num_groups: i32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_argmax_blocks_f16(stream: cutile_stream_t, logits: *const cutile_tensor_arg_t, block_max: *const cutile_partition_arg_t, block_idx: *const cutile_partition_arg_t, len: i32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_lm_head_argmax_blocks_f16(stream: cutile_stream_t, weights: *const cutile_tensor_arg_t, hidden: *const cutile_tensor_arg_t, block_max: *const cutile_partition_arg_t, block_idx: *const cutile_partition_arg_t, vocab_size: i32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_argmax_reduce_blocks_to_u32(stream: cutile_stream_t, block_max: *const cutile_tensor_arg_t, block_idx: *const cutile_tensor_arg_t, out: *const cutile_partition_arg_t, num_blocks: i32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_embedding_batch_f16(stream: cutile_stream_t, token_ids: *const cutile_tensor_arg_t, table: *const cutile_tensor_arg_t, out: *const cutile_partition_arg_t, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_gather_row_f16(stream: cutile_stream_t, src: *const cutile_tensor_arg_t, out: *const cutile_partition_arg_t, row_idx: i32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_fmha_seq_f16(stream: cutile_stream_t, q: *const cutile_tensor_arg_t, k: *const cutile_tensor_arg_t, v: *const cutile_tensor_arg_t, out: *const cutile_partition_arg_t, qk_scale: f32, query_group_size: i32, kv_len: i32, query_start: i32, position_start: *const cutile_tensor_arg_t, kv_len_from_position: i32, causal: i32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_fmha_prefill_gqa_lpt_raw_f16(stream: cutile_stream_t, q: *const c_void, k: *const c_void, v: *const c_void, out: *mut c_void, qk_scale: f32, query_group_size: i32, q_len: i32, kv_len: i32, query_start: i32, num_head_groups: i32, group: i32, d: i32, causal: i32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_fmha(stream: cutile_stream_t, out: *const cutile_partition_arg_t, q: *const cutile_tensor_arg_t, k: *const cutile_tensor_arg_t, v: *const cutile_tensor_arg_t, qk_scale: f32, input_pos: i32, query_group_size: i32, causal: i32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_linear_tile_mxfp8(stream: cutile_stream_t, z: *const cutile_partition_arg_t, x: *const cutile_tensor_arg_t, y: *const cutile_tensor_arg_t, x_scales: *const cutile_tensor_arg_t, y_scales: *const cutile_tensor_arg_t, alpha: f32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_linear_tile_nvfp4(stream: cutile_stream_t, z: *const cutile_partition_arg_t, x: *const cutile_tensor_arg_t, y: *const cutile_tensor_arg_t, x_scales: *const cutile_tensor_arg_t, y_scales: *const cutile_tensor_arg_t, alpha: f32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_block_quantize(stream: cutile_stream_t, x: *const cutile_tensor_arg_t, out: *const cutile_partition_arg_t, scales: *const cutile_partition_arg_t, tensor_scale: f32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_block_dequantize(stream: cutile_stream_t, x: *const cutile_tensor_arg_t, scales: *const cutile_tensor_arg_t, tensor_scale: f32, out: *const cutile_partition_arg_t, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_rms_norm_quantize(stream: cutile_stream_t, x: *const cutile_tensor_arg_t, w: *const cutile_tensor_arg_t, out: *const cutile_partition_arg_t, scales: *const cutile_partition_arg_t, eps: f32, tensor_scale: f32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_add_rms_norm_quantize(stream: cutile_stream_t, residual: *const cutile_tensor_arg_t, x: *const cutile_tensor_arg_t, w: *const cutile_tensor_arg_t, out: *const cutile_partition_arg_t, scales: *const cutile_partition_arg_t, residual_out: *const cutile_partition_arg_t, eps: f32, tensor_scale: f32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_silu_mul_quantize(stream: cutile_stream_t, gate: *const cutile_tensor_arg_t, up: *const cutile_tensor_arg_t, out: *const cutile_partition_arg_t, scales: *const cutile_partition_arg_t, tensor_scale: f32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_linear_tile_mxfp4(stream: cutile_stream_t, z: *const cutile_partition_arg_t, x: *const cutile_tensor_arg_t, y: *const cutile_tensor_arg_t, x_scales: *const cutile_tensor_arg_t, y_scales: *const cutile_tensor_arg_t, alpha: f32, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_paged_cache_write(stream: cutile_stream_t, new_k: *const cutile_tensor_arg_t, new_v: *const cutile_tensor_arg_t, k_cache: *const cutile_tensor_arg_t, v_cache: *const cutile_tensor_arg_t, k_scales: *const cutile_tensor_arg_t, v_scales: *const cutile_tensor_arg_t, page_table: *const cutile_tensor_arg_t, starts: *const cutile_tensor_arg_t, context_lens: *const cutile_tensor_arg_t, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_paged_cache_read(stream: cutile_stream_t, k_cache: *const cutile_tensor_arg_t, v_cache: *const cutile_tensor_arg_t, k_scales: *const cutile_tensor_arg_t, v_scales: *const cutile_tensor_arg_t, page_table: *const cutile_tensor_arg_t, starts: *const cutile_tensor_arg_t, context_lens: *const cutile_tensor_arg_t, out_k: *const cutile_partition_arg_t, out_v: *const cutile_partition_arg_t, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_paged_attention(stream: cutile_stream_t, q: *const cutile_tensor_arg_t, k_cache: *const cutile_tensor_arg_t, v_cache: *const cutile_tensor_arg_t, k_scales: *const cutile_tensor_arg_t, v_scales: *const cutile_tensor_arg_t, page_table: *const cutile_tensor_arg_t, starts: *const cutile_tensor_arg_t, context_lens: *const cutile_tensor_arg_t, out: *const cutile_partition_arg_t, qk_scale: f32, window: i32, max_new: i32, max_context: i32, workspace: *const cutile_tensor_arg_t, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_launch_adjust_logits(stream: cutile_stream_t, logits: *const cutile_tensor_arg_t, out: *const cutile_partition_arg_t, tokens: *const cutile_tensor_arg_t, prompt_lens: *const cutile_tensor_arg_t, token_lens: *const cutile_tensor_arg_t, repetition: *const cutile_tensor_arg_t, presence: *const cutile_tensor_arg_t, frequency: *const cutile_tensor_arg_t, bias_ids: *const cutile_tensor_arg_t, bias_values: *const cutile_tensor_arg_t, allowed: *const cutile_tensor_arg_t, opts: *const cutile_launch_opts_t) -> cutile_status_t;
    pub fn cutile_execution_lock_acquire() -> cutile_status_t;
    pub fn cutile_execution_lock_release();
    pub fn cutile_execution_lock_held() -> i32;
    pub fn cutile_get_default_device() -> i32;
    pub fn cutile_set_default_device(ordinal: i32);
    pub fn cutile_init_device_contexts(default_device: i32, num_devices: i32) -> cutile_status_t;
    pub fn cutile_init_device(ordinal: i32, kind: cutile_policy_kind_t, num_streams: i32) -> cutile_status_t;
    pub fn cutile_policy_next_stream(ordinal: i32, stream: *mut cutile_stream_t) -> cutile_status_t;
    pub fn cutile_deallocator_stream(ordinal: i32, stream: *mut cutile_stream_t) -> cutile_status_t;
    pub fn cutile_set_device_pool(ordinal: i32, pool: cutile_mempool_t) -> cutile_status_t;
    pub fn cutile_get_device_pool(ordinal: i32, pool: *mut cutile_mempool_t) -> cutile_status_t;
    pub fn cutile_reactor_register(stream: cutile_stream_t, waker: cutile_waker_fn_t, user: *mut c_void) -> cutile_status_t;
    pub fn cutile_completion_register(stream: cutile_stream_t, waker: cutile_waker_fn_t, user: *mut c_void) -> cutile_status_t;
    pub fn cutile_reactor_registrations() -> u64;
    pub fn cutile_reactor_wakes() -> u64;
    pub fn cutile_reactor_armed() -> i32;
}
