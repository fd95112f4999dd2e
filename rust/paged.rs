// src/engine/gpu/paged.rs for gguf-runner: the declarations of include/gr_paged.h (paged
// KV cache, attention over packed batches).  Every struct is a #[repr(C)] copy of the
// header's struct, field for field and in order (tests/test_paged_args.py checks them);
// status codes, element types and gr_last_error() are in ffi.rs.
#![allow(non_camel_case_types, dead_code)]
use std::ffi::c_void;

#[repr(C)]
pub struct GrPagedCache {
    pub n_pages: i32,
    pub page_size: i32,
    pub n_kv_heads: i32,
    pub head_dim: i32,
    pub kv_dtype: i32,
    pub k_pages: *mut c_void,
    pub v_pages: *mut c_void,
    pub page_stride: i64,
    pub row_stride: i64,
    pub head_stride: i64,
    pub k_scale: *mut f32,
    pub v_scale: *mut f32,
    pub scale_page_stride: i64,
    pub scale_row_stride: i64,
    pub scale_head_stride: i64,
}

#[repr(C)]
pub struct GrPagedBatch {
    pub n_seq: i32,
    pub n_rows: i32,
    pub max_rows: i32,
    pub max_len: i32,
    pub row_start: *const i32,
    pub kv_len: *const i32,
    pub page_table: *const i32,
    pub table_stride: i64,
    pub table_pages: i32,
}

#[repr(C)]
pub struct GrPagedRows {
    pub dtype: i32,
    pub k: *mut c_void,
    pub v: *mut c_void,
    pub row_stride: i64,
    pub head_stride: i64,
}

#[repr(C)]
pub struct GrPagedAttentionArgs {
    pub n_heads: i32,
    pub dtype: i32,
    pub window: i32,
    pub score_scale: f32,
    pub q: *const c_void,
    pub q_row_stride: i64,
    pub q_head_stride: i64,
    pub out: *mut c_void,
    pub out_row_stride: i64,
    pub out_head_stride: i64,
    pub workspace: *mut c_void,
}

#[repr(C)]
pub struct GrPackedArgs {
    pub n_seq: i32,
    pub n_rows: i32,
    pub max_rows: i32,
    pub n_heads: i32,
    pub n_kv_heads: i32,
    pub head_dim: i32,
    pub dtype: i32,
    pub window: i32,
    pub score_scale: f32,
    pub seq_start: *const i32,
    pub q: *const c_void,
    pub q_row_stride: i64,
    pub q_head_stride: i64,
    pub k: *const c_void,
    pub v: *const c_void,
    pub kv_row_stride: i64,
    pub kv_head_stride: i64,
    pub out: *mut c_void,
    pub out_row_stride: i64,
    pub out_head_stride: i64,
    pub workspace: *mut c_void,
}

unsafe extern "C" {
    pub fn gr_paged_kv_write(c: *const GrPagedCache, b: *const GrPagedBatch, rows: *const GrPagedRows, stream: *mut c_void) -> i32;
    pub fn gr_paged_kv_read(c: *const GrPagedCache, b: *const GrPagedBatch, rows: *const GrPagedRows, stream: *mut c_void) -> i32;
    pub fn gr_paged_attention_workspace_size(c: *const GrPagedCache, b: *const GrPagedBatch, a: *const GrPagedAttentionArgs) -> usize;
    pub fn gr_paged_attention(c: *const GrPagedCache, b: *const GrPagedBatch, a: *const GrPagedAttentionArgs, stream: *mut c_void) -> i32;
    pub fn gr_packed_attention_workspace_size(a: *const GrPackedArgs) -> usize;
    pub fn gr_packed_attention(a: *const GrPackedArgs, stream: *mut c_void) -> i32;
}
