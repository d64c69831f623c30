//! Raw declarations of include/lum_tree.h: the operators of speculative decoding as single calls.
//!
//! Kept in the header's order; tests/test_drafts_cpu.py parses both files and fails when a function, an argument type or a struct field differs.
#![allow(non_camel_case_types, dead_code)]

use std::os::raw::c_void;

#[repr(C)]
pub struct lum_draft_tree {
    pub row_start: *const i32,
    pub prefix: *const i32,
    pub parent: *const i32,
    pub slot: *const i32,
    pub n_seq: i32,
    pub n_rows: i32,
    pub max_rows: i32,
    pub max_prefix: i32,
}
#[repr(C)]
pub struct lum_kv_map {
    pub page_table: *const i32,
    pub rows: i64,
    pub slots: i32,
    pub max_seq: i32,
    pub page_rows: i32,
    pub pages_per_seq: i32,
}
#[repr(C)]
pub struct lum_tree_attn {
    pub q_dtype: u32,
    pub kv_dtype: u32,
    pub n_q_heads: i32,
    pub n_kv_heads: i32,
    pub head_dim: i32,
    pub window: i32,
    pub scale: f32,
    pub reserved: i32,
    pub q_stride: i64,
    pub kv_stride: i64,
    pub out_stride: i64,
}
#[repr(C)]
pub struct lum_kv_plane {
    pub rows: *mut c_void,
    pub row_bytes: u64,
}

extern "C" {
    pub fn lum_op_attn_tree_workspace(desc: *const lum_tree_attn, tree: *const lum_draft_tree, map: *const lum_kv_map) -> usize;
    pub fn lum_op_attn_tree(desc: *const lum_tree_attn, tree: *const lum_draft_tree, map: *const lum_kv_map, q_dev: *const c_void, k_dev: *const c_void, v_dev: *const c_void,
        sinks_dev: *const f32, out_dev: *mut c_void, workspace_dev: *mut c_void, workspace_bytes: usize, stream: *mut c_void) -> i32;
    pub fn lum_op_tree_accept_workspace(tree: *const lum_draft_tree, vocab: i32) -> usize;
    pub fn lum_op_tree_accept(tree: *const lum_draft_tree, tokens_dev: *const i32, logits_dev: *const f32, vocab: i32, logits_stride: i64, picks_dev: *const i32, path_dev: *mut i32,
        path_len: i32, n_accepted_dev: *mut i32, next_dev: *mut i32, workspace_dev: *mut c_void, workspace_bytes: usize, stream: *mut c_void) -> i32;
    pub fn lum_op_kv_compact(planes_dev: *const lum_kv_plane, n_planes: i32, map: *const lum_kv_map, tree: *const lum_draft_tree, path_dev: *const i32, path_len: i32,
        n_accepted_dev: *const i32, stream: *mut c_void) -> i32;
    pub fn lum_op_kv_copy(planes_dev: *const lum_kv_plane, n_planes: i32, rows: i64, spans_dev: *const i32, n_spans: i32, max_rows: i32, stream: *mut c_void) -> i32;
}
