//! Attention over packed prompts, a paged key/value cache and shared prefixes, and the cache's page
//! keeping (include/hq_attn.h), for `crates/nebula-hydrogen` (Linux / ROCm); beside qgemm.rs, whose
//! types, errors and conventions it shares. Every entry point of the header is declared below, with the
//! same names, arity and types (tests/test_rust_attn_binding.py checks them against the header). All
//! pointers are device pointers; nothing waits for the device.
#![allow(dead_code)]

use std::ffi::{c_char, c_int, c_void};
use std::ptr;

use crate::qgemm::{check, Dtype, QgemmError, Status, Stream};

/// hq_attn_kind, of the workspace query.
#[repr(C)]
#[derive(Clone, Copy, Debug, PartialEq, Eq)]
pub enum AttnKind {
    Prompt = 1,
    Paged = 2,
    Shared = 3,
}

/// hq_attn_io: queries and outputs of a call, strides in elements.
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct AttnIo {
    pub q: *const c_void,
    pub o: *mut c_void,
    pub lse: *mut f32,
    pub q_row: i64,
    pub q_head: i64,
    pub o_row: i64,
    pub o_head: i64,
    pub rows: u32,
    pub heads: u32,
    pub head_dim: u32,
    pub dtype: Dtype,
    pub scale: f32,
}
const _: () = assert!(std::mem::size_of::<AttnIo>() == 80);

/// hq_kv_cache: a paged cache over the caller's memory.
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct KvCache {
    pub k: *mut c_void,
    pub v: *mut c_void,
    pub layer_stride: i64,
    pub page_stride: i64,
    pub head_stride: i64,
    pub token_stride: i64,
    pub layers: u32,
    pub pages: u32,
    pub kv_heads: u32,
    pub page_tokens: u32,
    pub head_dim: u32,
    pub dtype: Dtype,
    pub table: *mut i32,
    pub table_stride: i64,
    pub rows: u32,
    pub max_pages: u32,
    pub lens: *mut i32,
    pub refs: *mut i32,
    pub status: *mut u32,
    pub refused: *mut i32,
}
const _: () = assert!(std::mem::size_of::<KvCache>() == 128);

/// Faults that calls report in the cache's status word.
pub const CACHE_BAD_ROW: u32 = 1;
pub const CACHE_NO_PAGES: u32 = 2;
pub const CACHE_ROW_FULL: u32 = 4;
pub const CACHE_BAD_PAGE: u32 = 8;
/// Sequences of one cache call.
pub const CACHE_MAX_BATCH: u32 = 1024;

extern "C" {
    pub fn hq_attn_workspace_bytes(kind: AttnKind, rows: u32, seqs: u32, groups: u32, heads: u32, kv_heads: u32,
                                   head_dim: u32, max_keys: u32, max_prefix: u32, bytes: *mut usize) -> Status;
    pub fn hq_describe_attn(kind: AttnKind, rows: u32, seqs: u32, groups: u32, heads: u32, kv_heads: u32,
                            head_dim: u32, max_keys: u32, max_prefix: u32, buf: *mut c_char,
                            buf_len: usize) -> Status;
    pub fn hq_attn_prompt(io: *const AttnIo, k: *const c_void, k_row: i64, k_head: i64, v: *const c_void,
                          v_row: i64, v_head: i64, kv_heads: u32, total_k: u32, cu_q: *const i32,
                          cu_k: *const i32, seqs: u32, causal: c_int, max_k: u32, workspace: *mut c_void,
                          workspace_bytes: usize, stream: Stream) -> Status;
    pub fn hq_attn_paged(io: *const AttnIo, cache: *const KvCache, layer: u32, rows: *const i32,
                         cu_q: *const i32, seqs: u32, max_len: u32, workspace: *mut c_void,
                         workspace_bytes: usize, stream: Stream) -> Status;
    pub fn hq_attn_shared_prefix(io: *const AttnIo, cache: *const KvCache, layer: u32, rows: *const i32,
                                 seqs: u32, starts: *const i32, prefix_lens: *const i32, groups: u32,
                                 max_prefix: u32, max_len: u32, workspace: *mut c_void, workspace_bytes: usize,
                                 stream: Stream) -> Status;
    pub fn hq_cache_workspace_bytes(cache: *const KvCache, bytes: *mut usize) -> Status;
    pub fn hq_cache_reserve(cache: *const KvCache, rows: *const i32, counts: *const i32, n: u32,
                            stream: Stream) -> Status;
    pub fn hq_cache_append(cache: *const KvCache, layer: u32, k: *const c_void, k_row: i64, k_head: i64,
                           v: *const c_void, v_row: i64, v_head: i64, tokens: u32, rows: *const i32,
                           cu: *const i32, n: u32, stream: Stream) -> Status;
    pub fn hq_cache_fork(cache: *const KvCache, parents: *const i32, children: *const i32, n: u32,
                         workspace: *mut c_void, workspace_bytes: usize, stream: Stream) -> Status;
    pub fn hq_cache_free(cache: *const KvCache, rows: *const i32, n: u32, stream: Stream) -> Status;
    pub fn hq_cache_copy_pages(cache: *const KvCache, src: *const i32, dst: *const i32, n: u32,
                               stream: Stream) -> Status;
    pub fn hq_cache_compact(cache: *const KvCache, out_table: *mut i32, out_stride: i64, out_refs: *mut i32,
                            workspace: *mut c_void, workspace_bytes: usize, stream: Stream) -> Status;
}

/// Workspace bytes of fork and compact on this cache.
pub fn cache_workspace_bytes(cache: &KvCache) -> Result<usize, QgemmError> {
    let mut bytes = 0usize;
    // SAFETY: reads the descriptor alone and writes `bytes`.
    check(unsafe { hq_cache_workspace_bytes(cache, &mut bytes) })?;
    Ok(bytes)
}

/// One decode token a sequence over a layer of the cache: row `rows[i]` (device, or null: row i) of `seqs`.
///
/// # Safety
/// `io` and `cache` describe live device memory, `rows` holds `seqs` entries, the workspace `workspace_bytes`
/// bytes that were zero before its first use, until the work on `stream` is done.
pub unsafe fn decode(io: &AttnIo, cache: &KvCache, layer: u32, rows: *const i32, max_len: u32, workspace: *mut c_void,
                     workspace_bytes: usize, stream: Stream) -> Result<(), QgemmError> {
    // SAFETY: as the caller promises.
    check(unsafe { hq_attn_paged(io, cache, layer, rows, ptr::null(), io.rows, max_len, workspace, workspace_bytes, stream) })
}
