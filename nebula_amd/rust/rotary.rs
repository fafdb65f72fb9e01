//! Norms and rotary positions of query and key heads, to tensors or into the cache's pages (include/hq_rotary.h), for
//! `crates/nebula-hydrogen` (Linux / ROCm); beside qgemm.rs and attn.rs, whose types, errors and conventions it shares.
//! Every entry point of the header is declared below, with the same names, arity and types
//! (tests/test_rust_mixer_bindings.py checks them against the header). All pointers are device pointers; nothing waits
//! for the device.
#![allow(dead_code)]

use std::ffi::c_void;
use std::ptr;

use crate::attn::KvCache;
use crate::qgemm::{check, Dtype, QgemmError, Status, Stream};

/// hq_rotary_layout.
#[repr(C)]
#[derive(Clone, Copy, Debug, PartialEq, Eq)]
pub enum RotaryLayout {
    Half = 1,
    Interleaved = 2,
}

/// hq_rotary: how heads are rotated; `turns` is a device pointer to dim / 2 doubles.
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct Rotary {
    pub turns: *const f64,
    pub dim: u32,
    pub layout: RotaryLayout,
    pub scale: f32,
}
const _: () = assert!(std::mem::size_of::<Rotary>() == 24);

/// hq_rotary_heads: heads of a call, strides in elements.
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct RotaryHeads {
    pub r#in: *const c_void,
    pub out: *mut c_void,
    pub in_row: i64,
    pub in_head: i64,
    pub out_row: i64,
    pub out_head: i64,
    pub weight: *const f32,
    pub heads: u32,
    pub eps: f32,
}
const _: () = assert!(std::mem::size_of::<RotaryHeads>() == 64);

extern "C" {
    pub fn hq_rotate(rotary: *const Rotary, q: *const RotaryHeads, k: *const RotaryHeads, tokens: u32, head_dim: u32,
                     dtype: Dtype, positions: *const i32, stream: Stream) -> Status;
    pub fn hq_cache_append_rotated(cache: *const KvCache, layer: u32, rotary: *const Rotary, q: *const RotaryHeads,
                                   k: *const RotaryHeads, v: *const c_void, v_row: i64, v_head: i64, tokens: u32,
                                   rows: *const i32, cu: *const i32, n: u32, stream: Stream) -> Status;
}

/// One decode token a sequence: `k` normed and rotated into the pages of row `rows[i]` beside `v`, `q` to its output.
///
/// # Safety
/// Everything describes live device memory of `n` tokens, `rows` holds `n` entries, until the work on `stream` is done.
pub unsafe fn append_rotated(cache: &KvCache, layer: u32, rotary: &Rotary, q: &RotaryHeads, k: &RotaryHeads, v: *const c_void,
                             v_row: i64, v_head: i64, rows: *const i32, n: u32, stream: Stream) -> Result<(), QgemmError> {
    // SAFETY: as the caller promises.
    check(unsafe { hq_cache_append_rotated(cache, layer, rotary, q, k, v, v_row, v_head, n, rows, ptr::null(), n, stream) })
}
