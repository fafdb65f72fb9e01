//! A state space layer's mixer between its projections: the short causal convolution, the selective scan and the states
//! that sequences keep (include/hq_ssm.h), for `crates/nebula-hydrogen` (Linux / ROCm); beside qgemm.rs, whose types,
//! errors and conventions it shares. Every entry point of the header is declared below, with the same names, arity and types
//! (tests/test_rust_mixer_bindings.py checks them against the header). All pointers are device pointers; nothing waits
//! for the device.
#![allow(dead_code)]

use std::ffi::{c_char, c_int, c_void};
use std::ptr;

use crate::qgemm::{check, Dtype, QgemmError, Status, Stream};

/// Sequences of one call.
pub const SSM_MAX_BATCH: u32 = 1024;

/// hq_state_cache: the states of sequences over the caller's memory.
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct StateCache {
    pub conv: *mut c_void,
    pub ssm: *mut f32,
    pub conv_layer: i64,
    pub conv_row: i64,
    pub ssm_layer: i64,
    pub ssm_row: i64,
    pub layers: u32,
    pub rows: u32,
    pub channels: u32,
    pub width: u32,
    pub heads: u32,
    pub head_dim: u32,
    pub state_dim: u32,
    pub dtype: Dtype,
    pub status: *mut u32,
    pub refused: *const i32,
}
const _: () = assert!(std::mem::size_of::<StateCache>() == 96);

/// hq_ssm_io: inputs and outputs of a scan, strides in elements.
#[repr(C)]
#[derive(Clone, Copy, Debug)]
pub struct SsmIo {
    pub x: *const c_void,
    pub b: *const c_void,
    pub c: *const c_void,
    pub dt: *const c_void,
    pub z: *const c_void,
    pub y: *mut c_void,
    pub a: *const f32,
    pub d: *const f32,
    pub dt_bias: *const f32,
    pub x_row: i64,
    pub x_head: i64,
    pub b_row: i64,
    pub b_group: i64,
    pub c_row: i64,
    pub c_group: i64,
    pub dt_row: i64,
    pub z_row: i64,
    pub z_head: i64,
    pub y_row: i64,
    pub y_head: i64,
    pub tokens: u32,
    pub groups: u32,
    pub dt_f32: c_int,
    pub softplus: c_int,
}
const _: () = assert!(std::mem::size_of::<SsmIo>() == 176);

extern "C" {
    pub fn hq_ssm_conv(cache: *const StateCache, layer: u32, x: *const c_void, ldx: i64, y: *mut c_void, ldy: i64,
                       w: *const f32, bias: *const f32, silu: c_int, tokens: u32, rows: *const i32, held: *const i32,
                       cu: *const i32, n: u32, stream: Stream) -> Status;
    pub fn hq_ssm_workspace_bytes(tokens: u32, n: u32, cu: c_int, heads: u32, groups: u32, head_dim: u32, state_dim: u32,
                                  max_len: u32, bytes: *mut usize) -> Status;
    pub fn hq_describe_ssm(tokens: u32, n: u32, cu: c_int, heads: u32, groups: u32, head_dim: u32, state_dim: u32,
                           max_len: u32, buf: *mut c_char, buf_len: usize) -> Status;
    pub fn hq_ssm_scan(cache: *const StateCache, layer: u32, io: *const SsmIo, rows: *const i32, held: *const i32,
                       cu: *const i32, n: u32, max_len: u32, workspace: *mut c_void, workspace_bytes: usize,
                       stream: Stream) -> Status;
}

/// Workspace bytes of a scan of packed sequences (0: none).
pub fn workspace_bytes(tokens: u32, n: u32, heads: u32, groups: u32, head_dim: u32, state_dim: u32, max_len: u32) -> Result<usize, QgemmError> {
    let mut bytes = 0usize;
    // SAFETY: writes `bytes`.
    check(unsafe { hq_ssm_workspace_bytes(tokens, n, 1, heads, groups, head_dim, state_dim, max_len, &mut bytes) })?;
    Ok(bytes)
}

/// One decode token of each of the `io.tokens` sequences, which hold rows `rows[i]` of the states (device, or null: row i).
///
/// # Safety
/// `cache` and `io` describe live device memory, `rows` holds `io.tokens` entries, until the work on `stream` is done.
pub unsafe fn decode(cache: &StateCache, layer: u32, io: &SsmIo, rows: *const i32, stream: Stream) -> Result<(), QgemmError> {
    // SAFETY: as the caller promises; single tokens need no workspace.
    check(unsafe { hq_ssm_scan(cache, layer, io, rows, ptr::null(), ptr::null(), io.tokens, 1, ptr::null_mut(), 0, stream) })
}
