//! A paged cache of keys and values held in 8 bits: appending to it and attention over it (no
//! counterpart in the reference, whose cache is a dense fp32 tensor that ScatterND writes,
//! runtime/src/providers/cuda/backend/scatter_nd.rs:78-225).
use crate::device::HipStream;
use crate::error::{check, Result};
use crate::ffi;
use crate::kernels::int8::Activation;
use std::os::raw::c_void;

pub use crate::ffi::{rmlk_paged_batch as PagedBatch, rmlk_paged_cache as PagedCache};

/// Rows of queries that are rotated along with the keys.
#[derive(Clone, Copy)]
pub struct Queries {
    pub heads: usize,
    pub q: *const c_void,
    pub q_stride: usize,
    pub q_out: *mut c_void,
}

/// Rotary tables, `[positions, head_dim]` floats each.
#[derive(Clone, Copy)]
pub struct Tables {
    pub cos: *const f32,
    pub sin: *const f32,
    pub positions: usize,
}

/// Appends the new tokens' keys and values (rows `k_stride` / `v_stride` elements apart).
///
/// # Safety
/// The pointers are device memory of the sizes `include/rmlk_hip.h` gives, valid until the stream has run
/// the call; a page that receives tokens belongs to one sequence of the call.
pub unsafe fn append(
    stream: &HipStream,
    kind: Activation,
    cache: &PagedCache,
    batch: &PagedBatch,
    k: *const c_void,
    k_stride: usize,
    v: *const c_void,
    v_stride: usize,
    tables: Option<Tables>,
    queries: Option<Queries>,
    err_flag: *mut i32,
) -> Result<()> {
    let t = tables.unwrap_or(Tables { cos: std::ptr::null(), sin: std::ptr::null(), positions: 0 });
    let q = queries.unwrap_or(Queries { heads: 0, q: std::ptr::null(), q_stride: 0, q_out: std::ptr::null_mut() });
    check(
        ffi::rmlk_hip_paged_append(
            stream.raw(),
            kind.dtype(),
            cache,
            batch,
            k,
            k_stride as i64,
            v,
            v_stride as i64,
            t.cos,
            t.sin,
            t.positions as i64,
            q.heads as i64,
            q.q,
            q.q_stride as i64,
            q.q_out,
            err_flag,
        ),
        "paged_append",
    )
}

/// Bytes of device scratch `attention` needs.
pub fn attention_workspace_size(kind: Activation, cache: &PagedCache, batch: &PagedBatch, heads: usize) -> usize {
    unsafe { ffi::rmlk_hip_paged_attention_workspace_size(kind.dtype(), cache, batch, heads as i64) }
}

/// Causal attention of the batch's rows over the cached tokens of their sequences; scores are multiplied
/// by `scale`.
///
/// # Safety
/// As `append`; the workspace belongs to the call until its kernels have run.
pub unsafe fn attention(
    stream: &HipStream,
    kind: Activation,
    cache: &PagedCache,
    batch: &PagedBatch,
    heads: usize,
    q: *const c_void,
    q_stride: usize,
    scale: f32,
    workspace: *mut c_void,
    workspace_bytes: usize,
    out: *mut c_void,
    err_flag: *mut i32,
) -> Result<()> {
    check(
        ffi::rmlk_hip_paged_attention(
            stream.raw(),
            kind.dtype(),
            cache,
            batch,
            heads as i64,
            q,
            q_stride as i64,
            1,
            scale,
            workspace,
            workspace_bytes,
            out,
            err_flag,
        ),
        "paged_attention",
    )
}
