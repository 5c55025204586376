//! Rows as int8 with one scale each, and products of such rows (no counterpart in the reference's
//! kernel crate, which holds fp32 only). Operands are raw device pointers: activations are often
//! views into larger tensors.
use crate::device::HipStream;
use crate::error::{check, Result};
use crate::ffi;
use std::os::raw::c_void;

/// Element type of the activations of the 8-bit operators.
#[derive(Clone, Copy, Debug, PartialEq, Eq)]
pub enum Activation {
    F32,
    F16,
    BF16,
}

impl Activation {
    pub fn dtype(self) -> i32 {
        match self {
            Activation::F32 => ffi::RMLK_FLOAT,
            Activation::F16 => ffi::RMLK_FLOAT16,
            Activation::BF16 => ffi::RMLK_BFLOAT16,
        }
    }
}

/// `scale[r] = max|x[r]| / 127`, `q[r] = x[r] / scale[r]` to nearest even.
///
/// # Safety
/// The pointers are device memory of the sizes `include/rmlk_hip.h` gives, valid until the stream has run
/// the call.
pub unsafe fn quantize_rows(
    stream: &HipStream,
    kind: Activation,
    rows: usize,
    cols: usize,
    x: *const c_void,
    ldx: usize,
    q: *mut c_void,
    ldq: usize,
    scale: *mut f32,
) -> Result<()> {
    check(
        ffi::rmlk_hip_quantize_rows(
            stream.raw(),
            kind.dtype(),
            rows as i64,
            cols as i64,
            x,
            ldx as i64,
            q,
            ldq as i64,
            scale,
        ),
        "quantize_rows",
    )
}

/// `quantize_rows` of `x / sqrt(mean(x^2) + eps) * gamma`; with `b` (and `sum_out`) of `x + b`.
///
/// # Safety
/// As `quantize_rows`; `b` and `sum_out` are both null or both not.
pub unsafe fn rmsnorm_quantize_rows(
    stream: &HipStream,
    kind: Activation,
    rows: usize,
    cols: usize,
    x: *const c_void,
    b: *const c_void,
    gamma: *const f32,
    eps: f32,
    sum_out: *mut c_void,
    q: *mut c_void,
    ldq: usize,
    scale: *mut f32,
) -> Result<()> {
    check(
        ffi::rmlk_hip_rmsnorm_quantize_rows(
            stream.raw(),
            kind.dtype(),
            rows as i64,
            cols as i64,
            x,
            b,
            gamma,
            eps,
            sum_out,
            q,
            ldq as i64,
            scale,
        ),
        "rmsnorm_quantize_rows",
    )
}

/// Bytes of device scratch `matmul_int8` needs for a size (0 for most).
pub fn matmul_int8_workspace_size(m: usize, n: usize, k: usize) -> usize {
    unsafe { ffi::rmlk_hip_matmul_int8_workspace_size(m as i64, n as i64, k as i64) }
}

/// `c = (a . wt^T) * a_scale[row] * w_scale[column] (+ residual)`.
///
/// # Safety
/// As `quantize_rows`; the workspace belongs to the call until its kernels have run.
pub unsafe fn matmul_int8(
    stream: &HipStream,
    kind: Activation,
    m: usize,
    n: usize,
    k: usize,
    a: *const c_void,
    lda: usize,
    a_scale: *const f32,
    wt: *const c_void,
    ldw: usize,
    w_scale: *const f32,
    residual: *const c_void,
    ldr: usize,
    workspace: *mut c_void,
    workspace_bytes: usize,
    c: *mut c_void,
    ldc: usize,
) -> Result<()> {
    check(
        ffi::rmlk_hip_matmul_int8(
            stream.raw(),
            kind.dtype(),
            m as i64,
            n as i64,
            k as i64,
            a,
            lda as i64,
            a_scale,
            wt,
            ldw as i64,
            w_scale,
            residual,
            ldr as i64,
            workspace,
            workspace_bytes,
            c,
            ldc as i64,
        ),
        "matmul_int8",
    )
}
