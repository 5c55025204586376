//! Raw bindings of `include/rmlk_hip.h` (generated by `gen_ffi.py`; do not edit by hand).
#![allow(non_camel_case_types)]
use std::os::raw::{c_char, c_void};

pub const RMLK_MAX_RANK: usize = 8;
pub const RMLK_HIP_MATMUL_NOALLOC_SCRATCH_BYTES: usize = 32 << 20;

/// `hipStream_t`; null is the default stream.
pub type rmlk_stream_t = *mut c_void;

// rmlk_status
pub const RMLK_OK: i32 = 0;
pub const RMLK_ERR_BAD_RANK: i32 = -1;
pub const RMLK_ERR_UNSUPPORTED: i32 = -2;
pub const RMLK_ERR_NULL_POINTER: i32 = -3;
pub const RMLK_ERR_SIZE_MISMATCH: i32 = -4;
pub const RMLK_ERR_INVALID_ARGUMENT: i32 = -5;
pub const RMLK_ERR_WORKSPACE: i32 = -6;
pub const RMLK_ERR_TOO_LARGE: i32 = -7;
pub const RMLK_ERR_SCRATCH_LIMIT: i32 = -8;

// rmlk_dtype (ONNX TensorProto.DataType numbers)
pub const RMLK_FLOAT: i32 = 1;
pub const RMLK_UINT8: i32 = 2;
pub const RMLK_INT8: i32 = 3;
pub const RMLK_UINT16: i32 = 4;
pub const RMLK_INT16: i32 = 5;
pub const RMLK_INT32: i32 = 6;
pub const RMLK_INT64: i32 = 7;
pub const RMLK_BOOL: i32 = 9;
pub const RMLK_FLOAT16: i32 = 10;
pub const RMLK_DOUBLE: i32 = 11;
pub const RMLK_UINT32: i32 = 12;
pub const RMLK_UINT64: i32 = 13;
pub const RMLK_BFLOAT16: i32 = 16;

// rmlk_binary_op
pub const RMLK_ADD: i32 = 0;
pub const RMLK_SUB: i32 = 1;
pub const RMLK_MUL: i32 = 2;
pub const RMLK_DIV: i32 = 3;
pub const RMLK_POW: i32 = 4;
pub const RMLK_EQUAL: i32 = 5;
pub const RMLK_GREATER: i32 = 6;

// rmlk_unary_op
pub const RMLK_SQRT: i32 = 0;
pub const RMLK_NEG: i32 = 1;
pub const RMLK_SIN: i32 = 2;
pub const RMLK_COS: i32 = 3;
pub const RMLK_SIGMOID: i32 = 4;

// rmlk_scatter_reduction
pub const RMLK_SCATTER_NONE: i32 = 0;
pub const RMLK_SCATTER_ADD: i32 = 1;
pub const RMLK_SCATTER_MUL: i32 = 2;
pub const RMLK_SCATTER_MAX: i32 = 3;
pub const RMLK_SCATTER_MIN: i32 = 4;

// kinds of rmlk_hip_stream_yardstick
pub const RMLK_YARDSTICK_READ: i32 = 0;
pub const RMLK_YARDSTICK_COPY: i32 = 1;

/// Shape or stride vector passed by value.
#[repr(C)]
#[derive(Clone, Copy, Debug, Default)]
pub struct rmlk_dims {
    pub rank: i32,
    pub v: [i64; RMLK_MAX_RANK],
}

/// One stream of head rows (see `rmlk_hip_head_rows`).
#[repr(C)]
#[derive(Clone, Copy)]
pub struct rmlk_row_stream {
    pub shape: rmlk_dims,
    pub x_stride: rmlk_dims,
    pub x: *const c_void,
    pub cos: *const c_void,
    pub sin: *const c_void,
    pub cos_stride: rmlk_dims,
    pub sin_stride: rmlk_dims,
    pub out: *mut c_void,
    pub idx: *const i64,
    pub tuple_size: i32,
    pub data_shape: rmlk_dims,
    pub partials: i32,
    pub partial_stride: i64,
}

/// A paged int8 cache of keys and values (see `rmlk_hip_paged_append`).
#[repr(C)]
#[derive(Clone, Copy)]
pub struct rmlk_paged_cache {
    pub pages: i64,
    pub page_size: i32,
    pub kv_heads: i32,
    pub head_dim: i32,
    pub k: *mut c_void,
    pub v: *mut c_void,
    pub k_scale: *mut f32,
    pub v_scale: *mut f32,
}

/// The ragged sequences of one call over a paged cache.
#[repr(C)]
#[derive(Clone, Copy)]
pub struct rmlk_paged_batch {
    pub seqs: i64,
    pub rows: i64,
    pub max_new: i64,
    pub max_length: i64,
    pub table_stride: i64,
    pub first: *const i32,
    pub length: *const i32,
    pub page_table: *const i32,
}

#[repr(C)]
#[derive(Clone, Copy)]
pub struct rmlk_device_info {
    pub name: [c_char; 128],
    pub arch: [c_char; 64],
    pub compute_units: i32,
    pub wavefront_size: i32,
    pub lds_bytes_per_block: i32,
    pub clock_khz: i32,
    pub total_mem_bytes: i64,
}

extern "C" {
    pub fn rmlk_hip_binary(
        stream: rmlk_stream_t,
        op: i32,
        dtype_a: i32,
        dtype_b: i32,
        out_shape: *const rmlk_dims,
        a_stride: *const rmlk_dims,
        b_stride: *const rmlk_dims,
        a: *const c_void,
        b: *const c_void,
        out: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_where(
        stream: rmlk_stream_t,
        dtype: i32,
        out_shape: *const rmlk_dims,
        x_stride: *const rmlk_dims,
        y_stride: *const rmlk_dims,
        cond_stride: *const rmlk_dims,
        x: *const c_void,
        y: *const c_void,
        cond: *const c_void,
        out: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_unary(
        stream: rmlk_stream_t,
        op: i32,
        dtype: i32,
        n: i64,
        input: *const c_void,
        out: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_cast(
        stream: rmlk_stream_t,
        src_dtype: i32,
        dst_dtype: i32,
        n: i64,
        input: *const c_void,
        out: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_reduce_mean(
        stream: rmlk_stream_t,
        dtype: i32,
        in_shape: *const rmlk_dims,
        axes: *const i64,
        n_axes: i32,
        input: *const c_void,
        out: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_softmax(
        stream: rmlk_stream_t,
        dtype: i32,
        outer: i64,
        axis_len: i64,
        inner: i64,
        input: *const c_void,
        out: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_matmul(
        stream: rmlk_stream_t,
        dtype: i32,
        batch: i64,
        m: i64,
        n: i64,
        k: i64,
        a: *const c_void,
        lda: i64,
        stride_a: i64,
        trans_a: i32,
        b: *const c_void,
        ldb: i64,
        stride_b: i64,
        trans_b: i32,
        c: *mut c_void,
        ldc: i64,
        stride_c: i64,
        workspace: *mut c_void,
        workspace_bytes: usize,
    ) -> i32;
    pub fn rmlk_hip_matmul_workspace_size(dtype: i32, batch: i64, m: i64, n: i64, k: i64) -> usize;
    pub fn rmlk_hip_matmul_describe(
        dtype: i32,
        batch: i64,
        m: i64,
        n: i64,
        k: i64,
        buf: *mut c_char,
        size: i32,
    ) -> i32;
    pub fn rmlk_hip_matmul_noalloc(
        stream: rmlk_stream_t,
        dtype: i32,
        batch: i64,
        m: i64,
        n: i64,
        k: i64,
        a: *const c_void,
        lda: i64,
        stride_a: i64,
        trans_a: i32,
        b: *const c_void,
        ldb: i64,
        stride_b: i64,
        trans_b: i32,
        c: *mut c_void,
        ldc: i64,
        stride_c: i64,
    ) -> i32;
    pub fn rmlk_hip_transpose(
        stream: rmlk_stream_t,
        dtype: i32,
        in_shape: *const rmlk_dims,
        perm: *const i64,
        input: *const c_void,
        out: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_expand(
        stream: rmlk_stream_t,
        dtype: i32,
        in_shape: *const rmlk_dims,
        out_shape: *const rmlk_dims,
        input: *const c_void,
        out: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_slice(
        stream: rmlk_stream_t,
        dtype: i32,
        in_shape: *const rmlk_dims,
        starts: *const rmlk_dims,
        steps: *const rmlk_dims,
        out_shape: *const rmlk_dims,
        input: *const c_void,
        out: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_concat(
        stream: rmlk_stream_t,
        dtype: i32,
        in_shape: *const rmlk_dims,
        out_shape: *const rmlk_dims,
        axis: i32,
        axis_offset: i64,
        input: *const c_void,
        out: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_concat_many(
        stream: rmlk_stream_t,
        dtype: i32,
        n_inputs: i32,
        in_shapes: *const rmlk_dims,
        ins: *const *const c_void,
        out_shape: *const rmlk_dims,
        axis: i32,
        out: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_gather(
        stream: rmlk_stream_t,
        dtype: i32,
        idx_dtype: i32,
        data_shape: *const rmlk_dims,
        axis: i32,
        n_idx: i64,
        data: *const c_void,
        idx: *const c_void,
        out: *mut c_void,
        err_flag: *mut i32,
    ) -> i32;
    pub fn rmlk_hip_scatter_nd(
        stream: rmlk_stream_t,
        reduction: i32,
        dtype: i32,
        data_shape: *const rmlk_dims,
        n_tuples: i64,
        tuple_size: i32,
        idx: *const i64,
        updates: *const c_void,
        out: *mut c_void,
        err_flag: *mut i32,
    ) -> i32;
    pub fn rmlk_hip_scatter_nd_copy(
        stream: rmlk_stream_t,
        dtype: i32,
        data_shape: *const rmlk_dims,
        n_tuples: i64,
        tuple_size: i32,
        idx: *const i64,
        updates: *const c_void,
        data: *const c_void,
        out: *mut c_void,
        err_flag: *mut i32,
    ) -> i32;
    pub fn rmlk_hip_trilu(
        stream: rmlk_stream_t,
        dtype: i32,
        batch: i64,
        rows: i64,
        cols: i64,
        upper: i32,
        k: i64,
        input: *const c_void,
        out: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_rmsnorm(
        stream: rmlk_stream_t,
        dtype: i32,
        rows: i64,
        cols: i64,
        x: *const c_void,
        gamma: *const c_void,
        eps: f32,
        reciprocal_form: i32,
        out: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_add_rmsnorm(
        stream: rmlk_stream_t,
        dtype: i32,
        rows: i64,
        cols: i64,
        a: *const c_void,
        b: *const c_void,
        gamma: *const c_void,
        eps: f32,
        reciprocal_form: i32,
        sum_out: *mut c_void,
        out: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_scale_mask_softmax(
        stream: rmlk_stream_t,
        dtype: i32,
        shape: *const rmlk_dims,
        mask_stride: *const rmlk_dims,
        scale_is_mul: i32,
        scale: f32,
        x: *const c_void,
        mask: *const c_void,
        out: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_swiglu(
        stream: rmlk_stream_t,
        dtype: i32,
        n: i64,
        gate: *const c_void,
        up: *const c_void,
        out: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_gemv_partials_workspace_size(dtype: i32, n: i64, k: i64) -> usize;
    pub fn rmlk_hip_gemv_partials(
        stream: rmlk_stream_t,
        dtype: i32,
        n: i64,
        k: i64,
        x: *const c_void,
        b: *const c_void,
        ldb: i64,
        workspace: *mut c_void,
        workspace_bytes: usize,
        splits_out: *mut i32,
    ) -> i32;
    pub fn rmlk_hip_splitk_swiglu(
        stream: rmlk_stream_t,
        dtype: i32,
        n: i64,
        partials: *const c_void,
        splits: i32,
        slab: i64,
        gate_offset: i64,
        up_offset: i64,
        out: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_attention(
        stream: rmlk_stream_t,
        dtype: i32,
        batch: i64,
        kv_heads: i64,
        rep: i64,
        q_len: i64,
        kv_len: i64,
        head_dim: i64,
        q: *const c_void,
        k: *const c_void,
        v: *const c_void,
        mask: *const c_void,
        mask_stride: *const rmlk_dims,
        scale_is_mul: i32,
        scale: f32,
        out_seq_major: i32,
        out: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_attention_workspace_size(
        dtype: i32,
        batch: i64,
        kv_heads: i64,
        rep: i64,
        q_len: i64,
        kv_len: i64,
        head_dim: i64,
        mask_stride: *const rmlk_dims,
    ) -> usize;
    pub fn rmlk_hip_attention_ws(
        stream: rmlk_stream_t,
        dtype: i32,
        batch: i64,
        kv_heads: i64,
        rep: i64,
        q_len: i64,
        kv_len: i64,
        head_dim: i64,
        q: *const c_void,
        k: *const c_void,
        v: *const c_void,
        mask: *const c_void,
        mask_stride: *const rmlk_dims,
        scale_is_mul: i32,
        scale: f32,
        out_seq_major: i32,
        workspace: *mut c_void,
        workspace_bytes: usize,
        out: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_attention_map_size(
        dtype: i32,
        batch: i64,
        kv_heads: i64,
        rep: i64,
        q_len: i64,
        kv_len: i64,
        head_dim: i64,
        mask_stride: *const rmlk_dims,
    ) -> usize;
    pub fn rmlk_hip_attention_map(
        stream: rmlk_stream_t,
        dtype: i32,
        batch: i64,
        kv_heads: i64,
        rep: i64,
        q_len: i64,
        kv_len: i64,
        head_dim: i64,
        mask: *const c_void,
        mask_stride: *const rmlk_dims,
        map: *mut c_void,
        map_bytes: usize,
    ) -> i32;
    pub fn rmlk_hip_attention_mapped(
        stream: rmlk_stream_t,
        dtype: i32,
        batch: i64,
        kv_heads: i64,
        rep: i64,
        q_len: i64,
        kv_len: i64,
        head_dim: i64,
        q: *const c_void,
        k: *const c_void,
        v: *const c_void,
        mask: *const c_void,
        mask_stride: *const rmlk_dims,
        scale_is_mul: i32,
        scale: f32,
        out_seq_major: i32,
        map: *const c_void,
        map_bytes: usize,
        out: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_attention_mapped_pieces(
        stream: rmlk_stream_t,
        dtype: i32,
        batch: i64,
        kv_heads: i64,
        rep: i64,
        q_len: i64,
        kv_len: i64,
        head_dim: i64,
        q: *const c_void,
        k: *const c_void,
        v: *const c_void,
        mask: *const c_void,
        mask_stride: *const rmlk_dims,
        scale_is_mul: i32,
        scale: f32,
        map: *const c_void,
        map_bytes: usize,
        out: *mut c_void,
        out_pieces: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_attention_ws_pieces(
        stream: rmlk_stream_t,
        dtype: i32,
        batch: i64,
        kv_heads: i64,
        rep: i64,
        q_len: i64,
        kv_len: i64,
        head_dim: i64,
        q: *const c_void,
        k: *const c_void,
        v: *const c_void,
        mask: *const c_void,
        mask_stride: *const rmlk_dims,
        scale_is_mul: i32,
        scale: f32,
        workspace: *mut c_void,
        workspace_bytes: usize,
        out: *mut c_void,
        out_pieces: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_attention_few_rows_workspace_size(
        dtype: i32,
        batch: i64,
        kv_heads: i64,
        rep: i64,
        q_len: i64,
        kv_len: i64,
        head_dim: i64,
    ) -> usize;
    pub fn rmlk_hip_attention_few_rows(
        stream: rmlk_stream_t,
        dtype: i32,
        batch: i64,
        kv_heads: i64,
        rep: i64,
        q_len: i64,
        kv_len: i64,
        head_dim: i64,
        q: *const c_void,
        k: *const c_void,
        v: *const c_void,
        mask: *const c_void,
        mask_stride: *const rmlk_dims,
        scale_is_mul: i32,
        scale: f32,
        out_seq_major: i32,
        workspace: *mut c_void,
        workspace_bytes: usize,
        out: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_attention_few_rows_one_launch(
        stream: rmlk_stream_t,
        dtype: i32,
        batch: i64,
        kv_heads: i64,
        rep: i64,
        q_len: i64,
        kv_len: i64,
        head_dim: i64,
        q: *const c_void,
        k: *const c_void,
        v: *const c_void,
        mask: *const c_void,
        mask_stride: *const rmlk_dims,
        scale_is_mul: i32,
        scale: f32,
        out_seq_major: i32,
        workspace: *mut c_void,
        workspace_bytes: usize,
        counters: *mut i32,
        out: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_store_weights(
        stream: rmlk_stream_t,
        w_dtype: i32,
        n: i64,
        src: *const c_void,
        dst: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_weights_fit(
        stream: rmlk_stream_t,
        w_dtype: i32,
        n: i64,
        src: *const c_void,
        fits: *mut i32,
    ) -> i32;
    pub fn rmlk_hip_matmul_grouped_workspace_size(
        dtype: i32,
        m: i64,
        k: i64,
        groups: i32,
        widths: *const i64,
    ) -> usize;
    pub fn rmlk_hip_matmul_grouped(
        stream: rmlk_stream_t,
        dtype: i32,
        m: i64,
        k: i64,
        a: *const c_void,
        lda: i64,
        w_dtype: i32,
        b: *const c_void,
        ldb: i64,
        trans_b: i32,
        groups: i32,
        widths: *const i64,
        outs: *const *mut c_void,
        workspace: *mut c_void,
        workspace_bytes: usize,
    ) -> i32;
    pub fn rmlk_hip_matmul_swiglu(
        stream: rmlk_stream_t,
        dtype: i32,
        m: i64,
        n: i64,
        k: i64,
        a: *const c_void,
        lda: i64,
        w_dtype: i32,
        b: *const c_void,
        ldb: i64,
        trans_b: i32,
        gate_offset: i64,
        up_offset: i64,
        out: *mut c_void,
        ldc: i64,
    ) -> i32;
    pub fn rmlk_hip_gemv_kmajor(
        stream: rmlk_stream_t,
        dtype: i32,
        n: i64,
        k: i64,
        x: *const c_void,
        w_dtype: i32,
        wt: *const c_void,
        ldw: i64,
        y: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_gemv_kmajor_swiglu(
        stream: rmlk_stream_t,
        dtype: i32,
        n: i64,
        k: i64,
        x: *const c_void,
        w_dtype: i32,
        wt: *const c_void,
        ldw: i64,
        gate_row: i64,
        up_row: i64,
        y: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_gemv_kmajor_add(
        stream: rmlk_stream_t,
        dtype: i32,
        n: i64,
        k: i64,
        x: *const c_void,
        w_dtype: i32,
        wt: *const c_void,
        ldw: i64,
        residual: *const c_void,
        y: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_gemv_kmajor_normed(
        stream: rmlk_stream_t,
        dtype: i32,
        n: i64,
        k: i64,
        x: *const c_void,
        gamma: *const c_void,
        eps: f32,
        reciprocal_form: i32,
        w_dtype: i32,
        wt: *const c_void,
        ldw: i64,
        y: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_gemv_kmajor_swiglu_normed(
        stream: rmlk_stream_t,
        dtype: i32,
        n: i64,
        k: i64,
        x: *const c_void,
        gamma: *const c_void,
        eps: f32,
        reciprocal_form: i32,
        w_dtype: i32,
        wt: *const c_void,
        ldw: i64,
        gate_row: i64,
        up_row: i64,
        y: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_matmul_partials_workspace_size(dtype: i32, m: i64, n: i64, k: i64) -> usize;
    pub fn rmlk_hip_matmul_partials(
        stream: rmlk_stream_t,
        dtype: i32,
        m: i64,
        n: i64,
        k: i64,
        a: *const c_void,
        lda: i64,
        w_dtype: i32,
        b: *const c_void,
        ldb: i64,
        trans_b: i32,
        workspace: *mut c_void,
        workspace_bytes: usize,
        splits_out: *mut i32,
    ) -> i32;
    pub fn rmlk_hip_splitk_add_rmsnorm(
        stream: rmlk_stream_t,
        dtype: i32,
        rows: i64,
        cols: i64,
        partials: *const c_void,
        splits: i32,
        slab: i64,
        b: *const c_void,
        gamma: *const c_void,
        eps: f32,
        reciprocal_form: i32,
        sum_out: *mut c_void,
        out: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_bf16x3_pieces_size(m: i64, k: i64) -> usize;
    pub fn rmlk_hip_bf16x3_split(
        stream: rmlk_stream_t,
        m: i64,
        k: i64,
        a: *const c_void,
        lda: i64,
        pieces: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_bf16x3_splits(m: i64, n: i64, k: i64) -> i32;
    pub fn rmlk_hip_matmul_bf16x3(
        stream: rmlk_stream_t,
        m: i64,
        n: i64,
        k: i64,
        pieces: *const c_void,
        wt: *const c_void,
        ldw: i64,
        splits: i32,
        c: *mut c_void,
        ldc: i64,
        slab: i64,
    ) -> i32;
    pub fn rmlk_hip_matmul_bf16x3_swiglu(
        stream: rmlk_stream_t,
        m: i64,
        n: i64,
        k: i64,
        pieces: *const c_void,
        wt: *const c_void,
        ldw: i64,
        gate_row: i64,
        up_row: i64,
        out: *mut c_void,
        ldc: i64,
        out_pieces: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_rmsnorm_pieces(
        stream: rmlk_stream_t,
        rows: i64,
        cols: i64,
        partials: *const c_void,
        splits: i32,
        slab: i64,
        b: *const c_void,
        gamma: *const c_void,
        eps: f32,
        reciprocal_form: i32,
        sum_out: *mut c_void,
        out: *mut c_void,
        pieces: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_matmul_bf16x3_grouped(
        stream: rmlk_stream_t,
        m: i64,
        k: i64,
        pieces: *const c_void,
        wt: *const c_void,
        ldw: i64,
        groups: i32,
        widths: *const i64,
        outs: *const *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_rotary(
        stream: rmlk_stream_t,
        dtype: i32,
        shape: *const rmlk_dims,
        x_stride: *const rmlk_dims,
        cos_stride: *const rmlk_dims,
        sin_stride: *const rmlk_dims,
        x: *const c_void,
        cos: *const c_void,
        sin: *const c_void,
        out: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_head_rows(
        stream: rmlk_stream_t,
        dtype: i32,
        n_streams: i32,
        streams: *const rmlk_row_stream,
        err_flag: *mut i32,
    ) -> i32;
    pub fn rmlk_hip_gemv_kmajor_head_rows(
        stream: rmlk_stream_t,
        dtype: i32,
        k: i64,
        x: *const c_void,
        gamma: *const c_void,
        eps: f32,
        reciprocal_form: i32,
        w_dtype: i32,
        wt: *const c_void,
        ldw: i64,
        n_streams: i32,
        streams: *const rmlk_row_stream,
        first_col: *const i64,
        err_flag: *mut i32,
    ) -> i32;
    pub fn rmlk_hip_quantize_rows(
        stream: rmlk_stream_t,
        dtype: i32,
        rows: i64,
        cols: i64,
        x: *const c_void,
        ldx: i64,
        q: *mut c_void,
        ldq: i64,
        scale: *mut f32,
    ) -> i32;
    pub fn rmlk_hip_rmsnorm_quantize_rows(
        stream: rmlk_stream_t,
        dtype: i32,
        rows: i64,
        cols: i64,
        x: *const c_void,
        b: *const c_void,
        gamma: *const f32,
        eps: f32,
        sum_out: *mut c_void,
        q: *mut c_void,
        ldq: i64,
        scale: *mut f32,
    ) -> i32;
    pub fn rmlk_hip_matmul_int8_workspace_size(m: i64, n: i64, k: i64) -> usize;
    pub fn rmlk_hip_matmul_int8(
        stream: rmlk_stream_t,
        dtype: i32,
        m: i64,
        n: i64,
        k: i64,
        a: *const c_void,
        lda: i64,
        a_scale: *const f32,
        wt: *const c_void,
        ldw: i64,
        w_scale: *const f32,
        residual: *const c_void,
        ldr: i64,
        workspace: *mut c_void,
        workspace_bytes: usize,
        c: *mut c_void,
        ldc: i64,
    ) -> i32;
    pub fn rmlk_hip_paged_append(
        stream: rmlk_stream_t,
        dtype: i32,
        cache: *const rmlk_paged_cache,
        batch: *const rmlk_paged_batch,
        k: *const c_void,
        k_stride: i64,
        v: *const c_void,
        v_stride: i64,
        cos: *const f32,
        sin: *const f32,
        positions: i64,
        heads: i64,
        q: *const c_void,
        q_stride: i64,
        q_out: *mut c_void,
        err_flag: *mut i32,
    ) -> i32;
    pub fn rmlk_hip_paged_attention_workspace_size(
        dtype: i32,
        cache: *const rmlk_paged_cache,
        batch: *const rmlk_paged_batch,
        heads: i64,
    ) -> usize;
    pub fn rmlk_hip_paged_attention(
        stream: rmlk_stream_t,
        dtype: i32,
        cache: *const rmlk_paged_cache,
        batch: *const rmlk_paged_batch,
        heads: i64,
        q: *const c_void,
        q_stride: i64,
        scale_is_mul: i32,
        scale: f32,
        workspace: *mut c_void,
        workspace_bytes: usize,
        out: *mut c_void,
        err_flag: *mut i32,
    ) -> i32;
    pub fn rmlk_hip_batch_begin(stream: rmlk_stream_t) -> i32;
    pub fn rmlk_hip_batch_flush(stream: rmlk_stream_t) -> i32;
    pub fn rmlk_hip_batch_end(stream: rmlk_stream_t) -> i32;
    pub fn rmlk_hip_batch_collects(
        shape: *const rmlk_dims,
        n_in: i32,
        strides: *const rmlk_dims,
    ) -> i32;
    pub fn rmlk_hip_fill(
        stream: rmlk_stream_t,
        dtype: i32,
        n: i64,
        value: *const c_void,
        out: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_range(
        stream: rmlk_stream_t,
        dtype: i32,
        n: i64,
        start: *const c_void,
        delta: *const c_void,
        out: *mut c_void,
    ) -> i32;
    pub fn rmlk_hip_stream_yardstick(
        stream: rmlk_stream_t,
        kind: i32,
        bytes: usize,
        src: *const c_void,
        dst: *mut c_void,
        stamps: *mut u64,
    ) -> i32;
    pub fn rmlk_hip_issue_yardstick(
        stream: rmlk_stream_t,
        kind: i32,
        second_wavefront: i32,
        iterations: i32,
        blocks: i32,
        cycles: *mut u64,
    ) -> i32;
    pub fn rmlk_hip_write_small(
        stream: rmlk_stream_t,
        dst: *mut c_void,
        src: *const c_void,
        bytes: usize,
    ) -> i32;
    pub fn rmlk_hip_malloc(ptr: *mut *mut c_void, bytes: usize) -> i32;
    pub fn rmlk_hip_free(ptr: *mut c_void) -> i32;
    pub fn rmlk_hip_memcpy_htod(
        stream: rmlk_stream_t,
        dst: *mut c_void,
        src: *const c_void,
        bytes: usize,
    ) -> i32;
    pub fn rmlk_hip_memcpy_dtoh(
        stream: rmlk_stream_t,
        dst: *mut c_void,
        src: *const c_void,
        bytes: usize,
    ) -> i32;
    pub fn rmlk_hip_memcpy_dtod(
        stream: rmlk_stream_t,
        dst: *mut c_void,
        src: *const c_void,
        bytes: usize,
    ) -> i32;
    pub fn rmlk_hip_memcpy_dtod_many(
        stream: rmlk_stream_t,
        n_copies: i32,
        dsts: *const *mut c_void,
        srcs: *const *const c_void,
        bytes: *const usize,
    ) -> i32;
    pub fn rmlk_hip_memset(stream: rmlk_stream_t, dst: *mut c_void, byte: i32, bytes: usize) -> i32;
    pub fn rmlk_hip_stream_sync(stream: rmlk_stream_t) -> i32;
    pub fn rmlk_hip_device_info(device: i32, info: *mut rmlk_device_info) -> i32;
    pub fn rmlk_hip_status_string(status: i32) -> *const c_char;
    pub fn rmlk_hip_version() -> *const c_char;
}
