#!/usr/bin/env python3
"""Writes src/ffi.rs from include/rmlk_hip.h: one `extern "C"` declaration per entry point.

    python hip/gen_ffi.py            # rewrite hip/src/ffi.rs
    python hip/gen_ffi.py --check    # exit 1 when the checked-in file is out of date

The types of the header map one to one (int32_t -> i32, size_t -> usize, `const T *` -> *const T,
`T *` -> *mut T); structs and constants are written out by hand in PREAMBLE below and checked
against the header by tests/test_hip_crate.py.
"""
import os
import re
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
HEADER = os.path.join(HERE, "..", "include", "rmlk_hip.h")
OUT = os.path.join(HERE, "src", "ffi.rs")

PREAMBLE = '''//! Raw bindings of `include/rmlk_hip.h` (generated by `gen_ffi.py`; do not edit by hand).
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

'''

SCALARS = {
    "int32_t": "i32", "int64_t": "i64", "size_t": "usize", "float": "f32", "double": "f64",
    "rmlk_stream_t": "rmlk_stream_t", "void": "c_void", "char": "c_char", "uint8_t": "u8", "uint64_t": "u64",
    "rmlk_dims": "rmlk_dims", "rmlk_row_stream": "rmlk_row_stream", "rmlk_device_info": "rmlk_device_info",
    "rmlk_paged_cache": "rmlk_paged_cache", "rmlk_paged_batch": "rmlk_paged_batch",
}
RESERVED = {"in": "input", "type": "kind", "ref": "reference", "fn": "func", "mod": "modulus"}


def rust_type(c_type: str) -> str:
    """`const void *const *` -> `*const *const c_void` and the like."""
    toks = c_type.replace("*", " * ").split()
    base, i, const_base = None, 0, False
    while i < len(toks) and toks[i] != "*":
        if toks[i] == "const":
            const_base = True
        else:
            base = toks[i]
        i += 1
    if base not in SCALARS:
        raise ValueError(f"unmapped C type `{c_type}`")
    ty = SCALARS[base]
    pointee_const = const_base
    while i < len(toks):
        assert toks[i] == "*", c_type
        i += 1
        ty = ("*const " if pointee_const else "*mut ") + ty
        pointee_const = False
        if i < len(toks) and toks[i] == "const":
            pointee_const = True
            i += 1
    return ty


def prototypes(text: str):
    text = re.sub(r"/\*.*?\*/", " ", text, flags=re.S)
    text = re.sub(r"^\s*#.*$", " ", text, flags=re.M)
    pat = re.compile(r"((?:const\s+)?[A-Za-z_0-9]+\s*\*?)\s*(rmlk_hip_\w+)\s*\(([^()]*)\)\s*$", re.S)
    for stmt in re.split(r"[;{}]", text):
        m = pat.search(stmt)
        if not m:
            continue
        ret, name, params = m.group(1).strip(), m.group(2), m.group(3).strip()
        args = []
        if params and params != "void":
            for p in params.split(","):
                p = " ".join(p.split())
                pm = re.match(r"(.*?)(\w+)$", p)
                ctype, pname = pm.group(1).strip(), pm.group(2)
                args.append((RESERVED.get(pname, pname), rust_type(ctype)))
        yield name, (None if ret == "void" else rust_type(ret)), args


def render() -> str:
    with open(HEADER) as f:
        text = f.read()
    lines = [PREAMBLE, 'extern "C" {\n']
    for name, ret, args in prototypes(text):
        sig = ", ".join(f"{n}: {t}" for n, t in args)
        decl = f"    pub fn {name}({sig})" + (f" -> {ret}" if ret else "") + ";"
        if len(decl) > 100:
            body = ",\n".join(f"        {n}: {t}" for n, t in args)
            decl = f"    pub fn {name}(\n{body},\n    )" + (f" -> {ret}" if ret else "") + ";"
        lines.append(decl + "\n")
    lines.append("}\n")
    return "".join(lines)


def main() -> int:
    new = render()
    if "--check" in sys.argv:
        with open(OUT) as f:
            return 0 if f.read() == new else 1
    with open(OUT, "w") as f:
        f.write(new)
    return 0


if __name__ == "__main__":
    sys.exit(main())
