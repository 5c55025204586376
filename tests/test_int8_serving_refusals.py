"""Calls of the 8-bit serving operators that the header rules out answer with the documented status before anything
is launched: the entry points check their arguments on the host, so no GPU is needed (the addresses handed over
are never read)."""
import ctypes
import os

import pytest

import rmlk_amd
from rmlk_amd import _lib

OK, UNSUPPORTED, NULL_POINTER, SIZE_MISMATCH, INVALID_ARGUMENT, WORKSPACE, TOO_LARGE = 0, -2, -3, -4, -5, -6, -7
FLOAT, INT8, FLOAT16, DOUBLE, BFLOAT16 = 1, 3, 10, 11, 16
P = 1 << 20           # a 16-byte aligned address that nothing may touch


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(rmlk_amd.library_path()):
        pytest.fail(f"{rmlk_amd.library_path()} is not built: run `make -C rmlk_amd/csrc`")
    return _lib.lib()


def _cache(**kw):
    f = dict(pages=10, page_size=16, kv_heads=2, head_dim=64, k=P, v=P, k_scale=P, v_scale=P)
    f.update(kw)
    return _lib.PagedCacheStruct(*[f[n] for n, _ in _lib.PagedCacheStruct._fields_])


def _batch(**kw):
    f = dict(seqs=2, rows=4, max_new=3, max_length=40, table_stride=5, first=P, length=P, page_table=P)
    f.update(kw)
    return _lib.PagedBatchStruct(*[f[n] for n, _ in _lib.PagedBatchStruct._fields_])


def test_quantize_rows(L):
    def call(dtype=FLOAT, rows=4, cols=40, x=P, ldx=40, q=P, ldq=48, scale=P):
        return L.rmlk_hip_quantize_rows(None, dtype, rows, cols, x, ldx, q, ldq, scale)
    for bad in (DOUBLE, INT8, 99):
        assert call(dtype=bad) == UNSUPPORTED
    assert call(rows=-1) == INVALID_ARGUMENT and call(cols=-1) == INVALID_ARGUMENT
    assert call(ldq=47) == UNSUPPORTED and call(q=P + 8) == UNSUPPORTED
    assert call(ldq=32) == SIZE_MISMATCH and call(ldx=39) == SIZE_MISMATCH
    assert call(x=0) == NULL_POINTER and call(q=0) == NULL_POINTER and call(scale=0) == NULL_POINTER
    assert call(cols=1 << 30, ldx=1 << 30, ldq=1 << 30) == TOO_LARGE
    assert call(rows=0, x=0, scale=0) == OK and call(cols=0, x=0, scale=0) == OK


def test_rmsnorm_quantize_rows(L):
    def call(dtype=FLOAT, rows=4, cols=40, x=P, b=P, gamma=P, s=P, q=P, ldq=48, scale=P):
        return L.rmlk_hip_rmsnorm_quantize_rows(None, dtype, rows, cols, x, b, gamma, 1e-5, s, q, ldq, scale)
    assert call(dtype=DOUBLE) == UNSUPPORTED
    assert call(rows=-1) == INVALID_ARGUMENT
    assert call(ldq=40) == UNSUPPORTED and call(ldq=32) == SIZE_MISMATCH
    for name in ("x", "gamma", "q", "scale"):
        assert call(**{name: 0}) == NULL_POINTER
    assert call(b=0) == NULL_POINTER and call(s=0) == NULL_POINTER      # both or neither
    assert call(rows=0, x=0) == OK


def test_matmul_int8(L):
    def call(dtype=FLOAT, m=70, n=100, k=200, a=P, lda=208, sa=P, w=P, ldw=208, sw=P, res=0, ldr=0, ws=0, wsb=0, c=P,
             ldc=100):
        return L.rmlk_hip_matmul_int8(None, dtype, m, n, k, a, lda, sa, w, ldw, sw, res, ldr, ws, wsb, c, ldc)
    assert call(dtype=DOUBLE) == UNSUPPORTED and call(dtype=INT8) == UNSUPPORTED
    for name in ("m", "n", "k"):
        assert call(**{name: -1}) == INVALID_ARGUMENT
    assert call(res=P, ldr=-1) == INVALID_ARGUMENT
    for name in ("a", "sa", "w", "sw", "c"):
        assert call(**{name: 0}) == NULL_POINTER
    assert call(lda=192) == SIZE_MISMATCH and call(ldw=192) == SIZE_MISMATCH and call(ldc=99) == SIZE_MISMATCH
    assert call(res=P, ldr=99) == SIZE_MISMATCH
    assert call(lda=201) == UNSUPPORTED and call(ldw=216) == UNSUPPORTED
    assert call(a=P + 4) == UNSUPPORTED and call(w=P + 1) == UNSUPPORTED
    assert call(k=131072, lda=131072, ldw=131072) == TOO_LARGE
    assert call(lda=1 << 23) == TOO_LARGE
    need = L.rmlk_hip_matmul_int8_workspace_size(64, 512, 8192)
    assert need > 0
    split = dict(m=64, n=512, k=8192, lda=8192, ldw=8192, ldc=512)
    assert call(**split) == NULL_POINTER
    assert call(**split, ws=P + 8, wsb=need) == UNSUPPORTED
    assert call(**split, ws=P, wsb=need - 1) == WORKSPACE
    assert call(m=0, a=0, c=0) == OK and call(n=0, w=0, c=0) == OK
    assert L.rmlk_hip_matmul_int8_workspace_size(0, 5, 5) == 0
    assert L.rmlk_hip_matmul_int8_workspace_size(5, 5, -5) == 0


@pytest.mark.parametrize("which", ["append", "attention"])
def test_paged_structs(L, which):
    def call(cache=None, batch=None, dtype=FLOAT):
        c = _cache() if cache is None else cache
        b = _batch() if batch is None else batch
        c = ctypes.byref(c) if c else None
        b = ctypes.byref(b) if b else None
        if which == "append":
            return L.rmlk_hip_paged_append(None, dtype, c, b, P, 128, P, 128, 0, 0, 0, 0, 0, 0, 0, 0)
        return L.rmlk_hip_paged_attention(None, dtype, c, b, 4, P, 256, 1, 0.125, 0, 0, P, 0)
    assert call(cache=False) == NULL_POINTER and call(batch=False) == NULL_POINTER
    assert call(dtype=DOUBLE) == UNSUPPORTED
    for f in (dict(page_size=8), dict(page_size=24), dict(page_size=256), dict(page_size=0), dict(head_dim=32),
              dict(head_dim=96), dict(head_dim=256), dict(k=P + 8), dict(v=P + 4)):
        assert call(cache=_cache(**f)) == UNSUPPORTED, f
    for f in (dict(pages=-1), dict(pages=0), dict(kv_heads=0), dict(kv_heads=-2)):
        assert call(cache=_cache(**f)) == INVALID_ARGUMENT, f
    for name in ("k", "v", "k_scale", "v_scale"):
        assert call(cache=_cache(**{name: 0})) == NULL_POINTER, name
    for f in (dict(seqs=-1), dict(rows=-1), dict(max_new=-1), dict(max_length=-1), dict(table_stride=-1)):
        assert call(batch=_batch(**f)) == INVALID_ARGUMENT, f
    for f in (dict(seqs=1 << 16), dict(rows=1 << 30), dict(max_new=1 << 30), dict(max_length=1 << 30)):
        assert call(batch=_batch(**f)) == TOO_LARGE, f
    assert call(cache=_cache(pages=1 << 31)) == TOO_LARGE
    for name in ("first", "length", "page_table"):
        assert call(batch=_batch(**{name: 0})) == NULL_POINTER, name
    assert call(batch=_batch(seqs=0, first=0, length=0, page_table=0)) == OK
    assert call(batch=_batch(rows=0, first=0, length=0, page_table=0)) == OK


def test_paged_append(L):
    def call(k=P, ks=128, v=P, vs=128, cos=P, sin=P, positions=50, heads=4, q=P, qs=256, q_out=P, dtype=FLOAT):
        return L.rmlk_hip_paged_append(None, dtype, ctypes.byref(_cache()), ctypes.byref(_batch()), k, ks, v, vs, cos, sin,
                                       positions, heads, q, qs, q_out, 0)
    assert call(k=0) == NULL_POINTER and call(v=0) == NULL_POINTER
    assert call(cos=0) == NULL_POINTER and call(sin=0) == NULL_POINTER          # both or neither
    assert call(q=0) == NULL_POINTER and call(q_out=0) == NULL_POINTER
    assert call(positions=-1) == INVALID_ARGUMENT and call(heads=0) == INVALID_ARGUMENT
    assert call(heads=3) == SIZE_MISMATCH
    assert call(ks=127) == SIZE_MISMATCH and call(vs=64) == SIZE_MISMATCH and call(qs=255) == SIZE_MISMATCH
    assert call(ks=130) == UNSUPPORTED and call(vs=129) == UNSUPPORTED and call(qs=258) == UNSUPPORTED
    assert call(ks=132, dtype=FLOAT16) == UNSUPPORTED
    for name in ("k", "v", "q", "q_out", "cos", "sin"):
        assert call(**{name: P + 4}) == UNSUPPORTED, name


def test_paged_attention(L):
    def call(dtype=FLOAT, heads=4, q=P, qs=256, ws=0, wsb=0, out=P, **batch):
        return L.rmlk_hip_paged_attention(None, dtype, ctypes.byref(_cache(pages=4000)), ctypes.byref(_batch(**batch)), heads,
                                          q, qs, 1, 0.125, ws, wsb, out, 0)
    assert call(q=0) == NULL_POINTER and call(out=0) == NULL_POINTER
    assert call(heads=0) == INVALID_ARGUMENT and call(heads=3) == SIZE_MISMATCH and call(heads=1 << 16) == TOO_LARGE
    assert call(qs=255) == SIZE_MISMATCH and call(qs=257) == UNSUPPORTED
    assert call(q=P + 8) == UNSUPPORTED and call(out=P + 8) == UNSUPPORTED
    long = dict(max_length=30000, table_stride=2000)
    need = L.rmlk_hip_paged_attention_workspace_size(FLOAT, ctypes.byref(_cache(pages=4000)), ctypes.byref(_batch(**long)), 4)
    assert need > 0
    assert call(**long) == NULL_POINTER
    assert call(**long, ws=P + 8, wsb=need) == UNSUPPORTED
    assert call(**long, ws=P, wsb=need - 1) == WORKSPACE
    size = L.rmlk_hip_paged_attention_workspace_size
    assert size(DOUBLE, ctypes.byref(_cache()), ctypes.byref(_batch(**long)), 4) == 0
    assert size(FLOAT, ctypes.byref(_cache()), ctypes.byref(_batch(seqs=0, **long)), 4) == 0
    assert size(FLOAT, None, None, 4) == 0


def test_sizes_beyond_a_launch(L):
    """More channels than a launch has work items for."""
    n = (1 << 27) + 16
    assert L.rmlk_hip_matmul_int8(None, FLOAT, 1, n, 16, P, 16, P, P, 16, P, 0, 0, 0, 0, P, n) == TOO_LARGE


def test_paged_append_rotation_in_place_needs_dense_rows(L):
    """q_out is dense: over a q whose rows lie apart it would overwrite rows that are still to be read."""
    def call(q_out, stride):
        return L.rmlk_hip_paged_append(None, FLOAT, ctypes.byref(_cache()), ctypes.byref(_batch(rows=4)), P, 128, P, 128, 0, 0,
                                       0, 4, P, stride, q_out, 0)
    assert call(P, 512) == INVALID_ARGUMENT and call(P, 260) == INVALID_ARGUMENT


def test_paged_attention_workspace_without_new_tokens(L):
    """max_new 0 (a padded batch): an answer, whatever the lengths."""
    size = L.rmlk_hip_paged_attention_workspace_size
    for max_length in (0, 40, 5000, 100000):
        for seqs in (1, 2, 70):
            b = _batch(seqs=seqs, max_new=0, max_length=max_length, table_stride=7000)
            assert size(FLOAT, ctypes.byref(_cache()), ctypes.byref(b), 4) >= 0
