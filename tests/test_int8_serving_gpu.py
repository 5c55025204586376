"""The 8-bit serving operators on the GPU against their definitions in float64 (int8_reference.py).

Where the result is integers and scales (row quantisation, the cache), it is compared for equality: the
kernels decide roundings as in exact arithmetic. Where it is a float, the tolerance counts the roundings:
u = 2^-24 per float operation, and half a step of the output type, u_out (2^-24, 2^-11, 2^-8)."""
import numpy as np
import pytest

import int8_reference as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24
U_OUT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}    # the step among subnormals


def _k():
    from rmlk_amd import kernels
    return kernels


def _dev(a, device, kind=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).to(device)
    return t.to(kind) if kind is not None else t


def _f64(t):
    return t.double().cpu().numpy()


def _padded(cols):
    return (cols + 15) // 16 * 16


def _check_rows(q, scale, y, cols, exact_scale):
    """q, scale of the kernel against the real rows y; integers are compared where y / scale is not within 1e-9
    of a border (a double evaluation of the norm cannot decide there); scales to one rounding."""
    want_q, want_s = ref.quantize_rows(y)
    got_q, got_s = q.cpu().numpy(), scale.cpu().numpy()
    nan = np.isnan(want_s)
    assert np.array_equal(np.isnan(got_s), nan)
    if exact_scale:
        assert np.array_equal(got_s[~nan], want_s[~nan])
    else:
        np.testing.assert_allclose(got_s[~nan], want_s[~nan], rtol=2 * U, atol=0)
    safe = np.ones(y.shape, bool)
    if not exact_scale:
        with np.errstate(all="ignore"):
            z = np.abs(y / np.where(want_s > 0, want_s, 1).astype(np.float64)[:, None])
            safe = ~(np.abs(z - np.floor(z) - 0.5) < 1e-9)
    assert np.array_equal(got_q[:, :cols][safe], want_q[safe])
    assert not got_q[:, cols:_padded(cols)].any()


# ---- rows to int8 ---------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 17), (1, 2048), (5, 4096), (2, 8200), (3, 16384), (2, 16392),
                                       (2, 33000), (300, 64)])
def test_quantize_rows(device, kind, rows, cols):
    rng = np.random.default_rng(rows * 100003 + cols)
    x = _dev(rng.standard_normal((rows, cols)).astype(np.float32) * 3, device, TYPES[kind])
    q = torch.full((rows, _padded(cols) + 32), 77, dtype=torch.int8, device=device)
    scale = torch.full((rows,), -1.0, device=device)
    _k().quantize_rows(x, q, scale)
    _check_rows(q, scale, _f64(x), cols, True)
    assert bool((q[:, _padded(cols):] == 77).all())


@pytest.mark.parametrize("kind", TYPES)
def test_quantize_rows_that_lie_apart_and_odd_starts(device, kind):
    """Rows of a wider tensor, starting at an element that no wide load can start at."""
    rng = np.random.default_rng(5)
    wide = _dev(rng.standard_normal((7, 700)).astype(np.float32), device, TYPES[kind])
    for first, cols in ((0, 256), (3, 256), (1, 511), (8, 130)):
        x = wide[:, first:first + cols]
        q = torch.zeros(7, _padded(cols), dtype=torch.int8, device=device)
        scale = torch.zeros(7, device=device)
        _k().quantize_rows(x, q, scale)
        _check_rows(q, scale, _f64(x), cols, True)


def test_quantize_rows_at_borders(device):
    """Values at and next to k + 1/2 steps, scales that are no powers of two."""
    rows = []
    for top in (127.0, 1.0, 0.1, 3.3e-5, 1e30, 2.0 ** -99):
        s = np.float32(np.float32(top) / np.float32(127))
        steps = np.arange(-126, 127) + 0.5
        v = (steps * np.float64(s)).astype(np.float32)
        up, down = np.nextafter(v, np.float32(np.inf)), np.nextafter(v, np.float32(-np.inf))
        rows.append(np.concatenate([[np.float32(top)], v, up, down]))
    x = np.stack(rows).astype(np.float32)
    q = torch.zeros(x.shape[0], _padded(x.shape[1]), dtype=torch.int8, device=device)
    scale = torch.zeros(x.shape[0], device=device)
    _k().quantize_rows(_dev(x, device), q, scale)
    _check_rows(q, scale, x.astype(np.float64), x.shape[1], True)


def test_quantize_rows_that_are_zero_tiny_or_not_finite(device):
    x = np.zeros((8, 40), np.float32)
    x[1, 3], x[2, 5], x[3, 39] = np.nan, np.inf, -np.inf
    x[4, 0] = 2.0 ** -101          # below what a row can hold
    x[5, :2] = 2.0 ** -100, -2.0 ** -107
    x[6] = 3.4e38
    x[7, 0], x[7, 1] = 1e-45, -1e-45
    q = torch.full((8, 48), 9, dtype=torch.int8, device=device)
    scale = torch.zeros(8, device=device)
    _k().quantize_rows(_dev(x, device), q, scale)
    _check_rows(q, scale, x.astype(np.float64), 40, True)
    assert scale[4].item() == 0 and not q[4].any() and not q[1].any() and not q[0].any()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("with_add", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 2048), (3, 17), (4, 4096), (2, 8200), (2, 20000), (40, 512)])
def test_rmsnorm_quantize_rows(device, kind, with_add, rows, cols):
    rng = np.random.default_rng(cols)
    x = _dev(rng.standard_normal((rows, cols)).astype(np.float32), device, TYPES[kind])
    add = _dev(rng.standard_normal((rows, cols)).astype(np.float32), device, TYPES[kind]) if with_add else None
    gamma = rng.uniform(0.5, 1.5, cols).astype(np.float32)
    q = torch.zeros(rows, _padded(cols), dtype=torch.int8, device=device)
    scale = torch.zeros(rows, device=device)
    total = torch.zeros_like(x) if with_add else None
    _k().rmsnorm_quantize_rows(x, _dev(gamma, device), 1e-5, q, scale, add=add, sum_out=total)
    s = x
    if with_add:
        s = (x.float() + add.float()).to(x.dtype)
        assert torch.equal(total, s)
    _check_rows(q, scale, ref.rmsnorm(_f64(s), gamma, 1e-5), cols, False)


def test_rmsnorm_quantize_rows_in_place_and_not_finite(device):
    rng = np.random.default_rng(8)
    x = rng.standard_normal((4, 96)).astype(np.float32)
    x[1, 5], x[2, 7] = np.nan, np.inf
    x[3] = 0
    a, b = _dev(x, device), _dev(np.ones_like(x) * 0, device)
    gamma = np.ones(96, np.float32)
    q = torch.zeros(4, 96, dtype=torch.int8, device=device)
    scale = torch.zeros(4, device=device)
    _k().rmsnorm_quantize_rows(a, _dev(gamma, device), 1e-5, q, scale, add=b, sum_out=a)   # the sum over its operand
    with np.errstate(all="ignore"):
        y = ref.rmsnorm(x.astype(np.float64), gamma, 1e-5)
    y[1] = y[2] = np.nan
    _check_rows(q, scale, y, 96, False)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("cols", [4099, 8201, 16400])
def test_rmsnorm_quantize_rows_long_odd_rows_in_place(device, kind, cols):
    """Rows that start at odd addresses and are read twice, the sum over its first or its second operand."""
    rng = np.random.default_rng(cols)
    for over in (0, 1):
        ops = [_dev(rng.standard_normal((3, cols)).astype(np.float32), device, TYPES[kind]) for _ in range(2)]
        total = (ops[0].float() + ops[1].float()).to(TYPES[kind])
        gamma = rng.uniform(0.5, 1.5, cols).astype(np.float32)
        q = torch.full((3, _padded(cols)), 5, dtype=torch.int8, device=device)
        scale = torch.zeros(3, device=device)
        _k().rmsnorm_quantize_rows(ops[0], _dev(gamma, device), 1e-5, q, scale, add=ops[1], sum_out=ops[over])
        assert torch.equal(ops[over], total)
        _check_rows(q, scale, ref.rmsnorm(_f64(total), gamma, 1e-5), cols, False)


# ---- int8 products --------------------------------------------------------------------------------

def _product_case(device, kind, m, n, k, residual, seed, lda=None, values=127):
    rng = np.random.default_rng(seed)
    lda = lda or _padded(k)
    # what lies behind k in a row must not matter
    a = rng.integers(-values - 1, values + 1, (m, lda)).astype(np.int8)
    w = rng.integers(-values - 1, values + 1, (n, _padded(k))).astype(np.int8)
    sa = rng.uniform(0.001, 0.1, m).astype(np.float32)
    sw = rng.uniform(0.0001, 0.01, n).astype(np.float32)
    res = None
    if residual == "rows":
        res = _dev(rng.standard_normal((m, n)).astype(np.float32), device, TYPES[kind])
    elif residual == "bias":
        res = _dev(rng.standard_normal(n).astype(np.float32), device, TYPES[kind])
    out = torch.full((m, n), float("nan"), dtype=TYPES[kind], device=device)
    da, dw = _dev(a, device), _dev(w, device)
    _k().matmul_int8(da, _dev(sa, device), dw, _dev(sw, device), out, k=k, residual=res)
    # (integer products below 2^53 are exact in float64)
    sums = a[:, :k].astype(np.float64) @ w[:, :k].astype(np.float64).T
    want = sums * sa[:, None].astype(np.float64) * sw[None, :].astype(np.float64)
    # float(sum), two products: three roundings; the sum with the residual, then the output's
    tol = 3.01 * U * np.abs(want)
    if res is not None:
        want = want + _f64(res)
        tol = tol + U * np.abs(want)
    tol = tol + 1.01 * U_OUT[kind] * np.abs(want) + TINY[kind]
    got = _f64(out)
    assert np.all(np.abs(got - want) <= tol), float(np.max(np.abs(got - want) / tol))


@pytest.mark.parametrize("m,n,k", [
    (1, 16, 32), (1, 2048, 2048), (1, 33, 100), (2, 128, 64), (3, 1000, 4096), (7, 65, 8192), (8, 130, 2048),
    (16, 512, 512), (17, 515, 1040), (31, 64, 16), (33, 257, 272), (64, 256, 1024), (65, 129, 640), (100, 640, 320),
    (128, 256, 256), (129, 257, 129), (200, 2048, 2048), (256, 1024, 5000), (300, 770, 1), (509, 1024, 2048),
    (1, 1, 1), (1, 5000, 31), (12, 4096, 48), (48, 48, 4800), (6, 16400, 100), (8, 16384, 2064), (20, 17000, 530),
    (32, 16387, 4096), (4, 20000, 64), (64, 100, 8200), (40, 70, 131071), (300, 130, 9000), (513, 33000, 64),
    (256, 12300, 150), (70, 40000, 96)])
def test_matmul_int8_sizes(device, m, n, k):
    _product_case(device, "f32", m, n, k, None, m * 31 + n * 7 + k)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("residual", [None, "rows", "bias"])
@pytest.mark.parametrize("m", [1, 5, 40, 150, 520])
def test_matmul_int8_types_and_residuals(device, kind, residual, m):
    _product_case(device, kind, m, 384, 512, residual, m)
    _product_case(device, kind, m, 333, 200, residual, m + 1, lda=256)


@pytest.mark.parametrize("kind,residual", [("f32", None), ("f16", "rows"), ("bf16", "bias"), ("f32", "rows")])
def test_matmul_int8_many_tiles(device, kind, residual):
    """Sizes that take the largest tiles, whole and ragged in every direction."""
    _product_case(device, kind, 509, 32704, 384, residual, 71)
    _product_case(device, kind, 511, 32697, 130, residual, 72)
    _product_case(device, kind, 385, 32520, 48, residual, 73, lda=64)


def test_matmul_int8_largest_sums(device):
    """k at its limit and every product at its largest: the sums stay inside 32 bits."""
    k = 131071
    a = torch.full((2, k + 1), -128, dtype=torch.int8, device=device)
    w = torch.full((20, k + 1), -128, dtype=torch.int8, device=device)
    w[1::2] = 127
    one = torch.ones(20, device=device)
    out = torch.zeros(2, 20, device=device)
    _k().matmul_int8(a, one[:2], w, one, out, k=k)
    want = np.where(np.arange(20) % 2, -128 * 127 * k, 128 * 128 * k).astype(np.float64)
    assert np.array_equal(_f64(out), np.broadcast_to(want.astype(np.float32), (2, 20)))


@pytest.mark.parametrize("m,n", [(1, 48), (8, 16400), (20, 17000), (40, 96), (300, 520)])
def test_matmul_int8_without_columns(device, m, n):
    """k = 0, on every route a size can take: the sums are empty, nothing is read of either operand."""
    from rmlk_amd._lib import lib
    one_m, one_n = torch.ones(m, device=device), torch.ones(n, device=device)
    res = torch.randn(m, n, device=device)
    a, w = (torch.full((r, 16), 99, dtype=torch.int8, device=device) for r in (m, n))
    for residual, want in ((None, torch.zeros_like(res)), (res, res)):
        out = torch.full_like(res, float("nan"))
        _k().matmul_int8(a, one_m, w, one_n, out, k=0, residual=residual)
        assert torch.equal(out, want)
    out = torch.full_like(res, float("nan"))
    status = lib().rmlk_hip_matmul_int8(torch.cuda.current_stream().cuda_stream, 1, m, n, 0, 0, 0, one_m.data_ptr(), 0, 0,
                                        one_n.data_ptr(), res.data_ptr(), n, 0, 0, out.data_ptr(), n)
    assert status == 0 and torch.equal(out, res)


def test_matmul_int8_scale_that_is_not_a_number_stays_in_its_row(device):
    rng = np.random.default_rng(2)
    for m in (4, 70):
        a = _dev(rng.integers(-127, 128, (m, 64)).astype(np.int8), device)
        w = _dev(rng.integers(-127, 128, (96, 64)).astype(np.int8), device)
        sa, sw = torch.ones(m, device=device), torch.ones(96, device=device)
        sa[1] = float("nan")
        out = torch.zeros(m, 96, device=device)
        _k().matmul_int8(a, sa, w, sw, out, k=64)
        bad = torch.isnan(out)
        assert bool(bad[1].all()) and int(bad.sum()) == 96


def test_matmul_int8_rows_that_lie_apart_and_result_over_residual(device):
    rng = np.random.default_rng(4)
    m, n, k = 70, 200, 96
    wide_a = _dev(rng.integers(-127, 128, (m, 160)).astype(np.int8), device)
    wide_w = _dev(rng.integers(-127, 128, (n, 128)).astype(np.int8), device)
    a, w = wide_a[:, 32:144], wide_w[:, 16:112]
    one_m, one_n = torch.full((m,), 0.5, device=device), torch.full((n,), 0.25, device=device)
    wide_c = torch.zeros(m, n + 13, device=device)
    c = wide_c[:, 5:5 + n]
    c.copy_(torch.from_numpy(rng.standard_normal((m, n)).astype(np.float32)))
    before = _f64(c)
    _k().matmul_int8(a, one_m, w, one_n, c, k=k, residual=c)
    want = _f64(a[:, :k]) @ _f64(w[:, :k]).T * 0.125 + before
    assert np.all(np.abs(_f64(c) - want) <= 4 * U * (np.abs(want) + np.abs(before)))
    assert not wide_c[:, :5].any() and not wide_c[:, 5 + n:].any()


# ---- the paged cache --------------------------------------------------------------------------------

class Paged:
    """A cache on the device and its double in numpy, with ragged sequences in shuffled pages."""

    def __init__(self, device, seqs, size, heads, dim, capacity, seed, spare=1):
        self.rng = np.random.default_rng(seed)
        self.device, self.size, self.heads, self.dim = device, size, heads, dim
        per = -(-capacity // size)
        pages = seqs * per + spare
        order = self.rng.permutation(pages)
        self.table = order[:seqs * per].reshape(seqs, per).astype(np.int32)
        k = self.rng.integers(-127, 128, (pages, heads, size, dim)).astype(np.int8)
        v = self.rng.integers(-127, 128, (pages, heads, dim, size)).astype(np.int8)
        # exponents that differ from block to block
        ks = (2.0 ** self.rng.integers(-7, -3, (pages, heads))).astype(np.float32)
        vs = (2.0 ** self.rng.integers(-9, 1, (pages, heads))).astype(np.float32)
        self.ref = ref.Cache(k, v, ks, vs)
        self.dev = _k().PagedCache(_dev(k, device), _dev(v, device), _dev(ks, device), _dev(vs, device))

    def batch(self, first, length, rows, max_new, max_len):
        return _k().PagedBatch(_dev(np.asarray(first, np.int32), self.device),
                               _dev(np.asarray(length, np.int32), self.device), _dev(self.table, self.device),
                               tokens=rows, max_new=max_new, max_len=max_len)

    def check_cache(self):
        for name in ("k", "v", "k_scale", "v_scale"):
            got, want = getattr(self.dev, name).cpu().numpy(), getattr(self.ref, name)
            assert np.array_equal(got, want, equal_nan=got.dtype == np.float32), name


def _tables(rng, positions, dim):
    angle = rng.uniform(-3, 3, (positions, dim // 2))
    angle = np.concatenate([angle, angle], axis=1)
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


def _append(p, kind, new, length, rep=2, pad=0, rotate=True, strided=False, values=None, with_q=True):
    first = np.concatenate([[0], np.cumsum(new)])
    rows = int(first[-1]) + pad
    rng, device = p.rng, p.device
    heads = p.heads * rep
    shape_kv, shape_q = (rows, p.heads, p.dim), (rows, heads, p.dim)
    k = rng.standard_normal(shape_kv).astype(np.float32) if values is None else values[0]
    v = rng.standard_normal(shape_kv).astype(np.float32) * 2 if values is None else values[1]
    q = rng.standard_normal(shape_q).astype(np.float32)
    cos, sin = _tables(rng, max(max(length), 1), p.dim)
    if strided:      # slices of one joint projection
        joint = np.concatenate([a.reshape(rows, -1) for a in (q, k, v)], axis=1)
        joint = _dev(joint, device, TYPES[kind])
        wq, wk = heads * p.dim, p.heads * p.dim
        dq = joint[:, :wq].view(rows, heads, p.dim)
        dk = joint[:, wq:wq + wk].view(rows, p.heads, p.dim)
        dv = joint[:, wq + wk:].view(rows, p.heads, p.dim)
    else:
        dq, dk, dv = (_dev(a, device, TYPES[kind]) for a in (q, k, v))
    q_out = torch.full(shape_q, 7.0, dtype=TYPES[kind], device=device)
    flag = torch.zeros(1, dtype=torch.int32, device=device)
    batch = p.batch(first, length, rows, max(list(new) + [0]), max(list(length) + [0]))
    dc, ds = (_dev(cos, device), _dev(sin, device)) if rotate else (None, None)
    _k().paged_append(p.dev, batch, dk, dv, cos=dc, sin=ds, q=dq if with_q else None,
                      q_out=q_out if with_q else None, err_flag=flag)
    assert flag.item() == 0
    c64, s64 = cos.astype(np.float64), sin.astype(np.float64)
    k64, v64, q64 = _f64(dk), _f64(dv), _f64(dq)
    want_q = np.full(shape_q, 7.0)
    for s, (n, l) in enumerate(zip(new, length)):
        at = slice(first[s], first[s + 1])
        p.ref.append(p.table[s], l - n, k64[at], v64[at], c64 if rotate else None, s64 if rotate else None)
        for i in range(n):
            want_q[first[s] + i] = (ref.rotate(q64[first[s] + i], c64[l - n + i], s64[l - n + i]) if rotate
                                    else q64[first[s] + i])
    p.check_cache()
    if with_q:
        tol = 1.01 * U_OUT[kind] * np.abs(want_q) + TINY[kind]
        assert np.all(np.abs(_f64(q_out) - want_q) <= tol)
    return batch, q_out


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("size", [16, 32, 64, 128])
@pytest.mark.parametrize("dim", [64, 128])
def test_paged_append_ragged(device, kind, size, dim):
    p = Paged(device, 5, size, 2, dim, 4 * size + 64, size * dim)
    _append(p, kind, [1, size, 3 * size + 5, 0, 7], [1, size, 3 * size + 5, 9, 2 * size + 2], pad=3)
    _append(p, kind, [1, 1, 1, 1, 1], [2, size + 1, 3 * size + 6, 10, 2 * size + 3], strided=True)
    _append(p, kind, [2, 0, 40, 1, size], [4, size + 1, 3 * size + 46, 11, 3 * size + 3], rotate=False, rep=3)


def test_paged_append_token_by_token_grows_blocks(device):
    """Values that grow from token to token: every append raises the step and re-rounds what is held."""
    p = Paged(device, 1, 16, 1, 64, 40, 3)
    rng = np.random.default_rng(1)
    for t in range(36):
        grow = 1.7 ** (t % 16)
        k = rng.standard_normal((1, 1, 64)).astype(np.float32) * np.float32(grow)
        v = rng.standard_normal((1, 1, 64)).astype(np.float32) * np.float32(1 / grow)
        _append(p, "f32", [1], [t + 1], values=(k, v), with_q=False, rotate=t % 2 == 0)


def test_paged_append_borders_of_the_step(device):
    """Largest magnitudes at and next to 127 * 2^e, zeros, the smallest and the largest floats."""
    tops = [127.0, np.nextafter(np.float32(127), np.float32(128)), 128.0, 1.0, 127 / 128, 0.0, 2.0 ** -126,
            2.0 ** -149, 127 * 2.0 ** -126, 3.4028234e38, 63.5, 64.0]
    p = Paged(device, len(tops), 16, 1, 64, 16, 5)
    rng = np.random.default_rng(6)
    k = np.zeros((len(tops), 1, 64), np.float32)
    for i, t in enumerate(tops):
        k[i, 0] = (rng.uniform(-1, 1, 64) * np.float64(t)).astype(np.float32)
        k[i, 0, 5] = np.float32(t)
    v = -k[:, :, ::-1].copy()
    _append(p, "f32", [1] * len(tops), [1] * len(tops), values=(k, v), rotate=False, with_q=False)


def test_paged_append_not_finite_values_mark_their_block(device):
    p = Paged(device, 1, 16, 2, 64, 48, 9)
    k = np.ones((20, 2, 64), np.float32)
    v = np.ones((20, 2, 64), np.float32)
    k[3, 1, 7] = np.nan
    v[18, 0, 2] = -np.inf
    _append(p, "f32", [20], [20], values=(k, v), rotate=False, with_q=False)
    assert np.isnan(p.ref.k_scale[p.table[0, 0], 1]) and np.isnan(p.ref.v_scale[p.table[0, 1], 0])
    one = np.ones((1, 2, 64), np.float32)
    _append(p, "f32", [1], [21], values=(one, one), rotate=False, with_q=False)      # stays marked
    many = np.ones((20, 2, 64), np.float32)
    _append(p, "f32", [20], [20], values=(many, many), rotate=False, with_q=False)   # started anew
    assert not np.isnan(p.ref.k_scale).any()


@pytest.mark.parametrize("kind", TYPES)
def test_paged_append_rotates_queries_that_are_not_finite_or_large(device, kind):
    """Infinities, NaN and the type's largest values go where the formula sends them, and only there."""
    kk = _k()
    p = Paged(device, 1, 16, 1, 64, 16, 12)
    dt = TYPES[kind]
    most = torch.finfo(dt).max
    q = torch.ones(6, 2, 64, device=device, dtype=dt)
    for i, value in enumerate((float("inf"), -float("inf"), float("nan"), most, -most)):
        q[i, 0, 3] = value          # the first half of the row
        q[i, 1, 35] = value         # the second
    kv = torch.ones(6, 1, 64, device=device, dtype=dt)
    cos, sin = (_dev(t, device) for t in _tables(np.random.default_rng(1), 6, 64))
    out = torch.zeros_like(q)
    kk.paged_append(p.dev, p.batch([0, 6], [6], 6, 6, 6), kv, kv, cos=cos, sin=sin, q=q, q_out=out)
    x, c, s = _f64(q), _f64(cos)[:, None], _f64(sin)[:, None]
    turned = np.concatenate([-x[..., 32:], x[..., :32]], axis=-1)
    with np.errstate(all="ignore"):
        want = x * c + turned * s
    got, bound = _f64(out), float(most)
    nan, inside = np.isnan(want), np.abs(want) < bound
    assert np.array_equal(np.isnan(got), nan)
    beyond = ~nan & ~inside          # (the largest value or an infinity: one rounding apart)
    assert np.all(np.sign(got[beyond]) == np.sign(want[beyond])) and np.all(np.abs(got[beyond]) >= bound)
    assert np.all(np.abs(got[inside] - want[inside]) <= 1.01 * U_OUT[kind] * np.abs(want[inside]) + TINY[kind])


def test_paged_append_bad_numbers_are_reported_and_skipped(device):
    kk = _k()
    p = Paged(device, 3, 16, 2, 64, 40, 11)
    k = torch.ones(9, 2, 64, device=device)
    flag = torch.zeros(1, dtype=torch.int32, device=device)
    cos = torch.ones(18, 64, device=device)

    def go(first, length, table=None, max_new=9, max_len=40, rotate=False):
        flag.zero_()
        t = p.table if table is None else table
        batch = kk.PagedBatch(_dev(np.asarray(first, np.int32), device), _dev(np.asarray(length, np.int32), device),
                              _dev(np.asarray(t, np.int32), device), tokens=9, max_new=max_new, max_len=max_len)
        kk.paged_append(p.dev, batch, k, k, cos=cos if rotate else None, sin=cos if rotate else None, err_flag=flag)
        return flag.item()

    assert go([0, 5, 3, 9], [5, 5, 9]) == 1                # does not ascend: nothing is done
    p.check_cache()
    assert go([-1, 3, 6, 9], [3, 3, 3]) == 1
    p.check_cache()
    assert go([0, 3, 6, 10], [3, 3, 4]) == 1               # more rows than there are
    p.check_cache()
    ones = np.ones((9, 2, 64))
    for bad in (dict(length=[3, 2, 3]), dict(length=[3, 41, 3]), dict(length=[3, -5, 3]),
                dict(length=[3, 1 << 30, 3])):              # fewer tokens than rows, beyond max_len, negative
        assert go([0, 3, 6, 9], bad["length"]) == 1
        for s in (0, 2):
            p.ref.append(p.table[s], 0, ones[:3], ones[:3])
        p.check_cache()
    assert go([0, 1, 8, 9], [1, 7, 1], max_new=5) == 1      # more rows than the bound
    for s in (0, 2):
        p.ref.append(p.table[s], 0, ones[:1], ones[:1])
    p.check_cache()
    table = p.table.copy()
    table[1, 1] = p.ref.k.shape[0]
    table[2, 0] = -1
    assert go([0, 3, 6, 9], [3, 18, 3], table=table) == 1   # pages outside the cache
    p.ref.append(p.table[0], 0, ones[:3], ones[:3])
    p.ref.append(p.table[1][:1], 15, ones[:1], ones[:1])    # position 15; 16 and 17 lie in the bad page
    p.check_cache()
    assert go([0, 3, 6, 9], [3, 20, 3], rotate=True) == 1   # positions 18 and 19 have no row in the tables
    turned = np.concatenate([np.zeros((3, 2, 32)), np.full((3, 2, 32), 2.0)], axis=2)
    p.ref.append(p.table[0], 0, turned, ones[:3])
    p.ref.append(p.table[1], 17, turned[:1], ones[:1])
    p.ref.append(p.table[2], 0, turned, ones[:3])
    p.check_cache()


# ---- attention --------------------------------------------------------------------------------------

def _attend(p, kind, new, length, rep=2, pad=0, scale=None, is_mul=True, strided=False, q_std=1.0, bounds=None,
            table=None, q=None, stream=None):
    first = np.concatenate([[0], np.cumsum(new)])
    rows = int(first[-1]) + pad
    heads = p.heads * rep
    scale = p.dim ** -0.5 if scale is None else scale
    if q is None:
        q = p.rng.standard_normal((rows, heads, p.dim)).astype(np.float32) * q_std
    if strided:
        wide = _dev(np.concatenate([q.reshape(rows, -1), q.reshape(rows, -1) * 0 + 5], axis=1), p.device, TYPES[kind])
        dq = wide[:, :heads * p.dim].view(rows, heads, p.dim)
    else:
        dq = _dev(q, p.device, TYPES[kind])
    out = torch.full((rows, heads, p.dim), 7.0, dtype=TYPES[kind], device=p.device)
    flag = torch.zeros(1, dtype=torch.int32, device=p.device)
    max_new, max_len = bounds or (max(list(new) + [0]), max(list(length) + [0]))
    batch = p.batch(first, length, rows, max_new, max_len)
    arg = scale if is_mul else 1 / scale
    _k().paged_attention(p.dev, batch, dq, out, scale=arg, scale_is_mul=is_mul, err_flag=flag)
    assert flag.item() == 0
    _check_attention(p, kind, dq, out, first, new, length, scale, rep)
    assert bool((out[int(first[-1]):] == 7).all()), "rows behind the last sequence were written"
    return out


def _check_attention(p, kind, dq, out, first, new, length, scale, rep, table=None):
    """Tolerance. A score is a sum of dim products of a query's value (22 bits: 2^-22 off) and an integer, summed and
    scaled in float: off by at most (2^-22 + (dim + 4) u) * bound, bound = sum |q||k| * scale; the exponential of
    a difference from the maximum (two such errors, and its own few roundings) is off by that much relative to
    itself, the weighted mean of v by twice that (numerator and denominator) times max |v|. The weights of the
    16-bit types are rounded to half (2^-11). Sums over the tokens round a few times: 64 u covers the tree of
    running sums at these lengths. Then the output's rounding."""
    q64, got = _f64(dq), _f64(out)
    table = p.table if table is None else table
    for s, (n, l) in enumerate(zip(new, length)):
        if n == 0:
            continue
        for g in range(p.heads):
            k, v = p.ref.tokens(table[s], l, g)
            for r in range(rep):
                h = g * rep + r
                want, bound = ref.attend(q64[first[s]:first[s + 1], h], k, v, l, scale)
                mine = got[first[s]:first[s + 1], h]
                vmax = np.abs(v[np.isfinite(v)]).max() if v.size and np.isfinite(v).any() else 0.0
                delta = (2.0 ** -22 + (p.dim + 4) * U) * bound[:, None]
                weights = 0.0 if kind == "f32" else 2.0 ** -11
                tol = (4 * delta + weights + 64 * U) * vmax + 1.01 * U_OUT[kind] * np.abs(want) + TINY[kind]
                nan = np.isnan(want)
                assert np.array_equal(np.isnan(mine), nan), (s, h)
                assert np.all((np.abs(mine - want) <= tol) | nan), (s, h, float(np.nanmax(np.abs(mine - want) / tol)))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("size", [16, 32, 64, 128])
def test_paged_attention_single_tokens(device, kind, dim, size):
    p = Paged(device, 9, size, 2, dim, 1000, size + dim)
    length = [1, 2, size - 1, size, size + 1, 63, 65, 200, 1000]
    _attend(p, kind, [1] * 9, length, rep=4, pad=2)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rep", [1, 2, 3, 5, 8])
def test_paged_attention_ragged_prompts(device, kind, rep):
    p = Paged(device, 6, 32, 2, 64, 400, rep)
    _attend(p, kind, [1, 64, 130, 0, 17, 33], [1, 64, 130, 50, 300, 97], rep=rep, pad=1)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("dim,size", [(64, 64), (128, 16), (128, 128)])
def test_paged_attention_long_prompt(device, kind, dim, size):
    p = Paged(device, 2, size, 1, dim, 700, dim + size)
    _attend(p, kind, [600, 5], [600, 690], rep=2, strided=True)


@pytest.mark.parametrize("kind", TYPES)
def test_paged_attention_long_cache(device, kind):
    """Keys split over many blocks, sequences of very different lengths, bounds far above what is there."""
    p = Paged(device, 3, 64, 1, 64, 9000, 21)
    _attend(p, kind, [1, 2, 1], [9000, 5000, 3], rep=4, bounds=(4, 9000))
    _attend(p, kind, [1, 1, 1], [70, 2, 0], rep=4, bounds=(3, 9000))


def test_paged_attention_many_heads_and_sequences(device):
    p = Paged(device, 33, 16, 8, 64, 90, 8)
    rng = np.random.default_rng(3)
    _attend(p, "f32", [1] * 33, [int(x) for x in rng.integers(1, 90, 33)], rep=8)
    _attend(p, "f32", [int(x) for x in rng.integers(0, 6, 33)], [int(x) for x in rng.integers(6, 90, 33)], rep=1)


@pytest.mark.parametrize("dim", [64, 128])
def test_paged_attention_rows_that_see_nothing(device, dim):
    """More rows than tokens: the first rows have negative positions and get zeros; sequences of no tokens."""
    p = Paged(device, 4, 16, 1, dim, 64, 2)
    out = _attend(p, "f32", [5, 3, 40, 1], [3, 0, 20, 0], rep=2)
    assert not out[:2].any() and not out[5:8].any() and not out[8:28].any() and not out[48].any()


@pytest.mark.parametrize("is_mul", [True, False])
def test_paged_attention_scales(device, is_mul):
    p = Paged(device, 2, 32, 2, 64, 200, 13)
    _attend(p, "f32", [3, 100], [180, 190], scale=0.37, is_mul=is_mul)


@pytest.mark.parametrize("kind", TYPES)
def test_paged_attention_steep_scores(device, kind):
    """Scores that differ by hundreds: all the weight on a few keys."""
    p = Paged(device, 2, 16, 1, 64, 500, 31)
    _attend(p, kind, [1, 70], [500, 400], rep=2, q_std=40.0)


def test_paged_attention_scores_that_rise_along_the_keys(device):
    """The maximum moves with every key: the sums held so far are rescaled all the way."""
    p = Paged(device, 1, 64, 1, 64, 512, 17)
    ramp = np.clip(np.arange(512) // 4, 0, 127).astype(np.int8)
    for page in range(8):
        p.ref.k[p.table[0, page], 0] = ramp[page * 64:(page + 1) * 64, None]
    p.ref.k_scale[:] = 0.25
    p.dev.k.copy_(torch.from_numpy(p.ref.k))
    p.dev.k_scale.copy_(torch.from_numpy(p.ref.k_scale))
    for std in (0.01, 0.3, 3.0):
        q = np.abs(p.rng.standard_normal((130, 2, 64))).astype(np.float32) * np.float32(std)
        _attend(p, "f32", [130], [512], rep=2, q=q)
        _attend(p, "f32", [130], [512], rep=2, q=-q)


def test_paged_attention_blocks_of_very_different_steps(device):
    """Steps of V a factor 2^20 apart between pages: the small ones keep their precision where the weight is
    theirs alone (a sequence within them)."""
    p = Paged(device, 2, 16, 1, 64, 200, 19)
    p.ref.v_scale[:] = 2.0 ** -3
    for page in range(0, p.table.shape[1], 2):
        p.ref.v_scale[p.table[0, page], 0] = 2.0 ** -23
    p.ref.v_scale[p.table[1], 0] = 2.0 ** -90
    p.dev.v_scale.copy_(torch.from_numpy(p.ref.v_scale))
    _attend(p, "f32", [3, 70], [200, 180], rep=4)


def test_paged_attention_queries_of_every_magnitude(device):
    p = Paged(device, 1, 16, 1, 64, 40, 23)
    q = p.rng.standard_normal((6, 2, 64)).astype(np.float32)
    for i, f in enumerate((1e-38, 1e-20, 1e-6, 1.0, 30.0, 0.0)):
        q[i] *= np.float32(f)
    _attend(p, "f32", [6], [40], q=q)


def test_paged_attention_marked_blocks_and_masked_garbage(device):
    """A block whose scale is NaN makes the queries that see it NaN and no others; nothing behind a sequence's
    tokens (other values of its last page, scales of pages it does not hold) reaches any result."""
    p = Paged(device, 3, 16, 2, 64, 64, 29, spare=3)
    for which in (p.ref.k_scale, p.ref.v_scale):
        which[p.table[0, 1], 1] = np.nan                      # tokens 16 .. 31 of sequence 0, head 1
        which[p.table[1, 2]] = np.nan                         # a page behind sequence 1's tokens
        which[p.table[2, 3]] = np.inf
    p.dev.k_scale.copy_(torch.from_numpy(p.ref.k_scale))
    p.dev.v_scale.copy_(torch.from_numpy(p.ref.v_scale))
    out = _attend(p, "f32", [40, 20, 40], [40, 32, 48], rep=2)
    assert torch.isnan(out[16:40, 2:]).all() and torch.isfinite(out[16:40, :2]).all()
    assert torch.isfinite(out[:16]).all() and torch.isfinite(out[40:]).all()
    p.ref.k_scale[p.table[0, 1], 1] = 1.0                     # of V alone
    p.dev.k_scale.copy_(torch.from_numpy(p.ref.k_scale))
    _attend(p, "f32", [40, 20, 40], [40, 32, 48], rep=2)
    _attend(p, "bf16", [1, 1, 1], [40, 32, 48], rep=2)


def test_paged_attention_query_that_is_not_finite_stays_alone(device):
    p = Paged(device, 1, 16, 1, 64, 64, 37)
    for rows in (5, 64):
        q = p.rng.standard_normal((rows, 2, 64)).astype(np.float32)
        q[1, 0, 3], q[2, 1, 60] = np.nan, np.inf
        first, new, length = [0, rows], [rows], [64]
        dq = _dev(q, device)
        out = torch.zeros(rows, 2, 64, device=device)
        _k().paged_attention(p.dev, p.batch(first, length, rows, rows, 64), dq, out, scale=0.125, scale_is_mul=True)
        bad = torch.isnan(out).any(dim=2)
        assert bool(bad[1, 0]) and bool(bad[2, 1]) and int(bad.sum()) == 2


def test_paged_attention_bad_numbers_are_reported_and_skipped(device):
    kk = _k()
    p = Paged(device, 3, 16, 2, 64, 64, 41)
    q = torch.from_numpy(p.rng.standard_normal((9, 4, 64)).astype(np.float32)).to(device)
    flag = torch.zeros(1, dtype=torch.int32, device=device)

    def go(first, length, table=None, max_new=9, max_len=64):
        flag.zero_()
        out = torch.full((9, 4, 64), 7.0, device=device)
        t = p.table if table is None else table
        batch = kk.PagedBatch(_dev(np.asarray(first, np.int32), device), _dev(np.asarray(length, np.int32), device),
                              _dev(np.asarray(t, np.int32), device), tokens=9, max_new=max_new, max_len=max_len)
        kk.paged_attention(p.dev, batch, q, out, scale=0.125, scale_is_mul=True, err_flag=flag)
        assert flag.item() == 1
        return out

    for first in ([0, 5, 3, 9], [-1, 3, 6, 9], [0, 3, 6, 10]):
        assert bool((go(first, [20, 20, 20]) == 7).all())
    for length in ([40, 65, 40], [40, -1, 40], [40, 1 << 30, 40]):
        out = go([0, 3, 6, 9], length)
        assert bool((out[3:6] == 7).all())
        _check_attention(p, "f32", q, out, [0, 3, 6, 9], [3, 0, 3], [40, 0, 40], 0.125, 2)
    out = go([0, 1, 8, 9], [40, 40, 40], max_new=5)
    assert bool((out[1:8] == 7).all())
    table = p.table.copy()
    table[1, 1] = p.ref.k.shape[0]          # tokens 16 .. 31 of sequence 1 are hidden
    table[2, 0] = -3                        # sequence 2: nothing is left
    out = go([0, 3, 6, 9], [40, 40, 3], table=table)
    _check_attention(p, "f32", q, out, [0, 3, 6, 9], [3, 0, 0], [40, 0, 0], 0.125, 2)
    assert not out[6:9].any()
    q64 = _f64(q)
    for h in range(4):
        k, v = p.ref.tokens(p.table[1], 40, h // 2)
        for i in range(3):
            see = [t for t in range(38 + i) if not 16 <= t < 32]
            want, bound = ref.attend(q64[3 + i:4 + i, h], k[see], v[see], len(see), 0.125)
            tol = (4 * (2.0 ** -22 + 68 * U) * bound[0] + 64 * U) * np.abs(v).max() + U * np.abs(want)
            assert np.all(np.abs(_f64(out[3 + i, h]) - want[0]) <= tol[0])


def test_paged_calls_of_a_padded_batch_without_new_tokens(device):
    """Rows, but none of them a sequence's (max_new 0): nothing is written; a sequence that has some is reported."""
    kk = _k()
    p = Paged(device, 3, 16, 2, 64, 64, 47)
    x = torch.ones(9, 2, 64, device=device)
    for max_len in (64, 1 << 20):
        for first, bad in (([0, 0, 0, 0], 0), ([4, 4, 4, 4], 0), ([0, 0, 2, 2], 1)):
            flag = torch.zeros(2, dtype=torch.int32, device=device)
            out = torch.full((9, 4, 64), 7.0, device=device)
            batch = kk.PagedBatch(_dev(np.asarray(first, np.int32), device), _dev(np.asarray([20, 20, 0], np.int32), device),
                                  _dev(p.table, device), tokens=9, max_new=0, max_len=max_len)
            kk.paged_append(p.dev, batch, x, x, err_flag=flag[:1])
            kk.paged_attention(p.dev, batch, torch.ones_like(out), out, scale=0.125, err_flag=flag[1:])
            assert flag.tolist() == [bad, bad] and bool((out == 7).all())
            p.check_cache()


def test_paged_attention_sequences_that_share_pages(device):
    """A common prefix: the same pages in two page tables (read only)."""
    p = Paged(device, 2, 16, 2, 64, 64, 43)
    p.table[1, :2] = p.table[0, :2]
    _attend(p, "f32", [1, 20], [60, 50], rep=4)
    p.table[1] = p.table[1, 0]              # one page again and again
    _attend(p, "f32", [1, 20], [60, 50], rep=4)


def test_paged_cache_offsets_beyond_32_bits(device):
    """Pages that begin more than 2^32 bytes into the cache."""
    kk = _k()
    heads, size, dim = 16, 128, 128
    per_page = heads * size * dim
    pages = (1 << 32) // per_page + 3
    if torch.cuda.mem_get_info()[0] < 3 * pages * per_page:
        pytest.skip("not enough free memory")
    k = torch.zeros(pages, heads, size, dim, dtype=torch.int8, device=device)
    v = torch.zeros(pages, heads, dim, size, dtype=torch.int8, device=device)
    cache = kk.PagedCache(k, v, torch.ones(pages, heads, device=device), torch.ones(pages, heads, device=device))
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device=device)
    rows = 300
    gen = torch.Generator(device=device).manual_seed(3)
    x = torch.randn(rows, heads, dim, generator=gen, device=device)
    first = torch.tensor([0, rows], dtype=torch.int32, device=device)
    length = torch.tensor([rows], dtype=torch.int32, device=device)
    batch = kk.PagedBatch(first, length, table, tokens=rows, max_new=rows, max_len=rows)
    kk.paged_append(cache, batch, x, x)
    out = torch.zeros_like(x)
    kk.paged_attention(cache, batch, x, out, scale=0.05, scale_is_mul=True)
    small = kk.PagedCache(k[[pages - 1, 0, pages - 2]].contiguous(), v[[pages - 1, 0, pages - 2]].contiguous(),
                          cache.k_scale[[pages - 1, 0, pages - 2]].contiguous(),
                          cache.v_scale[[pages - 1, 0, pages - 2]].contiguous())
    assert int(small.k.abs().amax()) > 63 and bool((small.k_scale <= 2.0 ** -4).all())
    near = torch.tensor([[0, 1, 2]], dtype=torch.int32, device=device)
    again = torch.zeros_like(x)
    kk.paged_attention(small, kk.PagedBatch(first, length, near, tokens=rows, max_new=rows, max_len=rows), x, again,
                       scale=0.05, scale_is_mul=True)
    assert torch.equal(out, again)


# ---- together, streams, graphs --------------------------------------------------------------------

def _layer(kk, w, cache, batch, x, cos, sin, buf):
    """One attention layer of a decoder in 8 bits; every buffer is the caller's."""
    heads, kv_heads, dim = w["heads"], w["kv_heads"], w["dim"]
    kk.rmsnorm_quantize_rows(x, w["gamma"], 1e-5, buf["xq"], buf["xs"])
    kk.matmul_int8(buf["xq"], buf["xs"], w["qkv"], w["qkv_s"], buf["joint"], k=x.shape[1])
    rows = x.shape[0]
    a, b = heads * dim, (heads + kv_heads) * dim
    kk.paged_append(cache, batch, buf["joint"][:, a:b].view(rows, kv_heads, dim),
                    buf["joint"][:, b:].view(rows, kv_heads, dim), cos=cos, sin=sin,
                    q=buf["joint"][:, :a].view(rows, heads, dim), q_out=buf["q"])
    kk.paged_attention(cache, batch, buf["q"], buf["ctx"], scale=dim ** 0.5, workspace=buf.get("ws"))
    kk.quantize_rows(buf["ctx"].view(rows, a), buf["cq"], buf["cs"])
    kk.matmul_int8(buf["cq"], buf["cs"], w["o"], w["o_s"], buf["out"], k=a, residual=x)
    return buf["out"]


def _layer_weights(kk, device, hidden, heads, kv_heads, dim, seed):
    gen = torch.Generator(device=device).manual_seed(seed)
    w = dict(heads=heads, kv_heads=kv_heads, dim=dim)
    w["gamma"] = 0.5 + torch.rand(hidden, generator=gen, device=device)
    for name, n, k in (("qkv", (heads + 2 * kv_heads) * dim, hidden), ("o", hidden, heads * dim)):
        full = torch.randn(n, k, generator=gen, device=device) * 0.05
        w[name] = torch.zeros(n, _padded(k), dtype=torch.int8, device=device)
        w[name + "_s"] = torch.zeros(n, device=device)
        kk.quantize_rows(full, w[name], w[name + "_s"])        # one scale per output channel
    return w


def _layer_buffers(device, rows, hidden, heads, kv_heads, dim, kind=torch.float32):
    z = lambda *s, t=kind: torch.zeros(*s, dtype=t, device=device)
    return dict(xq=z(rows, _padded(hidden), t=torch.int8), xs=z(rows, t=torch.float32),
                joint=z(rows, (heads + 2 * kv_heads) * dim), q=z(rows, heads, dim), ctx=z(rows, heads, dim),
                cq=z(rows, heads * dim, t=torch.int8), cs=z(rows, t=torch.float32), out=z(rows, hidden))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_decoder_layer_prompt_then_tokens(device, kind):
    """The operators in a row as a decoder layer uses them: a ragged prompt, then single tokens; every stage is
    compared with its definition on the operands it really had."""
    kk = _k()
    hidden, heads, kv_heads, dim, size = 192, 4, 2, 64, 16
    t = TYPES[kind]
    w = _layer_weights(kk, device, hidden, heads, kv_heads, dim, 1)
    p = Paged(device, 3, size, kv_heads, dim, 64, 51)
    cos, sin = _tables(p.rng, 64, dim)
    dcos, dsin = _dev(cos, device), _dev(sin, device)
    lengths = [0, 0, 0]
    for new in ([20, 7, 33], [1, 1, 1], [1, 1, 1], [4, 1, 2]):
        lengths = [l + n for l, n in zip(lengths, new)]
        first = np.concatenate([[0], np.cumsum(new)])
        rows = int(first[-1])
        batch = p.batch(first, lengths, rows, max(new), 64)
        x = torch.from_numpy(p.rng.standard_normal((rows, hidden)).astype(np.float32)).to(device).to(t)
        buf = _layer_buffers(device, rows, hidden, heads, kv_heads, dim, t)
        out = _layer(kk, w, p.dev, batch, x, dcos, dsin, buf)
        _check_rows(buf["xq"], buf["xs"], ref.rmsnorm(_f64(x), w["gamma"].cpu().numpy(), 1e-5), hidden, False)
        joint = _f64(buf["joint"])
        want = (_f64(buf["xq"])[:, :hidden] @ _f64(w["qkv"])[:, :hidden].T) * _f64(buf["xs"])[:, None] * _f64(w["qkv_s"])
        assert np.all(np.abs(joint - want) <= (4 * U + 1.01 * U_OUT[kind]) * np.abs(want) + TINY[kind])
        a, b = heads * dim, (heads + kv_heads) * dim
        for s in range(3):
            at = slice(first[s], first[s + 1])
            p.ref.append(p.table[s], lengths[s] - new[s], joint[at, a:b].reshape(-1, kv_heads, dim),
                         joint[at, b:].reshape(-1, kv_heads, dim), cos.astype(np.float64), sin.astype(np.float64))
        p.check_cache()
        _check_attention(p, kind, buf["q"], buf["ctx"], first, new, lengths, dim ** -0.5, heads // kv_heads)
        _check_rows(buf["cq"], buf["cs"], _f64(buf["ctx"]).reshape(rows, a), a, True)
        want = (_f64(buf["cq"]) @ _f64(w["o"])[:, :a].T) * _f64(buf["cs"])[:, None] * _f64(w["o_s"]) + _f64(x)
        tol = 4 * U * (np.abs(want) + np.abs(want - _f64(x))) + 1.01 * U_OUT[kind] * np.abs(want) + TINY[kind]
        assert np.all(np.abs(_f64(out) - want) <= tol)


def test_decoder_layer_on_another_stream_and_replayed_from_a_graph(device):
    """The decode step of the layer recorded once and replayed with new inputs and lengths in the same buffers; its
    results equal the eager ones bit for bit, in every replay, with eager work and waits in between."""
    kk = _k()
    hidden, heads, kv_heads, dim, size, seqs = 128, 8, 2, 64, 16, 5
    w = _layer_weights(kk, device, hidden, heads, kv_heads, dim, 2)
    rng = np.random.default_rng(4)
    cos, sin = (_dev(a, device) for a in _tables(rng, 600, dim))
    start = [1, 15, 16, 200, 500]

    def fresh():
        q = Paged(device, seqs, size, kv_heads, dim, 600, 61)
        first = torch.arange(seqs + 1, dtype=torch.int32, device=device)
        length = torch.tensor(start, dtype=torch.int32, device=device)
        batch = kk.PagedBatch(first, length, _dev(q.table, device), tokens=seqs, max_new=1, max_len=600)
        buf = _layer_buffers(device, seqs, hidden, heads, kv_heads, dim)
        need = kk.paged_attention_workspace_size(q.dev, batch, torch.float32, heads)
        buf["ws"] = torch.full((max(need, 16),), 0xEE, dtype=torch.uint8, device=device)
        return q, batch, buf

    inputs = [torch.from_numpy(rng.standard_normal((seqs, hidden)).astype(np.float32)).to(device) for _ in range(6)]
    eager_p, eager_b, eager_buf = fresh()
    want = []
    for x in inputs:
        want.append(_layer(kk, w, eager_p.dev, eager_b, x, cos, sin, eager_buf).clone())
        eager_b.length += 1

    p, batch, buf = fresh()
    x = inputs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _layer(kk, w, p.dev, batch, x, cos, sin, buf)          # another stream, eager
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(buf["out"], want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _layer(kk, w, p.dev, batch, x, cos, sin, buf)
    for i, xi in enumerate(inputs):                            # (step 0 again: the same token into the same slot)
        x.copy_(xi)
        buf["ws"].fill_(0x11 * (i + 1))
        graph.replay()
        if i % 2:
            torch.cuda.synchronize()
            torch.ones(1000, device=device).sum().item()
        assert torch.equal(buf["out"], want[i]), i
        batch.length += 1
    for name in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(p.dev, name), getattr(eager_p.dev, name))


def test_paged_attention_repeats_bit_for_bit(device):
    p = Paged(device, 4, 64, 2, 128, 3000, 71)
    new, length = [1, 1, 9, 1], [3000, 900, 2500, 64]
    q = p.rng.standard_normal((12, 8, 128)).astype(np.float32)
    outs = [_attend(p, "f16", new, length, rep=4, q=q) for _ in range(3)]
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
