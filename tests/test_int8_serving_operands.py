"""Tensors whose rows repeat or overlap, handed to the wrappers of the 8-bit serving operators: nothing may reach the
library that would be read or written as if such rows lay one behind the other. Runs without a GPU: the library is
replaced by one that notes its arguments."""
import pytest

torch = pytest.importorskip("torch")

from rmlk_amd import kernels as kk      # noqa: E402


class _Noted:
    """A library that launches nothing and keeps the arguments of every call."""

    def __init__(self):
        self.calls = {}

    def __getattr__(self, name):
        def call(*args):
            self.calls[name] = args
            return 0
        return call


@pytest.fixture
def noted(monkeypatch):
    library = _Noted()
    monkeypatch.setattr(kk, "lib", lambda: library)
    monkeypatch.setattr(kk, "_raw_stream", lambda *tensors: 0)
    monkeypatch.setattr(kk, "_ptr", lambda t: t.data_ptr())
    return library.calls


def _overlapping(rows, cols, pitch, dtype=torch.float32):
    return torch.zeros(rows * cols + cols, dtype=dtype).as_strided((rows, cols), (pitch, 1))


def test_pitches():
    z = torch.zeros
    assert kk._pitch2(z(4, 64)) == 64 and kk._pitch2(z(4, 100)[:, 16:48]) == 100 and kk._pitch2(z(8, 64)[::2]) == 128
    assert kk._pitch2(z(1, 64)) == 64 and kk._pitch2(z(1, 100)[:, :64]) == 64 and kk._pitch2(z(64).expand(1, 64)) == 64
    assert kk._pitch2(z(5, 1)) == 1 and kk._pitch2(z(5, 9)[:, 2:3]) == 9 and kk._pitch2(z(0, 64)) == 64
    assert kk._pitch(z(4, 2, 64), 128) == 128 and kk._pitch(z(4, 6, 64)[:, 1:3], 128) == 384
    assert kk._pitch(z(4, 300)[:, 40:168].view(4, 2, 64), 128) == 300
    assert kk._pitch(z(1, 2, 64).expand(1, 2, 64), 128) == 128 and kk._pitch(z(0, 2, 64), 128) == 128
    for bad in (z(64).expand(4, 64), z(1, 64).expand(2, 64), _overlapping(4, 100, 50), _overlapping(3, 64, 63)):
        with pytest.raises(AssertionError):
            kk._pitch2(bad)
    for bad in (z(1, 8, 64).expand(5, 8, 64), _overlapping(5, 512, 256).view(5, 8, 64), z(5, 1, 64).expand(5, 8, 64)):
        with pytest.raises(AssertionError):
            kk._pitch(bad, 512)


@pytest.mark.parametrize("repeat", [lambda t: t[:1].expand_as(t), lambda t: t.new_zeros(t.numel()).as_strided(t.shape, (t.shape[1] // 2, 1))])
def test_matrices_whose_rows_overlap(noted, repeat):
    """Every operand of the row quantisation and of the product in turn."""
    x, q, scale = torch.zeros(4, 64), torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4)
    with pytest.raises(AssertionError):
        kk.quantize_rows(repeat(x), q, scale)
    with pytest.raises(AssertionError):
        kk.quantize_rows(x, repeat(q), scale)
    gamma = torch.ones(64)
    for bad in (dict(x=repeat(x)), dict(q=repeat(q)), dict(add=repeat(x)), dict(sum_out=repeat(x))):
        with pytest.raises(AssertionError):
            kk.rmsnorm_quantize_rows(**{**dict(x=x, gamma=gamma, eps=1e-5, q=q, scale=scale, add=x, sum_out=x), **bad})
    a, wt, out = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(32, 64, dtype=torch.int8), torch.zeros(4, 32)
    for bad in (dict(a=repeat(a)), dict(wt=repeat(wt)), dict(out=repeat(out))):
        with pytest.raises(AssertionError):
            kk.matmul_int8(**{**dict(a=a, a_scale=scale, wt=wt, w_scale=torch.ones(32), out=out, k=64), **bad})
    assert not any(name in noted for name in ("rmlk_hip_quantize_rows", "rmlk_hip_rmsnorm_quantize_rows",
                                              "rmlk_hip_matmul_int8"))


def test_residuals_of_the_product(noted):
    """One row for all rows is a bias, however it is given; rows that overlap otherwise are refused."""
    a, wt, out = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(32, 64, dtype=torch.int8), torch.zeros(4, 32)

    def pitch(residual):
        noted.clear()
        kk.matmul_int8(a, torch.ones(4), wt, torch.ones(32), out, k=64, residual=residual)
        args = noted["rmlk_hip_matmul_int8"]
        assert args[11] == residual.data_ptr()
        return args[12]

    bias = torch.zeros(32)
    assert pitch(bias) == 0 and pitch(bias.expand(4, 32)) == 0 and pitch(torch.zeros(1, 40)[:, 8:].expand(4, 32)) == 0
    assert pitch(torch.zeros(4, 32)) == 32 and pitch(torch.zeros(4, 40)[:, :32]) == 40
    for bad in (_overlapping(4, 32, 16), torch.zeros(4, 1).expand(4, 32), torch.zeros(1).expand(4, 32),
                torch.zeros(64)[::2].expand(4, 32), torch.zeros(64)[::2]):
        with pytest.raises(AssertionError):
            pitch(bad)


def test_rows_of_the_paged_calls_that_overlap(noted):
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    cache = kk.PagedCache.allocate(4, 16, 2, 64, "cpu")
    batch = kk.PagedBatch(i32(2), i32(1), i32(1, 4), tokens=5, max_new=5, max_len=64)
    kv, q, out = torch.zeros(5, 2, 64), torch.zeros(5, 8, 64), torch.zeros(5, 8, 64)
    for repeat in (lambda t: t[:1].expand_as(t), lambda t: t[:, :1].expand_as(t),
                   lambda t: torch.zeros(t.numel()).as_strided(t.shape, (64, 64, 1))):
        for bad in (dict(k=repeat(kv)), dict(v=repeat(kv)), dict(q=repeat(q)), dict(q_out=repeat(q))):
            with pytest.raises(AssertionError):
                kk.paged_append(cache, batch, **{**dict(k=kv, v=kv, q=q, q_out=out), **bad})
        for bad in (dict(q=repeat(q)), dict(out=repeat(q))):
            with pytest.raises(AssertionError):
                kk.paged_attention(cache, batch, **{**dict(q=q, out=out, scale=8.0), **bad})
    assert "rmlk_hip_paged_append" not in noted and "rmlk_hip_paged_attention" not in noted
    kk.paged_append(cache, batch, kv, kv, q=q, q_out=out)
    kk.paged_attention(cache, batch, q, out, scale=8.0)
    assert noted["rmlk_hip_paged_append"][5] == 128 and noted["rmlk_hip_paged_attention"][6] == 512


@pytest.mark.gpu
def test_product_with_an_expanded_bias(device):
    """The bias as [n] and as its expansion to [m, n]: the same bits."""
    gen = torch.Generator(device=device).manual_seed(3)
    ints = lambda *s: torch.randint(-127, 128, s, generator=gen, device=device, dtype=torch.int8)
    for m, n in ((3, 48), (40, 200), (150, 333)):
        a, wt, bias = ints(m, 128), ints(n, 128), torch.randn(n, generator=gen, device=device)
        one_m, one_n = torch.full((m,), 0.01, device=device), torch.full((n,), 0.02, device=device)
        outs = []
        for residual in (bias, bias.expand(m, n)):
            outs.append(torch.empty(m, n, device=device))
            kk.matmul_int8(a, one_m, wt, one_n, outs[-1], k=128, residual=residual)
        assert torch.equal(outs[0], outs[1])
