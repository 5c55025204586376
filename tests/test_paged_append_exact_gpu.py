"""Rotated keys next to the borders of their rounding: the rotation is a sum of two products, and the integers and
the step of a block are those of the real number, here in fractions, also where its double would lie on a border."""
from fractions import Fraction

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

SIZE = 16


def _exact(x, cos, sin):
    """x [new, dim], cos and sin [new, dim]: the rotated rows in fractions."""
    half = x.shape[1] // 2
    f = lambda v: Fraction(float(v))
    rows = []
    for t in range(x.shape[0]):
        lo = [f(x[t, d]) * f(cos[t, d]) - f(x[t, d + half]) * f(sin[t, d]) for d in range(half)]
        hi = [f(x[t, d + half]) * f(cos[t, d + half]) + f(x[t, d]) * f(sin[t, d + half]) for d in range(half)]
        rows.append(lo + hi)
    return rows


def _rounded(rows):
    top, e = max(abs(v) for row in rows for v in row), -126
    while top > 127 * Fraction(2) ** e:
        e += 1
    return np.array([[max(-127, min(127, round(v / Fraction(2) ** e))) for v in row] for row in rows], np.int8), e


def _appended(device, x, cos, sin):
    """Blocks [n, new, dim] appended in one call, one sequence and page each: integers, scales."""
    from rmlk_amd import kernels as kk
    n, new, dim = x.shape
    cache = kk.PagedCache.allocate(n, SIZE, 1, dim, device)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=device)
    batch = kk.PagedBatch(i32([new * i for i in range(n + 1)]), i32([new] * n), i32([[i] for i in range(n)]),
                          tokens=n * new, max_new=new, max_len=SIZE)
    k = torch.from_numpy(x.reshape(n * new, 1, dim)).to(device)
    kk.paged_append(cache, batch, k, k, cos=torch.from_numpy(cos).to(device), sin=torch.from_numpy(sin).to(device))
    return cache.k[:, 0, :new].cpu().numpy(), cache.k_scale[:, 0].cpu().numpy()


def _compare(device, x, cos, sin):
    got, scale = _appended(device, x, cos, sin)
    for i in range(x.shape[0]):
        want, e = _rounded(_exact(x[i], cos, sin))
        assert scale[i] == 2.0 ** e, (i, scale[i], e)
        assert np.array_equal(got[i], want), (i, np.argwhere(got[i] != want)[:4])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [1, 3, 16])
@pytest.mark.parametrize("tiny", [2.0 ** -40, 2.0 ** -60, 2.0 ** -100])
def test_borders_between_integers(device, dim, new, tiny):
    """(j + 1/2) steps and a tail on either side, or none."""
    half = dim // 2
    cos, sin = np.ones((new, dim), np.float32), np.full((new, dim), tiny, np.float32)
    blocks = []
    for step, sign in ((1.0, 1), (1.0, -1), (2.0 ** -11, 1), (2.0 ** 20, -1)):
        x = np.zeros((new, dim), np.float32)
        for t in range(new):
            j = np.arange(half) * 2 - half + t
            x[t, :half] = (j + 0.5) * step * sign
            x[t, half:] = np.where(np.arange(half) % 3 == 0, 0, np.where(np.arange(half) % 3 == 1, 1, -1)) * step
        x[0, 0] = 100 * step                   # the block's step
        blocks.append(x)
    _compare(device, np.stack(blocks), cos, sin)
    _compare(device, np.stack(blocks)[:, :, ::-1].copy(), cos, sin)          # the tails in the second half's sums


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [1, 7])
def test_borders_of_the_step(device, dim, new):
    """A largest magnitude of 127 * 2^e with a tail outwards, inwards or none, in either half, of either sign."""
    half = dim // 2
    cos, sin = np.ones((new, dim), np.float32), np.full((new, dim), 2.0 ** -70, np.float32)
    blocks = []
    for top in (127.0, -127.0, 127 * 2.0 ** -9, -127 * 2.0 ** 30):
        for tail in (1.0, -1.0, 0.0):
            for at, other in ((3, half + 3), (half + 5, 5)):
                x = np.full((new, dim), top / 8, np.float32)
                x[new - 1, at], x[new - 1, other] = top, tail * abs(top) / 127
                blocks.append(x)
    _compare(device, np.stack(blocks), cos, sin)


@pytest.mark.parametrize("seed", range(3))
def test_products_of_any_sizes(device, seed):
    """Tables and values whose products lie 0 to 80 bits apart, cancel, or are nearly a border."""
    rng = np.random.default_rng(seed)
    cos = (rng.integers(-8, 9, (4, 64)) * 0.25).astype(np.float32)
    sin = (rng.integers(-1, 2, (4, 64)) * 2.0 ** rng.integers(-80, 1, (4, 64))).astype(np.float32)
    x = (rng.integers(-250, 251, (24, 4, 64)) * 0.5).astype(np.float32)
    x[:8] += np.float32(2.0 ** -14) * rng.integers(-1, 2, (8, 4, 64)).astype(np.float32)
    _compare(device, x, cos, sin)
