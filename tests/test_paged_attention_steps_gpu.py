"""Attention over a paged cache whose blocks have very different steps of V: a row is as exact as what it sees, whatever
the steps of pages that it does not see, or sees with next to no weight."""
import numpy as np
import pytest

import int8_reference as ref
import test_int8_serving_gpu as serving

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES, U, U_OUT, TINY = serving.TYPES, serving.U, serving.U_OUT, serving.TINY


def _paged(device, seqs, size, heads, dim, capacity, seed, v_steps, scores=None):
    """A cache whose page j of sequence s has V's step v_steps[s][j] (lists repeat); with `scores`, keys that give
    every token of the page the score scores[s][j] (in units of scale) under a query that is 8 in dim 0 and 0 beyond."""
    p = serving.Paged(device, seqs, size, heads, dim, capacity, seed)
    for s in range(seqs):
        for j, page in enumerate(p.table[s]):
            p.ref.v_scale[page] = v_steps[s % len(v_steps)][j % len(v_steps[s % len(v_steps)])]
            if scores is not None:
                p.ref.k[page], p.ref.k_scale[page] = 0, 1.0
                p.ref.k[page][..., 0] = scores[s % len(scores)][j % len(scores[s % len(scores)])]
    for name in ("k", "k_scale", "v_scale"):
        getattr(p.dev, name).copy_(torch.from_numpy(getattr(p.ref, name)))
    return p


def _run(p, kind, new, length, rep, q=None, bounds=None):
    """Tolerance, row by row. p_t: the weights of the tokens that the row sees. The relative error of a weight (a score's
    4 (2^-22 + (dim + 4) u) * bound, 64 u of the running sums; 2^-11 where 16-bit types round it) reaches the result times
    sum p_t |v_t|. A weight is a half (or two), relative to a reference that leaves the largest product of a weight and
    a step at least 2^(1/2): what lies below the last bit of a half, 2^-25, is lost, for each of n tokens of at most 127
    steps. Then the output's rounding."""
    first = np.concatenate([[0], np.cumsum(new)])
    rows, heads = int(first[-1]), p.heads * rep
    if q is None:
        q = p.rng.standard_normal((rows, heads, p.dim)).astype(np.float32)
    dq = serving._dev(q, p.device, TYPES[kind])
    out = torch.full((rows, heads, p.dim), 7.0, dtype=TYPES[kind], device=p.device)
    flag = torch.zeros(1, dtype=torch.int32, device=p.device)
    max_new, max_len = bounds or (max(new), max(length))
    scale = 0.125
    serving._k().paged_attention(p.dev, p.batch(first, length, rows, max_new, max_len), dq, out, scale=scale,
                                 scale_is_mul=True, err_flag=flag)
    assert flag.item() == 0
    q64, got = serving._f64(dq), serving._f64(out)
    for s, (n, l) in enumerate(zip(new, length)):
        for g in range(p.heads):
            k, v = p.ref.tokens(p.table[s], l, g)
            steps = np.repeat([np.float64(p.ref.v_scale[p.table[s, j], g]) for j in range(-(-l // p.size))], p.size)[:l]
            for r in range(rep):
                h = g * rep + r
                mine, x = got[first[s]:first[s + 1], h], q64[first[s]:first[s + 1], h]
                want, bound = ref.attend(x, k, v, l, scale)
                for i in range(n):
                    sees = l - n + i + 1
                    if sees <= 0:
                        assert not mine[i].any()
                        continue
                    score = k[:sees] @ x[i] * scale
                    w = np.exp(score - score.max())
                    w /= w.sum()
                    relative = 4 * (2.0 ** -22 + (p.dim + 4) * U) * bound[i] + 64 * U + (0.0 if kind == "f32" else 2.0 ** -11)
                    tol = (relative * (w @ np.abs(v[:sees])) + sees * 127 * 2.0 ** -25.5 * (w * np.abs(steps[:sees])).max()
                           + 1.01 * U_OUT[kind] * np.abs(want[i]) + TINY[kind])
                    off = np.abs(mine[i] - want[i])
                    assert np.all(off <= tol), (s, h, i, float(np.max(off / tol)), float(np.abs(want[i]).max()))
    return out


def _query(rows, heads, dim, value=8.0):
    q = np.zeros((rows, heads, dim), np.float32)
    q[..., 0] = value
    return q


GAPS = [0, 3, 6, 7, 12, 15, 20, 24, 25, 26, 30, 45, 70]


@pytest.mark.parametrize("gap", GAPS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,rep", [(4, 4), (8, 2), (60, 2), (60, 4)])
def test_hidden_page_of_a_larger_step(device, gap, dim, new, rep):
    """A prompt (few rows and many) whose first rows see only pages of a small step; a later page of the same tile
    of keys has a step 2^gap larger, then it falls again."""
    low = 2.0 ** -30
    for kind in ("f32", "bf16"):
        for steps in ([low, low * 2.0 ** gap], [low, low, low * 2.0 ** gap, low], [low * 2.0 ** gap, low]):
            p = _paged(device, 2, 16, 2, dim, 160, gap + new, [steps, steps[::-1]])
            _run(p, kind, [new, new], [new + 12, new + 75], rep)


@pytest.mark.parametrize("gap", [0, 5, 9, 13])
def test_hidden_page_of_a_larger_step_half(device, gap):
    low = 2.0 ** -9
    for new, rep in ((4, 4), (60, 2)):
        p = _paged(device, 2, 16, 2, 64, 160, gap, [[low, low * 2.0 ** gap], [low * 2.0 ** gap, low, low]])
        _run(p, "f16", [new, new], [new + 12, new + 75], rep)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("new,length", [(1, 400), (3, 333), (2, 2500), (70, 400), (200, 1500)])
@pytest.mark.parametrize("seed", range(4))
def test_steps_and_weights_that_move_apart(device, kind, new, length, seed):
    """Steps from 2^-100 to 2^20 and weights from e^-254 up, page by page in every order; keys split over blocks in
    the longer calls."""
    rng = np.random.default_rng(seed)
    pages = -(-length // 16)
    scores = rng.integers(-127, 128, pages)
    exps = rng.integers(-100, 21, pages)
    if seed == 1:        # large steps where there is no weight, the weight on ever smaller ones
        scores, exps = np.sort(scores), np.sort(exps)[::-1]
    elif seed == 2:      # the products of weight and step nearly alike
        exps = np.clip(np.rint(-scores * np.log2(np.e)) % 120 - 100, -100, 20).astype(int)
    elif seed == 3:      # long runs within a few steps, then a jump
        exps, scores = np.repeat(exps[::6], 6)[:pages] + rng.integers(0, 5, pages), scores // 8
    p = _paged(device, 2, 16, 1, 64, length, seed, [2.0 ** exps.astype(np.float64)], [scores])
    _run(p, kind, [new, min(new, 2)], [length, max(2, length - 37)], 2, q=_query(new + min(new, 2), 2, 64))


@pytest.mark.parametrize("new", [1, 80])
def test_pages_of_zeros_beside_others(device, new):
    """Blocks of nothing but zeros have the smallest step there is; they carry weight all the same."""
    p = _paged(device, 2, 32, 2, 64, 320, 5, [[1.0, 2.0 ** -126, 0.5], [2.0 ** -126]])
    zeros = p.ref.v_scale == np.float32(2.0 ** -126)
    p.ref.v[zeros] = 0
    p.dev.v.copy_(torch.from_numpy(p.ref.v))
    for kind in TYPES:
        _run(p, kind, [new, new], [300, 200], 4)


def test_marked_pages_among_far_steps(device):
    """A block that is no number reaches the rows that see it and no others, beside steps of any distance."""
    for new, rep in ((5, 2), (70, 2)):
        p = _paged(device, 1, 16, 2, 64, 160, 7, [[2.0 ** -20, 2.0 ** 15, 2.0 ** -40]])
        p.ref.v_scale[p.table[0, 3], 1] = np.nan            # tokens 48 .. 63 of head 1
        p.dev.v_scale.copy_(torch.from_numpy(p.ref.v_scale))
        length = 50
        q = p.rng.standard_normal((new, 4, 64)).astype(np.float32)
        out = torch.zeros(new, 4, 64, device=device)
        batch = p.batch([0, new], [length], new, new, length)
        serving._k().paged_attention(p.dev, batch, serving._dev(q, device), out, scale=0.125, scale_is_mul=True)
        sees = length - new + np.arange(new) + 1
        bad = torch.isnan(out).any(dim=2).cpu().numpy()
        assert np.array_equal(bad[:, 2], sees > 48) and np.array_equal(bad[:, 3], sees > 48) and not bad[:, :2].any()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,rep", [(1, 4), (8, 4), (60, 3)])
def test_steps_that_are_no_powers_of_two(device, kind, dim, new, rep):
    """Scales of the caller's own making; some pages of theirs beside some of powers of two, near and far."""
    for steps in ([0.0131], [0.0156, 4 / 3], [0.25, 0.3], [0.5, 0.25, 0.125, 0.7], [1.9999999, 2.0 ** -30, 0.01]):
        p = _paged(device, 2, 16, 2, dim, 240, 3, [steps, steps[::-1]])
        _run(p, kind, [new, new], [new + 12, new + 170], rep)


@pytest.mark.parametrize("new", [1, 60])
def test_odd_steps_of_zeros_and_of_constants(device, new):
    """A V of zeros gives zeros, one of ones its step, whatever the step."""
    for kind in TYPES:
        for step in (0.0131, 0.0156, 4 / 3, 5e-3, 0.9999):
            p = _paged(device, 1, 16, 1, 64, 120, 4, [[step]])
            for value in (0, 1, -1):
                p.ref.v[:] = value
                p.dev.v.copy_(torch.from_numpy(p.ref.v))
                out = _run(p, kind, [new], [new + 50], 2)
                if value == 0:
                    assert not out.any()


@pytest.mark.parametrize("new", [1, 60])
def test_steps_of_a_caller_that_are_subnormal_zero_or_negative(device, new):
    for steps in ([3e-40], [1e-39, 2.0 ** -126], [0.0], [0.0, 0.5, 0.0], [-0.3, 0.3], [-0.5]):
        p = _paged(device, 1, 16, 1, 64, 120, 8, [steps])
        _run(p, "f32", [new], [new + 50], 2)


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_extreme_steps(device, kind, new):
    """The smallest and the largest step a float has."""
    p = _paged(device, 1, 16, 1, 64, 200, 6, [[2.0 ** -126, 2.0 ** -126, 2.0 ** 119, 2.0 ** -126]])
    _run(p, kind, [new], [new], 2)
    _run(p, kind, [new], [new + 60], 2)


@pytest.mark.parametrize("new,length", [(1, 50), (1, 900), (3, 5000), (60, 200), (60, 3000)])
def test_values_next_to_the_largest_float(device, new, length):
    """Every value as large as a float can be: the results are means of them, in one piece, of wavefronts, of splits."""
    p = _paged(device, 2, 16, 1, 64, length, 9, [[2.0 ** 121]])
    p.ref.v[:] = np.where(p.ref.v < 0, -127, 127)
    p.dev.v.copy_(torch.from_numpy(p.ref.v))
    for scores in ([0], [5, -5, 3]):
        for j, page in enumerate(p.table.reshape(-1)):
            p.ref.k[page], p.ref.k_scale[page] = 0, 1.0
            p.ref.k[page][..., 0] = scores[j % len(scores)]
        p.dev.k.copy_(torch.from_numpy(p.ref.k))
        p.dev.k_scale.copy_(torch.from_numpy(p.ref.k_scale))
        _run(p, "f32", [new, new], [length, length - 7], 2, q=_query(2 * new, 2, 64))
