"""The 8-bit serving operators of this library as measurable cases: rows quantised to int8 (with or
without the norm in front), products of int8 rows and channels, keys and values rotated and appended to
a paged int8 cache, attention over that cache.

`run` computes a case either in plain torch operations (own = False) or through the library
(own = True); `exact` gives the same results from the definitions in 64 bits.

The definitions:
  row quantisation   s = fp32(max|y| / 127), q = round_half_even(y / s); s = 0 and q = 0 where max|y| < 2^-100
                     (with the norm: y = x / sqrt(mean(x^2) + eps) * gamma, x = round(a + b) to the type)
  int8 product       c[i, j] = sum_k a[i, k] w[j, k] * sa[i] * sw[j] (+ residual[i, j])
  cache block        one page of one head holds int8 values times 2^e; 2^e is the smallest power of two
                     with max|x| <= 127 * 2^e over what was appended to it since its first token; when a
                     later token raises e, the values held already are rounded to the new step
  attention          softmax over the cached tokens j <= position of the query, rows with none: zeros
"""
import math
import random

import numpy as np
import torch

own = False

EPS = float(np.float32(1e-5))
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SMALLEST = 2.0 ** -100   # rows whose largest magnitude lies below it are stored as zeros
LOWEST_EXPONENT = -126


# ---- the cases ------------------------------------------------------------------------------------

def listed():
    return [
        # the norm in front of a projection, one token being decoded: latency
        dict(name="norm_quantize_token", op="quantize", type="f32", rows=1, cols=2048, norm=True, add=True),
        # the input of a down projection, a whole prefill batch: bandwidth
        dict(name="quantize_prefill", op="quantize", type="f32", rows=4096, cols=8192, norm=False, add=False),
        # output projection of one decoded token, residual added: latency
        dict(name="product_token", op="product", type="f32", m=1, n=2048, k=2048, residual=True),
        # vocabulary projection of a few sequences: streams the weights
        dict(name="product_vocab", op="product", type="f32", m=8, n=128256, k=2048, residual=False),
        # gate projection of a ragged prefill
        dict(name="product_prefill", op="product", type="f32", m=509, n=8192, k=2048, residual=False),
        # down projection of a large batch of prompts: the matrix cores' rate
        dict(name="product_batch", op="product", type="bf16", m=4096, n=8192, k=8192, residual=True),
        # one new token of each of 64 short conversations
        dict(name="append_tokens", op="append", type="f32", seqs=64, new_lo=1, new_hi=1, len_lo=1, len_hi=64,
             kv_heads=8, rep=4, head_dim=64, page=32, pad=0, lengths=1),
        # prompts entering the cache, ragged, some of them behind what is cached already
        dict(name="append_prompts", op="append", type="bf16", seqs=8, new_lo=65, new_hi=1024, len_lo=65,
             len_hi=1300, kv_heads=8, rep=4, head_dim=128, page=64, pad=5, lengths=2),
        # decoding one sequence (prompt of 512 and 128 tokens behind it): latency
        dict(name="attend_token", op="attend", type="f32", seqs=1, new_lo=1, new_hi=1, len_lo=640, len_hi=640,
             kv_heads=8, rep=4, head_dim=64, page=64, pad=0, lengths=3),
        # decoding a batch of long ragged sequences: reads the cache once
        dict(name="attend_batch", op="attend", type="bf16", seqs=64, new_lo=1, new_hi=1, len_lo=100, len_hi=16384,
             kv_heads=8, rep=4, head_dim=128, page=64, pad=0, lengths=4),
        # prefill of one prompt: the matrix cores
        dict(name="attend_prompt", op="attend", type="f32", seqs=1, new_lo=2048, new_hi=2048, len_lo=2048,
             len_hi=2048, kv_heads=8, rep=4, head_dim=64, page=64, pad=0, lengths=5),
        # prompts fed in chunks, mixed with sequences that decode, small pages
        dict(name="attend_chunks", op="attend", type="f16", seqs=6, new_lo=1, new_hi=512, len_lo=512, len_hi=16384,
             kv_heads=8, rep=4, head_dim=128, page=16, pad=3, lengths=6),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["quantize", "product", "product", "append", "attend", "attend"])
    kind = rng.choice(["f32", "f32", "f16", "bf16"])
    if op == "quantize":
        norm = rng.random() < 0.6
        while True:
            rows, cols = _log_int(rng, 1, 8192), _log_int(rng, 17, 16384)
            if rng.random() < 0.6:
                cols = max(64, cols // 64 * 64)
            if rows * cols <= 4096 * 8192 // (2 if norm else 1):
                break
        return dict(op=op, type=kind, rows=rows, cols=cols, norm=norm, add=norm and rng.random() < 0.5)
    if op == "product":
        while True:
            m, n, k = _log_int(rng, 1, 4096), _log_int(rng, 16, 32768), _log_int(rng, 32, 16384)
            if rng.random() < 0.7:
                n, k = max(16, n // 64 * 64), max(32, k // 64 * 64)
            if m * n * k <= 4096 * 8192 * 8192 and n * k <= 128256 * 2048:
                break
        return dict(op=op, type=kind, m=m, n=n, k=k, residual=rng.random() < 0.4)
    heads = dict(kv_heads=rng.choice([1, 2, 4, 8, 16]), rep=rng.choice([1, 2, 3, 4, 6, 8]),
                 head_dim=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128]),
                 pad=rng.choice([0, 0, 1, 7]), lengths=rng.randrange(1 << 30))
    while True:
        seqs = _log_int(rng, 1, 128)
        new_hi = 1 if rng.random() < 0.4 else _log_int(rng, 1, 2048)
        len_hi = _log_int(rng, 1, 16384)
        case = dict(op=op, type=kind, seqs=seqs, new_lo=1, new_hi=new_hi, len_lo=1, len_hi=len_hi, **heads)
        new, length = _lengths(case)
        held = sum(length) * case["kv_heads"] * case["head_dim"]
        if op == "append":
            if held <= 1 << 23:
                return case
        elif held <= 200 << 20 and _pairs(new, length) * case["kv_heads"] * case["rep"] * case["head_dim"] <= 1 << 34:
            return case


def _lengths(case):
    """(new tokens, tokens held with them) of every sequence of a case."""
    rng = random.Random(case["lengths"])
    length = [_log_int(rng, case["len_lo"], case["len_hi"]) for _ in range(case["seqs"])]
    if case["seqs"] > 1:
        length[rng.randrange(case["seqs"])] = case["len_hi"]
    new = [min(n, _log_int(rng, case["new_lo"], case["new_hi"])) for n in length]
    return new, length


def _pairs(new, length):
    """Visible (query, key) pairs: query i of a sequence sees length - new + i + 1 tokens."""
    return sum(n * (l - n) + n * (n + 1) // 2 for n, l in zip(new, length))


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "quantize":
        elems = case["rows"] * case["cols"]
        moved = elems * (size + 1) + case["rows"] * 4
        if case["norm"]:
            moved += case["cols"] * 4
        if case["add"]:
            moved += 2 * elems * size
        return {"bytes": moved, "flops": elems * (8 if case["norm"] else 4)}
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + 4 * (m + n) + m * n * size * (2 if case["residual"] else 1),
                "flops": 2 * m * n * k}
    new, length = _lengths(case)
    g, d, heads, page = case["kv_heads"], case["head_dim"], case["kv_heads"] * case["rep"], case["page"]
    tokens = sum(new)
    if case["op"] == "append":
        touched = sum((l - 1) // page - (l - n) // page + 1 for n, l in zip(new, length))
        return {"bytes": tokens * d * (2 * heads * size + 2 * g * (size + 1)) + tokens * d * 8 + touched * g * 16
                + touched * 4 + case["seqs"] * 8, "flops": tokens * d * (3 * heads + 6 * g)}
    held = sum((l + page - 1) // page for l in length)
    return {"bytes": 2 * tokens * heads * d * size + 2 * sum(length) * g * d + held * (8 * g + 4) + case["seqs"] * 8,
            "flops": 4 * _pairs(new, length) * heads * d}


# ---- inputs ---------------------------------------------------------------------------------------

class State:
    pass


def _normal(gen, shape, kind=torch.float32, std=1.0):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * std).to(kind)


def _int8(gen, shape, std):
    out = torch.empty(shape, dtype=torch.int8, device="cuda")
    flat = out.view(-1)
    step = 1 << 26
    for i in range(0, flat.numel(), step):
        part = torch.randn(min(step, flat.numel() - i), generator=gen, device="cuda")
        flat[i:i + step] = (part * std).round_().clamp_(-127, 127).to(torch.int8)
    return out


def _padded(cols):
    return (cols + 15) // 16 * 16


def prepare(case, seed):
    st = _inputs(case, seed)
    if own:
        from rmlk_amd import kernels
        st.lib = kernels
        if case["op"] in ("append", "attend"):
            st.cache = kernels.PagedCache(st.k_cache, st.v_cache, st.k_scale, st.v_scale)
            st.batch = kernels.PagedBatch(st.first, st.length, st.table, tokens=st.tokens, max_new=max(st.new),
                                          max_len=max(st.lengths))
    return st


def _inputs(case, seed):
    st = State()
    st.case = case
    kind = TYPES[case["type"]]
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    if case["op"] == "quantize":
        rows, cols = case["rows"], case["cols"]
        # activations: most channels alike, a few much larger
        channel = torch.exp(0.5 * torch.randn(cols, generator=gen, device="cuda"))
        st.x = (torch.randn(rows, cols, generator=gen, device="cuda") * channel).to(kind)
        st.add = (torch.randn(rows, cols, generator=gen, device="cuda") * channel).to(kind) if case["add"] else None
        st.gamma = 0.5 + torch.rand(cols, generator=gen, device="cuda") if case["norm"] else None
        st.sum_out = torch.zeros_like(st.x) if case["add"] else None
        st.q = torch.zeros(rows, _padded(cols), dtype=torch.int8, device="cuda")
        st.scale = torch.zeros(rows, device="cuda")
    elif case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        st.a = torch.zeros(m, _padded(k), dtype=torch.int8, device="cuda")
        st.w = torch.zeros(n, _padded(k), dtype=torch.int8, device="cuda")
        st.a[:, :k] = _int8(gen, (m, k), 32.0)
        st.w[:, :k] = _int8(gen, (n, k), 32.0)
        st.a_scale = (0.5 + torch.rand(m, generator=gen, device="cuda")) * (4.0 / 127)
        st.w_scale = (0.5 + torch.rand(n, generator=gen, device="cuda")) * (0.08 / 127)
        st.residual = _normal(gen, (m, n), kind) if case["residual"] else None
        st.out = torch.zeros(m, n, dtype=kind, device="cuda")
    else:
        _paged_inputs(st, case, kind, gen)
    return st


def _paged_inputs(st, case, kind, gen):
    g, d, page = case["kv_heads"], case["head_dim"], case["page"]
    heads = g * case["rep"]
    st.new, st.lengths = _lengths(case)
    counts = [(l + page - 1) // page for l in st.lengths]
    pages = sum(counts) + 2
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    st.table = torch.zeros(case["seqs"], max(counts), dtype=torch.int32, device="cuda")
    at = 0
    for s, c in enumerate(counts):
        st.table[s, :c] = order[at:at + c]
        at += c
    first = [0]
    for n in st.new:
        first.append(first[-1] + n)
    st.rows = first[-1]
    st.tokens = st.rows + case["pad"]     # a padded batch: rows behind the last sequence belong to nobody
    st.starts = first
    st.first = torch.tensor(first, dtype=torch.int32, device="cuda")
    st.length = torch.tensor(st.lengths, dtype=torch.int32, device="cuda")
    # the cache as earlier appends left it: values of about 4 steps' deviation, steps that differ by block
    st.k_cache = _int8(gen, (pages, g, page, d), 30.0)
    st.v_cache = _int8(gen, (pages, g, d, page), 30.0)
    choice = torch.tensor([2.0 ** -6, 2.0 ** -5, 2.0 ** -5, 2.0 ** -4], device="cuda")
    st.k_scale = choice[torch.randint(0, 4, (pages, g), generator=gen, device="cuda")].contiguous()
    st.v_scale = choice[torch.randint(0, 4, (pages, g), generator=gen, device="cuda")].contiguous()
    st.q = _normal(gen, (st.tokens, heads, d), kind, 1.5)
    st.out = torch.zeros(st.tokens, heads, d, dtype=kind, device="cuda")
    if case["op"] == "append":
        st.k = _normal(gen, (st.tokens, g, d), kind)
        st.v = _normal(gen, (st.tokens, g, d), kind)
        half = d // 2
        freq = 500000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) * 2 / d)
        angle = torch.arange(max(st.lengths), device="cuda", dtype=torch.float64)[:, None] * freq
        angle = torch.cat([angle, angle], dim=1)
        st.cos, st.sin = angle.cos().float(), angle.sin().float()


# ---- one pass -------------------------------------------------------------------------------------

def run(st):
    op = st.case["op"]
    if op == "quantize":
        return _run_quantize(st)
    if op == "product":
        return _run_product(st)
    if op == "append":
        return _run_append(st)
    return _run_attend(st)


def _run_quantize(st):
    cols = st.case["cols"]
    if own:
        if st.case["norm"]:
            st.lib.rmsnorm_quantize_rows(st.x, st.gamma, EPS, st.q, st.scale, add=st.add, sum_out=st.sum_out)
        else:
            st.lib.quantize_rows(st.x, st.q, st.scale)
        values, scale, total = st.q[:, :cols] * st.scale[:, None], st.scale, st.sum_out
    else:
        x, total = st.x, None
        if st.add is not None:
            x = total = (st.x.float() + st.add.float()).to(st.x.dtype)
        y = x.double()                    # (the rounding to a step decides at borders: 64 bits)
        if st.gamma is not None:
            y = y / torch.sqrt((y * y).mean(dim=1, keepdim=True) + EPS) * st.gamma.double()
        top = y.abs().amax(dim=1, keepdim=True)
        scale = torch.where(top < SMALLEST, torch.zeros_like(top), top / 127).float()
        step = torch.where(scale > 0, scale, torch.ones_like(scale)).double()
        q = torch.where(scale > 0, (y / step).round().clamp(-127, 127), torch.zeros_like(y)).to(torch.int8)
        values, scale = q.float() * scale, scale[:, 0]
    return [values, scale] if total is None else [values, scale, total]


def _run_product(st):
    if own:
        st.lib.matmul_int8(st.a, st.a_scale, st.w, st.w_scale, st.out, k=st.case["k"], residual=st.residual)
        return st.out
    k = st.case["k"]
    c = (st.a[:, :k].float() @ st.w[:, :k].float().t()) * st.a_scale[:, None] * st.w_scale[None, :]
    if st.residual is not None:
        c = c + st.residual.float()
    return c.to(st.out.dtype)


def _rotate(x, cos, sin):
    half = x.shape[-1] // 2
    turned = torch.cat([-x[..., half:], x[..., :half]], dim=-1)
    return x * cos[:, None] + turned * sin[:, None]


def _power(e):
    return torch.ldexp(torch.ones_like(e, dtype=torch.float64), e)


def _append_blocks(cache, scale, page, slot, x, slots_last):
    """One of K and V: x [tokens, heads, dim] in 64 bits goes to (page, slot) of the int8 cache."""
    pages, heads = scale.shape
    size = cache.shape[3] if slots_last else cache.shape[2]
    top = torch.zeros(pages, heads, dtype=torch.float64, device=x.device)
    top.scatter_reduce_(0, page[:, None].expand(-1, heads), x.abs().amax(dim=2), "amax")
    start = torch.full((pages,), size, dtype=torch.int64, device=x.device)
    start.scatter_reduce_(0, page, slot, "amin")                # first new slot; size: block not touched
    mant, expo = torch.frexp(top)
    need = torch.where(mant <= 127 / 128, expo - 7, expo - 6)
    need = torch.where(top > 0, need, torch.full_like(need, LOWEST_EXPONENT)).clamp(LOWEST_EXPONENT, 127)
    held = torch.frexp(scale.double())[1] - 1
    fresh = (start == 0)[:, None]
    e = torch.where(fresh, need, torch.maximum(need, held))
    touched = (start < size)[:, None]
    e = torch.where(touched, e, held)
    # values held already, in the new step
    old = torch.arange(size, device=x.device)[None, :] < torch.where(start < size, start, torch.zeros_like(start))[:, None]
    shrink = _power(torch.where(fresh, torch.zeros_like(e), held - e)).float()
    if slots_last:
        rounded = (cache.float() * shrink[:, :, None, None]).round()
        cache.copy_(torch.where(old[:, None, None, :], rounded, cache.float()))
    else:
        rounded = (cache.float() * shrink[:, :, None, None]).round()
        cache.copy_(torch.where(old[:, None, :, None], rounded, cache.float()))
    q = (x * _power(-e)[page][:, :, None]).round().clamp(-127, 127).to(torch.int8)
    if slots_last:
        cache[page, :, :, slot] = q
    else:
        cache[page, :, slot] = q
    scale.copy_(torch.where(touched, _power(e).float(), scale))


def _run_append(st):
    if own:
        st.lib.paged_append(st.cache, st.batch, st.k, st.v, cos=st.cos, sin=st.sin, q=st.q, q_out=st.out)
    else:
        size = st.case["page"]
        t = torch.arange(st.rows, device="cuda")
        first, length = st.first.long(), st.length.long()
        seq = torch.searchsorted(first[1:], t, right=True)
        pos = length[seq] - (first[seq + 1] - t)
        page, slot = st.table[seq, pos // size].long(), pos % size
        cos, sin = st.cos[pos].double(), st.sin[pos].double()
        # (which step a value is rounded to decides at borders: 64 bits)
        _append_blocks(st.k_cache, st.k_scale, page, slot, _rotate(st.k[:st.rows].double(), cos, sin), False)
        _append_blocks(st.v_cache, st.v_scale, page, slot, st.v[:st.rows].double(), True)
        st.out[:st.rows] = _rotate(st.q[:st.rows].double(), cos, sin).to(st.out.dtype)
    return [st.out, st.k_cache * st.k_scale[:, :, None, None], st.v_cache * st.v_scale[:, :, None, None],
            st.k_scale, st.v_scale]


def _run_attend(st):
    case = st.case
    scale = 1.0 / math.sqrt(case["head_dim"])
    if own:
        st.lib.paged_attention(st.cache, st.batch, st.q, st.out, scale=scale, scale_is_mul=True)
        return st.out
    g, rep, d, size = case["kv_heads"], case["rep"], case["head_dim"], case["page"]
    for s in range(case["seqs"]):
        n, l, at = st.new[s], st.lengths[s], st.starts[s]
        pages = st.table[s, :(l + size - 1) // size].long()
        k = (st.k_cache[pages].float() * st.k_scale[pages][:, :, None, None]).permute(1, 0, 2, 3).reshape(g, -1, d)
        v = (st.v_cache[pages].float() * st.v_scale[pages][:, :, None, None]).permute(1, 0, 3, 2).reshape(g, -1, d)
        k, v = k[:, :l], v[:, :l]
        q = st.q[at:at + n].float().reshape(n, g, rep, d).permute(1, 2, 0, 3).reshape(g, rep * n, d)
        scores = (q @ k.transpose(1, 2).contiguous()) * scale
        last = torch.arange(l - n, l, device="cuda").repeat(rep)
        scores = scores.masked_fill(torch.arange(l, device="cuda")[None, :] > last[:, None], -math.inf)
        p = torch.exp(scores - scores.amax(dim=2, keepdim=True))
        o = (p @ v.contiguous()) / p.sum(dim=2, keepdim=True)
        st.out[at:at + n] = o.reshape(g, rep, n, d).permute(2, 0, 1, 3).reshape(n, g * rep, d).to(st.out.dtype)
    return st.out


# ---- the same from the definitions, in 64 bits ------------------------------------------------------

def exact(case, seed):
    st = _inputs(case, seed)
    if case["op"] == "quantize":
        total = None
        x = st.x.double()
        if case["add"]:
            total = x + st.add.double()
            x = total.to(st.x.dtype).double()
        if case["norm"]:
            x = x * (st.gamma.double() * torch.rsqrt(x.square().sum(1, keepdim=True) / case["cols"] + EPS))
        top = x.abs().max(dim=1, keepdim=True).values
        scale = (top / 127).to(torch.float32).double() * (top >= SMALLEST)
        q = torch.nan_to_num(torch.round(x / scale), nan=0.0, posinf=0.0, neginf=0.0)
        out = [torch.clamp(q, -127, 127) * scale, scale[:, 0]]
        return out if total is None else out + [total]
    if case["op"] == "product":
        k = case["k"]
        c = torch.matmul(st.a[:, :k].double() * st.a_scale.double()[:, None],
                         (st.w[:, :k].double() * st.w_scale.double()[:, None]).t().contiguous())
        return c if st.residual is None else c + st.residual.double()
    if case["op"] == "append":
        return _exact_append(st)
    return _exact_attend(st)


def _exact_append(st):
    case, size = st.case, st.case["page"]
    half = case["head_dim"] // 2
    out = torch.zeros(st.out.shape, dtype=torch.float64, device="cuda")
    k_held, v_held = st.k_cache.double(), st.v_cache.double()
    k_step, v_step = st.k_scale.double(), st.v_scale.double()

    def turn(x, lo, hi):
        c, s = st.cos[lo:hi].double().unsqueeze(1), st.sin[lo:hi].double().unsqueeze(1)
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * c[..., :half] - b * s[..., :half], b * c[..., half:] + a * s[..., half:]], dim=-1)

    def put(held, step, page, begin, x):
        """x [heads, tokens, dim] behind `begin` tokens of a block held as [heads, size, dim] integers."""
        for h in range(x.shape[0]):
            top = float(x[h].abs().max())
            new = LOWEST_EXPONENT if top == 0 else max(LOWEST_EXPONENT, math.ceil(math.log2(top)) - 8)
            while 127 * 2.0 ** new < top:
                new += 1
            if begin > 0:
                before = round(math.log2(float(step[page, h])))
                new = max(new, before)
                held[h, :begin] = torch.round(held[h, :begin] * 2.0 ** (before - new))
            held[h, begin:begin + x.shape[1]] = torch.clamp(torch.round(x[h] * 2.0 ** -new), -127, 127)
            step[page, h] = 2.0 ** new

    for s in range(case["seqs"]):
        n, l, at = st.new[s], st.lengths[s], st.starts[s]
        out[at:at + n] = turn(st.q[at:at + n].double(), l - n, l)
        k = turn(st.k[at:at + n].double(), l - n, l).transpose(0, 1)
        v = st.v[at:at + n].double().transpose(0, 1)
        pos = l - n
        while pos < l:
            page, begin = int(st.table[s, pos // size]), pos % size
            take = min(size - begin, l - pos)
            i = pos - (l - n)
            put(k_held[page], k_step, page, begin, k[:, i:i + take])
            put(v_held[page].transpose(1, 2), v_step, page, begin, v[:, i:i + take])
            pos += take
    return [out, k_held * k_step[..., None, None], v_held * v_step[..., None, None], k_step, v_step]


def _exact_attend(st):
    case, size, rep = st.case, st.case["page"], st.case["rep"]
    out = torch.zeros(st.out.shape, dtype=torch.float64, device="cuda")
    for s in range(case["seqs"]):
        n, l, at = st.new[s], st.lengths[s], st.starts[s]
        pages = st.table[s, :-(-l // size)].long()
        hidden = torch.ones(n, l, dtype=torch.bool, device="cuda").triu(l - n + 1)
        for h in range(case["kv_heads"]):
            k = (st.k_cache[pages, h].double() * st.k_scale[pages, h].double()[:, None, None]).flatten(0, 1)[:l]
            v = (st.v_cache[pages, h].double() * st.v_scale[pages, h].double()[:, None, None]).transpose(1, 2)
            v = v.reshape(-1, case["head_dim"])[:l]
            for r in range(h * rep, (h + 1) * rep):
                scores = st.q[at:at + n, r].double() @ k.t() / math.sqrt(case["head_dim"])
                out[at:at + n, r] = torch.softmax(scores.masked_fill(hidden, -math.inf), dim=1) @ v
    return out
