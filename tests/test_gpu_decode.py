"""The decoding operators on the GPU against plain implementations in 64 bits.

Tolerances, from the arithmetic (u = 2^-11 for fp16, 2^-8 for bf16, the rounding of the compute dtype):
  rotated Q: one rounding of the result and fp32 arithmetic on it: u·|q| + 2^-21·(|a| + |b|).
  8-bit codes: x·(c/A) in fp32 has a relative error below 2^-21, so a code differs from the 64-bit quotient by at
    most half a step plus 127·2^-21 (int8), half of e4m3's spacing plus 448·2^-21 (e4m3); scales by 2^-21 relative.
  reading back: code·scale is one fp32 product rounded once: equal bit for bit.
  attention: the weights (each <= 1 before the sum divides them) are rounded to the compute dtype, the output once
    more: 2u·max|v|, plus 2^-25 per key (fp16 weights below 2^-14) and 1e-4·max|v| for fp32 scores of up to ~30.
    Log-sum-exp, no 16-bit rounding in it: 1e-4.
  sampling: weights within 2^-22 relative of the 64-bit ones plus half a unit, so the running sum at a token is
    within total·2^-22 + vocab/2 of the 64-bit one, and the drawn token's interval holds u·total to twice that.
"""
import math

import numpy as np
import pytest
import torch

from autoane_b200 import _lib, decode

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F16, BF16, I8, E4 = torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


# ---- cache ----------------------------------------------------------------------------------------------------
def rotated(x, table, positions, rot, interleaved):
    """x [n, heads, 64] in 64 bits, turned by the table's angles."""
    if not rot:
        return x
    t = table.double()[positions.long()][:, None]
    y = x.clone()
    i = torch.arange(rot // 2, device="cuda")
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    y[..., ia] = x[..., ia] * t[..., 0] - x[..., ib] * t[..., 1]
    y[..., ib] = x[..., ib] * t[..., 0] + x[..., ia] * t[..., 1]
    return y


KV_CASES = [  # tokens, heads, kv_heads, cache type, compute dtype, page, rot, interleaved
    (1, 15, 5, I8, F16, 16, 64, False),
    (1, 1, 1, E4, BF16, 8, 16, True),
    (7, 9, 3, I8, BF16, 8, 48, False),
    (37, 8, 2, E4, F16, 32, 48, True),
    (300, 12, 12, F16, F16, 64, 32, False),
    (1001, 15, 5, BF16, BF16, 128, 0, False),
    (3000, 24, 6, I8, F16, 256, 32, True),
    (2500, 32, 8, E4, BF16, 1024, 64, False),
]


@pytest.mark.parametrize("n,heads,kv,kind,dtype,page,rot,inter", KV_CASES)
def test_kv_append_and_read(b2p, n, heads, kv, kind, dtype, page, rot, inter):
    g = gen(n + heads)
    cols = 64 * (heads + 2 * kv)
    wide = (randn(g, n, cols + 24) * 3).to(dtype)
    qkv = wide[:, 16:16 + cols] if n > 1 else wide[:, :cols]  # a view with a pitch of its own
    if n > 5:
        qkv[2, heads * 64:(heads + 2 * kv) * 64] = 0  # vectors of zeros
        qkv[4, heads * 64:heads * 64 + 64] *= 1e-3
    pages = -(-n // page) + 2
    table = decode.rope_table(5000, rot, theta=10000.0) if rot else None
    positions = torch.randint(0, 5000, (n,), device="cuda", generator=g).int()
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:n].int()
    if n > 5:
        slots[3] = -1
    cache = decode.KVCache.empty(pages, page, kv, kind)
    for t in (cache.k, cache.v):
        t.view(torch.uint8).fill_(0x5a)
    q = cache.append(qkv, heads, slots, positions if rot else None, table, inter)
    x = qkv.double().reshape(n, heads + 2 * kv, 64)
    turned = rotated(x[:, :heads + kv], table, positions, rot, inter)
    size = x.abs().amax(-1, keepdim=True) * 2
    err = (q.double().reshape(n, heads, 64) - turned[:, :heads]).abs()
    assert (err <= U[dtype] * turned[:, :heads].abs() + 2.0 ** -21 * size[:, :heads]).all()
    held = torch.cat((turned[:, heads:], x[:, heads + kv:]), 1).reshape(n, 2, kv, 64)
    live = slots >= 0
    at = (slots[live].long() // page, slice(None), slots[live].long() % page)
    k_out = torch.full((n, 64 * kv + 8), 7.0, device="cuda").to(dtype)[:, :64 * kv]
    k, v = cache.read(slots, dtype, k_out=k_out)
    assert k.data_ptr() == k_out.data_ptr()
    for which, (codes, scales, back) in enumerate(((cache.k, cache.k_scale, k), (cache.v, cache.v_scale, v))):
        want, got = held[live][:, which], codes.view(torch.uint8)[at].view(codes.dtype).double()
        if codes.dtype == dtype:
            assert ((got - want).abs() <= U[dtype] * want.abs() + 2.0 ** -21 * want.abs().amax(-1, keepdim=True)).all()
            plain = got.to(dtype)
        else:
            top = 127.0 if kind == I8 else 448.0
            unit = want.abs().amax(-1).clamp_min(1e-30) / top
            assert ((scales[at].double() - unit).abs() <= 2.0 ** -21 * unit).all()
            y = want / unit[..., None]
            half = torch.full_like(y, 0.5) if kind == I8 else torch.exp2(
                torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 4)
            assert ((got - y).abs() <= half + top * 2.0 ** -21).all()
            plain = (got.float() * scales[at][..., None]).to(dtype)
        assert torch.equal(back.reshape(n, kv, 64)[live], plain)
        assert (back[~live] == 0).all()
        untouched = torch.ones(pages, page, dtype=torch.bool, device="cuda")
        untouched[slots[live].long() // page, slots[live].long() % page] = False
        assert (codes.view(torch.uint8).movedim(1, 2)[untouched] == 0x5a).all()  # nothing else is written
    decode.check()


@pytest.mark.parametrize("kind", [I8, E4])
def test_kv_extremes(b2p, kind):
    """Subnormal, huge and non-finite vectors: each reads back as itself or, where it has a non-finite value, as NaN."""
    x = torch.zeros(6, 3 * 64, device="cuda", dtype=BF16)
    x[0, 64:] = 1e-38
    x[1, 64:] = 3e38
    x[2, 70], x[2, 140] = float("inf"), float("-inf")
    x[3, 64:] = float("nan")
    x[4, 64:] = torch.linspace(-2, 2, 128, device="cuda").to(BF16)
    cache = decode.KVCache.empty(1, 8, 1, kind)
    slots = torch.arange(6, device="cuda").int()
    cache.append(x, 1, slots)
    k, v = cache.read(slots, BF16)
    assert (k[0].float().abs() <= 1e-30).all() and (k[5] == 0).all() and (v[5] == 0).all()
    assert torch.allclose(k[1].float(), x[1, 64:128].float(), rtol=2.0 ** -6)
    assert k[2].isnan().any() and v[2].isnan().any() and k[3].isnan().all() and v[3].isnan().all()
    assert torch.allclose(k[4].float(), x[4, 64:128].float(), rtol=0.07, atol=2 / 127)


def test_kv_in_place_and_bad_indices(b2p):
    """Q may be written over itself; indices out of range are skipped and reported."""
    g = gen(3)
    qkv = randn(g, 40, 64 * 25).half()
    table, pos = decode.rope_table(64), torch.arange(40, device="cuda").int()
    slots = torch.arange(40, device="cuda").int()
    one, two = decode.KVCache.empty(4, 16, 5), decode.KVCache.empty(4, 16, 5)
    apart = one.append(qkv, 15, slots, pos, table)
    here = qkv.clone()
    two.append(here, 15, slots, pos, table, out=here[:, :960])
    assert torch.equal(here[:, :960], apart) and torch.equal(here[:, 960:], qkv[:, 960:])
    assert torch.equal(one.read(slots, F16)[0], two.read(slots, F16)[0])
    decode.check()
    bad = slots.clone()
    bad[5] = 64
    two.append(qkv, 15, bad, pos, table)
    with pytest.raises(decode.B2PError):
        decode.check()
    far = pos.clone()
    far[0] = 64
    two.append(qkv, 15, slots, far, table)
    with pytest.raises(decode.B2PError):
        decode.check()
    assert (two.read(bad, F16)[0][5] == 0).all()
    with pytest.raises(decode.B2PError):
        decode.check()
    decode.check()


def test_kv_beyond_32_bits(b2p):
    """Slots whose byte offsets pass 2^32."""
    pages = (1 << 32) // (5 * 64 * 64) + 40
    cache = decode.KVCache.empty(pages, 64, 5)
    slots = (pages * 64 - 1 - torch.arange(70, device="cuda") * 3).int()
    qkv = randn(gen(1), 70, 64 * 25).half()
    cache.append(qkv, 15, slots)
    k, v = cache.read(slots, F16)
    size = qkv[:, 960:].float().reshape(70, 10, 64).abs().amax(-1).amax()
    assert (k.float() - qkv[:, 960:1280].float()).abs().max() <= size / 254 * 1.01
    assert (v.float() - qkv[:, 1280:].float()).abs().max() <= size / 254 * 1.01
    att = decode.PrefixAttention(1, 1, 15, 5, 64, 3)
    q = randn(gen(2), 1, 960).half()
    page = torch.tensor([pages - 1], device="cuda").int()
    near = decode.KVCache(cache.k[-1:].clone(), cache.v[-1:].clone(), cache.k_scale[-1:].clone(),
                          cache.v_scale[-1:].clone())
    for t in (near, cache):  # the last page is written only in part: give every slot finite contents
        (t.k if t is near else t.k[-1:]).clamp_(-9, 9)
        for s in (t.k_scale[-1:], t.v_scale[-1:]):
            s.copy_(torch.full_like(s, 0.01))
    a = att(q, cache, page, 64, None, None)
    b = att(q, near, torch.zeros_like(page), 64, None, None)
    assert torch.equal(a, b)


# ---- attention ------------------------------------------------------------------------------------------------
def make_cache(g, pages, kv, page, kind, dtype, spread=1.0):
    shape = (pages, kv, page, 64)
    k, v = randn(g, *shape) * 1.2, randn(g, *shape)
    if spread != 1.0:  # values of very different sizes
        v = v * torch.exp2(torch.randint(-12, 3, shape[:3], device="cuda", generator=g).float() * spread)[..., None]
    if kind in (F16, BF16):
        return decode.KVCache(k.to(kind), v.to(kind))
    top = 127.0 if kind == I8 else 448.0
    made = []
    for x in (k, v):
        unit = x.abs().amax(-1) / top
        y = x / unit[..., None]
        made.append((y.round().to(I8) if kind == I8 else y.to(E4), unit.contiguous()))
    return decode.KVCache(made[0][0], made[1][0], made[0][1], made[1][1])


def dense(codes, scale, pages, count):
    x = codes.view(torch.uint8)[pages.long()].view(codes.dtype).double() if codes.dtype == E4 else codes[pages.long()].double()
    if scale is not None:
        x = x * scale[pages.long()].double()[..., None]
    return x.movedim(1, 0).reshape(codes.shape[1], -1, 64)[:, :count]


def attend64(q, cache, pp, plen, sp, lens, q_len):
    batch, kv = lens.numel(), cache.kv_heads
    heads = q.shape[1] // 64
    out = torch.zeros(batch, q_len, heads, 64, dtype=torch.float64, device="cuda")
    lse = torch.full((batch, q_len, heads), -math.inf, dtype=torch.float64, device="cuda")
    vmax = torch.zeros(batch, q_len, heads, dtype=torch.float64, device="cuda")
    x = q.double().reshape(batch, q_len, kv, heads // kv, 64)
    for b in range(batch):
        for i in range(q_len):
            own = max(0, int(lens[b]) - (q_len - 1 - i))
            k = torch.cat((dense(cache.k, cache.k_scale, pp, plen), dense(cache.k, cache.k_scale, sp[b], own)), 1)
            v = torch.cat((dense(cache.v, cache.v_scale, pp, plen), dense(cache.v, cache.v_scale, sp[b], own)), 1)
            if k.shape[1] == 0:
                continue
            s = torch.einsum("gad,gkd->gak", x[b, i], k) / 8
            lse[b, i] = torch.logsumexp(s, -1).reshape(-1) / math.log(2)
            p = torch.softmax(s, -1)
            out[b, i] = torch.einsum("gak,gkd->gad", p, v).reshape(heads, 64)
            # the largest value that a row's weights can meet
            vmax[b, i] = (p.sqrt() * v.abs().amax(-1)[:, None]).amax(-1).reshape(-1)
    return out.reshape(batch * q_len, -1), lse.reshape(batch * q_len, -1), vmax.reshape(batch * q_len, heads)


ATTN_CASES = [  # batch, q_len, heads, kv_heads, cache, dtype, page, prefix, suffix
    (1, 1, 8, 2, F16, F16, 16, 1, 0),
    (1, 1, 8, 2, F16, F16, 16, 0, 1),
    (1, 1, 15, 5, I8, F16, 16, 200, 33),
    (3, 1, 15, 5, I8, BF16, 8, 129, 70),
    (2, 5, 16, 1, E4, F16, 32, 257, 40),
    (8, 1, 15, 5, E4, BF16, 16, 1023, 129),
    (5, 4, 24, 6, BF16, BF16, 64, 1000, 300),
    (4, 1, 4, 4, F16, F16, 128, 5000, 17),
    (3, 8, 32, 8, I8, F16, 1024, 2049, 1500),
    (2, 3, 9, 3, E4, F16, 8, 4500, 9),
    (33, 1, 15, 5, I8, F16, 64, 3001, 100),
    (70, 2, 12, 4, E4, BF16, 16, 700, 65),
    (130, 1, 12, 12, F16, F16, 32, 1111, 20),
    (45, 1, 15, 5, I8, BF16, 256, 8191, 3),
    (1, 200, 15, 5, I8, F16, 64, 640, 450),
]


@pytest.mark.parametrize("batch,q_len,heads,kv,kind,dtype,page,prefix,suffix", ATTN_CASES)
@pytest.mark.parametrize("spread", [1.0, 0.9])
def test_prefix_attention(b2p, batch, q_len, heads, kv, kind, dtype, page, prefix, suffix, spread):
    """Against 64 bits, with lengths from none to the longest, pages in no order, garbage in unused slots."""
    g = gen(batch * 1000 + prefix)
    first, each = -(-prefix // page), -(-suffix // page)
    pages = first + batch * each + 2
    cache = make_cache(g, pages, kv, page, kind, dtype, spread)
    order = torch.randperm(pages, device="cuda", generator=g).int()
    pp, sp = order[:first].contiguous(), order[first:first + batch * each].reshape(batch, each).contiguous()
    lens = torch.randint(0, suffix + 1, (batch,), device="cuda", generator=g).int()
    lens[0] = suffix
    if batch > 1:
        lens[1] = 0
    # what lies beyond the end of a list must not count, whatever it is
    used = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    at = torch.arange(first * page, device="cuda").reshape(first, page)
    used[pp.long()] = at < prefix
    if each:
        at = torch.arange(each * page, device="cuda").reshape(1, each, page)
        used[sp.long()] = at < lens[:, None, None]
    for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        hole = ~used[:, None, :].expand(pages, kv, page)
        if scale is not None:
            scale[hole] = float("nan")
        if codes.dtype in (F16, BF16):
            codes[hole] = float("nan")
        else:
            codes.view(torch.uint8)[hole] = 0x7f  # the largest int8, the NaN of e4m3
    wide = (randn(g, batch * q_len, heads * 64 + 8) * 1.5).to(dtype)
    q = wide[:, :heads * 64]
    att = decode.PrefixAttention(batch, q_len, heads, kv, prefix, suffix)
    out, lse = att(q, cache, pp, prefix, sp, lens, return_lse=True)
    again = att(q, cache, pp, prefix, sp, lens)
    decode.check()
    assert torch.equal(out, again)  # bit for bit
    want, wlse, vmax = attend64(q, cache, pp, prefix, sp, lens.cpu(), q_len)
    empty = wlse.isinf()
    assert torch.equal(lse.isinf(), empty) and (out.reshape(*lse.shape, 64)[empty] == 0).all()
    assert ((lse.double() - wlse)[~empty].abs() <= 1e-4).all()
    bound = (2 * U[dtype] + (prefix + suffix) * 2.0 ** -25 + 1e-4) * cache_max(cache, used)
    assert ((out.double() - want).abs() <= bound).all(), ((out.double() - want).abs().max(), bound)
    # and row by row: no worse than rounding each weight and the output, over the values the row's weights meet
    err = (out.double() - want).reshape(*lse.shape, 64)
    rel = err.norm() / want.norm().clamp_min(1e-30)
    assert rel <= 3 * U[dtype], rel


def cache_max(cache, used):
    v = cache.v.double() if cache.v.dtype != E4 else cache.v.float().double()
    if cache.v_scale is not None:
        v = v * cache.v_scale.double()[..., None]
    return v.movedim(1, 2)[used].abs().max()


def test_prefix_attention_nan_and_stream(b2p):
    """A visible NaN reaches only the rows that see it; work on another stream; no suffix at all."""
    g = gen(9)
    cache = make_cache(g, 12, 2, 16, I8, F16)
    pp = torch.arange(4, device="cuda").int()
    sp = torch.arange(4, 12, device="cuda").int().reshape(2, 4)
    lens = torch.tensor([50, 40], device="cuda").int()
    q = randn(g, 2, 512).half()
    att = decode.PrefixAttention(2, 1, 8, 2, 64, 64)
    good = att(q, cache, pp, 60, sp, lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = att(q, cache, pp, 60, sp, lens)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(good, other)
    cache.k_scale[4, 1, 3] = float("nan")  # sequence 0's suffix, KV head 1
    out = att(q, cache, pp, 60, sp, lens)
    assert out[0, 256:].isnan().all() and torch.equal(out[0, :256], good[0, :256]) and torch.equal(out[1], good[1])
    alone = att(q, cache, pp, 60, None, None)
    zero = att(q, cache, pp, 60, sp, torch.zeros_like(lens))
    assert torch.equal(alone, zero)
    nothing, lse = att(q, cache, None, 0, None, None, return_lse=True)
    assert (nothing == 0).all() and (lse == -math.inf).all()
    decode.check()


def test_prefix_attention_bad_indices(b2p):
    """Page ids and lengths out of range are reported and read nothing."""
    cache = make_cache(gen(4), 8, 2, 16, F16, F16)
    att = decode.PrefixAttention(2, 1, 4, 2, 64, 32)
    q = randn(gen(5), 2, 256).half()
    pp, sp = torch.arange(4, device="cuda").int(), torch.arange(4, 8, device="cuda").int().reshape(2, 2)
    lens = torch.tensor([20, 30], device="cuda").int()
    for bad in ("prefix", "suffix", "length", "negative"):
        p, s, n = pp.clone(), sp.clone(), lens.clone()
        if bad == "prefix":
            p[2] = 8
        elif bad == "suffix":
            s[1, 1] = -5
        else:
            n[0] = 33 if bad == "length" else -1
        att(q, cache, p, 64, s, n)
        with pytest.raises(decode.B2PError):
            decode.check()
    att(q, cache, pp, 64, sp, lens)
    decode.check()


# ---- sampling -------------------------------------------------------------------------------------------------
def ranked(logits, temp, top_k, top_p, min_p):
    """Kept weights of one row in 64 bits, in index order: keys by the operator's fp32 arithmetic, the rest exact."""
    x = logits.astype(np.float32)
    m = np.float32(np.nanmax(x))
    if temp <= 0:
        w = np.zeros(x.size)
        w[int(np.nanargmax(x))] = 2.0 ** 31
        return w
    c = np.float32(np.float32(1) / np.float32(temp)) * np.float32(1.4426950408889634)
    with np.errstate(invalid="ignore"):
        d = (m - x) * c
    d = np.where(x == m, np.float32(0), d)
    key = np.rint(np.where(d < 64, d, np.float32(64)).astype(np.float64) * 2.0 ** 20)
    w = np.rint(2.0 ** (31 - key / 2.0 ** 20))
    order = np.argsort(key, kind="stable")
    s = w[order]
    if 0 < top_k < x.size:
        s[top_k:] = 0
    keep = np.ones(x.size, bool)
    if top_p < 1:
        keep = np.cumsum(s) - s < float(np.float32(top_p)) * s.sum()
    if min_p > 0:
        keep &= s >= min(float(np.float32(min_p)), 1.0) * 2.0 ** 31
    keep[0] = True
    out = np.zeros(x.size)
    out[order] = np.where(keep, s, 0)
    return out


def check_draw(row, token, logprob, u, *params):
    w = ranked(row, *params)
    total, run = w.sum(), np.cumsum(w)
    slack = 2 * (total * 2.0 ** -22 + w.size / 2)
    assert w[token] > 0, (token, params)
    assert run[token] - w[token] - slack <= u * total <= run[token] + slack, (token, params)
    if logprob is not None:
        assert abs(logprob - math.log(w[token] / total)) <= 1e-5 + 1.0 / w[token]


SAMPLE_CASES = [  # rows, vocab, dtype
    (1, 1, torch.float32),
    (3, 2, torch.float16),
    (5, 31, torch.bfloat16),
    (4, 1000, torch.float32),
    (33, 16893, torch.bfloat16),
    (6, 32000, torch.float32),
    (9, 49152, torch.float16),
    (2, 70001, torch.float32),
    (300, 2049, torch.float32),
]


@pytest.mark.parametrize("rows,vocab,dtype", SAMPLE_CASES)
@pytest.mark.parametrize("filters", ["none", "k", "p", "min", "all", "cold"])
def test_sample(b2p, rows, vocab, dtype, filters):
    g = gen(rows + vocab)
    wide = (randn(g, rows, vocab + 3) * 3).to(dtype)
    logits = wide[:, 1:vocab + 1] if filters in ("k", "all") else wide[:, :vocab].contiguous()
    if vocab > 100:
        logits[0, ::3] = -math.inf
        logits[rows // 2, 5:50] = float("nan")
    u = torch.rand(rows, device="cuda", generator=g)
    u[0] = 0.0
    temp = torch.rand(rows, device="cuda", generator=g) * 1.5 + 0.2
    k = torch.randint(1, max(2, min(vocab, 300)), (rows,), device="cuda", generator=g).int()
    p = torch.rand(rows, device="cuda", generator=g) * 0.98 + 0.01
    mp = torch.rand(rows, device="cuda", generator=g) * 0.1
    if filters == "cold":
        temp[:] = 0
    k, p, mp = (t if filters in (n, "all") else None for t, n in ((k, "k"), (p, "p"), (mp, "min")))
    tokens, logprobs = decode.sample(logits, u, temp, k, p, mp)
    again, _ = decode.sample(logits, u, temp, k, p, mp)
    assert torch.equal(tokens, again)
    x = logits.float().cpu().numpy()
    for r in range(rows):
        check_draw(x[r], int(tokens[r]), float(logprobs[r]), float(u[r]), float(temp[r]),
                   0 if k is None else int(k[r]), 1.0 if p is None else float(p[r]), 0.0 if mp is None else float(mp[r]))


def test_sample_ties(b2p):
    """Equal logits: the filters keep the lowest indices, and the draw goes through them in order."""
    n, vocab = 64, 5000
    logits = torch.full((n, vocab), 2.5, device="cuda", dtype=F16)
    u = (torch.arange(n, device="cuda") + 0.5) / n
    k = torch.full((n,), 40, device="cuda").int()
    tokens, logprobs = decode.sample(logits, u, top_k=k)
    assert torch.equal(tokens, (u * 40).int()) and torch.allclose(logprobs, torch.full_like(u, -math.log(40.0)))
    p = torch.full((n,), 0.1, device="cuda")
    kept = 501 if float(p[0]) > 0.1 else 500  # 0.1 in fp32 lies above 1/10
    tokens, _ = decode.sample(logits, u, top_p=p)
    assert torch.equal(tokens, (u.double() * kept).int())
    both, _ = decode.sample(logits, u, top_k=k, top_p=p)
    assert torch.equal(both, (u.double() * (5 if float(p[0]) > 0.1 else 4)).int())
    one, lp = decode.sample(logits, u, top_p=torch.zeros(n, device="cuda"))
    assert (one == 0).all() and (lp == 0).all()
    one, _ = decode.sample(logits, u, temperature=torch.zeros(n, device="cuda"))
    assert (one == 0).all()
    logits[:, 7] = 3.0
    one, _ = decode.sample(logits, u, min_p=torch.full((n,), 5.0, device="cuda"))
    assert (one == 7).all()


def test_sample_edges(b2p):
    """Rows of nothing, of one token, infinities, numbers at the ends of [0, 1)."""
    logits = torch.full((8, 300), -math.inf, device="cuda")
    logits[1, 200] = -5.0
    logits[2, 10], logits[2, 20] = math.inf, math.inf
    logits[3] = float("nan")
    logits[4, 299], logits[4, 0] = 1.0, 1.0
    logits[5, 299], logits[5, 0] = 1.0, 1.0
    logits[6] = 0.0
    logits[7] = -3e38
    logits[7, 100] = 3e38
    u = torch.tensor([0.5, 0.99, 0.6, 0.5, 0.0, 1 - 2.0 ** -24, 1 - 2.0 ** -24, 0.5], device="cuda")
    tokens, logprobs = decode.sample(logits, u, top_p=torch.full((8,), 0.999999, device="cuda"))
    assert tokens.tolist() == [-1, 200, 20, -1, 0, 299, 299, 100]
    assert logprobs[0].isnan() and logprobs[3].isnan() and logprobs[1] == 0
    assert abs(float(logprobs[2]) + math.log(2)) < 1e-6
    plain, _ = decode.sample(logits, u)
    assert plain.tolist() == tokens.tolist()


def test_sample_frequencies(b2p):
    """Over evenly spaced numbers each token comes as often as its probability says."""
    n, vocab = 20000, 40
    row = torch.linspace(0, 3, vocab, device="cuda")
    u = (torch.arange(n, device="cuda") + 0.5) / n
    tokens, _ = decode.sample(row.expand(n, vocab).contiguous(), u, temperature=torch.full((n,), 0.7, device="cuda"))
    seen = torch.bincount(tokens.long(), minlength=vocab) / n
    assert (seen - torch.softmax(row / 0.7, 0)).abs().max() <= 2.0 / n


@pytest.mark.parametrize("rows,vocab", [(2, 5000), (160, 5000), (310, 5000), (2, 70001)])
@pytest.mark.parametrize("std", [0.05, 3.0, 30.0])
def test_sample_wide_filters(b2p, rows, vocab, std):
    """top_k from a few to more than the threads, the list or the tokens that weigh anything; top_p to nearly 1."""
    g = gen(rows + vocab)
    logits = (randn(g, rows, vocab) * std).float()
    u = torch.rand(rows, device="cuda", generator=g)
    temp = torch.full((rows,), 0.7, device="cuda")
    ks = torch.tensor([1, 100, 129, 300, 513, 1400, 2500, vocab - 1], device="cuda").int()
    ps = torch.tensor([0.5, 0.9, 0.999, 0.9999999], device="cuda")
    k = ks[torch.arange(rows, device="cuda") % 8].contiguous()
    p = ps[torch.arange(rows, device="cuda") // 8 % 4].contiguous()
    if rows == 2:
        k, p = ks[[4, 6]].contiguous(), ps[[2, 3]].contiguous()
    x = logits.cpu().numpy()
    for kk, pp in ((k, None), (None, p), (k, p)):
        tokens, logprobs = decode.sample(logits, u, temp, kk, pp)
        for r in range(0, rows, max(1, rows // 32)):
            check_draw(x[r], int(tokens[r]), float(logprobs[r]), float(u[r]), float(temp[r]),
                       0 if kk is None else int(kk[r]), 1.0 if pp is None else float(pp[r]), 0.0)


def test_sample_tiny_temperature(b2p):
    """A temperature whose reciprocal is not finite leaves the largest logits alone."""
    logits = torch.zeros(4, 1000, device="cuda")
    logits[:, 100], logits[:, 900] = 1.0, 1.0
    u = torch.tensor([0.0, 0.49, 0.51, 0.99], device="cuda")
    for t in (1e-30, 1e-36, 1e-40):
        tokens, logprobs = decode.sample(logits, u, torch.full((4,), t, device="cuda"))
        assert tokens.tolist() == [100, 100, 900, 900]
        assert torch.allclose(logprobs, torch.full_like(u, -math.log(2.0)))


@pytest.mark.parametrize("batch,q_len,heads,kv,kind,dtype,page,prefix,suffix", [
    (40, 1, 15, 5, I8, F16, 64, 800, 300),     # single warps for the prefix and the suffixes
    (150, 1, 4, 1, E4, BF16, 16, 130, 40),
    (64, 2, 12, 4, I8, F16, 32, 0, 2500),      # suffixes alone, of several hundred keys a unit
    (160, 1, 2, 1, F16, F16, 8, 0, 2400),      # pages too small for such units
    (160, 1, 2, 1, I8, F16, 8, 100, 1500),
    (1, 1, 15, 5, F16, F16, 64, 8192, 30),     # the tcgen05 kernel for a few rows
    (2, 1, 9, 3, I8, BF16, 128, 9001, 0),
    (1, 3, 16, 1, E4, F16, 16, 8300, 700),
])
def test_prefix_attention_divisions(b2p, batch, q_len, heads, kv, kind, dtype, page, prefix, suffix):
    """Each way that the work is divided."""
    test_prefix_attention(b2p, batch, q_len, heads, kv, kind, dtype, page, prefix, suffix, 1.0)
