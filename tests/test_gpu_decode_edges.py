"""The decoding operators on the GPU where values, lengths and parameters reach their ends, against plain
implementations in 64 bits. Tolerances are those of test_gpu_decode.py, from the arithmetic; where a result must not
depend on something, it is compared bit for bit."""
import math

import pytest
import torch

from autoane_b200 import decode
from tests.test_gpu_decode import BF16, E4, F16, I8, U, attend64, gen, make_cache, randn

pytestmark = pytest.mark.gpu

NAN, INF = math.nan, math.inf


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---- cache ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", [I8, E4])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("bad", [INF, -INF, NAN])
def test_kv_nonfinite_vector_reads_back_nan(b2p, kind, dtype, bad):
    """One non-finite channel makes its (token, head) vector NaN, every channel of it and no other vector."""
    n, kv = 9, 3
    x = randn(gen(1), n, 64 * (1 + 2 * kv)).to(dtype)
    vectors = x.view(n, 1 + 2 * kv, 64)
    vectors[4, 1 + 1, 17] = bad      # K of token 4, head 1
    vectors[6, 1 + kv + 2, 63] = bad  # V of token 6, head 2
    cache = decode.KVCache.empty(2, 8, kv, kind)
    slots = torch.arange(n, device="cuda").int()
    cache.append(x, 1, slots)
    k, v = (t.view(n, kv, 64) for t in cache.read(slots, dtype))
    want = torch.zeros(n, kv, 64, dtype=torch.bool, device="cuda")
    for got, (t, h) in ((k, (4, 1)), (v, (6, 2))):
        want.zero_()
        want[t, h] = True
        assert torch.equal(got.isnan(), want)
    decode.check()


@pytest.mark.parametrize("kind", [I8, E4])
@pytest.mark.parametrize("prefix", [40, 8192])  # attn_rows_kernel and the tcgen05 kernel
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_infinite_key_is_not_lost(b2p, kind, prefix, sign):
    """A key with an infinite channel makes the rows that see it NaN, whatever the sign of the query's channel."""
    x = randn(gen(2), prefix, 3 * 64).half()
    x[7, 64 + 20] = INF
    cache = decode.KVCache.empty(-(-prefix // 64), 64, 1, kind)
    cache.append(x, 1, torch.arange(prefix, device="cuda").int())
    q = (torch.rand(1, 64, device="cuda", generator=gen(3)) + 0.5).half() * sign
    att = decode.PrefixAttention(1, 1, 1, 1, prefix, 0)
    out, lse = att(q, cache, torch.arange(cache.n_pages, device="cuda").int(), prefix, None, None, return_lse=True)
    assert out.isnan().all() and lse.isnan().all()
    decode.check()


# ---- attention: what a row does not see ---------------------------------------------------------------------
# batch, q_len, heads, kv_heads, prefix, suffix: a tile for the queries or several, units of one warp or of four
HIDDEN = [(2, 3, 3, 1, 70, 40), (1, 2, 8, 2, 0, 33), (2, 20, 6, 2, 0, 150), (1, 40, 3, 1, 30, 40), (150, 2, 2, 1, 64, 40),
          (80, 5, 16, 4, 0, 300), (3, 2, 30, 10, 8192, 65)]


@pytest.mark.parametrize("batch,q_len,heads,kv,prefix,suffix", HIDDEN)
@pytest.mark.parametrize("kind,dtype", [(F16, F16), (BF16, BF16), (I8, F16), (I8, BF16), (E4, F16), (E4, BF16)])
@pytest.mark.parametrize("where", ["k", "v", "inf"])
def test_later_tokens_do_not_reach_earlier_queries(b2p, batch, q_len, heads, kv, prefix, suffix, kind, dtype, where):
    """A non-finite key or value in the last token of a sequence: its last query has it, the others are as without."""
    page = 16
    g = gen(batch + q_len)
    first, each = -(-prefix // page), -(-suffix // page)
    cache = make_cache(g, first + batch * each, kv, page, kind, dtype)
    pp = torch.arange(first, device="cuda").int()
    sp = (first + torch.arange(batch * each, device="cuda")).int().reshape(batch, each)
    lens = torch.full((batch,), suffix, device="cuda").int()
    lens[-1] = max(suffix - 7, 1)
    q = randn(g, batch * q_len, heads * 64).to(dtype)
    att = decode.PrefixAttention(batch, q_len, heads, kv, prefix, suffix)
    clean, clean_lse = att(q, cache, pp, prefix, sp, lens, return_lse=True)
    b, h = batch - 1, kv - 1
    at = int(lens[b]) - 1
    spot = (int(sp[b, at // page]), h, at % page)
    bad = INF if where == "inf" else NAN
    codes, scale = (cache.k, cache.k_scale) if where == "k" else (cache.v, cache.v_scale)
    if scale is not None:
        scale[spot] = bad
    elif where == "k":
        codes[spot] = bad
    else:
        codes[spot][11] = bad
    if kind is E4 and where == "v":
        codes.view(torch.uint8)[spot] = 0x7f  # its codes are NaN too, as written by KVCache.append
    out, lse = att(q, cache, pp, prefix, sp, lens, return_lse=True)
    decode.check()
    shape = (batch, q_len, kv, heads // kv, 64)
    hit = torch.zeros(shape[:4], dtype=torch.bool, device="cuda")
    hit[b, -1, h] = True
    same = (out.view(shape) == clean.view(shape)).all(-1) & (lse.view(shape[:4]) == clean_lse.view(shape[:4]))
    assert torch.equal(same, ~hit)
    got = out.view(shape)[b, -1, h]
    if where == "k" or kind in (I8, E4):
        assert got.isnan().all() if where != "inf" else not got.isfinite().any()
    else:  # one channel of the value
        assert (got[:, 11] == INF).all() if where == "inf" else got[:, 11].isnan().all()
        got, ref = got.clone(), clean.view(shape)[b, -1, h].clone()
        got[:, 11] = ref[:, 11] = 0
        assert torch.equal(got, ref)


def test_infinite_values_of_both_signs(b2p):
    """Infinite values of both signs that one query sees make its channel NaN; of one sign, infinite."""
    g = gen(5)
    cache = make_cache(g, 4, 1, 16, F16, F16)
    cache.v[2, 0, 5, 3] = INF
    cache.v[2, 0, 6, 3] = -INF
    cache.v[2, 0, 6, 4] = -INF
    lens = ints(16 + 16 + 7)
    q = randn(g, 3, 64).half()
    out = decode.PrefixAttention(1, 3, 1, 1, 0, 64)(q, cache, None, 0, ints(0, 1, 2, 3).view(1, 4), lens)
    want, _, _ = attend64(q, cache, ints(), 0, ints(0, 1, 2, 3).view(1, 4), lens.cpu(), 3)
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.isinf(), want.isinf())
    assert out[0].isfinite().all() and out[1, 3] == INF and out[2, 3].isnan() and out[2, 4] == -INF
    decode.check()


@pytest.mark.parametrize("prefix,suffix", [(50, 20), (50, 0), (0, 20), (9000, 0), (9000, 300)])
def test_a_nan_query_has_a_nan_log_sum(b2p, prefix, suffix):
    """-inf says that a query sees nothing; one whose scores are all NaN has NaN, in the output and the log-sum-exp."""
    g = gen(6)
    first, each = -(-prefix // 16), -(-suffix // 16)
    cache = make_cache(g, first + 2 * each, 1, 16, F16, F16)
    q = randn(g, 2, 3 * 64).half()
    q[1, 64:128] = NAN
    sp = (first + torch.arange(2 * each, device="cuda")).int().view(2, each)
    att = decode.PrefixAttention(2, 1, 3, 1, prefix, suffix)
    out, lse = att(q, cache, torch.arange(first, device="cuda").int(), prefix, sp, ints(suffix, suffix),
                   return_lse=True)
    bad = torch.zeros(2, 3, dtype=torch.bool, device="cuda")
    bad[1, 1] = True
    assert torch.equal(out.view(2, 3, 64).isnan().all(-1), bad) and torch.equal(lse.isnan(), bad)
    assert lse[~bad].isfinite().all()
    decode.check()


# ---- attention: scales ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", [I8, E4])
@pytest.mark.parametrize("prefix", [100, 8192])
@pytest.mark.parametrize("scale", [0.0, 1e-40])
def test_values_of_vanishing_scale(b2p, kind, prefix, scale):
    """A value whose scale is zero or subnormal counts as (next to) zero, whatever its codes, and its weight counts."""
    g = gen(7)
    pages = -(-prefix // 64)
    cache = make_cache(g, pages, 1, 64, kind, F16)
    cache.v_scale[:, :, ::3] = scale
    q = randn(g, 4, 64).half()
    pp = torch.arange(pages, device="cuda").int()
    att = decode.PrefixAttention(4, 1, 1, 1, prefix, 0)
    out, lse = att(q, cache, pp, prefix, None, None, return_lse=True)
    none = torch.zeros(4, 0, dtype=torch.int32, device="cuda")
    want, wlse, _ = attend64(q, cache, pp, prefix, none, torch.zeros(4, dtype=torch.int32), 1)
    size = (cache.v.float() * cache.v_scale[..., None]).abs().max()
    assert ((lse - wlse).abs() <= 1e-4).all()
    assert ((out - want).abs() <= (2 * U[F16] + prefix * 2.0 ** -25 + 1e-4) * size).all()


@pytest.mark.parametrize("kind", [I8, E4])
def test_weights_of_zero_values_count_beside_large_ones(b2p, kind):
    """Vectors of zeros (written with the smallest scale) beside values of 2^18: each has its weight in the sum."""
    n = 128
    g = gen(8)
    x = randn(g, n, 3 * 64)
    x[:, :64] = 0
    x[:, 64:128] *= 0.02
    x[:, 128:] *= 2.0 ** 18
    x[0, 64:128] = 4.0      # the heaviest key, of a large value
    x[1:, 128:] = 0         # all others have none
    cache = decode.KVCache.empty(2, 64, 1, kind)
    cache.append(x.to(BF16), 1, torch.arange(n, device="cuda").int())
    q = torch.full((1, 64), 0.35, device="cuda").to(BF16)  # key 0 weighs 2^16 times each other: a 500th is theirs
    pp = ints(0, 1)
    out, lse = decode.PrefixAttention(1, 1, 1, 1, n, 0)(q, cache, pp, n, None, None, return_lse=True)
    want, wlse, _ = attend64(q, cache, pp, n, torch.zeros(1, 0, dtype=torch.int32, device="cuda"),
                             torch.zeros(1, dtype=torch.int32), 1)
    assert ((lse - wlse).abs() <= 1e-4).all()
    size = want.abs().max()
    assert ((out - want).abs() <= (2 * U[BF16] + n * 2.0 ** -25 + 1e-4) * size).all()


# ---- attention: lengths and sizes -------------------------------------------------------------------------------
def test_lengths_that_the_plan_leaves_no_room_for(b2p):
    """Suffix lengths above what the object was made for are reported, where that is none as well."""
    cache = make_cache(gen(10), 6, 1, 16, F16, F16)
    q = randn(gen(11), 2, 64).half()
    sp, pp = ints(2, 3, 4, 5).view(2, 2), ints(0, 1)
    att = decode.PrefixAttention(2, 1, 1, 1, 32, 0)
    plain = att(q, cache, pp, 32, None, None)
    assert torch.equal(att(q, cache, pp, 32, sp, ints(0, 0)), plain)
    decode.check()
    att(q, cache, pp, 32, sp, ints(0, 9))
    with pytest.raises(decode.B2PError):
        decode.check()
    roomy = decode.PrefixAttention(2, 1, 1, 1, 32, 64)
    roomy(q, cache, pp, 32, sp[:, :0], ints(3, 0))  # no pages for them
    with pytest.raises(decode.B2PError):
        decode.check()
    assert torch.equal(roomy(q, cache, pp, 32, sp[:, :0], ints(0, 0)), plain)
    decode.check()


def test_page_of_4_gb(b2p):
    """A page whose bytes pass 2^32: the second page is read as the second."""
    kv, page = 32768, 1024
    cache = decode.KVCache(*(torch.zeros(2, kv, page, 64, dtype=F16, device="cuda") for _ in range(2)))
    v = randn(gen(12), kv, 64).half()
    cache.v[1, :, 0] = v
    q = torch.zeros(1, 64 * kv, dtype=F16, device="cuda")
    out = decode.PrefixAttention(1, 1, kv, kv, 1, 0)(q, cache, ints(1), 1, None, None)
    decode.check()
    assert torch.equal(out.view(kv, 64), v)


def test_one_row_of_any_pitch(b2p):
    """The pitch of a matrix of one row is of no account."""
    g = gen(13)
    wide = randn(g, 1, 25 * 64 + 3).half()
    table, pos = decode.rope_table(8), ints(5)
    one, two = decode.KVCache.empty(1, 16, 5), decode.KVCache.empty(1, 16, 5)
    qkv = wide[:, :25 * 64]
    a = one.append(qkv, 15, ints(3), pos, table)
    b = two.append(qkv.clone(), 15, ints(3), pos, table)
    assert torch.equal(a, b)
    k = [torch.empty(1, 323, dtype=F16, device="cuda")[:, :320] for _ in range(2)]
    one.read(ints(3), F16, *k)
    assert all(torch.equal(x, y) for x, y in zip(k, two.read(ints(3), F16)))
    q = torch.empty(1, 15 * 64 + 1, dtype=F16, device="cuda")[:, :960]
    q.copy_(a)
    att = decode.PrefixAttention(1, 1, 15, 5, 16, 0)
    y = torch.empty(1, 967, dtype=F16, device="cuda")[:, :960]
    one.k[:], one.v[:], one.k_scale[:], one.v_scale[:] = 1, 2, 0.1, 0.1
    att(q, one, ints(0), 16, None, None, out=y)
    assert torch.equal(y, att(a, one, ints(0), 16, None, None))
    decode.check()


# ---- sampling -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, F16, BF16])
@pytest.mark.parametrize("vocab", [203, 500, 1000, 20000])
@pytest.mark.parametrize("rows", [5, 300])
def test_sample_infinite_temperature(b2p, dtype, vocab, rows):
    """Every finite logit weighs the same: the filters keep the lowest indices, and the draw goes through them evenly."""
    logits = (randn(gen(vocab), rows, vocab) * 3).to(dtype)
    u = (torch.arange(rows, device="cuda") + 0.5) / rows
    hot = torch.full((rows,), INF, device="cuda")
    for n in (1, 50, min(2 * vocab // 3, 500)):
        k = torch.full((rows,), n, device="cuda").int()
        tokens, logprobs = decode.sample(logits, u, hot, top_k=k)
        assert torch.equal(tokens, (u.double() * n).int())
        assert torch.allclose(logprobs, torch.full_like(u, -math.log(n)), atol=1e-5)
    for part in (0.25, 0.875):
        kept = math.ceil(vocab * part)  # the tokens before the last one kept weigh less than the part
        tokens, logprobs = decode.sample(logits, u, hot, top_p=torch.full((rows,), part, device="cuda"))
        assert torch.equal(tokens, (u.double() * kept).int())
        assert torch.allclose(logprobs, torch.full_like(u, -math.log(kept)), atol=1e-5)
    tokens, _ = decode.sample(logits, u, hot)
    assert torch.equal(tokens, (u.double() * vocab).int())
    logits[:, :10] = -INF
    tokens, _ = decode.sample(logits, u, hot, top_k=torch.full((rows,), 150, device="cuda").int())
    assert torch.equal(tokens, 10 + (u.double() * 150).int())
