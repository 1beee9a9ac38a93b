"""The decoding operators on the GPU where values, lengths and parameters reach their ends, against plain
implementations in 64 bits. Tolerances are those of test_gpu_decode.py, from the arithmetic; where a result must not
depend on something, it is compared bit for bit."""
import math

import pytest
import torch

from autoane_b200 import decode
from tests.test_gpu_decode import BF16, E4, F16, I8, gen, randn

pytestmark = pytest.mark.gpu

NAN, INF = math.nan, math.inf


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
