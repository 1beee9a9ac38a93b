"""The decoding operators on the host: argument checks of the C entry points (they precede any GPU work), the workspace
bound, the cache descriptor and the rotary tables."""
import ctypes as C
import math
import random
import re
from pathlib import Path

import pytest
import torch

from autoane_b200 import _lib, decode

ARG = -1


def desc(**kw):
    d = dict(k=16, v=16, k_scale=16, v_scale=16, n_pages=100, page_size=16, kv_heads=5, kind=_lib.KV_INT8)
    d.update(kw)
    return _lib.KVCacheDesc(*(d[n] for n, _ in _lib.KVCacheDesc._fields_))


def append(cache=None, qkv=16, ld_qkv=1600, heads=15, q_out=16, ld_q=960, slots=16, positions=16, rope=16, max_pos=8,
           rot=64, interleaved=0, n=1, dtype=0):
    d = cache or desc()
    return _lib.load().b2p_kv_append(C.addressof(d), qkv, ld_qkv, heads, q_out, ld_q, slots, positions, rope, max_pos,
                                     rot, interleaved, n, dtype, None)


def read(cache=None, slots=16, n=1, k_out=16, ld_k=320, v_out=16, ld_v=320, dtype=0):
    d = cache or desc()
    return _lib.load().b2p_kv_read(C.addressof(d), slots, n, k_out, ld_k, v_out, ld_v, dtype, None)


def attend(cache=None, q=16, ld_q=960, out=16, ld_out=960, batch=2, q_len=1, heads=15, prefix_pages=16, prefix_len=40,
           suffix_pages=16, suffix_pitch=2, suffix_lens=16, max_suffix=32, dtype=0, workspace=16, nbytes=1 << 30):
    d = cache or desc()
    return _lib.load().b2p_attention_prefix(C.addressof(d), q, ld_q, out, ld_out, None, batch, q_len, heads,
                                            prefix_pages, prefix_len, suffix_pages, suffix_pitch, suffix_lens,
                                            max_suffix, dtype, workspace, nbytes, None)


def sample(logits=16, ld=100, rows=1, vocab=100, dtype=2, u=16, tokens=16):
    return _lib.load().b2p_sample(logits, ld, rows, vocab, dtype, u, None, None, None, None, tokens, None, None)


REFUSED = [
    (append, dict(cache=desc(page_size=24)), "page_size"),
    (append, dict(cache=desc(page_size=4)), "page_size"),
    (append, dict(cache=desc(kind=3)), "kind"),
    (append, dict(cache=desc(k_scale=None)), "scale"),
    (append, dict(cache=desc(v=None)), "null"),
    (append, dict(cache=desc(k=24)), "aligned"),
    (append, dict(cache=desc(n_pages=1 << 28, page_size=16)), "2^31"),
    (append, dict(ld_qkv=1592), "columns"),
    (append, dict(ld_q=956), "columns"),
    (append, dict(ld_qkv=1604), "alignment"),
    (append, dict(qkv=24), "aligned"),
    (append, dict(rot=24), "rot"),
    (append, dict(rot=80), "rot"),
    (append, dict(rope=None), "rope"),
    (append, dict(max_pos=0), "max_pos"),
    (append, dict(slots=None), "slots"),
    (append, dict(dtype=2), "dtype"),
    (append, dict(n=-1), "n_tokens"),
    (append, dict(heads=0), "heads"),
    (read, dict(ld_k=312), "columns"),
    (read, dict(v_out=None), "null"),
    (read, dict(slots=None), "slots"),
    (attend, dict(heads=14), "multiple"),
    (attend, dict(batch=0), "range"),
    (attend, dict(q_len=0), "range"),
    (attend, dict(prefix_len=-1), "range"),
    (attend, dict(prefix_pages=None), "prefix_pages"),
    (attend, dict(suffix_lens=None), "suffix"),
    (attend, dict(suffix_pitch=1), "suffix_pitch"),
    (attend, dict(ld_out=952), "columns"),
    (attend, dict(q=24), "aligned"),
    (attend, dict(workspace=None), "workspace"),
    (attend, dict(nbytes=100), "workspace"),
    (attend, dict(workspace=24), "aligned"),
    (attend, dict(dtype=2), "dtype"),
    (sample, dict(vocab=0), "vocab"),
    (sample, dict(vocab=1 << 21, ld=1 << 21), "vocab"),
    (sample, dict(ld=99), "ld"),
    (sample, dict(u=None), "null"),
    (sample, dict(tokens=None), "null"),
    (sample, dict(dtype=3), "dtype"),
    (sample, dict(rows=-1), "rows"),
]


@pytest.mark.parametrize("fn,kw,word", REFUSED, ids=[f"{f.__name__}-{i}" for i, (f, _, _) in enumerate(REFUSED)])
def test_refusals(fn, kw, word):
    """Each bad argument is refused with a status and a message that names it, before any GPU work."""
    assert fn(**kw) == ARG
    assert word in _lib.load().b2p_last_error().decode()


def test_no_tokens_or_rows_is_no_work():
    assert append(n=0) == 0 and read(n=0) == 0 and sample(rows=0) == 0


def test_valid_arguments_reach_the_device():
    """With every argument valid the calls get as far as the device (absent here, so B2P_ERR_CUDA)."""
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible: these addresses are not real")
    for fn in (append, read, attend, sample):
        assert fn() not in (0, ARG), fn.__name__


def test_workspace_serves_every_smaller_call():
    """The workspace of a call holds what any call with no larger arguments uses."""
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible: these addresses are not real")
    rng = random.Random(7)
    size = lambda a, b: int(math.exp(rng.uniform(math.log(a), math.log(b + 1))))  # noqa: E731
    for _ in range(4000):
        heads, kv = rng.choice([(15, 5), (9, 3), (8, 2), (32, 8), (12, 12), (16, 1), (64, 1)])
        batch, q_len = size(1, 600), size(1, 16)
        prefix, suffix = rng.choice([0, size(1, 200000)]), rng.choice([0, size(1, 200000)])
        bound = _lib.load().b2p_attention_prefix_workspace(batch, q_len, heads, kv, prefix, suffix)
        less = lambda n: size(1, n) if n else 0  # noqa: E731
        rc = attend(cache=desc(kv_heads=kv), ld_q=heads * 64, ld_out=heads * 64, heads=heads, batch=less(batch),
                    q_len=less(q_len), prefix_len=less(prefix), max_suffix=less(suffix), suffix_pitch=1 << 20,
                    nbytes=bound)
        assert rc != ARG, _lib.load().b2p_last_error()


def test_workspace_serves_every_cache():
    """Nor does it depend on the pages or the kind of the cache."""
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible: these addresses are not real")
    rng = random.Random(8)
    size = lambda a, b: int(math.exp(rng.uniform(math.log(a), math.log(b + 1))))  # noqa: E731
    for _ in range(4000):
        heads, kv = rng.choice([(15, 5), (9, 3), (8, 2), (12, 12), (16, 1), (64, 1)])
        batch, q_len = size(1, 600), size(1, 8)
        prefix, suffix = rng.choice([0, size(1, 200000)]), rng.choice([0, size(1, 200000)])
        bound = _lib.load().b2p_attention_prefix_workspace(batch, q_len, heads, kv, prefix, suffix)
        kind = rng.choice([dict(kind=_lib.KV_16, k_scale=None, v_scale=None), dict()])
        rc = attend(cache=desc(kv_heads=kv, page_size=8 << rng.randrange(8), **kind), ld_q=heads * 64,
                    ld_out=heads * 64, heads=heads, batch=batch, q_len=q_len, prefix_len=prefix, max_suffix=suffix,
                    suffix_pitch=1 << 20, nbytes=bound)
        assert rc != ARG, _lib.load().b2p_last_error()


def test_descriptor_matches_header():
    text = (Path(__file__).resolve().parents[1] / "include" / "b2p.h").read_text()
    for name, value in (("B2P_KV_16", _lib.KV_16), ("B2P_KV_INT8", _lib.KV_INT8), ("B2P_KV_E4M3", _lib.KV_E4M3)):
        assert int(re.search(rf"#define\s+{name}\s+(\d+)", text).group(1)) == value
    assert C.sizeof(_lib.KVCacheDesc) == 4 * 8 + 4 * 4


def test_rope_table():
    t = decode.rope_table(50, 32, theta=100000.0, device="cpu")
    assert t.shape == (50, 16, 2) and t.dtype == torch.float32
    for p, i in ((0, 3), (49, 0), (31, 15)):
        a = p * 100000.0 ** (-2 * i / 32)
        assert abs(t[p, i, 0].item() - math.cos(a)) < 1e-7 and abs(t[p, i, 1].item() - math.sin(a)) < 1e-7
    half = decode.rope_table(50, 32, theta=100000.0, scale=2.0, device="cpu")
    assert torch.allclose(half[::2], t[:25], atol=1e-7)
    y = decode.rope_table(50, 64, theta=10000.0, scale=4.0, yarn=(2048, 32.0, 1.0), device="cpu")
    size = 0.1 * math.log(4.0) + 1
    assert torch.allclose(y.square().sum(-1), torch.full((50, 32), size * size), atol=1e-5)
    plain = decode.rope_table(50, 64, theta=10000.0, device="cpu")
    assert torch.allclose(y[:, 0], plain[:, 0] * size, atol=1e-6)  # the fastest pair keeps its angles
    slow = decode.rope_table(50, 64, theta=10000.0, scale=4.0, device="cpu")
    assert torch.allclose(y[:, -1], slow[:, -1] * size, atol=1e-6)  # the slowest is divided by 4
    with pytest.raises(ValueError):
        decode.rope_table(50, 24, device="cpu")


def test_tensors_are_checked():
    with pytest.raises(ValueError):
        decode.KVCache(torch.zeros(2, 5, 16, 64), torch.zeros(2, 5, 16, 64))  # neither on a GPU nor of a cache type
    with pytest.raises(ValueError):
        decode.sample(torch.zeros(2, 10), torch.zeros(2))
    with pytest.raises(ValueError):
        decode.PrefixAttention(1, 1, 5, 2, 10, 10, device="cpu")
