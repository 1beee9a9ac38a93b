"""examples/complete.py over a compacted vocabulary: what is drawn goes on as the embedding row that it stands for."""
import numpy as np
import pytest
import torch

from autoane_b200 import decode
from autoane_b200.model import Config
from tests import _models as M
from tests.test_gpu_complete import example

pytestmark = pytest.mark.gpu


def test_compact_vocabulary(b2p):
    """The same completions as by a model whose embedding has only the compacted rows, bit for bit."""
    cfg = M.small_cfg(nlayers=2, seq=64)
    syn = M.make_model(cfg, n_active=1500, seed=5, rms_jitter=0.05)
    mc = Config(dim=cfg.dim, hidden=cfg.hidden, heads=cfg.heads, kv_heads=cfg.kv_heads, head_dim=cfg.hd, seq=64,
                nlayers=2, vocab=cfg.vocab, rank=cfg.rank, rope_theta=cfg.rope_theta, max_groups=4)
    rms = np.stack([syn.theta[s] for s in M.rms_slices(syn)])
    rows = np.random.default_rng(1).permutation(cfg.vocab)[:1500]
    compact = np.ascontiguousarray(syn.embed[rows])
    batch, prompt = 3, torch.arange(20) * 71 % 1500
    ex = example()
    small = ex.Completer(mc, syn.weights, rms, compact, compact, batch, 20, 16)
    whole = ex.Completer(mc, syn.weights, rms, syn.embed, compact, batch, 20, 16, ids=rows)
    u = torch.rand(12, batch, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    want = small.complete(prompt, 12, u)
    got = whole.complete(torch.from_numpy(rows)[prompt], 12, u)
    decode.check()
    assert torch.equal(got, want) and not torch.equal(got[0], got[1])
    with pytest.raises(ValueError, match="ids"):
        ex.Completer(mc, syn.weights, rms, syn.embed, compact, batch, 20, 16, ids=rows[:10])
