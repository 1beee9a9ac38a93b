"""The decoding operators in a model (examples/complete.py) against `Model`'s forward pass.

The same weights and tokens give the same mean loss by two ways: `Model.eval` over whole sequences, and the prompt's
pass followed by single tokens over the shared prefix. Both compute in fp16 with fp32 sums, so they agree to the 1e-3
nats that the workload allows of a loss. An int8 cache changes a logit by at most about 0.4% of its spread (0.6 here), a
mean of 128 losses by a few 1e-4: 2e-3.
"""
import importlib.util
import os

import numpy as np
import pytest
import torch

from autoane_b200 import decode
from autoane_b200.model import Config, Model, load_synthetic
from tests import _models as M

pytestmark = pytest.mark.gpu


def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "complete.py")
    spec = importlib.util.spec_from_file_location("complete", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def setup(prompt_len, seq=128, n_active=3000, batch=2, kv=torch.float16):
    cfg = M.small_cfg(nlayers=2, seq=seq)
    syn = M.make_model(cfg, n_active=n_active, seed=11, rms_jitter=0.05)
    mc = Config(dim=cfg.dim, hidden=cfg.hidden, heads=cfg.heads, kv_heads=cfg.kv_heads, head_dim=cfg.hd, seq=seq,
                nlayers=2, vocab=cfg.vocab, rank=cfg.rank, rope_theta=cfg.rope_theta, max_groups=4)
    rms = np.stack([syn.theta[s] for s in M.rms_slices(syn)])
    c = example().Completer(mc, syn.weights, rms, syn.embed, syn.cembed, batch, max(prompt_len, 1), seq, kv)
    return syn, mc, c


@pytest.mark.parametrize("prompt_len", [1, 64, 77])
@pytest.mark.parametrize("kv,tol", [(torch.float16, 1e-3), (torch.int8, 2e-3)])
def test_loss_matches_the_models(b2p, prompt_len, kv, tol):
    seq, batch = 128, 2
    syn, mc, c = setup(prompt_len, seq, kv=kv)
    model = Model(mc)
    load_synthetic(model, syn.weights, syn.embed, syn.compact_to_full, syn.theta)
    toks = M.make_tokens(2 * seq + 2, 3000, seed=3).reshape(batch, seq + 1)
    toks[1, :prompt_len] = toks[0, :prompt_len]
    want = []
    for b in range(batch):
        tgt = syn.full_to_compact[toks[b, 1:]].astype(np.uint16)
        want.append(float(model.eval(toks[b:b + 1, :seq], tgt[None], [(0, 0, 0.0, 0.0)])[0]))
    model.close()

    ids = torch.from_numpy(toks.astype(np.int64)).cuda()  # compact ids are the full ones here
    nll = torch.zeros(batch, seq, device="cuda")
    first = torch.log_softmax(c.prefill(ids[0, :prompt_len], all_logits=True).double(), 1)
    for b in range(batch):
        nll[b, :prompt_len] = -first.gather(1, ids[b, 1:prompt_len + 1, None])[:, 0]
    for i in range(prompt_len, seq):
        logp = torch.log_softmax(c.step(ids[:, i]).double(), 1)
        nll[:, i] = -logp.gather(1, ids[:, i + 1:i + 2])[:, 0]
    decode.check()
    got = nll.mean(1).tolist()
    assert np.abs(np.array(got) - want).max() < tol, (got, want)


def test_complete(b2p):
    """Greedy samples are the same in every row and the argmax of the logits; draws repeat for the same numbers."""
    syn, mc, c = setup(70, batch=3, kv=torch.int8)
    prompt = torch.arange(70, device="cuda") * 37 % 3000
    g = torch.Generator(device="cuda").manual_seed(0)
    u = torch.rand(9, 3, device="cuda", generator=g)
    cold = c.complete(prompt, 9, u, temperature=torch.zeros(3, device="cuda"))
    assert cold.shape == (3, 9) and torch.equal(cold, cold[:1].expand(3, 9))
    assert int(c.prefill(prompt)[0].argmax()) == int(cold[0, 0])
    filters = dict(temperature=torch.full((3,), 0.9, device="cuda"), top_p=torch.full((3,), 0.9, device="cuda"))
    a = c.complete(prompt, 9, u, **filters)
    assert torch.equal(a, c.complete(prompt, 9, u, **filters)) and not torch.equal(a[0], a[1])
    with pytest.raises(ValueError, match="prompt"):
        c.prefill(torch.zeros(71, dtype=torch.int64))
    decode.check()


def test_graph_replays(b2p):
    """A captured decoding step gives what the plain one gives."""
    syn, mc, c = setup(70, batch=2, kv=torch.int8)
    c.prefill(torch.arange(70, device="cuda") * 37 % 3000)
    tokens, u = torch.tensor([5, 2900], device="cuda"), torch.tensor([0.2, 0.7], device="cuda")
    k = torch.full((2,), 40, dtype=torch.int32, device="cuda")
    want = decode.sample(c.step(tokens), u, top_k=k)
    c.new = 0  # the same token again
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        decode.sample(c.step(tokens), u, top_k=k)
        c.new = 0
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = decode.sample(c.step(tokens), u, top_k=k)
    for t in got:
        t.zero_()
    graph.replay()
    decode.check()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    del graph
