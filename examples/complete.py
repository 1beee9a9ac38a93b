"""Complete one prompt many times: the decoding operators together.

A randomly initialised model of SmolLM2-360M's shape (or fewer layers of it)
reads a prompt once and continues it as `--batch` samples that share the
prompt's keys and values. The reference completes text one sample at a time on
the CPU (generate.py:161).

    python examples/complete.py --prompt 1000 --batch 16 --new 64

A layer's projections run on b2p_gemm. For the prompt, `KVCache.append` rotates
and quantises, `KVCache.read` gives back the keys and values as the cache has
them, and b2p_attention takes them; for every later token, `append` and
`PrefixAttention` do. `sample` draws the tokens. Between these, RMSNorm, SiLU
and the residual sums are torch's.
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from autoane_b200 import _lib, decode  # noqa: E402
from autoane_b200.model import Config  # noqa: E402

PAGE = 64


def gemm(x: torch.Tensor, w: torch.Tensor, out_f32: bool = False) -> torch.Tensor:
    """x [n, k] · w [m, k]ᵀ on the tile engine."""
    y = torch.empty(x.shape[0], w.shape[0], dtype=torch.float32 if out_f32 else x.dtype, device=x.device)
    _lib.call("b2p_gemm", x.data_ptr(), w.data_ptr(), y.data_ptr(), x.shape[0], w.shape[0], x.shape[1], w.shape[0],
              0 if x.dtype is torch.float16 else 1, int(out_f32), torch.cuda.current_stream().cuda_stream)
    return y


class Completer:
    """`weights`: lists by layer of Wq, Wk, Wv, Wo, W1, W2, W3 [out, in] (adapters merged); `rms` [2·layers + 1, dim]:
    the attention's and the feed-forward's norm of every layer, then the last one; `embed` [vocab, dim]; `head`
    [tokens, dim]: the rows of the embedding that a token may be drawn from, and `ids` which rows of `embed` they are (a
    compacted vocabulary's ids; None: the first ones, in order)."""

    def __init__(self, cfg: Config, weights: dict, rms, embed, head, batch: int, max_prompt: int, max_new: int,
                 kv: torch.dtype = torch.int8, dtype: torch.dtype = torch.float16, ids=None):
        put = lambda a: torch.as_tensor(a).to("cuda", dtype).contiguous()  # noqa: E731
        self.cfg, self.batch, self.max_prompt, self.max_new, self.dtype = cfg, batch, max_prompt, max_new, dtype
        layers = range(cfg.nlayers)
        w = {k: [put(a) for a in v] for k, v in weights.items()}
        self.qkv = [torch.cat([w["Wq"][l], w["Wk"][l], w["Wv"][l]]) for l in layers]
        self.up = [torch.cat([w["W1"][l], w["W3"][l]]) for l in layers]
        self.o, self.down = w["Wo"], w["W2"]
        self.rms = torch.as_tensor(rms).to("cuda", torch.float32)
        self.embed, self.head = torch.as_tensor(embed).to("cuda", torch.float32), put(head)
        self.ids = torch.arange(len(head), device="cuda") if ids is None else torch.as_tensor(ids).to("cuda", torch.long)
        if self.ids.shape != (self.head.shape[0],):
            raise ValueError("ids must name an embedding row for each row of head")

        prompt_pages, own_pages = -(-max_prompt // PAGE), -(-max_new // PAGE)
        self.cache = [decode.KVCache.empty(prompt_pages + batch * own_pages, PAGE, cfg.kv_heads, kv) for _ in layers]
        self.prompt_pages = torch.arange(prompt_pages, dtype=torch.int32, device="cuda")
        self.own_pages = (prompt_pages + torch.arange(batch * own_pages, dtype=torch.int32, device="cuda")).view(
            batch, own_pages)
        self.attend = decode.PrefixAttention(batch, 1, cfg.heads, cfg.kv_heads, max_prompt, max_new)
        self.table = decode.rope_table(PAGE * (prompt_pages + own_pages), decode.HEAD_DIM, cfg.rope_theta)
        self.prompt_len = self.new = 0

    def _norm(self, x, i):
        return (x * torch.rsqrt(x.square().mean(1, keepdim=True) + 1e-5) * self.rms[i]).to(self.dtype)

    def _layers(self, tokens, slots, positions, attend):
        """Hidden states of the tokens; attend(layer, qkv) sees rotated queries in qkv's first columns."""
        cfg, q_cols = self.cfg, self.cfg.heads * decode.HEAD_DIM
        x = self.embed[tokens]
        for l in range(cfg.nlayers):
            qkv = gemm(self._norm(x, 2 * l), self.qkv[l])
            self.cache[l].append(qkv, cfg.heads, slots, positions, self.table, interleaved=True, out=qkv[:, :q_cols])
            x = x + cfg.res_alpha * gemm(attend(l, qkv), self.o[l], True)
            gate, up = gemm(self._norm(x, 2 * l + 1), self.up[l], True).chunk(2, 1)
            x = x + cfg.res_alpha * gemm((torch.nn.functional.silu(gate) * up).to(self.dtype), self.down[l], True)
        return x

    def _logits(self, x):
        return gemm(self._norm(x, 2 * self.cfg.nlayers), self.head, True)

    def prefill(self, prompt: torch.Tensor, all_logits: bool = False) -> torch.Tensor:
        """Reads the prompt (token ids); logits after its last token, or after each."""
        n, cfg = prompt.numel(), self.cfg
        if not 1 <= n <= self.max_prompt:
            raise ValueError(f"the prompt must have 1 to {self.max_prompt} tokens")
        padded = -(-n // 64) * 64  # b2p_attention's step; the tokens added are behind all others and keep no slot
        q_cols, kv_cols = cfg.heads * decode.HEAD_DIM, cfg.kv_heads * decode.HEAD_DIM
        positions = torch.arange(padded, dtype=torch.int32, device="cuda")
        slots = torch.where(positions < n, positions, -1)  # the prompt's pages are the first ones, in order

        def attend(l, qkv):
            self.cache[l].read(slots, self.dtype, qkv[:, q_cols:q_cols + kv_cols], qkv[:, q_cols + kv_cols:])
            out = torch.empty(padded, q_cols, dtype=self.dtype, device="cuda")
            _lib.call("b2p_attention", qkv.data_ptr(), qkv.stride(0), out.data_ptr(), q_cols, None, 1, padded,
                      cfg.heads, cfg.kv_heads, 0 if self.dtype is torch.float16 else 1,
                      torch.cuda.current_stream().cuda_stream)
            return out

        tokens = torch.nn.functional.pad(prompt.cuda().long(), (0, padded - n))
        x = self._layers(tokens, slots, positions, attend)
        self.prompt_len, self.new = n, 0
        return self._logits(x[:n] if all_logits else x[n - 1:n])

    def step(self, tokens: torch.Tensor) -> torch.Tensor:
        """Appends one token to each sample; logits [batch, tokens] after it."""
        if self.new == self.max_new:
            raise ValueError(f"the cache holds {self.max_new} new tokens a sample")
        at = self.new
        slots = self.own_pages[:, at // PAGE] * PAGE + at % PAGE
        positions = torch.full_like(slots, self.prompt_len + at)
        lens = torch.full_like(slots, at + 1)
        q_cols = self.cfg.heads * decode.HEAD_DIM
        x = self._layers(tokens.long(), slots, positions, lambda l, qkv: self.attend(
            qkv[:, :q_cols], self.cache[l], self.prompt_pages, self.prompt_len, self.own_pages, lens))
        self.new += 1
        return self._logits(x)

    def complete(self, prompt: torch.Tensor, new: int, u: torch.Tensor, **filters) -> torch.Tensor:
        """`new` tokens for every sample after a prompt of `embed`'s rows, drawn by u [new, batch]: indices into `head`'s
        rows, [batch, new]. The filters are `sample`'s."""
        logits = self.prefill(prompt).expand(self.batch, -1).contiguous()
        out = []
        for i in range(new):
            tokens, _ = decode.sample(logits, u[i], **filters)
            out.append(tokens)
            if i + 1 < new:
                logits = self.step(self.ids[tokens.long()])
        return torch.stack(out, 1)


def random_weights(cfg: Config, seed: int = 0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda *shape: torch.randn(*shape, device="cuda", generator=g) * 0.02  # noqa: E731
    q, kv, d, h = cfg.heads * 64, cfg.kv_heads * 64, cfg.dim, cfg.hidden
    shapes = {"Wq": (q, d), "Wk": (kv, d), "Wv": (kv, d), "Wo": (d, q), "W1": (h, d), "W2": (d, h), "W3": (h, d)}
    weights = {k: [new(*s) for _ in range(cfg.nlayers)] for k, s in shapes.items()}
    return weights, torch.ones(2 * cfg.nlayers + 1, d), new(cfg.vocab, d)


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=32)
    ap.add_argument("--prompt", type=int, default=1000, help="tokens of the prompt")
    ap.add_argument("--batch", type=int, default=16, help="samples")
    ap.add_argument("--new", type=int, default=64, help="tokens of each sample")
    ap.add_argument("--kv", choices=["int8", "e4m3", "f16"], default="int8")
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args()
    _lib.call("b2p_init", torch.cuda.current_device())
    cfg = Config(nlayers=a.layers)
    weights, rms, embed = random_weights(cfg, a.seed)
    kv = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn, "f16": torch.float16}[a.kv]
    c = Completer(cfg, weights, rms, embed, embed, a.batch, a.prompt, a.new, kv)
    g = torch.Generator(device="cuda").manual_seed(a.seed + 1)
    prompt = torch.randint(cfg.vocab, (a.prompt,), device="cuda", generator=g)
    u = torch.rand(a.new, a.batch, device="cuda", generator=g)
    per = lambda v, t=torch.float32: torch.full((a.batch,), v, dtype=t, device="cuda")  # noqa: E731
    filters = dict(temperature=per(0.8), top_k=per(50, torch.int32), top_p=per(0.95))
    c.complete(prompt, min(a.new, 4), u, **filters)  # the first pass loads the kernels
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    tokens = c.complete(prompt, a.new, u, **filters)
    decode.check()
    t1 = time.perf_counter()
    print(tokens[:2].tolist())
    print(f"{a.layers} layers, prompt {a.prompt}, {a.batch} x {a.new} tokens, {a.kv} cache: {t1 - t0:.3f} s, "
          f"{a.batch * a.new / (t1 - t0):.0f} tokens/s")


if __name__ == "__main__":
    main()
