"""Decoding on the GPU: a paged key/value cache, attention of a batch whose
sequences share a long prefix, and sampling.

A thin layer over b2p_kv_append, b2p_kv_read, b2p_attention_prefix and
b2p_sample (include/b2p.h has their definitions) for torch tensors. All work
goes to torch's current stream of the current device, which has to be the
tensors' own (the library launches there); nothing synchronises. There is no
backward pass: under autograd, inputs that require a gradient are refused.
Argument errors raise `B2PError` (from the library) or `ValueError` (shapes and
types of the tensors). Indices on the device (slots, positions, page ids,
lengths) are checked there: `check()` raises if any was out of range.

The reference generates with a numpy forward and top-k sampling
(generate.py:161); a step here is

    q = cache.append(qkv, heads, slots, positions, table)      # rotate, quantise, write
    y = attend(q, cache, prefix_pages, prefix_len, suffix_pages, suffix_lens)
    tokens, logprobs = sample(logits, u, temperature, top_k, top_p, min_p)

with the projections between them on b2p_gemm (examples/complete.py).
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib
from ._lib import KV_16, KV_E4M3, KV_INT8, B2PError, KVCacheDesc

HEAD_DIM = 64
_DTYPE = {torch.float16: 0, torch.bfloat16: 1}
_LOGITS = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_KIND = {torch.int8: KV_INT8, torch.float8_e4m3fn: KV_E4M3, torch.float16: KV_16, torch.bfloat16: KV_16}


_bound: dict = {}


def _fn(name):
    """The library's entry point."""
    f = _bound.get(name)
    if f is None:
        f = _bound[name] = getattr(_lib.load(), name)
    return f


def _raise(name: str, rc: int):
    raise B2PError(name, rc, _lib.load().b2p_last_error().decode(errors="replace"))


_stream = torch._C._cuda_getCurrentRawStream  # of a device index
_current = torch._C._cuda_getDevice


def _on(device: int) -> int:
    """The current stream of the tensors' device. The library launches on the current device and keeps its status word
    there, so another one is refused: a kernel would start on the wrong GPU with this one's addresses."""
    if device != _current():
        raise ValueError(f"the tensors are on cuda:{device}, the current device is cuda:{_current()}: make theirs "
                         f"current (torch.cuda.set_device or torch.cuda.device) for the call")
    return _stream(device)


def _rows(t: torch.Tensor, name: str, dtypes=_DTYPE) -> torch.Tensor:
    if t.dim() != 2 or t.dtype not in dtypes or not t.is_cuda or (t.stride(1) != 1 and t.shape[1] > 1):
        raise ValueError(f"{name} must be a CUDA matrix of {[str(d) for d in dtypes]} with contiguous rows")
    if t.requires_grad and torch.is_grad_enabled():  # (what comes back would have no history, without a word)
        raise ValueError(f"{name} requires a gradient and these operators have none: detach it, or call under no_grad")
    return t


def _vec(t, name: str, dtype, n: int, device: int):
    """A contiguous vector's address; None gives NULL."""
    if t is None:
        return None
    if t.dtype is not dtype or t.numel() != n or t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of {n} values on cuda:{device}")
    return t.data_ptr()


def _ld(t: torch.Tensor) -> int:
    if t.shape[0] <= 1:  # no second row: any pitch that keeps 16 bytes does
        return t.shape[1] + -t.shape[1] % 8
    ld = t.stride(0)
    if ld >= 1 << 31:  # (ctypes would cut it off)
        raise ValueError(f"a row pitch of {ld} elements is more than the library takes (2^31 - 1)")
    return ld


def check(stream: int | None = None) -> None:
    """Wait for `stream` (default: the current one) and raise if a kernel on the current device recorded a bad index or
    a failed wait."""
    if stream is None:
        stream = torch.cuda.current_stream().cuda_stream
    _lib.call("b2p_device_status", stream)


def rope_table(positions: int, rot: int = HEAD_DIM, theta: float = 10000.0, scale: float = 1.0,
               yarn: tuple[float, float, float] | None = None, device="cuda") -> torch.Tensor:
    """Cosine and sine of every position's angles, computed in 64 bits: fp32 [positions, rot/2, 2].

    Pair i turns by position·theta^(-2i/rot) (training/cpu_ops.h:303-307). For contexts longer than the training's:
    `scale` s divides every angle by s (position interpolation); with yarn = (trained_positions, fast, slow) a pair
    that makes more than `fast` turns over trained_positions keeps its angle, one that makes fewer than `slow` is
    divided by s, those between are blended linearly in the pair index, and cosines and sines carry the factor
    0.1·ln(s) + 1 (the attention temperature of that scheme: YaRN, Peng, Quesnelle, Fan and Shippole, 2023, from
    which the steps are)."""
    if rot % 16 or not 0 < rot <= HEAD_DIM:
        raise ValueError(f"rot must be 16, 32, 48 or {HEAD_DIM} (got {rot})")
    i = torch.arange(rot // 2, dtype=torch.float64)
    freq = theta ** (-2.0 * i / rot)
    size = 1.0
    if yarn is not None:
        trained, fast, slow = yarn
        pair = lambda turns: rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        lo, hi = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), rot - 1)
        blend = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        blend[i >= pair(slow)] = 1.0  # (the first pair, too, where none makes as many turns)
        freq = freq * (1 - blend) + freq / scale * blend
        size = 0.1 * math.log(scale) + 1.0 if scale > 1 else 1.0
    else:
        freq = freq / scale
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * freq
    return (torch.stack((angle.cos(), angle.sin()), -1) * size).float().to(device)


class KVCache:
    """A paged cache over the caller's tensors: k and v [n_pages, kv_heads, page_size, 64] of int8, float8_e4m3fn or
    the compute dtype; 8-bit caches have k_scale and v_scale, fp32 [n_pages, kv_heads, page_size]."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None):
        if k.dim() != 4 or k.shape[3] != HEAD_DIM or k.dtype not in _KIND or not k.is_cuda:
            raise ValueError("k must be a CUDA tensor [n_pages, kv_heads, page_size, 64] of int8, float8_e4m3fn, "
                             "float16 or bfloat16")
        if v.shape != k.shape or v.dtype != k.dtype or v.device != k.device:
            raise ValueError("v must be like k")
        kind = _KIND[k.dtype]
        scales = [] if kind == KV_16 else [k_scale, v_scale]
        for s in scales:
            if s is None or s.dtype != torch.float32 or s.shape != k.shape[:3] or s.device != k.device:
                raise ValueError("8-bit caches need fp32 k_scale and v_scale [n_pages, kv_heads, page_size]")
        if not all(t.is_contiguous() for t in (k, v, *scales)):
            raise ValueError("cache tensors must be contiguous")
        self.k, self.v = k, v
        self.k_scale, self.v_scale = scales or (None, None)
        self.n_pages, self.kv_heads, self.page_size, _ = k.shape
        self.kind, self.device, self._dev = kind, k.device, k.get_device()
        self._desc = KVCacheDesc(k.data_ptr(), v.data_ptr(), *(s.data_ptr() for s in scales or ()),
                                 *((None, None) if not scales else ()), self.n_pages, self.page_size, self.kv_heads,
                                 kind)
        self._ref = C.addressof(self._desc)

    @classmethod
    def empty(cls, n_pages: int, page_size: int, kv_heads: int, dtype: torch.dtype = torch.int8,
              device="cuda") -> "KVCache":
        """A new cache of `n_pages` pages (uninitialised)."""
        shape = (n_pages, kv_heads, page_size, HEAD_DIM)
        new = lambda: torch.empty(shape, dtype=dtype, device=device)  # noqa: E731
        scale = (lambda: torch.empty(shape[:3], device=device)) if _KIND.get(dtype) != KV_16 else (lambda: None)
        return cls(new(), new(), scale(), scale())

    def _dtype(self, dtype: torch.dtype) -> int:
        if dtype not in _DTYPE or (self.kind == KV_16 and dtype != self.k.dtype):
            raise ValueError(f"the cache holds {self.k.dtype}: {dtype} does not go with it")
        return _DTYPE[dtype]

    def append(self, qkv: torch.Tensor, heads: int, slots: torch.Tensor, positions: torch.Tensor | None = None,
               table: torch.Tensor | None = None, interleaved: bool = False,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """Write the K and V of qkv [n, 64·(heads + 2·kv_heads)] to `slots` (int32 [n]; negative: skip), rotated by
        `table` (see rope_table; None: no rotation) at `positions` (int32 [n]). Returns rotated Q [n, 64·heads]
        (`out`, which may be a view of qkv)."""
        n, cols = _rows(qkv, "qkv").shape
        q_cols, dev, stream = heads * HEAD_DIM, self._dev, _on(self._dev)
        if cols < q_cols + 2 * HEAD_DIM * self.kv_heads or qkv.get_device() != dev:
            raise ValueError(f"qkv must have {q_cols + 2 * HEAD_DIM * self.kv_heads} columns, on {self.device}")
        if out is None:
            out = qkv.new_empty((n, q_cols))
            ld_out = q_cols
        else:
            if out.shape != (n, q_cols) or out.dtype is not qkv.dtype or out.get_device() != dev:
                raise ValueError(f"out must be {qkv.dtype} [{n}, {q_cols}] on {self.device}")
            ld_out = _ld(_rows(out, "out"))
        max_pos = rot = 0
        angles = None
        if table is not None:
            if table.dim() != 3 or table.shape[2] != 2 or positions is None:
                raise ValueError("table must be [positions, rot/2, 2], and goes with positions")
            max_pos, rot = table.shape[0], 2 * table.shape[1]
            angles = _vec(table, "table", torch.float32, max_pos * rot, dev)
        rc = _fn("b2p_kv_append")(
            self._ref, qkv.data_ptr(), _ld(qkv), heads, out.data_ptr(), ld_out,
            _vec(slots, "slots", torch.int32, n, dev), _vec(positions, "positions", torch.int32, n, dev), angles,
            max_pos, rot, 1 if interleaved else 0, n, self._dtype(qkv.dtype), stream)
        if rc:
            _raise("b2p_kv_append", rc)
        return out

    def read(self, slots: torch.Tensor, dtype: torch.dtype, k_out: torch.Tensor | None = None,
             v_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The K and V of `slots` (int32 [n]; negative: zeros) as [n, 64·kv_heads] of `dtype`."""
        n, cols, dev = slots.numel(), HEAD_DIM * self.kv_heads, self._dev
        code, stream = self._dtype(dtype), _on(dev)
        for name, t in (("k_out", k_out), ("v_out", v_out)):
            if t is not None and (t.shape != (n, cols) or t.dtype is not dtype or t.get_device() != dev):
                raise ValueError(f"{name} must be {dtype} [{n}, {cols}] on {self.device}")
        k = torch.empty((n, cols), dtype=dtype, device=self.device) if k_out is None else _rows(k_out, "k_out")
        v = torch.empty_like(k) if v_out is None else _rows(v_out, "v_out")
        rc = _fn("b2p_kv_read")(self._ref, _vec(slots, "slots", torch.int32, n, dev), n, k.data_ptr(),
                                cols if k_out is None else _ld(k), v.data_ptr(), cols if v_out is None else _ld(v),
                                code, stream)
        if rc:
            _raise("b2p_kv_read", rc)
        return k, v


class PrefixAttention:
    """Attention of `batch` sequences with `q_len` queries each over a shared prefix and their own suffixes, with the
    workspace that calls up to max_prefix and max_suffix tokens need. Calls on one object share it: keep them on one
    stream, or ordered."""

    def __init__(self, batch: int, q_len: int, heads: int, kv_heads: int, max_prefix: int, max_suffix: int,
                 device="cuda"):
        size = _fn("b2p_attention_prefix_workspace")(batch, q_len, heads, kv_heads, max_prefix, max_suffix)
        if not size:
            raise ValueError("batch, q_len, heads, kv_heads, max_prefix or max_suffix out of range")
        self.batch, self.q_len, self.heads, self.kv_heads = batch, q_len, heads, kv_heads
        self.max_prefix, self.max_suffix = max_prefix, max_suffix
        self.workspace = torch.empty(size, dtype=torch.uint8, device=device)
        self._ws, self._ws_bytes = self.workspace.data_ptr(), size

    def __call__(self, q: torch.Tensor, cache: KVCache, prefix_pages: torch.Tensor | None, prefix_len: int,
                 suffix_pages: torch.Tensor | None, suffix_lens: torch.Tensor | None, out: torch.Tensor | None = None,
                 return_lse: bool = False):
        """q [batch·q_len, 64·heads]; prefix_pages int32 [ceil(prefix_len/page_size)]; suffix_pages int32
        [batch, pages]; suffix_lens int32 [batch] (None: no suffixes; lengths above max_suffix or the pages are reported
        by `check()`). Returns out, or (out, lse [batch·q_len, heads])."""
        n, cols, dev = self.batch * self.q_len, self.heads * HEAD_DIM, cache._dev
        if _rows(q, "q").shape != (n, cols) or q.get_device() != dev or cache.kv_heads != self.kv_heads:
            raise ValueError(f"q must be [{n}, {cols}] on {cache.device}, the cache have {self.kv_heads} KV heads")
        stream = _on(dev)
        if self.workspace.get_device() != dev:
            raise ValueError(f"the workspace is on {self.workspace.device}, the cache on {cache.device}")
        if not 0 <= prefix_len <= self.max_prefix:
            raise ValueError(f"prefix_len must be from 0 to {self.max_prefix}")
        prefix = pages = lens = None
        pitch = most = 0
        if prefix_len:
            if prefix_pages is None or prefix_pages.numel() * cache.page_size < prefix_len:
                raise ValueError(f"prefix_pages must name {-(-prefix_len // cache.page_size)} pages")
            prefix = _vec(prefix_pages, "prefix_pages", torch.int32, prefix_pages.numel(), dev)
        if suffix_lens is not None:  # (where there is no room for a suffix, the lengths are still checked)
            lens = _vec(suffix_lens, "suffix_lens", torch.int32, self.batch, dev)
            if self.max_suffix:
                if suffix_pages is None or suffix_pages.dim() != 2 or suffix_pages.shape[0] != self.batch:
                    raise ValueError("suffix_pages must be [batch, pages]")
                pitch = suffix_pages.shape[1]
                most = min(self.max_suffix, pitch * cache.page_size)
                if most:
                    pages = _vec(suffix_pages, "suffix_pages", torch.int32, self.batch * pitch, dev)
        ld_q = _ld(q)
        if out is None:
            out = torch.empty_like(q) if ld_q == cols else q.new_empty((n, cols))
        elif out.shape != q.shape or out.dtype is not q.dtype or out.get_device() != dev:
            raise ValueError("out must be like q")
        lse = q.new_empty((n, self.heads), dtype=torch.float32) if return_lse else None
        rc = _fn("b2p_attention_prefix")(
            cache._ref, q.data_ptr(), ld_q, out.data_ptr(), _ld(_rows(out, "out")),
            None if lse is None else lse.data_ptr(), self.batch, self.q_len, self.heads, prefix, prefix_len, pages,
            pitch, lens, most, cache._dtype(q.dtype), self._ws, self._ws_bytes, stream)
        if rc:
            _raise("b2p_attention_prefix", rc)
        return (out, lse) if return_lse else out


def sample(logits: torch.Tensor, u: torch.Tensor, temperature: torch.Tensor | None = None,
           top_k: torch.Tensor | None = None, top_p: torch.Tensor | None = None, min_p: torch.Tensor | None = None,
           out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """A token for each row of logits [n, vocab] (float16, bfloat16 or float32) from uniform numbers u (fp32 [n]),
    with per-row temperature, top_p, min_p (fp32 [n]) and top_k (int32 [n]); None turns a filter off. Returns tokens
    (int32 [n]; `out`) and the natural logs of their probabilities among the kept tokens (fp32 [n])."""
    n, vocab = _rows(logits, "logits", _LOGITS).shape
    dev = logits.get_device()
    stream = _on(dev)
    if u is None:
        raise ValueError("u is needed")
    logprobs = torch.empty_like(u)
    f32, i32 = torch.float32, torch.int32
    if out is None:
        out = torch.empty_like(u, dtype=i32)
    rc = _fn("b2p_sample")(
        logits.data_ptr(), _ld(logits), n, vocab, _LOGITS[logits.dtype], _vec(u, "u", f32, n, dev),
        _vec(temperature, "temperature", f32, n, dev), _vec(top_k, "top_k", i32, n, dev),
        _vec(top_p, "top_p", f32, n, dev), _vec(min_p, "min_p", f32, n, dev), _vec(out, "out", i32, n, dev),
        logprobs.data_ptr(), stream)
    if rc:
        _raise("b2p_sample", rc)
    return out, logprobs
