"""The decoding operators' cases, and their plain forms.

Three operators make one decoding step: writing new tokens' keys and values into a paged cache (rotated and
quantised) and reading them back; attention of a batch whose sequences share a long prefix, over that cache; and
sampling the next tokens from the logits. A head has 64 channels throughout.
"""
import math

import numpy as np
import torch

own = False

HD = 64
LOG2E = 1.4426950408889634
KINDS = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
TINY = 1e-30        # smallest |x| maximum a vector is scaled by
KEY = float(1 << 20)  # sampling: steps of log2 probability below the maximum
ONE = float(1 << 31)  # sampling: the weight of the likeliest token
BOTTOM = 64.0       # sampling: the depth, in log2, below which nothing is told apart


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decoding step of eight completions of one prompt: the smallest write, where latency counts
        dict(name="kv_step", op="kv", tokens=8, heads=15, kv_heads=5, kind="int8", dtype="f16", page=16, rot=64,
             interleaved=False, base=1000),
        # a ragged chunk of a prompt far into a long context; rotation of half the head, interleaved pairs
        dict(name="kv_chunk", op="kv", tokens=2051, heads=24, kv_heads=6, kind="e4m3", dtype="bf16", page=64, rot=32,
             interleaved=True, base=60000),
        # a whole long prompt, written at once and read back for dense attention
        dict(name="kv_prompt", op="kv", tokens=65536, heads=15, kv_heads=5, kind="int8", dtype="f16", page=64, rot=64,
             interleaved=False, base=0),
        # a single completion of a short prompt, unquantised cache: the smallest attention
        dict(name="attn_one", op="attn", batch=1, queries=1, heads=8, kv_heads=2, kind="16", dtype="f16", page=16,
             prefix=200, suffix=33),
        # eight completions of a prompt, soon after it
        dict(name="attn_samples", op="attn", batch=8, queries=1, heads=15, kv_heads=5, kind="int8", dtype="f16",
             page=16, prefix=1023, suffix=129),
        # several queries per sequence (drafted tokens being checked), unquantised cache, odd lengths
        dict(name="attn_verify", op="attn", batch=20, queries=4, heads=24, kv_heads=6, kind="16", dtype="bf16",
             page=64, prefix=4001, suffix=700),
        # a batch under one long system prompt, a key head for every query head
        dict(name="attn_wide", op="attn", batch=64, queries=1, heads=12, kv_heads=12, kind="e4m3", dtype="bf16",
             page=32, prefix=8192, suffix=300),
        # many completions of one long document: the largest attention
        dict(name="attn_long", op="attn", batch=256, queries=1, heads=15, kv_heads=5, kind="int8", dtype="f16",
             page=64, prefix=32768, suffix=512),
        # one row of logits, as a single completion samples it: the smallest sampling
        dict(name="sample_one", op="sample", rows=1, vocab=49152, dtype="f32", top_k=50, top_p=1.0, min_p=0.0),
        # a batch over a compacted vocabulary of odd size, by nucleus alone
        dict(name="sample_compact", op="sample", rows=33, vocab=16893, dtype="bf16", top_k=0, top_p=0.95, min_p=0.0),
        # a batch with every filter in use
        dict(name="sample_batch", op="sample", rows=256, vocab=49152, dtype="f16", top_k=200, top_p=0.9, min_p=0.02),
        # many rows of 32-bit logits from the whole distribution
        dict(name="sample_rows", op="sample", rows=1024, vocab=32000, dtype="f32", top_k=0, top_p=1.0, min_p=0.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["kv", "attn", "attn", "sample"])
    heads, kv_heads = rng.choice([(15, 5), (9, 3), (8, 2), (24, 6), (32, 8), (12, 12), (16, 1)])
    dtype = rng.choice(["f16", "bf16"])
    if op == "kv":
        rot = rng.choice([64, 64, 32, 16, 0])
        tokens = min(_log(rng, 1, 65536), 65536 * 25 // (heads + 2 * kv_heads))
        return dict(op="kv", tokens=tokens, heads=heads, kv_heads=kv_heads, kind=rng.choice(["int8", "e4m3", "16"]),
                    dtype=dtype, page=rng.choice([8, 16, 32, 64, 128, 256]), rot=rot,
                    interleaved=rng.random() < 0.5, base=rng.randrange(0, 60000))
    if op == "attn":
        queries = rng.choice([1, 1, 1, 2, 3, 5, 8])
        prefix = 0 if rng.random() < 0.1 else _log(rng, 1, 32768)
        suffix = 0 if prefix and rng.random() < 0.1 else _log(rng, 1, 4096)
        batch = _log(rng, 1, 256)
        # no more than the largest listed case: its rows times its keys, and the keys held by all sequences
        while batch > 1 and (batch * queries * heads * (prefix + suffix) > 256 * 15 * 33000
                             or batch * suffix * kv_heads > 256 * 512 * 5):
            batch = batch * 2 // 3
        while queries > 1 and batch * queries * heads * (prefix + suffix) > 256 * 15 * 33000:
            queries -= 1
        return dict(op="attn", batch=batch, queries=queries, heads=heads, kv_heads=kv_heads,
                    kind=rng.choice(["int8", "e4m3", "16"]), dtype=dtype, page=rng.choice([8, 16, 32, 64, 128]),
                    prefix=prefix, suffix=suffix)
    vocab = rng.choice([49152, 32000, 16893, 8191, _log(rng, 100, 50000)])
    return dict(op="sample", rows=_log(rng, 1, min(1024, 1024 * 32000 // vocab)), vocab=vocab,
                dtype=rng.choice(["f16", "bf16", "f32"]), top_k=rng.choice([0, 0, 1, 20, 50, 1000]),
                top_p=rng.choice([1.0, 0.99, 0.9, 0.5]), min_p=rng.choice([0.0, 0.0, 0.01, 0.1]))


def _suffix_lens(case):
    """Completions are of every length from none to the longest; which sequence has which goes by the seed."""
    b, n = case["batch"], case["suffix"]
    return [n] if b == 1 else [n * i // (b - 1) for i in range(b)]


def work(case):
    if case["op"] == "kv":
        n, h, g = case["tokens"], case["heads"], case["kv_heads"]
        held = 2 * g * (HD + 4 if case["kind"] in KINDS else 2 * HD)
        read = (h + 2 * g) * HD * 2 + 8 + case["rot"] * 4
        return {"bytes": n * (read + h * HD * 2 + 2 * held + 2 * g * HD * 2 + 4),
                "flops": n * ((h + g) * case["rot"] * 3 + 2 * g * HD * 3)}
    if case["op"] == "attn":
        lens, q = _suffix_lens(case), case["queries"]
        rows = case["batch"] * q * case["heads"]
        held = 2 * case["kv_heads"] * (HD + 4 if case["kind"] in KINDS else 2 * HD)
        seen = sum(max(0, n - (q - 1 - i)) for n in lens for i in range(q))
        return {"bytes": rows * (2 * HD * 2 + 4) + (case["prefix"] + sum(lens)) * held,
                "flops": 4 * HD * (rows * case["prefix"] + case["heads"] * seen)}
    size = DTYPES[case["dtype"]].itemsize
    return {"bytes": case["rows"] * (case["vocab"] * size + 28), "flops": 6 * case["rows"] * case["vocab"]}


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _table(base, count, rot, theta=100000.0):
    """cos and sin of every position's angles up to the last one used, rounded once from 64 bits: [position, rot/2, 2]."""
    if not rot:
        return None
    freq = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    ang = torch.arange(base + count, dtype=torch.float64, device="cuda")[:, None] * freq
    return torch.stack((ang.cos(), ang.sin()), -1).float().contiguous()


def _held(case, pages, g):
    """A cache of `pages` pages with keys and values in every slot: channels of unequal size, as trained keys have."""
    shape = (pages, case["kv_heads"], case["page"], HD)
    size = torch.rand((1, case["kv_heads"], 1, HD), device="cuda", generator=g) * 1.5 + 0.25
    k = torch.randn(shape, device="cuda", generator=g) * size
    v = torch.randn(shape, device="cuda", generator=g)
    if case["kind"] == "16":
        return k.to(DTYPES[case["dtype"]]), v.to(DTYPES[case["dtype"]]), None, None
    (k, ks), (v, vs) = _quantise(k, case["kind"]), _quantise(v, case["kind"])
    return k, v, ks, vs


def prepare(case, seed):
    g = _gen(seed)
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "kv":
        n, h, kv, page = case["tokens"], case["heads"], case["kv_heads"], case["page"]
        s["qkv"] = (torch.randn((n, (h + 2 * kv) * HD), device="cuda", generator=g) * 1.3).to(dtype)
        pages = -(-n // page) + 3
        order = torch.randperm(pages, device="cuda", generator=g)
        at = torch.arange(n, device="cuda")
        s["slots"] = (order[at // page] * page + at % page).int()
        s["positions"] = (case["base"] + at).int()
        s["table"] = _table(case["base"], n, case["rot"])
        kind = KINDS.get(case["kind"], dtype)
        shape = (pages, kv, page, HD)
        s["k"], s["v"] = torch.zeros(shape, device="cuda").to(kind), torch.zeros(shape, device="cuda").to(kind)
        scaled = case["kind"] in KINDS
        s["ks"] = torch.zeros(shape[:3], device="cuda") if scaled else None
        s["vs"] = torch.zeros(shape[:3], device="cuda") if scaled else None
    elif case["op"] == "attn":
        b, page = case["batch"], case["page"]
        first = -(-case["prefix"] // page)
        each = -(-case["suffix"] // page)
        pages = first + b * each + 1
        s["k"], s["v"], s["ks"], s["vs"] = _held(case, pages, g)
        order = torch.randperm(pages, device="cuda", generator=g).int()
        s["prefix_pages"] = order[:first].contiguous()
        s["suffix_pages"] = order[first:first + b * each].reshape(b, each).contiguous()
        lens = np.random.RandomState(seed % (1 << 32)).permutation(np.array(_suffix_lens(case), np.int32))
        s["suffix_lens"] = torch.from_numpy(lens.astype(np.int32)).cuda()
        s["q"] = (torch.randn((b * case["queries"], case["heads"] * HD), device="cuda", generator=g) * 1.5).to(dtype)
    else:
        n, vocab = case["rows"], case["vocab"]
        s["logits"] = (torch.randn((n, vocab), device="cuda", generator=g) * 2.5
                       + torch.randn((1, vocab), device="cuda", generator=g)).to(dtype)
        s["u"] = torch.rand((n,), device="cuda", generator=g)
        s["temperature"] = torch.rand((n,), device="cuda", generator=g) * 0.9 + 0.4
        full = lambda v, t: torch.full((n,), v, dtype=t, device="cuda")  # noqa: E731
        s["top_k"] = full(case["top_k"], torch.int32)
        s["top_p"] = full(case["top_p"], torch.float32)
        s["min_p"] = full(case["min_p"], torch.float32)
    if own:
        from autoane_b200 import decode
        if case["op"] != "sample":
            s["cache"] = decode.KVCache(s["k"], s["v"], s["ks"], s["vs"])
        if case["op"] == "attn":
            s["attend"] = decode.PrefixAttention(case["batch"], case["queries"], case["heads"], case["kv_heads"],
                                                 max_prefix=case["prefix"], max_suffix=case["suffix"])
        s["decode"] = decode
    return s


# ---------------------------------------------------------------------------------------------------------------
# the operators
# ---------------------------------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    if case["op"] == "kv":
        return _run_kv(s, case)
    return _run_attn(s, case) if case["op"] == "attn" else _run_sample(s, case)


def _run_kv(s, case):
    if own:
        q = s["cache"].append(s["qkv"], case["heads"], s["slots"], s["positions"], s["table"], case["interleaved"])
        k, v = s["cache"].read(s["slots"], s["qkv"].dtype)
        return {"q": q, "k": k, "v": v}
    dtype, kv, page = s["qkv"].dtype, case["kv_heads"], case["page"]
    n = case["tokens"]
    x = s["qkv"].float().reshape(n, -1, HD)
    q, k, v = x[:, :case["heads"]], x[:, case["heads"]:case["heads"] + kv], x[:, case["heads"] + kv:]
    q, k = _rotate(q, s, case), _rotate(k, s, case)
    at = (s["slots"].long() // page, slice(None), s["slots"].long() % page)
    if case["kind"] == "16":
        s["k"][at], s["v"][at] = k.to(dtype), v.to(dtype)
        back = s["k"][at], s["v"][at]
    else:
        s["k"][at], s["ks"][at] = _quantise(k, case["kind"])
        s["v"][at], s["vs"][at] = _quantise(v, case["kind"])
        back = s["k"][at].float() * s["ks"][at][..., None], s["v"][at].float() * s["vs"][at][..., None]
    return {"q": q.to(dtype).reshape(n, -1), "k": back[0].to(dtype).reshape(n, -1), "v": back[1].to(dtype).reshape(n, -1)}


def _rotate(x, s, case):
    rot = case["rot"]
    if not rot:
        return x
    t = s["table"][s["positions"].long()].to(x.dtype)
    c, d = t[:, None, :, 0], t[:, None, :, 1]
    if case["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack((a * c - b * d, b * c + a * d), -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat((a * c - b * d, b * c + a * d), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _quantise(x, kind):
    """Codes and scales: every vector of 64 by its own largest value."""
    top = x.abs().amax(-1).clamp_min(TINY)
    scaled = x * (top.reciprocal() * TOP[kind])[..., None]
    code = scaled.round().to(torch.int8) if kind == "int8" else scaled.to(torch.float8_e4m3fn)
    return code, top * (1.0 / TOP[kind])


def _gathered(s, pages, count):
    """Keys and values of `count` slots of a list of pages (or of each of many lists): [..., kv_heads, count, HD]."""
    def one(held, scale):
        x = held[pages.long()].float()
        if scale is not None:
            x = x * scale[pages.long()][..., None]
        x = x.movedim(-3, -4)
        return x.reshape(*x.shape[:-3], x.shape[-3] * x.shape[-2], HD)[..., :count, :]
    return one(s["k"], s["ks"]), one(s["v"], s["vs"])


def _run_attn(s, case):
    if own:
        out, lse = s["attend"](s["q"], s["cache"], s["prefix_pages"], case["prefix"], s["suffix_pages"],
                               s["suffix_lens"], return_lse=True)
        return {"out": out, "lse": lse}
    out, lse = _attend(s, case, torch.float32)
    return {"out": out.to(s["q"].dtype), "lse": lse}


def _attend(s, case, t):
    b, n, h, kv = case["batch"], case["queries"], case["heads"], case["kv_heads"]
    r = h // kv
    q = s["q"].to(t).reshape(b, n, kv, r, HD)
    pk, pv = (x.to(t) for x in _gathered(s, s["prefix_pages"], case["prefix"]))
    sk, sv = (x.to(t) for x in _gathered(s, s["suffix_pages"], case["suffix"]))
    shared = q.permute(2, 0, 1, 3, 4).reshape(kv, b * n * r, HD)
    sp = (torch.matmul(shared, pk.transpose(-1, -2)) / 8).reshape(kv, b, n, r, case["prefix"])
    ss = torch.matmul(q.permute(2, 0, 1, 3, 4).reshape(kv, b, n * r, HD),
                      sk.permute(1, 0, 3, 2)).reshape(kv, b, n, r, case["suffix"]) / 8
    seen = s["suffix_lens"].long()[:, None] - (n - 1 - torch.arange(n, device="cuda"))[None, :]
    hidden = torch.arange(case["suffix"], device="cuda")[None, None, :] >= seen[..., None]
    ss = ss.masked_fill(hidden[None, :, :, None, :], -math.inf)
    none = torch.full((kv, b, n, r, 1), -math.inf, dtype=t, device="cuda")
    top = torch.cat((sp, ss, none), -1).amax(-1, keepdim=True)
    ref = torch.where(top.isinf(), torch.zeros_like(top), top)
    ep, es = (sp - ref).exp(), (ss - ref).exp()
    total = ep.sum(-1, keepdim=True) + es.sum(-1, keepdim=True)
    keep = (seen[None, :, :, None, None] > 0) | (case["prefix"] > 0)
    acc = torch.matmul(ep.reshape(kv, b * n * r, -1), pv).reshape(kv, b, n, r, HD)
    acc = acc + torch.matmul(es.reshape(kv, b, n * r, -1), sv.permute(1, 0, 2, 3)).reshape(kv, b, n, r, HD)
    out = torch.where(keep, acc / total, torch.zeros_like(acc))
    lse = torch.where(keep, ref * LOG2E + total.log2(), torch.full_like(total, -math.inf))
    return (out.permute(1, 2, 0, 3, 4).reshape(b * n, h * HD),
            lse.permute(1, 2, 0, 3, 4).reshape(b * n, h).contiguous())


def _run_sample(s, case):
    if own:
        tokens, logprobs = s["decode"].sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
        return {"tokens": tokens, "logprobs": logprobs}
    x = s["logits"].float()
    depth = (x.amax(-1, keepdim=True) - x) * (s["temperature"].reciprocal() * LOG2E)[:, None]
    key = (depth.clamp_max(BOTTOM) * KEY).round()
    weight = (torch.exp2(-key * (1 / KEY)) * ONE).round().to(torch.int64)
    order = torch.sort(key, dim=-1, stable=True).indices
    w = weight.gather(-1, order)
    rank = torch.arange(case["vocab"], device="cuda")[None, :]
    k = torch.where(s["top_k"] > 0, s["top_k"], case["vocab"])[:, None]
    w = torch.where(rank < k, w, 0)
    sums = w.cumsum(-1)
    within = (sums - w).double() < s["top_p"].double()[:, None] * sums[:, -1:].double()
    kept = (rank == 0) | ((within | (s["top_p"] >= 1)[:, None]) & (w.double() >= s["min_p"].double()[:, None] * ONE))
    w = torch.where(kept, w, 0)
    total = w.sum(-1, keepdim=True)
    aim = torch.minimum((s["u"].double()[:, None] * total.double()).floor().long(), total - 1)
    w = torch.zeros_like(w).scatter(-1, order, w)
    token = (w.cumsum(-1) <= aim).sum(-1, keepdim=True)
    logprob = -key.gather(-1, token) * (1 / KEY) * math.log(2.0) - (total.double() / ONE).float().log()
    return {"tokens": token[:, 0].int(), "logprobs": logprob[:, 0]}


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "kv":
        return _exact_kv(s, case)
    if case["op"] == "attn":
        return _exact_attn(s, case)
    return _exact_sample(s, case)


def _exact_kv(s, case):
    h, kv, rot, n = case["heads"], case["kv_heads"], case["rot"], case["tokens"]
    x = s["qkv"].double().reshape(n, h + 2 * kv, HD)
    if rot:
        turn = torch.view_as_complex(s["table"][s["positions"].long()].double())[:, None, :]
        part = x[:, :h + kv, :rot]
        pairs = part.unflatten(-1, (-1, 2)) if case["interleaved"] else part.unflatten(-1, (2, -1)).transpose(-1, -2)
        turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        x[:, :h + kv, :rot] = (turned if case["interleaved"] else turned.transpose(-1, -2)).flatten(-2)
    held = x[:, h:]
    if case["kind"] == "int8":
        unit = held.abs().amax(-1, keepdim=True).clamp_min(TINY) / 127
        held = (held / unit).round() * unit
    elif case["kind"] == "e4m3":
        unit = held.abs().amax(-1, keepdim=True).clamp_min(TINY) / 448
        y = held / unit
        grid = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
        held = (y / grid).round() * grid * unit
    return {"q": x[:, :h].reshape(n, -1), "k": held[:, :kv].reshape(n, -1), "v": held[:, kv:].reshape(n, -1)}


def _exact_attn(s, case):
    """Row by row of the batch: softmax over the keys that a query sees, written out."""
    n, h, kv = case["queries"], case["heads"], case["kv_heads"]
    lens = s["suffix_lens"].tolist()

    def keys(pages, count):
        got = []
        for held, scale in ((s["k"], s["ks"]), (s["v"], s["vs"])):
            x = held[pages.long()].double()
            x = x if scale is None else x * scale[pages.long()].double().unsqueeze(-1)
            got.append(x.transpose(0, 1).reshape(kv, -1, HD)[:, :count])
        return got

    pk, pv = keys(s["prefix_pages"], case["prefix"])
    out = torch.zeros((case["batch"], n, h, HD), dtype=torch.float64, device="cuda")
    lse = torch.full((case["batch"], n, h), -math.inf, dtype=torch.float64, device="cuda")
    for b, held in enumerate(lens):
        sk, sv = keys(s["suffix_pages"][b], held)
        q = s["q"].double().reshape(case["batch"], n, kv, h // kv, HD)[b]
        scores = torch.einsum("ngrd,gkd->ngrk", q, torch.cat((pk, sk), 1)) * 0.125
        values = torch.cat((pv, sv), 1)
        for i in range(n):
            count = case["prefix"] + max(0, held - (n - 1 - i))
            if count:
                row = scores[i, :, :, :count]
                lse[b, i] = torch.logsumexp(row, -1).reshape(h) / math.log(2.0)
                out[b, i] = torch.einsum("grk,gkd->grd", torch.softmax(row, -1), values[:, :count]).reshape(h, HD)
    return {"out": out.reshape(case["batch"] * n, h * HD), "lse": lse.reshape(case["batch"] * n, h)}


def _exact_sample(s, case):
    """One row at a time: the filters as they are usually stated, on probabilities in 64 bits."""
    logits, got = s["logits"].double(), []
    for i in range(case["rows"]):
        p = torch.softmax(logits[i] / s["temperature"][i].double(), -1)
        p, order = torch.sort(p, descending=True, stable=True)
        if case["top_k"]:
            p = torch.where(torch.arange(case["vocab"], device="cuda") < case["top_k"], p, 0)
        p = p / p.sum()
        keep = p >= float(np.float32(case["min_p"])) * p[0]
        if case["top_p"] < 1:
            keep &= p.cumsum(0) - p < float(np.float32(case["top_p"]))
        p = torch.where(keep, p, 0)
        p = p / p.sum()
        placed = torch.zeros_like(p).scatter(0, order, p)
        at = torch.searchsorted(placed.cumsum(0), s["u"][i].double(), right=True).clamp_max(case["vocab"] - 1)
        got.append(placed[at].log())
    return {"tokens": None, "logprobs": torch.stack(got)}
