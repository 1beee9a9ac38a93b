"""What the decoding calls refuse or pass on before any GPU work, with tensors that stand in for another GPU's: no
launch is made."""
import math
from pathlib import Path

import pytest
import torch

from autoane_b200 import decode


class Elsewhere(torch.Tensor):
    """A CPU tensor that gives itself out as one of cuda:1."""
    is_cuda = property(lambda self: True)

    def get_device(self):
        return 1


def on_1(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(Elsewhere)


@pytest.fixture
def calls(monkeypatch):
    """The library's calls, recorded and not made; the current device is cuda:0."""
    made = []

    def fn(name):
        def call(*a):
            made.append((name, a))
            return 1 << 10 if name.endswith("workspace") else 0
        return call

    monkeypatch.setattr(decode, "_fn", fn)
    monkeypatch.setattr(decode, "_stream", lambda dev: 0)
    monkeypatch.setattr(decode, "_current", lambda: 0)
    return made


def cache_1():
    return decode.KVCache(on_1(2, 1, 8, 64), on_1(2, 1, 8, 64))


def vec(n, dtype=torch.int32):
    return on_1(n, dtype=dtype)


@pytest.mark.parametrize("what", ["append", "read", "attend", "sample"])
def test_tensors_of_another_device_are_refused(calls, monkeypatch, what):
    """The library launches on the current device: tensors of another one must not get there."""
    cache = cache_1()
    monkeypatch.setattr(decode, "_current", lambda: 1)
    att = decode.PrefixAttention(1, 1, 1, 1, 8, 0, device="cpu")
    att.workspace = att.workspace.as_subclass(Elsewhere)
    call = {
        "append": lambda: cache.append(on_1(2, 192), 1, vec(2)),
        "read": lambda: cache.read(vec(2), torch.float16, on_1(2, 64), on_1(2, 64)),
        "attend": lambda: att(on_1(1, 64), cache, vec(1), 8, None, None),
        "sample": lambda: decode.sample(on_1(2, 10), vec(2, torch.float32)),
    }[what]
    calls.clear()
    call()
    assert len(calls) == 1  # with cuda:1 current it is made
    monkeypatch.setattr(decode, "_current", lambda: 0)
    with pytest.raises(ValueError, match="cuda:1"):
        call()
    assert len(calls) == 1


def test_workspace_of_another_device_is_refused(calls, monkeypatch):
    """A PrefixAttention made on one device does not work on a cache of another."""
    monkeypatch.setattr(decode, "_current", lambda: 1)
    att = decode.PrefixAttention(1, 1, 1, 1, 8, 0, device="cpu")
    calls.clear()
    with pytest.raises(ValueError, match="workspace"):
        att(on_1(1, 64), cache_1(), vec(1), 8, None, None)
    assert not calls


def test_tensors_that_require_a_gradient_are_refused(calls, monkeypatch):
    """The operators have no backward pass: under autograd their inputs may not require one."""
    monkeypatch.setattr(decode, "_current", lambda: 1)
    logits, u = on_1(2, 10, dtype=torch.float32).requires_grad_(), vec(2, torch.float32)
    with pytest.raises(ValueError, match="gradient"):
        decode.sample(logits, u)
    with pytest.raises(ValueError, match="gradient"):
        cache_1().append(on_1(2, 192).requires_grad_(), 1, vec(2))
    assert not calls
    with torch.no_grad():
        decode.sample(logits, u)
    decode.sample(logits.detach(), u)
    assert len(calls) == 2


def test_large_pitches():
    """A pitch beyond the library's 32 bits is refused, not cut off."""
    far = torch.empty_strided((2, 64), (1 << 31, 1), dtype=torch.float16, device="meta")
    with pytest.raises(ValueError, match="pitch"):
        decode._ld(far)
    assert decode._ld(torch.empty_strided((2, 64), ((1 << 31) - 8, 1), device="meta")) == (1 << 31) - 8


def test_pitch_of_one_row():
    """The pitch of a matrix of one row is of no account; any other's is passed on."""
    one = torch.empty(1, 1603, device="meta")
    assert decode._ld(one[:, :1600]) == 1600
    assert decode._ld(one) >= 1603 and decode._ld(one) % 8 == 0
    assert decode._ld(torch.empty(3, 1603, device="meta")[:, :1600]) == 1603


@pytest.mark.parametrize("rot,theta,trained,fast,slow", [
    (64, 10000.0, 2048, 32.0, 1.0), (64, 10000.0, 1 << 17, 32.0, 1.0), (16, 10000.0, 32768, 32.0, 1.0),
    (32, 500.0, 8192, 32.0, 2.0), (64, 10000.0, 4, 32.0, 1.0), (16, 100000.0, 1 << 20, 2.0, 1.0)])
def test_yarn_keeps_and_divides_by_turns(rot, theta, trained, fast, slow):
    """A pair that makes more than `fast` turns over the trained positions keeps its angle, one that makes fewer than
    `slow` is divided by the scale, and those between go from the one to the other without a step back."""
    scale = 8.0
    size = 0.1 * math.log(scale) + 1
    t = decode.rope_table(2, rot, theta, scale, (trained, fast, slow), device="cpu").double()[1] / size
    freq = theta ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot)
    turns = trained * freq / (2 * math.pi)
    part = torch.atan2(t[:, 1], t[:, 0]) / freq  # of the plain angle
    tol = 1e-6 / freq
    assert ((part - 1).abs() <= tol)[turns > fast].all()
    assert ((part - 1 / scale).abs() <= tol)[turns < slow].all()
    # the whole ramp: from 0 at the last pair above `fast` to 1 at the first one below `slow`
    at = lambda n: rot * math.log(trained / (n * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
    lo, hi = max(math.floor(at(fast)), 0), math.ceil(at(slow))
    for i in range(rot // 2):
        if slow <= turns[i] <= fast and hi > lo:
            blend = min(max((i - lo) / (hi - lo), 0.0), 1.0)
            assert abs(part[i] - (1 - blend + blend / scale)) <= tol[i], (i, part[i])


def test_kernels_read_their_inputs_by_ordinary_loads():
    """These kernels start while the one before them still runs (programmatic launch), and wait for it before they read
    what it writes. The read-only path (ld.global.nc) is for data that nothing writes while a kernel runs: its loads
    may come from before the wait."""
    csrc = Path(decode.__file__).parent / "csrc"
    names = ["decode.cuh", "kv_cache.cu", "attn_prefix.cuh", "attn_prefix.cu", "attn_prefix_tc.cu", "sample.cu"]
    for name in names:
        text = (csrc / name).read_text()
        assert not any(w in text for w in ("__ldg", "__restrict__", "global.nc")), name
