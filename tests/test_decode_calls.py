"""What the decoding calls refuse or pass on before any GPU work, with tensors that stand in for another GPU's: no
launch is made."""
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
