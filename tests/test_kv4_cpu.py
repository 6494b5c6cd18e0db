"""CPU checks of the 4-bit cache and the log probabilities: refusals that need no device, and the reference form itself."""
import contextlib
import ctypes
import math
import types

import pytest
import torch

import daiza_amd as dz
import kv4_ref as ref


def test_refusals_without_a_device():
    L = dz.lib()
    h = ctypes.c_void_p()
    assert L.dz_kv4_create(0, 64, 8, ctypes.byref(h)) == dz.DZ_ERR_TENSOR
    assert L.dz_kv4_create(4, 96, 8, ctypes.byref(h)) == dz.DZ_ERR_UNSUPPORTED
    assert L.dz_kv4_create(4, 64, 0, ctypes.byref(h)) == dz.DZ_ERR_TENSOR
    assert L.dz_kv4_create(4, 64, 8, None) == dz.DZ_ERR_MODEL
    assert not h.value
    assert L.dz_kv4_len(None) == -1
    assert L.dz_kv4_free(None) == dz.DZ_OK
    assert L.dz_kv4_truncate(None, 0) == dz.DZ_ERR_MODEL
    assert L.dz_kv4_append_dev(None, None, 0, None, 0, 0, 1, None) == dz.DZ_ERR_MODEL
    assert L.dz_kv4_read_dev(None, 0, 1, None, None, None) == dz.DZ_ERR_MODEL
    assert L.dz_kv4_attend_dev(None, None, 0, 0, 1, 1, 1.0, None, 0, None, 0, None, None) == dz.DZ_ERR_MODEL
    assert L.dz_kv4_evict_dev(None, None, 0, 0, 0, None, None, 0, None, None) == dz.DZ_ERR_MODEL
    assert L.dz_kv4_attend_work_bytes(None, 4, 1) == 0


def test_logprobs_refusals_without_a_device():
    L = dz.lib()

    def call(type=0, n=1, vocab=10, ld=10, top=0):
        return L.dz_logprobs_dev(None, ld, type, n, vocab, None, top, None, None, None, None, None, None)

    assert call(type=7) == dz.DZ_ERR_UNSUPPORTED
    assert call(n=-1) == dz.DZ_ERR_TENSOR
    assert call(vocab=0) == dz.DZ_ERR_TENSOR
    assert call(ld=9) == dz.DZ_ERR_TENSOR
    assert call(top=11) == dz.DZ_ERR_UNSUPPORTED
    assert call(top=65, vocab=100, ld=100) == dz.DZ_ERR_UNSUPPORTED
    assert call(n=0) == dz.DZ_OK
    assert call() == dz.DZ_ERR_MODEL
    assert L.dz_logprobs_work_bytes(0, 10, 0) == 0 and L.dz_logprobs_work_bytes(1, 10, 65) == 0


def test_host_tensors_are_refused():
    with pytest.raises(dz.DaizaError):
        dz.logprobs_dev(torch.zeros(1, 4))


def test_reference_of_stored_values():
    """The reference against the format's definition by hand."""
    x = torch.zeros(1, 1, 64)
    x[0, 0, :8] = torch.tensor([6.0, 0.25, 0.75, -1.25, 1.75, 2.5, 3.5, -5.0])
    x[0, 0, 32:36] = torch.tensor([7.0, 0.5, 1.5, -3.0])  # 7 does not fit under 6: the next power of two
    got = ref.stored(x)[0, 0]
    assert got[:8].tolist() == [6, 0, 1, -1, 2, 2, 4, -4]
    assert got[32:36].tolist() == [8, 0, 2, -3]
    assert torch.equal(ref.stored(got.reshape(1, 1, 64))[0, 0], got)
    x[0, 0, 3] = math.inf
    got = ref.stored(x)[0, 0]
    assert bool(torch.isnan(got[:32]).all()) and bool(torch.isfinite(got[32:]).all())


class _Torch:
    """What _work uses of torch, keeping account of the stream that each block is allocated on."""
    uint8 = "uint8"

    def __init__(self, current):
        self.current, self.blocks, self.cuda = current, [], self

    def empty(self, n, dtype, device):
        self.blocks.append((n, self.current))
        return self

    def record_stream(self, stream):  # says when a block is free again, nothing of when it was
        pass

    class ExternalStream(int):
        def __new__(cls, handle, device=None):
            assert handle, "torch takes 0 for a stream of its pool"
            return int.__new__(cls, handle)

    def default_stream(self, device):
        return 0

    @contextlib.contextmanager
    def stream(self, s):
        before, self.current = self.current, int(s)
        yield
        self.current = before


@pytest.mark.parametrize("current", [0, 0x1000])
@pytest.mark.parametrize("stream", [0, 0x1000, 0x2000])
def test_work_memory_is_allocated_on_the_calls_stream(monkeypatch, current, stream):
    """A block of the current stream's may still be in use there when the call runs on its own stream."""
    fake = _Torch(current)
    monkeypatch.setattr(dz, "_torch", fake)
    monkeypatch.setattr(dz, "_current_stream", lambda t: fake.current)
    dz._work(types.SimpleNamespace(device="cuda:0"), 100, stream)
    assert fake.blocks == [(100, stream)] and fake.current == current
