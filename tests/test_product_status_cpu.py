"""kernels.product_status and product_reset around the C calls, without a GPU."""

import contextlib
import types

import pytest
import torch

from fused_decode_b200 import _capi, kernels


class FakeLib:
    """The word behind fd_product_status / fd_product_reset; ``code`` is what both return."""

    def __init__(self):
        self.word, self.code, self.streams = 0, 0, []

    def fd_product_status(self, out, stream):
        self.streams.append(stream)
        out.value = self.word
        return self.code

    def fd_product_reset(self, stream):
        self.streams.append(stream)
        self.word = 0
        return self.code

    def fd_status_string(self, code):
        return b"device query failed"


@pytest.fixture
def lib(monkeypatch):
    fake = FakeLib()
    monkeypatch.setattr(_capi, "load", lambda: fake)
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: types.SimpleNamespace(cuda_stream=7))
    return fake


def test_an_expired_wait_shows_until_it_is_reset(lib):
    assert kernels.product_status() == 0
    lib.word = 1  # a bounded wait expired
    assert kernels.product_status() == 1 and kernels.product_status() == 1
    kernels.product_reset()
    assert kernels.product_status() == 0
    assert set(lib.streams) == {7}


def test_errors_are_raised(lib):
    lib.code = 5
    with pytest.raises(RuntimeError):
        kernels.product_status()
    with pytest.raises(RuntimeError):
        kernels.product_reset()


@pytest.mark.gpu
def test_reset_on_the_device():
    from fused_decode_b200 import linear_act

    kernels.product_reset()
    x = torch.ones(2, 64, device="cuda", dtype=torch.bfloat16)
    assert (linear_act(x, x) == 64).all()
    assert kernels.product_status() == 0
