"""
The host side of the latent-attention functions without a GPU: what they ask of the library and when, seen
through a stand-in for it; and, in the kernels' source, that no warp can leave a loop apart.
"""
import os
import re

import pytest
import torch

from lazylora_b200 import _lib


class _Status:
    """A library whose two status words hold what the test puts there, each cleared when it is read."""

    def __init__(self, latent, dense):
        self.words = {"latent": latent, "dense": dense}

    def _read(self, name):
        code, self.words[name] = self.words[name], 0
        return code

    def ll_latent_status(self, stream):
        return self._read("latent")

    def ll_gemm_bf16_status(self, stream):
        return self._read("dense")

    def ll_last_cuda_error(self):
        return b"device status"


@pytest.mark.parametrize("latent,dense", [(0, 3), (5, 0), (5, 3)])
def test_check_status_covers_the_per_head_products(monkeypatch, latent, dense):
    """head_linear's launches record a wait that ran out in the dense products' word."""
    from lazylora_b200.core import latent_attention as A
    lib = _Status(latent, dense)
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(_lib, "stream_ptr", lambda stream=None: 0)
    with pytest.raises(_lib.LLError):
        A.check_status()
    assert lib.words == {"latent": 0, "dense": 0}, "both are read, whichever raised"
    A.check_status()


def test_paged_workspace_is_the_current_devices(monkeypatch):
    """The size goes by the device's SMs, so one device's is not handed to another."""
    from lazylora_b200.core import latent_attention as A
    sizes, given, device = {0: 1000, 1: 5000}, [], [0]

    class Lib:
        def ll_paged_latent_workspace_bytes(self, *a):
            return sizes[device[0]]

        def ll_paged_latent_attention(self, *a):
            given.append((device[0], a[-2]))
            return 0

    monkeypatch.setattr(A, "_library", Lib())
    monkeypatch.setattr(A, "_device", lambda: device[0])
    monkeypatch.setattr(A, "_stream", lambda *tensors: 0)
    A._paged_workspace.cache_clear()
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt)  # noqa: E731
    try:
        for device[0] in (0, 1, 0):
            A.paged_latent_attention(z(1, 1, 2, 192), z(2, 8, 192), z(1, 1, dt=torch.int32), z(1, dt=torch.int32), 128, 0.1)
    finally:
        A._paged_workspace.cache_clear()
    assert given == [(0, 1000), (1, 5000), (0, 1000)]


def test_epilogue_waits_have_one_outcome_a_warp():
    """A bounded wait that runs out in some lanes only would let them leave a loop in which the others wait for
    them (__syncwarp, tcgen05.ld): the dense products' epilogues, whose loops a wait can end, vote on it."""
    csrc = os.path.join(os.path.dirname(os.path.abspath(_lib.__file__)), "csrc")
    with open(os.path.join(csrc, "dense_gemm.cu")) as fh:
        waits = re.findall(r"ok = (\w+)\(&accfull\[ab\], abph", fh.read())
    assert len(waits) == 2 and set(waits) == {"warp_wait_sleep"}, waits
