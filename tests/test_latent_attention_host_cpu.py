"""
The host side of the latent-attention functions without a GPU: what they ask of the library and when, seen
through a stand-in for it.
"""
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
