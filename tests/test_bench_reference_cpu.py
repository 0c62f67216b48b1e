"""
The bench's reference arm without the compiled reference: one line that says so, at once.
"""
import json
from types import SimpleNamespace

import torch

import bench
from oracle import moe_oracle as O


def test_reference_arm_without_the_reference_is_unavailable(monkeypatch, capsys):
    """It neither makes the layer's inputs nor times another implementation in the reference's place."""
    import lazylora_b200.synthetic as S

    def never(*a, **k):
        raise AssertionError("nothing is made or timed")
    monkeypatch.setattr(O, "REF_SO", "/nonexistent/libmxfp4_ref.so")
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(S, "make_layer_device", never)
    monkeypatch.setattr(bench, "cpu_reference_sample", never)
    bench.run_reference(SimpleNamespace(steps=20, warmup=5), S.CONFIGS["c1"], 0, 1, None)
    line = json.loads(capsys.readouterr().out)
    assert line["impl"] == "reference" and "not been compiled" in line["unavailable"]
