"""
The latent-attention entry points without a GPU: argument checks of the C functions return before any CUDA
call, the Python functions refuse CPU tensors, and the operators' measured cases are well formed.
"""
import ctypes
import os
import random
import sys

import pytest
import torch

from lazylora_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_c_entry_points_check_arguments():
    lib = _lib.load()
    p, one = ctypes.c_void_p(16), ctypes.c_float(1.0)              # never dereferenced: the checks come first

    def append(kv_stride=576, T=4, d_c=512, d_r=64, dtype=1, page=8, q=p, qs=64, H=2, kv=p, rows=10):
        return lib.ll_latent_append(kv, kv_stride, p, p, p, rows, T, d_c, d_r, dtype, 0, p, 8 * 576, 576, 4, page, q,
                                    128, qs, H, p, 128, 64, None)
    assert append(T=0) == 0
    for bad in (dict(T=-1), dict(d_c=100), dict(d_r=24), dict(dtype=0), dict(page=0), dict(kv_stride=577), dict(qs=60),
                dict(kv=None), dict(rows=0), dict(H=-1)):
        assert append(**bad) == 1, bad

    def paged(row=576, page=16, B=2, Tq=1, H=4, d_c=512, d_r=64, scale=1.0, dtype=1, q=p, ws=1 << 40):
        return lib.ll_paged_latent_attention(q, 4 * 576, row, p, 16 * 576, 576, 4, page, p, 3, 3, p, B, Tq, H, d_c, d_r,
                                             ctypes.c_float(scale), dtype, p, p, p, ws, None)
    assert paged(B=0) == 0
    for bad in (dict(page=12), dict(d_c=192), dict(d_r=32), dict(scale=0.0), dict(scale=float("nan")), dict(dtype=3),
                dict(q=None), dict(row=580), dict(Tq=0), dict(H=0)):
        assert paged(**bad) == 1, bad
    assert paged(ws=0) == 4

    def packed(**kw):
        a = dict(B=2, Tq=8, Tk=8, H=2, d_n=128, d_r=64, d_v=128, causal=1, dtype=1, scale=0.1, q=16, q_stride_t=384,
                 q_stride_h=192, k_nope=16, k_stride_t=256, k_stride_h=128, k_pe=16, kpe_stride_t=64, v=16, v_stride_t=256,
                 v_stride_h=128, cu_q=16, cu_k=16)
        a.update(kw)
        return _lib.LatentPacked(**a)
    fwd = lambda a, out=p: lib.ll_latent_forward(ctypes.byref(a), out, p, None)  # noqa: E731
    assert fwd(packed(B=0)) == 0 and fwd(packed(Tq=0)) == 0
    for bad in (dict(d_n=96), dict(d_r=32), dict(d_v=256), dict(H=0), dict(scale=0.0), dict(dtype=0), dict(q=None),
                dict(q=8), dict(q_stride_t=12), dict(k_pe=None), dict(cu_q=None), dict(v_stride_h=0), dict(Tq=-1)):
        assert fwd(packed(**bad)) == 1, bad
    assert fwd(packed(), None) == 1

    def bwd(a, g=p, ws=1 << 40, dk_pe=p):
        return lib.ll_latent_backward(ctypes.byref(a), g, 256, 128, p, p, p, p, dk_pe, p, p, ws, None)
    assert bwd(packed(B=0)) == 0
    assert bwd(packed(), g=None) == 1 and bwd(packed(), dk_pe=None) == 1 and bwd(packed(d_n=32)) == 1
    assert bwd(packed(), ws=16) == 4
    assert lib.ll_latent_backward_workspace_bytes(ctypes.byref(packed())) >= 4 * (2 * 8 * 64 + 2 * 8)

    def heads(T=4, H=2, N=64, K=64, x=p, st=128, ldw=64):
        return lib.ll_gemm_bf16_heads(T, H, N, K, x, st, 64, p, 4096, ldw, 1, p, 128, 64, None)
    assert heads(T=0) == 0
    for bad in (dict(N=0), dict(K=-1), dict(x=None), dict(st=12), dict(ldw=0)):
        assert heads(**bad) == 1, bad
    assert one.value == 1.0


def test_python_functions_refuse_cpu_tensors():
    from lazylora_b200.core import latent_attention as A
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt)  # noqa: E731
    i32, i64 = (lambda *s: z(*s, dt=torch.int32)), (lambda *s: z(*s, dt=torch.int64))
    for call in (lambda: A.append_latent(z(2, 8, 192), z(1, 192), i64(1), i64(1), torch.zeros(4, 64)),
                 lambda: A.rotate_positions(z(2, 3, 64), i64(2), torch.zeros(4, 64)),
                 lambda: A.paged_latent_attention(z(1, 1, 2, 192), z(2, 8, 192), i32(1, 1), i32(1), 128, 0.1),
                 lambda: A.latent_attention_forward(z(4, 2, 192), z(4, 2, 128), z(4, 64), z(4, 2, 128), i32(2), i32(2), 0.1),
                 lambda: A.head_linear(z(2, 2, 64), z(2, 64, 64))):
        with pytest.raises(ValueError):
            call()


def test_layout_rules_of_views():
    """What is read in place and what is copied: inner stride 1, other strides positive multiples of 8."""
    from lazylora_b200.core.latent_attention import _view
    t = torch.zeros(4, 3, 72, dtype=torch.bfloat16)
    assert _view(t[..., :64])[0].data_ptr() == t.data_ptr()
    assert _view(t[..., 8:])[0].data_ptr() == t[..., 8:].data_ptr()
    assert _view(t[..., 4:68], copy=False) is None                  # starts 8 bytes into a row
    assert _view(t[0].t(), copy=False) is None                      # inner stride not 1
    broadcast = torch.zeros(1, 3, 64, dtype=torch.bfloat16).expand(4, 3, 64)
    copied, strides = _view(broadcast)
    assert copied.data_ptr() != broadcast.data_ptr() and tuple(strides) == (192, 64, 1)
    one = torch.zeros(1, 64, dtype=torch.bfloat16).as_strided((1, 64), (5, 1))
    assert _view(one)[1][0] % 8 == 0                                # the stride of a single row does not matter


def test_measured_cases():
    sys.path.insert(0, ROOT)
    import perf.operators as P
    names = [c["name"] for c in P.listed()]
    assert len(set(names)) == len(names) == 12
    flops = [P.work(c)["flops"] for c in P.listed()]
    assert max(flops) >= 16 * min(flops)
    rng = random.Random(0)
    most = {k: max(P.work(c)[k] for c in P.listed()) for k in ("bytes", "flops")}
    for _ in range(50):
        w = P.work(P.draw(rng))
        assert 0 < w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"]
