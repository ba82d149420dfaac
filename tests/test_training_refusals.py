"""Host-side refusals of the adapter and router-training entry points. CPU only."""

from __future__ import annotations

from deepseek_v41_mlx_b200 import _lib as L


def _fwd(T=4, K=64, n=2, R=8, N=32, x=16, out=L.F32, ws=None, ws_bytes=0):
    return L.load().dsv41_lora_forward(x, T, K, x, x, n, R, N, None, x, None, out, x, None, ws,
                                       ws_bytes, None)


def test_lora_forward_refuses_before_any_device_work():
    assert _fwd(K=60) == L.BAD_SHAPE and "multiple of 8" in L.last_error()
    assert _fwd(T=-1) == L.BAD_SHAPE and _fwd(N=0) == L.BAD_SHAPE and _fwd(n=0) == L.BAD_SHAPE
    assert _fwd(n=8193) == L.BAD_SHAPE and _fwd(T=(1 << 30) + 1) == L.BAD_SHAPE
    assert _fwd(R=12) == L.UNSUPPORTED and _fwd(R=136) == L.UNSUPPORTED
    assert _fwd(out=L.F16) == L.BAD_DTYPE
    assert _fwd(x=None) == L.BAD_ARG and _fwd(x=24) == L.MISALIGNED
    assert _fwd(T=5000) == L.WORKSPACE
    assert _fwd(T=0) == L.OK


def _bwd(T=4, K=64, n=2, R=8, N=32, p=16, dt=L.F32, gdt=L.F32):
    return L.load().dsv41_lora_backward(p, p, p, p, p, T, K, N, n, R, None, p, None, dt, p, gdt,
                                        p, p, None, 0, None)


def test_lora_backward_refuses_before_any_device_work():
    assert _bwd(K=4) == L.BAD_SHAPE and _bwd(R=7) == L.UNSUPPORTED
    assert _bwd(dt=L.U8) == L.BAD_DTYPE and _bwd(gdt=L.F16) == L.BAD_DTYPE
    assert _bwd(p=None) == L.BAD_ARG and _bwd(p=8) == L.MISALIGNED and _bwd() == L.WORKSPACE


def _bal(T=4, E=8, k=2, S=1, p=16, dt=L.F32, off=None, score=0, temp=1.0, gl=None, dz=None):
    return L.load().dsv41_moe_balance(p, dt, T, E, p, k, off, S, None, score, temp, gl, None, 1,
                                      1.0, p, p, dz, None, 0, None)


def test_balance_refuses_before_any_device_work():
    assert _bal(dt=L.F16) == L.BAD_DTYPE
    assert _bal(E=1025) == L.BAD_SHAPE and _bal(E=0) == L.BAD_SHAPE and _bal(T=-1) == L.BAD_SHAPE
    assert _bal(k=9) == L.BAD_ARG and _bal(k=0) == L.BAD_ARG and _bal(score=3) == L.BAD_ARG
    assert _bal(temp=0.0) == L.BAD_ARG and _bal(S=2) == L.BAD_ARG and _bal(gl=16) == L.BAD_ARG
    assert _bal(p=None) == L.BAD_ARG and _bal(T=5000) == L.WORKSPACE


def test_workspaces_stay_proportionate():
    lib = L.load()
    for T in (1, 64, 777, 8192):
        for n in (1, 64, 1024):
            # three bf16 values a token and rank (an adapter's tokens padded to 64); for the
            # gradients twice that and at most two partial sums a CTA
            f = lib.dsv41_lora_workspace_size(T, 7168, 4096, n, 64, 0)
            g = lib.dsv41_lora_workspace_size(T, 7168, 4096, n, 64, 1)
            pad = min(n, T) * 64 * 64 * 6
            assert f <= T * (64 * 6 + 64) + pad + n * 64 + (1 << 20)
            assert g <= 2 * (f + T * 64 * 6 + pad + (1 << 20)) + 2 * 2 * 148 * 64 * 128 * 4 + n * 64
    assert lib.dsv41_moe_balance_workspace_size(65536, 384, 16) <= 65536 * 8 + 4096


def test_cpu_tensors_are_refused():
    import pytest
    import torch

    import deepseek_v41_mlx_b200 as q
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    a, b = torch.zeros(2, 8, 64, dtype=torch.bfloat16), torch.zeros(2, 32, 8, dtype=torch.bfloat16)
    ids = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(q.DSV41Error):
        q.lora.lora_forward(x, a, b, ids)
    with pytest.raises(q.DSV41Error):
        q.moe.balance_loss(torch.zeros(4, 8), ids.view(4, 1))


def test_missing_ids_are_refused():
    import pytest
    import torch

    import deepseek_v41_mlx_b200 as q
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    a, b = torch.zeros(2, 8, 64, dtype=torch.bfloat16), torch.zeros(2, 32, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="ids"):
        q.lora.lora_forward(x, a, b, None)
    with pytest.raises(ValueError, match="ids"):
        q.lora.LoRA(a, b).backward(x, x, x, None)
