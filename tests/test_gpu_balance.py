"""The router's training pass: balance loss, counts, gradients, refusals.

Counts must be equal; the loss and the gradients are compared with float64.  The loss sums p (a
ratio of fp32 scores, each off by a few steps of 2^-24) with equal signs, so its relative error
is that of one term: 32 steps of 2^-24 allowed (the score's exponential contributes up to about
|z| / 8 steps, |z| < 40 here, the square root, the normalising sum and the division the rest).
A gradient is a difference, c_e - sum_j c_j p_j and dw_j - sum_l dw_l w_l: its terms are known to
a few steps of their own size, so it is compared against the sum of its terms' magnitudes (where c
is close to the mean, or one choice carries all the weight, the difference is far smaller).
"""

from __future__ import annotations

import types

import pytest
import torch

import deepseek_v41_mlx_b200 as q

pytestmark = pytest.mark.gpu

BF, F32, D = torch.bfloat16, torch.float32, torch.float64


def _eq(a, b):
    return bool(torch.equal(a, b))
FUNCS = ["sqrtsoftplus", "sigmoid", "softmax"]


def _score(z, func):
    if func == "softmax":
        return torch.softmax(z, -1)
    if func == "sigmoid":
        # s = e^(log s): its derivative s (1 - s) keeps 1 - s, which float64 sigmoid(z) rounds away
        # from z = 20 on (2^-53 against e^-z)
        return torch.nn.functional.logsigmoid(z).exp()
    return torch.logaddexp(z, torch.zeros_like(z)).sqrt()


def _ref(z, idx, offsets, mask, func, temp, gl, dw, norm, scale):
    """loss, counts, dlogits (autograd) and the magnitudes of the terms of dlogits, float64."""
    z = z.to(D).detach().requires_grad_(True)
    T, E = z.shape
    k = idx.shape[1]
    live = torch.ones(T, dtype=torch.bool, device="cuda") if mask is None else mask.bool()
    off = [0, T] if offsets is None else offsets.tolist()
    s = _score(z / temp, func)
    losses, counts, aim = [], [], 0.0
    mag = torch.zeros_like(z)
    for a, b in zip(off[:-1], off[1:]):
        rows = torch.arange(a, b, device="cuda")
        rows = rows[live[rows]]
        i = idx[rows].long()
        ok = (i >= 0) & (i < E)
        c = torch.bincount(i[ok], minlength=E)
        counts.append(c)
        m = max(rows.numel(), 1)
        p = s[rows] / (s[rows].sum(1, keepdim=True) + 1e-20)
        losses.append((c.to(D) * p).sum() * E / (k * m * m))
        if gl is not None:
            aim = aim + losses[-1] * gl[len(losses) - 1].to(D)
            up = gl[len(losses) - 1].to(D).abs() * E / (k * m * m)
            mag[rows] += up * (c + (c * p).sum(1, keepdim=True)) / s[rows].sum(1, keepdim=True)
        if dw is not None:
            w = torch.where(ok, torch.gather(s[rows], 1, i.clamp(0, E - 1)), 0.0)
            d = dw[rows].to(D).abs() * ok
            if norm and k > 1:
                d = (d + (d * w).sum(1, keepdim=True) / (w.sum(1, keepdim=True) + 1e-20)) \
                    / (w.sum(1, keepdim=True) + 1e-20)
                w = w / (w.sum(1, keepdim=True) + 1e-20)
            aim = aim + (scale * w * dw[rows].to(D) * ok).sum()
            mag[rows] = mag[rows].scatter_add(1, i.clamp(0, E - 1), scale * d * ok)
    loss = torch.stack(losses).detach() if losses else torch.zeros(0, dtype=D, device="cuda")
    cnt = torch.stack(counts).int() if counts else torch.zeros(0, E, dtype=torch.int32,
                                                               device="cuda")
    if not torch.is_tensor(aim):
        return loss, cnt, torch.zeros_like(z), torch.zeros_like(z)
    mag = mag.detach()
    if func == "softmax":
        sd = s.detach()
        mag = sd * (mag + (mag * sd).sum(1, keepdim=True)) / temp
    else:
        mag = mag * torch.autograd.grad(s.sum(), z, retain_graph=True)[0]
    return loss, cnt, torch.autograd.grad(aim, z)[0], mag


def _inputs(seed, T, E, k, dtype=F32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = (torch.randn(T, E, generator=g, device="cuda") * 1.5).to(dtype)
    idx = torch.topk(z.float(), k, dim=1).indices.int() if T else \
        torch.empty(0, k, dtype=torch.int32, device="cuda")
    dw = torch.randn(T, k, generator=g, device="cuda")
    return g, z, idx, dw


def _check(z, idx, offsets=None, mask=None, func="sqrtsoftplus", temp=1.0, gl=None, dw=None,
           norm=True, scale=1.5):
    loss, cnt, dz = q.moe.balance_loss(z, idx, offsets, mask, func, temp, gl, dw, norm, scale)
    wl, wc, wd, mag = _ref(z, idx, offsets, mask, func, temp, gl, dw, norm, scale)
    assert _eq(cnt, wc) and cnt.dtype == torch.int32
    assert ((loss.to(D) - wl).abs() <= 32 * 2.0 ** -24 * wl.abs()).all()
    if gl is None and dw is None:
        assert dz is None
        return loss, cnt, dz
    # 32 steps of the terms (as for the loss), and the type's own rounding
    tol = 32 * 2.0 ** -24 * mag + torch.finfo(z.dtype).eps / 2 * 1.01 * wd.abs()
    assert dz.dtype == z.dtype and ((dz.to(D) - wd).abs() <= tol + 1e-30).all()
    again = q.moe.balance_loss(z, idx, offsets, mask, func, temp, gl, dw, norm, scale)
    assert _eq(loss, again[0]) and _eq(dz, again[2])
    return loss, cnt, dz


@pytest.mark.parametrize("func", FUNCS)
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("T,E,k", [(1, 8, 1), (1, 384, 6), (5, 33, 3), (64, 384, 6), (130, 60, 8),
                                   (257, 1024, 32), (700, 256, 8), (3001, 96, 2), (2500, 129, 64)])
def test_one_sequence(cuda, T, E, k, dtype, func):
    g, z, idx, dw = _inputs(T + E + k, T, E, k, dtype)
    gl = torch.rand(1, generator=g, device="cuda") + 0.5
    _check(z, idx, func=func)
    _check(z, idx, func=func, gl=gl)
    _check(z, idx, func=func, dw=dw, temp=1.7)
    _check(z, idx, func=func, gl=gl, dw=dw, norm=False)
    _check(z, idx, func=func, gl=gl * 1e3, dw=dw, scale=2.5, temp=0.6)


@pytest.mark.parametrize("T,S", [(40, 3), (900, 60), (900, 900), (5000, 7), (20000, 2)])
def test_ragged_sequences(cuda, T, S):
    """Sequences of many lengths (one token and none among them), tokens before the first and
    behind the last, and padding."""
    E, k = 96, 4
    g, z, idx, dw = _inputs(T + S, T, E, k)
    cuts = torch.randint(2, T - 1, (S + 1,), generator=g, device="cuda").sort().values
    cuts[S // 2] = cuts[S // 2 - 1] if S > 2 else cuts[S // 2]
    offsets = cuts.int()
    mask = torch.rand(T, generator=g, device="cuda") > 0.3
    gl = torch.randn(S, generator=g, device="cuda")
    for m in (None, mask, torch.zeros_like(mask)):
        loss, cnt, dz = _check(z, idx, offsets, m, gl=gl, dw=dw)
    assert (loss == 0).all() and (cnt == 0).all() and (dz == 0).all()
    loss, cnt, dz = _check(z, idx, offsets, mask.to(torch.uint8), gl=gl)
    out = torch.ones(T, dtype=torch.bool, device="cuda")
    out[int(offsets[0]):int(offsets[-1])] = False
    assert (dz[out | ~mask] == 0).all()


@pytest.mark.parametrize("T", [20, 4000])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_unaligned_rows(cuda, T, dtype):
    g, z, idx, dw = _inputs(8, T, 96, 5, dtype)
    flat = torch.empty(T * 96 + 1, dtype=dtype, device="cuda")
    flat[1:] = z.reshape(-1)
    _check(flat[1:].view(T, 96), idx, gl=torch.ones(1, device="cuda"), dw=dw)


@pytest.mark.parametrize("k", [1, 3, 32, 33, 64])
@pytest.mark.parametrize("func", FUNCS)
def test_choices_repeated_and_missing(cuda, k, func):
    """Any number of choices a token, with the same expert more than twice and with none."""
    T, E = 300, 70
    g, z, _, dw = _inputs(k, T, E, k)
    idx = torch.randint(-2, 9, (T, k), generator=g, device="cuda").int()
    idx[7] = -1
    gl = torch.ones(1, device="cuda")
    for norm in (True, False):
        _check(z, idx, func=func, gl=gl, dw=dw, norm=norm)
    mask = torch.rand(T, generator=g, device="cuda") > 0.4
    _check(z, idx, mask=mask, func=func, dw=dw)


def test_more_than_2_31_values(cuda):
    """Offsets into the logits past 32 bits: the last rows' gradients against the formula."""
    T, E, k = 2_150_000, 1000, 4
    g = torch.Generator(device="cuda").manual_seed(2)
    z = torch.randn(1000, E, generator=g, device="cuda").repeat(T // 1000, 1)
    idx = torch.randint(0, E, (T, k), generator=g, device="cuda").int()
    loss, cnt, dz = q.moe.balance_loss(z, idx, grad_loss=1e6)
    assert _eq(cnt[0], torch.bincount(idx.reshape(-1).long(), minlength=E).int())
    zl = z[-50:].to(D).requires_grad_(True)
    s = _score(zl, "sqrtsoftplus")
    p = s / (s.sum(1, keepdim=True) + 1e-20)
    coef = 1e6 * E / (k * T * T)
    want = torch.autograd.grad((p * cnt[0].to(D)).sum() * coef, zl)[0]
    ds = torch.autograd.grad(_score(zl, "sqrtsoftplus").sum(), zl)[0]
    # terms c and sum c p, each about T k / E times coef ds / sum s
    mag = 2 * cnt[0].to(D).max() * coef * ds / s.sum(1, keepdim=True)
    assert ((dz[-50:].to(D) - want).abs() <= 32 * 2.0 ** -24 * mag.detach()).all()


@pytest.mark.parametrize("T", [60, 3000])
@pytest.mark.parametrize("func", FUNCS)
def test_padding_may_hold_anything(cuda, T, func):
    g, z, idx, dw = _inputs(T, T, 64, 4)
    mask = torch.rand(T, generator=g, device="cuda") > 0.5
    offsets = torch.tensor([0, T // 3, T - 5], dtype=torch.int32, device="cuda")
    gl = torch.ones(2, device="cuda")
    want = _check(z, idx, offsets, mask, func, gl=gl, dw=dw)
    idle = ~mask
    idle[T - 5:] = True
    z2, idx2, dw2 = z.clone(), idx.clone(), dw.clone()
    z2[idle], dw2[idle] = float("nan"), float("inf")
    idx2[idle] = -1
    z2[T - 1] = float("-inf")
    got = q.moe.balance_loss(z2, idx2, offsets, mask, func, 1.0, gl, dw2, True, 1.5)
    assert all(_eq(u, v) for u, v in zip(got, want))
    assert (got[2][idle] == 0).all()


@pytest.mark.parametrize("func", FUNCS)
def test_extreme_logits(cuda, func):
    """Far logits keep the scores' relative precision; a row of the type's lowest value or of
    -inf has zero scores, adds nothing and gets no loss gradient."""
    T, E, k = 200, 64, 4
    g, z, idx, dw = _inputs(3, T, E, k)
    z = z * 20
    gl = torch.ones(1, device="cuda")
    _check(z, torch.topk(z, k, 1).indices.int(), func=func, gl=gl)
    if func != "softmax":
        z[5], z[77] = float("-inf"), torch.finfo(F32).min
        loss, cnt, dz = q.moe.balance_loss(z, idx, None, None, func, 1.0, gl)
        assert torch.isfinite(loss).all() and torch.isfinite(dz).all()
        assert (dz[5] == 0).all() and (dz[77] == 0).all()
    else:
        z[5] = float("-inf")
        z[6, 1:] = float("-inf")
        loss, cnt, dz = q.moe.balance_loss(z, idx, None, None, func, 1.0, gl)
        assert torch.isfinite(loss).all() and torch.isfinite(dz).all()
        assert (dz[5] == 0).all()
    z[9, 3] = float("nan")                                   # a live NaN is seen, in its row
    loss, cnt, dz = q.moe.balance_loss(z, idx, None, None, func, 1.0, gl)
    rows = torch.isnan(dz).any(1)
    assert torch.isnan(loss).all() and rows[9] and int(rows.sum()) == 1


@pytest.mark.parametrize("T", [60, 3000])
@pytest.mark.parametrize("E, k", [(64, 4), (33, 4), (64, 40)])
@pytest.mark.parametrize("func", FUNCS)
def test_a_row_of_nan_is_seen(cuda, func, E, k, T):
    """A live token whose logits are all NaN, or NaN and -inf, makes its sequence's loss and its own
    gradient NaN; the other sequences and rows keep their bits."""
    g, z, idx, dw = _inputs(T + E, T, E, k)
    offsets = torch.tensor([0, T // 2, T], dtype=torch.int32, device="cuda")
    gl = torch.ones(2, device="cuda")
    z2 = z.clone()
    z2[9] = float("nan")
    z2[11] = float("-inf")
    z2[11, E - 1] = float("nan")
    rest = torch.ones(T, dtype=torch.bool, device="cuda")
    rest[9] = rest[11] = False
    for kw in (dict(), dict(grad_loss=gl), dict(dweights=dw), dict(grad_loss=gl, dweights=dw)):
        want = q.moe.balance_loss(z, idx, offsets, score_func=func, **kw)
        loss, cnt, dz = q.moe.balance_loss(z2, idx, offsets, score_func=func, **kw)
        assert torch.isnan(loss[0]) and loss[1] == want[0][1] and _eq(cnt, want[1])
        if kw:
            assert torch.isnan(dz[9]).all() and torch.isnan(dz[11]).any()
            assert _eq(dz[rest], want[2][rest])


def test_same_expert_twice_and_missing_choices(cuda):
    T, E, k = 500, 40, 5
    g, z, _, dw = _inputs(4, T, E, k)
    idx = torch.randint(-1, 4, (T, k), generator=g, device="cuda").int()
    _check(z, idx, gl=torch.ones(1, device="cuda"), dw=dw)
    bad = idx.clone()
    bad[idx < 0] = E + 3
    a = q.moe.balance_loss(z, idx, grad_loss=1.0, dweights=dw)
    b = q.moe.balance_loss(z, bad, grad_loss=1.0, dweights=dw)
    assert all(_eq(u, v) for u, v in zip(a, b))
    import ctypes as C
    from deepseek_v41_mlx_b200 import _lib as L
    flags = C.c_uint32(0)
    L.call("dsv41_device_status", torch.cuda.current_stream().cuda_stream, C.byref(flags))
    assert flags.value & 2


def test_gradient_by_differences(cuda):
    """(loss(z + h d) - loss(z - h d)) / 2h against dlogits, counts held by the given indices.
    h = 2^-4: the third-order term of the quotient is below 1e-3 of the first for unit d, and
    fp32 losses of about 1 leave 2^-24 / h of error."""
    T, E, k = 64, 48, 4
    g, z, idx, _ = _inputs(6, T, E, k)
    for func in FUNCS:
        dz = q.moe.balance_loss(z, idx, score_func=func, grad_loss=1.0)[2].to(D)
        d = dz / dz.norm()                                   # along the gradient
        step = 2.0 ** -4 * 8
        lo, hi = ((z.to(D) + sgn * step * d).float() for sgn in (-1, 1))
        lo, hi = (_ref(v, idx, None, None, func, 1.0, None, None, True, 1.0)[0] for v in (lo, hi))
        quot = (hi - lo) / (2 * step)
        assert abs(quot - (dz * d).sum()) <= 0.02 * abs(quot)


def _gate(E=64, D_=256, k=4, func="sqrtsoftplus"):
    args = types.SimpleNamespace(n_activated_experts=k, score_func=func, gate_temp=1.3,
                                 norm_topk_prob=True, route_scale=1.5, n_routed_experts=E, dim=D_)
    gate = q.moe.Gate(args)
    gen = torch.Generator(device="cuda").manual_seed(1)
    gate.weight = (torch.randn(E, D_, generator=gen, device="cuda") * D_ ** -0.5).to(BF)
    gate.bias = torch.randn(E, generator=gen, device="cuda") * 0.01
    return gate, gen


@pytest.mark.parametrize("func", FUNCS)
@pytest.mark.parametrize("T", [1, 37, 900])
def test_router_training_step(cuda, T, func):
    """Gate -> logits -> loss, counts and gradients, as a training step runs them: the weights
    that the gradient belongs to are the gate's own."""
    gate, gen = _gate(func=func)
    x = torch.randn(T, 256, generator=gen, device="cuda").to(BF)
    w, idx = gate(x)
    z = gate.logits(x)
    z64 = x.to(D) @ gate.weight.to(D).T
    mag = x.to(D).abs() @ gate.weight.to(D).abs().T
    assert z.dtype == F32 and ((z.to(D) - z64).abs() <= 4 * 256 ** 0.5 * 2.0 ** -23 * mag).all()
    s = torch.gather(_score(z.to(D) / 1.3, func), 1, idx.long())
    assert torch.allclose(w.to(D), 1.5 * s / (s.sum(1, keepdim=True) + 1e-20), rtol=1e-5)
    dw = torch.randn(T, 4, generator=gen, device="cuda")
    loss, counts, dz = gate.balance_loss(z, idx, grad_loss=0.01, dweights=dw)
    want = _ref(z, idx, None, None, func, 1.3, torch.full((1,), 0.01, device="cuda"), dw, True,
                1.5)
    assert _eq(counts, want[1]) and int(counts.sum()) == T * 4
    assert ((dz.to(D) - want[2]).abs() <= 32 * 2.0 ** -24 * want[3]).all()
    same = gate.balance_loss(z.view(1, T, 64), idx.view(1, T, 4).long(), grad_loss=0.01,
                             dweights=dw.view(1, T, 4))
    assert same[2].shape == (1, T, 64) and _eq(same[2][0], dz)


@pytest.mark.parametrize("T, E, K", [(2400, 64, 256), (400, 384, 512), (1301, 100, 32)])
def test_router_logits_of_many_tokens(cuda, T, E, K):
    """Enough tiles for all SMs: the products are written by one launch, K not split."""
    gate, gen = _gate(E, K)
    x = torch.randn(T, K, generator=gen, device="cuda").to(BF)
    z = gate.logits(x)
    z64 = x.to(D) @ gate.weight.to(D).T
    mag = x.to(D).abs() @ gate.weight.to(D).abs().T
    assert z.shape == (T, E) and ((z.to(D) - z64).abs() <= 4 * K ** 0.5 * 2.0 ** -23 * mag).all()


def test_graph_replay(cuda):
    graphs = []
    for T in (50, 4000):
        g, z, idx, dw = _inputs(T, T, 96, 4)
        offsets = torch.tensor([0, T // 3, T], dtype=torch.int32, device="cuda")

        gl = torch.ones(2, device="cuda")

        def step(z=z, idx=idx, offsets=offsets, dw=dw, gl=gl):
            return q.moe.balance_loss(z, idx, offsets, grad_loss=gl, dweights=dw)
        step()
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs = step()
        graphs.append((gr, outs, step, z, idx, g))
    for _ in range(3):
        for gr, outs, step, z, idx, g in graphs:
            z.copy_(torch.randn(z.shape, generator=g, device="cuda"))
            idx.copy_(torch.topk(z, 4, 1).indices.int())
        torch.cuda.synchronize()
        for gr, *_ in graphs:
            with torch.cuda.stream(torch.cuda.Stream()):
                gr.replay()
        torch.cuda.synchronize()
        for gr, outs, step, *_ in graphs:
            assert all(_eq(u, v) for u, v in zip(outs, step()))


def test_empty(cuda):
    g, z, idx, dw = _inputs(0, 0, 16, 2)
    loss, cnt, dz = q.moe.balance_loss(z, idx, grad_loss=1.0, dweights=dw)
    assert loss.tolist() == [0.0] and (cnt == 0).all() and dz.shape == (0, 16)
    z, idx = torch.randn(9, 16, device="cuda"), torch.zeros(9, 2, dtype=torch.int32, device="cuda")
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    loss, cnt, dz = q.moe.balance_loss(z, idx, none, grad_loss=torch.empty(0, device="cuda"))
    assert loss.shape == (0,) and cnt.shape == (0, 16) and (dz == 0).all()


def test_refusals(cuda):
    g, z, idx, dw = _inputs(1, 8, 16, 2)
    f = q.moe.balance_loss
    off = torch.tensor([0, 8], dtype=torch.int32, device="cuda")
    for bad in (lambda: f(z.half(), idx), lambda: f(z, idx.float()), lambda: f(z, idx[:7]),
                lambda: f(z, idx, off.long()), lambda: f(z, idx, off[:0]),
                lambda: f(z, idx, mask=torch.ones(7, dtype=torch.bool, device="cuda")),
                lambda: f(z, idx, mask=torch.ones(8, device="cuda")),
                lambda: f(z, idx, grad_loss=torch.ones(2, device="cuda")),
                lambda: f(z, idx, dweights=dw[:, :1]), lambda: f(z, idx, dweights=dw.to(BF)),
                lambda: f(z, idx, score_func="relu"), lambda: f(z, idx, gate_temp=0.0),
                lambda: f(torch.zeros(2, 1025, device="cuda"), idx[:2]),
                lambda: f(z[:, :1].contiguous(), idx)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(q.DSV41Error):
        f(z.cpu(), idx)
