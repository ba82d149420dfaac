"""Timed cases of the adapter and router-training operators, with their plain forms.

Two families:

* low-rank adapters of many requests beside one shared projection
  (``lora.lora_forward`` / ``lora.lora_backward``): y[t] = base[t] + s_i (x[t] A_i^T) B_i^T with
  i = ids[t], rows with a negative id keep their base; and the gradients of x, A and B;
* the router's training pass (``moe.balance_loss``): per-sequence balance loss, per-expert
  counts, and the gradient of that loss and of the routing weights to the router's logits.

``run`` computes a case in elementary torch operations (``own`` false) or by the package's
operators (``own`` true); ``exact`` computes the same outputs from the definitions in float64.
"""

from __future__ import annotations

import importlib.util
import math
import os
import random
import sys

import torch

own = False


def _package():
    name = "deepseek_v41_mlx_b200"
    if name not in sys.modules:
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                           "deepseek-v41-mlx_b200")
        spec = importlib.util.spec_from_file_location(
            name, os.path.join(pkg, "__init__.py"), submodule_search_locations=[pkg])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


# ------------------------------------------------------------------------------- the cases

def _lora(name, op, tokens, inp, out, rank, adapters, requests, out_dtype="bf16", base=True):
    return dict(name=name, op=op, tokens=tokens, inp=inp, out=out, rank=rank, adapters=adapters,
                requests=requests, out_dtype=out_dtype, base=base)


def _bal(name, tokens, experts, topk, sequences, score, dtype, grad, routed, padded):
    return dict(name=name, op="balance", tokens=tokens, experts=experts, topk=topk,
                sequences=sequences, score=score, dtype=dtype, grad=grad, routed=routed,
                padded=padded)


def listed():
    return [
        # one request decoding one token through the fp8 projection of the headline GEMV
        _lora("lora_decode_1", "lora", 1, 7168, 4096, 16, 8, 1),
        # a decode batch, a token from each of 64 requests on 32 adapters, some on none
        _lora("lora_decode_64", "lora", 64, 7168, 4096, 16, 32, 64),
        # decode rows of many requests next to a prefill chunk, an odd token count, odd output
        # width, fp32 output
        _lora("lora_mixed_777", "lora", 777, 2048, 1153, 64, 24, 40, out_dtype="f32"),
        # a prefill of four requests through the wide projection of the affine workload
        _lora("lora_prefill_8192", "lora", 8192, 7168, 14336, 32, 4, 5),
        # training forward: the delta alone and the rank-sized product kept for the backward
        _lora("lora_train_4096", "lora_train", 4096, 4096, 7168, 128, 2, 4, base=False),
        # gradients of a few short sequences
        _lora("lora_grad_500", "lora_grad", 500, 2048, 1000, 8, 3, 6, base=False),
        # gradients of eight adapters trained side by side, added to the projection's own dx
        _lora("lora_grad_4096", "lora_grad", 4096, 7168, 4096, 16, 8, 16),
        # gradients of one adapter of a large rank over long sequences
        _lora("lora_grad_8192", "lora_grad", 8192, 7168, 4096, 64, 1, 4),
        # load statistics and loss of a decode batch's routing
        _bal("balance_64", 64, 384, 6, 1, "sqrtsoftplus", "f32", False, False, False),
        # training micro-batch of ragged padded sequences, loss and routing-weight gradients
        _bal("balance_5000", 5000, 384, 6, 7, "sqrtsoftplus", "f32", True, True, True),
        # softmax router with bf16 logits, one batch-wide loss
        _bal("balance_16384", 16384, 256, 8, 1, "softmax", "bf16", True, True, False),
        # a large step of sixteen sequences
        _bal("balance_65536", 65536, 384, 6, 16, "sqrtsoftplus", "f32", True, True, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["lora", "lora", "lora_train", "lora_grad", "lora_grad", "balance",
                       "balance"])
    if kind == "balance":
        experts = rng.choice([8, 60, 64, 96, 160, 256, 300, 384])
        return dict(op="balance", tokens=_log(rng, 1, 65536), experts=experts,
                    topk=rng.randint(1, 8), sequences=_log(rng, 1, 64),
                    score=rng.choice(["sqrtsoftplus", "sigmoid", "softmax"]),
                    dtype=rng.choice(["f32", "bf16"]), grad=rng.random() < 0.8,
                    routed=rng.random() < 0.7, padded=rng.random() < 0.5)
    tokens = _log(rng, 1, 4096)
    inp = 8 * _log(rng, 32, 896)
    out = _log(rng, 65, 7168)
    if rng.random() < 0.6:
        out = (out + 7) // 8 * 8
    return dict(op=kind, tokens=tokens, inp=inp, out=out, rank=8 * _log(rng, 1, 16),
                adapters=_log(rng, 1, 32), requests=_log(rng, 1, 64),
                out_dtype=rng.choice(["bf16", "bf16", "f32"]), base=rng.random() < 0.7)


# ----------------------------------------------------------------------------- the inputs

def _randn(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _request_ids(case, seed):
    """Adapter of every token: requests one after another, each a run of tokens on one adapter;
    one request in eight is on none.  With a token a request it is a decode batch."""
    r = random.Random(seed)
    T, n = case["tokens"], case["adapters"]
    q = min(case["requests"], T)
    cuts = sorted(r.sample(range(1, T), q - 1)) if q > 1 else []
    bounds = [0] + cuts + [T]
    order = list(range(n))
    r.shuffle(order)
    ids, j = [], 0
    for i in range(q):
        if i % 8 == 7:
            a = -1
        else:
            a = order[j % n]
            j += 1
        ids += [a] * (bounds[i + 1] - bounds[i])
    return ids


def _prepare_lora(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    T, K, N, R, n = (case[k] for k in ("tokens", "inp", "out", "rank", "adapters"))
    bf, f32 = torch.bfloat16, torch.float32
    odt = f32 if case["out_dtype"] == "f32" else bf
    ids = _request_ids(case, seed)
    st = dict(op=case["op"], n=n, odt=odt,
              x=_randn(gen, (T, K), bf), a=_randn(gen, (n, R, K), bf, K ** -0.5),
              b=_randn(gen, (n, N, R), bf, R ** -0.5),
              ids=torch.tensor(ids, dtype=torch.int32, device="cuda"),
              scaling=torch.rand(n, generator=gen, device="cuda") + 0.5, base=None)
    # the tokens of each adapter, as a program that looped over its requests would know them
    st["groups"] = [(i, torch.tensor([t for t, v in enumerate(ids) if v == i], device="cuda"))
                    for i in sorted(set(ids)) if i >= 0]
    if case["op"] == "lora_grad":
        st["dy"] = _randn(gen, (T, N), bf, 1e-2)
        h = torch.zeros((T, R), dtype=f32, device="cuda")
        for i, t in st["groups"]:
            h[t] = st["x"][t].float() @ st["a"][i].float().T
        st["h"] = h
        if case["base"]:
            st["base"] = _randn(gen, (T, K), odt, 1e-2)
    elif case["base"]:
        st["base"] = _randn(gen, (T, N), odt)
    return st


_FUNCS = ("sqrtsoftplus", "sigmoid", "softmax")


def _prepare_balance(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = random.Random(seed)
    T, E, k, S = (case[c] for c in ("tokens", "experts", "topk", "sequences"))
    dt = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
    S = min(S, T)
    # some experts are preferred, as in a router before its loads are balanced
    logits = _randn(gen, (T, E), torch.float32) + 0.7 * _randn(gen, (1, E), torch.float32)
    logits = logits.to(dt)
    mask = None
    if case["padded"]:
        end = T - T // 16                     # a tail behind the last sequence, and padding
        mask = torch.rand(T, generator=gen, device="cuda") > 0.1
    else:
        end = T
    S = min(S, end)
    cuts = sorted(r.sample(range(1, end), S - 1)) if S > 1 else []
    offsets = torch.tensor([0] + cuts + [end], dtype=torch.int32, device="cuda")
    indices = torch.topk(logits.float(), k, dim=1).indices.to(torch.int32)
    return dict(op="balance", logits=logits, indices=indices, offsets=offsets, mask=mask,
                score=case["score"], grad=case["grad"],
                grad_loss=(torch.full((S,), 1e-2 / S, device="cuda") if case["grad"] else None),
                dweights=(_randn(gen, (T, k), torch.float32, 1e-2)
                          if case["grad"] and case["routed"] else None))


def prepare(case, seed):
    return _prepare_balance(case, seed) if case["op"] == "balance" else _prepare_lora(case, seed)


# ------------------------------------------------------------------------------ the passes

def _plain_lora(s):
    x, a, b, scaling = s["x"], s["a"], s["b"], s["scaling"]
    T, N, R = x.shape[0], b.shape[1], a.shape[1]
    y = s["base"].float() if s["base"] is not None else torch.zeros((T, N), device=x.device)
    y = y.clone() if s["odt"] == torch.float32 else y
    h = torch.zeros((T, R), device=x.device)
    for i, t in s["groups"]:
        hi = x[t].float() @ a[i].float().T
        y[t] += scaling[i] * (hi @ b[i].float().T)
        h[t] = hi
    y = y.to(s["odt"])
    return (y, h) if s["op"] == "lora_train" else y


def _plain_lora_grad(s):
    x, a, b, h, dy, scaling = s["x"], s["a"], s["b"], s["h"], s["dy"], s["scaling"]
    dx = s["base"].float() if s["base"] is not None else torch.zeros(x.shape, device=x.device)
    dx = dx.clone() if s["odt"] == torch.float32 else dx
    da = torch.zeros(a.shape, device=x.device)
    db = torch.zeros(b.shape, device=x.device)
    for i, t in s["groups"]:
        dyi = dy[t].float() * scaling[i]
        g = dyi @ b[i].float()
        dx[t] += g @ a[i].float()
        da[i] = g.T @ x[t].float()
        db[i] = dyi.T @ h[t]
    return dx.to(s["odt"]), da.to(a.dtype), db.to(b.dtype)


def _plain_balance(s):
    z = s["logits"].float()
    T, E = z.shape
    idx = s["indices"].long()
    k = idx.shape[1]
    S = s["offsets"].numel() - 1
    seq = torch.bucketize(torch.arange(T, device=z.device), s["offsets"].long(), right=True) - 1
    live = seq < S
    if s["mask"] is not None:
        live = live & s["mask"]
    seq = torch.where(live, seq, S)
    # the sum of a row's scores normalises it; the chosen experts count for its sequence
    if s["score"] == "softmax":
        ex = torch.exp(z - z.amax(1, keepdim=True))
        sc = ex / ex.sum(1, keepdim=True)
    elif s["score"] == "sigmoid":
        sc = 1 / (1 + torch.exp(-z))
    else:
        sc = torch.sqrt(torch.clamp(z, min=0) + torch.log1p(torch.exp(-z.abs())))
    total = sc.sum(1, keepdim=True) + 1e-20
    p = sc / total
    one = torch.ones_like(idx, dtype=torch.int32)
    counts = torch.zeros((S + 1) * E, dtype=torch.int32, device=z.device)
    counts = counts.index_add(0, (seq[:, None] * E + idx).reshape(-1), one.reshape(-1))
    counts = counts.reshape(S + 1, E)
    m = torch.zeros(S + 1, device=z.device).index_add(0, seq, torch.ones(T, device=z.device))
    f = counts.float()[seq]
    dot = (f * p).sum(1)
    coef = E / (k * torch.clamp(m, min=1) ** 2)
    loss = (torch.zeros(S + 1, device=z.device).index_add(0, seq, dot) * coef)[:S]
    if not s["grad"]:
        return loss, counts[:S]
    up = torch.zeros(S + 1, device=z.device)
    up[:S] = s["grad_loss"] * coef[:S]
    ds = up[seq][:, None] * (f - dot[:, None]) / total
    if s["dweights"] is not None:
        ws = torch.gather(sc, 1, idx)
        z0 = ws.sum(1, keepdim=True) + 1e-20
        dw = s["dweights"]
        if k > 1:
            w = ws / z0
            dw = (dw - (dw * w).sum(1, keepdim=True)) / z0
        dw = torch.where(live[:, None], 1.5 * dw, 0.0)
        ds = ds.scatter_add(1, idx, dw)
    if s["score"] == "softmax":
        dz = sc * (ds - (ds * sc).sum(1, keepdim=True))
    elif s["score"] == "sigmoid":
        dz = ds * sc * (1 - sc)
    else:
        dz = ds / (1 + torch.exp(-z)) / (2 * sc)
    return loss, counts[:S], dz.to(s["logits"].dtype)


def run(state):
    s = state
    if s["op"] == "balance":
        if not own:
            return _plain_balance(s)
        loss, counts, dz = _package().moe.balance_loss(
            s["logits"], s["indices"], offsets=s["offsets"], mask=s["mask"],
            score_func=s["score"], grad_loss=s["grad_loss"], dweights=s["dweights"],
            route_scale=1.5)
        return (loss, counts, dz) if s["grad"] else (loss, counts)
    if s["op"] == "lora_grad":
        if not own:
            return _plain_lora_grad(s)
        return _package().lora.lora_backward(
            s["dy"], s["x"], s["h"], s["a"], s["b"], s["ids"], scaling=s["scaling"],
            dx_base=s["base"], dx_dtype=s["odt"])
    if not own:
        return _plain_lora(s)
    return _package().lora.lora_forward(
        s["x"], s["a"], s["b"], s["ids"], scaling=s["scaling"], base=s["base"],
        out_dtype=s["odt"], return_h=s["op"] == "lora_train")


# --------------------------------------------------------------------- what a pass is worth

def work(case):
    T = case["tokens"]
    if case["op"] == "balance":
        E, k = case["experts"], case["topk"]
        S = min(case["sequences"], T)
        e = 4 if case["dtype"] == "f32" else 2
        by = T * E * e + T * k * 4 + S * (4 + 4 * E) + (T if case["padded"] else 0)
        fl = T * E * 8
        if case["grad"]:
            by += T * E * e + S * 4 + (T * k * 4 if case["routed"] else 0)
            fl += T * E * 10
        return {"bytes": by, "flops": fl}
    K, N, R, n = (case[c] for c in ("inp", "out", "rank", "adapters"))
    q = min(case["requests"], T)
    used = min(n, q - q // 8)
    o = 4 if case["out_dtype"] == "f32" else 2
    by = T * K * 2 + used * R * (K + N) * 2 + T * 4 + n * 4
    if case["op"] == "lora_grad":
        by += T * N * 2 + T * R * 4 + T * K * o * (2 if case["base"] else 1)
        by += n * R * (K + N) * 2
        return {"bytes": by, "flops": 4 * T * R * (K + N)}
    by += T * N * o * (2 if case["base"] else 1)
    if case["op"] == "lora_train":
        by += T * R * 4
    return {"bytes": by, "flops": 2 * T * R * (K + N)}


# --------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    d = torch.float64
    if case["op"] == "balance":
        return _exact_balance(case, s)
    x, a, b, sc = s["x"].to(d), s["a"].to(d), s["b"].to(d), s["scaling"].to(d)
    ids = s["ids"].long()
    grad = case["op"] == "lora_grad"
    first = (s["base"].to(d) if s["base"] is not None else
             torch.zeros((x.shape[0], x.shape[1] if grad else b.shape[1]), dtype=d, device="cuda"))
    if grad:
        dy, h = s["dy"].to(d), s["h"].to(d)
        da, db, dx = torch.zeros_like(a), torch.zeros_like(b), first.clone()
        for i in range(case["adapters"]):
            rows = torch.nonzero(ids == i)[:, 0]
            if rows.numel():
                g = torch.einsum("tn,nr->tr", dy[rows], b[i]) * sc[i]
                dx[rows] += torch.einsum("tr,rk->tk", g, a[i])
                da[i] = torch.einsum("tr,tk->rk", g, x[rows])
                db[i] = torch.einsum("tn,tr->nr", dy[rows], h[rows]) * sc[i]
        return dx, da, db
    y = first.clone()
    hs = torch.zeros((x.shape[0], a.shape[1]), dtype=d, device="cuda")
    for i in range(case["adapters"]):
        rows = torch.nonzero(ids == i)[:, 0]
        if rows.numel():
            hs[rows] = torch.einsum("tk,rk->tr", x[rows], a[i])
            y[rows] += torch.einsum("tr,nr->tn", hs[rows], b[i]) * sc[i]
    return (y, hs) if case["op"] == "lora_train" else y


def _exact_balance(case, s):
    d = torch.float64
    z = s["logits"].to(d).requires_grad_(True)
    E, k = z.shape[1], s["indices"].shape[1]
    off = s["offsets"].tolist()
    live = torch.ones(z.shape[0], dtype=torch.bool, device="cuda") if s["mask"] is None \
        else s["mask"]
    if case["score"] == "softmax":
        score = torch.softmax(z, 1)
    elif case["score"] == "sigmoid":
        score = torch.sigmoid(z)
    else:
        score = torch.logaddexp(z, torch.zeros_like(z)).sqrt()
    losses, counts, aim = [], [], 0.0
    for q in range(len(off) - 1):
        rows = torch.arange(off[q], off[q + 1], device="cuda")
        rows = rows[live[rows]]
        idx = s["indices"][rows].long()
        c = torch.bincount(idx.reshape(-1), minlength=E)
        counts.append(c)
        m = max(rows.numel(), 1)
        f = c.to(d) * E / (k * m)
        mean_p = (score[rows] / (score[rows].sum(1, keepdim=True) + 1e-20)).sum(0) / m
        losses.append((f * mean_p).sum())
        if case["grad"]:
            aim = aim + losses[-1] * s["grad_loss"][q].to(d)
            if s["dweights"] is not None:
                w = torch.gather(score[rows], 1, idx)
                if k > 1:
                    w = w / (w.sum(1, keepdim=True) + 1e-20)
                aim = aim + (1.5 * w * s["dweights"][rows].to(d)).sum()
    loss, cnt = torch.stack(losses).detach(), torch.stack(counts).to(torch.int32)
    if not case["grad"]:
        return loss, cnt
    return loss, cnt, torch.autograd.grad(aim, z)[0]
