"""Low-rank adapters beside a projection: forward, gradients, layers, refusals.

Every output is compared element by element with the formula in float64.  Tolerances count
rounding steps: a sum of m fp32 terms is off by about sqrt(m) steps of 2^-23 of the sum of the
terms' magnitudes (4 standard deviations allowed; a tensor core's truncating accumulator stays
inside that, since its partial sums are about 1 / sqrt(m) of that sum), the rank-sized
intermediate keeps at least 17 significant bits, and the output is rounded once, half a step of
its type.
"""

from __future__ import annotations

import ctypes as C
import threading

import pytest
import torch

import deepseek_v41_mlx_b200 as q
from deepseek_v41_mlx_b200 import _lib as L

pytestmark = pytest.mark.gpu

BF, F32, D = torch.bfloat16, torch.float32, torch.float64


def _eq(a, b):
    return bool(torch.equal(a, b))


def _randn(gen, *shape, scale=1.0, dtype=BF):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _case(seed, T, K, N, R, n):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return dict(x=_randn(g, T, K), a=_randn(g, n, R, K, scale=K ** -0.5),
                b=_randn(g, n, N, R, scale=R ** -0.5),
                s=torch.rand(n, generator=g, device="cuda") + 0.5, g=g)


def _ids(kind, T, n, g):
    if kind == "none":
        return torch.full((T,), -1, dtype=torch.int32, device="cuda")
    if kind == "runs":
        return (torch.arange(T, device="cuda") * (n + 1) // max(T, 1) - 1).to(torch.int32)
    if kind == "one":
        return torch.full((T,), n - 1, dtype=torch.int32, device="cuda")
    return torch.randint(-1, n, (T,), generator=g, device="cuda").to(torch.int32)


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _sel(w, ids):
    """w[ids] in float64, zero for rows without an adapter."""
    live = (ids >= 0) & (ids < w.shape[0])
    out = w.to(D)[ids.clamp(0, w.shape[0] - 1).long()]
    return out * live.view(-1, *([1] * (w.dim() - 1)))


def _rows(fn, ids, n):
    """fn(i, rows) for every adapter that has rows."""
    for i in range(n):
        rows = torch.nonzero(ids == i)[:, 0]
        if rows.numel():
            fn(i, rows)


def _forward64(c, ids, base):
    """(y, h, the sum of magnitudes behind y, behind h) in float64."""
    x, a, b, s = c["x"].to(D), c["a"].to(D), c["b"].to(D), c["s"].to(D)
    T, N, R = x.shape[0], b.shape[1], a.shape[1]
    y = base.to(D).clone() if base is not None else torch.zeros(T, N, dtype=D, device="cuda")
    h = torch.zeros(T, R, dtype=D, device="cuda")
    ya, ha = torch.zeros_like(y), torch.zeros_like(h)

    def one(i, t):
        h[t] = x[t] @ a[i].T
        ha[t] = x[t].abs() @ a[i].abs().T
        y[t] += s[i] * (h[t] @ b[i].T)
        ya[t] = s[i] * (ha[t] @ b[i].abs().T)
    _rows(one, ids, a.shape[0])
    return y, h, ya, ha


def _check_forward(c, ids, base, odt, y, h=None):
    K, R = c["a"].shape[2], c["a"].shape[1]
    y64, h64, ya, ha = _forward64(c, ids, base)
    step = 2.0 ** -23 * 4 * (K + R) ** 0.5
    tol = step * ya + 2.0 ** -17 * ya + _half_step(odt) * y64.abs() * 1.01
    assert ((y.to(D) - y64).abs() <= tol + 1e-30).all()
    if h is not None:
        assert ((h.to(D) - h64).abs() <= 2.0 ** -23 * 4 * K ** 0.5 * ha).all()
    idle = (ids < 0) | (ids >= c["a"].shape[0])
    if base is not None:
        assert _eq(y[idle], base[idle])
    else:
        assert (y[idle] == 0).all()
    return y64


# one token; one tile and its neighbours; more tokens than a tile; ragged K, N, R
SHAPES = [(1, 64, 8, 8, 1), (1, 7168, 4096, 16, 3), (3, 72, 33, 8, 2), (17, 256, 130, 24, 5),
          (64, 1032, 200, 16, 32), (127, 512, 96, 40, 4), (129, 520, 257, 64, 3),
          (300, 1024, 1000, 128, 7), (1025, 768, 384, 72, 2), (2000, 136, 1153, 16, 600)]


@pytest.mark.parametrize("kind", ["mixed", "runs", "one", "none"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward(cuda, shape, kind):
    T, K, N, R, n = shape
    c = _case(sum(shape), *shape)
    ids = _ids(kind, T, n, c["g"])
    for odt in (BF, F32):
        for with_base in (True, False):
            base = _randn(c["g"], T, N, dtype=odt) if with_base else None
            y, h = q.lora.lora_forward(c["x"], c["a"], c["b"], ids, c["s"], base, odt,
                                       return_h=True)
            assert y.dtype == odt and h.dtype == F32
            _check_forward(c, ids, base, odt, y, h)
            y2 = q.lora.lora_forward(c["x"], c["a"], c["b"], ids, c["s"], base, odt)
            assert _eq(y, y2)


@pytest.mark.parametrize("shape", [(40, 16384, 64, 16, 4), (513, 14336, 136, 32, 3)], ids=str)
def test_forward_long_rows(cuda, shape):
    c = _case(5, *shape)
    ids = _ids("mixed", shape[0], shape[4], c["g"])
    y, h = q.lora.lora_forward(c["x"], c["a"], c["b"], ids, c["s"], out_dtype=F32, return_h=True)
    _check_forward(c, ids, None, F32, y, h)


@pytest.mark.parametrize("kind", ["mixed", "runs", "none"])
@pytest.mark.parametrize("shape", [(3000, 72, 33, 8, 2), (2500, 264, 130, 24, 5),
                                   (1300, 1032, 200, 104, 9), (1100, 520, 256, 48, 1),
                                   (1030, 8, 1, 8, 3), (2049, 4096, 64, 128, 2)], ids=str)
def test_forward_many_tokens(cuda, shape, kind):
    """Sorted tiles: ranks of every piece width, odd and single columns, short contractions."""
    T, K, N, R, n = shape
    c = _case(sum(shape), *shape)
    ids = _ids(kind, T, n, c["g"])
    for odt in (BF, F32):
        base = _randn(c["g"], T, N, dtype=odt)
        y, h = q.lora.lora_forward(c["x"], c["a"], c["b"], ids, c["s"], base, odt, return_h=True)
        _check_forward(c, ids, base, odt, y, h)
        y = q.lora.lora_forward(c["x"], c["a"], c["b"], ids, c["s"], out_dtype=odt)
        _check_forward(c, ids, None, odt, y)


@pytest.mark.parametrize("T", [3, 1500])
def test_unaligned_base_and_output(cuda, T):
    """Rows of base and the output may start at any element."""
    c = _case(14, T, 256, 128, 16, 3)
    ids = _ids("mixed", T, 3, c["g"])
    dy = _randn(c["g"], T, 128)
    _, h = q.lora.lora_forward(c["x"], c["a"], c["b"], ids, c["s"], return_h=True)
    for dt in (BF, F32):
        flat = _randn(c["g"], T * 128 + 1, dtype=dt)
        base = flat[1:].view(T, 128)
        want = q.lora.lora_forward(c["x"], c["a"], c["b"], ids, c["s"], base.clone(), dt)
        assert _eq(q.lora.lora_forward(c["x"], c["a"], c["b"], ids, c["s"], base, dt), want)
        out = torch.empty(T * 128 + 1, dtype=dt, device="cuda")[1:].view(T, 128)
        q.lora.lora_forward(c["x"], c["a"], c["b"], ids, c["s"], base, dt, out=out)
        assert _eq(out, want)
        xb = _randn(c["g"], T * 256 + 1, dtype=dt)[1:].view(T, 256)
        g1 = q.lora.lora_backward(dy, c["x"], h, c["a"], c["b"], ids, c["s"], xb, dt)
        g2 = q.lora.lora_backward(dy, c["x"], h, c["a"], c["b"], ids, c["s"], xb.clone(), dt)
        assert all(_eq(u, v) for u, v in zip(g1, g2))


def test_more_than_2_31_values(cuda):
    """Offsets into x, y and their gradients past 32 bits: rows at both ends against the formula."""
    T, K, N, R, n = 300_000, 7200, 7208, 8, 2
    g = torch.Generator(device="cuda").manual_seed(3)
    c = dict(a=_randn(g, n, R, K, scale=K ** -0.5), b=_randn(g, n, N, R), g=g,
             s=torch.ones(n, device="cuda"))
    x = torch.randn(1000, K, generator=g, device="cuda").to(BF).repeat(T // 1000, 1)
    ids = _ids("mixed", T, n, g)
    y, h = q.lora.lora_forward(x, c["a"], c["b"], ids, c["s"], return_h=True)
    rows = torch.cat([torch.arange(200), torch.arange(T - 200, T)]).cuda()
    _check_forward(dict(c, x=x[rows]), ids[rows], None, BF, y[rows], h[rows])
    dx, da, db = q.lora.lora_backward(y, x, h, c["a"], c["b"], ids, c["s"])
    (dx64, _, _), (mag, _, _) = _backward64(dict(c, x=x[rows]), ids[rows], y[rows], h[rows], None)
    tol = (2.0 ** -23 * 4 * N ** 0.5 + 2.0 ** -17) * mag + _half_step(BF) * dx64.abs() * 1.01
    assert ((dx[rows].to(D) - dx64).abs() <= tol).all()
    # db in slices of the tokens: sums of 1.5e5 terms, in fp32 partial sums of 64-token stages
    want, mag = torch.zeros(n, N, R, dtype=D, device="cuda"), torch.zeros(n, N, R, device="cuda")
    for t0 in range(0, T, 20000):
        t = slice(t0, t0 + 20000)
        for i in range(n):
            k = torch.nonzero(ids[t] == i)[:, 0]
            yi, hi = y[t][k], h[t][k]
            want[i] += yi.to(D).T @ hi.to(D)
            mag[i] += yi.float().abs().T @ hi.abs()
    tol = (2.0 ** -23 * 4 * T ** 0.5 + 2.0 ** -17) * mag + _half_step(BF) * want.abs() * 1.01
    assert ((db.to(D) - want).abs() <= tol).all()


def test_more_than_2_31_parts(cuda):
    """Many short rows: the parts of h and g are past 2^31 values; rows at both ends and whole
    gradients against the formula."""
    T, K, N, R, n = 60_000_000, 8, 8, 8, 2
    g = torch.Generator(device="cuda").manual_seed(4)
    c = dict(a=_randn(g, n, R, K), b=_randn(g, n, N, R), g=g, s=torch.ones(n, device="cuda"))
    x = torch.randn(1000, K, generator=g, device="cuda").to(BF).repeat(T // 1000, 1)
    ids = _ids("mixed", T, n, g)
    y, h = q.lora.lora_forward(x, c["a"], c["b"], ids, c["s"], return_h=True)
    dx, da, db = q.lora.lora_backward(y, x, h, c["a"], c["b"], ids, c["s"])
    rows = torch.cat([torch.arange(200), torch.arange(T - 200, T)]).cuda()
    _check_forward(dict(c, x=x[rows]), ids[rows], None, BF, y[rows], h[rows])
    (dx64, _, _), (mag, _, _) = _backward64(dict(c, x=x[rows]), ids[rows], y[rows], h[rows], None)
    tol = (2.0 ** -23 * 4 * N ** 0.5 + 2.0 ** -17) * mag + _half_step(BF) * dx64.abs() * 1.01
    assert ((dx[rows].to(D) - dx64).abs() <= tol).all()
    want, mag = (torch.zeros(n, N, R, dtype=D, device="cuda") for _ in range(2))
    for t0 in range(0, T, 4_000_000):
        t = slice(t0, t0 + 4_000_000)
        for i in range(n):
            k = ids[t] == i
            yi, hi = y[t][k].to(D), h[t][k].to(D)
            want[i] += yi.T @ hi
            mag[i] += yi.abs().T @ hi.abs()
    tol = (2.0 ** -23 * 4 * T ** 0.5 + 2.0 ** -17) * mag + _half_step(BF) * want.abs() * 1.01
    assert ((db.to(D) - want).abs() <= tol).all()


def test_forward_in_place_leading_shape_and_int64_ids(cuda):
    c = _case(9, 24, 256, 120, 16, 4)
    ids = _ids("mixed", 24, 4, c["g"])
    base = _randn(c["g"], 24, 120)
    want = q.lora.lora_forward(c["x"], c["a"], c["b"], ids, c["s"], base)
    y = base.clone()
    got = q.lora.lora_forward(c["x"].view(2, 3, 4, 256), c["a"], c["b"], ids.long().view(2, 3, 4),
                              c["s"], y, out=y)
    assert got is y and _eq(got, want)
    x2 = torch.cat([c["x"], c["x"]], 1)[:, :256]               # row stride 512
    assert _eq(q.lora.lora_forward(x2, c["a"], c["b"], ids, c["s"], base), want)
    out = torch.empty(24, 120, dtype=BF, device="cuda")
    q.lora.lora_forward(c["x"], c["a"], c["b"], ids, c["s"], base, out=out)
    assert _eq(out, want)
    # scaling None is 1
    one = torch.ones(4, device="cuda")
    assert _eq(q.lora.lora_forward(c["x"], c["a"], c["b"], ids, None, base),
                       q.lora.lora_forward(c["x"], c["a"], c["b"], ids, one, base))


@pytest.mark.parametrize("T", [5, 700])
def test_idle_rows_and_unused_adapters_may_hold_anything(cuda, T):
    """Infinities and NaN in rows on no adapter, and in adapters nobody uses, stay where they
    are: every other row keeps its bits, forward and backward."""
    c = _case(11, T, 264, 136, 16, 6)
    ids = _ids("mixed", T, 6, c["g"])
    ids[ids == 2] = -1
    ids[0], ids[1], ids[T - 1] = 1, -1, -1
    base = _randn(c["g"], T, 136)
    dy = _randn(c["g"], T, 136)
    y, h = q.lora.lora_forward(c["x"], c["a"], c["b"], ids, c["s"], base, return_h=True)
    grads = q.lora.lora_backward(dy, c["x"], h, c["a"], c["b"], ids, c["s"])
    idle = ids < 0
    x2, dy2, a2, b2, s2 = (v.clone() for v in (c["x"], dy, c["a"], c["b"], c["s"]))
    x2[idle], dy2[idle] = float("nan"), float("inf")
    a2[2], b2[2], s2[2] = float("inf"), float("nan"), float("nan")
    y2, h2 = q.lora.lora_forward(x2, a2, b2, ids, s2, base, return_h=True)
    assert _eq(y, y2) and _eq(h, h2)
    h2[idle] = float("nan")
    for g, g2 in zip(grads, q.lora.lora_backward(dy2, x2, h2, a2, b2, ids, s2)):
        assert _eq(g, g2)
    assert (grads[1][2] == 0).all() and (grads[2][2] == 0).all() and (grads[0][idle] == 0).all()


def test_non_finite_rows_stay_in_their_rows(cuda):
    c = _case(12, 200, 256, 128, 8, 2)
    ids = _ids("mixed", 200, 2, c["g"])
    ids[7] = 0
    want = q.lora.lora_forward(c["x"], c["a"], c["b"], ids, c["s"])
    x2 = c["x"].clone()
    x2[7, 3] = float("inf")
    y = q.lora.lora_forward(x2, c["a"], c["b"], ids, c["s"])
    rest = torch.arange(200, device="cuda") != 7
    assert _eq(y[rest], want[rest]) and not torch.isfinite(y[7]).all()


@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
@pytest.mark.parametrize("T, N", [(5, 64), (700, 64), (700, 65)])
def test_rows_without_adapter_keep_every_bit_of_base(cuda, T, N, dtype):
    c = _case(14, T, 64, N, 16, 3)
    ids = _ids("mixed", T, 3, c["g"])
    base = _randn(c["g"], T, N, dtype=dtype)
    base[:, ::3] = -0.0
    y = q.lora.lora_forward(c["x"], c["a"], c["b"], ids, c["s"], base=base)
    bits = torch.int16 if dtype is BF else torch.int32
    idle = ids < 0
    assert idle.any() and _eq(y[idle].view(bits), base[idle].view(bits))


@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
@pytest.mark.parametrize("T, N", [(5, 64), (5, 65), (3000, 64), (3000, 65)])
def test_rows_without_adapter_keep_nan_payloads(cuda, T, N, dtype):
    """Few tokens and sorted tiles alike: base's NaN of both kinds, infinities and zeros of both
    signs come out as they are, and zeros where there is no base."""
    c = _case(15, T, 64, N, 16, 3)
    ids = _ids("mixed", T, 3, c["g"])
    ids[0], ids[T // 2:] = -1, -1                  # whole tiles without an adapter among them
    bits, shift = (torch.int16, 0) if dtype is BF else (torch.int32, 16)
    words = [0x7F81, 0x7FC5, 0x7F80, 0x0000, 0x7FFF, 0x0001, 0x3F80]
    words = [w << shift | (3 if shift and w & 0x7F else 0) for w in words]
    top = 16 + shift
    words += [w - (1 << (top - 1)) for w in words]     # the same with the sign bit
    base = torch.tensor(words, dtype=bits, device="cuda").repeat(T * N // len(words) + 1)
    base = base[:T * N].view(T, N).view(dtype)
    idle = ids < 0
    y = q.lora.lora_forward(c["x"], c["a"], c["b"], ids, c["s"], base=base)
    assert _eq(y[idle].view(bits), base[idle].view(bits))
    y = base.clone()
    q.lora.lora_forward(c["x"], c["a"], c["b"], ids, c["s"], base=y, out=y)
    assert _eq(y[idle].view(bits), base[idle].view(bits))
    y = q.lora.lora_forward(c["x"], c["a"], c["b"], ids, c["s"], out_dtype=dtype)
    assert (y[idle].view(bits) == 0).all()
    dy, h = _randn(c["g"], T, N), _randn(c["g"], T, 16, dtype=F32)
    xb = torch.tensor(words, dtype=bits, device="cuda").repeat(T * 64 // len(words) + 1)
    xb = xb[:T * 64].view(T, 64).view(dtype)
    dx = q.lora.lora_backward(dy, c["x"], h, c["a"], c["b"], ids, c["s"], xb)[0]
    assert _eq(dx[idle].view(bits), xb[idle].view(bits))


def test_calls_from_several_threads(cuda):
    """Each thread has a stream and sizes of its own; the results are those of calls in turn."""
    jobs = []
    for k, (T, R) in enumerate([(900, 128), (700, 16), (800, 64), (600, 32)]):
        c = _case(40 + k, T, 264, 392, R, 5)
        ids = _ids("mixed", T, 5, c["g"])
        jobs.append((c, ids, _randn(c["g"], T, 392)))

    def run(c, ids, dy):
        y, h = q.lora.lora_forward(c["x"], c["a"], c["b"], ids, c["s"], return_h=True)
        return (y, h) + q.lora.lora_backward(dy, c["x"], h, c["a"], c["b"], ids, c["s"])
    got, errors = [[] for _ in jobs], []
    start = threading.Barrier(len(jobs))
    torch.cuda.synchronize()

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                for _ in range(5):
                    got[k].append(run(*jobs[k]))
                torch.cuda.current_stream().synchronize()
        except Exception as e:                       # shown by the assertion below
            errors.append(e)
    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(jobs))]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors
    for k, job in enumerate(jobs):
        want = run(*job)
        assert len(got[k]) == 5 and all(_eq(u, v) for r in got[k] for u, v in zip(r, want))


def test_ids_past_the_bank_count_as_none(cuda):
    c = _case(13, 40, 64, 32, 8, 3)
    ids = _ids("mixed", 40, 3, c["g"])
    base = _randn(c["g"], 40, 32)
    dy = _randn(c["g"], 40, 32)
    bad = ids.clone()
    bad[ids < 0] = 3
    bad[0] = 2147483647
    ids[0] = -1
    flags = C.c_uint32(0)
    stream = torch.cuda.current_stream().cuda_stream
    L.call("dsv41_device_status", stream, C.byref(flags))
    y, h = q.lora.lora_forward(c["x"], c["a"], c["b"], bad, c["s"], base, return_h=True)
    L.call("dsv41_device_status", stream, C.byref(flags))
    assert flags.value & 2
    assert _eq(y, q.lora.lora_forward(c["x"], c["a"], c["b"], ids, c["s"], base))
    g1 = q.lora.lora_backward(dy, c["x"], h, c["a"], c["b"], bad, c["s"])
    g2 = q.lora.lora_backward(dy, c["x"], h, c["a"], c["b"], ids, c["s"])
    assert all(_eq(u, v) for u, v in zip(g1, g2))
    L.call("dsv41_device_status", stream, C.byref(flags))


# ------------------------------------------------------------------------------- gradients

def _backward64(c, ids, dy, h, base):
    x, a, b, s = c["x"].to(D), c["a"].to(D), c["b"].to(D), c["s"].to(D)
    dy, h = dy.to(D), h.to(D)
    dx = base.to(D).clone() if base is not None else torch.zeros_like(x)
    dxa = torch.zeros_like(x)
    da, db, daa, dba = (torch.zeros_like(v) for v in (a, b, a, b))

    def one(i, t):
        g = s[i] * (dy[t] @ b[i])
        ga = s[i] * (dy[t].abs() @ b[i].abs())
        dx[t] += g @ a[i]
        dxa[t] = ga @ a[i].abs()
        da[i], daa[i] = g.T @ x[t], ga.T @ x[t].abs()
        db[i], dba[i] = s[i] * (dy[t].T @ h[t]), s[i] * (dy[t].abs().T @ h[t].abs())
    _rows(one, ids, a.shape[0])
    return (dx, da, db), (dxa, daa, dba)


@pytest.mark.parametrize("kind", ["mixed", "runs", "one", "none"])
@pytest.mark.parametrize("shape", SHAPES[:9] + [(2000, 136, 257, 16, 300)], ids=str)
def test_backward(cuda, shape, kind):
    T, K, N, R, n = shape
    c = _case(sum(shape) + 1, *shape)
    ids = _ids(kind, T, n, c["g"])
    dy = _randn(c["g"], T, N)
    _, h = q.lora.lora_forward(c["x"], c["a"], c["b"], ids, c["s"], return_h=True)
    for dt, with_base in ((BF, True), (F32, False), (F32, True), (BF, False)):
        base = _randn(c["g"], T, K, dtype=dt) if with_base else None
        got = q.lora.lora_backward(dy, c["x"], h, c["a"], c["b"], ids, c["s"], base, dt, dt)
        want, mag = _backward64(c, ids, dy, h, base)
        for g, w, m, terms in zip(got, want, mag, (N + R, N + T, T)):
            tol = (2.0 ** -23 * 4 * terms ** 0.5 + 2.0 ** -17) * m \
                + _half_step(dt) * w.abs() * 1.01
            assert g.dtype == dt and ((g.to(D) - w).abs() <= tol + 1e-30).all()
        again = q.lora.lora_backward(dy, c["x"], h, c["a"], c["b"], ids, c["s"], base, dt, dt)
        assert all(_eq(u, v) for u, v in zip(got, again))


# the weight gradients' ring has 5, 4, 6, 5, 4 stages for these ranks with bf16 gradients and
# 5, 6, 5, 4, 3, 3, 3 with fp32
@pytest.mark.parametrize("N", [1000, 1001])
@pytest.mark.parametrize("kind, n", [("one", 1), ("mixed", 3)])
@pytest.mark.parametrize("R, dt", [(16, BF), (32, BF), (64, BF), (96, BF), (128, BF), (8, F32),
                                   (32, F32), (64, F32), (96, F32), (104, F32), (112, F32),
                                   (128, F32)], ids=str)
def test_backward_pieces_of_many_rings(cuda, R, dt, kind, n, N):
    """13 stages of 64 tokens a CTA or more: every slot of its ring is used more than twice."""
    T, K = 14000, 2048
    c = _case(R + N + n, T, K, N, R, n)
    ids = _ids(kind, T, n, c["g"])
    dy, h = _randn(c["g"], T, N), _randn(c["g"], T, R, dtype=F32)
    got = q.lora.lora_backward(dy, c["x"], h, c["a"], c["b"], ids, c["s"], None, dt, dt)
    want, mag = _backward64(c, ids, dy, h, None)
    parts = 2.0 ** -17 if dt is BF else 0.0      # fp32 results keep all of g's and h's 24 bits
    for g, w, m, terms in zip(got, want, mag, (N + R, N + T, T)):
        tol = (2.0 ** -23 * 4 * terms ** 0.5 + parts) * m + _half_step(dt) * w.abs() * 1.01
        assert ((g.to(D) - w).abs() <= tol + 1e-30).all()
    for _ in range(3):
        again = q.lora.lora_backward(dy, c["x"], h, c["a"], c["b"], ids, c["s"], None, dt, dt)
        assert all(_eq(u, v) for u, v in zip(got, again))


# Sums of a single term: what is left of an error is the rounding of scaling times h or g (half a
# step of 2^-23), and at most one truncated or rounded step for each of the three additions that
# join the parts.  (A result from two parts, 17 bits, would be off by up to 64 steps.)
_SINGLE = 4 * 2.0 ** -23


def _one_row_a_column(gen, rows, cols):
    """bf16 [rows, cols] with one value in every column, in different rows."""
    v = torch.zeros(rows, cols, dtype=BF, device="cuda")
    at = torch.randperm(rows, generator=gen, device="cuda")[:cols]
    v[at, torch.arange(cols, device="cuda")] = _randn(gen, cols) + 2
    return v


@pytest.mark.parametrize("R", [8, 24, 64, 96, 104, 128])
@pytest.mark.parametrize("T, N", [(5, 200), (3000, 200), (3000, 201)])
def test_fp32_results_keep_every_bit_of_h_and_g(cuda, T, N, R):
    n, K = 3, 256
    c = _case(R + T + N, T, K, N, R, n)
    ids = _ids("mixed", T, n, c["g"])
    for w in (c["b"], c["a"].transpose(1, 2)):     # one rank in every column
        w *= torch.eye(R, device="cuda").repeat(w.shape[1] // R + 1, 1)[:w.shape[1]].to(BF)
    full = torch.randn(n, R, K, generator=c["g"], device="cuda").to(BF)
    y, h = q.lora.lora_forward(c["x"], full, c["b"], ids, c["s"], out_dtype=F32, return_h=True)
    live = ids >= 0
    hs = h.to(D) * (c["s"].to(D)[ids.clamp(min=0).long()] * live)[:, None]
    want = torch.einsum("tr,tcr->tc", hs, _sel(c["b"], ids))
    assert want[live].abs().min() > 0 and ((y.to(D) - want).abs() <= _SINGLE * want.abs()).all()
    if T < K:
        return
    c["x"], dy = _one_row_a_column(c["g"], T, K), _one_row_a_column(c["g"], T, N)
    c["b"] = _randn(c["g"], n, N, R)
    h = _randn(c["g"], T, R, dtype=F32)
    got = q.lora.lora_backward(dy, c["x"], h, c["a"], c["b"], ids, c["s"], None, F32, F32)
    want, _ = _backward64(c, ids, dy, h, None)
    for g, w in zip(got, want):
        assert (w != 0).any() and ((g.to(D) - w).abs() <= _SINGLE * w.abs()).all()


@pytest.mark.parametrize("shape", [(700, 512, 1000, 16, 4), (700, 512, 1001, 64, 4),
                                   (3000, 264, 96, 128, 3), (130, 72, 33, 8, 2)], ids=str)
def test_backward_of_mixed_types(cuda, shape):
    """dx and the weights' gradients have types of their own: the bits of one do not depend on the
    other's type."""
    T, K, N, R, n = shape
    c = _case(sum(shape), *shape)
    ids = _ids("mixed", T, n, c["g"])
    dy, h = _randn(c["g"], T, N), _randn(c["g"], T, R, dtype=F32)

    def grads(xdt, gdt):
        return q.lora.lora_backward(dy, c["x"], h, c["a"], c["b"], ids, c["s"], None, xdt, gdt)
    same = {dt: grads(dt, dt) for dt in (BF, F32)}
    for xdt, gdt in ((BF, F32), (F32, BF)):
        dx, da, db = grads(xdt, gdt)
        assert dx.dtype == xdt and da.dtype == db.dtype == gdt
        assert _eq(dx, same[xdt][0]) and _eq(da, same[gdt][1]) and _eq(db, same[gdt][2])


@pytest.mark.parametrize("dt", [BF, F32], ids=str)
@pytest.mark.parametrize("T", [6, 3000])
def test_infinities_stay_where_they_enter(cuda, T, dt):
    """Exactly the elements whose sums an infinity enters are not finite (infinite, or NaN where
    its products with the parts of h or g do not add up); all others keep their bits."""
    inf, n, R, K, N = float("inf"), 3, 16, 136, 72
    c = _case(90, T, K, N, R, n)
    ids = _ids("mixed", T, n, c["g"])
    ids[T - 1], ids[0] = 1, 0                      # the last row: the one that padding repeats
    mine, t0 = ids == 1, T - 1
    x, a, b, s = c["x"], c["a"], c["b"], c["s"]
    dy, h = _randn(c["g"], T, N), _randn(c["g"], T, R, dtype=F32)

    def put(v, *at):
        v = v.clone()
        v[at] = inf
        return v

    def fwd(x, a, b):
        return q.lora.lora_forward(x, a, b, ids, s, out_dtype=dt, return_h=True)

    def bwd(dy, x, a, b):
        return q.lora.lora_backward(dy, x, h, a, b, ids, s, None, dt, dt)

    def only(got, want, *where):
        for v, w, at in zip(got, want, where):
            bad = torch.zeros_like(v, dtype=torch.bool)
            if at is not None:
                bad[at] = True
            assert _eq(torch.isfinite(v), ~bad) and _eq(v[~bad], w[~bad])
    y, g = fwd(x, a, b), bwd(dy, x, a, b)
    every = slice(None)
    only(fwd(put(x, t0, 5), a, b), y, (t0,), (t0,))
    only(fwd(x, put(a, 1, 2, 5), b), y, (mine,), (mine, 2))
    only(fwd(x, a, put(b, 1, 7, 3)), y, (mine, 7), None)
    only(bwd(dy, put(x, t0, 5), a, b), g, None, (1, every, 5), None)
    only(bwd(dy, x, put(a, 1, 2, 5), b), g, (mine, 5), None, None)
    only(bwd(put(dy, t0, 7), x, a, b), g, (t0,), (1,), (1, 7))
    only(bwd(dy, x, a, put(b, 1, 7, 3)), g, (mine,), (1, 3), None)


@pytest.mark.parametrize("T", [6, 3000])
def test_values_past_the_largest_bf16(cuda, T):
    """h and g up to fp32's largest value, which a bf16 rounds to infinity: products that fit stay
    finite and keep every bit (sums of single terms and powers of two: no rounding at all)."""
    n, K, N, R = 2, 16, 24, 8
    ids = (torch.arange(T, device="cuda") % n).int()
    x, a = torch.zeros(T, K, dtype=BF, device="cuda"), torch.zeros(n, R, K, dtype=BF, device="cuda")
    b = torch.zeros(n, N, R, dtype=BF, device="cuda")
    x[:, 0], x[:, 1] = 2.0 ** 64, 2.0 ** 50
    a[:, 0, 0], a[:, 0, 1] = 2.0 ** 63 * 255 / 128, 2.0 ** 69 * 1.25
    a[1] *= -1
    b[:, :, 0] = 2.0 ** -10
    y, h = q.lora.lora_forward(x, a, b, ids, out_dtype=F32, return_h=True)
    big = 2.0 ** 127 * (255 / 128 + 1.25 * 2.0 ** -8)          # past the middle to 2^128
    sign = torch.where(ids == 0, 1.0, -1.0).to(D)[:, None]
    assert (h[:, :1].to(D) == big * sign).all() and (y.to(D) == big * 2.0 ** -10 * sign).all()
    y = q.lora.lora_forward(x, a, b, ids)
    assert (y.to(D) == 2.0 ** 118 * sign).all()
    dy = torch.zeros(T, N, dtype=BF, device="cuda")
    dy[0, 3] = dy[1, 3] = 2.0 ** -20
    dx, da, db = q.lora.lora_backward(dy, x, h, a, b, ids, dx_dtype=F32, grad_dtype=F32)
    assert (db[:, 3, 0].to(D) == big * 2.0 ** -20 * sign[:2, 0]).all()


def test_two_captured_graphs_of_sorted_tiles_at_once(cuda):
    cs = [_case(150 + i, T, 520, 264, R, 4) for i, (T, R) in enumerate(((2000, 16), (3000, 104)))]
    graphs = []
    for c, dt in zip(cs, (BF, F32)):
        T = c["x"].shape[0]
        c["ids"] = _ids("mixed", T, 4, c["g"])
        c["dy"] = _randn(c["g"], T, 264)

        def step(c=c, dt=dt):
            y, h = q.lora.lora_forward(c["x"], c["a"], c["b"], c["ids"], c["s"], out_dtype=dt,
                                       return_h=True)
            return (y, h) + q.lora.lora_backward(c["dy"], c["x"], h, c["a"], c["b"], c["ids"],
                                                 c["s"], None, dt, dt)
        step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step()
        graphs.append((g, outs, step, torch.cuda.Stream()))
    for rnd in range(3):
        for c in cs:
            c["x"].copy_(_randn(c["g"], *c["x"].shape))
            c["ids"].copy_(_ids(("mixed", "runs", "none")[rnd], c["x"].shape[0], 4, c["g"]))
        torch.cuda.synchronize()
        for g, _, _, st in graphs:
            with torch.cuda.stream(st):
                for _ in range(4):
                    g.replay()
        torch.cuda.synchronize()
        for _, outs, step, _ in graphs:
            assert all(_eq(o, w) for o, w in zip(outs, step()))


def test_gradients_by_differences(cuda):
    """d sum(y * dy) / d(x, a, b) along a direction, from two forward passes.  y is linear in
    each of x, a and b, so the difference quotient is exact but for rounding."""
    c = _case(31, 90, 128, 72, 16, 3)
    ids = _ids("mixed", 90, 3, c["g"])
    dy = _randn(c["g"], 90, 72)
    _, h = q.lora.lora_forward(c["x"], c["a"], c["b"], ids, c["s"], return_h=True)
    grads = q.lora.lora_backward(dy, c["x"], h, c["a"], c["b"], ids, c["s"], dx_dtype=F32,
                                 grad_dtype=F32)
    for name, grad in zip(("x", "a", "b"), grads):
        lo = dict(c)
        lo[name] = torch.zeros_like(c[name])
        d = _randn(c["g"], *c[name].shape)
        hi = dict(c)
        hi[name] = d                                     # y(d) - y(0): the derivative along d
        y = [q.lora.lora_forward(v["x"], v["a"], v["b"], ids, v["s"], out_dtype=F32).to(D)
             for v in (hi, lo)]
        quot = ((y[0] - y[1]) * dy.to(D)).sum()
        dot = (grad.to(D) * d.to(D)).sum()
        scale = ((y[0] - y[1]).abs() * dy.to(D).abs()).sum()
        assert abs(quot - dot) <= 2.0 ** -17 * 4 * scale


# ------------------------------------------------------------- in use: layers, streams, graphs

def test_layers_take_adapters(cuda):
    import numpy as np
    from gen import affine_weight, bf16_acts, fp4_weight, fp8_weight
    rng = np.random.default_rng(3)
    N, K, n = 256, 512, 3

    def d(v):
        return torch.from_numpy(np.ascontiguousarray(v)).cuda()

    w8, s8 = fp8_weight(rng, N, K)
    w4, s4 = fp4_weight(rng, N, K)
    wq, sc, bi = affine_weight(rng, N, K, 4)
    bf = lambda v: d(v.view(np.int16)).view(BF)               # noqa: E731
    layers = [q.linear.FP8Linear(d(w8), d(s8)), q.linear.FP4Linear(d(w4), d(s4)),
              q.linear.QuantizedLinear(d(wq.view(np.int32)), bf(sc), bf(bi))]
    for T in (1, 5, 200):
        c = _case(T, T, K, N, 16, n)
        bank = q.lora.LoRA(c["a"], c["b"], c["s"])
        ids = _ids("mixed", T, n, c["g"])
        x = bf(bf16_acts(rng, T, K)[0])
        for layer in layers:
            for odt in (None, F32):
                base = layer(x, out_dtype=odt)
                y = layer(x, out_dtype=odt, lora=bank, lora_ids=ids)
                assert y.dtype == base.dtype
                assert _eq(y, bank(x, ids, base=base))
                assert _eq(layer(x, out_dtype=odt), base)


def test_training_step_through_a_layer(cuda):
    """Forward through a frozen fp8 layer with adapters and the gradients of a squared loss,
    against autograd in float64 on the decoded weight."""
    import numpy as np
    from gen import fp8_weight
    rng = np.random.default_rng(8)
    T, K, N, R, n = 96, 256, 160, 8, 2
    w, s = (torch.from_numpy(v).cuda() for v in fp8_weight(rng, N, K, 116, 120))
    c = _case(77, T, K, N, R, n)
    ids = _ids("mixed", T, n, c["g"])
    layer, bank = q.linear.FP8Linear(w, s), q.lora.LoRA(c["a"], c["b"], c["s"])
    y, h = bank(c["x"], ids, base=layer(c["x"], out_dtype=F32), return_h=True)
    dy = (2 * y).to(BF)
    wd = q.dequant.dequant_fp8(w, s).to(D)
    dx, da, db = bank.backward(dy, c["x"], h, ids, dx_base=(dy.to(D) @ wd).to(BF))
    x64, a64, b64 = (c[k].to(D).requires_grad_(True) for k in ("x", "a", "b"))
    live = (ids >= 0).to(D)[:, None]
    i = ids.clamp(min=0).long()
    y64 = x64 @ wd.T + live * c["s"].to(D)[i][:, None] * torch.einsum(
        "tnr,tr->tn", b64[i], torch.einsum("trk,tk->tr", a64[i], x64))
    want = torch.autograd.grad(y64, (x64, a64, b64), dy.to(D))
    for g, w64 in zip((dx, da, db), want):
        # dx_base and the result are each rounded to bf16: two half steps of the norm
        assert (g.to(D) - w64).norm() <= 2 * 2.0 ** -8 * w64.norm()


def test_graph_replay_and_two_captures(cuda):
    """Captured calls replayed with new contents give the bits of eager calls, and two captured
    graphs replayed in turn and at once do not disturb each other."""
    cs = [_case(50 + i, T, 512, 256, 16, 4) for i, T in enumerate((7, 400))]
    graphs = []
    for c in cs:
        T = c["x"].shape[0]
        c["ids"] = _ids("mixed", T, 4, c["g"])
        c["dy"] = _randn(c["g"], T, 256)

        def step(c=c):
            y, h = q.lora.lora_forward(c["x"], c["a"], c["b"], c["ids"], c["s"], return_h=True)
            return (y, h) + q.lora.lora_backward(c["dy"], c["x"], h, c["a"], c["b"], c["ids"],
                                                 c["s"])
        step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step()
        graphs.append((g, outs, step))
    for rnd in range(3):
        for c in cs:
            T = c["x"].shape[0]
            c["x"].copy_(_randn(c["g"], T, 512))
            c["ids"].copy_(_ids(("mixed", "runs", "none")[rnd], T, 4, c["g"]))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for (g, _, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for g, outs, step in graphs:
            for o, w in zip(outs, step()):
                assert _eq(o, w)


def test_side_stream(cuda):
    c = _case(61, 300, 1024, 512, 32, 4)
    ids = _ids("mixed", 300, 4, c["g"])
    want = q.lora.lora_forward(c["x"], c["a"], c["b"], ids, c["s"])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [q.lora.lora_forward(c["x"], c["a"], c["b"], ids, c["s"]) for _ in range(4)]
    s.synchronize()
    assert all(_eq(v, want) for v in got)


@pytest.mark.parametrize("T, K, N, n, R, few", [
    (1, 7168, 4096, 8, 16, True), (64, 7168, 4096, 32, 16, True), (8, 7168, 14336, 4, 64, True),
    (24, 7168, 14336, 4, 128, False), (384, 4096, 4096, 4, 32, False)], ids=str)
def test_few_token_form_where_it_is_faster(cuda, T, K, N, n, R, few):
    """The one-launch form (no workspace) at sizes where the other takes 1.4 times as long or more,
    and the other way round; either gives the formula."""
    nb = L.load().dsv41_lora_workspace_size(T, K, N, n, R, 0)
    assert (nb == 0) == few
    c = _case(T + R, T, K, N, R, n)
    ids = _ids("mixed", T, n, c["g"])
    y, h = q.lora.lora_forward(c["x"], c["a"], c["b"], ids, c["s"], return_h=True)
    _check_forward(c, ids, None, BF, y, h)


def test_every_launch_is_counted(cuda):
    """The launches that dsv41_prof_launches counts are the kernels that a call launches."""
    def launches(fn):
        fn()
        L.prof_enable(True)
        fn()
        torch.cuda.synchronize()
        report = {k: v[0] for k, v in L.prof_report().items()}
        n = L.prof_launches()
        L.prof_enable(False)
        assert n == sum(report.values())
        return report
    c = _case(71, 3000, 264, 136, 16, 3)
    ids = _ids("mixed", 3000, 3, c["g"])
    dy, h = _randn(c["g"], 3000, 136), _randn(c["g"], 3000, 16, dtype=F32)
    one = dict.fromkeys
    assert launches(lambda: q.lora.lora_forward(c["x"][:4], c["a"], c["b"], ids[:4])) == \
        one(["lora_decode"], 1)
    assert launches(lambda: q.lora.lora_forward(c["x"], c["a"], c["b"], ids)) == \
        one(["lora_plan", "lora_shrink", "lora_expand"], 1)
    assert launches(lambda: q.lora.lora_backward(dy, c["x"], h, c["a"], c["b"], ids)) == \
        one(["lora_plan", "lora_shrink", "lora_wgrad", "lora_join", "lora_expand"], 1)
    for T, names in ((64, ["balance"]), (5000, ["balance_count", "balance"]),
                     (20000, ["balance_zero", "balance_count", "balance"])):
        z = torch.zeros(T, 64, device="cuda")
        idx = torch.zeros(T, 4, dtype=torch.int32, device="cuda")
        assert launches(lambda: q.moe.balance_loss(z, idx, grad_loss=1.0)) == one(names, 1)


def test_no_tokens(cuda):
    c = _case(70, 0, 64, 40, 8, 3)
    ids = torch.empty(0, dtype=torch.int32, device="cuda")
    y, h = q.lora.lora_forward(c["x"], c["a"], c["b"], ids, c["s"], return_h=True)
    assert y.shape == (0, 40) and h.shape == (0, 8)
    dx, da, db = q.lora.lora_backward(y, c["x"], h, c["a"], c["b"], ids, c["s"])
    assert dx.shape == (0, 64) and (da == 0).all() and (db == 0).all()


def test_refusals(cuda):
    c = _case(80, 4, 64, 32, 8, 2)
    x, a, b, s = c["x"], c["a"], c["b"], c["s"]
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    f = q.lora.lora_forward
    base = torch.zeros(4, 32, device="cuda")
    for bad in (lambda: f(x[:, :56], a, b, ids), lambda: f(x, a, b, ids[:3]),
                lambda: f(x, a.float(), b, ids), lambda: f(x, a, b[:1], ids),
                lambda: f(x, a, b, ids.float()), lambda: f(x, a, b, ids, s[:1]),
                lambda: f(x, a, b, ids, s.double()), lambda: f(x, a, b, ids, s, base, BF),
                lambda: f(x, a, b, ids, s, base[:3]),
                lambda: f(x, a, b, ids, out=torch.zeros(32, 4, device="cuda").T),
                lambda: f(x, a, b, ids, out_dtype=torch.float16),
                lambda: f(x[:, :60].contiguous(), a[..., :60].contiguous(), b, ids)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(q.DSV41Error):                       # rank 12
        f(x, torch.zeros(2, 12, 64, dtype=BF, device="cuda"),
          torch.zeros(2, 32, 12, dtype=BF, device="cuda"), ids)
    with pytest.raises(q.DSV41Error):                       # rank 136
        f(x, torch.zeros(2, 136, 64, dtype=BF, device="cuda"),
          torch.zeros(2, 32, 136, dtype=BF, device="cuda"), ids)
    with pytest.raises(q.DSV41Error):
        f(x.cpu(), a, b, ids)
    dy, h = torch.zeros(4, 32, dtype=BF, device="cuda"), torch.zeros(4, 8, device="cuda")
    g = q.lora.lora_backward
    for bad in (lambda: g(dy.float(), x, h, a, b, ids), lambda: g(dy, x, h.to(BF), a, b, ids),
                lambda: g(dy[:3], x, h, a, b, ids), lambda: g(dy, x, h[:, :4], a, b, ids),
                lambda: g(dy, x, h, a, b, ids, dx_base=torch.zeros(4, 32, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(ValueError):                         # an unaligned view
        flat = torch.zeros(4 * 64 + 1, dtype=BF, device="cuda")
        f(flat[1:].view(4, 64), a, b, ids)
