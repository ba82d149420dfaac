"""Low-rank adapters of many requests beside one shared projection.

A bank holds ``n`` adapters of one projection [N, K]: ``a`` bf16 [n, R, K], ``b`` bf16 [n, N, R]
and ``scaling`` f32 [n].  Every token names its adapter (``ids`` int32; negative: none), so one
call serves a batch whose requests use different adapters, or none:

    y[t] = base[t] + scaling[i] * (x[t] @ a[i].T) @ b[i].T        i = ids[t]

``lora_forward`` adds the adapters' part to the projection's output (``base``), ``lora_backward``
gives the gradients of x, a and b for training them beside frozen weights.  ``LoRA`` is a bank as
an object; the layers of ``linear`` take one (``FP8Linear(...)(x, lora=bank, lora_ids=ids)``).
The rank is a multiple of 8 up to 128 (pad a and b with zeros to mix ranks in one bank), K a
multiple of 8.  Ids at or past n count as none and raise bit 1 of ``dsv41_device_status``.
"""

from __future__ import annotations

from . import _lib as L


def _bank(a, b, scaling, device):
    t = L.torch()
    a, b = L.cuda_tensor(a, "a"), L.cuda_tensor(b, "b")
    if a.dtype != t.bfloat16 or b.dtype != t.bfloat16:
        raise ValueError("a and b must be bfloat16")
    if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2]:
        raise ValueError("a must be [n, R, K] and b [n, N, R]")
    if scaling is not None:
        scaling = L.cuda_tensor(scaling, "scaling")
        if scaling.dtype != t.float32 or tuple(scaling.shape) != (a.shape[0],):
            raise ValueError("scaling must be float32 [n]")
    _same_device(device, a=a, b=b, scaling=scaling)
    return a, b, scaling


def _same_device(device, **tensors):
    for name, v in tensors.items():
        if v is not None and v.device != device:
            raise ValueError(f"{name} is on {v.device}, x on {device}")


def _ids(ids, T, device):
    t = L.torch()
    ids = L.cuda_tensor(ids, "ids")
    if ids.dtype not in (t.int32, t.int64):
        raise ValueError("ids must be int32 (or int64)")
    if ids.numel() != T:
        raise ValueError(f"ids must name the adapter of each of the {T} tokens")
    _same_device(device, ids=ids)
    # ids that int32 cannot hold are no adapter's
    return ids if ids.dtype == t.int32 else ids.clamp(-1, 0x7FFFFFFF).to(t.int32)


def _addend(v, name, shape, dtype, device):
    """base / dx_base: any leading shape, the output's rows."""
    if v is None:
        return None
    v = L.cuda_tensor(v, name)
    if v.numel() != shape[0] * shape[1] or v.shape[-1] != shape[1]:
        raise ValueError(f"{name} must be [..., {shape[1]}] with {shape[0]} rows")
    if v.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, the output's dtype")
    _same_device(device, **{name: v})
    return v


def _odt(dtype, default):
    t = L.torch()
    dtype = dtype or default
    if dtype not in (t.float32, t.bfloat16):
        raise ValueError("output dtypes must be float32 or bfloat16")
    return dtype


def lora_forward(x, a, b, ids, scaling=None, base=None, out_dtype=None, out=None,
                 return_h=False):
    """``base + scaling[i] * (x @ a[i].T) @ b[i].T`` row by row, i = ids[row].

    x [..., K] bf16 (other dtypes are converted), base [..., N] of the output's dtype or None;
    ``out`` (may be ``base`` itself) receives the result.  ``out_dtype`` defaults to base's or
    out's dtype, else bf16.  With ``return_h`` also h = x @ a[i].T, float32 [..., R], which
    ``lora_backward`` takes."""
    t = L.torch()
    x = L.cuda_tensor(x, "x")
    if x.dtype != t.bfloat16:
        x = x.to(t.bfloat16)
    dev = x.device
    a, b, scaling = _bank(a, b, scaling, dev)
    n, R, K = a.shape
    N = b.shape[1]
    if x.shape[-1] != K:
        raise ValueError(f"x must be [..., {K}]")
    T = x.numel() // K
    ids = _ids(ids, T, dev)
    like = base if base is not None else out
    odt = _odt(out_dtype, t.bfloat16 if like is None else like.dtype)
    base = _addend(base, "base", (T, N), odt, dev)
    lead = tuple(x.shape[:-1])
    if out is None:
        y = t.empty(lead + (N,), dtype=odt, device=dev)
    else:
        y = out
        if not (isinstance(y, t.Tensor) and y.is_contiguous()
                and _addend(y, "out", (T, N), odt, dev) is y):
            raise ValueError("out must be a contiguous CUDA tensor")
    h = t.empty(lead + (R,), dtype=t.float32, device=dev) if return_h else None
    with L.on(dev):
        nb = L.load().dsv41_lora_workspace_size(T, K, N, n, R, 0)
        ws = L.workspace(nb, dev)
        L.call("dsv41_lora_forward", L.ptr(x), T, K, L.ptr(a), L.ptr(b), n, R, N, L.ptr(scaling),
               L.ptr(ids), L.ptr(base), L.dtype_code(odt), L.ptr(y), L.ptr(h), L.ptr(ws), nb,
               L.stream_of(x))
    return (y, h) if return_h else y


def lora_backward(dy, x, h, a, b, ids, scaling=None, dx_base=None, dx_dtype=None,
                  grad_dtype=None):
    """Gradients (dx, da, db) of ``lora_forward`` from dy [..., N] bf16.

    h float32 [..., R] is what the forward pass returned (``return_h``).  dx_base [..., K] (the
    projection's own gradient, of dx's dtype) is added to dx; dx_dtype defaults to dx_base's
    dtype, else bf16.  da [n, R, K] and db [n, N, R] are ``grad_dtype`` (default: a's) and whole:
    zeros for adapters without tokens.  base's gradient is dy itself."""
    t = L.torch()
    x, dy, h = L.cuda_tensor(x, "x"), L.cuda_tensor(dy, "dy"), L.cuda_tensor(h, "h")
    dev = x.device
    if x.dtype != t.bfloat16:
        x = x.to(t.bfloat16)
    if dy.dtype != t.bfloat16:
        raise ValueError("dy must be bfloat16")
    if h.dtype != t.float32:
        raise ValueError("h must be float32, as lora_forward returns it")
    a, b, scaling = _bank(a, b, scaling, dev)
    n, R, K = a.shape
    N = b.shape[1]
    if x.shape[-1] != K:
        raise ValueError(f"x must be [..., {K}]")
    T = x.numel() // K
    if dy.shape[-1] != N or dy.numel() != T * N or h.shape[-1] != R or h.numel() != T * R:
        raise ValueError("dy must be [..., N] and h [..., R] for x's tokens")
    _same_device(dev, dy=dy, h=h)
    ids = _ids(ids, T, dev)
    xdt = _odt(dx_dtype, t.bfloat16 if dx_base is None else dx_base.dtype)
    gdt = _odt(grad_dtype, a.dtype)
    dx_base = _addend(dx_base, "dx_base", (T, K), xdt, dev)
    dx = t.empty(x.shape, dtype=xdt, device=dev)
    da = t.empty(a.shape, dtype=gdt, device=dev)
    db = t.empty(b.shape, dtype=gdt, device=dev)
    with L.on(dev):
        nb = L.load().dsv41_lora_workspace_size(T, K, N, n, R, 1)
        ws = L.workspace(nb, dev)
        L.call("dsv41_lora_backward", L.ptr(dy), L.ptr(x), L.ptr(h), L.ptr(a), L.ptr(b), T, K, N,
               n, R, L.ptr(scaling), L.ptr(ids), L.ptr(dx_base), L.dtype_code(xdt), L.ptr(dx),
               L.dtype_code(gdt), L.ptr(da), L.ptr(db), L.ptr(ws), nb, L.stream_of(x))
    return dx, da, db


class LoRA:
    """A bank of adapters for one projection: a bf16 [n, R, K], b bf16 [n, N, R], scaling f32
    [n] (None: 1)."""

    def __init__(self, a, b, scaling=None):
        self.a, self.b, self.scaling = a, b, scaling

    def __call__(self, x, ids, base=None, out_dtype=None, out=None, return_h=False):
        return lora_forward(x, self.a, self.b, ids, self.scaling, base, out_dtype, out, return_h)

    def backward(self, dy, x, h, ids, dx_base=None, dx_dtype=None, grad_dtype=None):
        return lora_backward(dy, x, h, self.a, self.b, ids, self.scaling, dx_base, dx_dtype,
                             grad_dtype)
