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

Tensors are taken as values: a result has no autograd history, even where an input requires a
gradient; ``lora_backward`` is the gradient.  x, a, b, dy and h must start on 16 bytes (views that
do not are refused); base, out and dx_base may start anywhere.  An infinity in x, a, b or dy makes
the elements whose sums it enters infinite or NaN, and no others.
"""

from __future__ import annotations

import functools

from . import _lib as L


@functools.lru_cache(maxsize=1024)
def _workspace_size(device, T, K, N, n, R, backward):
    # (by device too: the grids follow its number of SMs)
    with L.torch().cuda.device(device):
        return L.load().dsv41_lora_workspace_size(T, K, N, n, R, backward)


def _tensor(v, name, dtype, device):
    """v as a contiguous CUDA tensor of ``dtype`` on ``device``."""
    if type(v) is L.torch().Tensor and v.dtype is dtype and v.device == device \
            and v.is_contiguous():
        return v
    v = L.cuda_tensor(v, name)
    if v.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, not {v.dtype}")
    if v.device != device:
        raise ValueError(f"{name} is on {v.device}, x on {device}")
    return v


def _operands(x, a, b, ids, scaling):
    """x bf16, the bank, the ids int32, the device and the sizes T, K, N, n, R."""
    t = L.torch()
    if ids is None:
        raise ValueError("ids must name the adapter of each token (negative: none)")
    x = L.cuda_tensor(x, "x")
    if x.dtype != t.bfloat16:
        x = x.to(t.bfloat16)
    dev = x.device
    a, b = _tensor(a, "a", t.bfloat16, dev), _tensor(b, "b", t.bfloat16, dev)
    sa, sb = a.shape, b.shape
    if len(sa) != 3 or len(sb) != 3 or sa[0] != sb[0] or sa[1] != sb[2]:
        raise ValueError("a must be [n, R, K] and b [n, N, R]")
    n, R, K = sa
    if scaling is not None:
        scaling = _tensor(scaling, "scaling", t.float32, dev)
        if scaling.shape != (n,):
            raise ValueError("scaling must be float32 [n]")
    if x.dim() == 0 or x.shape[-1] != K or K == 0:
        raise ValueError(f"x must be [..., {K}]")
    T = x.numel() // K
    if ids.dtype is t.int64:             # ids that int32 cannot hold are no adapter's
        ids = L.as_tensor(ids).clamp(-1, 0x7FFFFFFF).to(t.int32)
    ids = _tensor(ids, "ids", t.int32, dev)
    if ids.numel() != T:
        raise ValueError(f"ids must name the adapter of each of the {T} tokens")
    return x, a, b, ids, scaling, dev, T, K, sb[1], n, R


def _rows(v, name, rows, cols, dtype, device):
    """[..., cols] with ``rows`` rows, or None."""
    if v is None:
        return None
    v = _tensor(v, name, dtype, device)
    if v.numel() != rows * cols or v.shape[-1] != cols:
        raise ValueError(f"{name} must be [..., {cols}] with {rows} rows")
    return v


def _code(dtype):
    t = L.torch()
    if dtype == t.bfloat16:
        return L.BF16
    if dtype == t.float32:
        return L.F32
    raise ValueError("output dtypes must be float32 or bfloat16")


def lora_forward(x, a, b, ids, scaling=None, base=None, out_dtype=None, out=None,
                 return_h=False):
    """``base + scaling[i] * (x @ a[i].T) @ b[i].T`` row by row, i = ids[row].

    x [..., K] bf16 (other dtypes are converted), base [..., N] of the output's dtype or None;
    ``out`` (may be ``base`` itself) receives the result.  ``out_dtype`` defaults to base's or
    out's dtype, else bf16.  With ``return_h`` also h = x @ a[i].T, float32 [..., R], which
    ``lora_backward`` takes."""
    t = L.torch()
    x, a, b, ids, scaling, dev, T, K, N, n, R = _operands(x, a, b, ids, scaling)
    lead = x.shape[:-1]
    like = base if base is not None else out
    odt = out_dtype or (t.bfloat16 if like is None else like.dtype)
    code = _code(odt)
    base = _rows(base, "base", T, N, odt, dev)
    if out is None:
        if base is not None and base.shape[:-1] == lead:
            out = t.empty_like(base)
        else:
            out = x.new_empty(lead + (N,), dtype=odt)
    elif _rows(out, "out", T, N, odt, dev) is not out:
        raise ValueError("out must be a contiguous CUDA tensor")
    h = x.new_empty(lead + (R,), dtype=t.float32) if return_h else None
    nb = _workspace_size(dev, T, K, N, n, R, 0)
    ws = L.workspace(nb, dev) if nb else None
    L.call_on(dev, "dsv41_lora_forward", x.data_ptr(), T, K, a.data_ptr(), b.data_ptr(), n, R, N,
              L.ptr(scaling), ids.data_ptr(), L.ptr(base), code, out.data_ptr(), L.ptr(h),
              L.ptr(ws), nb, L.stream_of(x))
    return (out, h) if return_h else out


def lora_backward(dy, x, h, a, b, ids, scaling=None, dx_base=None, dx_dtype=None,
                  grad_dtype=None):
    """Gradients (dx, da, db) of ``lora_forward`` from dy [..., N] bf16.

    h float32 [..., R] is what the forward pass returned (``return_h``).  dx_base [..., K] (the
    projection's own gradient, of dx's dtype) is added to dx; dx_dtype defaults to dx_base's
    dtype, else bf16.  da [n, R, K] and db [n, N, R] are ``grad_dtype`` (default: a's) and whole:
    zeros for adapters without tokens.  base's gradient is dy itself."""
    t = L.torch()
    x, a, b, ids, scaling, dev, T, K, N, n, R = _operands(x, a, b, ids, scaling)
    dy = _rows(dy, "dy", T, N, t.bfloat16, dev)
    h = _rows(h, "h", T, R, t.float32, dev)
    xdt = dx_dtype or (t.bfloat16 if dx_base is None else dx_base.dtype)
    gdt = grad_dtype or t.bfloat16
    xcode, gcode = _code(xdt), _code(gdt)
    dx_base = _rows(dx_base, "dx_base", T, K, xdt, dev)
    dx = t.empty_like(x, dtype=xdt)
    da, db = t.empty_like(a, dtype=gdt), t.empty_like(b, dtype=gdt)
    nb = _workspace_size(dev, T, K, N, n, R, 1)
    ws = L.workspace(nb, dev) if nb else None
    L.call_on(dev, "dsv41_lora_backward", dy.data_ptr(), x.data_ptr(), h.data_ptr(), a.data_ptr(),
              b.data_ptr(), T, K, N, n, R, L.ptr(scaling), ids.data_ptr(), L.ptr(dx_base), xcode,
              dx.data_ptr(), gcode, da.data_ptr(), db.data_ptr(), L.ptr(ws), nb, L.stream_of(x))
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
