"""Low-rank adapters of many requests at once beside a shared projection (csrc/adapter.hip; no
counterpart in the reference): one frozen table -- the entity table of a trained model, or any
[m, d] map -- serves many clients, domains or relations, each with a small correction of its own.

    y_i = W x_i + scales_t B_t (A_t x_i),   t = ids[i]             (t = -1: no adapter)

``adapted_projection`` is the operator, differentiable in x, a and b (W stays frozen);
``LowRankAdapters`` holds the parameters; ``KgeModel.score_sp_adapted`` / ``score_po_adapted`` score
queries against all entities with it.  fp32 tables use the fp32 matrix instruction, bf16 tables the bf16 one;
sums are fp32 in both, results are rounded once.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib as L
from .label_losses import _capturing, first_order, is_on_current_device, on_device_of

MAX_RANK = 1024
FEW = 32  # rows that take the path for few requests, which needs no workspace (the C entry has the same number)


def _matrix(t: torch.Tensor) -> torch.Tensor:
    """[rows, cols] with unit column stride and rows that do not overlap."""
    if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
    return t


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _padded(rows: int, cols: int, like: torch.Tensor) -> torch.Tensor:
    """[rows, cols] whose rows start on 16 bytes.  No view of a wider buffer: a Function's output that is a view
    cannot be changed in place (known answers masked with -inf)."""
    per = 16 // like.element_size()
    return like.new_empty_strided((rows, cols), ((cols + per - 1) // per * per, 1))


def _forward(x, w, a, b, ids, scales, for_backward):
    """(y, what the backward pass needs)"""
    n, d = x.shape
    k, m, r = b.shape
    y = _padded(n, m, x)
    lib, dtype = L.lib(), L.DTYPES[x.dtype]
    size = lib.kge_adapter_save_size(n, d, k, r)
    save = torch.empty(size, device=x.device, dtype=torch.uint8)
    ws, ws_size = None, 0
    if for_backward or n > FEW:
        ws_size = lib.kge_adapter_forward_ws_size(dtype, n, d, m, k, r, for_backward)
        if ws_size:
            ws = torch.empty(ws_size, device=x.device, dtype=torch.uint8)
    L._check(lib.kge_adapter_forward(
        x.data_ptr(), dtype, _ld(x), n, d, w.data_ptr(), _ld(w), m, a.data_ptr(), b.data_ptr(), k, r, ids.data_ptr(),
        L.ptr(scales), y.data_ptr(), _ld(y), save.data_ptr(), size, for_backward, L.ptr(ws), ws_size, L.stream()),
        "kge_adapter_forward")
    return y, save


class _AdaptedProjection(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, a, b, ids, scales):
        y, save = _forward(x, w, a, b, ids, scales, True)
        ctx.save_for_backward(x, w, a, b, scales, save)
        return y

    @first_order
    def backward(ctx, dy):
        if not is_on_current_device(dy):
            with torch.cuda.device(dy.get_device()):
                return _gradients(ctx, dy)
        return _gradients(ctx, dy)


def _gradients(ctx, dy):
    x, w, a, b, scales, save = ctx.saved_tensors
    n, d = x.shape
    k, m, r = b.shape
    want_x, _, want_a, want_b, _, _ = ctx.needs_input_grad
    dy = _matrix(dy)
    dx, da, db = dx_at, da_at, db_at = None, None, None
    ldx = d
    if want_x:
        dx = _padded(n, d, x)
        dx_at, ldx = dx.data_ptr(), _ld(dx)
    if want_a:
        da = torch.empty_like(a)
        da_at = da.data_ptr()
    if want_b:
        db = torch.empty_like(b)
        db_at = db.data_ptr()
    lib, dtype = L.lib(), L.DTYPES[x.dtype]
    size = lib.kge_adapter_backward_ws_size(dtype, n, d, m, k, r, want_x, want_a, want_b)
    ws = torch.empty(size, device=x.device, dtype=torch.uint8)
    status = lib.kge_adapter_backward(
        dy.data_ptr(), dtype, _ld(dy), n, m, x.data_ptr(), _ld(x), d, w.data_ptr(), _ld(w), a.data_ptr(), b.data_ptr(),
        k, r, None if scales is None else scales.data_ptr(), save.data_ptr(), save.numel(), dx_at, ldx, da_at, db_at,
        ws.data_ptr(), size, L.stream())
    if status:
        L._check(status, "kge_adapter_backward")
    return dx, None, da, db, None, None


def _as_they_are(x, w, a, b, ids, scales) -> bool:
    """Whether the arguments are what the kernels take, with nothing to convert or to refuse (the usual case, seen
    with few tensor accesses: a serving call is launch-bound); otherwise _checked says what is wrong."""
    if L.CHECK_INDEX:
        return False
    dtype, dev, bs = x.dtype, x.get_device(), b.shape
    if (dtype not in (torch.bfloat16, torch.float32) or w.dtype is not dtype or a.dtype is not dtype
            or b.dtype is not dtype or len(bs) != 3 or w.get_device() != dev or a.get_device() != dev or b.get_device() != dev
            or ids.get_device() != dev or ids.dtype is not torch.int64):
        return False
    k, m, r = bs
    if len(a.shape) != 3 or len(x.shape) != 2:
        return False
    n, d = x.shape
    if scales is not None and not (scales.dtype is torch.float32 and scales.shape == (k,) and scales.get_device() == dev
                                   and scales.is_contiguous() and not scales.requires_grad):
        return False
    return (w.shape == (m, d) and a.shape == (k, r, d) and ids.shape == (n,) and min(d, m, k) >= 1 and 1 <= r <= MAX_RANK
            and not w.requires_grad and x.is_contiguous() and w.is_contiguous() and a.is_contiguous()
            and b.is_contiguous() and ids.is_contiguous())


def _checked(x, w, a, b, ids, scales):
    """The arguments as the kernels take them, or an error that says what is wrong."""
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"x: expected float32 or bfloat16, got {x.dtype}")
    dtype, dev = x.dtype, x.get_device()  # (-1: CPU)
    for t, dim, what in ((x, 2, "x [n, d]"), (w, 2, "w [m, d]"), (a, 3, "a [k, r, d]"), (b, 3, "b [k, m, r]")):
        if t.dim() != dim or t.dtype != dtype:
            raise ValueError(f"{what}: expected {dim} dimensions of {dtype}, got {list(t.shape)} {t.dtype}")
        if t.get_device() != dev:
            raise ValueError(f"{what}: on {t.device}, x is on {x.device}")
    (n, d), m, (k, r) = x.shape, w.shape[0], a.shape[:2]
    if w.shape[1] != d or a.shape[2] != d or tuple(b.shape) != (k, m, r):
        raise ValueError(f"x {list(x.shape)}, w {list(w.shape)}, a {list(a.shape)}, b {list(b.shape)}: expected "
                         "[n, d], [m, d], [k, r, d], [k, m, r]")
    if min(d, m, k) < 1 or not 1 <= r <= MAX_RANK:
        raise ValueError(f"d={d}, m={m}, k={k}, r={r}: expected at least 1 each, ranks up to {MAX_RANK}")
    if w.requires_grad and torch.is_grad_enabled():
        raise ValueError("w: the shared projection is frozen, pass it detached")
    if ids.dim() != 1 or ids.numel() != n or ids.is_floating_point() or ids.dtype == torch.bool:
        raise ValueError(f"ids: expected {n} integers, got {list(ids.shape)} {ids.dtype}")
    if scales is not None:
        if scales.dim() != 1 or scales.numel() != k or not scales.is_floating_point():
            raise ValueError(f"scales: expected {k} floating point numbers, got {list(scales.shape)} {scales.dtype}")
        if scales.requires_grad and torch.is_grad_enabled():
            raise ValueError("scales: no gradient flows into them, pass them detached")
        scales = scales.detach().to(torch.float32).contiguous()
    for t, what in ((ids, "ids"), (scales, "scales")):
        if t is not None and t.get_device() != dev:
            raise ValueError(f"{what}: on {t.device}, x is on {x.device}")
    ids = L.idx64(ids)
    if L.CHECK_INDEX and n > 0 and not _capturing():
        lo, hi = int(ids.min()), int(ids.max())
        if lo < -1 or hi >= k:
            raise IndexError(f"adapter id: out of range [{lo}, {hi}] for {k} adapters (-1: none)")
    return _matrix(x), _matrix(w), a.contiguous(), b.contiguous(), ids, scales


def adapted_projection(x: torch.Tensor, w: torch.Tensor, a: torch.Tensor, b: torch.Tensor, ids: torch.Tensor,
                       scales: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y [n, m]: y_i = w x_i + scales[t] b[t] (a[t] x_i) for t = ids[i], y_i = w x_i for ids[i] = -1.

    x [n, d] requests in any order, w [m, d] shared and frozen (pass it detached), a [k, r, d] and
    b [k, m, r] the adapters (ranks below r: padded with zeros), scales [k] (None: 1), all of one type, fp32
    or bf16 (scales in any floating type, used in fp32).  Differentiable in x, a and b."""
    if not _as_they_are(x, w, a, b, ids, scales):
        x, w, a, b, ids, scales = _checked(x, w, a, b, ids, scales)
    L.require_device(x)
    with on_device_of(x):
        if torch.is_grad_enabled() and (x.requires_grad or a.requires_grad or b.requires_grad):
            return _AdaptedProjection.apply(x, w, a, b, ids, scales)
        return _forward(x, w, a, b, ids, scales, False)[0]


class LowRankAdapters(torch.nn.Module):
    """k adapters of rank r beside a [num_out, num_in] projection: ``a`` starts as N(0, 1 / num_in), ``b``
    as zeros, so that a new adapter changes nothing.  ``alpha``: scales = alpha / r."""

    def __init__(self, num_adapters: int, rank: int, num_in: int, num_out: int, alpha: Optional[float] = None,
                 device=None, dtype=torch.float32):
        super().__init__()
        if min(num_adapters, num_in, num_out) < 1 or not 1 <= rank <= MAX_RANK:
            raise ValueError(f"num_adapters={num_adapters}, rank={rank}, num_in={num_in}, num_out={num_out}: expected "
                             f"at least 1 each, ranks up to {MAX_RANK}")
        a = torch.randn(num_adapters, rank, num_in, device=device).mul_(num_in ** -0.5)
        self.a = torch.nn.Parameter(a.to(dtype))
        self.b = torch.nn.Parameter(torch.zeros(num_adapters, num_out, rank, device=device, dtype=dtype))
        scale = 1.0 if alpha is None else float(alpha) / rank
        self.register_buffer("scales", torch.full((num_adapters,), scale, device=device, dtype=torch.float32))

    def forward(self, x: torch.Tensor, w: torch.Tensor, ids: torch.Tensor) -> torch.Tensor:
        return adapted_projection(x, w, self.a, self.b, ids, self.scales)
