"""The library's stand-alone operators (include/vtc_amd.h, "Operators") on torch tensors.

Rotary positions, group norm with an activation on channel-last rows and the gated feed-forward block: what an encoder variant
(VtcEngine(variant=...)) runs inside the library, for callers that run such layers themselves or adapt them to new recordings.
Every function launches on the current stream of its tensors' device and neither synchronises nor copies to the host.

Each operator has explicit forward and backward calls (`*_forward`, `*_backward`, `inverse=True`) and, where that is handier, a
differentiable one (`rotary`, `rotary_qk`, `group_norm_act`, `gated_ffn`) whose gradient is those calls.  A program that captures
a training step into a graph uses the explicit ones, or makes the differentiable call inside the capture as well.
"""

from __future__ import annotations

import ctypes as C
import math

import numpy as np
import torch

from . import lib as L

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
ACTS = {"none": 0, "gelu": 1, "silu": 2, "sigmoid": 3}
LAYOUTS = {"half": 0, "interleaved": 1}
SCALINGS = ("none", "linear", "ntk", "by_parts")


def _need_gpu(x: torch.Tensor, what: str) -> int:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{what}: expected a tensor, got {type(x).__name__}")
    if x.device.type != "cuda":
        raise ValueError(f"{what}: tensors must be on a ROCm GPU (there is no CPU path), got {x.device}")
    return x.device.index


def _same(what: str, x: torch.Tensor, **others) -> None:
    for name, t in others.items():
        if t is not None and (t.device != x.device or t.dtype != x.dtype):
            raise ValueError(f"{what}: {name} is {t.dtype} on {t.device}, expected {x.dtype} on {x.device}")


def _dtype(x: torch.Tensor, what: str, allowed=(torch.float32, torch.float16, torch.bfloat16)) -> int:
    if x.dtype not in allowed:
        raise ValueError(f"{what}: type {x.dtype} is not one of {', '.join(str(a) for a in allowed)}")
    return _DTYPES[x.dtype]


def _stream(device) -> C.c_void_p:
    return C.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _ptr(t) -> C.c_void_p:
    return C.c_void_p(0 if t is None else t.data_ptr())


def _workspace(n: int, device) -> torch.Tensor:
    # the allocator's blocks start at multiples of 512 bytes; inside a graph capture they come from the graph's own pool
    return torch.empty(max(int(n), 1), dtype=torch.uint8, device=device)


# ------------------------------------------------------------------------------------------------ rotary positions
class Rotary:
    """What a rotation is: pairs of the first `rotary_dim` elements of a head (all of them by default, see rotary()), their layout
    ("half": j with j + rotary_dim / 2; "interleaved": 2j with 2j + 1) and their angular frequencies, base ** (-2 j / rotary_dim)
    unless scaled for positions beyond those a model was trained on:

    "linear":   frequency / factor
    "ntk":      base * factor ** (rotary_dim / (rotary_dim - 2)) in place of base
    "by_parts": pairs that turn more than 32 times over `original_length` positions keep their frequency, those that turn less
                than once are divided by `factor`, between them a ramp linear in the pair's index; the result is multiplied by
                1 + 0.1 ln(factor)

    Frequencies are 64-bit; `frequency` and `amplitude` may be replaced by the caller's own."""

    def __init__(self, rotary_dim: int, layout: str = "half", base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                 original_length: int = 0):
        r, s = int(rotary_dim), float(factor)
        if r < 2 or r % 2 or r > 512:
            raise ValueError(f"rotary_dim must be even and in 2..512, got {rotary_dim}")
        if layout not in LAYOUTS:
            raise ValueError(f"layout must be one of {list(LAYOUTS)}, got {layout!r}")
        if scaling not in SCALINGS:
            raise ValueError(f"scaling must be one of {list(SCALINGS)}, got {scaling!r}")
        if not (base > 1.0 and math.isfinite(base)) or not (s > 0.0 and math.isfinite(s)):
            raise ValueError("base must be above 1 and factor above 0, both finite")
        if scaling == "by_parts" and original_length < 1:
            raise ValueError("by_parts scaling needs original_length")
        self.rotary_dim, self.layout = r, layout
        j = np.arange(r // 2, dtype=np.float64)
        self.amplitude = 1.0
        if scaling == "ntk":
            base = base * s ** (r / max(r - 2, 1))
        f = float(base) ** (-2.0 * j / r)
        if scaling == "linear":
            f = f / s
        elif scaling == "by_parts":
            def index(turns):   # the pair that turns this often over the original length
                return r * math.log(original_length / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))
            low, high = max(math.floor(index(32.0)), 0), min(math.ceil(index(1.0)), r // 2 - 1)
            ramp = np.clip((j - low) / max(high - low, 1e-3), 0.0, 1.0)
            f = f / s * ramp + f * (1.0 - ramp)
            self.amplitude = 0.1 * math.log(s) + 1.0 if s > 1.0 else 1.0
        self.frequency = np.ascontiguousarray(f)

    def _struct(self, head_dim: int):
        f = np.ascontiguousarray(self.frequency, dtype=np.float64)
        if f.shape != (self.rotary_dim // 2,):
            raise ValueError(f"frequency must have {self.rotary_dim // 2} entries, got shape {f.shape}")
        s = L.VtcRotary(head_dim=head_dim, rotary_dim=self.rotary_dim, layout=LAYOUTS[self.layout], amplitude=float(self.amplitude),
                        frequency=f.ctypes.data_as(L._f64p))
        return s, f   # f has to live until the call returns


def _rotary_call(tensors, spec: Rotary, positions, offset: int, inverse: bool, outs):
    x0 = tensors[0]
    index = _need_gpu(x0, "rotary")
    dt = _dtype(x0, "rotary")
    if not isinstance(spec, Rotary):
        raise TypeError("rotary: expected a Rotary")
    if x0.dim() not in (3, 4):
        raise ValueError(f"rotary: tensors are (batch, length, heads, head_dim) or (length, heads, head_dim), got {tuple(x0.shape)}")
    batch, length = (x0.shape[0], x0.shape[1]) if x0.dim() == 4 else (1, x0.shape[0])
    head_dim = x0.shape[-1]
    if spec.rotary_dim > head_dim:
        raise ValueError(f"rotary: rotary_dim {spec.rotary_dim} is more than head_dim {head_dim}")
    arr = (L.VtcHeads * len(tensors))()
    given = outs
    outs = []
    for i, x in enumerate(tensors):
        _same("rotary", x0, tensor=x)
        if x.dim() != x0.dim() or x.shape[:-2] != x0.shape[:-2] or x.shape[-1] != head_dim:
            raise ValueError(f"rotary: shapes {tuple(x0.shape)} and {tuple(x.shape)} do not go together")
        if x.numel() and x.stride(-1) != 1:
            raise ValueError("rotary: the elements of a head must be contiguous")
        y = given[i] if given is not None else None
        if y is None:
            y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        else:
            _same("rotary", x0, out=y)
            if y.shape != x.shape or (y.numel() and y.stride(-1) != 1):
                raise ValueError(f"rotary: out must have shape {tuple(x.shape)} with contiguous heads, got {tuple(y.shape)}")
        outs.append(y)
        sx = ((0,) if x.dim() == 3 else ()) + x.stride()
        sy = ((0,) if y.dim() == 3 else ()) + y.stride()
        arr[i] = L.VtcHeads(x=x.data_ptr(), y=y.data_ptr(), x_batch=sx[0], x_row=sx[1], x_head=sx[2], y_batch=sy[0], y_row=sy[1],
                            y_head=sy[2], heads=x.shape[-2])
    pos, pos64, pb, pt = None, 0, 0, 0
    if positions is not None:
        if positions.device != x0.device or positions.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"rotary: positions must be int32 or int64 on {x0.device}")
        if positions.shape not in ((length,), (batch, length)):
            raise ValueError(f"rotary: positions must have shape ({length},) or ({batch}, {length}), got {tuple(positions.shape)}")
        pos, pos64 = positions, int(positions.dtype == torch.int64)
        pb, pt = positions.stride() if positions.dim() == 2 else (0, positions.stride(0))
    if batch == 0 or length == 0 or any(x.shape[-2] == 0 for x in tensors):
        if all(y.numel() == 0 for y in outs):
            return outs
        raise ValueError("rotary: a tensor without heads beside one with heads")
    s, keep = spec._struct(head_dim)
    L.check(L.load().vtc_rotary_heads(index, dt, C.byref(s), batch, length, arr, len(tensors), _ptr(pos), pos64, pb, pt, int(offset),
                                      int(bool(inverse)), _stream(x0.device)))
    del keep
    return outs


class _RotaryFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, spec, positions, offset, inverse, *tensors):
        ctx.args = (spec, offset, inverse)
        ctx.save_for_backward(*(() if positions is None else (positions,)))
        return tuple(_rotary_call(tensors, spec, positions, offset, inverse, None))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        spec, offset, inverse = ctx.args
        positions = ctx.saved_tensors[0] if ctx.saved_tensors else None
        grads = [g if g.stride(-1) == 1 or not g.numel() else g.contiguous() for g in grads]
        return (None, None, None, None) + tuple(_rotary_call(grads, spec, positions, offset, not inverse, None))


def rotary_qk(q: torch.Tensor, k: torch.Tensor, spec: Rotary, positions: torch.Tensor | None = None, offset: int = 0,
              inverse: bool = False, out=None):
    """Rotate q and k in one launch: (batch, length, heads, head_dim) or (length, heads, head_dim) each, the heads of q and k may
    differ in number, any strides but the last.  positions: int32 / int64 (batch, length) or (length,), default 0, 1, ..; `offset`
    is added.  inverse turns the other way, which is also the gradient.  out = (q_out, k_out): write there (q and k themselves for
    in place), without a gradient."""
    _need_gpu(q, "rotary")
    _need_gpu(k, "rotary")
    if out is not None:
        if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad):
            raise ValueError("rotary: out= has no gradient; detach the inputs")
        return tuple(_rotary_call((q, k), spec, positions, offset, inverse, tuple(out)))
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad):
        return _RotaryFunction.apply(spec, positions, offset, inverse, q, k)
    return tuple(_rotary_call((q, k), spec, positions, offset, inverse, None))


def rotary(x: torch.Tensor, spec: Rotary, positions: torch.Tensor | None = None, offset: int = 0, inverse: bool = False, out=None):
    """rotary_qk for one tensor."""
    _need_gpu(x, "rotary")
    if out is not None:
        if torch.is_grad_enabled() and x.requires_grad:
            raise ValueError("rotary: out= has no gradient; detach the input")
        return _rotary_call((x,), spec, positions, offset, inverse, (out,))[0]
    if torch.is_grad_enabled() and x.requires_grad:
        return _RotaryFunction.apply(spec, positions, offset, inverse, x)[0]
    return _rotary_call((x,), spec, positions, offset, inverse, None)[0]


# ------------------------------------------------------------------------------------------------ group norm + activation
def _gn_args(what, x, groups, weight, bias, lengths, act):
    index = _need_gpu(x, what)
    dt = _dtype(x, what)
    if x.dim() != 3:
        raise ValueError(f"{what}: rows are (batch, length, channels), got {tuple(x.shape)}")
    if x.numel() and x.stride(2) != 1:
        raise ValueError(f"{what}: the channels of a row must be contiguous")
    n, t, c = x.shape
    if groups < 1 or c < 1 or c % groups:
        raise ValueError(f"{what}: {c} channels do not divide into {groups} groups")
    if act not in ("none", "gelu", "silu"):
        raise ValueError(f"{what}: act must be 'none', 'gelu' or 'silu', got {act!r}")
    f32 = 0
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.device != x.device or p.shape != (c,) or not p.is_contiguous():
            raise ValueError(f"{what}: {name} must be contiguous with shape ({c},) on {x.device}")
        if p.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"{what}: {name} must be {x.dtype} or float32, got {p.dtype}")
        f32 = int(p.dtype == torch.float32)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"{what}: weight and bias must have one type")
    if lengths is not None and (lengths.device != x.device or lengths.dtype != torch.int32 or lengths.shape != (n,) or not lengths.is_contiguous()):
        raise ValueError(f"{what}: lengths must be a contiguous int32 tensor of shape ({n},) on {x.device}")
    return index, dt, f32


def _rows3(t):
    return L.VtcRows3(p=t.data_ptr(), batch=t.stride(0), row=t.stride(1))


def group_norm_act_forward(x: torch.Tensor, groups: int, weight=None, bias=None, eps: float = 1e-5, act: str = "none", lengths=None,
                           out=None):
    """(y, mean, rstd): y = act(group_norm(x)) on channel-last rows (batch, length, channels), statistics per sample and group of
    neighbouring channels over the first lengths[n] rows (int32 tensor, default all).  Rows behind a sample's length are not read
    and come out as zero.  weight / bias: of x's type or float32.  out: where y goes (x itself for in place).  mean and rstd
    (batch, groups, float32) are what the backward call needs."""
    what = "group_norm_act"
    index, dt, f32 = _gn_args(what, x, groups, weight, bias, lengths, act)
    n, t, c = x.shape
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    else:
        _same(what, x, out=out)
        if out.shape != x.shape or (out.numel() and out.stride(2) != 1):
            raise ValueError(f"{what}: out must have shape {tuple(x.shape)} with contiguous channels")
    mean = torch.empty((n, groups), dtype=torch.float32, device=x.device)
    rstd = torch.empty_like(mean)
    if n == 0 or t == 0:
        mean.zero_()
        rstd.zero_()
        return out, mean, rstd
    so = L.load()
    size = so.vtc_group_norm_act_workspace(n, t, c, groups, 0)
    if size < 0:
        L.check(int(size))
    ws = _workspace(size, x.device)
    L.check(so.vtc_group_norm_act(index, dt, C.byref(_rows3(x)), C.byref(_rows3(out)), n, t, c, int(groups), _ptr(weight), _ptr(bias), f32,
                                  float(eps), ACTS[act], _ptr(lengths), _ptr(mean), _ptr(rstd), _ptr(ws), ws.numel(), _stream(x.device)))
    return out, mean, rstd


def group_norm_act_backward(dy: torch.Tensor, x: torch.Tensor, groups: int, mean, rstd, weight=None, bias=None, act: str = "none",
                            lengths=None, out=None):
    """(dx, dweight, dbias) for dy = dLoss / dy and the statistics of the forward call; dweight / dbias have the affine's type (None
    where there is none).  out: where dx goes (dy or x for in place)."""
    what = "group_norm_act_backward"
    index, dt, f32 = _gn_args(what, x, groups, weight, bias, lengths, act)
    n, t, c = x.shape
    _same(what, x, dy=dy, out=out)
    if dy.shape != x.shape or (dy.numel() and dy.stride(2) != 1):
        raise ValueError(f"{what}: dy must have shape {tuple(x.shape)} with contiguous channels")
    for s in (mean, rstd):
        if s.device != x.device or s.dtype != torch.float32 or s.shape != (n, groups) or not s.is_contiguous():
            raise ValueError(f"{what}: mean and rstd are the forward call's, float32 of shape ({n}, {groups})")
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    elif out.shape != x.shape or (out.numel() and out.stride(2) != 1):
        raise ValueError(f"{what}: out must have shape {tuple(x.shape)} with contiguous channels")
    dw = None if weight is None else torch.empty_like(weight)
    db = None if bias is None else torch.empty_like(bias)
    so = L.load()
    size = so.vtc_group_norm_act_workspace(n, t, c, groups, 1)
    if size < 0:
        L.check(int(size))
    ws = _workspace(size, x.device)
    L.check(so.vtc_group_norm_act_backward(index, dt, C.byref(_rows3(dy)), C.byref(_rows3(x)), C.byref(_rows3(out)), n, t, c, int(groups),
                                           _ptr(weight), _ptr(bias), f32, ACTS[act], _ptr(lengths), _ptr(mean), _ptr(rstd), _ptr(dw),
                                           _ptr(db), _ptr(ws), ws.numel(), _stream(x.device)))
    return out, dw, db


class _GroupNormActFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, groups, weight, bias, eps, act, lengths):
        y, mean, rstd = group_norm_act_forward(x, groups, weight, bias, eps, act, lengths)
        ctx.save_for_backward(x, weight, bias, lengths, mean, rstd)
        ctx.args = (groups, act)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, lengths, mean, rstd = ctx.saved_tensors
        if dy.numel() and dy.stride(2) != 1:
            dy = dy.contiguous()
        dx, dw, db = group_norm_act_backward(dy, x, ctx.args[0], mean, rstd, weight, bias, ctx.args[1], lengths)
        return dx, None, dw, db, None, None, None


def group_norm_act(x: torch.Tensor, groups: int, weight=None, bias=None, eps: float = 1e-5, act: str = "none", lengths=None) -> torch.Tensor:
    """act(group_norm(x)) with a gradient for x, weight and bias; see group_norm_act_forward."""
    _need_gpu(x, "group_norm_act")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _GroupNormActFunction.apply(x, groups, weight, bias, eps, act, lengths)
    return group_norm_act_forward(x, groups, weight, bias, eps, act, lengths)[0]


# ------------------------------------------------------------------------------------------------ gated feed-forward
def _mat(t):
    return L.VtcMat(p=t.data_ptr(), row=max(t.stride(0), t.shape[1]) if t.shape[0] <= 1 else t.stride(0))


def _ffn_args(what, x, w_gate, w_up, w_down, biases, act):
    index = _need_gpu(x, what)
    dt = _dtype(x, what, (torch.float16, torch.bfloat16))
    _same(what, x, w_gate=w_gate, w_up=w_up, w_down=w_down)
    if w_gate.dim() != 2 or w_up.shape != w_gate.shape or w_down.dim() != 2 or w_down.shape[1] != w_gate.shape[0] or x.dim() < 1 or x.shape[-1] != w_gate.shape[1]:
        raise ValueError(f"{what}: x (.., width), w_gate and w_up (inner, width), w_down (out, inner) do not go together: {tuple(x.shape)}, "
                         f"{tuple(w_gate.shape)}, {tuple(w_up.shape)}, {tuple(w_down.shape)}")
    for name, t in (("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down)):
        if t.stride(1) != 1 or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
            raise ValueError(f"{what}: {name} must be stored row by row")
    if act not in ACTS:
        raise ValueError(f"{what}: act must be one of {list(ACTS)}, got {act!r}")
    f32, kinds = 0, set()
    for name, b, n in zip(("b_gate", "b_up", "b_down"), biases, (w_gate.shape[0], w_gate.shape[0], w_down.shape[0])):
        if b is None:
            continue
        if b.device != x.device or b.shape != (n,) or not b.is_contiguous() or b.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"{what}: {name} must be contiguous, of shape ({n},) and type {x.dtype} or float32 on {x.device}")
        kinds.add(b.dtype)
        f32 = int(b.dtype == torch.float32)
    if len(kinds) > 1:
        raise ValueError(f"{what}: the biases must have one type")
    return index, dt, f32


def _rows2(t, what):
    """t (.., n) as rows (m, n) whose elements are contiguous; a view where the strides allow it."""
    r = t.reshape(-1, t.shape[-1])
    if r.numel() and (r.stride(1) != 1 or (r.shape[0] > 1 and r.stride(0) < r.shape[1])):
        r = r.contiguous()
    return r


def gated_ffn_forward(x: torch.Tensor, w_gate, w_up, w_down, b_gate=None, b_up=None, b_down=None, act: str = "silu", save: bool = False):
    """(y, saved): y = (act(x w_gate^T + b_gate) * (x w_up^T + b_up)) w_down^T + b_down on rows x (.., width) in float16 or bfloat16,
    sums in fp32; w_gate, w_up (inner, width), w_down (out, inner); biases of x's type or float32.  With save, `saved` is what
    gated_ffn_backward needs (three times rows x inner in x's type), else None."""
    what = "gated_ffn"
    index, dt, f32 = _ffn_args(what, x, w_gate, w_up, w_down, (b_gate, b_up, b_down), act)
    rows = _rows2(x, what)
    m, k = rows.shape
    f, n = w_gate.shape[0], w_down.shape[0]
    y = torch.empty(x.shape[:-1] + (n,), dtype=x.dtype, device=x.device)
    so = L.load()
    size = so.vtc_gated_ffn_workspace(m, k, f, n, 0)
    if size < 0:
        L.check(int(size))
    saved = _workspace(so.vtc_gated_ffn_saved(m, f), x.device) if save else None
    if m == 0:
        return y, saved
    ws = _workspace(size, x.device)
    L.check(so.vtc_gated_ffn(index, dt, m, k, f, n, C.byref(_mat(rows)), C.byref(_mat(w_gate)), C.byref(_mat(w_up)), C.byref(_mat(w_down)),
                             _ptr(b_gate), _ptr(b_up), _ptr(b_down), f32, ACTS[act], C.byref(L.VtcMat(y.data_ptr(), n)), _ptr(saved),
                             0 if saved is None else saved.numel(), _ptr(ws), ws.numel(), _stream(x.device)))
    return y, saved


def gated_ffn_backward(dy: torch.Tensor, x: torch.Tensor, w_gate, w_up, w_down, saved, act: str = "silu", biases: bool = True,
                       bias_dtype=None, need_dx: bool = True, need_dw: bool = True):
    """(dx, dw_gate, dw_up, dw_down, db_gate, db_up, db_down) for dy = dLoss / dy and the forward call's `saved`; what is not asked for
    (biases, need_dx, need_dw) is None.  Gradients have the type of what they belong to (biases: bias_dtype, default x's)."""
    what = "gated_ffn_backward"
    index, dt, _ = _ffn_args(what, x, w_gate, w_up, w_down, (None, None, None), act)
    _same(what, x, dy=dy)
    f, n = w_gate.shape[0], w_down.shape[0]
    if dy.shape != x.shape[:-1] + (n,):
        raise ValueError(f"{what}: dy must have shape {tuple(x.shape[:-1] + (n,))}, got {tuple(dy.shape)}")
    bias_dtype = bias_dtype or x.dtype
    if bias_dtype not in (x.dtype, torch.float32):
        raise ValueError(f"{what}: bias_dtype must be {x.dtype} or float32")
    rows, drows = _rows2(x, what), _rows2(dy, what)
    m, k = rows.shape
    new = lambda shape, kind: torch.empty(shape, dtype=kind, device=x.device)  # noqa: E731
    dx = new(x.shape, x.dtype) if need_dx else None
    dw = tuple(new(w.shape, x.dtype) if need_dw else None for w in (w_gate, w_up, w_down))
    db = tuple(new((c,), bias_dtype) if biases else None for c in (f, f, n))
    if m == 0:
        for t in dw + db:
            if t is not None:
                t.zero_()
        return (dx,) + dw + db
    so = L.load()
    size = so.vtc_gated_ffn_workspace(m, k, f, n, 1)
    if size < 0:
        L.check(int(size))
    if saved is None or saved.device != x.device or saved.dtype != torch.uint8 or saved.numel() < so.vtc_gated_ffn_saved(m, f):
        raise ValueError(f"{what}: saved is the forward call's (with save=True)")
    ws = _workspace(size, x.device)
    adr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    grads = L.VtcFfnGrads(adr(dx), k, *(adr(t) for t in dw + db))
    L.check(so.vtc_gated_ffn_backward(index, dt, m, k, f, n, C.byref(_mat(drows)), C.byref(_mat(rows)), C.byref(_mat(w_gate)),
                                      C.byref(_mat(w_up)), C.byref(_mat(w_down)), _ptr(saved), saved.numel(),
                                      int(bias_dtype == torch.float32), ACTS[act], C.byref(grads), _ptr(ws), ws.numel(), _stream(x.device)))
    return (dx,) + dw + db


class _GatedFfnFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, b_gate, b_up, b_down, act):
        y, saved = gated_ffn_forward(x, w_gate, w_up, w_down, b_gate, b_up, b_down, act, save=True)
        ctx.save_for_backward(x, w_gate, w_up, w_down, saved)
        ctx.act, ctx.kinds = act, tuple(None if b is None else b.dtype for b in (b_gate, b_up, b_down))
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w_gate, w_up, w_down, saved = ctx.saved_tensors
        kinds = [k for k in ctx.kinds if k is not None]
        need = ctx.needs_input_grad
        got = gated_ffn_backward(dy, x, w_gate, w_up, w_down, saved, ctx.act, biases=bool(kinds) and any(need[4:7]),
                                 bias_dtype=kinds[0] if kinds else None, need_dx=need[0], need_dw=any(need[1:4]))
        return tuple(t if i < 4 or ctx.kinds[i - 4] is not None else None for i, t in enumerate(got)) + (None,)


def gated_ffn(x: torch.Tensor, w_gate, w_up, w_down, b_gate=None, b_up=None, b_down=None, act: str = "silu") -> torch.Tensor:
    """The block with a gradient for x, the weights and the biases; see gated_ffn_forward."""
    _need_gpu(x, "gated_ffn")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, w_gate, w_up, w_down, b_gate, b_up, b_down)):
        return _GatedFfnFunction.apply(x, w_gate, w_up, w_down, b_gate, b_up, b_down, act)
    return gated_ffn_forward(x, w_gate, w_up, w_down, b_gate, b_up, b_down, act)[0]
