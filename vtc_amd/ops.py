"""The library's stand-alone operators (include/vtc_amd.h, "Operators") on torch tensors.

Rotary positions, group norm with an activation on channel-last rows and the gated feed-forward block: what an encoder variant
(VtcEngine(variant=...)) runs inside the library, for callers that run such layers themselves or adapt them to new recordings.
Every function launches on the current stream of its tensors' device and neither synchronises nor copies to the host.

Each operator has explicit forward and backward calls (`*_forward`, `*_backward`, `inverse=True`) and, where that is handier, a
differentiable one (`rotary`, `rotary_qk`, `group_norm_act`, `gated_ffn`) whose gradient is those calls (reverse mode; a
forward-mode tangent is refused).  The explicit calls and what is written through out= carry no gradient.  A program that captures a
training step into a graph uses the explicit ones, or makes the differentiable call inside the capture as well.
"""

from __future__ import annotations

import ctypes as C
import functools
import math

import numpy as np
import torch
import torch.autograd.forward_ad as forward_ad
from torch.autograd.graph import increment_version

from . import lib as L

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
ACTS = {"none": 0, "gelu": 1, "silu": 2, "sigmoid": 3}
LAYOUTS = {"half": 0, "interleaved": 1}
SCALINGS = ("none", "linear", "ntk", "by_parts")


_so = None


def _library():
    global _so
    if _so is None:
        _so = L.load()
    return _so


def _need_gpu(x: torch.Tensor, what: str) -> int:
    """The index of x's GPU."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{what}: expected a tensor, got {type(x).__name__}")
    if not x.is_cuda:
        raise ValueError(f"{what}: tensors must be on a ROCm GPU (there is no CPU path), got {x.device}")
    return x.get_device()


def _same(what: str, x: torch.Tensor, name: str, t) -> None:
    if t.dtype is not x.dtype or not t.is_cuda or t.get_device() != x.get_device():
        raise ValueError(f"{what}: {name} is {t.dtype} on {t.device}, expected {x.dtype} on {x.device}")


def _dtype(x: torch.Tensor, what: str, allowed=_DTYPES) -> int:
    dt = allowed.get(x.dtype)
    if dt is None:
        raise ValueError(f"{what}: type {x.dtype} is not one of {', '.join(str(a) for a in allowed)}")
    return dt


# the raw handle without a Stream object around it, which costs several microseconds per call
_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _ptr(t):
    return None if t is None else t.data_ptr()


@functools.lru_cache(maxsize=1024)
def _bytes(entry: str, *sizes) -> int:
    """What a size query of the library answers; it depends on nothing but the sizes."""
    n = getattr(_library(), entry)(*sizes)
    if n < 0:
        L.check(int(n))
    return n


def _empty(t: torch.Tensor) -> torch.Tensor:
    """An uninitialised contiguous tensor like t (empty_like without a format is the cheapest way to one)."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty_like(t, memory_format=torch.contiguous_format)


def _workspace(n: int, x: torch.Tensor) -> torch.Tensor:
    # the allocator's blocks start at multiples of 512 bytes; inside a graph capture they come from the graph's own pool
    return torch.empty(n if n > 0 else 1, dtype=torch.uint8, device=x.device)


def _tracked(*tensors) -> bool:
    """Whether autograd has to hear of a call on these tensors.  A forward-mode tangent counts: the operators have none of their own, and
    the autograd functions below say so, where the plain call would drop it."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _check_out(what: str, out) -> None:
    if torch.is_grad_enabled() and out.requires_grad:
        raise ValueError(f"{what}: out= has no gradient, and the tensor given requires one; detach it")


# ------------------------------------------------------------------------------------------------ rotary positions
class Rotary:
    """What a rotation is: pairs of the first `rotary_dim` elements of a head (all of them by default, see rotary()), their layout
    ("half": j with j + rotary_dim / 2; "interleaved": 2j with 2j + 1) and their angular frequencies, base ** (-2 j / rotary_dim)
    unless scaled for positions beyond those a model was trained on:

    "linear":   frequency / factor
    "ntk":      base * factor ** (rotary_dim / (rotary_dim - 2)) in place of base
    "by_parts": pairs that turn more than 32 times over `original_length` positions keep their frequency, those that turn less
                than once are divided by `factor`, between them (from pair 0 on, if none turns that often) a ramp linear in the
                pair's index; the result is multiplied by 1 + 0.1 ln(factor)

    Frequencies are 64-bit; frequency= and amplitude= give the caller's own instead.  The object does not change once it is made."""

    def __init__(self, rotary_dim: int, layout: str = "half", base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                 original_length: int = 0, frequency=None, amplitude: float | None = None):
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
            # the ramp may end behind the last pair (index(1) counts on): clamped to it, a pair that still turns twice would be slowed
            # by the whole factor.  Where not even pair 0 turns once, the ramp lies in front of it
            high = min(math.ceil(index(1.0)), r - 1)
            low = min(max(math.floor(index(32.0)), 0), high - 1)
            ramp = np.clip((j - low) / (high - low), 0.0, 1.0)
            f = f / s * ramp + f * (1.0 - ramp)
            self.amplitude = 0.1 * math.log(s) + 1.0 if s > 1.0 else 1.0
        if frequency is not None:
            f = np.array(frequency, dtype=np.float64)
        if amplitude is not None:
            self.amplitude = float(amplitude)
        if f.shape != (r // 2,):
            raise ValueError(f"frequency must have {r // 2} entries, got shape {f.shape}")
        f.setflags(write=False)
        self.frequency = f
        self._structs = {}

    def __getstate__(self):   # copies and pickles leave the C descriptions, which hold addresses, behind
        return {"rotary_dim": self.rotary_dim, "layout": self.layout, "amplitude": self.amplitude, "frequency": self.frequency}

    def __setstate__(self, state):
        self.__dict__.update(state, frequency=np.array(state["frequency"]), _structs={})
        self.frequency.setflags(write=False)

    def _struct(self, head_dim: int) -> L.VtcRotary:
        """The C description for heads of this size (it points into self.frequency)."""
        s = self._structs.get(head_dim)
        if s is None:
            s = self._structs[head_dim] = L.VtcRotary(head_dim, self.rotary_dim, LAYOUTS[self.layout], 0, self.amplitude,
                                                      self.frequency.ctypes.data_as(L._f64p))
        return s


def _rotary_call(tensors, spec: Rotary, positions, offset: int, inverse: bool, outs):
    x0 = tensors[0]
    index = _need_gpu(x0, "rotary")
    dt = _dtype(x0, "rotary")
    if not isinstance(spec, Rotary):
        raise TypeError("rotary: expected a Rotary")
    shape0 = x0.shape
    nd = len(shape0)
    if nd == 4:
        batch, length, _, head_dim = shape0
    elif nd == 3:
        (length, _, head_dim), batch = shape0, 1
    else:
        raise ValueError(f"rotary: tensors are (batch, length, heads, head_dim) or (length, heads, head_dim), got {tuple(shape0)}")
    if spec.rotary_dim > head_dim:
        raise ValueError(f"rotary: rotary_dim {spec.rotary_dim} is more than head_dim {head_dim}")
    heads, results, empty = [], [], batch == 0 or length == 0
    for i, x in enumerate(tensors):
        shape = shape0
        if x is not x0:
            _same("rotary", x0, "a tensor", x)
            shape = x.shape
            if len(shape) != nd or shape[:-2] != shape0[:-2] or shape[-1] != head_dim:
                raise ValueError(f"rotary: shapes {tuple(shape0)} and {tuple(shape)} do not go together")
        sx = x.stride()
        empty = empty or shape[-2] == 0
        if sx[-1] != 1 and not empty:
            raise ValueError("rotary: the elements of a head must be contiguous")
        if outs is None:
            y = torch.empty_like(x)
            if y.stride(-1) != 1:   # (sizes of one leave empty_like's order open)
                y = torch.empty(shape, dtype=x.dtype, device=x.device)
        else:
            y = outs[i]
            _same("rotary", x0, "out", y)
            _check_out("rotary", y)
            if y.shape != shape or (y.stride(-1) != 1 and not empty):
                raise ValueError(f"rotary: out must have shape {tuple(shape)} with contiguous heads, got {tuple(y.shape)}")
        results.append(y)
        sy = y.stride()
        if nd == 3:
            sx, sy = (0,) + sx, (0,) + sy
        heads.append((x.data_ptr(), y.data_ptr(), sx[0], sx[1], sx[2], sy[0], sy[1], sy[2], shape[-2]))
    pos, pos64, pb, pt = None, 0, 0, 0
    if positions is not None:
        if not positions.is_cuda or positions.get_device() != index or positions.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"rotary: positions must be int32 or int64 on {x0.device}")
        shape = positions.shape
        if shape != (batch, length) and shape != (length,):
            raise ValueError(f"rotary: positions must have shape ({length},) or ({batch}, {length}), got {tuple(shape)}")
        pos, pos64 = positions.data_ptr(), int(positions.dtype is torch.int64)
        pb, pt = positions.stride() if len(shape) == 2 else (0, positions.stride(0))
    if empty:
        if all(y.numel() == 0 for y in results):
            return results
        raise ValueError("rotary: a tensor without heads beside one with heads")
    rc = _library().vtc_rotary_heads(index, dt, spec._struct(head_dim), batch, length, (L.VtcHeads * len(heads))(*heads), len(heads), pos, pos64,
                                     pb, pt, offset, 1 if inverse else 0, _stream(index))
    if rc:
        L.check(rc)
    if outs is not None:
        increment_version(results)   # a gradient that has kept what was there before has to notice
    return results


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
        if _tracked(q, k):
            raise ValueError("rotary: out= has no gradient; detach the inputs")
        return tuple(_rotary_call((q, k), spec, positions, offset, inverse, tuple(out)))
    if _tracked(q, k):
        return _RotaryFunction.apply(spec, positions, offset, inverse, q, k)
    return tuple(_rotary_call((q, k), spec, positions, offset, inverse, None))


def rotary(x: torch.Tensor, spec: Rotary, positions: torch.Tensor | None = None, offset: int = 0, inverse: bool = False, out=None):
    """rotary_qk for one tensor."""
    _need_gpu(x, "rotary")
    if out is not None:
        if _tracked(x):
            raise ValueError("rotary: out= has no gradient; detach the input")
        return _rotary_call((x,), spec, positions, offset, inverse, (out,))[0]
    if _tracked(x):
        return _RotaryFunction.apply(spec, positions, offset, inverse, x)[0]
    return _rotary_call((x,), spec, positions, offset, inverse, None)[0]


def _dense_last(t) -> bool:
    """Whether the elements of the last dimension are neighbours (one element has no stride, whatever the tensor says)."""
    return t.stride(-1) == 1 or t.shape[-1] == 1 or not t.numel()


# ------------------------------------------------------------------------------------------------ group norm + activation
_GN_ACTS = ("none", "gelu", "silu")


def _gn_args(what, x, groups, weight, bias, lengths, act):
    index = _need_gpu(x, what)
    dt = _dtype(x, what)
    shape = x.shape
    if len(shape) != 3:
        raise ValueError(f"{what}: rows are (batch, length, channels), got {tuple(shape)}")
    n, t, c = shape
    if not _dense_last(x):
        raise ValueError(f"{what}: the channels of a row must be contiguous")
    if groups < 1 or c < 1 or c % groups:
        raise ValueError(f"{what}: {c} channels do not divide into {groups} groups")
    if act not in _GN_ACTS:
        raise ValueError(f"{what}: act must be 'none', 'gelu' or 'silu', got {act!r}")
    f32 = 0
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if not p.is_cuda or p.get_device() != index or p.shape != (c,) or not p.is_contiguous():
            raise ValueError(f"{what}: {name} must be contiguous with shape ({c},) on {x.device}")
        kind = p.dtype
        if kind is not x.dtype and kind is not torch.float32:
            raise ValueError(f"{what}: {name} must be {x.dtype} or float32, got {kind}")
        f32 = 1 if kind is torch.float32 else 0
    if weight is not None and bias is not None and weight.dtype is not bias.dtype:
        raise ValueError(f"{what}: weight and bias must have one type")
    if lengths is not None and (not lengths.is_cuda or lengths.get_device() != index or lengths.dtype is not torch.int32 or lengths.shape != (n,) or
                                not lengths.is_contiguous()):
        raise ValueError(f"{what}: lengths must be a contiguous int32 tensor of shape ({n},) on {x.device}")
    return index, dt, f32, n, t, c


def _rows3(t):
    s = t.stride()
    return L.VtcRows3(t.data_ptr(), s[0], s[1])


def _gn_out(what, x, out):
    if out is None:
        return _empty(x)
    _same(what, x, "out", out)
    _check_out(what, out)
    if out.shape != x.shape or not _dense_last(out):
        raise ValueError(f"{what}: out must have shape {tuple(x.shape)} with contiguous channels")
    return out


def group_norm_act_forward(x: torch.Tensor, groups: int, weight=None, bias=None, eps: float = 1e-5, act: str = "none", lengths=None,
                           out=None):
    """(y, mean, rstd): y = act(group_norm(x)) on channel-last rows (batch, length, channels), statistics per sample and group of
    neighbouring channels over the first lengths[n] rows (int32 tensor, default all).  Rows behind a sample's length are not read
    and come out as zero.  weight / bias: of x's type or float32.  out: where y goes (x itself for in place).  mean and rstd
    (batch, groups, float32) are what the backward call needs.  A sample's result does not depend on the rest of its batch (of tensors
    with the same strides and alignment)."""
    what = "group_norm_act"
    index, dt, f32, n, t, c = _gn_args(what, x, groups, weight, bias, lengths, act)
    given, out = out, _gn_out(what, x, out)
    mean, rstd = torch.empty((2, n, groups), dtype=torch.float32, device=x.device).unbind(0)
    so = _library()
    size = _bytes("vtc_group_norm_act_workspace", n, t, c, groups, 0)
    ws = _workspace(size, x)
    rc = so.vtc_group_norm_act(index, dt, _rows3(x), _rows3(out), n, t, c, groups, _ptr(weight), _ptr(bias), f32, eps, ACTS[act], _ptr(lengths),
                               mean.data_ptr(), rstd.data_ptr(), ws.data_ptr(), size, _stream(index))
    if rc:
        L.check(rc)
    if given is not None:
        increment_version(given)
    return out, mean, rstd


def group_norm_act_backward(dy: torch.Tensor, x: torch.Tensor, groups: int, mean, rstd, weight=None, bias=None, act: str = "none",
                            lengths=None, out=None):
    """(dx, dweight, dbias) for dy = dLoss / dy and the statistics of the forward call; dweight / dbias have the affine's type (None
    where there is none).  out: where dx goes (dy or x for in place)."""
    what = "group_norm_act_backward"
    index, dt, f32, n, t, c = _gn_args(what, x, groups, weight, bias, lengths, act)
    _same(what, x, "dy", dy)
    if dy.shape != x.shape or not _dense_last(dy):
        raise ValueError(f"{what}: dy must have shape {tuple(x.shape)} with contiguous channels")
    for s in (mean, rstd):
        if not s.is_cuda or s.get_device() != index or s.dtype is not torch.float32 or s.shape != (n, groups) or not s.is_contiguous():
            raise ValueError(f"{what}: mean and rstd are the forward call's, float32 of shape ({n}, {groups})")
    given, out = out, _gn_out(what, x, out)
    dw = None if weight is None else torch.empty_like(weight)
    db = None if bias is None else torch.empty_like(bias)
    so = _library()
    size = _bytes("vtc_group_norm_act_workspace", n, t, c, groups, 1)
    ws = _workspace(size, x)
    rc = so.vtc_group_norm_act_backward(index, dt, _rows3(dy), _rows3(x), _rows3(out), n, t, c, groups, _ptr(weight), _ptr(bias), f32, ACTS[act],
                                        _ptr(lengths), mean.data_ptr(), rstd.data_ptr(), _ptr(dw), _ptr(db), ws.data_ptr(), size, _stream(index))
    if rc:
        L.check(rc)
    if given is not None:
        increment_version(given)
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
        if not _dense_last(dy):
            dy = dy.contiguous()
        dx, dw, db = group_norm_act_backward(dy, x, ctx.args[0], mean, rstd, weight, bias, ctx.args[1], lengths)
        return dx, None, dw, db, None, None, None


def group_norm_act(x: torch.Tensor, groups: int, weight=None, bias=None, eps: float = 1e-5, act: str = "none", lengths=None) -> torch.Tensor:
    """act(group_norm(x)) with a gradient for x, weight and bias; see group_norm_act_forward."""
    _need_gpu(x, "group_norm_act")
    if _tracked(x, weight, bias):
        return _GroupNormActFunction.apply(x, groups, weight, bias, eps, act, lengths)
    return group_norm_act_forward(x, groups, weight, bias, eps, act, lengths)[0]


# ------------------------------------------------------------------------------------------------ gated feed-forward
_FFN_TYPES = {torch.float16: 1, torch.bfloat16: 2}


_MAX_PITCH = 1 << 20   # the library's limit for matrices of more than one row


def _mat(t, cols):
    row = t.stride(0)
    return L.VtcMat(t.data_ptr(), row if row > cols else cols)   # a single row may have any stride


def _ffn_args(what, x, w_gate, w_up, w_down, biases, act):
    index = _need_gpu(x, what)
    dt = _dtype(x, what, _FFN_TYPES)
    _same(what, x, "w_gate", w_gate)
    _same(what, x, "w_up", w_up)
    _same(what, x, "w_down", w_down)
    sg, su, sd = w_gate.shape, w_up.shape, w_down.shape
    if len(sg) != 2 or su != sg or len(sd) != 2 or sd[1] != sg[0] or x.dim() < 1 or x.shape[-1] != sg[1]:
        raise ValueError(f"{what}: x (.., width), w_gate and w_up (inner, width), w_down (out, inner) do not go together: {tuple(x.shape)}, "
                         f"{tuple(sg)}, {tuple(su)}, {tuple(sd)}")
    for name, t in (("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down)):
        row, col = t.stride()
        if (col != 1 and t.shape[1] > 1) or (row < t.shape[1] and t.shape[0] > 1):
            raise ValueError(f"{what}: {name} must be stored row by row")
    if act not in ACTS:
        raise ValueError(f"{what}: act must be one of {list(ACTS)}, got {act!r}")
    kind = None
    for i, b in enumerate(biases):
        if b is None:
            continue
        if not b.is_cuda or b.get_device() != index or b.shape != ((sg[0],) if i < 2 else (sd[0],)) or not b.is_contiguous() or (
                b.dtype is not x.dtype and b.dtype is not torch.float32):
            raise ValueError(f"{what}: {('b_gate', 'b_up', 'b_down')[i]} must be contiguous, of shape ({sg[0] if i < 2 else sd[0]},) and type "
                             f"{x.dtype} or float32 on {x.device}")
        if kind is not None and b.dtype is not kind:
            raise ValueError(f"{what}: the biases must have one type")
        kind = b.dtype
    return index, dt, 1 if kind is torch.float32 else 0, sg[1], sg[0], sd[0]


def _rows2(t):
    """t (.., n) as rows (m, n) whose elements are contiguous; a view where the strides allow it, else a copy (also of rows that are
    further apart than the library takes, such as the last frames of several long recordings: those are few)."""
    r = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
    row, col = r.stride()
    if (col != 1 or (not r.shape[1] <= row <= _MAX_PITCH and r.shape[0] > 1)) and r.numel():
        r = r.contiguous()
    return r


def gated_ffn_forward(x: torch.Tensor, w_gate, w_up, w_down, b_gate=None, b_up=None, b_down=None, act: str = "silu", save: bool = False):
    """(y, saved): y = (act(x w_gate^T + b_gate) * (x w_up^T + b_up)) w_down^T + b_down on rows x (.., width) in float16 or bfloat16,
    sums in fp32; w_gate, w_up (inner, width), w_down (out, inner); biases of x's type or float32.  With save, `saved` is what
    gated_ffn_backward needs, an opaque buffer of vtc_gated_ffn_saved bytes; else None.  The order in which a row's products are added
    follows the number of rows, so its last bits do."""
    what = "gated_ffn"
    index, dt, f32, k, f, n = _ffn_args(what, x, w_gate, w_up, w_down, (b_gate, b_up, b_down), act)
    rows = _rows2(x)
    m = rows.shape[0]
    y = _empty(x) if n == k else torch.empty(x.shape[:-1] + (n,), dtype=x.dtype, device=x.device)
    so = _library()
    size = _bytes("vtc_gated_ffn_workspace", m, k, f, n, 0)
    saved, saved_size = None, 0
    if save:
        saved_size = _bytes("vtc_gated_ffn_saved", m, f)
        saved = _workspace(saved_size, x)
    if m == 0:
        return y, saved
    ws = _workspace(size, x)
    rc = so.vtc_gated_ffn(index, dt, m, k, f, n, _mat(rows, k), _mat(w_gate, k), _mat(w_up, k), _mat(w_down, f), _ptr(b_gate), _ptr(b_up),
                          _ptr(b_down), f32, ACTS[act], L.VtcMat(y.data_ptr(), n), _ptr(saved), saved_size, ws.data_ptr(), size, _stream(index))
    if rc:
        L.check(rc)
    return y, saved


def gated_ffn_backward(dy: torch.Tensor, x: torch.Tensor, w_gate, w_up, w_down, saved, act: str = "silu", biases: bool = True,
                       bias_dtype=None, need_dx: bool = True, need_dw: bool = True):
    """(dx, dw_gate, dw_up, dw_down, db_gate, db_up, db_down) for dy = dLoss / dy and the forward call's `saved`; what is not asked for
    (biases, need_dx, need_dw) is None.  Gradients have the type of what they belong to (biases: bias_dtype, default x's).  act is the
    forward call's; its slopes are part of `saved`."""
    what = "gated_ffn_backward"
    index, dt, _, k, f, n = _ffn_args(what, x, w_gate, w_up, w_down, (), act)
    _same(what, x, "dy", dy)
    if dy.shape != x.shape[:-1] + (n,):
        raise ValueError(f"{what}: dy must have shape {tuple(x.shape[:-1] + (n,))}, got {tuple(dy.shape)}")
    bias_dtype = bias_dtype or x.dtype
    if bias_dtype not in (x.dtype, torch.float32):
        raise ValueError(f"{what}: bias_dtype must be {x.dtype} or float32")
    rows, drows = _rows2(x), _rows2(dy)
    m = rows.shape[0]
    dx = _empty(x) if need_dx else None
    dw = (_empty(w_gate), _empty(w_up), _empty(w_down)) if need_dw else (None, None, None)
    db = tuple(x.new_empty((c,)) if bias_dtype is x.dtype else x.new_empty((c,), dtype=bias_dtype) for c in (f, f, n)) if biases else (None, None, None)
    if m == 0:
        for t in dw + db:
            if t is not None:
                t.zero_()
        return (dx,) + dw + db
    so = _library()
    size = _bytes("vtc_gated_ffn_workspace", m, k, f, n, 1)
    if saved is None or not saved.is_cuda or saved.get_device() != index or saved.dtype is not torch.uint8 or saved.numel() < _bytes("vtc_gated_ffn_saved", m, f):
        raise ValueError(f"{what}: saved is the forward call's (with save=True)")
    ws = _workspace(size, x)
    grads = L.VtcFfnGrads(_ptr(dx), k, *(_ptr(t) for t in dw + db))
    rc = so.vtc_gated_ffn_backward(index, dt, m, k, f, n, _mat(drows, n), _mat(rows, k), _mat(w_gate, k), _mat(w_up, k), _mat(w_down, f),
                                   saved.data_ptr(), saved.numel(), 1 if bias_dtype is torch.float32 else 0, grads, ws.data_ptr(), size,
                                   _stream(index))
    if rc:
        L.check(rc)
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
    if _tracked(x, w_gate, w_up, w_down, b_gate, b_up, b_down):
        return _GatedFfnFunction.apply(x, w_gate, w_up, w_down, b_gate, b_up, b_down, act)
    return gated_ffn_forward(x, w_gate, w_up, w_down, b_gate, b_up, b_down, act)[0]
