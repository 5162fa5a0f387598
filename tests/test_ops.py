"""The stand-alone operators (vtc_amd.ops): rotary positions and group norm with an activation, against 64-bit definitions.

Tolerances: a result rounded to type t is off by at most eps(t) / 2 of its value; the fp32 arithmetic in front of it is bounded term
by term beside each check.  Refusals run without a GPU (the library checks its arguments before it looks for a device)."""

import ctypes as C
import math

import numpy as np
import pytest
import torch

from vtc_amd import lib as L
from vtc_amd import ops

gpu = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def half_step(t, v):
    """Largest rounding of v to type t: half a step relative, half a subnormal step near zero."""
    i = torch.finfo(t)
    return v.abs() * (i.eps / 2) + i.smallest_normal * i.eps / 2


def close(got, want, tol, what=""):
    d = (got.double().cpu() - want).abs()
    assert got.shape == want.shape
    bad = ~(d <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((d / tol).max()):.3g} x the tolerance"


# --------------------------------------------------------------------------------------------- rotary
def rotary_64(x, spec, pos, inverse=False):
    x = x.double().cpu()
    a = pos.double().cpu()[..., None] * torch.from_numpy(spec.frequency)
    c, s = (torch.cos(a) * spec.amplitude)[..., None, :], (torch.sin(a) * spec.amplitude * (-1 if inverse else 1))[..., None, :]
    y, r = x.clone(), spec.rotary_dim
    if spec.layout == "half":
        u, v = x[..., : r // 2], x[..., r // 2: r]
        y[..., : r // 2], y[..., r // 2: r] = u * c - v * s, u * s + v * c
        mag = torch.cat([u.abs() + v.abs()] * 2, -1)
    else:
        u, v = x[..., 0:r:2], x[..., 1:r:2]
        y[..., 0:r:2], y[..., 1:r:2] = u * c - v * s, u * s + v * c
        mag = torch.stack([u.abs() + v.abs()] * 2, -1).flatten(-2)
    return y, mag


def check_rotary(got, x, spec, pos, inverse=False):
    want, mag = rotary_64(x, spec, pos, inverse)
    r = spec.rotary_dim
    # cos and sin are within 2^-22 (argument 2^-24 pi / 4, five fp32 operations), each product and the sum round once more.
    # The angle itself: the definition rounds position * frequency to 53 bits and the library rounds the frequency in turns, each
    # 2^-53 of the angle, which is 1e-6 rad at the 2^33 rad of the farthest positions here
    angle = (pos.double().cpu().abs()[..., None] * torch.from_numpy(np.abs(spec.frequency)))[..., None, :]
    angle = torch.cat([angle] * 2, -1) if spec.layout == "half" else torch.stack([angle] * 2, -1).flatten(-2)
    tol = half_step(x.dtype, want)[..., :r] + mag * spec.amplitude * (2.0 ** -21 + angle * 2.0 ** -52)
    close(got[..., :r], want[..., :r], tol, "rotated")
    assert torch.equal(got[..., r:].cpu(), x[..., r:].cpu()), "the part behind the rotation is copied"


@gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("batch,length,hq,hk,dim,rot", [(1, 1, 1, 1, 2, 2), (3, 1, 12, 12, 64, 64), (2, 77, 12, 4, 64, 48), (1, 300, 3, 1, 130, 130),
                                                        (2, 19, 5, 5, 24, 14), (1, 9, 2, 2, 640, 512), (5, 1031, 1, 1, 16, 16)])
def test_rotary_against_the_definition(kind, layout, batch, length, hq, hk, dim, rot):
    g = torch.Generator(device="cuda").manual_seed(dim + length)
    q = torch.randn((batch, length, hq, dim), generator=g, device="cuda").to(TYPES[kind])
    k = torch.randn((batch, length, hk, dim), generator=g, device="cuda").to(TYPES[kind])
    spec = ops.Rotary(rot, layout=layout)
    pos = torch.randint(0, 3_000_000, (batch, length), generator=g, device="cuda")
    q2, k2 = ops.rotary_qk(q, k, spec, positions=pos)
    check_rotary(q2, q, spec, pos)
    check_rotary(k2, k, spec, pos)
    q3 = ops.rotary(q, spec, positions=pos.to(torch.int32), inverse=True)
    check_rotary(q3, q, spec, pos, inverse=True)
    k3 = ops.rotary(k, spec, offset=7)
    check_rotary(k3, k, spec, (torch.arange(length) + 7).expand(batch, length))


@gpu
@pytest.mark.parametrize("scaling,factor", [("linear", 4.0), ("ntk", 8.0), ("by_parts", 32.0), ("by_parts", 0.5)])
def test_rotary_scalings_far_and_negative_positions(scaling, factor):
    spec = ops.Rotary(96, scaling=scaling, factor=factor, original_length=2048, layout="interleaved")
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn((2, 50, 3, 128), generator=g, device="cuda")
    pos = torch.randint(-2 ** 33, 2 ** 33, (2, 50), generator=g, device="cuda")
    check_rotary(ops.rotary(x, spec, positions=pos), x, spec, pos)


@gpu
def test_rotary_strides_in_place_and_broadcast():
    g = torch.Generator(device="cuda").manual_seed(6)
    spec = ops.Rotary(64)
    qkv = torch.randn((3, 40, 3 * 12 * 64), generator=g, device="cuda").half()      # a fused projection's rows
    before = qkv.clone()
    q, k = qkv[..., :768].unflatten(-1, (12, 64)), qkv[..., 768:1536].unflatten(-1, (12, 64))
    ops.rotary_qk(q, k, spec, out=(q, k))
    pos = torch.arange(40).expand(3, 40)
    check_rotary(q, before[..., :768].unflatten(-1, (12, 64)), spec, pos)
    check_rotary(k, before[..., 768:1536].unflatten(-1, (12, 64)), spec, pos)
    assert torch.equal(qkv[..., 1536:], before[..., 1536:])
    heads_first = torch.randn((2, 5, 33, 64), generator=g, device="cuda")             # (batch, heads, length, dim)
    x = heads_first.transpose(1, 2)
    check_rotary(ops.rotary(x, spec), x, spec, torch.arange(33).expand(2, 33))
    odd = torch.randn((2, 33, 5, 67), generator=g, device="cuda").bfloat16()[..., 1:65]   # rows that are not 16-byte aligned
    check_rotary(ops.rotary(odd, spec), odd, spec, torch.arange(33).expand(2, 33))
    same = torch.randn((1, 33, 1, 64), generator=g, device="cuda").expand(4, 33, 6, 64)   # one head for all
    check_rotary(ops.rotary(same, spec), same, spec, torch.arange(33).expand(4, 33))
    rows = torch.randn((33, 5, 64), generator=g, device="cuda")
    check_rotary(ops.rotary(rows, spec), rows, spec, torch.arange(33))
    assert ops.rotary(rows[:0], spec).shape == (0, 5, 64)
    inf = torch.full((1, 2, 1, 64), float("inf"), device="cuda")
    assert not torch.isfinite(ops.rotary(inf, spec)[0, 1]).any()


@gpu
def test_rotary_gradient_formula_and_differences():
    g = torch.Generator(device="cuda").manual_seed(7)
    spec = ops.Rotary(24, scaling="by_parts", factor=4.0, original_length=100)
    pos = torch.randint(0, 500, (2, 9), generator=g, device="cuda")
    q = torch.randn((2, 9, 3, 32), generator=g, device="cuda", requires_grad=True)
    k = torch.randn((2, 9, 1, 32), generator=g, device="cuda", requires_grad=True)
    dq, dk = torch.randn((2, 9, 3, 32), generator=g, device="cuda"), torch.randn((2, 9, 1, 32), generator=g, device="cuda")
    yq, yk = ops.rotary_qk(q, k, spec, positions=pos)
    gq, gk = torch.autograd.grad((yq, yk), (q, k), (dq, dk))
    check_rotary(gq, dq, spec, pos, inverse=True)
    check_rotary(gk, dk, spec, pos, inverse=True)
    # the map is linear: differences along a direction are exact up to rounding
    v = torch.randn((2, 9, 3, 32), generator=g, device="cuda")
    with torch.no_grad():
        along = (ops.rotary(q + v, spec, positions=pos) - ops.rotary(q - v, spec, positions=pos)) / 2
    lhs, rhs = float((along.double() * dq.double()).sum()), float((gq.double() * v.double()).sum())
    # each of the 1728 products is off by at most 2^-20 of its factors (|q| + |v| below 10, |dq| below 5)
    assert abs(lhs - rhs) <= q.numel() * 50 * 2.0 ** -20


def _rotary_c(**over):
    f = (C.c_double * 32)(*([0.5] * 32))
    spec = dict(head_dim=64, rotary_dim=64, layout=0, amplitude=1.0, frequency=f)
    t = dict(x=1 << 20, y=2 << 20, x_batch=64 * 12 * 10, x_row=64 * 12, x_head=64, y_batch=64 * 12 * 10, y_row=64 * 12, y_head=64, heads=12)
    a = dict(dtype=1, batch=2, length=10, n=1, positions=None, pos64=0, pb=0, pt=0)
    second = dict(t, x=4 << 20, y=5 << 20)
    for key, v in over.items():
        group, name = key.split("__")
        {"spec": spec, "t": t, "a": a, "u": second}[group][name] = v
    arr = (L.VtcHeads * 2)(L.VtcHeads(**t), L.VtcHeads(**second))
    rc = L.load().vtc_rotary_heads(0, a["dtype"], C.byref(L.VtcRotary(**spec)), a["batch"], a["length"], arr, a["n"], a["positions"], a["pos64"],
                                   a["pb"], a["pt"], 0, 0, None)
    return rc, L.last_error(None)


@pytest.mark.parametrize("over,text", [
    (dict(a__dtype=3), "type"), (dict(a__n=0), "one or two"), (dict(a__n=3), "one or two"), (dict(a__batch=-1), "negative size"),
    (dict(spec__head_dim=1), "head_dim"), (dict(spec__rotary_dim=63), "rotary_dim"), (dict(spec__rotary_dim=66), "rotary_dim"),
    (dict(spec__layout=2), "layout"), (dict(spec__frequency=None), "frequencies"), (dict(spec__amplitude=float("nan")), "amplitude"),
    (dict(spec__frequency=(C.c_double * 32)(*([float("inf")] * 32))), "frequency 0"),
    (dict(t__x=None), "null"), (dict(t__heads=0), "heads"), (dict(t__x_row=-64), "negative stride"), (dict(t__x=(1 << 20) + 1), "aligned"),
    (dict(t__y_row=0), "overlaps itself"), (dict(t__y_head=32), "overlaps itself"), (dict(t__y_batch=64), "overlaps itself"),
    (dict(t__y=(1 << 20) + 128), "overlap without being the same"), (dict(t__y=1 << 20, t__x_row=0), "overlap without being the same"),
    (dict(a__positions=2, a__pos64=1), "positions"), (dict(a__positions=8, a__pt=-1), "position stride"),
    (dict(a__n=2, u__y=2 << 20), "shares memory"), (dict(a__n=2, u__x=2 << 20, u__y=5 << 20), "shares memory"),
    (dict(a__n=2, u__y=1 << 20), "shares memory"),
    (dict(a__n=2, t__y=1 << 20, u__x=(1 << 20) + 64, u__y=(1 << 20) + 64), "shares memory"),
])
def test_rotary_refusals_of_the_library(over, text):
    rc, msg = _rotary_c(**over)
    assert rc == L.ERR_ARG and text in msg, (rc, msg)


def test_rotary_refusals_of_the_wrapper():
    with pytest.raises(ValueError, match="no CPU path"):
        ops.rotary(torch.zeros(2, 3, 4, 8), ops.Rotary(8))
    with pytest.raises(TypeError):
        ops.rotary(None, ops.Rotary(8))
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=514), dict(rotary_dim=8, layout="full"), dict(rotary_dim=8, scaling="x"),
                dict(rotary_dim=8, base=1.0), dict(rotary_dim=8, scaling="linear", factor=0.0), dict(rotary_dim=8, scaling="by_parts", factor=2.0)):
        with pytest.raises(ValueError):
            ops.Rotary(**bad)


@gpu
def test_rotary_refusals_with_tensors():
    x = torch.zeros((2, 3, 4, 8), device="cuda")
    spec = ops.Rotary(8)
    for bad in (lambda: ops.rotary(x[0, 0], spec), lambda: ops.rotary(x.double(), spec), lambda: ops.rotary(x, ops.Rotary(16)),
                lambda: ops.rotary(x.transpose(2, 3), spec), lambda: ops.rotary(x, spec, positions=torch.zeros(3)),
                lambda: ops.rotary(x, spec, positions=torch.zeros((3, 2), dtype=torch.int64, device="cuda")),
                lambda: ops.rotary(x, spec, positions=torch.zeros(3, dtype=torch.float32, device="cuda")),
                lambda: ops.rotary(x, spec, out=x[:, :, :2]), lambda: ops.rotary_qk(x, x[:, :2], spec), lambda: ops.rotary_qk(x, x.half(), spec),
                lambda: ops.rotary(x.requires_grad_(), spec, out=x)):
        with pytest.raises(ValueError):
            bad()
    x = x.detach()
    y = torch.zeros(2 * 96 + 8, device="cuda")
    with pytest.raises(L.VtcError, match="overlap"):
        ops.rotary(y[:192].view(2, 3, 4, 8), spec, out=y[8:].view(2, 3, 4, 8))


# --------------------------------------------------------------------------------------------- group norm + activation
def act_64(name, z):
    if name == "gelu":
        p = torch.special.ndtr(z)
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name in ("silu", "sigmoid"):
        s = torch.sigmoid(z)
        return (z * s, s * (1 + z * (1 - s))) if name == "silu" else (s, s * (1 - s))
    return z, torch.ones_like(z)


# largest error of the activation and its slope in fp32 arithmetic: 16-bit results use a fit of Phi that is 1.7e-5 off in gelu and
# 0.25 x 1.4e-4 in Phi; 2^-20 covers v_exp_f32 / v_rcp_f32 and the rounding of their arguments (|z s'(z)| below 1)
def act_tol(name, kind):
    return (5e-5 if name == "gelu" and kind != "f32" else 0.0) + 2.0 ** -20


def gn_64(x, groups, w, b, act, lengths, dy=None, eps=1e-5):
    x = x.double().cpu()
    n, t, c = x.shape
    w = torch.ones(c, dtype=torch.float64) if w is None else w.double().cpu()
    b = torch.zeros(c, dtype=torch.float64) if b is None else b.double().cpu()
    lens = [t] * n if lengths is None else [int(v) for v in lengths.cpu().clamp(0, t)]
    out = {k: torch.zeros((n, t, c), dtype=torch.float64) for k in ("y", "dx", "tol_y", "tol_dx")}
    out |= {k: torch.zeros(c, dtype=torch.float64) for k in ("dw", "db", "tol_dw", "tol_db")}
    out["mean"], out["rstd"] = torch.zeros((n, groups), dtype=torch.float64), torch.zeros((n, groups), dtype=torch.float64)
    for i, l in enumerate(lens):
        if l == 0:
            continue
        v = x[i, :l].view(l, groups, -1)
        mean = v.mean((0, 2), keepdim=True)
        rstd = 1 / torch.sqrt(((v - mean) ** 2).mean((0, 2), keepdim=True) + eps)
        out["mean"][i], out["rstd"][i] = mean.flatten(), rstd.flatten()
        h = ((v - mean) * rstd).reshape(l, c)
        z = h * w + b
        y, d = act_64(act, z)
        out["y"][i, :l] = y
        scale = (mean.abs() * rstd).expand(1, groups, c // groups).reshape(1, c)     # the mean's fp32 rounding, in units of the spread
        tz = 2.0 ** -20 * (1 + h.abs() * w.abs() + b.abs()) + 2.0 ** -22 * scale * w.abs()
        out["tol_y"][i, :l] = 1.13 * tz
        if dy is not None:
            g = dy[i, :l].double().cpu()
            dz = g * d
            dh = (dz * w).view(l, groups, -1)
            hh = h.view(l, groups, -1)
            A, B = dh.mean((0, 2), keepdim=True), (dh * hh).mean((0, 2), keepdim=True)
            r = rstd.expand(1, groups, c // groups)
            out["dx"][i, :l] = ((dh - A - hh * B) * r).reshape(l, c)
            out["dw"] += (dz * h).sum(0)
            out["db"] += dz.sum(0)
            # slope off by its own error plus that of z (|act''| below 1.2); A and B are means of terms with the same error
            slope = 1.2 * tz
            e = (g.abs() * slope * w.abs()).view(l, groups, -1)
            eh = (2.0 ** -20 * (1 + h.abs()) + 2.0 ** -22 * scale).view(l, groups, -1)
            spread = (dh.abs() * 2.0 ** -20 + e)
            out["tol_dx"][i, :l] = ((spread + spread.mean((0, 2), keepdim=True) + hh.abs() * (spread * hh.abs() + dh.abs() * eh).mean((0, 2), keepdim=True)
                                     + eh * B.abs() + 2.0 ** -20 * (A.abs() + (hh * B).abs())) * r).reshape(l, c)
            # a thread adds at most 256 rows in fp32, the rest is 64-bit
            out["tol_dw"] += (dz.abs() * h.abs()).sum(0) * 2.0 ** -16 + (g.abs() * slope * h.abs()).sum(0) + (dz.abs() * eh.reshape(l, c)).sum(0)
            out["tol_db"] += dz.abs().sum(0) * 2.0 ** -16 + (g.abs() * slope).sum(0)
    return out


def check_gn(kind, x, groups, w, b, act, lengths, dy, got):
    want = gn_64(x, groups, w, b, act, lengths, dy)
    t = TYPES[kind]
    at = act_tol(act, kind)
    y, mean, rstd, dx, dw, db = got
    # a mean is off by its own rounding plus 2^-20 of the spread; rstd by 2^-18 relative (sums of squares over a row block in fp32)
    spread = 1 / want["rstd"].clamp_min(1e-30)
    close(mean, want["mean"], half_step(torch.float32, want["mean"]) + 2.0 ** -20 * torch.where(want["rstd"] > 0, spread, 0.0) + 2.0 ** -24 * want["mean"].abs(), "mean")
    close(rstd, want["rstd"], want["rstd"] * 2.0 ** -18, "rstd")
    close(y, want["y"], half_step(t, want["y"]) + want["tol_y"] + at, "y")
    if dy is None:
        return
    gmax = dy.double().cpu().abs()
    r = want["rstd"].repeat_interleave(x.shape[2] // groups, 1)[:, None]
    wabs = torch.ones(x.shape[2], dtype=torch.float64) if w is None else w.double().cpu().abs()
    h = torch.nan_to_num((x.double().cpu() - want["mean"].repeat_interleave(x.shape[2] // groups, 1)[:, None]) * r, 0.0, 0.0, 0.0)
    lens = torch.full((x.shape[0],), x.shape[1]) if lengths is None else lengths.cpu().clamp(0, x.shape[1])
    real = (torch.arange(x.shape[1])[None] < lens[:, None])[..., None].double()
    h, gmax = h * real, gmax.nan_to_num(0.0) * real
    # every dz is off by at * |dy|: its own term, and A and B, means whose terms are at most `worst`
    worst = (gmax * wabs).amax((1, 2), keepdim=True) * (1 + h.abs().amax((1, 2), keepdim=True))
    extra = at * r * (gmax * wabs + worst * (1 + h.abs()))
    close(dx, want["dx"], half_step(t, want["dx"]) + want["tol_dx"] + extra, "dx")
    if dw is not None:
        close(dw, want["dw"], half_step(dw.dtype, want["dw"]) + want["tol_dw"] + at * (gmax * h.abs()).sum((0, 1)), "dweight")
    if db is not None:
        close(db, want["db"], half_step(db.dtype, want["db"]) + want["tol_db"] + at * gmax.sum((0, 1)), "dbias")


def run_gn(x, groups, w, b, act, lengths, dy):
    y, mean, rstd = ops.group_norm_act_forward(x, groups, w, b, act=act, lengths=lengths)
    dx = dw = db = None
    if dy is not None:
        dx, dw, db = ops.group_norm_act_backward(dy, x, groups, mean, rstd, w, b, act=act, lengths=lengths)
    return y, mean, rstd, dx, dw, db


GN_SHAPES = [(1, 1, 1, 1), (2, 5, 7, 7), (3, 33, 48, 3), (1, 499, 512, 32), (2, 300, 512, 512), (1, 64, 512, 1), (2, 37, 2056, 8), (1, 70, 8192, 16),
             (4, 129, 24, 6), (70, 3, 16, 2), (2, 1999, 64, 4), (1, 5001, 40, 5), (3, 260, 201, 3)]


@gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n,t,c,groups", GN_SHAPES)
def test_group_norm_forward_and_backward(kind, n, t, c, groups):
    g = torch.Generator(device="cuda").manual_seed(n * 1000 + t)
    act = ("none", "gelu", "silu")[(n + t + c) % 3]
    x = (torch.randn((n, t, c), generator=g, device="cuda") * (torch.rand(c, generator=g, device="cuda") * 2 + 0.1) + torch.randn(c, generator=g, device="cuda")).to(TYPES[kind])
    w, b = (1 + 0.3 * torch.randn(c, generator=g, device="cuda")).to(TYPES[kind]), (0.3 * torch.randn(c, generator=g, device="cuda")).to(TYPES[kind])
    dy = torch.randn((n, t, c), generator=g, device="cuda").to(TYPES[kind])
    check_gn(kind, x, groups, w, b, act, None, dy, run_gn(x, groups, w, b, act, None, dy))


@gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("act", ["none", "gelu", "silu"])
@pytest.mark.parametrize("c,groups", [(64, 4), (64, 64), (45, 5), (512, 32)])
def test_group_norm_padded_batches(kind, act, c, groups):
    """Lengths of zero, one, all and out of range; what lies behind a length is NaN or infinite and must not matter."""
    n, t = 7, 131
    g = torch.Generator(device="cuda").manual_seed(c)
    lengths = torch.tensor([0, 1, t, 64, 130, -5, t + 9], dtype=torch.int32, device="cuda")
    x, dy = (torch.randn((n, t, c), generator=g, device="cuda").to(TYPES[kind]) for _ in range(2))
    behind = torch.arange(t, device="cuda")[None] >= lengths[:, None]
    x[behind], dy[behind] = float("nan"), float("inf")
    w, b = torch.randn(c, generator=g, device="cuda"), torch.randn(c, generator=g, device="cuda")      # an fp32 affine
    got = run_gn(x, groups, w, b, act, lengths, dy)
    assert not got[0][behind].any() and not got[3][behind].any()
    check_gn(kind, x, groups, w, b, act, lengths, dy, got)


@gpu
@pytest.mark.parametrize("kind", list(TYPES))
def test_group_norm_without_affine_strides_in_place_and_empty(kind):
    g = torch.Generator(device="cuda").manual_seed(3)
    wide = torch.randn((2, 50, 3, 96), generator=g, device="cuda").to(TYPES[kind])
    x, dy = wide[:, :, 1], wide[:, :, 2]                                     # rows 288 elements apart
    check_gn(kind, x, 8, None, None, "gelu", None, dy, run_gn(x, 8, None, None, "gelu", None, dy))
    odd = torch.randn((2, 50, 99), generator=g, device="cuda").to(TYPES[kind])[..., 1:97]
    check_gn(kind, odd, 8, None, None, "silu", None, dy, run_gn(odd, 8, None, None, "silu", None, dy))
    shared = torch.randn((1, 50, 96), generator=g, device="cuda").to(TYPES[kind]).expand(3, 50, 96)
    check_gn(kind, shared, 8, None, None, "none", None, None, run_gn(shared, 8, None, None, "none", None, None))
    want = run_gn(x, 8, None, None, "gelu", None, dy)
    z = x.clone()
    y, mean, rstd = ops.group_norm_act_forward(z, 8, act="gelu", out=z)
    assert y is z and torch.equal(z, want[0])
    d = dy.clone()
    dx, _, _ = ops.group_norm_act_backward(d, x, 8, mean, rstd, act="gelu", out=d)
    assert torch.equal(dx, want[3])
    w = torch.ones(96, device="cuda")
    for empty in (x[:0], x[:, :0]):
        y, mean, rstd = ops.group_norm_act_forward(empty, 8, w, w)
        dx, dw, db = ops.group_norm_act_backward(empty, empty, 8, mean, rstd, w, w)
        assert y.shape == dx.shape == empty.shape and not dw.any() and not db.any()


@gpu
def test_group_norm_offset_far_from_zero_and_constant_rows():
    """A mean 1000 times the spread does not cancel; constant rows have rstd = 1 / sqrt(eps)."""
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn((2, 700, 64), generator=g, device="cuda") + 1000.0
    dy = torch.randn((2, 700, 64), generator=g, device="cuda")
    check_gn("f32", x, 4, None, None, "silu", None, dy, run_gn(x, 4, None, None, "silu", None, dy))
    y, mean, rstd = ops.group_norm_act_forward(torch.full((1, 700, 64), 3.0, device="cuda"), 4)
    assert (mean == 3).all() and torch.allclose(rstd, torch.full_like(rstd, 1e-5 ** -0.5)) and not y.any()
    bad = torch.zeros((2, 9, 8), device="cuda")
    bad[0, 3, 1] = float("inf")
    y, _, _ = ops.group_norm_act_forward(bad, 2)
    assert y[0, :, :4].isnan().all() and torch.isfinite(y[0, :, 4:]).all() and torch.isfinite(y[1]).all()


@gpu
def test_group_norm_differentiable_call_against_differences():
    g = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randn((2, 30, 24), generator=g, device="cuda", requires_grad=True)
    w, b = (torch.randn(24, generator=g, device="cuda", requires_grad=True) for _ in range(2))
    lengths = torch.tensor([30, 11], dtype=torch.int32, device="cuda")
    dy = torch.randn((2, 30, 24), generator=g, device="cuda")
    grads = torch.autograd.grad(ops.group_norm_act(x, 3, w, b, act="gelu", lengths=lengths), (x, w, b), dy)
    for i, t in enumerate((x, w, b)):
        v = torch.randn(t.shape, generator=g, device="cuda")
        args = [x.detach(), w.detach(), b.detach()]
        f = []
        for s in (1e-3, -1e-3):
            a = list(args)
            a[i] = args[i] + s * v
            want = gn_64(a[0], 3, a[1], a[2], "gelu", lengths)["y"]
            f.append(float((want * dy.double().cpu()).sum()))
        num = (f[0] - f[1]) / 2e-3
        ana = float((grads[i].double() * v.double()).sum())
        # central differences of a 64-bit definition: the inputs a +- s v are rounded to fp32 (2^-24 / s relative), the third
        # derivative leaves s^2 times a few
        assert abs(num - ana) <= 2e-3 * (abs(num) + float((grads[i].abs() * v.abs()).sum()) ** 0.5 + 1), (i, num, ana)


@gpu
def test_operators_on_a_side_stream_and_in_a_graph():
    """Replays of a captured step give the eager bits, with other work and synchronisation between them."""
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn((3, 700, 96), generator=g, device="cuda").half()
    dy = torch.randn((3, 700, 96), generator=g, device="cuda").half()
    w = torch.randn(96, generator=g, device="cuda").half()
    lengths = torch.tensor([700, 0, 333], dtype=torch.int32, device="cuda")
    spec = ops.Rotary(16)

    def step():
        y, m, r = ops.group_norm_act_forward(x, 6, w, None, act="silu", lengths=lengths)
        q = ops.rotary(y.view(3, 700, 6, 16), spec, offset=5)
        d = ops.rotary(dy.view(3, 700, 6, 16), spec, offset=5, inverse=True)
        return (q,) + ops.group_norm_act_backward(d.view(3, 700, 96), x, 6, m, r, w, None, act="silu", lengths=lengths)[:2]

    eager = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        x.copy_(torch.randn((3, 700, 96), generator=g, device="cuda").half())
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        for a, c in zip(out, want):
            assert torch.equal(a, c)
        (out[0] * 2).sum().item()
    assert not torch.equal(eager[0], out[0])


def _gn_c(backward=False, **over):
    t = dict(x=L.VtcRows3(1 << 20, 6400, 64), y=L.VtcRows3(2 << 20, 6400, 64), dy=L.VtcRows3(3 << 20, 6400, 64))
    a = dict(dtype=1, n=2, l=100, c=64, g=4, w=None, b=None, f32=0, eps=1e-5, act=1, mean=1 << 24, rstd=1 << 24, ws=1 << 25, size=1 << 24)
    for k, v in over.items():
        if k in t:
            t[k] = v
        else:
            a[k] = v
    fp = lambda v: C.c_void_p(v)  # noqa: E731
    ref = lambda s: None if s is None else C.byref(s)  # noqa: E731
    so = L.load()
    if backward:
        rc = so.vtc_group_norm_act_backward(0, a["dtype"], ref(t["dy"]), ref(t["x"]), ref(t["y"]), a["n"], a["l"], a["c"], a["g"], a["w"], a["b"],
                                            a["f32"], a["act"], None, fp(a["mean"]), fp(a["rstd"]), None, None, fp(a["ws"]), a["size"], None)
    else:
        rc = so.vtc_group_norm_act(0, a["dtype"], ref(t["x"]), ref(t["y"]), a["n"], a["l"], a["c"], a["g"], a["w"], a["b"], a["f32"], a["eps"],
                                   a["act"], None, fp(a["mean"]), fp(a["rstd"]), fp(a["ws"]), a["size"], None)
    return rc, L.last_error(None)


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("over,text", [
    (dict(dtype=5), "type"), (dict(f32=2), "affine_f32"), (dict(act=3), "activation"), (dict(act=-1), "activation"), (dict(n=-1), "negative size"),
    (dict(c=0), "channels"), (dict(c=8193), "channels"), (dict(g=5), "groups"), (dict(g=0), "groups"), (dict(x=None), "null"),
    (dict(x=L.VtcRows3(None, 6400, 64)), "null"), (dict(x=L.VtcRows3(1 << 20, -1, 64)), "negative stride"),
    (dict(x=L.VtcRows3((1 << 20) + 1, 6400, 64)), "aligned"), (dict(y=L.VtcRows3(2 << 20, 6400, 63)), "overlaps itself"),
    (dict(y=L.VtcRows3(2 << 20, 0, 64)), "overlaps itself"), (dict(y=L.VtcRows3((1 << 20) + 64, 6400, 64)), "overlap without"),
    (dict(y=L.VtcRows3(1 << 20, 12800, 128)), "overlap without"), (dict(l=1 << 39), "too many rows"),
])
def test_group_norm_refusals_of_the_library(backward, over, text):
    rc, msg = _gn_c(backward, **over)
    assert rc == L.ERR_ARG and text in msg, (rc, msg)


def test_group_norm_refusals_forward_only():
    for over, text, code in ((dict(eps=-1.0), "eps", L.ERR_ARG), (dict(eps=float("nan")), "eps", L.ERR_ARG), (dict(mean=None), "mean", L.ERR_ARG),
                             (dict(size=16), "workspace", L.ERR_CAPACITY), (dict(ws=None), "workspace", L.ERR_CAPACITY), (dict(ws=(1 << 25) + 8), "256", L.ERR_ARG)):
        rc, msg = _gn_c(**over)
        assert rc == code and text in msg, (rc, msg)
    assert L.load().vtc_group_norm_act_workspace(-1, 5, 8, 2, 0) == L.ERR_ARG
    assert L.load().vtc_group_norm_act_workspace(0, 5, 8, 2, 0) == 0


@gpu
def test_group_norm_refusals_with_tensors():
    x = torch.zeros((2, 9, 8), device="cuda")
    w = torch.zeros(8, device="cuda")
    ok = torch.tensor([3, 4], dtype=torch.int32, device="cuda")
    for bad in (lambda: ops.group_norm_act(x[0], 2), lambda: ops.group_norm_act(x, 3), lambda: ops.group_norm_act(x, 2, act="relu"),
                lambda: ops.group_norm_act(x.double(), 2), lambda: ops.group_norm_act(x.transpose(1, 2), 9), lambda: ops.group_norm_act(x, 2, w[:4]),
                lambda: ops.group_norm_act(x, 2, w.half(), w), lambda: ops.group_norm_act(x.half(), 2, w.half(), w),
                lambda: ops.group_norm_act(x, 2, lengths=ok.long()), lambda: ops.group_norm_act(x, 2, lengths=ok[:1]),
                lambda: ops.group_norm_act(x.cpu(), 2), lambda: ops.group_norm_act_forward(x, 2, out=x.half()),
                lambda: ops.group_norm_act_backward(x[:, :4], x, 2, *ops.group_norm_act_forward(x, 2)[1:])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(L.VtcError, match="eps"):
        ops.group_norm_act(x, 2, eps=-1.0)
