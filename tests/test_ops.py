"""The stand-alone operators (vtc_amd.ops): rotary positions and group norm with an activation, against 64-bit definitions.

Tolerances: a result rounded to type t is off by at most eps(t) / 2 of its value; the fp32 arithmetic in front of it is bounded term
by term beside each check.  Refusals run without a GPU (the library checks its arguments before it looks for a device)."""

import copy
import ctypes as C
import math
import pickle

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
    a = pos.double().cpu()[..., None] * torch.tensor(spec.frequency)
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
    angle = (pos.double().cpu().abs()[..., None] * torch.tensor(np.abs(spec.frequency)))[..., None, :]
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


@pytest.mark.parametrize("rotary_dim", [2, 4, 6, 32, 64, 128])
@pytest.mark.parametrize("base", [100.0, 10000.0, 500000.0])
@pytest.mark.parametrize("length", [1, 3, 6, 7, 30, 200, 201, 202, 2048, 47_000, 48_000, 100_000, 3_000_000])
def test_rotary_by_parts_frequencies_by_counting_turns(rotary_dim, base, length):
    """The ramp's ends found by counting turns over the original length, pair by pair, on an index that runs on past the last pair."""
    r, s = rotary_dim, 8.0
    spec = ops.Rotary(r, base=base, scaling="by_parts", factor=s, original_length=length)
    turns = [length * base ** (-2.0 * j / r) / (2.0 * math.pi) for j in range(r)]
    if any(abs(t - e) < 1e-9 * e for t in turns for e in (1.0, 32.0)):
        pytest.skip("a pair on the border itself")
    low = max([j for j in range(r) if turns[j] > 32.0], default=0)
    high = min([j for j in range(r) if turns[j] < 1.0], default=r - 1)
    for j in range(r // 2):
        f = base ** (-2.0 * j / r)
        share = 1.0 if j >= high else 0.0 if j <= low else (j - low) / (high - low)   # of the division by the factor
        assert spec.frequency[j] == pytest.approx(f * (1.0 - share) + f / s * share, rel=1e-12), j
        if turns[j] < 1.0:
            assert spec.frequency[j] == pytest.approx(f / s, rel=1e-12), j
        if turns[j] > 32.0:
            assert spec.frequency[j] == pytest.approx(f, rel=1e-12), j
    assert spec.amplitude == pytest.approx(1.0 + 0.1 * math.log(s))


@pytest.mark.parametrize("rotary_dim", [4, 64, 128])
def test_rotary_ntk_and_linear_frequencies(rotary_dim):
    """ntk leaves the first pair alone, divides the last one by the factor and spaces the others evenly in the logarithm between."""
    r, s = rotary_dim, 8.0
    plain, ntk, linear = (ops.Rotary(r, scaling=k, factor=s) for k in ("none", "ntk", "linear"))
    j = np.arange(r // 2)
    assert np.allclose(plain.frequency, 10000.0 ** (-j / (r / 2)), rtol=1e-13, atol=0)
    assert np.allclose(ntk.frequency, plain.frequency * s ** (-j / (r / 2 - 1)), rtol=1e-12, atol=0)
    assert np.allclose(linear.frequency * s, plain.frequency, rtol=1e-13, atol=0)
    assert plain.amplitude == ntk.amplitude == linear.amplitude == 1.0


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


def test_rotary_description_is_copied_and_pickled_without_addresses():
    spec = ops.Rotary(48, layout="interleaved", scaling="by_parts", factor=8.0, original_length=500)
    first = spec._struct(64)
    for other in (copy.deepcopy(spec), copy.copy(spec), pickle.loads(pickle.dumps(spec))):
        assert np.array_equal(other.frequency, spec.frequency) and not other.frequency.flags.writeable
        s = other._struct(64)
        assert (s.rotary_dim, s.layout, s.amplitude) == (first.rotary_dim, first.layout, first.amplitude)
        assert C.cast(s.frequency, C.c_void_p).value == other.frequency.ctypes.data != spec.frequency.ctypes.data


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
@pytest.mark.parametrize("n,t,c,groups", [(2, 8000, 32, 2), (2, 8192, 16, 16), (2, 8193, 16, 16), (3, 700, 128, 4), (2, 500, 128, 2), (2, 2049, 64, 8),
                                          (9, 1, 64, 4), (2, 515, 128, 1)])
def test_group_norm_samples_that_fit_on_chip_and_just_do_not(kind, n, t, c, groups):
    test_group_norm_forward_and_backward(kind, n, t, c, groups)


@gpu
@pytest.mark.parametrize("kind", list(TYPES))
def test_group_norm_sample_does_not_depend_on_its_batch(kind):
    g = torch.Generator(device="cuda").manual_seed(21)
    for t, c, groups in ((300, 64, 4), (9000, 32, 2), (130, 45, 5)):
        x, dy = (torch.randn((5, t, c), generator=g, device="cuda").to(TYPES[kind]) for _ in range(2))
        y, m, r = ops.group_norm_act_forward(x, groups, act="gelu")
        dx, _, _ = ops.group_norm_act_backward(dy, x, groups, m, r, act="gelu")
        y1, m1, r1 = ops.group_norm_act_forward(x[3:4], groups, act="gelu")
        assert torch.equal(y[3:4], y1) and torch.equal(m[3:4], m1)
        assert torch.equal(dx[3:4], ops.group_norm_act_backward(dy[3:4], x[3:4], groups, m1, r1, act="gelu")[0])


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


# --------------------------------------------------------------------------------------------- gated feed-forward
def ffn_64(x, wg, wu, wd, bg, bu, bd, act, dy=None):
    x, wg, wu, wd = (t.double() for t in (x, wg, wu, wd))
    z = lambda t: 0.0 if t is None else t.double()  # noqa: E731
    g, u = x @ wg.t() + z(bg), x @ wu.t() + z(bu)
    a, d = act_64(act, g)
    h = a * u
    out = {"y": h @ wd.t() + z(bd)}
    if dy is not None:
        dy = dy.double()
        dh = dy @ wd
        dg, du = dh * u * d, dh * a
        out |= {"dx": dg @ wg + du @ wu, "dw_gate": dg.t() @ x, "dw_up": du.t() @ x, "dw_down": dy.t() @ h, "db_gate": dg.sum(0),
                "db_up": du.sum(0), "db_down": dy.sum(0)}
    return out


def ffn_tolerances(x, wg, wu, wd, bg, bu, bd, act, dy, kind):
    """Worst case of every rounding, carried through the formulas with absolute values.  e = half a step of the type for what is
    stored between the products (h; g, u, dg, du in the backward pass), s = fp32 sums: at most n 2^-24 of the sum of magnitudes."""
    e = torch.finfo(kind).eps / 2
    tiny = torch.finfo(kind).smallest_normal * torch.finfo(kind).eps
    x, wg, wu, wd = (t.double() for t in (x, wg, wu, wd))
    z = lambda t: 0.0 if t is None else t.double()  # noqa: E731
    m, k = x.shape
    f, n = wd.shape[1], wd.shape[0]
    s = lambda c: (c + 16) * 2.0 ** -24  # noqa: E731
    at = act_tol(act, "bf16")
    g, u = x @ wg.t() + z(bg), x @ wu.t() + z(bu)
    ag, au = x.abs() @ wg.abs().t() + abs(z(bg)), x.abs() @ wu.abs().t() + abs(z(bu))
    a, d = act_64(act, g)
    eg, eu = ag * s(k), au * s(k)                        # g and u in fp32
    ea = 1.13 * eg + at                                  # slopes of the activations are below 1.13
    h = a * u
    eh = ea * u.abs() + a.abs() * eu + ea * eu + e * h.abs() + tiny
    tol = {"y": eh @ wd.abs().t() + (h.abs() + eh) @ wd.abs().t() * s(f) + abs(z(bd)) * 2.0 ** -24}
    if dy is not None:
        dy = dy.double()
        egr, eur = eg + e * g.abs() + tiny, eu + e * u.abs() + tiny          # g and u as stored
        dh, adh = dy @ wd, dy.abs() @ wd.abs()
        edh = adh * s(n)
        ed, ear = 1.2 * egr + at, 1.13 * egr + at                            # |act''| is below 1.2
        dg, du = dh * u * d, dh * a
        edg = edh * (u.abs() + eur) * (d.abs() + ed) + dh.abs() * (eur * (d.abs() + ed) + u.abs() * ed) + e * dg.abs() + tiny
        edu = edh * (a.abs() + ear) + dh.abs() * ear + e * du.abs() + tiny
        prod = lambda err, val, w: err @ w.abs() + (val.abs() + err) @ w.abs() * s(w.shape[0])  # noqa: E731
        tol["dx"] = prod(edg, dg, wg) + prod(edu, du, wu)
        tol["dw_gate"], tol["dw_up"] = prod(edg.t(), dg.t(), x), prod(edu.t(), du.t(), x)
        tol["dw_down"] = prod(torch.zeros_like(dy.t()), dy.t(), h) + dy.abs().t() @ eh
        tol["db_gate"], tol["db_up"] = edg.sum(0) + dg.abs().sum(0) * s(256), edu.sum(0) + du.abs().sum(0) * s(256)
        tol["db_down"] = dy.abs().sum(0) * s(256)
    return tol


def make_ffn(kind, m, k, f, n, bias, seed=0, bias_kind=None):
    g = torch.Generator(device="cuda").manual_seed(seed + m + 7 * k + 13 * f)
    r = lambda *shape, std=1.0: (torch.randn(shape, generator=g, device="cuda") * std)  # noqa: E731
    x, dy = r(m, k).to(kind), r(m, n).to(kind)
    w = (r(f, k, std=k ** -0.5).to(kind), r(f, k, std=k ** -0.5).to(kind), r(n, f, std=f ** -0.5).to(kind))
    b = tuple((r(c, std=0.3).to(bias_kind or kind) if bias else None) for c in (f, f, n))
    return x, w, b, dy


NAMES = ("dx", "dw_gate", "dw_up", "dw_down", "db_gate", "db_up", "db_down")


def check_ffn(kind, x, w, b, act, dy, y, grads):
    want = ffn_64(x, *w, *b, act, dy)
    tol = ffn_tolerances(x, *w, *b, act, dy, kind)
    for name, got in (("y", y),) + tuple(zip(NAMES, grads or ())):
        if got is not None:
            ref = want[name].cpu()
            close(got, ref, half_step(got.dtype, ref) + tol[name].cpu() * 1.001, name)


FFN_SIZES = [(1, 64, 64, 64), (1, 8, 8, 8), (3, 1, 1, 1), (16, 768, 2048, 768), (17, 40, 72, 24), (33, 389, 131, 77), (64, 256, 512, 256),
             (65, 256, 512, 256), (200, 64, 128, 192), (257, 129, 250, 311), (511, 768, 512, 768), (1030, 100, 300, 50), (2048, 192, 384, 192)]


@gpu
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("m,k,f,n", FFN_SIZES)
def test_gated_ffn_forward_and_backward(kind, m, k, f, n):
    act = ("silu", "gelu", "sigmoid", "none")[(m + f) % 4]
    bias = (m + k) % 3 != 0
    x, w, b, dy = make_ffn(TYPES[kind], m, k, f, n, bias)
    y, saved = ops.gated_ffn_forward(x, *w, *b, act=act, save=True)
    y2, none = ops.gated_ffn_forward(x, *w, *b, act=act)
    assert none is None and torch.equal(y, y2)
    grads = ops.gated_ffn_backward(dy, x, *w, saved, act=act, biases=bias)
    check_ffn(TYPES[kind], x, w, b, act, dy, y, grads)


@gpu
@pytest.mark.parametrize("act", ["none", "gelu", "silu", "sigmoid"])
@pytest.mark.parametrize("m", [5, 300])
def test_gated_ffn_activations_and_fp32_biases(act, m):
    x, w, b, dy = make_ffn(torch.float16, m, 96, 160, 96, True, bias_kind=torch.float32)
    y, saved = ops.gated_ffn_forward(x, *w, *b, act=act, save=True)
    grads = ops.gated_ffn_backward(dy, x, *w, saved, act=act, bias_dtype=torch.float32)
    check_ffn(torch.float16, x, w, b, act, dy, y, grads)


@gpu
@pytest.mark.parametrize("bits", [0x7FFFFFFF, -1, 0x7F800001, 0x7F800000])   # NaN of both signs with every bit set, the least one, inf
@pytest.mark.parametrize("m,k,f", [(5, 64, 136), (300, 64, 136), (9000, 768, 2048)])
def test_gated_ffn_gradients_of_bias_values_that_are_no_numbers(bits, m, k, f):
    for which in (0, 1):
        x, w, b, dy = make_ffn(torch.bfloat16, m, k, f, k, True, bias_kind=torch.float32)
        b[which].view(torch.int32)[77] = bits
        y, saved = ops.gated_ffn_forward(x, *w, *b, act="sigmoid", save=True)
        dx, dwg, dwu, dwd, dbg, dbu, _ = ops.gated_ffn_backward(dy, x, *w, saved, act="sigmoid", bias_dtype=torch.float32)
        clean = torch.arange(f, device="cuda") != 77
        for t in (dwg[clean], dwu[clean], dwd[:, clean], dbg[clean], dbu[clean]):
            assert torch.isfinite(t).all()
        nan = bits != 0x7F800000
        if which == 0:     # sigmoid(inf) = 1 with slope 0
            assert torch.isnan(y).all() == nan and torch.isfinite(y).all() != nan
            assert torch.isnan(dx).all() == nan and torch.isfinite(dx).all() != nan
            assert torch.isnan(dwg[77]).all() == nan and torch.isnan(dbg[77]) == nan and torch.isnan(dwu[77]).all() == nan
        else:              # u = inf: h and dg are infinite, so sums over them are inf or NaN; du does not depend on u
            assert not torch.isfinite(y).any() and not torch.isfinite(dx).any() and not torch.isfinite(dwg[77]).any()
            assert torch.isfinite(dwu[77]).all() and torch.isfinite(dbu[77]) and not torch.isfinite(dwd[:, 77]).any()


@gpu
@pytest.mark.parametrize("bits", [0x7FFF, -1])   # NaN of both signs with every bit set
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("m,k,f", [(5, 64, 136), (300, 64, 136), (9000, 768, 2048)])
def test_gated_ffn_gradients_of_a_row_that_is_no_number(kind, bits, m, k, f):
    x, w, b, dy = make_ffn(TYPES[kind], m, k, f, k, True)
    x.view(torch.int16)[2, 11] = bits
    y, saved = ops.gated_ffn_forward(x, *w, *b, save=True)
    dx, dwg, dwu, dwd, dbg, dbu, dbd = ops.gated_ffn_backward(dy, x, *w, saved)
    clean = torch.arange(m, device="cuda") != 2
    assert torch.isnan(y[2]).all() and torch.isnan(dx[2]).all() and torch.isfinite(y[clean]).all() and torch.isfinite(dx[clean]).all()
    assert all(torch.isnan(t).all() for t in (dwg, dwu, dwd, dbg, dbu)) and torch.isfinite(dbd).all()


@gpu
@pytest.mark.parametrize("m", [1, 40, 700])
def test_gated_ffn_strides_shapes_and_partial_gradients(m):
    kind = torch.bfloat16
    x, w, b, dy = make_ffn(kind, m, 96, 160, 64, True)
    want, saved = ops.gated_ffn_forward(x, *w, *b, save=True)
    grads = ops.gated_ffn_backward(dy, x, *w, saved)
    wide = torch.zeros((m, 3 * 96), dtype=kind, device="cuda")
    wide[:, 96:192] = x
    for view in (wide[:, 96:192], torch.cat([x, x], 1)[:, :96]):               # rows that are further apart
        assert torch.equal(ops.gated_ffn_forward(view, *w, *b)[0], want)
    off = torch.zeros(m * 96 + 1, dtype=kind, device="cuda")[1:].view(m, 96)    # rows that are not aligned to 16 bytes
    off.copy_(x)
    wide_w = torch.zeros((160, 2, 96), dtype=kind, device="cuda")               # gate and up interleaved row by row
    wide_w[:, 0], wide_w[:, 1] = w[0], w[1]
    odd_w = torch.zeros(64 * 163 + 1, dtype=kind, device="cuda")[1:].view(64, 163)[:, :160]
    odd_w.copy_(w[2])
    y, s2 = ops.gated_ffn_forward(off, wide_w[:, 0], wide_w[:, 1], odd_w, *b, save=True)
    assert torch.equal(y, want)
    for a, c in zip(ops.gated_ffn_backward(dy, off, wide_w[:, 0], w[1].clone(), odd_w, s2), grads):
        assert torch.equal(a, c)
    y3 = ops.gated_ffn(x.view(1, m, 1, 96), *w, *b)
    assert y3.shape == (1, m, 1, 64) and torch.equal(y3.view(m, 64), want)
    for kw in (dict(need_dx=False), dict(need_dw=False), dict(biases=False)):
        got = ops.gated_ffn_backward(dy, x, *w, saved, **kw)
        for i, (a, c) in enumerate(zip(got, grads)):
            gone = (i == 0 and "need_dx" in kw) or (1 <= i <= 3 and "need_dw" in kw) or (i >= 4 and "biases" in kw)
            assert a is None if gone else torch.equal(a, c)
    y, s = ops.gated_ffn_forward(x[:0], *w, *b, save=True)
    assert y.shape == (0, 64)
    assert not any(t.any() for t in ops.gated_ffn_backward(dy[:0], x[:0], *w, s)[1:])


@gpu
def test_gated_ffn_rows_do_not_reach_each_other():
    """An infinite row stays alone, in every kernel the rows can take; so do rows next to the end of a tile."""
    for m in (40, 300):
        x, w, b, _ = make_ffn(torch.float16, m, 100, 132, 60, True)
        want = ops.gated_ffn(x, *w, *b)
        x[7] = float("nan")
        got = ops.gated_ffn(x, *w, *b)
        assert got[7].isnan().all() and torch.equal(got[:7], want[:7]) and torch.equal(got[8:], want[8:])


@gpu
def test_gated_ffn_differentiable_call_formula_and_differences():
    x, w, b, dy = make_ffn(torch.float16, 70, 48, 64, 40, True)
    leaves = [t.detach().clone().requires_grad_() for t in (x,) + w + b]
    y = ops.gated_ffn(*leaves, act="gelu")
    grads = torch.autograd.grad(y, leaves, dy)
    check_ffn(torch.float16, x, w, b, "gelu", dy, y.detach(), grads)
    only = ops.gated_ffn(x, w[0], w[1], w[2], leaves[4], None, None, act="gelu")
    (db,) = torch.autograd.grad(only, (leaves[4],), dy)
    assert db.shape == (64,)
    # central differences of the 64-bit definition along a direction, against the returned gradients
    g = torch.Generator(device="cuda").manual_seed(11)
    tol = ffn_tolerances(x, *w, *b, "gelu", dy, torch.float16)
    base = [t.double() for t in (x,) + w + b]
    for i, name in enumerate(NAMES):
        v = torch.randn(base[i].shape, generator=g, device="cuda", dtype=torch.float64)
        f = [float((ffn_64(*(t + (s * v if j == i else 0) for j, t in enumerate(base)), "gelu")["y"] * dy.double()).sum()) for s in (1e-4, -1e-4)]
        num, ana = (f[0] - f[1]) / 2e-4, float((grads[i].double() * v).sum())
        room = float(((tol[name] + half_step(torch.float16, grads[i].double())) * v.abs()).sum())
        assert abs(num - ana) <= room + 1e-5 * abs(num) + 1e-4, (name, num, ana, room)   # 64-bit differences: 1e-16 / 1e-4 and 1e-8 of f'''


@gpu
def test_gated_ffn_long_contraction_offsets_beyond_32_bits():
    """rows x inner beyond 2^31 elements: the last rows and the sums over all of them are right."""
    m, k, f, n = 1_100_000, 8, 2048, 8
    g = torch.Generator(device="cuda").manual_seed(12)
    kind = torch.bfloat16
    x = torch.zeros((m, k), dtype=kind, device="cuda")
    dy = torch.zeros((m, n), dtype=kind, device="cuda")
    x[-300:], dy[-300:] = torch.randn((300, k), generator=g, device="cuda").to(kind), torch.randn((300, n), generator=g, device="cuda").to(kind)
    w = tuple((torch.randn(s, generator=g, device="cuda") * s[1] ** -0.5).to(kind) for s in ((f, k), (f, k), (n, f)))
    y, saved = ops.gated_ffn_forward(x, *w, save=True)
    grads = ops.gated_ffn_backward(dy, x, *w, saved, biases=False)
    assert not y[:-300].any() and not grads[0][:-300].any()
    check_ffn(kind, x[-300:], w, (None,) * 3, "silu", dy[-300:], y[-300:], (grads[0][-300:],) + grads[1:4])


@gpu
def test_gated_ffn_in_a_graph():
    x, w, b, dy = make_ffn(torch.bfloat16, 600, 136, 200, 136, True)

    def step():
        y, saved = ops.gated_ffn_forward(x, *w, *b, act="gelu", save=True)
        small = ops.gated_ffn_forward(x[:9], *w, *b, act="gelu")[0]
        return (y, small) + ops.gated_ffn_backward(dy, x, *w, saved, act="gelu")

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        x.mul_(-0.9)
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        assert all(torch.equal(a, c) for a, c in zip(out, want))
        (out[0].float() * 2).sum().item()


@gpu
def test_calls_on_two_streams_at_once_do_not_disturb_each_other():
    """Each call brings its own workspace: interleaved calls on two streams give the bits of lone ones."""
    g = torch.Generator(device="cuda").manual_seed(31)
    sets = []
    for i in range(2):
        x, w, b, dy = make_ffn(torch.float16, 900, 264, 520, 264, True, seed=i)
        n = torch.randn((4, 3000, 48), generator=g, device="cuda").half()
        sets.append((x, w, b, dy, n))

    def work(x, w, b, dy, n):
        y, saved = ops.gated_ffn_forward(x, *w, *b, save=True)
        out = (y,) + ops.gated_ffn_backward(dy, x, *w, saved)
        z, m, r = ops.group_norm_act_forward(n, 3, act="silu")
        return out + (z, ops.group_norm_act_backward(n, n, 3, m, r, act="silu")[0], ops.rotary(z.view(4, 3000, 3, 16), ops.Rotary(16)))

    want = [[t.clone() for t in work(*s)] for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(work(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert all(torch.equal(a, c) for a, c in zip(out, want[i]))


@gpu
def test_rotary_and_group_norm_beyond_32_bit_offsets():
    """More than 2^31 elements: the last rows are those of a call on them alone."""
    spec = ops.Rotary(64)
    x = torch.zeros((1, 130_000, 130, 128), dtype=torch.float16, device="cuda")
    tail = torch.randn((1, 40, 130, 128), device="cuda").half()
    x[:, -40:] = tail
    y = ops.rotary(x, spec)
    assert x.numel() > 2 ** 31 and torch.equal(y[:, -40:], ops.rotary(tail, spec, offset=130_000 - 40)) and not y[:, :40].any()
    del x, y
    z = torch.zeros((3, 1_450_000, 512), dtype=torch.bfloat16, device="cuda")
    z[2].normal_()
    y, m, r = ops.group_norm_act_forward(z, 16, act="gelu")
    y2, m2, r2 = ops.group_norm_act_forward(z[2:], 16, act="gelu")
    assert z.numel() > 2 ** 31 and torch.equal(y[2:], y2) and torch.equal(r[2:], r2) and not y[:2].any()
    assert abs(float(y2.float().mean()) - 0.2821) < 1e-3      # E[gelu(standard normal)] = 1 / (2 sqrt(pi)); 7e8 values
    del y
    dx, _, _ = ops.group_norm_act_backward(z, z, 16, m, r, act="gelu")
    assert torch.equal(dx[2:], ops.group_norm_act_backward(z[2:], z[2:], 16, m2, r2, act="gelu")[0])


@gpu
def test_rotary_between_columns_of_one_buffer():
    """Input and output interleaved in the rows of one buffer share no element and are taken; shared ones are refused."""
    g = torch.Generator(device="cuda").manual_seed(33)
    rows = torch.randn((2, 30, 4 * 64 * 2), generator=g, device="cuda").half()
    x, y = rows[..., :256].unflatten(-1, (4, 64)), rows[..., 256:].unflatten(-1, (4, 64))
    keep = x.clone()
    ops.rotary(x, ops.Rotary(64), out=y)
    assert torch.equal(x, keep)
    check_rotary(y, keep, ops.Rotary(64), torch.arange(30).expand(2, 30))
    with pytest.raises(L.VtcError, match="overlap"):
        ops.rotary(x, ops.Rotary(64), out=rows[..., 192:448].unflatten(-1, (4, 64)))


def _ffn_c(backward=False, **over):
    a = dict(dtype=1, m=100, k=64, f=128, n=64, f32=0, act=2, x=L.VtcMat(1 << 20, 64), wg=L.VtcMat(2 << 20, 64), wu=L.VtcMat(3 << 20, 64),
             wd=L.VtcMat(4 << 20, 128), y=L.VtcMat(5 << 20, 64), saved=6 << 20, saved_size=1 << 20, ws=8 << 20, size=1 << 30, dx=7 << 20, dx_row=64, dw=1 << 28,
             dw2=(1 << 28) + (1 << 20), dw3=(1 << 28) + (2 << 20))
    a.update(over)
    ref = lambda s: None if s is None else C.byref(s)  # noqa: E731
    so = L.load()
    mats = [ref(a[n]) for n in ("x", "wg", "wu", "wd")]
    if backward:
        grads = L.VtcFfnGrads(a["dx"], a["dx_row"], a["dw"], a["dw2"], a["dw3"])
        rc = so.vtc_gated_ffn_backward(0, a["dtype"], a["m"], a["k"], a["f"], a["n"], ref(a["y"]), *mats, a["saved"], a["saved_size"], a["f32"],
                                       C.byref(grads), a["ws"], a["size"], None)
    else:
        rc = so.vtc_gated_ffn(0, a["dtype"], a["m"], a["k"], a["f"], a["n"], *mats, None, None, None, a["f32"], a["act"], ref(a["y"]), a["saved"],
                              a["saved_size"], a["ws"], a["size"], None)
    return rc, L.last_error(None)


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("over,text,code", [
    (dict(dtype=0), "f16 or bf16", L.ERR_ARG), (dict(f32=2), "bias_f32", L.ERR_ARG),
    (dict(m=-1), "rows", L.ERR_ARG), (dict(m=1 << 31), "rows", L.ERR_ARG), (dict(k=0), "width", L.ERR_ARG), (dict(f=(1 << 18) + 1), "width", L.ERR_ARG),
    (dict(x=None), "x is null", L.ERR_ARG), (dict(wg=L.VtcMat(None, 64)), "w_gate is null", L.ERR_ARG), (dict(wd=L.VtcMat(4 << 20, 127)), "pitch", L.ERR_ARG),
    (dict(x=L.VtcMat(1 << 20, (1 << 20) + 1)), "pitch", L.ERR_ARG), (dict(x=L.VtcMat((1 << 20) + 1, 64)), "aligned", L.ERR_ARG),
    (dict(y=L.VtcMat(5 << 20, 63)), "pitch", L.ERR_ARG), (dict(size=10, x=L.VtcMat((1 << 20) + 2, 64)), "workspace", L.ERR_CAPACITY),
    (dict(saved_size=10), "saved", L.ERR_CAPACITY), (dict(ws=(8 << 20) + 16), "256", L.ERR_ARG), (dict(saved=(6 << 20) + 16), "256", L.ERR_ARG)])
def test_gated_ffn_refusals_of_the_library(backward, over, text, code):
    rc, msg = _ffn_c(backward, **over)
    assert rc == code and text in msg, (rc, msg)


def test_gated_ffn_refusals_of_one_direction():
    for backward, over, text in ((False, dict(y=L.VtcMat((1 << 20) + 64, 64)), "overlaps x"), (False, dict(act=4), "activation"), (True, dict(dx=1 << 20), "overlaps"),
                                 (True, dict(dx=5 << 20), "overlaps"), (True, dict(dx_row=63), "pitch"), (True, dict(dw=None), "go together"),
                                 (True, dict(m=0), "no rows"), (True, dict(dx=(7 << 20) + 1), "aligned"), (False, dict(y=L.VtcMat(4 << 20, 64)), "overlaps w_down"),
                                 (True, dict(dw=2 << 20), "overlaps w_gate"), (True, dict(dw2=1 << 28), "overlaps dw_gate"),
                                 (True, dict(dw3=5 << 20), "overlaps dy"), (False, dict(m=1 << 30, f=1 << 18, wd=L.VtcMat(4 << 20, 1 << 18)), "too many")):
        rc, msg = _ffn_c(backward, **over)
        assert rc == L.ERR_ARG and text in msg, (rc, msg)
    so = L.load()
    assert so.vtc_gated_ffn_workspace(10, 0, 8, 8, 0) == L.ERR_ARG and so.vtc_gated_ffn_workspace(0, 8, 8, 8, 1) == 0
    assert so.vtc_gated_ffn_saved(-1, 8) == L.ERR_ARG


@gpu
def test_gated_ffn_refusals_with_tensors():
    x, w, b, dy = make_ffn(torch.float16, 6, 16, 24, 8, True)
    y, saved = ops.gated_ffn_forward(x, *w, *b, save=True)
    for bad in (lambda: ops.gated_ffn(x.float(), *w), lambda: ops.gated_ffn(x, w[0].bfloat16(), w[1], w[2]), lambda: ops.gated_ffn(x[:, :8], *w),
                lambda: ops.gated_ffn(x, w[0], w[1][:8], w[2]), lambda: ops.gated_ffn(x, w[0], w[1], w[2].t()), lambda: ops.gated_ffn(x, *w, act="relu"),
                lambda: ops.gated_ffn(x, w[0].t().contiguous().t(), w[1], w[2]), lambda: ops.gated_ffn(x, *w, b[0][:4]),
                lambda: ops.gated_ffn(x, *w, b[0], b[1].float()), lambda: ops.gated_ffn(x.cpu(), *w), lambda: ops.gated_ffn_backward(dy, x, *w, None),
                lambda: ops.gated_ffn_backward(dy[:3], x, *w, saved), lambda: ops.gated_ffn_backward(dy, x, *w, saved[:100]),
                lambda: ops.gated_ffn_backward(dy, x, *w, saved, bias_dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("backward", [False, True])
def test_gated_ffn_pitch_of_a_single_row_is_not_looked_at(backward):
    """x[:, -1] of a long recording.  No such device: what the argument checks let pass goes no further."""
    so, far = L.load(), 1_536_000
    mat = lambda at, row: C.byref(L.VtcMat(at, row))  # noqa: E731
    for rows, pitch, ok in ((1, far, True), (1, 0, True), (1, -5, True), (2, far, False), (2, 767, False)):
        x, w = mat(1 << 20, pitch), (mat(4 << 20, 768), mat(8 << 20, 768), mat(12 << 20, 256))
        if backward:
            grads = L.VtcFfnGrads(1 << 28, pitch, None, None, None)
            rc = so.vtc_gated_ffn_backward(-1, 1, rows, 768, 256, 768, mat(16 << 20, pitch), x, *w, 32 << 20, 1 << 20, 0, C.byref(grads), 64 << 20, 1 << 27, None)
        else:
            rc = so.vtc_gated_ffn(-1, 1, rows, 768, 256, 768, x, *w, None, None, None, 0, 2, mat(16 << 20, pitch), None, 0, 64 << 20, 1 << 27, None)
        msg = L.last_error(None)
        assert rc != 0 and ("device" in msg if ok else "pitch" in msg), (rows, pitch, msg)


@gpu
@pytest.mark.parametrize("batch", [1, 2, 8, 70])
def test_gated_ffn_on_the_last_frames_of_long_recordings(batch):
    t, k, f = 2000, 768, 256
    x, w, b, dy = make_ffn(torch.float16, batch, k, f, k, True)
    wide, wide_dy = (torch.zeros((batch, t, k), dtype=torch.float16, device="cuda") for _ in range(2))
    wide[:, -1], wide_dy[:, -1] = x, dy
    want, saved = ops.gated_ffn_forward(x, *w, *b, save=True)
    grads = ops.gated_ffn_backward(dy, x, *w, saved)
    for view, dview in ((wide[:, -1], wide_dy[:, -1]), (wide[:, -1:], wide_dy[:, -1:])):
        y, s = ops.gated_ffn_forward(view, *w, *b, save=True)
        assert y.shape == view.shape and torch.equal(y.view(batch, k), want)
        got = ops.gated_ffn_backward(dview, view, *w, s)
        assert got[0].shape == view.shape and torch.equal(got[0].reshape(batch, k), grads[0])
        assert all(torch.equal(a, c) for a, c in zip(got[1:], grads[1:]))


@gpu
@pytest.mark.parametrize("call", ["rotary", "rotary_qk", "group_norm_act", "gated_ffn"])
def test_forward_mode_tangents_are_refused(call):
    forward_ad = torch.autograd.forward_ad
    x, w, b, _ = make_ffn(torch.float16, 6, 16, 24, 16, True)
    h = x.view(1, 6, 1, 16)
    calls = {"rotary": lambda t: ops.rotary(t.view(1, 6, 1, 16), ops.Rotary(16)), "rotary_qk": lambda t: ops.rotary_qk(h, t.view(1, 6, 1, 16), ops.Rotary(16)),
             "group_norm_act": lambda t: ops.group_norm_act(t.view(1, 6, 16), 2), "gated_ffn": lambda t: ops.gated_ffn(t, *w, *b)}
    plain = calls[call](x)
    with forward_ad.dual_level():
        again = calls[call](x)
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError):
            calls[call](dual)
        with pytest.raises(ValueError, match="no gradient"):
            ops.rotary(dual.view(1, 6, 1, 16), ops.Rotary(16), out=torch.empty_like(h))
    for a, c in zip(plain if isinstance(plain, tuple) else (plain,), again if isinstance(again, tuple) else (again,)):
        assert torch.equal(a, c)


@gpu
@pytest.mark.parametrize("call", ["rotary", "rotary_qk", "group_norm", "group_norm_backward"])
def test_writing_through_out_is_seen_by_autograd(call):
    """A value that an earlier operation keeps for its gradient is overwritten: the gradient refuses, as for torch's own operations."""
    leaf = torch.randn((2, 5, 24), device="cuda", requires_grad=True)
    y = leaf * 2
    z = (y * y).sum()
    d = y.detach()
    heads = d.view(2, 5, 3, 8)
    spec = ops.Rotary(8)
    if call == "rotary":
        assert ops.rotary(heads, spec, out=heads) is heads
    elif call == "rotary_qk":
        ops.rotary_qk(torch.zeros_like(heads), heads, spec, out=(torch.empty_like(heads), heads))
    else:
        x = torch.randn_like(d)
        _, mean, rstd = ops.group_norm_act_forward(x, 3, out=d if call == "group_norm" else None)
        if call == "group_norm_backward":
            ops.group_norm_act_backward(x, x, 3, mean, rstd, out=d)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
    # a tensor that itself requires a gradient is not written to while gradients are recorded
    for bad in (lambda: ops.rotary(heads, spec, out=y.view(2, 5, 3, 8)), lambda: ops.group_norm_act_forward(d, 3, out=y)):
        with pytest.raises(ValueError, match="no gradient"):
            bad()
    with torch.no_grad():
        assert ops.group_norm_act_forward(d, 3, out=y)[0] is y


@gpu
@pytest.mark.parametrize("n,c,groups", [((1 << 18) + 3, 512, 32), ((1 << 19) + 5, 512, 32), ((1 << 24) + 9, 8, 1), ((1 << 22) + 1, 24, 12)])
def test_group_norm_of_more_samples_than_a_launch_holds(n, c, groups):
    """Single frames, more of them than 2^32 threads take: the kernels go in several launches each.  The borders of 512-, 256- and 1024-thread
    kernels; a sample's bits are those of a call on a few samples alone, and the affine's gradients are sums over all."""
    g = torch.Generator(device="cuda").manual_seed(c)
    x, dy = (torch.randn((n, 1, c), generator=g, device="cuda").half() for _ in range(2))
    w, b = (1 + 0.3 * torch.randn(c, generator=g, device="cuda")).half(), (0.3 * torch.randn(c, generator=g, device="cuda")).half()
    lengths = torch.ones(n, dtype=torch.int32, device="cuda")
    lengths[-2] = 0
    y, mean, rstd = ops.group_norm_act_forward(x, groups, w, b, lengths=lengths)
    dx, dw, db = ops.group_norm_act_backward(dy, x, groups, mean, rstd, w, b, lengths=lengths)
    for at in (0, (1 << 22) - 2, (1 << 23) // (c // 16 or 1) - 2, (1 << 24) // (c // 16 or 1) - 2, n // 2, n - 4):
        part = slice(at, at + 4)
        if at + 4 > n:
            continue
        y1, m1, r1 = ops.group_norm_act_forward(x[part], groups, w, b, lengths=lengths[part])
        dx1, _, _ = ops.group_norm_act_backward(dy[part], x[part], groups, m1, r1, w, b, lengths=lengths[part])
        assert torch.equal(y[part], y1) and torch.equal(mean[part], m1) and torch.equal(rstd[part], r1) and torch.equal(dx[part], dx1), at
    assert not y[-2].any() and not dx[-2].any()
    want_w, want_b = (torch.zeros(c, dtype=torch.float64, device="cuda") for _ in range(2))
    room_w, room_b = (torch.zeros(c, dtype=torch.float64, device="cuda") for _ in range(2))
    for rows in torch.arange(n, device="cuda").split(1 << 20):
        v, d = x[rows, 0].double().view(-1, groups, c // groups), dy[rows, 0].double() * lengths[rows, None]
        m = v.mean(2, keepdim=True)
        r = 1 / torch.sqrt(((v - m) ** 2).mean(2, keepdim=True) + 1e-5)
        h = ((v - m) * r).reshape(-1, c)
        # of a term: rstd 2^-18, the mean 2^-20 of the spread and 2^-24 of itself, the product 2^-24; the sums are 64-bit
        err = h.abs() * 2.0 ** -17 + 2.0 ** -20 + (m.abs() * r).expand(-1, -1, c // groups).reshape(-1, c) * 2.0 ** -23
        want_w, want_b = want_w + (d * h).sum(0), want_b + d.sum(0)
        room_w, room_b = room_w + (d.abs() * err).sum(0), room_b + d.abs().sum(0) * 2.0 ** -40
    for got, want, room in ((dw, want_w, room_w), (db, want_b, room_b)):
        close(got, want.cpu(), half_step(got.dtype, want).cpu() + room.cpu())


def test_group_norm_sample_counts_are_not_limited_by_the_grid():
    """No such device: what the argument checks let pass goes no further."""
    so = L.load()
    for n, l, ok in ((1 << 32, 1, True), (1 << 20, 1 << 16, True), (1, (1 << 30) - (1 << 17), True), (1, 1 << 30, False), (1 << 39, 4, False)):
        t = lambda at: C.byref(L.VtcRows3(at, 8 * l, 8))  # noqa: E731
        size = so.vtc_group_norm_act_workspace(n, min(l, 1 << 30), 8, 1, 0)
        rc = so.vtc_group_norm_act(-1, 1, t(1 << 20), t(1 << 50), n, l, 8, 1, None, None, 0, 1e-5, 0, None, 1 << 60, 1 << 60, 1 << 61, size, None)
        msg = L.last_error(None)
        assert rc != 0 and ("device" in msg if ok else "too many rows" in msg), (n, l, msg)


# Every product of these runs on 256-wide tiles (tests/test_op_extents.py asks the library's plan): several tiles of a block one after the
# other and fewer tiles than blocks, halves of a tile behind the matrix, K splits of the weights' gradients, rows that are copied first and rows that are not
FFN_WIDE_SIZES = [(9001, 773, 2051, 757), (24601, 1100, 700, 1300), (12013, 1096, 712, 1288)]


@gpu
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("m,k,f,n", FFN_WIDE_SIZES)
def test_gated_ffn_on_256_wide_tiles(kind, m, k, f, n):
    act = {9001: "silu", 24601: "gelu", 12013: "sigmoid"}[m]
    kind = TYPES[kind]
    x, w, b, dy = make_ffn(kind, m, k, f, n, True, bias_kind=torch.float32 if m == 24601 else None)
    y, saved = ops.gated_ffn_forward(x, *w, *b, act=act, save=True)
    assert torch.equal(y, ops.gated_ffn_forward(x, *w, *b, act=act)[0])
    grads = ops.gated_ffn_backward(dy, x, *w, saved, act=act, bias_dtype=b[0].dtype)
    check_ffn(kind, x, w, b, act, dy, y, grads)
    # the bounds above grow with the contraction; in the 2-norm, at most four half steps lie on the way to a result (h or dg / du, the other
    # factor of a product of two of them, the result, and Phi's fit), and n terms in fp32 add n 2^-24
    want = ffn_64(x, *w, *b, act, dy)
    for name, got in (("y", y),) + tuple(zip(NAMES, grads)):
        room = 2 * torch.finfo(kind).eps + m * 2.0 ** -24
        assert float((got.double() - want[name]).norm() / want[name].norm()) <= room, name


# Small tiles with the down product, dx and the weights' gradients in K splits, alone or together
FFN_SPLIT_SIZES = [(499, 768, 2048, 768), (301, 389, 2051, 261), (70, 100, 4100, 52), (1237, 389, 1031, 389)]


@gpu
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("m,k,f,n", FFN_SPLIT_SIZES)
def test_gated_ffn_in_k_splits(kind, m, k, f, n):
    x, w, b, dy = make_ffn(TYPES[kind], m, k, f, n, True)
    y, saved = ops.gated_ffn_forward(x, *w, *b, act="gelu", save=True)
    grads = ops.gated_ffn_backward(dy, x, *w, saved, act="gelu")
    check_ffn(TYPES[kind], x, w, b, "gelu", dy, y, grads)
    want = ffn_64(x, *w, *b, "gelu", dy)   # the 2-norm as in test_gated_ffn_on_256_wide_tiles
    for name, got in (("y", y),) + tuple(zip(NAMES, grads)):
        room = 2 * torch.finfo(TYPES[kind]).eps + max(m, f) * 2.0 ** -24
        assert float((got.double() - want[name]).norm() / want[name].norm()) <= room, name


@gpu
def test_gated_ffn_weights_of_more_than_2_to_the_29_elements():
    """K-tiles of dx whose k-rows lie more than 2^31 bytes behind the first, with a half-tile of columns behind the matrix; a sample of rows
    and columns of every result against the 64-bit definition."""
    m, k, f, n = 4100, 4160, 131080, 200
    kind = torch.bfloat16
    x, w, b, dy = make_ffn(kind, m, k, f, n, False)
    y, saved = ops.gated_ffn_forward(x, *w, save=True)
    dx, dwg, dwu, dwd = ops.gated_ffn_backward(dy, x, *w, saved, biases=False)[:4]
    del saved
    rows = torch.tensor([0, 1, 255, 256, 2047, 4095, 4096, 4099], device="cuda")
    want = ffn_64(x[rows], *w, *b, "silu", dy[rows])
    tol = ffn_tolerances(x[rows], *w, *b, "silu", dy[rows], kind)
    for name, got in (("y", y[rows]), ("dx", dx[rows])):
        close(got, want[name].cpu(), half_step(kind, want[name]).cpu() + tol[name].cpu() * 1.001, name)
    del want, tol
    cols = torch.tensor([0, 127, 128, 65535, 65536, 131071, 131072, 131079], device="cuda")
    part = (w[0][cols], w[1][cols], w[2][:, cols].contiguous())   # these inner columns alone: their weights' gradients do not depend on the others
    want = ffn_64(x, *part, *b, "silu", dy)
    tol = ffn_tolerances(x, *part, *b, "silu", dy, kind)
    for name, got in (("dw_gate", dwg[cols]), ("dw_up", dwu[cols]), ("dw_down", dwd[:, cols])):
        close(got, want[name].cpu(), half_step(kind, want[name]).cpu() + tol[name].cpu() * 1.001, name)


def fused_layouts(batch, length, heads, dim):
    """(shape, axis of the 3 projections, order that brings (batch, length, heads, dim)) of fused projections, by the order of their dimensions."""
    return {
        "rows": ((batch, length, 3, heads, dim), 2, (0, 1, 2, 3)),
        "sequence first": ((length, batch, 3, heads, dim), 2, (1, 0, 2, 3)),
        "heads first": ((batch, 3, heads, length, dim), 1, (0, 2, 1, 3)),
        "projection first": ((3, batch, length, heads, dim), 0, (0, 1, 2, 3)),
        "projections of a head together": ((batch, length, heads, 3, dim), 3, (0, 1, 2, 3)),
        "length last": ((heads, batch, 3, length, dim), 2, (1, 2, 0, 3)),
    }


LAYOUT_NAMES = list(fused_layouts(1, 1, 1, 2))


@gpu
@pytest.mark.parametrize("name", LAYOUT_NAMES)
@pytest.mark.parametrize("batch", [1, 4])
def test_rotary_in_place_in_fused_projections_of_any_order(name, batch):
    length, heads, dim = 33, 5, 24
    shape, axis, order = fused_layouts(batch, length, heads, dim)[name]
    g = torch.Generator(device="cuda").manual_seed(41)
    qkv = torch.randn(shape, generator=g, device="cuda").half()
    before = qkv.clone()
    spec = ops.Rotary(16, layout="interleaved")
    q, k = (qkv.select(axis, i).permute(order) for i in (0, 1))
    ops.rotary_qk(q, k, spec, out=(q, k))
    pos = torch.arange(length).expand(batch, length)
    for i, t in ((0, q), (1, k)):
        check_rotary(t, before.select(axis, i).permute(order), spec, pos)
    assert torch.equal(qkv.select(axis, 2), before.select(axis, 2))
    q2 = before.select(axis, 2).permute(order)   # and from one projection into another's place
    ops.rotary(q2, spec, out=before.select(axis, 0).permute(order))
    check_rotary(before.select(axis, 0).permute(order), q2, spec, pos)


def test_rotary_takes_what_is_apart_and_refuses_what_is_shared():
    """In place on two tensors of one buffer, by brute force over their elements.  No such device: what passes the checks goes no further."""
    f = (C.c_double * 32)(*([0.5] * 32))
    rng = np.random.default_rng(17)
    so = L.load()

    def accepted(base, strides, counts, heads, dim):
        spec = L.VtcRotary(dim, 2, 0, 0, 1.0, C.cast(f, L._f64p))
        arr = (L.VtcHeads * 2)(*(L.VtcHeads(1 << 20 if i == 0 else (1 << 20) + 2 * base, 1 << 20 if i == 0 else (1 << 20) + 2 * base, *strides, *strides, heads[i])
                                 for i in (0, 1)))
        rc = so.vtc_rotary_heads(-1, 1, C.byref(spec), counts[0], counts[1], arr, 2, None, 0, 0, 0, 0, 0, None)
        msg = L.last_error(None)
        assert rc != 0 and ("device" in msg or "shares memory" in msg or "overlaps itself" in msg), msg
        return None if "overlaps itself" in msg else "device" in msg

    def elements(base, strides, counts, heads, dim):
        n = [np.arange(c) for c in (counts[0], counts[1], heads, dim)]
        return set((base + n[0][:, None, None, None] * strides[0] + n[1][:, None, None] * strides[1] + n[2][:, None] * strides[2] + n[3]).ravel().tolist())

    for name in LAYOUT_NAMES:                    # whole projections: always apart
        shape, axis, order = fused_layouts(3, 4, 2, 6)[name]
        t = torch.empty(shape)
        a, b = (t.select(axis, i).permute(order) for i in (0, 1))
        for base in (b.storage_offset(), -b.storage_offset()):
            assert accepted(base, a.stride()[:3], (3, 4), (2, 2), 6), name
        assert accepted(b.storage_offset() - 1, a.stride()[:3], (3, 4), (2, 2), 6) is False, name   # the last element of the first one
    seen = {True: 0, False: 0}
    for _ in range(3000):
        counts, heads, dim = rng.integers(1, 4, 2).tolist(), rng.integers(1, 4, 2).tolist(), int(rng.choice([2, 4, 6]))
        sizes = [*counts, max(heads)]
        strides, span = [0, 0, 0], dim
        for i in rng.permutation(3).tolist():    # nested, with room between
            strides[i] = span + int(rng.choice([0, 0, 2, dim, 3 * dim]))
            span = strides[i] * (sizes[i] - 1) + span
        base = int(rng.integers(-span - 4, span + 4))
        got = accepted(base, strides, counts, heads, dim)
        if got is None:
            continue
        shared = bool(elements(0, strides, counts, heads[0], dim) & elements(base, strides, counts, heads[1], dim))
        assert got == (not shared), (base, strides, counts, heads, dim)
        seen[got] += 1
    assert min(seen.values()) > 300, seen


@gpu
def test_group_norm_statistics_of_samples_without_rows():
    """A call on samples of length 0 still writes their mean and rstd, from C as from Python."""
    mean, rstd = torch.full((2, 70000, 20), float("nan"), device="cuda")
    t = C.byref(L.VtcRows3(None, 0, 40))
    L.check(L.load().vtc_group_norm_act(0, 1, t, t, 70000, 0, 40, 20, None, None, 0, 1e-5, 0, None, mean.data_ptr(), rstd.data_ptr(), None, 0,
                                        torch.cuda.current_stream().cuda_stream))
    assert not mean.any() and not rstd.any()
    x = torch.zeros((3, 0, 40), device="cuda")
    y, mean, rstd = ops.group_norm_act_forward(x, 20)
    assert y.shape == x.shape and mean.shape == (3, 20) and not mean.any() and not rstd.any()
    assert ops.group_norm_act_forward(x[:0], 20)[1].shape == (0, 20)


@gpu
def test_one_channel_and_one_column_have_no_stride():
    """A single channel turned channel-last and weights of width one keep the stride of what they were; it means nothing."""
    g = torch.Generator(device="cuda").manual_seed(51)
    x, dy = (torch.randn((3, 1, 70), generator=g, device="cuda").transpose(1, 2) for _ in range(2))   # (3, 70, 1), strides (70, 1, 70)
    w = torch.randn(1, generator=g, device="cuda")
    assert x.stride(2) == 70
    check_gn("f32", x, 1, w, w, "silu", None, dy, run_gn(x, 1, w, w, "silu", None, dy))
    z = x.clone(memory_format=torch.preserve_format)
    assert torch.equal(ops.group_norm_act_forward(z, 1, out=z)[0], ops.group_norm_act_forward(x, 1)[0])
    leaf = x.detach().requires_grad_()
    (dx,) = torch.autograd.grad(ops.group_norm_act(leaf, 1, w, w, act="silu"), leaf, dy)
    assert torch.equal(dx, run_gn(x, 1, w, w, "silu", None, dy)[3])
    x, w, b, dy = make_ffn(torch.float16, 130, 1, 24, 8, True)
    turned = tuple(t.as_strided(t.shape, (1, t.shape[0])) for t in w[:2] + (x,))
    y, saved = ops.gated_ffn_forward(turned[2], *turned[:2], w[2], *b, save=True)
    check_ffn(torch.float16, x, w, b, "silu", dy, y, ops.gated_ffn_backward(dy, x, *turned[:2], w[2], saved))


@gpu
@pytest.mark.parametrize("m", [2, 16, 17, 32, 33, 64])
def test_gated_ffn_few_rows_do_not_reach_each_other(m):
    """A row that is no number stays alone on both sides of the border between the kernels of few and of many rows."""
    x, w, b, dy = make_ffn(torch.float16, m, 100, 132, 60, True)
    want, saved = ops.gated_ffn_forward(x, *w, *b, save=True)
    check_ffn(torch.float16, x, w, b, "silu", dy, want, ops.gated_ffn_backward(dy, x, *w, saved))
    x[1] = float("nan")
    got = ops.gated_ffn(x, *w, *b)
    clean = torch.arange(m, device="cuda") != 1
    assert got[1].isnan().all() and torch.equal(got[clean], want[clean])
