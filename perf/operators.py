"""The encoder-variant operators of vtc_amd.ops as cases to time and compare: rotary positions, group norm with an
activation (channels last) and the gated feed-forward block.

`own = False` computes the plain forms (elementary torch operations in 32 bits, 64 for the angles), `own = True` makes the
calls a user makes.  A case is a dict of plain values; `prepare` makes its inputs on the GPU from a seed, `run` is one pass.
"""

import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one new 20 ms frame of each of 8 live recordings, hours into them: q and k of a 12 x 64 head layer
        {"name": "rotary_frame", "op": "rotary", "type": "f16", "batch": 8, "length": 1, "q_heads": 12, "k_heads": 12, "head_dim": 64,
         "rotary_dim": 64, "layout": "half", "base": 10000.0, "scaling": "none", "factor": 1.0, "original": 0, "far": 2000000, "inverse": False},
        # q and k of a layer for 64 windows of 10 s, the batch the benchmark runs
        {"name": "rotary_windows", "op": "rotary", "type": "f16", "batch": 64, "length": 499, "q_heads": 12, "k_heads": 12, "head_dim": 64,
         "rotary_dim": 64, "layout": "half", "base": 10000.0, "scaling": "none", "factor": 1.0, "original": 0, "far": 0, "inverse": False},
        # the gradient's direction over 20 minutes of frames in 32 bits: grouped key heads, part of the head, stretched positions
        {"name": "rotary_long_inverse", "op": "rotary", "type": "f32", "batch": 1, "length": 60001, "q_heads": 16, "k_heads": 4, "head_dim": 128,
         "rotary_dim": 96, "layout": "interleaved", "base": 10000.0, "scaling": "by_parts", "factor": 32.0, "original": 2048, "far": 0,
         "inverse": True},
        # the last conv layer's output of one 10 s window: latency
        {"name": "norm_window", "op": "norm", "type": "f16", "batch": 1, "length": 499, "channels": 512, "groups": 32, "act": "gelu",
         "ragged": False, "train": False},
        # a conv layer's output for 64 windows of 10 s
        {"name": "norm_conv_batch", "op": "norm", "type": "f16", "batch": 64, "length": 3999, "channels": 512, "groups": 32, "act": "gelu",
         "ragged": False, "train": False},
        # a training step on recordings of different lengths, one group per channel
        {"name": "norm_ragged_step", "op": "norm", "type": "bf16", "batch": 24, "length": 1999, "channels": 512, "groups": 512, "act": "gelu",
         "ragged": True, "train": True},
        # an odd layer in 32 bits: 201 channels in 3 groups
        {"name": "norm_odd_step", "op": "norm", "type": "f32", "batch": 5, "length": 1531, "channels": 201, "groups": 3, "act": "silu",
         "ragged": True, "train": True},
        # one frame through a layer's feed-forward block (the dense block's parameters in gated form: 2/3 of its width)
        {"name": "ffn_frame", "op": "ffn", "type": "bf16", "rows": 1, "width": 768, "inner": 2048, "act": "silu", "bias": True, "train": False},
        # one 10 s window
        {"name": "ffn_window", "op": "ffn", "type": "f16", "rows": 499, "width": 768, "inner": 2048, "act": "gelu", "bias": True, "train": False},
        # 64 windows of 10 s, the batch the benchmark runs
        {"name": "ffn_windows", "op": "ffn", "type": "f16", "rows": 31936, "width": 768, "inner": 2048, "act": "silu", "bias": True, "train": False},
        # a training step on 32 windows of 10 s
        {"name": "ffn_step", "op": "ffn", "type": "bf16", "rows": 15968, "width": 768, "inner": 2048, "act": "silu", "bias": True, "train": True},
        # a training step at sizes that are no multiple of anything
        {"name": "ffn_odd_step", "op": "ffn", "type": "f16", "rows": 1237, "width": 389, "inner": 1031, "act": "gelu", "bias": False, "train": True},
    ]


def _spread(rng, low, high):
    """A whole number in low..high, uniform in its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["rotary", "norm", "ffn"])
    kind = rng.choice(["f32", "f16", "bf16"])
    if op == "rotary":
        head_dim = rng.choice([16, 24, 40, 64, 80, 96, 128, 130])
        rotary_dim = head_dim if rng.random() < 0.5 else 2 * rng.randint(2, head_dim // 2)
        batch, q_heads = _spread(rng, 1, 64), rng.choice([1, 3, 4, 8, 12, 16])
        k_heads = q_heads if rng.random() < 0.6 else rng.choice([1, 2])
        most = 32000000 // ((q_heads + k_heads) * head_dim * batch)
        length = _spread(rng, 1, max(1, min(60000, most)))
        scaling = rng.choice(["none", "linear", "ntk", "by_parts"])
        return {"op": op, "type": kind, "batch": batch, "length": length, "q_heads": q_heads, "k_heads": k_heads, "head_dim": head_dim,
                "rotary_dim": rotary_dim, "layout": rng.choice(["half", "interleaved"]), "base": rng.choice([10000.0, 500000.0]),
                "scaling": scaling, "factor": 1.0 if scaling == "none" else rng.choice([2.0, 7.5, 32.0]),
                "original": 2048 if scaling == "by_parts" else 0, "far": rng.choice([0, 0, 100000, 2000000]), "inverse": rng.random() < 0.4}
    if op == "norm":
        groups = rng.choice([1, 3, 8, 32, 48])
        channels = groups * rng.randint(1, max(1, 1024 // groups))
        batch = _spread(rng, 1, 64)
        length = _spread(rng, 1, max(1, min(8000, 60000000 // (batch * channels))))
        return {"op": op, "type": kind, "batch": batch, "length": length, "channels": channels, "groups": groups,
                "act": rng.choice(["none", "gelu", "silu"]), "ragged": rng.random() < 0.5, "train": rng.random() < 0.5}
    width = rng.choice([64, 96, 256, 512, 768, 1024, rng.randint(17, 1100)])
    inner = rng.choice([128, 512, 1024, 2048, 2736, rng.randint(33, 2800)])
    train = rng.random() < 0.5
    rows = _spread(rng, 1, max(1, min(32000, int((2.5e11 if train else 3e11) / ((18 if train else 6) * width * inner)))))
    return {"op": op, "type": rng.choice(["f16", "bf16"]), "rows": rows, "width": width, "inner": inner, "act": rng.choice(["gelu", "silu", "sigmoid"]),
            "bias": rng.random() < 0.5, "train": train}


# ---------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = _TYPES[case["type"]]

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(kind)

    state = {"case": case}
    if case["op"] == "rotary":
        b, t = case["batch"], case["length"]
        state["q"] = normal(b, t, case["q_heads"], case["head_dim"])
        state["k"] = normal(b, t, case["k_heads"], case["head_dim"])
        first = torch.randint(0, case["far"] + 1, (b, 1), generator=g, device="cuda")   # a recording's frames so far
        state["positions"] = first + torch.arange(t, device="cuda")
        state["frequency"], state["amplitude"] = _frequencies(case)
        if own:   # the description of the rotation, which a program makes once
            from vtc_amd import ops
            state["rotary"] = ops.Rotary(case["rotary_dim"], layout=case["layout"], base=case["base"], scaling=case["scaling"],
                                         factor=case["factor"], original_length=case["original"])
    elif case["op"] == "norm":
        b, t, c = case["batch"], case["length"], case["channels"]
        # a conv layer's output: channels of different scale and offset
        scale = torch.rand(c, generator=g, device="cuda") * 2.0 + 0.1
        offset = torch.randn(c, generator=g, device="cuda")
        state["x"] = (torch.randn((b, t, c), generator=g, device="cuda") * scale + offset).to(kind)
        state["weight"] = (1.0 + 0.2 * torch.randn(c, generator=g, device="cuda")).to(kind)
        state["bias"] = normal(c, std=0.2)
        state["lengths"] = torch.randint(1, t + 1, (b,), generator=g, device="cuda", dtype=torch.int32) if case["ragged"] else None
        state["dy"] = normal(b, t, c) if case["train"] else None
    else:
        m, k, f = case["rows"], case["width"], case["inner"]
        state["x"] = normal(m, k)                     # rows behind a LayerNorm
        state["w_gate"], state["w_up"] = normal(f, k, std=k ** -0.5), normal(f, k, std=k ** -0.5)
        state["w_down"] = normal(k, f, std=f ** -0.5)
        state["b_gate"], state["b_up"], state["b_down"] = (normal(n, std=0.1) if case["bias"] else None for n in (f, f, k))
        state["dy"] = normal(m, k) if case["train"] else None
    return state


def _frequencies(case):
    """Angular frequencies of the pairs in 64 bits and the amplitude of the rotation."""
    r, s = case["rotary_dim"], case["factor"]
    j = torch.arange(r // 2, dtype=torch.float64, device="cuda")
    base, amplitude = case["base"], 1.0
    if case["scaling"] == "ntk":
        base = base * s ** (r / max(r - 2, 1))
    f = base ** (-2.0 * j / r)
    if case["scaling"] == "linear":
        f = f / s
    elif case["scaling"] == "by_parts":
        # pairs that turn more than 32 times over the original length keep their frequency, those that turn less than once are
        # slowed by the factor, a ramp that is linear in the pair's index lies between
        def index(turns):
            return r * math.log(case["original"] / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))
        low, high = max(math.floor(index(32.0)), 0), min(math.ceil(index(1.0)), r // 2 - 1)
        ramp = ((j - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        f = f / s * ramp + f * (1.0 - ramp)
        amplitude = 0.1 * math.log(s) + 1.0 if s > 1.0 else 1.0
    return f, amplitude


# ---------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    if case["op"] == "rotary":
        angle = state["positions"].double()[..., None] * state["frequency"]
        sign = -1.0 if case["inverse"] else 1.0
        cos, sin = (angle.cos() * state["amplitude"]).float(), (angle.sin() * (sign * state["amplitude"])).float()
        return {"q": _rotate(case, state["q"], cos, sin), "k": _rotate(case, state["k"], cos, sin)}
    if case["op"] == "norm":
        return _norm(case, state)
    return _ffn(case, state)


def _run_own(case, state):
    from vtc_amd import ops
    if case["op"] == "rotary":
        q, k = ops.rotary_qk(state["q"], state["k"], state["rotary"], positions=state["positions"], inverse=case["inverse"])
        return {"q": q, "k": k}
    if case["op"] == "norm":
        args = dict(weight=state["weight"], bias=state["bias"], eps=1e-5, act=case["act"], lengths=state["lengths"])
        y, mean, rstd = ops.group_norm_act_forward(state["x"], case["groups"], **args)
        if not case["train"]:
            return {"y": y}
        dx, dw, db = ops.group_norm_act_backward(state["dy"], state["x"], case["groups"], mean, rstd, weight=state["weight"], bias=state["bias"],
                                                 act=case["act"], lengths=state["lengths"])
        return {"y": y, "dx": dx, "dweight": dw, "dbias": db}
    weights = (state["w_gate"], state["w_up"], state["w_down"])
    biases = dict(b_gate=state["b_gate"], b_up=state["b_up"], b_down=state["b_down"])
    y, saved = ops.gated_ffn_forward(state["x"], *weights, **biases, act=case["act"], save=case["train"])
    if not case["train"]:
        return {"y": y}
    g = ops.gated_ffn_backward(state["dy"], state["x"], *weights, saved, act=case["act"], biases=case["bias"])
    names = ("dx", "dw_gate", "dw_up", "dw_down") + (("db_gate", "db_up", "db_down") if case["bias"] else ())
    return {"y": y, **dict(zip(names, g))}


def _rotate(case, x, cos, sin):
    r = case["rotary_dim"]
    cos, sin = cos[:, :, None], sin[:, :, None]
    y = x.float().clone()
    if case["layout"] == "half":
        a, b = y[..., : r // 2].clone(), y[..., r // 2: r].clone()
        y[..., : r // 2], y[..., r // 2: r] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = y[..., 0:r:2].clone(), y[..., 1:r:2].clone()
        y[..., 0:r:2], y[..., 1:r:2] = a * cos - b * sin, a * sin + b * cos
    return y.to(x.dtype)


def _act(name, z):
    """act(z) and its derivative."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "gelu":
        p = 0.5 * torch.erfc(z * -math.sqrt(0.5))
        return z * p, p + z * torch.exp(-0.5 * z * z) * (2.0 * math.pi) ** -0.5
    s = torch.sigmoid(z)
    return (s, s * (1.0 - s)) if name == "sigmoid" else (z * s, s * (1.0 + z * (1.0 - s)))


def _norm(case, state):
    b, t, c, n = case["batch"], case["length"], case["channels"], case["groups"]
    x, w, bias = state["x"].float().view(b, t, n, c // n), state["weight"].float().view(n, c // n), state["bias"].float().view(n, c // n)
    if state["lengths"] is None:
        real = torch.ones((b, t, 1, 1), device="cuda")
    else:
        real = (torch.arange(t, device="cuda")[None] < state["lengths"][:, None]).float()[:, :, None, None]
    count = real.sum(1, keepdim=True) * (c // n)
    mean = (x * real).sum((1, 3), keepdim=True) / count
    rstd = 1.0 / torch.sqrt(((x - mean) ** 2 * real).sum((1, 3), keepdim=True) / count + 1e-5)
    hat = (x - mean) * rstd
    y, slope = _act(case["act"], hat * w + bias)
    out = {"y": (y * real).to(state["x"].dtype).view(b, t, c)}
    if case["train"]:
        dz = state["dy"].float().view(b, t, n, c // n) * slope * real
        dh = dz * w
        inner = dh.sum((1, 3), keepdim=True) / count
        along = (dh * hat).sum((1, 3), keepdim=True) / count
        out["dx"] = ((dh - inner - hat * along) * rstd * real).to(state["x"].dtype).view(b, t, c)
        out["dweight"] = (dz * hat).sum((0, 1)).to(state["x"].dtype).view(c)
        out["dbias"] = dz.sum((0, 1)).to(state["x"].dtype).view(c)
    return out


def _ffn(case, state):
    x, wg, wu, wd = (state[n].float() for n in ("x", "w_gate", "w_up", "w_down"))
    g, u = x @ wg.t(), x @ wu.t()
    if case["bias"]:
        g, u = g + state["b_gate"].float(), u + state["b_up"].float()
    a, slope = _act(case["act"], g)
    h = a * u
    y = h @ wd.t()
    if case["bias"]:
        y = y + state["b_down"].float()
    kind = state["x"].dtype
    out = {"y": y.to(kind)}
    if case["train"]:
        dy = state["dy"].float()
        dh = dy @ wd
        dg, du = dh * u * slope, dh * a
        out["dx"] = (dg @ wg + du @ wu).to(kind)
        out["dw_gate"], out["dw_up"], out["dw_down"] = (dg.t() @ x).to(kind), (du.t() @ x).to(kind), (dy.t() @ h).to(kind)
        if case["bias"]:
            out["db_gate"], out["db_up"], out["db_down"] = dg.sum(0).to(kind), du.sum(0).to(kind), dy.sum(0).to(kind)
    return out


# ---------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    e = _BYTES[case["type"]]
    if case["op"] == "rotary":
        n = case["batch"] * case["length"] * (case["q_heads"] + case["k_heads"])
        return {"bytes": 2 * n * case["head_dim"] * e + 8 * case["batch"] * case["length"], "flops": 3 * n * case["rotary_dim"]}
    if case["op"] == "norm":
        n = case["batch"] * case["length"] * case["channels"]
        # forward: x, y; a step: x, dy, y, dx
        return {"bytes": (4 if case["train"] else 2) * n * e + (4 if case["train"] else 2) * case["channels"] * e, "flops": (40 if case["train"] else 15) * n}
    m, k, f = case["rows"], case["width"], case["inner"]
    if case["train"]:   # x, dy, y, dx and the weights and their gradients
        return {"bytes": (4 * m * k + 6 * k * f) * e, "flops": 18 * m * k * f}
    return {"bytes": (2 * m * k + 3 * k * f) * e, "flops": 6 * m * k * f}


# ---------------------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        # as a product of complex numbers, a block of rows at a time
        f, amplitude = _frequencies(case)
        r = case["rotary_dim"]
        turn = -1.0 if case["inverse"] else 1.0
        out = {}
        for name in ("q", "k"):
            y = s[name].double()
            for b in range(y.shape[0]):
                angle = turn * s["positions"][b].double()[:, None] * f
                spin = torch.polar(torch.full_like(angle, amplitude), angle)[:, None]
                part = y[b, :, :, :r]
                if case["layout"] == "half":
                    z = torch.complex(part[..., : r // 2].contiguous(), part[..., r // 2:].contiguous()) * spin
                    y[b, :, :, :r] = torch.cat([z.real, z.imag], -1)
                else:
                    z = torch.complex(part[..., 0::2].contiguous(), part[..., 1::2].contiguous()) * spin
                    y[b, :, :, :r] = torch.stack([z.real, z.imag], -1).flatten(-2)
            out[name] = y
        return out
    if case["op"] == "norm":
        # one recording at a time, over its real rows alone; the gradient as the formula's projections
        t, c, n = case["length"], case["channels"], case["groups"]
        w, bias = s["weight"].double(), s["bias"].double()
        y = torch.zeros((case["batch"], t, c), dtype=torch.float64, device="cuda")
        dx, dw, db = torch.zeros_like(y), torch.zeros_like(w), torch.zeros_like(w)
        for i in range(case["batch"]):
            real = t if s["lengths"] is None else int(s["lengths"][i])
            x = s["x"][i, :real].double().view(real, n, -1).permute(1, 0, 2).reshape(n, -1)
            var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
            std = torch.sqrt(var + 1e-5)
            hat = ((x - mean) / std).view(n, real, -1).permute(1, 0, 2).reshape(real, c)
            z = hat * w + bias
            a, slope = _exact_act(case["act"], z)
            y[i, :real] = a
            if case["train"]:
                dz = s["dy"][i, :real].double() * slope
                dw += (dz * hat).sum(0)
                db += dz.sum(0)
                d = (dz * w).view(real, n, -1).permute(1, 0, 2).reshape(n, -1)
                h = (x - mean) / std
                d = d - d.mean(1, keepdim=True) - h * (d * h).mean(1, keepdim=True)
                dx[i, :real] = (d / std).view(n, real, -1).permute(1, 0, 2).reshape(real, c)
        return {"y": y, "dx": dx, "dweight": dw, "dbias": db} if case["train"] else {"y": y}
    x, wg, wu, wd = (s[n].double() for n in ("x", "w_gate", "w_up", "w_down"))
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    bg, bu, bd = (zero if s[n] is None else s[n].double() for n in ("b_gate", "b_up", "b_down"))
    out = {n: [] for n in ("y", "dx")}
    sums = {}
    for i in range(0, case["rows"], 8192):
        rows = x[i: i + 8192]
        g, u = torch.nn.functional.linear(rows, wg) + bg, torch.nn.functional.linear(rows, wu) + bu
        a, slope = _exact_act(case["act"], g)
        out["y"].append(torch.nn.functional.linear(a * u, wd) + bd)
        if case["train"]:
            dy = s["dy"][i: i + 8192].double()
            dh = torch.mm(dy, wd)
            dg, du = dh * u * slope, dh * a
            out["dx"].append(torch.mm(dg, wg) + torch.mm(du, wu))
            parts = [torch.mm(dg.t(), rows), torch.mm(du.t(), rows), torch.mm(dy.t(), a * u)]
            if case["bias"]:
                parts += [dg.sum(0), du.sum(0), dy.sum(0)]
            for name, p in zip(("dw_gate", "dw_up", "dw_down", "db_gate", "db_up", "db_down"), parts):
                sums[name] = sums[name] + p if name in sums else p
    y = torch.cat(out["y"])
    return {"y": y, "dx": torch.cat(out["dx"]), **sums} if case["train"] else {"y": y}


def _exact_act(name, z):
    if name == "none":
        return z, torch.ones_like(z)
    if name == "gelu":
        phi = torch.special.ndtr(z)
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    s = 1.0 / (1.0 + torch.exp(-z))
    if name == "sigmoid":
        return s, s - s * s
    return z * s, s + z * (s - s * s)
