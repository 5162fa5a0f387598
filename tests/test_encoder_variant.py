"""Encoder variants (engine.EncoderVariant, the `encoder` block of a config): group norm behind the conv layers, rotary positions,
gated feed-forward, alone and together, through the library's own forward pass against the CPU oracle."""

import ctypes as C

import numpy as np
import pytest
import torch
import yaml

from oracle import vtc_oracle as O
from vtc_amd import lib as L
from vtc_amd import synth
from vtc_amd.engine import EncoderVariant, VtcEngine
from vtc_amd.ops import Rotary
from vtc_amd.segma_compat.config import load_config
from vtc_amd.segma_compat.models import Models, encoder_variant

gpu = pytest.mark.gpu
VARIANTS = {
    "rotary": EncoderVariant(rotary=Rotary(64)),
    "rotary_part": EncoderVariant(rotary=Rotary(48, layout="interleaved", scaling="by_parts", factor=8.0, original_length=199)),
    "gated_silu": EncoderVariant(ffn="gated_silu"),
    "gated_gelu": EncoderVariant(ffn="gated_gelu"),
    "conv_norm": EncoderVariant(conv_norm_groups=32),
    "all": EncoderVariant(rotary=Rotary(64), ffn="gated_silu", conv_norm_groups=16),
}


def variant_state(variant, seed=0, inner=2048):
    w = synth.make_weights(seed=seed, family="hubert")
    w = synth.variant_weights(w, seed, ffn=variant.ffn, conv_norm_groups=variant.conv_norm_groups, inner=inner, hub=True)
    if variant.rotary is not None:
        w = {k: v for k, v in w.items() if "pos_conv_embed" not in k}
    return w


def as_torch(w):
    return {k: torch.from_numpy(np.ascontiguousarray(v)) for k, v in w.items()}


@gpu
@pytest.mark.parametrize("name", list(VARIANTS))
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_every_stage_of_a_variant_against_the_oracle(name, dtype):
    """The bars of the base encoder's stage test (f16 storage: 1e-2 / 1.5e-2 on conv and hidden rows of unit scale, 2e-2 on logits;
    bf16 storage: 8 times the rounding)."""
    variant = VARIANTS[name]
    # Everything between two stores is fp32, so a stage's error is, to first order, linear in the stores' half step, 2^-11 (f16) and 2^-8
    # (bf16) of a value: 8 x 1e-2 on conv rows.  (The base encoder's bf16 bar of 6e-2 holds for one store per conv layer; a layer with
    # its own norm stores twice, the conv's rows and the normed ones: up to 2 x 6e-2.)
    conv_tol, hid_tol, logit_tol = (1e-2, 1.5e-2, 2e-2) if dtype == "f16" else (8e-2, 1.2e-1, 1.5e-1)
    w = variant_state(variant)
    B, W = 3, 16000
    T = O.conv_out_len(W)
    wav = np.random.default_rng(1).standard_normal((B, W), dtype=np.float32) * np.float32(0.1)
    wav[-1, W // 2:] = 0
    st = O.encoder_stages(as_torch(w), torch.from_numpy(wav), variant=variant)
    eng = VtcEngine(w, 4, 1.0, max_batch=B, mfma_dtype=dtype, variant=variant)
    arena = torch.from_numpy(wav.reshape(-1).copy()).cuda()
    start, valid = np.arange(B) * W, np.full(B, W)
    valid[-1] = W // 2
    dst, keep = np.arange(B) * T, np.full(B, T)
    logits = torch.zeros((B * T, 4), device="cuda")
    names = [f"conv{i}" for i in range(7)] + ["proj", "enc_in"] + [f"layer{l}" for l in range(12)]
    for stage, key in enumerate(names):
        eng.debug_stop_after(stage)
        eng.forward_windows(arena, start, valid, dst, keep, logits)
        ref = st[key].transpose(1, 2).contiguous() if stage <= 6 else st[key]
        got = torch.from_numpy(eng.debug_stage(stage, B, ref.numel()).reshape(ref.shape))
        scale = max(1.0, float(ref.std()))
        err = (got - ref).abs().max().item()
        assert err <= (conv_tol if stage <= 6 else hid_tol) * scale, f"{key}: max abs err {err}"
    eng.debug_stop_after(-1)
    eng.forward_windows(arena, start, valid, dst, keep, logits)
    torch.cuda.synchronize()
    err = (logits.cpu() - st["logits"].reshape(B * T, 4)).abs().max().item()
    assert err <= logit_tol, err
    eng.close()


@gpu
@pytest.mark.parametrize("name", [n for n, v in VARIANTS.items() if not v.conv_norm_groups])
def test_conv_layers_without_norms_keep_the_base_models_bf16_bar(name):
    """One store per conv layer, as in HuBERT-base: 6e-2 on conv rows, not the bar of layers that store twice."""
    variant = VARIANTS[name]
    w = variant_state(variant)
    B, W = 3, 16000
    T = O.conv_out_len(W)
    wav = np.random.default_rng(1).standard_normal((B, W), dtype=np.float32) * np.float32(0.1)
    st = O.encoder_stages(as_torch(w), torch.from_numpy(wav), variant=variant)
    eng = VtcEngine(w, 4, 1.0, max_batch=B, mfma_dtype="bf16", variant=variant)
    arena = torch.from_numpy(wav.reshape(-1).copy()).cuda()
    logits = torch.zeros((B * T, 4), device="cuda")
    for stage in range(7):
        eng.debug_stop_after(stage)
        eng.forward_windows(arena, np.arange(B) * W, np.full(B, W), np.arange(B) * T, np.full(B, T), logits)
        ref = st[f"conv{stage}"].transpose(1, 2).contiguous()
        got = torch.from_numpy(eng.debug_stage(stage, B, ref.numel()).reshape(ref.shape))
        err = (got - ref).abs().max().item()
        assert err <= 6e-2 * max(1.0, float(ref.std())), f"conv{stage}: max abs err {err}"
    eng.close()


@gpu
@pytest.mark.parametrize("variant,inner", [(EncoderVariant(ffn="gated_sigmoid"), 256), (EncoderVariant(ffn="gated_gelu"), 8192), (EncoderVariant(conv_norm_groups=1), 0),
                                           (EncoderVariant(conv_norm_groups=512), 0), (EncoderVariant(rotary=Rotary(2, layout="interleaved")), 0)])
def test_logits_at_the_limits_of_a_variants_sizes(variant, inner):
    """The narrowest and widest gated block, one group of all channels and one per channel, one rotated pair; the bar of the logits above."""
    w = variant_state(variant, inner=inner or 2048)
    B, W = 3, 16000
    T = O.conv_out_len(W)
    wav = np.random.default_rng(2).standard_normal((B, W), dtype=np.float32) * np.float32(0.1)
    want = O.encoder_stages(as_torch(w), torch.from_numpy(wav), variant=variant)["logits"]
    eng = VtcEngine(w, 4, 1.0, max_batch=B, variant=variant)
    logits = torch.zeros((B * T, 4), device="cuda")
    eng.forward_windows(torch.from_numpy(wav.reshape(-1).copy()).cuda(), np.arange(B) * W, np.full(B, W), np.arange(B) * T, np.full(B, T), logits)
    assert (logits.cpu() - want.reshape(B * T, 4)).abs().max().item() <= 2e-2
    eng.close()


@gpu
def test_variant_changes_the_result_and_the_base_model_is_untouched():
    w = synth.make_weights(seed=0, family="hubert")
    wav = torch.from_numpy(synth.synth_audio(3.0, 5)).cuda()
    base = VtcEngine(w, 4, 1.0, max_batch=4)
    same = VtcEngine(w, 4, 1.0, max_batch=4, variant=EncoderVariant())
    a = base.infer_waveform(wav)
    assert torch.equal(a, same.infer_waveform(wav))
    for e in (base, same):
        e.close()
    seen = [a]
    for variant in VARIANTS.values():
        eng = VtcEngine(variant_state(variant), 4, 1.0, max_batch=4, variant=variant)
        x = eng.infer_waveform(wav)
        assert torch.isfinite(x).all() and all(not torch.equal(x, s) for s in seen)
        # windows share no state: the same windows in other batches give the same bits
        assert torch.equal(x, eng.infer_waveform(wav, batch_size=1)) or variant.conv_norm_groups or variant.ffn != "gelu"
        torch.testing.assert_close(x, eng.infer_waveform(wav, batch_size=1), atol=2e-2, rtol=0)
        seen.append(x)
        eng.close()


@gpu
@pytest.mark.parametrize("name", list(VARIANTS))
def test_a_window_of_a_variant_does_not_depend_on_its_batch(name):
    """What lets recordings share forwards: a window's logits have the same bits in any batch."""
    variant = VARIANTS[name]
    eng = VtcEngine(variant_state(variant), 4, 4.0, max_batch=40, variant=variant)
    wav = torch.from_numpy(synth.synth_audio(40 * 3.98, 8)).cuda()
    full = eng.infer_waveform(wav)
    for batch in (1, 3, 17):
        assert torch.equal(full, eng.infer_waveform(wav, batch_size=batch))
    eng.close()


@gpu
def test_forward_of_a_variant_in_large_batches():
    """Full 10 s windows: many row blocks per window in the conv norms, many tiles in the gated block; windows agree with a batch of
    one window to the bar of the logits, and a batch repeated gives the same bits."""
    variant = VARIANTS["all"]
    eng = VtcEngine(variant_state(variant), 4, 10.0, max_batch=12, variant=variant)
    wav = torch.from_numpy(synth.synth_audio(12 * 9.98, 3)).cuda()
    a = eng.infer_waveform(wav)
    assert torch.equal(a, eng.infer_waveform(wav))
    b = eng.infer_waveform(wav, batch_size=5)
    assert (a - b).abs().max().item() <= 2e-2
    eng.close()


@gpu
def test_variant_through_config_and_model(tmp_path):
    from vtc_amd.segma_compat.inference import apply_model_on_audio
    from vtc_amd.segma_compat.utils.encoders import MultiLabelEncoder
    import wave
    path = tmp_path / "a.wav"
    pcm = (synth.synth_audio(2.5, 1) * 32767).astype("<i2")
    with wave.open(str(path), "wb") as f:
        f.setnchannels(1)
        f.setsampwidth(2)
        f.setframerate(16000)
        f.writeframes(pcm.tobytes())
    cfg_path = tmp_path / "c.yml"
    cfg_path.write_text(yaml.safe_dump({"audio": {"chunk_duration_s": 1.0}, "encoder": {"position": "rotary", "ffn": "gated_silu", "conv_norm_groups": 32}}))
    cfg = load_config(cfg_path)
    model = Models[cfg.model.name].load_from_checkpoint("synthetic:3", MultiLabelEncoder(cfg.data.classes), cfg).eval().to("cuda")
    logits = apply_model_on_audio(path, model, model.conv_settings, "cuda", 4, 1.0)
    sd = synth.variant_weights(synth.make_weights(seed=3), 3, ffn="gated_silu", conv_norm_groups=32)
    want = O.encoder_stages(as_torch(sd), torch.from_numpy(pcm[:16000].astype(np.float32) / 32768)[None], variant=encoder_variant(cfg.encoder))["logits"][0]
    assert logits.shape[1] == 4 and (logits[: want.shape[0]].cpu() - want).abs().max().item() <= 2e-2
    assert model.rescue_engine(1.0, 2).variant.ffn == "gated_silu"
    model.close_rescue()


def test_config_block_and_refusals(tmp_path):
    p = tmp_path / "c.yml"
    p.write_text(yaml.safe_dump({"encoder": {"position": "rotary", "rotary_dim": 32, "rotary_scaling": "linear", "rotary_factor": 2}}))
    v = encoder_variant(load_config(p).encoder)
    assert v.rotary.rotary_dim == 32 and v.ffn == "gelu" and np.allclose(v.rotary.frequency, Rotary(32).frequency / 2)
    p.write_text("{}\n")
    v = encoder_variant(load_config(p).encoder)
    assert v.rotary is None and v == EncoderVariant()
    for bad in (dict(ffn="dense"), dict(conv_norm_groups=5), dict(conv_norm_groups=-1), dict(rotary=Rotary(66))):
        with pytest.raises(ValueError):
            EncoderVariant(**bad)
    cfg = load_config(p).encoder
    cfg.position = "none"
    with pytest.raises(ValueError):
        encoder_variant(cfg)


def _create(**over):
    f = (C.c_double * 32)(*([1.0] * 32))
    spec = L.VtcSpec(abi_version=L.ABI_VERSION, n_labels=4, window_samples=16000, max_batch=1, mfma_dtype=1)
    v = L.VtcVariant()
    r = dict(head_dim=64, rotary_dim=0, layout=0, amplitude=1.0, frequency=f)
    fields = {k[3:]: x for k, x in over.items() if k.startswith("r__")}
    v.rotary = L.VtcRotary(**{**r, **fields})
    for k, x in over.items():
        if not k.startswith("r__"):
            setattr(v, k, x)
    h = C.c_void_p()
    rc = L.load().vtc_create_variant(C.byref(spec), C.byref(L.VtcWeights()), C.byref(v), 0, C.byref(h))
    return rc, L.last_error(None)


@pytest.mark.parametrize("over,text", [
    (dict(conv_norm_groups=3), "divide 512"), (dict(conv_norm_groups=-4), "divide 512"), (dict(conv_norm_groups=8), "conv layer 1"),
    (dict(ffn_act=9), "ffn_act"), (dict(ffn_act=2, ffn_inner=2000), "ffn_inner"), (dict(ffn_act=2, ffn_inner=128), "ffn_inner"),
    (dict(ffn_act=2, ffn_inner=1 << 20), "ffn_inner"), (dict(ffn_act=2, ffn_inner=2048), "gate tensor in layer 0"),
    (dict(r__rotary_dim=66), "rotary"), (dict(r__rotary_dim=3), "rotary"), (dict(r__rotary_dim=8, r__head_dim=32), "rotary"),
    (dict(r__rotary_dim=8, r__layout=4), "rotary"), (dict(r__rotary_dim=8, r__frequency=None), "rotary"),
    (dict(r__rotary_dim=2, r__frequency=(C.c_double * 1)(float("nan"))), "frequency 0")])
def test_library_refuses_bad_variants(over, text):
    rc, msg = _create(**over)
    assert rc == L.ERR_ARG and text in msg, (rc, msg)


@gpu
def test_engine_checks_the_variant_tensors():
    v = EncoderVariant(ffn="gated_silu")
    w = variant_state(v)
    with pytest.raises(KeyError):
        VtcEngine(synth.make_weights(seed=0), 4, 1.0, max_batch=1, variant=v)
    with pytest.raises(ValueError, match="intermediate_dense"):
        VtcEngine(w, 4, 1.0, max_batch=1)
    w["encoder.layers.3.feed_forward.gate_dense.bias"] = np.zeros(7, np.float32)
    with pytest.raises(ValueError, match="gate_dense.bias"):
        VtcEngine(w, 4, 1.0, max_batch=1, variant=v)


# ------------------------------------------------------------------------------------------------ the operators as a layer uses them
@gpu
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16])
def test_conv_norm_rotary_attention_and_gated_block_as_one_trained_run(kind):
    """A stage of such an encoder built from the public operators, forward and gradients, against the same chain in 64 bits: norm +
    GELU on conv rows, rotated q and k in plain attention, the gated block with its residual."""
    from vtc_amd import ops
    g = torch.Generator(device="cuda").manual_seed(2)
    n, t, heads, dim = 2, 70, 2, 32
    c = heads * dim
    r = lambda *s, std=1.0: (torch.randn(s, generator=g, device="cuda") * std).to(kind)  # noqa: E731
    x, lengths = r(n, t, c), torch.tensor([t, 41], dtype=torch.int32, device="cuda")
    gw, gb, wqk = (1 + 0.1 * torch.randn(c, generator=g, device="cuda")).to(kind), r(c, std=0.1), r(2 * c, c, std=c ** -0.5)
    ffn = (r(96, c, std=c ** -0.5), r(96, c, std=c ** -0.5), r(c, 96, std=96 ** -0.5))
    dy = r(n, t, c)
    spec = Rotary(dim)
    real = (torch.arange(t, device="cuda")[None] < lengths[:, None])

    def chain(x, gw, gb, wqk, ffn, norm, rotate, block):
        h = norm(x, gw, gb)
        qk = (h.reshape(-1, c) @ wqk.t()).view(n, t, 2, heads, dim)
        q, k = rotate(qk[:, :, 0], qk[:, :, 1])
        q, k, v = (z.permute(0, 2, 1, 3).reshape(n * heads, t, dim).to(torch.float64 if x.dtype == torch.float64 else torch.float32)
                   for z in (q, k, h.view(n, t, heads, dim)))
        s = (q[:, :, None] * k[:, None]).sum(-1) * dim ** -0.5
        s = s.masked_fill(~real.repeat_interleave(heads, 0)[:, None], float("-inf"))
        a = (torch.softmax(s, -1)[..., None] * v[:, None]).sum(2)
        a = a.view(n, heads, t, dim).permute(0, 2, 1, 3).reshape(n, t, c).to(x.dtype)
        u = h + a
        return u + block(u, *ffn)

    def plain_norm(x, w, b):
        rows = []
        for i in range(n):
            l = int(lengths[i])
            v = x[i, :l].view(l, 4, -1)
            z = (v - v.mean((0, 2), keepdim=True)) / torch.sqrt(v.var((0, 2), keepdim=True, correction=0) + 1e-5)
            rows.append(torch.nn.functional.pad(torch.nn.functional.gelu(z.reshape(l, c) * w + b), (0, 0, 0, t - l)))
        return torch.stack(rows)

    def plain_rotate(q, k):
        ang = torch.arange(t, dtype=torch.float64, device="cuda")[:, None] * torch.tensor(spec.frequency).cuda()
        cos, sin = ang.cos()[:, None], ang.sin()[:, None]
        turn = lambda z: torch.cat([z[..., :16] * cos - z[..., 16:] * sin, z[..., :16] * sin + z[..., 16:] * cos], -1)  # noqa: E731
        return turn(q), turn(k)

    leaves = [z.detach().clone().requires_grad_() for z in (x, gw, gb, wqk) + ffn]
    got = chain(*leaves[:4], leaves[4:], lambda x, w, b: ops.group_norm_act(x, 4, w, b, act="gelu", lengths=lengths),
                lambda q, k: ops.rotary_qk(q, k, spec), lambda u, *w: ops.gated_ffn(u, *w, act="silu"))
    grads = torch.autograd.grad(got, leaves, dy)
    exact = [z.detach().double().requires_grad_() for z in (x, gw, gb, wqk) + ffn]
    want = chain(*exact[:4], exact[4:], plain_norm, plain_rotate,
                 lambda u, a, b, d: (torch.nn.functional.silu(u @ a.t()) * (u @ b.t())) @ d.t())
    exact_grads = torch.autograd.grad(want, exact, dy.double())
    # about twelve roundings of half a step lie on the way to any gradient here, each relative to values of the tensor's own size;
    # in the 2-norm they add like 12 x eps / 2 at the very most
    room = 12 * torch.finfo(kind).eps / 2
    for a, b in [(got, want)] + list(zip(grads, exact_grads)):
        assert float((a.double() - b).norm() / b.norm()) <= room
