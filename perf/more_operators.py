"""Performance cases of the operators that a preference or policy fine-tuning step needs around a block's own weights.

Four families, called on device memory through `see_ai_b200.backend.CudaBackend`:

  join        a block joins the residual stream: the norm after the block, its gate, the scaled residual and the norm before
              the next block, forward and backward with the weights' gradients.
  preference  a loss of paired sequences by their log ratios to a reference model, with the gradient of the logits.
  policy      a clipped policy loss with a KL term, with the gradient of the logits.
  grad        the norm over all gradients and the factor that clips them, or the clipped gradients themselves.

`own` false: the same quantities by elementary torch operations in 32 bits, rounded once at the end.
"""

from __future__ import annotations

import functools
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}


# ---- the cases --------------------------------------------------------------------------------------

def _join(op, kind, rows, cols, x, y, post=True, gate=True, scale=1.0):
    return dict(op=op, kind=kind, rows=rows, cols=cols, x=x, y=y, post=post, gate=gate, scale=scale)


def _preference(kind, pairs, longest, classes, type, average=False, logit_scale=1.0):
    return dict(op="preference", kind=kind, pairs=pairs, longest=longest, classes=classes, type=type, average=average, logit_scale=logit_scale)


def _policy(rows, classes, type, kl=0.0, logit_scale=1.0):
    return dict(op="policy", rows=rows, classes=classes, type=type, kl=kl, logit_scale=logit_scale)


def _grad(op, layers, d_model, d_hidden, vocab, type, rank=0):
    return dict(op=op, layers=layers, d_model=d_model, d_hidden=d_hidden, vocab=vocab, type=type, rank=rank)


def listed():
    def named(name, case):
        return dict(case, name=name)

    return [
        # One token of a decoder 768 wide: latency alone.
        named("join_fwd_token", _join("join_fwd", "rms", 1, 768, "f32", "bf16")),
        # The benchmark's batch, 64 sequences of 512: an f32 residual stream, 16-bit products before and after.
        named("join_fwd_64x512", _join("join_fwd", "rms", 32768, 768, "f32", "bf16")),
        # A short ragged batch of an odd width on the way back.
        named("join_bwd_ragged", _join("join_bwd", "layer", 777, 1029, "f32", "f32")),
        # A wide model's rows in 16 bits on the way back, without a gate.
        named("join_bwd_4096", _join("join_bwd", "rms", 16384, 4096, "bf16", "bf16", gate=False, scale=0.9)),
        # A few short answers of a small vocabulary.
        named("preference_small", _preference("hinge", 3, 60, 250, "f32")),
        # Eight pairs of up to 512 tokens.
        named("preference_8x512", _preference("sigmoid", 8, 512, 32000, "bf16")),
        # Ragged pairs, an odd vocabulary, averaged over each answer.
        named("preference_odd", _preference("square", 3, 333, 50001, "f16", average=True)),
        # One short answer, logits in 32 bits.
        named("policy_answer", _policy(64, 32000, "f32", kl=0.05)),
        # Sixteen answers of 512 tokens.
        named("policy_16x512", _policy(8192, 32000, "bf16", kl=0.02)),
        # An odd, large vocabulary, sampled at another temperature.
        named("policy_odd", _policy(777, 128003, "bf16", logit_scale=1.25)),
        # All gradients of a decoder of twelve layers.
        named("grad_norm_decoder", _grad("grad_norm", 12, 768, 2048, 32000, "bf16")),
        # The f32 gradients of its rank-16 adapters, clipped.
        named("grad_clip_adapters", _grad("grad_clip", 12, 768, 0, 0, "f32", 16)),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


MOST_LOGITS = 1 << 28


def draw(rng):
    op = rng.choice(("join_fwd", "join_bwd", "preference", "policy", "grad_norm", "grad_clip"))
    if op.startswith("join"):
        cols = _log(rng, 16, 8192)
        if rng.random() < 0.7:   # widths are mostly multiples of 64
            cols = max(64, cols // 64 * 64)
        rows = _log(rng, 1, max(2, min(65536, (1 << 26) // cols)))
        x, y = rng.choice((("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "f16")))
        return _join(op, rng.choice(("layer", "rms")), rows, cols, x, y, rng.random() < 0.7, rng.random() < 0.5, rng.choice((1.0, 1.0, 0.9, 0.5)))
    if op == "preference":
        classes, pairs = _log(rng, 50, 130000), _log(rng, 1, 16)
        longest = _log(rng, 4, max(5, min(1024, 240000000 // (2 * pairs * classes))))
        kind = rng.choice(("sigmoid", "hinge", "square"))
        return _preference(kind, pairs, longest, classes, rng.choice(("f32", "bf16", "bf16", "f16")), rng.random() < 0.4, rng.choice((1.0, 1.0, 0.8)))
    if op == "policy":
        classes = _log(rng, 50, 130000)
        rows = _log(rng, 1, max(2, min(16384, 240000000 // classes)))
        return _policy(rows, classes, rng.choice(("f32", "bf16", "bf16", "f16")), rng.choice((0.0, 0.02, 0.1)), rng.choice((1.0, 1.0, 1.25)))
    d_model, type = _log(rng, 64, 1024) // 8 * 8, rng.choice(("f32", "bf16", "bf16", "f16"))
    if rng.random() < 0.4:
        return _grad(op, rng.randint(1, 24), d_model, 0, 0, type, rng.choice((4, 8, 16)))
    return _grad(op, rng.randint(1, 8), d_model, int(d_model * 8 / 3) // 8 * 8, _log(rng, 250, 32000), type)


# ---- inputs -------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _join_inputs(case, seed):
    """A residual stream whose channels are of unlike size, some far from zero; a block's output of about 1."""
    gen = _generator(seed)
    rows, cols, xt, yt = case["rows"], case["cols"], TYPES[case["x"]], TYPES[case["y"]]
    layer, post = case["kind"] == "layer", case["post"]
    s = dict(case, seed=seed, eps=1e-5, layer=layer)
    x = _randn(gen, rows, cols) * torch.exp(0.5 * _randn(gen, cols)) + 0.5 * _randn(gen, cols)
    s["x_in"] = (x * torch.exp(0.3 * _randn(gen, rows, 1))).to(xt)
    s["block"] = (_randn(gen, rows, cols) * torch.exp(0.3 * _randn(gen, cols)) + 0.2).to(yt)
    s["pre_gamma"], s["pre_beta"] = 1.0 + 0.1 * _randn(gen, cols), 0.1 * _randn(gen, cols) if layer else None
    s["post_gamma"] = 1.0 + 0.1 * _randn(gen, cols) if post else None
    s["post_beta"] = 0.1 * _randn(gen, cols) if post and layer else None
    s["gate_w"] = 0.5 + 0.2 * _randn(gen, cols) if case["gate"] else None
    f32 = dict(device="cuda", dtype=torch.float32)
    rows_of = lambda wanted: torch.empty(rows, **f32) if wanted else None  # noqa: E731
    s.update(post_mean=rows_of(post and layer), post_rstd=rows_of(post), pre_mean=rows_of(layer), pre_rstd=rows_of(True))
    if case["op"] == "join_fwd":
        s.update(x_out=torch.empty(rows, cols, device="cuda", dtype=xt), y_out=torch.empty(rows, cols, device="cuda", dtype=yt))
        return s
    out = _join_wide(s)   # what the forward pass kept
    s["x_out"] = out["x_out"].to(xt)
    for key in ("post_mean", "post_rstd", "pre_mean", "pre_rstd"):
        s[key] = out[key].float() if s[key] is not None else None
    s["dy"], s["dx_out"] = (_randn(gen, rows, cols) * 0.1).to(yt), (_randn(gen, rows, cols) * 0.1).to(xt)
    s.update(dx=torch.empty_like(s["x_out"]), dblock=torch.empty_like(s["block"]))
    for key in ("post_gamma", "post_beta", "gate_w", "pre_gamma", "pre_beta"):
        s["d" + key] = torch.empty(cols, **f32) if s[key] is not None else None
    return s


def _lengths(case):
    """The tokens of each sequence (chosen and rejected in turn) and of the prompt in front of its answer."""
    longest = case["longest"]
    lengths = [longest - (7 * i * i) % (longest // 2 + 1) for i in range(2 * case["pairs"])]
    return lengths, [n // 4 for n in lengths]


def _logits(gen, rows, classes, type, labels):
    """A trained model's: a label's chance from next to nothing up to next to one."""
    z = _randn(gen, rows, classes).mul_(2.0)
    lift = math.log(classes) * (0.4 + torch.rand(rows, generator=gen, device="cuda"))
    z.scatter_add_(1, labels.long().clamp(min=0)[:, None], lift[:, None])
    return z.to(TYPES[type])


def _wide_logp(s):
    """Log-probabilities of the labels in 64 bits, a few rows at a time."""
    out = torch.zeros(s["logits"].shape[0], device="cuda", dtype=torch.float64)
    step = max(1, (1 << 26) // s["classes"])
    for at in range(0, out.numel(), step):
        z = s["logits"][at:at + step].double() * s["logit_scale"]
        out[at:at + step] = z.gather(1, s["labels"][at:at + step].long().clamp(min=0)[:, None])[:, 0] - torch.logsumexp(z, 1)
    return torch.where(s["labels"] >= 0, out, 0.0)


def _preference_inputs(case, seed):
    gen = _generator(seed)
    lengths, prompts = _lengths(case)
    starts = np.concatenate([[0], np.cumsum(lengths)])
    rows = (int(starts[-1]) + 63) // 64 * 64   # a batch's buffer ends on a multiple of 64 tokens
    labels = torch.randint(case["classes"], (rows,), generator=gen, device="cuda", dtype=torch.int32)
    for at, n in zip(starts, prompts):
        labels[int(at):int(at) + n] = -1
    s = dict(case, seed=seed, rows=rows, labels=labels, logits=_logits(gen, rows, case["classes"], case["type"], labels),
             starts=torch.tensor(starts, device="cuda", dtype=torch.int32), beta=0.1, smoothing=0.05 if case["kind"] == "sigmoid" else 0.0,
             margin=0.2 if case["kind"] != "square" else 0.0)
    sums = _sequence_sums(s, _wide_logp(s))
    spread = 0.3 if case["average"] else 3.0
    reference = (sums + spread * _randn(gen, sums.numel())).float()
    # The hinge's corner is a point that no pair lies next to.
    near = ((_margins(s, sums, reference.double()) - 1.0).abs() < 1e-4).double().repeat_interleave(2)
    s["reference"] = (reference + 0.05 * near * torch.arange(sums.numel(), device="cuda").fmod(2)).float()
    f32 = dict(device="cuda", dtype=torch.float32)
    s.update(loss=torch.empty(1, **f32), margins=torch.empty(case["pairs"], **f32), sequence_logp=torch.empty(2 * case["pairs"], **f32),
             dlogits=torch.zeros_like(s["logits"]))
    return s


def _policy_inputs(case, seed):
    gen = _generator(seed)
    rows, classes = case["rows"], case["classes"]
    labels = torch.randint(classes, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    labels[_prompt_rows(rows)] = -1
    s = dict(case, seed=seed, labels=labels, logits=_logits(gen, rows, classes, case["type"], labels), clip_low=0.2, clip_high=0.28)
    logp = _wide_logp(s)
    ratio = torch.exp(0.15 * _randn(gen, rows)).double()
    for border in (1.0 - s["clip_low"], 1.0 + s["clip_high"]):   # points that no ratio lies next to
        ratio = torch.where((ratio - border).abs() < 1e-4, border + 2e-4, ratio)
    s["old_logp"], s["ref_logp"] = (logp - ratio.log()).float(), (logp + 0.3 * _randn(gen, rows)).float() if case["kl"] else None
    s["advantages"] = _randn(gen, rows)
    s["weights"] = torch.full((rows,), 1.0 / (rows - len(_prompt_rows(rows))), device="cuda")
    f32 = dict(device="cuda", dtype=torch.float32)
    s.update(loss=torch.empty(3, **f32), logp=torch.empty(rows, **f32), dlogits=torch.zeros_like(s["logits"]))
    return s


def _prompt_rows(rows):
    """The tokens of prompts, which the loss does not count."""
    return [r for r in range(rows) if r // 16 % 8 == 1]


def _grad_sizes(case):
    d, f = case["d_model"], case["d_hidden"]
    if case["rank"]:
        return [d * case["rank"]] * (8 * case["layers"])
    return ([d, d] + [d * d] * 4 + [d, d] + [d * f] * 3) * case["layers"] + [d * case["vocab"]]


def _grad_inputs(case, seed):
    """Gradients of unlike size, in tensors that lie one behind the other; their norm is above what is allowed."""
    gen = _generator(seed)
    sizes = _grad_sizes(case)
    starts = np.concatenate([[0], np.cumsum(sizes)]).tolist()
    g = torch.empty(starts[-1], device="cuda", dtype=TYPES[case["type"]])
    for n, at in zip(sizes, starts):
        g[at:at + n] = (_randn(gen, n) * (1e-3 * math.exp(math.sin(at + seed)))).to(g.dtype)
    f32 = dict(device="cuda", dtype=torch.float32)
    s = dict(case, seed=seed, sizes=sizes, starts=starts, g=g, norm=torch.empty(1, **f32), factor=torch.empty(1, **f32),
             loss_scale=torch.full((1,), 0.25, **f32), max_norm=0.1)
    s["out"] = torch.empty_like(g) if case["op"] == "grad_clip" else None
    return s


def prepare(case, seed):
    if case["op"].startswith("join"):
        return _join_inputs(case, seed)
    if case["op"].startswith("grad"):
        return _grad_inputs(case, seed)
    return _preference_inputs(case, seed) if case["op"] == "preference" else _policy_inputs(case, seed)


# ---- the plain forms ------------------------------------------------------------------------------------

def _plain_norm(s, v, gamma, beta):
    mean = v.mean(1) if s["layer"] else None
    centred = v - mean[:, None] if s["layer"] else v
    rstd = torch.rsqrt(centred.square().mean(1) + s["eps"])
    out = centred * rstd[:, None] * gamma
    return (out + beta if s["layer"] else out), mean, rstd


def _given(outputs):
    return {k: v for k, v in outputs.items() if v is not None}


def _join_fwd(s):
    u, post_mean, post_rstd = s["block"].float(), None, None
    if s["post"]:
        u, post_mean, post_rstd = _plain_norm(s, u, s["post_gamma"], s["post_beta"])
    if s["gate"]:
        u = u * s["gate_w"]
    x = s["x_in"].float() * s["scale"] + u
    y, pre_mean, pre_rstd = _plain_norm(s, x, s["pre_gamma"], s["pre_beta"])
    return _given(dict(x_out=x.to(TYPES[s["x"]]), y=y.to(TYPES[s["y"]]), post_mean=post_mean, post_rstd=post_rstd, pre_mean=pre_mean,
                       pre_rstd=pre_rstd))


def _plain_norm_bwd(s, q, unit, rstd):
    d = q - unit * (q * unit).mean(1, keepdim=True)
    if s["layer"]:
        d = d - q.mean(1, keepdim=True)
    return d * rstd[:, None]


def _join_bwd(s):
    unit_of = lambda v, mean, rstd: ((v - mean[:, None]) if s["layer"] else v) * rstd[:, None]  # noqa: E731
    dy = s["dy"].float()
    unit = unit_of(s["x_out"].float(), s["pre_mean"], s["pre_rstd"])
    d = _plain_norm_bwd(s, dy * s["pre_gamma"], unit, s["pre_rstd"]) + s["dx_out"].float()
    out = dict(dx=(d * s["scale"]).to(TYPES[s["x"]]), dpre_gamma=(dy * unit).sum(0), dpre_beta=dy.sum(0) if s["layer"] else None)
    u = s["block"].float()
    gated = d * s["gate_w"] if s["gate"] else d
    if not s["post"]:
        out.update(dblock=gated.to(TYPES[s["y"]]), dgate_w=(d * u).sum(0) if s["gate"] else None)
        return _given(out)
    unit = unit_of(u, s["post_mean"], s["post_rstd"])
    if s["gate"]:
        out["dgate_w"] = (d * (unit * s["post_gamma"] + s["post_beta"] if s["layer"] else unit * s["post_gamma"])).sum(0)
    out.update(dpost_gamma=(gated * unit).sum(0), dpost_beta=gated.sum(0) if s["layer"] else None)
    out["dblock"] = _plain_norm_bwd(s, gated * s["post_gamma"], unit, s["post_rstd"]).to(TYPES[s["y"]])
    return _given(out)


def _sequence_sums(s, logp):
    """Sums of the rows' log-probabilities over each sequence, or averages over those that count."""
    of = torch.searchsorted(s["starts"][1:].long(), torch.arange(s["rows"], device="cuda"), right=True)
    counted = (s["labels"] >= 0) & (of < 2 * s["pairs"])
    sums = torch.zeros(2 * s["pairs"] + 1, device="cuda", dtype=torch.float64).index_add_(0, of, torch.where(counted, logp, 0.0))[:-1]
    if s["average"]:
        sums = sums / torch.zeros(2 * s["pairs"] + 1, device="cuda", dtype=torch.float64).index_add_(0, of, counted.double())[:-1].clamp(min=1.0)
    return sums


def _margins(s, sums, reference):
    ratio = sums - reference
    return s["beta"] * (ratio[0::2] - ratio[1::2]) - s["margin"]


def _softmax(s):
    """Probabilities, and the labels' log-probabilities in 64 bits: the corners of the losses are next to them."""
    z = s["logits"].float() * s["logit_scale"]
    most = z.amax(1, keepdim=True)
    e = torch.exp(z - most)
    total = e.sum(1, keepdim=True, dtype=torch.float64)
    index = s["labels"].long().clamp(min=0)[:, None]
    logp = z.gather(1, index).double() - most.double() - total.log()
    return e / total.float(), torch.where(s["labels"] >= 0, logp[:, 0], 0.0), index


def _logit_gradient(s, p, index, slope):
    """slope (onehot - p) times the logits' scale; rows of no slope: zeros."""
    slope = (slope * s["logit_scale"]).float()[:, None]
    d = p.mul_(-slope).scatter_add_(1, index, slope)
    return torch.where(s["labels"][:, None] >= 0, d, 0.0).to(TYPES[s["type"]])


def _preference_loss(s):
    p, logp, index = _softmax(s)
    sums = _sequence_sums(s, logp)
    h = _margins(s, sums, s["reference"].double())
    if s["kind"] == "sigmoid":
        up, down = torch.exp(-h), torch.exp(h)
        losses = (1.0 - s["smoothing"]) * torch.log(1.0 + up) + s["smoothing"] * torch.log(1.0 + down)
        slope = -(1.0 - s["smoothing"]) * up / (1.0 + up) + s["smoothing"] * down / (1.0 + down)
    elif s["kind"] == "hinge":
        losses, slope = torch.relu(1.0 - h), -(h < 1.0).double()
    else:
        off = (h - 0.5) / s["beta"]
        losses, slope = off * off, 2.0 * off / s["beta"]
    slope = slope * s["beta"] / s["pairs"]
    slopes = torch.stack([slope, -slope], 1).reshape(-1)
    of = torch.searchsorted(s["starts"][1:].long(), torch.arange(s["rows"], device="cuda"), right=True)
    if s["average"]:
        counted = ((s["labels"] >= 0) & (of < 2 * s["pairs"])).double()
        slopes = slopes / torch.zeros(2 * s["pairs"] + 1, device="cuda", dtype=torch.float64).index_add_(0, of, counted)[:-1].clamp(min=1.0)
    row_slopes = torch.cat([slopes, slopes.new_zeros(1)])[of]
    return dict(loss=losses.mean().float().reshape(1), margins=h.float(), sequence_logp=sums.float(),
                dlogits=_logit_gradient(s, p, index, row_slopes))


def _policy_loss(s):
    p, logp, index = _softmax(s)
    counted = s["labels"] >= 0
    weights = torch.where(counted, s["weights"], 0.0).double()
    a = s["advantages"].double()
    r = torch.exp(logp - s["old_logp"].double())
    cut = r.clamp(1.0 - s["clip_low"], 1.0 + s["clip_high"])
    free = r * a <= cut * a
    losses, slope = -torch.minimum(r * a, cut * a), torch.where(free, -r * a, 0.0)
    kl = torch.zeros_like(losses)
    if s["kl"]:
        x = s["ref_logp"].double() - logp
        kl = torch.exp(x) - x - 1.0
        losses, slope = losses + s["kl"] * kl, slope + s["kl"] * (1.0 - torch.exp(x))
    sums = torch.stack([(weights * losses).sum(), (weights * kl).sum(), (weights * ~free).sum()])
    return dict(loss=sums.float(), logp=logp.float(), dlogits=_logit_gradient(s, p, index, weights * slope))


def _grad_pass(s):
    g = s["g"].float()
    norm = g.double().square().sum().sqrt() * s["loss_scale"].double().abs()
    factor = torch.where((norm <= s["max_norm"]) | (norm == 0), 1.0, s["max_norm"] / norm) * s["loss_scale"].double()
    out = dict(norm=norm.float(), factor=factor.float())
    return out if s["out"] is None else dict(out, out=(g * factor.float()).to(s["g"].dtype))


# ---- the framework's calls --------------------------------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _backend():
    from see_ai_b200 import backend as B
    be = B.CudaBackend(torch.cuda.current_device())
    be.set_stream(torch.cuda.current_stream().cuda_stream)
    return B, be


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _own_join(s):
    B, be = _backend()
    kind = B.NORM_LAYER if s["layer"] else B.NORM_RMS
    options = dict(x_type=B.TYPES[s["x"]], y_type=B.TYPES[s["y"]], residual_scale=s["scale"])
    names = ("post_gamma", "post_beta", "gate_w", "pre_gamma", "pre_beta")
    if "own_weights" not in s:   # a program lists its weights once
        s["own_weights"] = B.join_weights(**{k.removesuffix("_w"): _ptr(s[k]) for k in names})
        s["own_stats"] = B.join_stats(**{k: _ptr(s[k]) for k in ("post_mean", "post_rstd", "pre_mean", "pre_rstd")})
        if s["op"] == "join_bwd":
            s["own_grads"] = B.join_weights(**{k.removesuffix("_w"): _ptr(s["d" + k]) for k in names})
            s["work"] = torch.empty(B.join_backward_workspace(s["rows"], s["cols"]), device="cuda", dtype=torch.uint8)
    if s["op"] == "join_fwd":
        be.join_forward(kind, s["rows"], s["cols"], _ptr(s["x_in"]), _ptr(s["block"]), s["own_weights"], _ptr(s["x_out"]), _ptr(s["y_out"]),
                        s["own_stats"], eps=s["eps"], **options)
        return _given(dict(x_out=s["x_out"], y=s["y_out"], post_mean=s["post_mean"], post_rstd=s["post_rstd"], pre_mean=s["pre_mean"],
                           pre_rstd=s["pre_rstd"]))
    be.join_backward(kind, s["rows"], s["cols"], _ptr(s["dy"]), _ptr(s["dx_out"]), _ptr(s["x_out"]), _ptr(s["block"]), s["own_weights"],
                     s["own_stats"], _ptr(s["dx"]), _ptr(s["dblock"]), s["own_grads"], _ptr(s["work"]), s["work"].numel(), **options)
    return _given(dict(dx=s["dx"], dblock=s["dblock"], **{"d" + k: s["d" + k] for k in names}))


def _own_preference(s):
    B, be = _backend()
    if "work" not in s:
        s["work"] = torch.empty(B.preference_workspace(s["rows"], s["pairs"]), device="cuda", dtype=torch.uint8)
    be.preference_loss(s["rows"], s["classes"], s["pairs"], _ptr(s["logits"]), _ptr(s["labels"]), _ptr(s["starts"]), _ptr(s["loss"]),
                       _ptr(s["margins"]), _ptr(s["sequence_logp"]), _ptr(s["work"]), s["work"].numel(), ref_logp=_ptr(s["reference"]),
                       dlogits=_ptr(s["dlogits"]), type=B.TYPES[s["type"]], kind=B.PREFERENCES[s["kind"]], beta=s["beta"],
                       smoothing=s["smoothing"], margin=s["margin"], logit_scale=s["logit_scale"], average=s["average"])
    return {k: s[k] for k in ("loss", "margins", "sequence_logp", "dlogits")}


def _own_policy(s):
    B, be = _backend()
    if "work" not in s:
        s["work"] = torch.empty(B.policy_workspace(s["rows"]), device="cuda", dtype=torch.uint8)
    be.policy_loss(s["rows"], s["classes"], _ptr(s["logits"]), _ptr(s["labels"]), _ptr(s["old_logp"]), _ptr(s["advantages"]), _ptr(s["loss"]),
                   _ptr(s["logp"]), _ptr(s["work"]), s["work"].numel(), ref_logp=_ptr(s["ref_logp"]), weights=_ptr(s["weights"]),
                   dlogits=_ptr(s["dlogits"]), type=B.TYPES[s["type"]], clip_low=s["clip_low"], clip_high=s["clip_high"], kl_coef=s["kl"],
                   logit_scale=s["logit_scale"])
    return {k: s[k] for k in ("loss", "logp", "dlogits")}


def _own_grad(s):
    B, be = _backend()
    if "table" not in s:   # a program lists its tensors once
        at = lambda t, start: 0 if t is None else t.data_ptr() + start * t.element_size()  # noqa: E731
        s["table"] = B.grad_tensors([dict(g=at(s["g"], o), out=at(s["out"], o), n=n, type=B.TYPES[s["type"]])
                                     for n, o in zip(s["sizes"], s["starts"])])
        s["work"] = torch.empty(B.grad_workspace(), device="cuda", dtype=torch.uint8)
    call = be.grad_norm if s["out"] is None else be.grad_clip
    call(s["table"], s["max_norm"], _ptr(s["norm"]), _ptr(s["factor"]), _ptr(s["work"]), s["work"].numel(), grad_scale=_ptr(s["loss_scale"]))
    return _given(dict(norm=s["norm"], factor=s["factor"], out=s["out"]))


def run(state):
    op = state["op"]
    if own:
        family = {"join": _own_join, "preference": _own_preference, "policy": _own_policy, "grad": _own_grad}
        return family[op.split("_")[0]](state)
    return {"join_fwd": _join_fwd, "join_bwd": _join_bwd, "preference": _preference_loss, "policy": _policy_loss, "grad_norm": _grad_pass,
            "grad_clip": _grad_pass}[op](state)


# ---- the same in 64 bits ------------------------------------------------------------------------------------

def _join_wide(s):
    def norm(v, gamma, beta):
        n = v.shape[1]
        mean = v.sum(1) / n if s["layer"] else None
        off = v if mean is None else v - mean[:, None]
        rstd = 1.0 / ((off ** 2).sum(1) / n + s["eps"]).sqrt()
        out = gamma.double() * off / ((off ** 2).sum(1, keepdim=True) / n + s["eps"]).sqrt()
        return out if beta is None else out + beta.double(), mean, rstd

    u, post_mean, post_rstd = s["block"].double(), None, None
    if s["post"]:
        u, post_mean, post_rstd = norm(u, s["post_gamma"], s["post_beta"])
    x = float(np.float32(s["scale"])) * s["x_in"].double() + (u if not s["gate"] else u * s["gate_w"].double())
    y, pre_mean, pre_rstd = norm(x, s["pre_gamma"], s["pre_beta"])
    return _given(dict(x_out=x, y=y, post_mean=post_mean, post_rstd=post_rstd, pre_mean=pre_mean, pre_rstd=pre_rstd))


def _exact_join_bwd(s):
    """Each norm's Jacobian applied to the gradient that comes down through gamma."""
    def unit_of(v, mean, rstd):
        v = v.double() if mean is None else v.double() - mean.double()[:, None]
        return v * rstd.double()[:, None]

    def through(q, unit, rstd):
        n = q.shape[1]
        pull = torch.einsum("rc,rc->r", q, unit)[:, None] / n * unit
        return rstd.double()[:, None] * (q - pull - (q.sum(1, keepdim=True) / n if s["layer"] else 0.0))

    dy, cols = s["dy"].double(), s["block"].shape[1]
    one = torch.ones(cols, device="cuda", dtype=torch.float64)
    unit2 = unit_of(s["x_out"], s["pre_mean"], s["pre_rstd"])
    d = s["dx_out"].double() + through(dy * s["pre_gamma"].double(), unit2, s["pre_rstd"])
    gate = s["gate_w"].double() if s["gate"] else one
    out = dict(dx=float(np.float32(s["scale"])) * d, dpre_gamma=torch.einsum("rc,rc->c", dy, unit2), dpre_beta=dy.sum(0) if s["layer"] else None)
    if s["post"]:
        unit1 = unit_of(s["block"], s["post_mean"], s["post_rstd"])
        gamma, beta = s["post_gamma"].double(), s["post_beta"].double() if s["layer"] else 0.0
        out.update(dblock=through(d * gate * gamma, unit1, s["post_rstd"]), dpost_gamma=torch.einsum("rc,rc->c", d, unit1) * gate,
                   dpost_beta=d.sum(0) * gate if s["layer"] else None, dgate_w=torch.einsum("rc,rc->c", d, unit1 * gamma + beta) if s["gate"] else None)
    else:
        out.update(dblock=d * gate, dgate_w=torch.einsum("rc,rc->c", d, s["block"].double()) if s["gate"] else None)
    return _given(out)


def _exact_dlogits(s, slopes):
    """slopes: of the loss by each row's log-probability."""
    out = torch.zeros(s["logits"].shape, device="cuda", dtype=torch.float64)
    step = max(1, (1 << 26) // s["classes"])
    for at in range(0, out.shape[0], step):
        rows = slice(at, at + step)
        label = s["labels"][rows].long()
        onehot = torch.arange(s["classes"], device="cuda")[None, :] == label[:, None]
        p = torch.softmax(s["logits"][rows].double() * float(np.float32(s["logit_scale"])), 1)
        # Where the label's chance is next to one, what is left of it is the others' sum.
        left = torch.where(onehot, 0.0, p).sum(1, keepdim=True)
        out[rows] = slopes[rows, None] * float(np.float32(s["logit_scale"])) * torch.where(onehot, left, -p)
        out[rows][label < 0] = 0.0
    return out


def _exact_preference(s):
    logp = _wide_logp(s)
    starts = s["starts"].tolist()
    beta, margin, smoothing = (float(np.float32(s[k])) for k in ("beta", "margin", "smoothing"))
    sums, counts = [], []
    for a, b in zip(starts[:-1], starts[1:]):
        counts.append(max(1, int((s["labels"][a:b] >= 0).sum())) if s["average"] else 1)
        sums.append(float(logp[a:b].sum()) / counts[-1])
    reference = s["reference"].double().tolist()
    total, margins, slopes = 0.0, [], torch.zeros(s["rows"], device="cuda", dtype=torch.float64)
    for i in range(s["pairs"]):
        a, b = 2 * i, 2 * i + 1
        h = beta * ((sums[a] - reference[a]) - (sums[b] - reference[b])) - margin
        if s["kind"] == "sigmoid":
            chance = 1.0 / (1.0 + math.exp(-h))
            value, slope = -(1.0 - smoothing) * math.log(chance) - smoothing * math.log1p(-chance), smoothing * chance - (1.0 - smoothing) * (1.0 - chance)
        elif s["kind"] == "hinge":
            value, slope = max(0.0, 1.0 - h), -1.0 if h < 1.0 else 0.0
        else:
            value, slope = (h / beta - 0.5 / beta) ** 2, 2.0 * (h / beta - 0.5 / beta) / beta
        total += value
        margins.append(h)
        slopes[starts[a]:starts[a + 1]] = slope * beta / s["pairs"] / counts[a]
        slopes[starts[b]:starts[b + 1]] = -slope * beta / s["pairs"] / counts[b]
    f64 = dict(device="cuda", dtype=torch.float64)
    return dict(loss=torch.tensor([total / s["pairs"]], **f64), margins=torch.tensor(margins, **f64), sequence_logp=torch.tensor(sums, **f64),
                dlogits=_exact_dlogits(s, slopes))


def _exact_policy(s):
    logp = _wide_logp(s)
    low, high, kl_coef = (float(np.float32(s[k])) for k in ("clip_low", "clip_high", "kl"))
    w = s["weights"].double() * (s["labels"] >= 0)
    a, r = s["advantages"].double(), torch.exp(logp - s["old_logp"].double())
    plain, cut = -a * r, -a * torch.clamp(r, 1.0 - low, 1.0 + high)
    loss, slope, clipped = torch.maximum(plain, cut), torch.where(plain >= cut, plain, 0.0), (plain < cut).double()
    kl = torch.zeros_like(loss)
    if s["kl"]:
        x = s["ref_logp"].double() - logp
        kl = torch.expm1(x) - x
        slope = slope - kl_coef * torch.expm1(x)
    return dict(loss=torch.stack([(w * (loss + kl_coef * kl)).sum(), (w * kl).sum(), (w * clipped).sum()]), logp=logp,
                dlogits=_exact_dlogits(s, w * slope))


def _exact_grad(s):
    square = sum(torch.dot(t, t) for t in s["g"].double().split(s["sizes"]))
    scale, most = s["loss_scale"].double()[0], float(np.float32(s["max_norm"]))
    norm = square.sqrt() * scale.abs()
    factor = scale * (1.0 if float(norm) <= most else most / norm)
    out = dict(norm=norm.reshape(1), factor=factor.reshape(1))
    return out if s["out"] is None else dict(out, out=s["g"].double() * factor)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "join_fwd":
        return _join_wide(s)
    return {"join_bwd": _exact_join_bwd, "preference": _exact_preference, "policy": _exact_policy, "grad_norm": _exact_grad,
            "grad_clip": _exact_grad}[case["op"]](s)


# ---- what a pass cannot do without ---------------------------------------------------------------------------

def work(case):
    if case["op"].startswith("join"):
        rows, cols = case["rows"], case["cols"]
        n, x, y = float(rows * cols), SIZES[case["x"]], SIZES[case["y"]]
        vectors = 4.0 * cols * (1 + case["gate"] + case["post"]) * (1 if case["kind"] == "rms" else 2)
        if case["op"] == "join_fwd":
            return {"bytes": n * 2 * (x + y) + vectors + 8.0 * rows, "flops": 16.0 * n}
        return {"bytes": n * 3 * (x + y) + 2 * vectors + 8.0 * rows, "flops": 30.0 * n}
    if case["op"] == "preference":
        lengths, prompts = _lengths(case)
        rows, counted = sum(lengths), sum(lengths) - sum(prompts)
    elif case["op"] == "policy":
        rows, counted = case["rows"], case["rows"] - len(_prompt_rows(case["rows"]))
    else:
        n, size = float(sum(_grad_sizes(case))), SIZES[case["type"]]
        return {"bytes": n * size * (2 if case["op"] == "grad_clip" else 1), "flops": n * (3 if case["op"] == "grad_clip" else 2)}
    size = SIZES[case["type"]]
    return {"bytes": float(rows + counted) * case["classes"] * size + 24.0 * rows, "flops": 8.0 * counted * case["classes"]}
