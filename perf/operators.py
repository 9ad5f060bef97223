"""Performance cases of the operators that train a block's own weights beside an update plan.

Three families, called on device memory through `see_ai_b200.backend.CudaBackend`:

  norm   layer norm and root-mean-square norm: the forward pass, and the backward pass with the gradients
         of the weights (and the residual branch's gradient added to the input's).
  gated  the gated feed-forward block, hidden = act(x Wg) * (x Wu), and its backward pass.
  adamw  one AdamW step over many tensors, moments in 8 bits or in 32, with the 16-bit copy of the weights
         that the next forward pass multiplies by.

`own` false: the same quantities by elementary torch operations in 32 bits, rounded once at the end.
"""

from __future__ import annotations

import functools
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 256   # elements that share a scale where the moments have 8 bits
GELU_C, GELU_A = math.sqrt(2.0 / math.pi), 0.044715


# ---- the cases --------------------------------------------------------------------------------------

def _norm(op, kind, rows, cols, x, y, addend=False):
    return dict(op=op, kind=kind, rows=rows, cols=cols, x=x, y=y, addend=addend)


def _gated(op, rows, d_in, d_hidden, type="bf16", act="silu", keep=True):
    return dict(op=op, rows=rows, d_in=d_in, d_hidden=d_hidden, type=type, act=act, keep=keep)


def _adamw(bits, layers, d_model, d_hidden, vocab, grad, copy, rank=0):
    return dict(op="adamw", bits=bits, layers=layers, d_model=d_model, d_hidden=d_hidden, vocab=vocab, grad=grad, copy=copy, rank=rank)


def listed():
    def named(name, case):
        return dict(case, name=name)

    return [
        # One token of a decoder 768 wide: latency alone.
        named("norm_fwd_token", _norm("norm_fwd", "layer", 1, 768, "f32", "f32")),
        # The benchmark's batch, 64 sequences of 512, its f32 residual stream into a 16-bit product.
        named("norm_fwd_64x512", _norm("norm_fwd", "layer", 32768, 768, "f32", "bf16")),
        # The same on the way back, the residual branch's gradient joining in.
        named("norm_bwd_64x512", _norm("norm_bwd", "layer", 32768, 768, "f32", "bf16", True)),
        # A short ragged batch of an odd width.
        named("norm_bwd_ragged", _norm("norm_bwd", "layer", 777, 1029, "f32", "f32")),
        # A wide model's rows in 16 bits.
        named("norm_bwd_rms_4096", _norm("norm_bwd", "rms", 16384, 4096, "bf16", "bf16")),
        # One token through the block: the weights are read once.
        named("gated_fwd_token", _gated("gated_fwd", 1, 768, 2048, keep=False)),
        # A ragged evaluation batch: three sequences of 200 tokens.
        named("gated_fwd_600", _gated("gated_fwd", 600, 512, 1376, "f16", "gelu", False)),
        # A training step's forward pass of a wide model.
        named("gated_fwd_8192", _gated("gated_fwd", 8192, 4096, 12288)),
        # One rank's share of the benchmark's batch on the way back.
        named("gated_bwd_8x512", _gated("gated_bwd", 4096, 768, 2048)),
        # The backward pass of a wide model, an odd number of rows.
        named("gated_bwd_8191", _gated("gated_bwd", 8191, 2048, 6144, act="gelu")),
        # All weights of a decoder of twelve layers, moments in 8 bits, 16-bit gradients and copies.
        named("adamw8_decoder", _adamw(8, 12, 768, 2048, 32000, "bf16", "bf16")),
        # Its rank-16 adapters: 96 small tensors, f32 throughout.
        named("adamw32_adapters", _adamw(32, 12, 768, 0, 0, "f32", "none", 16)),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm_fwd", "norm_bwd", "gated_fwd", "gated_bwd", "adamw"))
    if op.startswith("norm"):
        cols = _log(rng, 16, 8192)
        if rng.random() < 0.7:   # widths are mostly multiples of 64
            cols = max(64, cols // 64 * 64)
        rows = _log(rng, 1, max(2, min(65536, (1 << 26) // cols)))
        x, y = rng.choice((("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "f16")))
        return _norm(op, rng.choice(("layer", "rms")), rows, cols, x, y, op == "norm_bwd" and rng.random() < 0.5)
    if op.startswith("gated"):
        d_in = _log(rng, 64, 4096) // 8 * 8
        d_hidden = max(64, int(d_in * rng.uniform(1.5, 4.0)) // 8 * 8)
        most = 4e11 / (d_in * d_hidden) / (2 if op == "gated_bwd" else 1)
        rows = _log(rng, 1, max(2, min(16384, most)))
        return _gated(op, rows, d_in, d_hidden, rng.choice(("bf16", "bf16", "f16")), rng.choice(("silu", "gelu", "relu")),
                      op == "gated_bwd" or rng.random() < 0.5)
    bits, d_model = rng.choice((8, 32)), _log(rng, 64, 1024) // 8 * 8
    grad = rng.choice(("f32", "bf16"))
    copy = rng.choice(("none", "bf16", "f16"))
    if rng.random() < 0.4:
        return _adamw(bits, rng.randint(1, 24), d_model, 0, 0, grad, copy, rng.choice((4, 8, 16)))
    return _adamw(bits, rng.randint(1, 8), d_model, int(d_model * 8 / 3) // 8 * 8, _log(rng, 250, 32000), grad, copy)


# ---- inputs -------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _norm_inputs(case, seed):
    """A residual stream: channels of unlike size, some of them far from zero, rows of unlike size."""
    gen = _generator(seed)
    rows, cols = case["rows"], case["cols"]
    x = _randn(gen, rows, cols) * torch.exp(0.5 * _randn(gen, cols)) + 0.5 * _randn(gen, cols)
    x = (x * torch.exp(0.3 * _randn(gen, rows, 1))).to(TYPES[case["x"]])
    s = dict(case, seed=seed, eps=1e-5, x_in=x, gamma=1.0 + 0.1 * _randn(gen, cols), beta=0.1 * _randn(gen, cols))
    f32 = dict(device="cuda", dtype=torch.float32)
    if case["op"] == "norm_fwd":
        s.update(y_out=torch.empty(rows, cols, device="cuda", dtype=TYPES[case["y"]]), mean=torch.empty(rows, **f32), rstd=torch.empty(rows, **f32))
        return s
    s["dy"] = (_randn(gen, rows, cols) * 0.1).to(TYPES[case["y"]])
    wide = x.double()
    mean = wide.mean(1) if case["kind"] == "layer" else torch.zeros(rows, device="cuda", dtype=torch.float64)
    s["mean"], s["rstd"] = mean.float(), ((wide - mean[:, None]).square().mean(1) + s["eps"]).rsqrt().float()
    s["add"] = (_randn(gen, rows, cols) * 0.1).to(TYPES[case["x"]]) if case["addend"] else None
    s.update(dx=torch.empty_like(x), dgamma=torch.empty(cols, **f32), dbeta=torch.empty(cols, **f32))
    return s


def _gated_inputs(case, seed):
    """Normalised rows and weights of a trained block's size: gate and up of about 1."""
    gen = _generator(seed)
    rows, d_in, d_hidden, t = case["rows"], case["d_in"], case["d_hidden"], TYPES[case["type"]]
    s = dict(case, seed=seed, x=_randn(gen, rows, d_in).to(t))
    s["wg"], s["wu"] = ((_randn(gen, d_in, d_hidden) * d_in ** -0.5).to(t) for _ in range(2))
    if case["op"] == "gated_fwd":
        s["hidden"] = torch.empty(rows, d_hidden, device="cuda", dtype=t)
        s["gate"], s["up"] = (torch.empty_like(s["hidden"]) if case["keep"] else None for _ in range(2))
        return s
    s["gate"], s["up"] = s["x"] @ s["wg"], s["x"] @ s["wu"]
    s["dh"] = _randn(gen, rows, d_hidden).to(t)
    s.update(dx=torch.empty_like(s["x"]), dwg=torch.empty_like(s["wg"]), dwu=torch.empty_like(s["wu"]))
    return s


def _adamw_sizes(case):
    """Elements of each tensor, and whether its weights decay."""
    d, f = case["d_model"], case["d_hidden"]
    if case["rank"]:
        return [(d * case["rank"], True)] * (8 * case["layers"])
    layer = [(d, False), (d, False)] + [(d * d, True)] * 4 + [(d, False), (d, False)] + [(d * f, True)] * 3
    return layer * case["layers"] + [(d * case["vocab"], True)]


def _adamw_inputs(case, seed):
    """A run's two hundredth step.  The tensors lie in flat buffers, each from a multiple of 256 elements on."""
    gen = _generator(seed)
    sizes = _adamw_sizes(case)
    lengths = [(n + BLOCK - 1) // BLOCK * BLOCK for n, _ in sizes]
    starts = np.concatenate([[0], np.cumsum(lengths)[:-1]]).tolist()
    total = sum(lengths)
    spread = torch.exp(_randn(gen, total // BLOCK, 1)).expand(-1, BLOCK).reshape(-1) * 1e-3
    p, g = _randn(gen, total) * 0.02, _randn(gen, total) * spread
    m, v = _randn(gen, total) * spread * 0.25, (spread * (0.3 + torch.rand(total, generator=gen, device="cuda"))).square()
    s = dict(case, seed=seed, sizes=sizes, starts=starts, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, decay=0.01, step=201)
    counts = torch.tensor([n for n, _ in sizes], device="cuda")
    of = torch.repeat_interleave(torch.arange(len(sizes), device="cuda"), torch.tensor(lengths, device="cuda"))
    index = torch.arange(total, device="cuda") - torch.tensor(starts, device="cuda")[of]
    inside = index < counts[of]
    for t in (p, g, m, v):
        t.mul_(inside)
    s["index"] = index
    s["decays"] = (torch.tensor([float(w) for _, w in sizes], device="cuda") * np.float32(s["decay"]).item())[of]
    s["p"], s["g"] = p, g.to(TYPES[case["grad"]])
    s["copy16"] = None if case["copy"] == "none" else p.to(TYPES[case["copy"]])
    if case["bits"] == 32:
        s["m"], s["v"] = m, v
    else:
        half = torch.full_like(index, 0x80000000)
        s["m"], s["ms"] = _encode(m, half, True)
        s["v"], s["vs"] = _encode(v.sqrt(), half, False)   # held as its root: half the range of exponents
    return s


def prepare(case, seed):
    if case["op"].startswith("norm"):
        return _norm_inputs(case, seed)
    return _gated_inputs(case, seed) if case["op"].startswith("gated") else _adamw_inputs(case, seed)


# ---- the plain forms ------------------------------------------------------------------------------------

def _act(kind, g):
    if kind == "relu":
        return torch.relu(g)
    if kind == "silu":
        return g * torch.sigmoid(g)
    return 0.5 * g * (1.0 + torch.tanh(GELU_C * (g + GELU_A * g * g * g)))


def _act_slope(kind, g):
    if kind == "relu":
        return (g > 0).to(g.dtype)
    if kind == "silu":
        s = torch.sigmoid(g)
        return s * (1.0 + g * (1.0 - s))
    t = torch.tanh(GELU_C * (g + GELU_A * g * g * g))
    return 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * GELU_C * (1.0 + 3.0 * GELU_A * g * g)


def _norm_fwd(s):
    x = s["x_in"].float()
    mean = x.mean(1) if s["kind"] == "layer" else torch.zeros_like(s["mean"])
    centred = x - mean[:, None]
    rstd = torch.rsqrt(centred.square().mean(1) + s["eps"])
    y = centred * rstd[:, None] * s["gamma"]
    y = y + s["beta"] if s["kind"] == "layer" else y
    return dict(y=y.to(TYPES[s["y"]]), mean=mean, rstd=rstd) if s["kind"] == "layer" else dict(y=y.to(TYPES[s["y"]]), rstd=rstd)


def _norm_bwd(s):
    x, dy, rstd = s["x_in"].float(), s["dy"].float(), s["rstd"][:, None]
    unit = (x - s["mean"][:, None]) * rstd
    q = dy * s["gamma"]
    dx = q - unit * (q * unit).mean(1, keepdim=True)
    if s["kind"] == "layer":
        dx = dx - q.mean(1, keepdim=True)
    dx = dx * rstd
    if s["add"] is not None:
        dx = dx + s["add"].float()
    out = dict(dx=dx.to(TYPES[s["x"]]), dgamma=(dy * unit).sum(0))
    return dict(out, dbeta=dy.sum(0)) if s["kind"] == "layer" else out


def _gated_fwd(s):
    t = TYPES[s["type"]]
    x = s["x"].float()
    g, u = x @ s["wg"].float(), x @ s["wu"].float()
    out = dict(hidden=(_act(s["act"], g) * u).to(t))
    return dict(out, gate=g.to(t), up=u.to(t)) if s["keep"] else out


def _gated_bwd(s):
    t = TYPES[s["type"]]
    x, g, u, dh = (s[k].float() for k in ("x", "gate", "up", "dh"))
    dg, du = dh * u * _act_slope(s["act"], g), dh * _act(s["act"], g)
    dx = dg @ s["wg"].float().T + du @ s["wu"].float().T
    return dict(dx=dx.to(t), dw_gate=(x.T @ dg).to(t), dw_up=(x.T @ du).to(t))


def _encode(x, word, signed):
    """Values to float8 (e4m3) and a scale for each 256 of them, the block's largest on 448.  The cut adds the word's top
    20 bits to the 20 mantissa bits that go, so that values between two neighbours go to either in proportion; a value
    that is not zero stays that where it has no sign (a second moment's root)."""
    largest = x.abs().reshape(-1, BLOCK).amax(1)
    live = largest >= 2.0 ** -100
    factor = torch.where(live, 448.0 / torch.where(live, largest, torch.ones_like(largest)), torch.zeros_like(largest))
    a = (x.abs().reshape(-1, BLOCK) * factor[:, None]).reshape(-1)
    low = a < 2.0 ** -6
    bits = torch.where(low, a + 2.0 ** -6, a).view(torch.int32)
    code = ((bits + (word >> 12).to(torch.int32)) >> 20) - torch.where(low, 968, 960)
    code = code.clamp(max=126)
    code = code + torch.where(x < 0, 128, 0) if signed else torch.where((code == 0) & (a > 0), 1, code)
    return code.to(torch.uint8).view(torch.float8_e4m3fn), torch.where(live, largest * (1.0 / 448.0), torch.zeros_like(largest))


def _decode(code, scale):
    return (code.float().reshape(-1, BLOCK) * scale[:, None]).reshape(-1)


def _word(index, step, shift):
    """Equally spread 32-bit words for the rounding of element `index` at `step`: the sum of a multiple of the golden
    section and one of the square root of two."""
    return (index * 0x9E3779B9 + step * 0x6A09E667 + shift) & 0xFFFFFFFF


def _corrections(s, dtype=np.float32):
    one, b1, b2 = dtype(1.0), dtype(np.float32(s["beta1"])), dtype(np.float32(s["beta2"]))
    return (float(b1), float(one - b1), float(one / (one - b1 ** dtype(s["step"]))),
            float(b2), float(one - b2), float(one / (one - b2 ** dtype(s["step"]))))


def _adamw_step(s):
    b1, c1, k1, b2, c2, k2 = _corrections(s)
    g, p = s["g"].float(), s["p"]
    if s["bits"] == 8:
        root = _decode(s["v"], s["vs"])
        m, v = _decode(s["m"], s["ms"]) * b1 + g * c1, root * root * b2 + g * c2 * g
        root = v.sqrt()
        size = root * float(np.sqrt(np.float32(k2)))
        for key, x, shift in (("m", m, 0), ("v", root, 0x80000000)):
            code, scale = _encode(x, _word(s["index"], s["step"], shift), key == "m")
            s[key].copy_(code)
            s[key + "s"].copy_(scale)
    else:
        m, v = s["m"] * b1 + g * c1, s["v"] * b2 + g * c2 * g
        size = (v * k2).sqrt()
        s["m"].copy_(m)
        s["v"].copy_(v)
    p.copy_(p - ((m * k1) / (size + s["eps"]) + p * s["decays"]) * s["lr"])
    if s["copy16"] is not None:
        s["copy16"].copy_(p)
    return _adamw_outputs(s)


def _adamw_outputs(s):
    return {k: s[k] for k in ("p", "m", "v", "ms", "vs", "copy16") if s.get(k) is not None}


# ---- the framework's calls --------------------------------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _backend():
    from see_ai_b200 import backend as B
    be = B.CudaBackend(torch.cuda.current_device())
    be.set_stream(torch.cuda.current_stream().cuda_stream)
    return B, be


def _own_norm(s):
    B, be = _backend()
    kind = B.NORM_LAYER if s["kind"] == "layer" else B.NORM_RMS
    types = dict(x_type=B.TYPES[s["x"]], y_type=B.TYPES[s["y"]])
    rows, cols = s["rows"], s["cols"]
    layer = s["kind"] == "layer"
    if s["op"] == "norm_fwd":
        be.norm_forward(kind, rows, cols, s["x_in"].data_ptr(), s["gamma"].data_ptr(), s["beta"].data_ptr() if layer else 0,
                        s["y_out"].data_ptr(), s["mean"].data_ptr() if layer else 0, s["rstd"].data_ptr(), eps=s["eps"], **types)
        return dict(y=s["y_out"], mean=s["mean"], rstd=s["rstd"]) if layer else dict(y=s["y_out"], rstd=s["rstd"])
    if "work" not in s:
        s["work"] = torch.empty(B.norm_backward_workspace(rows, cols), device="cuda", dtype=torch.uint8)
    be.norm_backward(kind, rows, cols, s["dy"].data_ptr(), s["x_in"].data_ptr(), s["gamma"].data_ptr(),
                     s["mean"].data_ptr() if layer else 0, s["rstd"].data_ptr(), s["dx"].data_ptr(), s["dgamma"].data_ptr(),
                     s["dbeta"].data_ptr() if layer else 0, s["work"].data_ptr(), s["work"].numel(),
                     addend=0 if s["add"] is None else s["add"].data_ptr(), **types)
    out = dict(dx=s["dx"], dgamma=s["dgamma"])
    return dict(out, dbeta=s["dbeta"]) if layer else out


def _own_gated(s):
    B, be = _backend()
    shape = (s["rows"], s["d_in"], s["d_hidden"])
    kinds = dict(type=B.TYPES[s["type"]], act=B.ACTS[s["act"]])
    if s["op"] == "gated_fwd":
        be.gated_forward(*shape, s["x"].data_ptr(), s["wg"].data_ptr(), s["wu"].data_ptr(), s["hidden"].data_ptr(),
                         s["gate"].data_ptr() if s["keep"] else 0, s["up"].data_ptr() if s["keep"] else 0, **kinds)
        return dict(hidden=s["hidden"], gate=s["gate"], up=s["up"]) if s["keep"] else dict(hidden=s["hidden"])
    if "work" not in s:
        s["work"] = torch.empty(B.gated_backward_workspace(*shape), device="cuda", dtype=torch.uint8)
    be.gated_backward(*shape, s["dh"].data_ptr(), s["x"].data_ptr(), s["wg"].data_ptr(), s["wu"].data_ptr(), s["gate"].data_ptr(),
                      s["up"].data_ptr(), s["dx"].data_ptr(), s["dwg"].data_ptr(), s["dwu"].data_ptr(), s["work"].data_ptr(),
                      s["work"].numel(), **kinds)
    return dict(dx=s["dx"], dw_gate=s["dwg"], dw_up=s["dwu"])


def _own_adamw(s):
    B, be = _backend()
    if "table" not in s:   # a program lists its tensors once
        at = lambda key, start: 0 if s.get(key) is None else s[key].data_ptr() + start * s[key].element_size()  # noqa: E731
        s["table"] = B.adamw_tensors([
            dict(p=at("p", o), g=at("g", o), m=at("m", o), v=at("v", o), m_scale=at("ms", o // BLOCK), v_scale=at("vs", o // BLOCK),
                 copy=at("copy16", o), n=n, g_type=B.TYPES[s["grad"]], copy_type=B.TYPES["f32" if s["copy"] == "none" else s["copy"]],
                 no_decay=not decays)
            for (n, decays), o in zip(s["sizes"], s["starts"])])
        s["params"] = B.StepParams(s["lr"], s["beta1"], s["beta2"], s["eps"], s["decay"], 0, s["step"])
    be.adamw_step(s["table"], s["params"], state_bits=s["bits"])
    return _adamw_outputs(s)


def run(state):
    if own:
        if state["op"].startswith("norm"):
            return _own_norm(state)
        return _own_gated(state) if state["op"].startswith("gated") else _own_adamw(state)
    return {"norm_fwd": _norm_fwd, "norm_bwd": _norm_bwd, "gated_fwd": _gated_fwd, "gated_bwd": _gated_bwd, "adamw": _adamw_step}[state["op"]](state)


# ---- the same in 64 bits ------------------------------------------------------------------------------------

def _exact_norm(s):
    x, gamma = s["x_in"].double(), s["gamma"].double()
    layer = s["kind"] == "layer"
    n = x.shape[1]
    if s["op"] == "norm_fwd":
        mean = x.sum(1) / n if layer else torch.zeros(x.shape[0], dtype=torch.float64, device=x.device)
        var = ((x - mean[:, None]) ** 2).sum(1) / n
        rstd = 1.0 / (var + s["eps"]).sqrt()
        y = (x - mean[:, None]) * rstd[:, None] * gamma + (s["beta"].double() if layer else 0.0)
        return dict(y=y, mean=mean, rstd=rstd) if layer else dict(y=y, rstd=rstd)
    dy, rstd = s["dy"].double(), s["rstd"].double()[:, None]
    unit = (x - s["mean"].double()[:, None]) * rstd
    q = gamma * dy
    pull = unit * ((unit * q).sum(1, keepdim=True) / n) + (q.sum(1, keepdim=True) / n if layer else 0.0)
    dx = (q - pull) * rstd + (0.0 if s["add"] is None else s["add"].double())
    out = dict(dx=dx, dgamma=torch.einsum("rc,rc->c", dy, unit))
    return dict(out, dbeta=dy.sum(0)) if layer else out


def _exact_gated(s):
    x, wg, wu = (s[k].double() for k in ("x", "wg", "wu"))

    def both(g):   # the activation and its slope
        if s["act"] == "relu":
            return g.clamp(min=0.0), (g > 0).double()
        if s["act"] == "silu":
            e = torch.exp(-g)
            return g / (1.0 + e), (1.0 + e + g * e) / (1.0 + e) ** 2
        inner = GELU_C * g * (1.0 + GELU_A * g ** 2)
        half = 1.0 / (1.0 + torch.exp(-2.0 * inner))
        return g * half, half + g * 2.0 * half * (1.0 - half) * GELU_C * (1.0 + 3.0 * GELU_A * g ** 2)

    if s["op"] == "gated_fwd":
        g, u = torch.matmul(x, wg), torch.matmul(x, wu)
        out = dict(hidden=both(g)[0] * u)
        return dict(out, gate=g, up=u) if s["keep"] else out
    value, slope = both(s["gate"].double())
    dh = s["dh"].double()
    dg, du = dh * s["up"].double() * slope, dh * value
    return dict(dx=torch.matmul(dg, wg.t()) + torch.matmul(du, wu.t()), dw_gate=torch.matmul(x.t(), dg), dw_up=torch.matmul(x.t(), du))


def _exact_adamw(s):
    b1, c1, k1, b2, c2, k2 = _corrections(s, np.float64)
    p, g = s["p"].double(), s["g"].double()
    m, v = s["m"].double(), s["v"].double()
    if s["bits"] == 8:
        wide = lambda scale: scale.double().repeat_interleave(BLOCK)  # noqa: E731
        m, v = m * wide(s["ms"]), (v * wide(s["vs"])) ** 2
    m, v = b1 * m + c1 * g, b2 * v + c2 * g * g
    p = p - float(np.float32(s["lr"])) * (k1 * m / ((k2 * v).sqrt() + float(np.float32(s["eps"]))) + s["decays"].double() * p)
    out = dict(p=p, m=m, v=v)
    if s["bits"] == 8:
        def held(x, shift):
            """What stands for x: its neighbours in e4m3 are a multiple of their distance, the lower one's share decides."""
            largest = x.abs().reshape(-1, BLOCK).amax(1)
            a = x.abs() * torch.where(largest > 0, 448.0 / largest, 0.0).repeat_interleave(BLOCK)
            distance = 2.0 ** (torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3.0)
            at = ((s["index"] * 0x9E3779B9 + s["step"] * 0x6A09E667 + shift) % (1 << 32)).div(4096, rounding_mode="floor").double() / (1 << 20)
            a = (torch.floor(a / distance + at) * distance).clamp(max=448.0)
            return x.sign() * a, largest / 448.0
        m8, ms = held(m, 0)
        v8, vs = held(v.sqrt(), 0x80000000)
        v8 = torch.where(v > 0, v8.clamp(min=2.0 ** -9), v8)
        out = dict(p=p, m=m8, v=v8, ms=ms, vs=vs)
    return out if s["copy16"] is None else dict(out, copy16=p)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"].startswith("norm"):
        return _exact_norm(s)
    return _exact_gated(s) if case["op"].startswith("gated") else _exact_adamw(s)


# ---- what a pass cannot do without ---------------------------------------------------------------------------

def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2, "none": 0}
    if case["op"].startswith("norm"):
        n, x, y = case["rows"] * case["cols"], size[case["x"]], size[case["y"]]
        if case["op"] == "norm_fwd":
            return {"bytes": n * (x + y) + 8.0 * (case["rows"] + case["cols"]), "flops": 7.0 * n}
        return {"bytes": n * (2 * x + y + (x if case["addend"] else 0)) + 8.0 * case["rows"] + 12.0 * case["cols"], "flops": 13.0 * n}
    if case["op"].startswith("gated"):
        m, d, f = float(case["rows"]), case["d_in"], case["d_hidden"]
        if case["op"] == "gated_fwd":
            return {"bytes": 2.0 * (m * d + 2 * d * f + m * f * (3 if case["keep"] else 1)), "flops": 4.0 * m * d * f}
        return {"bytes": 2.0 * (2 * m * d + 4 * d * f + 3 * m * f), "flops": 8.0 * m * d * f}
    n = float(sum(n for n, _ in _adamw_sizes(case)))
    states = 16.0 if case["bits"] == 32 else 4.0 + 16.0 / BLOCK
    return {"bytes": n * (8.0 + size[case["grad"]] + states + size[case["copy"]]), "flops": n * 14.0}
