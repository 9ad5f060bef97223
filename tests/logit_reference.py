"""Losses over rows of logits in 64 bits, with how far a sound f32 kernel may be off.

Let x = (z - max z) / ln 2 and e = 2^x.  A kernel's e is off by ex2.approx's 2^-22 and, relative, by ln 2 times what its exponent is off:
a rounding of the exponent and one of its factor, 2^-24 |x| each.  What else each exponent of a row has in common cancels.  A sum of
e has at most CHAIN(classes) additions on any path.  logp = (z_l - M) - log s adds roundings of its terms and results; where the label
holds more than half, -log1p(others / e_l) is off by the same relative to itself.
"""

import math

import torch

ULP = 2.0 ** -24
LN2 = math.log(2.0)
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def chain(classes):
    """Eight in a unit, a thread's units, and sixteen to join threads, warps and blocks (each with a factor, 2^-22 and a rounding: four)."""
    return 8 + max(16, classes // 4096 + 1) + 4 * 16


def rounding(dtype, value):
    if dtype == torch.float32:
        return ULP * value.abs() + 2.0 ** -126   # (results below are flushed)
    f = torch.finfo(dtype)
    return f.eps / 2 * value.abs() + f.smallest_normal * f.eps / 2


class Rows:
    """Log-probabilities of the labels and what dlogits are made of, with their errors' bounds; rows that do not count: zeros."""

    def __init__(self, logits, labels, logit_scale=1.0):
        self.classes, self.dtype = logits.shape[1], logits.dtype
        self.scale = float(torch.tensor(logit_scale, dtype=torch.float32))
        self.counts = (labels >= 0) & (labels < self.classes)
        self.index = labels.long().clamp(0, self.classes - 1)[:, None]
        z = logits.double() * self.scale
        z = torch.where(self.counts[:, None], z, 0.0)
        off = z - z.amax(1, keepdim=True)
        e = torch.exp(off)
        e = torch.where(off == -math.inf, 0.0, e)
        ex = torch.where(e > 0, e * off.abs(), 0.0)
        e_label, ex_label = e.gather(1, self.index), ex.gather(1, self.index)
        others, s = e.scatter(1, self.index, 0.0).sum(1, keepdim=True), e.sum(1, keepdim=True)
        z_label = off.gather(1, self.index)
        exact = torch.where(e_label > others, -torch.log1p(others / e_label), z_label - s.log())
        each = 2.0 ** -22 + chain(self.classes) * ULP
        off_s = each + 2 * ULP * ex.sum(1, keepdim=True) / s                       # relative, of s
        off_others = each + 2 * ULP * ex.scatter(1, self.index, 0.0).sum(1, keepdim=True) / others.clamp(min=1e-300)
        direct = off_s + 4 * ULP * (z_label.abs() + s.log() + exact.abs())
        near = exact.abs() * (off_others + each + 2 * ULP * ex_label / e_label.clamp(min=1e-300) + 8 * ULP) + 2.0 ** -126
        zero = lambda t: torch.where(self.counts, t[:, 0], 0.0)  # noqa: E731
        self.logp, self.logp_off = zero(exact), zero(torch.where(e_label > others, near, direct))
        self.p, self.left = e / s, others / s
        # An e below 2^-126 is flushed to zero: p = e / s loses at most that, for s is 1 at least (the maximum's own e).
        self.p_off = self.p * (off_s + each + 2 * ULP * off.abs().clamp(max=1e4) + 4 * ULP) + 2.0 ** -126
        self.left_off = self.left * (off_s + off_others + 4 * ULP)

    def check_logp(self, logp):
        assert ((logp.double() - self.logp).abs() <= self.logp_off + ULP * self.logp.abs()).all()

    def check_dlogits(self, d, slope, slope_off):
        """slope: of the loss by logp, [rows]."""
        want = -slope[:, None] * self.p * self.scale
        allowed = self.scale * (slope.abs()[:, None] * self.p_off + slope_off[:, None] * self.p)
        of_label, its_allowed = slope[:, None] * self.left * self.scale, self.scale * (slope.abs()[:, None] * self.left_off + slope_off[:, None] * self.left)
        want, allowed = want.scatter(1, self.index, of_label), allowed.scatter(1, self.index, its_allowed)
        want, allowed = (torch.where(self.counts[:, None], t, 0.0) for t in (want, allowed))
        allowed = allowed * 1.001 + 3 * ULP * want.abs()   # (three products)
        ok = (d.double() - want).abs() <= allowed + rounding(self.dtype, want.abs() + allowed)
        assert ok.all(), (int((~ok).sum()), float(((d.double() - want).abs() / (allowed + rounding(self.dtype, want))).max()))
        assert (d[~self.counts] == 0).all()


def policy(rows, old, ref, advantages, weights, clip_low, clip_high, kl_coef):
    """Per row: slope and its bound, loss, kl, clipped, each times the weight, and the loss's and kl's bounds."""
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))  # noqa: E731
    low, high, kl_coef = 1.0 - f32(clip_low), 1.0 + f32(clip_high), f32(kl_coef)
    a, w = advantages.double(), torch.where(rows.counts, weights.double() if weights is not None else 1.0, 0.0)
    diff = torch.where(rows.counts, rows.logp - old.double(), 0.0)
    off = rows.logp_off + ULP * (rows.logp.abs() + diff.abs())      # of the difference
    r = torch.exp(diff)
    cut = r.clamp(low, high)
    clipped = r * a > cut * a
    loss, slope = torch.where(clipped, -cut * a, -r * a), torch.where(clipped, 0.0, -r * a)
    slope_off = (r * a).abs() * (off + 6 * ULP) * (~clipped)
    loss_off = torch.where(clipped, (cut * a).abs() * 4 * ULP, slope_off)
    kl, kl_off = torch.zeros_like(loss), torch.zeros_like(loss)
    if ref is not None:
        x = torch.where(rows.counts, ref.double() - rows.logp, 0.0)
        off = rows.logp_off + ULP * (rows.logp.abs() + x.abs())
        grown = torch.expm1(x)
        kl = grown - x
        kl_off = grown.abs() * off + 3 * ULP * (grown.abs() + x.abs())
        loss, loss_off = loss + kl_coef * kl, loss_off + kl_coef * kl_off + 2 * ULP * (loss.abs() + kl_coef * kl)
        slope_off = slope_off + kl_coef * ((1 + grown.abs()) * off + 4 * ULP * grown.abs()) + ULP * (slope.abs() + kl_coef * grown.abs())
        slope = slope - kl_coef * grown
    near = ((r - low).abs() < 1e-5) | ((r - high).abs() < 1e-5)
    assert not (near & rows.counts).any(), "a ratio lies next to a corner"
    zero = lambda t: torch.where(rows.counts, t * w, 0.0)  # noqa: E731
    return dict(slope=zero(slope), slope_off=zero(slope_off).abs() + 2 * ULP * zero(slope).abs(), loss=zero(loss), kl=zero(kl),
                clipped=zero(clipped.double()), loss_off=zero(loss_off).abs() + ULP * zero(loss).abs(), kl_off=zero(kl_off).abs() + ULP * zero(kl).abs())


def preference(rows, starts, ref, kind, beta, smoothing, margin, average):
    """Loss, margins, sums, slopes of the rows, and their bounds."""
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))  # noqa: E731
    beta, smoothing, margin = f32(beta), f32(smoothing), f32(margin)
    starts = starts.tolist()
    pairs = (len(starts) - 1) // 2
    n = rows.logp.numel()
    sums, offs, counts = [], [], []
    for b, e in zip(starts[:-1], starts[1:]):
        c = int(rows.counts[b:e].sum())
        by = 1.0 / c if average and c else 1.0
        counts.append(by)
        sums.append(float(rows.logp[b:e].sum()) * by)
        offs.append(float((rows.logp_off[b:e] + ULP * rows.logp[b:e].abs()).sum()) * by)
    slopes, slopes_off = (torch.zeros(n, device=rows.logp.device, dtype=torch.float64) for _ in range(2))
    loss, loss_off, margins, margins_off = 0.0, 0.0, [], []
    for i in range(pairs):
        a, b = 2 * i, 2 * i + 1
        ra, rb = (float(ref[a]), float(ref[b])) if ref is not None else (0.0, 0.0)
        h = beta * ((sums[a] - ra) - (sums[b] - rb)) - margin
        off = beta * (offs[a] + offs[b])
        if kind == "sigmoid":
            soft = lambda v: max(v, 0.0) + math.log1p(math.exp(-abs(v)))  # noqa: E731
            chance = 1.0 / (1.0 + math.exp(h)) if h < 700 else 0.0   # of -h
            value, slope = (1 - smoothing) * soft(-h) + smoothing * soft(h), smoothing - chance
            value_off, slope_off = off, chance * (1.0 - chance) * off * math.exp(min(off, 1.0))
        elif kind == "hinge":
            assert abs(h - 1.0) > 2 * off, "a margin lies next to the corner"
            value, slope, value_off, slope_off = max(0.0, 1.0 - h), -1.0 if h < 1.0 else 0.0, off if h < 1.0 else 0.0, 0.0
        else:
            d = (h - 0.5) / beta
            value, slope, slope_off = d * d, 2.0 * d / beta, 2.0 * off / beta ** 2
            value_off = 2.0 * abs(d) * off / beta + (off / beta) ** 2
        loss, loss_off = loss + value / pairs, loss_off + value_off / pairs
        margins.append(h)
        margins_off.append(off)
        for seq, sign in ((a, 1.0), (b, -1.0)):
            by = beta / pairs * counts[seq]
            slopes[starts[seq]:starts[seq + 1]] = sign * slope * by
            slopes_off[starts[seq]:starts[seq + 1]] = slope_off * by + ULP * abs(slope * by)
    t = lambda v: torch.tensor(v, dtype=torch.float64)  # noqa: E731
    return dict(loss=loss, loss_off=loss_off + ULP * abs(loss), margins=t(margins), margins_off=t(margins_off) + ULP * t(margins).abs(), sums=t(sums),
                sums_off=t(offs) + ULP * t(sums).abs(), slopes=slopes, slopes_off=slopes_off)
