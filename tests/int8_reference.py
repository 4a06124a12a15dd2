"""Plain statements in 64 bits of the 8-bit rows, products and log probabilities,
and how far the operators' F32 arithmetic may be from them (u = 2^-24, half a step
of F32)."""
import numpy as np
import torch

U = 2.0 ** -24
LEAST = 127 * 2.0 ** -126


def check_rows(data, scale, y, rel):
    """8-bit rows against y (64 bits): rel bounds the relative error of the operator's
    F32 values of y. Its a = max |y| is within rel, the scale rounds once more; y * (127 / a)
    has rel from y, rel from a and two roundings, the integer half a step."""
    data, scale, y = data.cpu().to(torch.float64), scale.cpu().to(torch.float64), y.cpu()
    finite = torch.isfinite(y).all(-1)
    assert bool(torch.isnan(scale[~finite]).all()), "scales of rows with values that are not finite"
    amax = y.abs().amax(-1)
    none = finite & (amax < LEAST)
    assert bool((scale[none] == 0).all()) and bool((data[none | ~finite] == 0).all()), "rows of zeros"
    rows = finite & ~none
    data, scale, y, amax = data[rows], scale[rows], y[rows], amax[rows]
    if torch.is_tensor(rel):
        rel = rel.cpu()[rows]
    off = (scale * 127 / amax - 1).abs()
    assert bool((off <= rel + 1.01 * U).all()), f"scales off by {off.max().item():.3g}"
    limit = torch.as_tensor(0.5 + 127 * (2 * rel + 2.1 * U)).expand(len(y))
    away = (data - y * (127 / amax)[:, None]).abs().amax(-1)
    assert bool((away <= limit).all()), f"integers off by {away.max().item():.6g}"
    assert bool((data.abs() <= 127).all())


def norm(h, weight, eps):
    h = h.double()
    return h / (h.square().mean(-1, keepdim=True) + float(np.float32(eps))).sqrt() * weight.double()


# the sum of squares: at most 64 terms one after another, 6 steps of a tree, 16 waves, as
# many roundings; the division by the channels and eps one each, halved by the root; the root, its
# inverse and two products one each
NORM_REL = ((64 + 6 + 16 + 2) / 2 + 4) * U


def gated(gate, up):
    g = gate.double()
    return g * torch.sigmoid(g) * up.double()


def gated_rel(gate):
    """The exponent's product and constant are off by up to 1.5 u |g| together, 2^x and the
    reciprocal by a step (2 u), the sum and two products round once each."""
    return (1.5 * gate.double().abs().amax(-1) + 7) * U


def linear(x, w, dtype):
    """The definition's own roundings: the sum (exact in 64 bits) to F32, each product, the
    result's type."""
    (x, sx), (w, sw) = x, w
    sums = x.double() @ w.double().t().contiguous()
    return (sums.float() * sx[:, None] * sw).to(dtype)


# ---------------------------------------------------------- log probabilities


def logprobs(x, tokens, top):
    """(logprobs, entropy, top tokens, top logprobs) in 64 bits; tokens [rows, given]."""
    x = x.cpu().double().numpy()
    rows, vocab = x.shape
    tokens = tokens.cpu().numpy()
    lp, entropy = np.full(tokens.shape, np.nan), np.full(rows, np.nan)
    best, best_lp = np.zeros((rows, top), np.int64), np.full((rows, top), np.nan)
    for r in range(rows):
        # NaN first, then descending; a stable sort leaves the lowest index in front
        order = np.lexsort((-np.nan_to_num(x[r] + 0.0, nan=0.0, posinf=np.inf, neginf=-np.inf), ~np.isnan(x[r])))
        best[r] = order[:top]
        m = x[r].max()
        if not np.isfinite(m):
            continue
        d = x[r] - m
        e = np.exp(d)
        s = e.sum()
        entropy[r] = np.log(s) - (e * np.where(e > 0, d, 0.0)).sum() / s
        inside = (tokens[r] >= 0) & (tokens[r] < vocab)
        lp[r, inside] = d[tokens[r, inside]] - np.log(s)
        best_lp[r] = d[best[r]] - np.log(s)
    return lp, entropy, best, best_lp


def logprob_limits(x, d):
    """How far log probabilities of logits d below the maximum, and entropies, may be off. The
    weighted mean of |x - m| over a row, E, is entropy - log s, at most log(vocab). s: a term's exponent
    is off by 2.5 u |x - m| (so s by 2.5 u E), a term by a step more, and at most vocab / 256 + 64 terms
    are added one after another. log s rounds within two steps, d once, the difference once; the
    entropy's sum is off as s is, in terms of E."""
    vocab = x.shape[1]
    rows = x.cpu().double()
    m = rows.amax(-1, keepdim=True)
    log_s = np.log(np.exp((rows - m).numpy()).sum(-1))
    mean = np.log(vocab) + 1
    of_s = (2 + 2.5 * mean + vocab / 256 + 64) * U
    log_off = of_s + 4 * U * np.abs(log_s)
    lp = log_off[:, None] + 2 * U * (np.abs(d) + log_s[:, None])
    return lp, log_off + mean * (2 * of_s + 4 * U) + 2 * U * log_s
