"""Plain implementations of the operators of ``multigrid_amd.policy`` in 64 bits, on the CPU, one row or token at a time
where that is plainest, with the bounds that 32-bit arithmetic may be off by."""
import math

import numpy as np
import torch

U32 = 2.0 ** -24  # half a step of float32, relative
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SMALLEST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def np64(t):
    return t.detach().cpu().double().numpy()


def close(got, want, err, dtype):
    """``got`` (a tensor of ``dtype``) is ``want`` (64 bits) within ``err`` of 32-bit arithmetic and one rounding to its type;
    infinities and NaN have to be in the same places."""
    got = np64(got)
    assert got.shape == want.shape, (got.shape, want.shape)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    bound = err + HALF_STEP[dtype] * (np.abs(want) + err) + SMALLEST[dtype] / 2
    with np.errstate(invalid="ignore"):
        off = np.abs(got - want)
    bad = fine & ~(off <= bound)
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, e.g. {got[bad][0]} for {want[bad][0]} (bound {np.broadcast_to(bound, got.shape)[bad][0]})"


def embed(ids, table, sizes, scale):
    """(values, bound of the 32-bit sums): fields - 1 additions and a product, each off by half a step of what it gives."""
    w, ids = np64(table), ids.cpu().numpy().astype(np.int64).reshape(-1, len(sizes))
    out, size = np.zeros((len(ids), w.shape[1])), np.zeros((len(ids), w.shape[1]))
    base = 0
    for f, rows in enumerate(sizes):
        ok = (ids[:, f] >= 0) & (ids[:, f] < rows)
        out[ok] += w[base + ids[ok, f]]
        size[ok] += np.abs(w[base + ids[ok, f]])
        base += rows
    s = float(np.float32(scale))
    return out * s, size * abs(s) * U32 * (len(sizes) + 1)


def embed_grad(ids, grad, sizes, scale):
    """(values, bound): a sum of m numbers in any order is off by at most m half steps of the sum of their magnitudes."""
    g, ids = np64(grad).reshape(-1, grad.shape[-1]), ids.cpu().numpy().astype(np.int64).reshape(-1, len(sizes))
    out, size = np.zeros((sum(sizes), g.shape[1])), np.zeros((sum(sizes), g.shape[1]))
    many = np.zeros((sum(sizes), 1))
    base = 0
    for f, rows in enumerate(sizes):
        ok = (ids[:, f] >= 0) & (ids[:, f] < rows)
        with np.errstate(invalid="ignore"):
            np.add.at(out, base + ids[ok, f], g[ok])
        np.add.at(size, base + ids[ok, f], np.abs(g[ok]))
        np.add.at(many, base + ids[ok, f], 1.0)
        base += rows
    s = float(np.float32(scale))
    with np.errstate(invalid="ignore"):
        return out * s, size * abs(s) * U32 * (many + 2)


def history_counts(history, lengths, n, k):
    c = np.zeros((n, k))
    if history is None:
        return c
    h = history.cpu().numpy().astype(np.int64)
    h = np.broadcast_to(h, (n, h.shape[-1]))
    for i in range(n):
        length = h.shape[1] if lengths is None else min(max(int(lengths[i]), 0), h.shape[1])
        for j in h[i, :length]:
            if 0 <= j < k:
                c[i, j] += 1
    return c


def allowed(mask, n, k):
    if mask is None:
        return np.ones((n, k), bool)
    m = mask.cpu().numpy()
    if mask.dtype == torch.int32:
        at = np.arange(k)
        m = (m.astype(np.int64)[..., at // 32] >> (at % 32)) & 1
    return np.broadcast_to(m != 0, (n, k))


def per_row(v, n):
    v = np64(v) if isinstance(v, torch.Tensor) else np.float64(np.float32(v))
    return np.broadcast_to(v, (n,))[:, None]


def adjust(logits, history=None, lengths=None, repetition=1.0, presence=0.0, frequency=0.0, bias=None, mask=None):
    """(values, bound, factor of the gradient): at most six operations (1 / repetition, its product, presence, frequency times
    c, that, bias), each off by half a step of what it gives."""
    x = np64(logits)
    n, k = x.shape
    c, r = history_counts(history, lengths, n, k), per_row(repetition, n)
    with np.errstate(invalid="ignore", over="ignore"):
        factor = np.where(c > 0, np.where(x > 0, 1 / r, r), 1.0)
        b = 0.0 if bias is None else np64(bias)
        parts = (np.where(c > 0, np.where(x > 0, x / r, x * r), x), -np.where(c > 0, per_row(presence, n), 0.0), -per_row(frequency, n) * c, b)
        y = parts[0] + parts[1] + parts[2] + parts[3]
        size = sum(np.abs(p) for p in parts)
    ok = allowed(mask, n, k)
    return np.where(ok, y, -np.inf), np.where(ok & np.isfinite(size), 6 * U32 * size, 0.0), np.where(ok, factor, 0.0)


def draw(logits, uniforms, temperature=1.0):
    """(tokens, log-probabilities, distance of the nearest border relative to the total)."""
    x = np64(logits)
    n, k = x.shape
    t = per_row(temperature, n)[:, 0]
    tokens, lp, margin = np.zeros(n, np.int64), np.zeros(n), np.full(n, np.inf)
    for i in range(n):
        best = np.max(x[i])  # NaN if one is there
        if not np.isfinite(best):
            tokens[i], lp[i] = -1, -np.inf if best == -np.inf else np.nan
            continue
        z = (x[i] - best) / t[i]
        p = np.exp(z)
        upto = np.array([math.fsum(p[:1])]) if k == 1 else np.cumsum(p)
        if uniforms is None:
            tokens[i] = int(np.argmax(x[i]))
        else:
            border = float(uniforms[i]) * upto[-1]
            above = np.nonzero(upto > border)[0]
            tokens[i] = above[0] if len(above) else np.nonzero(p > 0)[0][-1]
            margin[i] = np.min(np.abs(upto - border)) / upto[-1]
        lp[i] = z[tokens[i]] - np.log(upto[-1])
    return tokens, lp, margin


def logprobs(logits, tokens, temperature, grad=None, grad_entropy=None):
    """Values and bounds of the log-probabilities, the entropies and (with gradients) the logits' gradient.

    z = (x - m) / T is off by 5 half steps of itself (difference, 1 / T, its product with log2(e) / 2, that constant, the product
    of both), so an exponential, the square of an instruction's result within one step, by (5 |z| + 5) of them; a sum over k
    numbers, in at least 64 parts, by k / 64 + 16.  The sum r of all exponentials but the maximum's own 1 is taken without that
    1 where it is small; from 1 / 17 on it may be a sum with it, less 1, whose roundings are of 1 + r."""
    x = np64(logits)
    n, k = x.shape
    t = per_row(temperature, n)
    m = np.max(x, 1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        z = (x - m) / t
        e = np.exp(z)
        live = e > 0
        az = np.where(live, np.abs(z), 0.0)
        rest = e.copy()
        rest[np.arange(n), np.argmax(x, 1)] = 0.0  # the maximum's own 1 is exact
        r = rest.sum(1, keepdims=True)
        log_total = np.log1p(r)
        depth = k / 64 + 16
        # an exponential below 2^-126 is held in steps of 2^-149 (of e^-101 and less nothing is left: 8.8e-44 of an entropy
        # becomes 0): 2 steps each, times |z| where z multiplies it; |z| above 110 adds less than a step
        grid = 2 * 2.0 ** -149
        dr = U32 * ((rest * (5 * az + 5)).sum(1, keepdims=True) + depth * np.where(r > 1 / 17, 1 + r, r)) + k * grid
        tz = np.where(live, e * z, 0.0).sum(1, keepdims=True)
        dt = U32 * ((e * az * (5 * az + 9)).sum(1, keepdims=True) + depth * np.abs(tz)) + grid * (1 + np.minimum(az, 110.0)).sum(1, keepdims=True)
        entropy = log_total - tz / (1 + r)
        d_log = dr / (1 + r) + 4 * U32 * log_total
        d_entropy = d_log + dt / (1 + r) + np.abs(tz) * dr / (1 + r) ** 2 + 4 * U32 * (log_total + np.abs(tz) / (1 + r))
        empty = m == -np.inf
        log_total, entropy = np.where(empty, 0.0, log_total), np.where(empty, 0.0, entropy)
        d_log, d_entropy = (np.where(empty, 0.0, v) for v in (d_log, d_entropy))
        lp = np.where(empty, -np.inf, z - log_total)
        d_lp = d_log + U32 * (4 * np.where(np.isfinite(z), np.abs(z), 0.0) + np.where(np.isfinite(lp), np.abs(lp), 0.0))
    tok = tokens.cpu().numpy().astype(np.int64)
    known = (tok >= 0) & (tok < k)
    at = np.where(known, tok, 0)
    taken = np.where(known, lp[np.arange(n), at], 0.0), np.where(known, d_lp[np.arange(n), at], 0.0)
    result = [taken, (entropy[:, 0], d_entropy[:, 0])]
    if grad is not None:
        with np.errstate(invalid="ignore", over="ignore"):
            g = np.where(known, np64(grad), 0.0)[:, None]
            h = np64(grad_entropy)[:, None]
            p = np.exp(lp)
            hot = np.zeros((n, k))
            hot[np.arange(n)[known], tok[known]] = 1.0
            none = x == -np.inf
            s = np.where(none, 0.0, lp + entropy)
            off = np.where(hot > 0, np.where(none, 0.0, -np.expm1(lp)), p)  # |1[a] - p|
            d = (g * np.where(hot > 0, off, -p) - h * p * s) / t
            d = np.where(none, 0.0, d)
            # a probability below 2^-126 is held in steps of 2^-149, however exact its exponent: half a step for its rounding,
            # one for the exponential, and what follows multiplies it (1.2e-43 as 1.18e-43, times a log-probability of -94,
            # moves the product by 1 in 60 of itself)
            dp = p * (d_lp + 4 * U32) + 2 * 2.0 ** -149
            err = (np.abs(g) * (np.where(hot > 0, dp + 4 * U32 * off, dp)) + np.abs(h) * (np.abs(s) * dp + p * (d_lp + d_entropy))
                   + 6 * U32 * (np.abs(g) * off + np.abs(h) * p * np.abs(s))) / t
        result.append((d, np.where(none, 0.0, err)))
    return result
