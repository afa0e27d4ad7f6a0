"""Rows of logits of large magnitude, and small temperatures: log-sum-exp, loss and gradients against float64
formed from differences to the row's maximum (exact rational numbers where a given log-sum-exp is subtracted).
`api` is the package or its CPU mode.

Tolerances, u = 2^-24 a float32 rounding.  With d = (x - max) / T, exact here:
  log q   the scaled difference is off by three roundings of itself, the sum by those of its terms (at most 40
          below the largest count), 8 u for exp and log and up to vocab / 256 + 72 additions in a row
          -> u (8 |log q| + vocab / 256 + 240); the same relative to q
  log p   likewise over k <= 16 entries: u (8 |log p| + 120), and relative to p
  lse     the sum as above, peak / T or its scaled form, product, sum and last factor: 6 u |lse|
  q from a given lse: exponent E = x / T - lse.  lse * T is rounded to m, and what that took off is put back: both
          parts, of size A = |x - m| / T + |lse T - m| / T, carry three roundings -> u (6 A + 60)
and half a step of the result's type on top."""

from fractions import Fraction

import numpy as np

from tests.logits_cases import HALF_STEP, SMALLEST, U, close, decode, encode, in_float32, np_dtype  # noqa: F401

K = 8


def rows_of(kind, magnitude, temperature, vocab, rng):
    """One row: float64 values, rounded to the type afterwards."""
    x = rng.standard_normal(vocab) * 3
    at = np.arange(vocab)
    if kind == "mostly masked":
        x[rng.random(vocab) < 0.9] = -magnitude
    elif kind == "masked":
        x[:] = -magnitude
    elif kind == "begins masked":                # whole lanes and wavefronts begin with masked entries
        x[at < vocab * 5 // 8] = -magnitude
    elif kind == "ends masked":
        x[at > vocab * 3 // 8] = -magnitude
    elif kind == "peaks":
        x[rng.integers(0, vocab, 3)] = magnitude
    elif kind == "peaks and masked":
        x[::2] = -magnitude
        x[rng.integers(0, vocab, 5)] = magnitude
    elif kind == "about":                        # all about the magnitude, a few steps of float32 apart
        step = float(np.spacing(np.float32(magnitude)))
        x = magnitude + step * rng.integers(0, 6, vocab)
    elif kind == "falling":                      # from large to small in long stretches
        x = x - magnitude * (at * 8 // vocab)
    elif kind == "rising":
        x = x + magnitude * (at * 8 // vocab)
    else:
        assert kind == "small temperature"
        x = x * magnitude
    return x


def exponent(x, temperature, lse):
    """x / temperature - lse in float64, formed exactly where it is not far from zero."""
    t, g = Fraction(temperature), Fraction(lse)
    out = np.empty(x.shape)
    values, back = np.unique(x, return_inverse=True)
    rough = values / temperature - lse
    unsure = np.abs(rough) < 1000 + 1e-14 * np.abs(lse)
    fine = np.where(unsure, 0.0, rough)
    for n in np.flatnonzero(unsure):
        e = Fraction(float(values[n])) / t - g
        fine[n] = float(max(min(e, Fraction(10) ** 300), -Fraction(10) ** 300))
    out[...] = fine[back.reshape(x.shape)]
    return out


def check(api, name, lines, temperature, copies=1, calls=("top", "loss", "both", "grad"), seed=0):
    """`lines`: rows, one after the other, each `copies` times over."""
    rng = np.random.default_rng(seed)
    t = float(np.float32(temperature))
    a, x = encode(np.stack(lines), name)
    rows, vocab = x.shape
    op = api.logits
    peak = x.max(1)
    d = (x - peak[:, None]) / t
    total = np.exp(d).sum(1)
    lse = in_float32(peak / t + np.log(total))
    log_q = d - np.log(total)[:, None]
    q = np.exp(np.maximum(log_q, -745))
    tol_lse = U * (6 * np.abs(np.where(np.isfinite(lse), lse, 0)) + vocab / 256 + 240)
    many = lambda v: np.repeat(v, copies, 0)                                    # noqa: E731
    send = lambda v: api.to_device(np.ascontiguousarray(many(v)))               # noqa: E731
    dx = send(a)

    if "top" in calls:
        got = op.top(dx, 3, lse=True, temperature=temperature)
        close(got[2].copy_to_host(), many(lse), many(tol_lse), "lse of top")
        order = np.argsort(-x, axis=1, kind="stable")[:, :3]
        assert np.array_equal(got[1].copy_to_host(), many(order))

    # a teacher whose entries are the student's largest, its smallest and others; one absent
    indices = np.stack([np.concatenate([[v.argmax(), v.argmin()], rng.permutation(vocab)[:K - 2]]) for v in x])
    indices[:, 5] = -1
    teacher = (rng.standard_normal((rows, K)) * 2 * min(t, 1.0)).astype(np.float32)
    there = indices >= 0
    z = np.where(there, teacher.astype(np.float64) / t, -np.inf)
    z = z - z.max(1, keepdims=True)
    log_p = np.where(there, z - np.log(np.exp(z).sum(1, keepdims=True)), 0)
    p = np.where(there, np.exp(log_p), 0)
    named = np.take_along_axis(log_q, np.maximum(indices, 0), 1)
    gap = np.where(there, log_p - named, 0)
    loss = (p * gap).sum(1)
    tol_p = U * (8 * np.abs(log_p) + 120)
    tol_loss = (p * (U * (8 * np.abs(named) + vocab / 256 + 240) + tol_p + tol_p * np.abs(gap))).sum(1) + 2.0 ** -149
    grad_loss = ((0.5 + rng.random(rows)) * t).astype(np.float32)
    factor = (grad_loss.astype(np.float64) / t)[:, None]
    share, tol_share = np.zeros_like(x), np.zeros_like(x)
    for r in range(rows):
        np.add.at(share[r], indices[r][there[r]], p[r][there[r]])
        np.add.at(tol_share[r], indices[r][there[r]], (p * tol_p)[r][there[r]])
    mass = p.sum(1, keepdims=True)

    def check_gradient(got, q, tol_q, what, unclear=False):
        with np.errstate(over="ignore", invalid="ignore"):
            want = factor * (mass * q - share)
            tol = factor * (q * tol_q + tol_share + 16 * U * (q + share)) + HALF_STEP[name] * np.abs(want) * (1 + 1e-6)
            tol = tol + SMALLEST[name] + 2.0 ** -125 * factor
            want = in_float32(want)
            limit = 65504.0 if name == "float16" else np.finfo(np.float32).max
            want = np.where(np.abs(want) > limit, np.sign(want) * np.inf, want)
        got = np.where(many(np.broadcast_to(unclear, x.shape)), many(want), decode(got.copy_to_host()))
        close(got, many(want), many(np.where(np.isfinite(tol), tol, 0)), what)

    dv, di, dg = send(teacher), send(indices.astype(np.int32)), send(grad_loss)
    if "loss" in calls:
        got = op.distill_loss(dx, dv, di, temperature=temperature)
        close(got[1].copy_to_host(), many(lse), many(tol_lse), "lse of the loss")
        close(got[0].copy_to_host(), many(in_float32(loss)), many(tol_loss), "loss")
    if "both" in calls:
        got = op.distill_loss_and_grad(dg, dx, dv, di, temperature=temperature)
        close(got[1].copy_to_host(), many(lse), many(tol_lse), "lse of both")
        close(got[0].copy_to_host(), many(in_float32(loss)), many(tol_loss), "loss of both")
        check_gradient(got[2], q, U * (8 * np.abs(np.maximum(log_q, -745)) + vocab / 256 + 240), "gradient of both")
    if "grad" in calls:
        given = lse.astype(np.float32)
        got = op.distill_grad(dg, dx, dv, di, send(given), temperature=temperature)
        q, tol_q, unclear = np.zeros_like(x), np.zeros_like(x), np.zeros(x.shape, bool)
        for r in np.flatnonzero(np.isfinite(given)):         # a row whose lse is -inf has q = 0
            e = exponent(x[r], t, float(given[r]))
            near = float(np.float32(float(given[r]) * t))
            rest = float(abs(Fraction(float(given[r])) * Fraction(t) - Fraction(near)))
            off = U * (6 * (np.abs(x[r] - near) + rest) / t + 60)
            q[r], tol_q[r] = np.exp(np.minimum(e, 709)), np.expm1(np.minimum(off, 600))
            # within its tolerance of the end of the type's range a result may be on either side (the factor is
            # between 1/2 and 3/2, the mass 1)
            unclear[r] = np.abs(e - np.log(65504.0 if name == "float16" else 2.0 ** 128)) < off + 1
        assert unclear.mean() < 0.2
        check_gradient(got, q, tol_q, "gradient by itself", unclear)


# (kind, magnitude, temperature)
ORDINARY = [(kind, m, t) for kind in ("mostly masked", "masked", "begins masked", "ends masked", "peaks", "peaks and masked")
            for m, t in ((1e9, 0.3), (1e9, 0.1), (1e10, 1.0), (1e15, 1.0), (1e20, 1.0))]
STEEP = [("small temperature", 1.0, 1e-9), ("small temperature", 1.0, 1e-20), ("small temperature", 20.0, 1e-5),
         ("mostly masked", 1e10, 1e-9), ("begins masked", 1e15, 1e-20), ("masked", 1e9, 1e-9), ("peaks", 1e4, 1e-3)]
# about the magnitude from which the exponent of the reference is no longer a product rounded once (2^22 powers of
# two), on both sides of it in one row, and values that differ by single steps of float32
BORDER = [("about", 2.0 ** 22 / 1.4426950408889634, 1.0), ("about", 2.0 ** 22 / 1.4426950408889634 - 0.5, 1.0),
          ("about", 1e10, 700.0), ("about", 1e10, 1024.0), ("about", 3.3e6, 0.4), ("about", 4.1e6, 1.5),
          ("falling", 1e6, 1.0), ("rising", 1e6, 1.0), ("rising", 2907260.0, 1.0), ("falling", 3e9, 0.3)]
