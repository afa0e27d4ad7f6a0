"""Inputs and checks of the operators over rows of logits, shared by the GPU and the CPU mode's
tests.  `api` is the package (or its CPU mode): to_device / device_array / logits.

Tolerances, all against the float64 oracle on the rounded inputs; u = 2^-24 is a float32 rounding:
  adjust  at most six float32 operations, each off by at most u times the largest intermediate
  lse     every term of the sum: 2 u |z - peak| for the scaled difference, 4 u for exp, and at most
          vocab / 256 + 40 additions one after the other on the longest path (16 more where a row is
          split); peak / T, the logarithm and the last addition 3 u |lse|
  loss, gradient  the same errors of p and q, weighted by the terms they appear in
and half a step of the result's type on top."""

import numpy as np

from numba_cuda_amd._logits_host import bfloat16, from_bfloat16, to_bfloat16
from oracle import logits64

U = 2.0 ** -24
HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
SMALLEST = {"float32": 2.0 ** -149, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}   # half the least step near zero
DTYPES = ["float32", "float16", "bfloat16"]
LOWEST = {"float32": -np.finfo(np.float32).max, "float16": -65504.0, "bfloat16": -3.3895313892515355e38}


def np_dtype(name):
    return bfloat16 if name == "bfloat16" else np.dtype(name)


def encode(x, name):
    """float values -> array of the type, and the float64 values it really holds."""
    with np.errstate(over="ignore"):
        a = to_bfloat16(x) if name == "bfloat16" else np.asarray(x).astype(name)
    return a, decode(a)


def decode(a):
    a = np.asarray(a)
    return (from_bfloat16(a) if a.dtype == bfloat16 else a).astype(np.float64)


def rows_like(rng, rows, vocab, name, kind="normal"):
    x = rng.standard_normal((rows, vocab)) * 3.0
    if kind == "edge":
        # one row each of what a row can be; the rest are ordinary
        special = [np.full(vocab, -np.inf), np.full(vocab, LOWEST[name]), np.zeros(vocab),
                   np.arange(vocab) * 0.01 - 2, 2 - np.arange(vocab) * 0.01,
                   np.where(np.arange(vocab) % 2, 0.0, -0.0), np.where(rng.random(vocab) < 0.9, -np.inf, x[0]),
                   np.where(rng.random(vocab) < 0.9, LOWEST[name], x[0])]
        for r, line in enumerate(special[:rows]):
            x[r] = line
    return encode(x, name)


def padded(api, a, pad, before=0):
    """`a` on the device as columns before..before+n of a wider buffer."""
    if not pad:
        return api.to_device(np.ascontiguousarray(a))
    wide = np.zeros((a.shape[0], before + a.shape[1] + pad), a.dtype)
    wide[:, before:before + a.shape[1]] = a
    return api.to_device(wide)[:, before:before + a.shape[1]]


def close(got, want, tol, what):
    got, want, tol = np.asarray(got, np.float64), np.asarray(want, np.float64), np.broadcast_to(tol, np.shape(want))
    assert got.shape == want.shape, what
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan), "%s: NaN elsewhere" % what
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf]), "%s: infinities differ" % what
    fine = ~(nan | inf)
    with np.errstate(invalid="ignore"):
        bad = ~(np.abs(got[fine] - want[fine]) <= tol[fine])
        # a value whose tolerance reaches past float32's largest may have become infinite
        bad &= ~((np.abs(want) + tol >= np.finfo(np.float32).max) & (got == np.sign(want) * np.inf))[fine]
    assert not bad.any(), "%s: %d of %d off, worst %g over its tolerance %g" % (
        what, bad.sum(), bad.size, np.abs(got[fine] - want[fine])[bad].max(), tol[fine][bad].max())


def in_float32(x):
    """What lies beyond float32's range is infinite there (all of a row at the type's lowest value,
    divided by a temperature below one)."""
    return np.where(np.abs(x) > np.finfo(np.float32).max, np.sign(x) * np.inf, x)


# ---- adjust --------------------------------------------------------------------------------

def adjust_inputs(rng, rows, vocab, longest, pairs):
    lengths = rng.integers(0, longest + 1, rows)
    lengths[0] = longest
    if rows > 2:
        lengths[1] = 0
    offsets = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)
    # a few words often, a few outside the vocabulary
    tokens = (rng.random(offsets[-1]) ** 3 * vocab).astype(np.int64)
    if len(tokens) > 4:
        tokens[1], tokens[3] = -1, vocab + 3
    prompts = np.array([rng.integers(0, n + 1) for n in lengths], np.int64)
    counts = rng.integers(0, pairs + 1, rows)
    bias_offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)
    bias_tokens = rng.integers(-1, vocab + 1, bias_offsets[-1])
    bias_values = rng.standard_normal(bias_offsets[-1]).astype(np.float32) * 4
    mask = rng.integers(0, 2 ** 32, (rows, (vocab + 31) // 32), dtype=np.uint64).astype(np.uint32)
    mask[rng.random(mask.shape) < 0.3] = 0
    if rows > 3:
        mask[2], mask[3] = 0, 0xffffffff         # nothing allowed; everything
    return dict(tokens=tokens, offsets=offsets, prompts=prompts, bias_tokens=bias_tokens, bias_values=bias_values,
                bias_offsets=bias_offsets, mask=mask, lengths=lengths)


def allowed_of(mask, vocab):
    v = np.arange(vocab)
    return ((mask[:, v >> 5] >> (v & 31).astype(np.uint32)) & 1).astype(bool)


def check_adjust(api, rows, vocab, name, out_name, longest, pairs, with_mask, index="int32", kind="normal", pad=0,
                 in_place=False, per_row=True, seed=0):
    rng = np.random.default_rng(seed + rows * 1000003 + vocab)
    a, x = rows_like(rng, rows, vocab, name, kind)
    n = adjust_inputs(rng, rows, vocab, longest, pairs)
    rep, pre, fre = 1.0 + rng.random(rows), rng.random(rows), rng.random(rows) * 0.3
    rep, pre, fre = (v.astype(np.float32) for v in (rep, pre, fre))
    if not per_row:
        rep, pre, fre = np.float32(1.25), np.float32(0.5), np.float32(0.125)
    send = lambda v: api.to_device(np.ascontiguousarray(v))                     # noqa: E731
    arg = (lambda v: send(v)) if per_row else float
    d = padded(api, a, pad, before=min(pad, 3))
    kw = dict(repetition=arg(rep), presence=arg(pre), frequency=arg(fre), tokens=send(n["tokens"].astype(index)),
              offsets=send(n["offsets"].astype(index)), prompt_lengths=send(n["prompts"].astype(index)))
    if pairs:
        kw.update(bias_tokens=send(n["bias_tokens"].astype(index)), bias_values=send(n["bias_values"]),
                  bias_offsets=send(n["bias_offsets"].astype(index)))
    if with_mask == "rows":
        kw["mask"] = send(n["mask"])
        allowed = allowed_of(n["mask"], vocab)
    elif with_mask == "shared":
        kw["mask"] = send(n["mask"][0].view(np.int32))
        allowed = allowed_of(n["mask"][:1], vocab)
    else:
        allowed = None
    listed = [[(int(v), float(b)) for v, b in zip(n["bias_tokens"][lo:hi], n["bias_values"][lo:hi])]
              for lo, hi in zip(n["bias_offsets"], n["bias_offsets"][1:])] if pairs else None
    want = logits64.adjust(x, n["tokens"], n["offsets"], n["prompts"], rep, pre, fre, listed, allowed)
    # the largest intermediate of every entry
    size = np.abs(x) * np.reshape(rep, (-1, 1) if per_row else ()) + np.reshape(pre, (-1, 1) if per_row else ())
    size = size + np.reshape(fre, (-1, 1) if per_row else ()) * n["lengths"][:, None]
    if pairs and len(n["bias_values"]):
        size = size + np.abs(n["bias_values"]).max()
    if in_place:
        out = api.logits.adjust(d, d, **kw)
        assert out is d
    elif out_name == name:
        out = api.logits.adjust(d, **kw)
    else:
        out = api.device_array((rows, vocab), np_dtype(out_name))
        assert api.logits.adjust(d, out, **kw) is out
    got = decode(out.copy_to_host())
    step = HALF_STEP[out_name]
    with np.errstate(invalid="ignore", over="ignore"):
        if kind == "edge":                       # what overflows float32, or the type, is infinite
            want = decode(encode(in_float32(want), out_name)[0])
        tol = 6 * U * size + (step * np.abs(want) + SMALLEST[out_name]) * (3 if kind == "edge" else 1)
    close(got, want, np.where(np.isfinite(tol), tol, 0), "adjust")
    return got


# ---- top -----------------------------------------------------------------------------------

def lse_tolerance(x, temperature, lse):
    with np.errstate(invalid="ignore", over="ignore"):
        z = np.where(np.isfinite(x), x, 0) / temperature
        near = np.where(z > z.max(1, keepdims=True) - 40, z, z.max(1, keepdims=True))   # the rest adds nothing
        spread = near.max(1) - near.min(1)
        return U * (2 * spread + 4 + x.shape[1] / 256 + 56) + 3 * U * np.abs(lse) + U


def check_top(api, rows, vocab, name, k, lse=True, temperature=1.0, kind="normal", pad=0, seed=0, data=None):
    rng = np.random.default_rng(seed + rows * 1000003 + vocab)
    a, x = rows_like(rng, rows, vocab, name, kind) if data is None else encode(data, name)
    d = padded(api, a, pad, before=min(pad, 3))
    got = api.logits.top(d, k, lse=True, temperature=temperature) if lse else api.logits.top(d, k)
    values, indices = got[0].copy_to_host(), got[1].copy_to_host()
    want = logits64.top(x, k)
    assert indices.dtype == np.int32 and np.array_equal(indices, want)
    assert values.tobytes() == np.take_along_axis(a, want, 1).tobytes()
    if lse:
        exact = in_float32(logits64.lse(x, float(np.float32(temperature))))
        with np.errstate(invalid="ignore"):
            tol = lse_tolerance(x, temperature, np.where(np.isfinite(exact), exact, 0))
        close(got[2].copy_to_host(), exact, tol, "lse")


# ---- distillation --------------------------------------------------------------------------

def distill_inputs(rng, rows, vocab, k, teacher, repeated=False):
    """Teacher entries: whole rows, short ones, empty ones, values of -inf, repeated indices."""
    indices = np.empty((rows, k), np.int64)
    for r in range(rows):
        indices[r] = rng.permutation(vocab)[:k] if k <= vocab and not repeated else rng.integers(0, max(vocab, 1), k)
    a, values = encode(rng.standard_normal((rows, k)) * 2 + 5, teacher)
    a, values = a.copy(), values.copy()
    if k > 2:
        indices[0, k // 2] = -1
        if rows > 1:
            indices[1, 0] = vocab + 5
        if rows > 2:
            indices[2] = -1
        if rows > 3:
            a[3, 0], values[3, 0] = encode(np.array(-np.inf), teacher)[0], -np.inf
    lse = np.array([np.log(np.exp(values[r][np.isfinite(values[r])] - 5).sum() + 0.5) + 5 for r in range(rows)])
    return a, values, indices, lse.astype(np.float32)


def check_distill(api, rows, vocab, name, k, temperature=1.0, teacher="float32", full=False, index="int32",
                  kind="normal", pad=0, repeated=False, in_place=False, what="both", seed=0):
    rng = np.random.default_rng(seed + rows * 1000003 + vocab * 31 + k)
    a, x = rows_like(rng, rows, vocab, name, kind)
    raw, values, indices, teacher_lse = distill_inputs(rng, rows, vocab, k, teacher, repeated)
    t = float(np.float32(temperature))
    if full:
        with np.errstate(divide="ignore"):
            live = np.where((indices >= 0) & (indices < vocab), values, -np.inf) / t
            peak = live.max(1, initial=-1e30)
            teacher_lse = (peak + np.log(np.exp(live - peak[:, None]).sum(1) + 0.25)).astype(np.float32)
            teacher_lse[~np.isfinite(teacher_lse)] = 0
    grad_loss = (rng.random(rows) + 0.5).astype(np.float32)
    if rows > 4:
        grad_loss[4] = 0
    send = lambda v: api.to_device(np.ascontiguousarray(v))                     # noqa: E731
    d = padded(api, a, pad, before=min(pad, 3))
    kw = dict(temperature=temperature, teacher_lse=send(teacher_lse) if full else None)
    dv, di, dg = padded(api, raw, 2 if pad else 0), send(indices.astype(index)), send(grad_loss)
    op = api.logits
    loss = lse = grad = None
    if what == "both":
        loss, lse, grad = op.distill_loss_and_grad(dg, d, dv, di, out=d if in_place else None, **kw)
    else:
        loss, lse = op.distill_loss(d, dv, di, **kw)
        if what == "apart":
            grad = op.distill_grad(dg, d, dv, di, lse, out=d if in_place else None, **kw)
    given = lse.copy_to_host().astype(np.float64) if what == "apart" else None
    want_loss, want_lse, _ = logits64.distill(x, values, indices, t, teacher_lse if full else None)
    want_lse = in_float32(want_lse)
    fine = np.isfinite(want_lse)
    tol_lse = lse_tolerance(x, t, np.where(fine, want_lse, 0))
    close(lse.copy_to_host(), want_lse, tol_lse, "lse")

    # errors of p and of the terms of the loss
    there = (indices >= 0) & (indices < vocab) & (values != -np.inf)
    size = np.where(there, np.abs(values) / t, 0)
    spread = size.max(1, initial=0) * 2 + np.abs(teacher_lse if full else 0)
    rel_p = U * (4 * spread + k / 256 + 40)
    mass = 1.0
    if full:
        mass = np.array([np.exp(values[r][there[r]] / t - teacher_lse[r]).sum() for r in range(rows)])
    with np.errstate(invalid="ignore"):
        named = np.where(there & np.isfinite(x[np.arange(rows)[:, None], np.clip(indices, 0, vocab - 1)]),
                         np.abs(x[np.arange(rows)[:, None], np.clip(indices, 0, vocab - 1)]) / t, 0)
    log_size = spread + named.max(1, initial=0) * 2 + np.where(fine, np.abs(want_lse), 0)
    with np.errstate(over="ignore"):
        tol_loss = mass * (rel_p * (log_size + 1) + tol_lse + 8 * U * log_size) + 2.0 ** -149
    close(loss.copy_to_host(), want_loss, np.where(np.isfinite(tol_loss), tol_loss, 0), "loss")
    if grad is None:
        return
    _, _, want = logits64.distill(x, values, indices, t, teacher_lse if full else None, grad_loss, given)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        norm = np.where(fine, want_lse if given is None else given, 0)[:, None]
        log_q = np.where(np.isfinite(x), x, 0) / t - norm
        q = np.where(x == -np.inf, 0, np.exp(np.minimum(log_q, 0.1)))
        rel_q = (U * (4 * np.abs(np.maximum(log_q, -200)) + 16) + (tol_lse if given is None else 0 * tol_lse)[:, None]
                 + rel_p[:, None] + 4 * U * np.abs(norm))
        p = np.zeros_like(want)
        for r in range(rows):
            share = values[r][there[r]] / t
            if len(share):
                share = np.exp(share - (teacher_lse[r] if full else share.max()))
                share = share if full else share / share.sum()
                np.add.at(p[r], indices[r][there[r]], share)
        factor = (np.abs(grad_loss) / t)[:, None]
        tol = factor * (np.reshape(mass, (-1, 1)) * q * rel_q + p * (rel_p[:, None] + 8 * U))
        tol = tol + HALF_STEP[name] * np.abs(want) * (1 + 1e-6) + SMALLEST[name] + 2.0 ** -126 * factor
    close(decode(grad.copy_to_host()), want, tol, "gradient")
