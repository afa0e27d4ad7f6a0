"""The operators over rows of logits in float64, straight from their definitions (test oracle)."""

import numpy as np


def bf16_round(x):
    """float32 values of `x` rounded to bfloat16, to nearest even."""
    bits = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32).astype(np.uint64)
    out = ((bits + 0x7fff + ((bits >> 16) & 1)) >> 16 << 16).astype(np.uint32).view(np.float32)
    return np.where(np.isfinite(x), out, np.asarray(x, np.float32))


def adjust(x, tokens=(), offsets=None, prompts=None, repetition=1.0, presence=0.0, frequency=0.0, pairs=None,
           allowed=None):
    """x: rows x vocab; pairs: per row a list of (entry, value); allowed: rows x vocab booleans."""
    y = np.array(x, dtype=np.float64)
    rows, vocab = y.shape
    number = lambda v, r: float(np.float32(v if np.ndim(v) == 0 else v[r]))     # noqa: E731
    with np.errstate(all="ignore"):
        for r in range(rows):
            history = list(tokens[offsets[r]:offsets[r + 1]]) if offsets is not None else []
            prompt = 0 if prompts is None else int(prompts[r])
            counts = {int(t): 0 for t in history if 0 <= t < vocab}
            for t in history[prompt:]:
                if 0 <= t < vocab:
                    counts[int(t)] += 1
            for v, count in counts.items():
                rep = number(repetition, r)
                y[r, v] = y[r, v] / rep if y[r, v] > 0 else y[r, v] * rep
                if count:
                    y[r, v] -= number(frequency, r) * count + number(presence, r)
            if pairs is not None:
                for v, b in dict(pairs[r]).items():
                    if 0 <= v < vocab:
                        y[r, v] += float(np.float32(b))
    if allowed is not None:
        y[~np.broadcast_to(allowed, y.shape)] = -np.inf
    return y


def lse(x, temperature=1.0):
    z = np.asarray(x, np.float64)
    out = np.empty(z.shape[0])
    for r in range(z.shape[0]):
        peak = z[r].max() if z.shape[1] else -np.inf
        if np.isnan(peak) or np.isinf(peak):
            out[r] = peak
        else:
            out[r] = peak / temperature + np.log(np.exp((z[r] - peak) / temperature).sum())
    return out


def top(x, k):
    """Indices of the k largest entries: NaN first, equal ones by index."""
    z = np.asarray(x, np.float64)
    out = np.empty((z.shape[0], k), np.int64)
    for r in range(z.shape[0]):
        line = z[r].tolist()
        order = sorted(range(len(line)), key=lambda v: (0, 0.0, v) if line[v] != line[v] else (1, -line[v], v))
        out[r] = order[:k]
    return out


def distill(x, values, indices, temperature=1.0, teacher_lse=None, grad_loss=None, given_lse=None):
    """(loss, lse, gradient or None) of every row."""
    z = np.asarray(x, np.float64)
    rows, vocab = z.shape
    norm = lse(z, temperature) if given_lse is None else np.asarray(given_lse, np.float64)
    loss, grad = np.zeros(rows), None if grad_loss is None else np.zeros_like(z)
    with np.errstate(all="ignore"):
        for r in range(rows):
            entries = [(int(v), float(t)) for v, t in zip(indices[r], values[r]) if 0 <= v < vocab and t != -np.inf]
            if not entries:
                continue
            t = np.array([e[1] for e in entries]) / temperature
            if teacher_lse is not None:
                log_p = t - float(teacher_lse[r])
            else:
                log_p = t - t.max() - np.log(np.exp(t - t.max()).sum())
            p = np.exp(log_p)
            log_q = np.full(vocab, -np.inf) if norm[r] == -np.inf else z[r] / temperature - norm[r]
            for (v, _), share, log_share in zip(entries, p, log_p):
                if share != 0:
                    loss[r] += share * (log_share - log_q[v])
            if grad is not None and grad_loss[r] != 0:
                grad[r] = p.sum() * np.exp(log_q)
                for (v, _), share in zip(entries, p):
                    grad[r, v] -= share
                grad[r] *= float(grad_loss[r]) / temperature
    return loss, norm, grad
