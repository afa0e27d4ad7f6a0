"""Calls of more workgroups than one launch holds (2^21): the rows on both sides of each cut."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import numba_cuda_amd as cuda
from numba_cuda_amd import logits

MOST = 1 << 21
U = 2.0 ** -24


def _small(vocab, seed):
    rng = np.random.default_rng(seed)
    return rng.integers(-40, 40, (MOST + 5, vocab)).astype(np.float32) / 8


@pytest.mark.parametrize("vocab", [1, 5])
def test_adjust(vocab):
    x = _small(vocab, 1)
    rows = len(x)
    token = (np.arange(rows) * 7 % (vocab + 1)).astype(np.int32)             # one a row, some outside
    prompts = (np.arange(rows) % 3 == 0).astype(np.int64)
    allowed = (np.arange(rows) * 5 % 31).astype(np.uint32) | 1
    pairs = (np.arange(rows) % vocab).astype(np.int32)
    values = (np.arange(rows) % 16).astype(np.float32)
    starts = cuda.to_device(np.arange(rows + 1))
    got = logits.adjust(cuda.to_device(x), tokens=cuda.to_device(token), offsets=starts,
                        prompt_lengths=cuda.to_device(prompts), repetition=2.0, presence=0.5, frequency=0.25,
                        bias_tokens=cuda.to_device(pairs), bias_values=cuda.to_device(values), bias_offsets=starts,
                        mask=cuda.to_device(allowed[:, None])).copy_to_host()
    want = x.copy()
    at = np.flatnonzero(token < vocab)
    here = want[at, token[at]]
    want[at, token[at]] = np.where(here > 0, here / 2, here * 2) - np.where(prompts[at] == 0, np.float32(0.75), np.float32(0))
    want[np.arange(rows), pairs] += values
    want[(allowed[:, None] >> np.arange(vocab, dtype=np.uint32)) & 1 == 0] = -np.inf
    assert np.array_equal(got, want)                                         # all exact in float32


@pytest.mark.parametrize("vocab, k", [(1, 1), (5, 3)])
def test_top(vocab, k):
    x = _small(vocab, 2)
    values, indices, lse = (a.copy_to_host() for a in logits.top(cuda.to_device(x), k, lse=True))
    order = np.argsort(-x, axis=1, kind="stable")[:, :k]
    assert np.array_equal(indices, order) and np.array_equal(values, np.take_along_axis(x, order, 1))
    # a handful of terms: 8 u each for the exponential, the logarithm and the sums, 6 u |lse|
    want = np.log(np.exp(x.astype(np.float64)).sum(1))
    assert (np.abs(lse - want) <= U * (40 + 6 * np.abs(want))).all()


@pytest.mark.parametrize("vocab", [1, 5])
def test_distill(vocab):
    x = _small(vocab, 3)
    rows = len(x)
    rng = np.random.default_rng(4)
    t, i = rng.integers(-8, 8, (rows, 2)).astype(np.float32) / 4, rng.integers(-1, vocab, (rows, 2)).astype(np.int32)
    g = rng.random(rows).astype(np.float32)
    dx, dt, di, dg = (cuda.to_device(a) for a in (x, t, i, g))
    z = x.astype(np.float64)
    log_q = z - np.log(np.exp(z).sum(1, keepdims=True))
    there = i >= 0
    p = np.where(there, np.exp(t.astype(np.float64)), 0)
    p = p / np.where(there.any(1), p.sum(1), 1)[:, None]
    picked = np.take_along_axis(log_q, np.maximum(i, 0), 1)
    with np.errstate(divide="ignore"):
        loss = np.where(there, p * (np.log(p) - picked), 0).sum(1)
    grad = p.sum(1, keepdims=True) * np.exp(log_q)
    for j in range(2):
        np.add.at(grad, (np.arange(rows), np.maximum(i[:, j], 0)), -p[:, j])
    grad *= g[:, None]
    # logarithms of up to 14, a few dozen roundings
    off = U * 60 * 14
    for got in (logits.distill_loss(dx, dt, di), logits.distill_loss_and_grad(dg, dx, dt, di)):
        assert (np.abs(got[0].copy_to_host() - loss) <= off).all()
        assert (np.abs(got[1].copy_to_host() - np.log(np.exp(z).sum(1))) <= off).all()
    assert (np.abs(got[2].copy_to_host() - grad) <= off).all()
    assert (np.abs(logits.distill_grad(dg, dx, dt, di, got[1]).copy_to_host() - grad) <= off).all()


def _windows(torch, rows, vocab):
    """Row r begins r entries into one array: many long, different rows in little memory."""
    line = ((torch.arange(rows + vocab, device="cuda") * 2654435761) % 4093).to(torch.float32) / 1024
    sums = torch.cat([torch.zeros(1, device="cuda", dtype=torch.float64), torch.cumsum(torch.exp(line.double()), 0)])
    lse = torch.log(sums[vocab:vocab + rows] - sums[:rows])
    return line, torch.as_strided(line, (rows, vocab), (1, 1)), lse


def test_a_loss_in_the_order_of_memory():
    """Three workgroups of the statistics a row."""
    torch = pytest.importorskip("torch")
    rows, vocab = MOST // 3 + 100, 4500
    assert logits.distill_workspace(rows, vocab, 2, np.float32) >= rows * 3 * 8
    line, x, lse = _windows(torch, rows, vocab)
    r = torch.arange(rows, device="cuda")
    indices = torch.stack([r % vocab, (r * 31 + 7) % vocab], 1).to(torch.int32)
    values = torch.stack([(r % 5).float() / 4, (r % 7).float() / 4], 1)
    loss, norm = (torch.empty(rows, device="cuda") for _ in range(2))
    logits.distill_loss(x, values, indices, loss=loss, lse=norm)
    torch.cuda.synchronize()
    log_p = torch.log_softmax(values.double(), 1)
    log_q = torch.gather(x, 1, indices.long()).double() - lse[:, None]
    want = (torch.exp(log_p) * (log_p - log_q)).sum(1)
    # 4500 terms: up to 4500 / 256 + 72 additions in a row, logarithms of up to 14
    off = U * (90 + 60 * 14)
    assert float((norm.double() - lse).abs().max()) <= off and float((loss.double() - want).abs().max()) <= off


def test_a_gradient_in_the_order_of_memory():
    torch = pytest.importorskip("torch")
    rows, vocab = 4096, 131100                   # 513 workgroups a row: 4087 rows a launch
    line, x, lse = _windows(torch, rows, vocab)
    r = torch.arange(rows, device="cuda")
    indices = torch.stack([r % vocab, (r * 31 + 7) % vocab, r % vocab], 1)
    values = torch.stack([(r % 5).float() / 4, (r % 7).float() / 4, (r % 3).float()], 1)
    weights = 1.0 + (r % 4).float()
    norm = lse.float()
    out = torch.full((rows, vocab), float("nan"), device="cuda")
    logits.distill_grad(weights, x, values, indices, norm, out=out)
    torch.cuda.synchronize()
    p = torch.softmax(values.double(), 1)
    for row in [*range(0, 3), *range(4080, 4096)]:
        want = torch.exp(x[row].double() - norm[row].double())
        tol = want * U * 8 * 20
        for j in range(3):
            want[indices[row, j]] -= p[row, j]
            tol[indices[row, j]] += p[row, j] * U * 60
        off = (out[row].double() - want * weights[row].double()).abs() - weights[row].double() * tol - want.abs() * U * 8
        assert float(off.max()) <= 0, row
    assert not bool(torch.isnan(out).any())


def test_loss_and_gradient_of_the_longest_rows():
    """Few long rows in parts: 65537 workgroups of the statistics a row, 31 rows a launch."""
    torch = pytest.importorskip("torch")
    rows, vocab = 33, (1 << 27) + 3
    line, x, lse = _windows(torch, rows, vocab)
    r = torch.arange(rows, device="cuda")
    indices = torch.stack([r, vocab - 1 - r], 1)
    values = torch.stack([(r % 5).float() / 4, (r % 7).float() / 4], 1)
    out = torch.full((rows, vocab), float("nan"), device="cuda")
    loss, norm = (torch.empty(rows, device="cuda") for _ in range(2))
    logits.distill_loss_and_grad(2.0 ** 24, x, values, indices, loss=loss, lse=norm, out=out)
    torch.cuda.synchronize()
    log_p = torch.log_softmax(values.double(), 1)
    p = torch.exp(log_p)
    log_q = torch.gather(x, 1, indices).double() - lse[:, None]
    want = (p * (log_p - log_q)).sum(1)
    # a wavefront adds up the 65537 parts: 1024 + 72 additions in a row, logarithms of up to 24
    off = U * (1100 + 60 * 24)
    assert float((norm.double() - lse).abs().max()) <= off and float((loss.double() - want).abs().max()) <= off
    for row in (0, 1, 15, 29, 30, 31, 32):
        for cut in (slice(0, 5000), slice(vocab // 2, vocab // 2 + 5000), slice(vocab - 5000, vocab)):
            place = torch.arange(vocab, device="cuda")[cut]
            want = torch.exp(x[row, cut].double() - lse[row]) * 2.0 ** 24
            tol = want * (off + U * 8 * 24)
            for j in range(2):
                here = place == indices[row, j]
                want[here] -= p[row, j] * 2.0 ** 24
                tol[here] += p[row, j] * U * 60 * 2.0 ** 24
            assert bool(((out[row, cut].double() - want).abs() <= tol + want.abs() * U).all()), (row, cut)
    for row in range(rows):
        assert not bool(torch.isnan(out[row]).any())
