"""Rows of more entries than a launch of the gradient in the order of memory holds."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from numba_cuda_amd import logits

U = 2.0 ** -24


@pytest.mark.parametrize("name, vocab", [("float32", (1 << 29) + 5), ("bfloat16", (1 << 30) - 3)])
def test_gradient_by_itself(name, vocab):
    torch = pytest.importorskip("torch")
    dtype = getattr(torch, name)
    x = torch.empty(1, vocab, dtype=dtype, device="cuda")
    part = 1 << 27
    for at in range(0, vocab, part):
        n = min(part, vocab - at)
        x[0, at:at + n] = torch.arange(at, at + n, device="cuda").remainder_(1009).to(torch.float32) * 0.01
    named = [0, vocab - 1, vocab // 2, (1 << 29) - 1]
    values = torch.tensor([[3.0, 1.0, 2.0, 2.5]], device="cuda")
    indices = torch.tensor([named], device="cuda")
    out = torch.full((1, vocab), float("nan"), dtype=dtype, device="cuda")
    # few distinct values: the sums are exact in float64
    distinct = (torch.arange(1009, device="cuda").to(torch.float32) * 0.01).to(dtype).double().cpu().numpy()
    counts = np.full(1009, vocab // 1009) + (np.arange(1009) < vocab % 1009)
    lse = float(np.log((counts * np.exp(distinct)).sum()))
    given = torch.tensor([lse], device="cuda")
    lse = float(given[0])
    logits.distill_grad(2.0 ** 20, x, values, indices, given, out=out)
    torch.cuda.synchronize()
    p = np.exp([3.0, 1.0, 2.0, 2.5])
    p /= p.sum()
    want = 2.0 ** 20 * np.exp(distinct - lse)
    # 8 roundings of the exponent's parts, of up to 21, and of the exponential; half a step of the result
    off = 30 * 8 * U + (U if name == "float32" else 2.0 ** -8)
    for at in range(0, vocab, part):
        n = min(part, vocab - at)
        got = out[0, at:at + n]
        place = torch.arange(at, at + n, device="cuda").remainder_(1009)
        expected = torch.from_numpy(want).to("cuda", torch.float32)[place]
        bad = ~((got.float() - expected).abs() <= off * expected)       # NaN too
        at_named = [v for v in named if at <= v < at + n]
        assert int(bad.sum()) == len(at_named), (at, int(bad.sum()))
        for v in at_named:
            exact = want[v % 1009] - 2.0 ** 20 * p[named.index(v)]
            assert abs(float(out[0, v]) - exact) <= off * abs(exact) + 40 * U * 2.0 ** 20
