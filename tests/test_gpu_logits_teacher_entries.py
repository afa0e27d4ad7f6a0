"""Loss and gradient of many rows at the numbers of teacher's entries and lengths where the lanes per row change."""

import pytest

pytestmark = pytest.mark.gpu

import numba_cuda_amd as cuda
from tests import logits_cases as cases


@pytest.mark.parametrize("name, vocab", [("float32", 16385), ("bfloat16", 33000), ("float16", 81920), ("float16", 81921)])
@pytest.mark.parametrize("rows, k", [(513, 300), (513, 301), (512, 301), (257, 513)])
def test_both(name, vocab, rows, k):
    cases.check_distill(cuda, rows, vocab, name, k, what="both", pad=3 if k % 2 else 0, in_place=k == 301, repeated=k == 513)
