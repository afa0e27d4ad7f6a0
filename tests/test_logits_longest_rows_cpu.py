"""How calls on the longest rows are spread, asked through the workspaces they need."""

import pytest

from numba_cuda_amd import _lib
from numba_cuda_amd.kernels import logits

GRAD = 2


@pytest.mark.parametrize("code, each", [(0, 256), (1, 512), (2, 512)])          # entries per workgroup
def test_a_gradient_of_the_longest_rows_needs_no_workspace(code, each):
    """Rows of more workgroups than a launch holds cannot take the launches in the order of memory."""
    need = _lib.load().nbh_rows_distill_workspace
    most = (1 << 21) * each                      # entries of a launch's workgroups
    # a row may begin up to seven entries behind a multiple of sixteen bytes
    for vocab in (most - 7, most // 2, most // 2 + 1):
        assert need(1, vocab, 8, code, GRAD) > 0
    for vocab in (most - 6, most, most + 1, 2 ** 31 - 1):
        assert need(1, vocab, 8, code, GRAD) == 0
    assert need(3, 2 ** 31 - 1, logits.MOST, code, GRAD) == 0
