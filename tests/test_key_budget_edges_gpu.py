"""A key-value cache with a budget on the device: values, shapes and calls at the edge of what the operators take."""
import pytest
import torch

from tests.key_budget_oracle import step
from tests.test_key_budget_gpu import _check_weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,BS,vt", [(128, 64, True), (64, 16, False)])
def test_weights_capped_rows_that_differ(D, BS, vt):
    """Capped scores, log-sum-exps that change from tile to tile: each tile has its own, in every run the same bits."""
    q, cache, md, scores = step([2300], [2300], 8, 2, D, BS, torch.bfloat16, "cuda", vt=vt, seed=5)
    lse = 4 + 6 * torch.rand(2300, 8, generator=torch.Generator().manual_seed(2)).cuda()
    want = None
    for _ in range(10):
        got = scores.clone()
        _check_weights(q, cache, md, got, cap=30.0, lse=lse)
        assert want is None or torch.equal(got, want)
        want = got
