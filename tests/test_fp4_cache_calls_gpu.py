"""A key-value cache in 4 bits on the device: calls that its documentation allows beside the usual ones."""
import pytest
import torch

from tests.test_fp4_cache_calls import LAYOUTS
from vllm_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H", [1, 2])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_keys_and_values_of_any_layout(layout, H):
    T, D, BS = 3, 16, 16
    with torch.device("cuda"):
        k, v = (LAYOUTS[layout](T, H, D) for _ in range(2))
    cache, want = (torch.zeros(ops.fp4_cache_shape(1, H, BS, D), dtype=torch.uint8, device=d) for d in ("cuda", "cpu"))
    slots = torch.tensor([5, 0, 9])
    ops.reshape_and_cache_fp4(k, v, cache, slots.cuda())
    ops.reshape_and_cache_fp4(k.cpu(), v.cpu(), want, slots)
    assert torch.equal(cache.cpu(), want)
