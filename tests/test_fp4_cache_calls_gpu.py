"""A key-value cache in 4 bits on the device: calls that its documentation allows beside the usual ones."""
import pytest
import torch

from tests.fp4_oracle import attend, step
from tests.test_fp4_cache_calls import LAYOUTS
from vllm_b200 import ops
from vllm_b200.ops import cuda_ops

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


@pytest.mark.parametrize("Hkv,G,D,few", [(64, 1, 128, 1100), (40, 1, 64, 1639), (32, 4, 192, 513)])
def test_many_heads_and_a_long_request_in_one_kernel(Hkv, G, D, few):
    """kv heads times query rows of a request beyond 16 bits, in the kernel of single tokens."""
    cu, Hq, BS, scale = cuda_ops(), Hkv * G, 32, D ** -0.5
    q, cache, md = step([40, 90], [3, 70], Hq, Hkv, D, BS, torch.bfloat16, "cuda", seed=D, spread=2.0)
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
    cu._fp4_few(q, cache, md, Hkv, D, BS, md.block_table.shape[1] * BS, scale, None, 0.0, out, lse, None, 1.0, few)
    want, norm, mass, terms, big = attend(q, cache, md, scale)
    # as for other steps: 32-bit sums of D products, a factor and an exponential; weights in fp16; 32-bit sums; the output's rounding
    eps = (D / 8 + 16) * 2.0 ** -23 * terms + 8 * 2.0 ** -24 * 1.5 * terms + 2.0 ** -21
    bound = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2 * eps + 2.0 ** -13) * mass + 90 * 2.0 ** -31 * big + 2.0 ** -25
    assert ((out.double().cpu() - want).abs() <= bound).all() and ((lse.double().cpu() - norm).abs() <= eps + 2.0 ** -20 + 2.0 ** -22 * norm.abs()).all()
