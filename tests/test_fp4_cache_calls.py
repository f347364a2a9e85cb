"""A key-value cache in 4 bits: calls that its documentation allows, as far as they show without a device."""
import pytest
import torch

from vllm_b200.ops import cuda


def _rnd(*shape):
    return torch.randn(shape, dtype=torch.bfloat16)


LAYOUTS = {
    "interleaved": lambda T, H, D: _rnd(T, H, D, 2)[..., 0],  # keys and values of a channel side by side
    "every other column": lambda T, H, D: _rnd(T, 2 * D)[:, ::2][:, None].expand(T, H, D),
    "one column": lambda T, H, D: _rnd(T, 8)[:, :1, None].expand(T, H, D),
    "heads first": lambda T, H, D: _rnd(H, T, D).transpose(0, 1),
    "columns first": lambda T, H, D: _rnd(H, D, T).permute(2, 0, 1),
    "a token for all": lambda T, H, D: _rnd(1, H, D).expand(T, H, D),
    "part of a projection": lambda T, H, D: _rnd(T, (H + 2) * D)[:, D:-D].unflatten(1, (H, D)),
}


@pytest.mark.parametrize("H", [1, 2])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_rows_lie_as_the_kernel_reads_them(layout, H):
    """Row t, at t times the row stride, has the H D values of a token next to each other, inside the memory that it belongs to."""
    T, D = 3, 16
    x = LAYOUTS[layout](T, H, D)
    rows = cuda._fp4_rows(x)
    step = rows.stride(0)
    assert rows.data_ptr() % 16 == 0 and step % 8 == 0
    assert rows.storage_offset() + (T - 1) * step + H * D <= rows.untyped_storage().nbytes() // 2
    assert torch.equal(rows.as_strided((T, H * D), (step, 1)), x.reshape(T, H * D))
