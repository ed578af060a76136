"""The layouts in which torch's engine hands gradients on, with meta tensors:
expanded from a sum, permuted by a consumer that transposed the output."""
import pytest
import torch

from hp_rms_norm_amd import ops

BF = torch.bfloat16


def t(*shape):
    return torch.empty(shape, dtype=BF, device="meta")


LAYOUTS = {
    "expanded from one element": lambda: t(1, 1, 1).expand(2, 6, 64),
    "expanded rows": lambda: t(1, 1, 64).expand(2, 6, 64),
    "expanded leading dimension": lambda: t(1, 6, 64).expand(2, 6, 64),
    "transposed leading dimensions": lambda: t(6, 2, 64).transpose(0, 1),
    "transposed rows": lambda: t(2, 64, 6).transpose(1, 2),
    "overlapping rows": lambda: torch.as_strided(t(1000), (2, 6, 64), (48, 8, 1)),
    "every other element": lambda: t(2, 6, 128)[..., ::2],
}


@pytest.mark.parametrize("layout", LAYOUTS)
def test_the_gradients_layout(layout):
    x, w, d = t(2, 6, 64), t(64), LAYOUTS[layout]()
    for dout, dres in ((d, None), (x, d), (d, d)):
        dx, dw = ops.rms_norm_backward(dout, x, w, 1e-6, dresidual=dres)
        assert dx.shape == (2, 6, 64) and dx.is_contiguous() and dx.dtype == BF and dw.shape == (64,)


def test_rows_of_a_wider_store_are_read_in_place():
    """Strided rows are no reason for a copy (which meta tensors would show as
    another storage); the gradient's own shape, type and device still count."""
    d = t(2, 6, 80)[..., :64]
    assert ops._rows(d) is d
    assert ops._rows(t(12, 80)[:, 8:72]).stride() == (80, 1)
    x, w = t(2, 6, 64), t(64)
    for bad in (t(1, 6, 64), t(2, 6, 64).to(torch.float16), t(6, 2, 64)):
        with pytest.raises(RuntimeError):
            ops.rms_norm_backward(bad, x, w, 1e-6)
