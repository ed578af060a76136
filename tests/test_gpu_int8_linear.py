"""The product of 8-bit integers on the GPU.  The sums are exact; from there

    |out - exact| <= u |exact| + 3 e (|sum * scale * weight_scale| + |bias|)

with u half a step of the output type (bf16 2^-8, fp16 2^-11) and e = 2^-24: the
sum's rounding to binary32, one product and one fused multiply-add.  binary64
holds the sums exactly (below 2^31), so its product is the oracle's."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
E = 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "the gpu tests need a HIP device"
    import hp_rms_norm_amd
    return hp_rms_norm_amd


def make(rows, inner, outer, seed, in_pad=0, in_offset=0, w_pad=0, w_offset=0):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def ints(n, pad, offset):
        v = torch.randint(-128, 128, (n * (inner + pad) + offset,), generator=g, device=DEV, dtype=torch.int8)
        return v[offset:].view(n, inner + pad)[:, :inner]
    x, w = ints(rows, in_pad, in_offset), ints(outer, w_pad, w_offset)
    scale = 0.01 * (0.5 + torch.rand(rows, generator=g, device=DEV))
    weight_scale = 0.001 * (0.5 + torch.rand(outer, generator=g, device=DEV))
    bias = torch.randn(outer, generator=g, device=DEV)
    return x, scale, w, weight_scale, bias


def check(out, x, scale, w, weight_scale, bias):
    y = x.double() @ w.double().t() * scale.double().view(-1, 1) * weight_scale.double()
    b = torch.zeros_like(weight_scale) if bias is None else bias
    want, size = y + b.double(), y.abs() + b.double().abs()
    u = U[out.dtype]
    off = (out.double() - want).abs()
    assert bool((off <= u * want.abs() + 3 * E * (1 + u) * size + TINY[out.dtype]).all()), off.max()


# both sides of every rule on rows and on outer, and of a tile's end
ROWS = [1, 2, 3, 4, 5, 7, 8, 9, 16, 17, 31, 48, 64, 65, 127, 128, 129, 256, 257, 700]


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_matches_the_formula(ops, rows, dtype):
    for i, (inner, outer) in enumerate(((64, 16), (16, 1), (128, 100), (1024, 4096), (1040, 4100), (2048, 257),
                                        (4096, 512), (4112, 130), (48, 66000), (9216, 33), (16400, 515))):
        x, scale, w, weight_scale, bias = make(rows, inner, outer, rows + i)
        bias = bias.to(dtype) if i % 2 else None
        out = ops.int8_linear(x, scale, w, weight_scale, bias=bias, dtype=dtype)
        assert out.shape == (rows, outer) and out.dtype == dtype
        check(out, x, scale, w, weight_scale, bias)


@pytest.mark.parametrize("rows", [1, 6, 13, 40, 100, 300])
@pytest.mark.parametrize("inner", [1, 2, 15, 17, 31, 100, 1001, 4095])
def test_odd_inner_sizes(ops, rows, inner):
    x, scale, w, weight_scale, bias = make(rows, inner, 77, rows + inner)
    check(ops.int8_linear(x, scale, w, weight_scale), x, scale, w, weight_scale, None)


@pytest.mark.parametrize("rows", [1, 8, 16, 50, 128, 600])
@pytest.mark.parametrize("pads", [(16, 16, 32, 16), (16, 0, 1, 0), (3, 1, 16, 0), (0, 8, 0, 4), (5, 3, 7, 1)])
def test_strided_and_misaligned_rows(ops, rows, pads):
    for inner, outer in ((256, 300), (1000, 70)):
        x, scale, w, weight_scale, bias = make(rows, inner, outer, 3, *pads)
        store = torch.zeros(rows * (outer + 5) + 1, device=DEV, dtype=torch.float16)[1:].view(rows, outer + 5)
        out = store[:, :outer]
        ops.int8_linear_out(out, x, scale, w, weight_scale, bias=bias.half())
        check(out, x, scale, w, weight_scale, bias.half())
        assert not bool(store[:, outer:].any())


@pytest.mark.parametrize("rows", [1, 5, 20, 60, 100, 128, 600])
def test_the_largest_sums(ops, rows):
    """131071 terms of 2^14 are 2^31 - 2^14; of both signs."""
    inner, outer = 131071, 40
    x = torch.full((rows, inner), -128, device=DEV, dtype=torch.int8)
    w = torch.full((outer, inner), -128, device=DEV, dtype=torch.int8)
    w[::2] = 127
    scale, weight_scale = torch.full((rows,), 2.0 ** -14, device=DEV), torch.full((outer,), 0.5, device=DEV)
    out = ops.int8_linear(x, scale, w, weight_scale)
    check(out, x, scale, w, weight_scale, None)
    assert bool((out[:, 1::2] > 0).all()) and bool((out[:, ::2] < 0).all())


def test_rows_do_not_depend_on_the_others(ops):
    x, scale, w, weight_scale, bias = make(700, 512, 333, 9)
    bias = bias.bfloat16()
    whole = ops.int8_linear(x, scale, w, weight_scale, bias=bias)
    for n in (1, 3, 8, 12, 33, 65, 129):
        assert torch.equal(ops.int8_linear(x[:n], scale[:n], w, weight_scale, bias=bias), whole[:n])


def test_leading_dimensions_and_scales_that_are_not_numbers(ops):
    x, scale, w, weight_scale, _ = make(24, 64, 40, 4)
    x3, s3 = x.view(2, 3, 4, 64), scale.view(2, 3, 4, 1).clone()
    out = ops.int8_linear(x3, s3, w, weight_scale.view(40, 1))
    assert out.shape == (2, 3, 4, 40)
    assert torch.equal(out.view(24, 40), ops.int8_linear(x, scale, w, weight_scale))
    s3[0, 1, 2, 0], s3[1, 0, 0, 0] = float("nan"), float("inf")
    bad = ops.int8_linear(x3, s3, w, weight_scale)
    assert bool(torch.isnan(bad[0, 1, 2]).all()) and not bool(torch.isfinite(bad[1, 0, 0]).any())
    keep = torch.ones((2, 3, 4), dtype=torch.bool, device=DEV)
    keep[0, 1, 2] = keep[1, 0, 0] = False
    assert torch.equal(bad[keep], out[keep])
    assert ops.int8_linear(x[:0], scale[:0], w, weight_scale).shape == (0, 40)


def test_a_large_product(ops):
    """More tiles than CUs, in both directions, on the largest tiles."""
    x, scale, w, weight_scale, bias = make(5000, 1024, 9000, 10)
    out = ops.int8_linear(x, scale, w, weight_scale, bias=bias.bfloat16())
    check(out, x, scale, w, weight_scale, bias.bfloat16())


@pytest.mark.parametrize("rows", [2, 3, 4])
def test_a_few_rows_of_odd_sizes_strides_and_the_largest_sums(ops, rows):
    for inner, outer, pads in ((1, 1, (0, 0, 0, 0)), (17, 3, (0, 0, 0, 0)), (1001, 6, (3, 1, 16, 0)),
                               (4096, 5, (16, 16, 32, 16)), (5000, 1027, (0, 8, 0, 4)),
                               (1024, 4, (0, 0, 0, 0)), (8208, 9, (0, 0, 0, 0))):
        x, scale, w, weight_scale, bias = make(rows, inner, outer, rows, *pads)
        out = ops.int8_linear(x, scale, w, weight_scale, bias=bias.half(), dtype=torch.float16)
        check(out, x, scale, w, weight_scale, bias.half())
    x = torch.full((rows, 131071), -128, device=DEV, dtype=torch.int8)
    w = torch.full((7, 131071), -128, device=DEV, dtype=torch.int8)
    scale, weight_scale = torch.full((rows,), 2.0 ** -14, device=DEV), torch.full((7,), 0.5, device=DEV)
    check(ops.int8_linear(x, scale, w, weight_scale), x, scale, w, weight_scale, None)
