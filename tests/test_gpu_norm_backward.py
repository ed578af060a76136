"""The gradient of RMSNorm on the GPU against its formula in binary64.

Bounds, element by element, with u half a step of the output type (bf16 2^-8,
fp16 2^-11 relative to the value, fp32 2^-24) and e = 2^-24: a row's two sums
run over at most 32 elements a lane and at most 12 joining steps, each step off
by at most e of the sum of magnitudes, and the few products and the square root
and division by a few e more, so with K = 64

    |dinput - exact|  <= u |exact| + K e (|r g| + |s| r^3 mean|g s| + |dresidual|)
    |dweight - exact| <= u |exact| + (K + rows / 32 + 64) e sum|dout s r|

(a column's terms are added over at most rows / workgroups in a lane, then
over the workgroups, 32 apart), plus half the smallest subnormal in float16.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}
E, K, EPS = 2.0 ** -24, 64, 1e-6


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "the gpu tests need a HIP device"
    import hp_rms_norm_amd
    return hp_rms_norm_amd


def make(rows, hidden, dtype, seed, residual=True, pad=0, offset=0):
    """Row tensors as views of wider rows that start `offset` elements in."""
    g = torch.Generator(device=DEV).manual_seed(seed)

    def rows_of():
        store = torch.randn(rows * (hidden + pad) + offset, generator=g, device=DEV).to(dtype)
        return store[offset:].view(rows, hidden + pad)[:, :hidden]
    x, dout = rows_of(), rows_of()
    dres = rows_of() if residual else None
    w = (1 + 0.1 * torch.randn(hidden + offset, generator=g, device=DEV)).to(dtype)[offset:]
    return x, dout, dres, w


def exact(x, dout, dres, w, eps=EPS):
    """(dinput, its bound's magnitude, dweight, its bound's magnitude) in binary64."""
    s, d, g = x.double(), dout.double(), dout.double() * w.double()
    r = (s.pow(2).mean(1, keepdim=True) + eps).rsqrt()
    dx = r * g - s * r ** 3 * (g * s).mean(1, keepdim=True)
    mag = (r * g).abs() + s.abs() * r ** 3 * (g * s).abs().mean(1, keepdim=True)
    if dres is not None:
        dx, mag = dx + dres.double(), mag + dres.double().abs()
    terms = d * s * r
    return dx, mag, terms.sum(0), terms.abs().sum(0)


def check(got_dx, got_dw, x, dout, dres, w, eps=EPS):
    dx, mag, dw, wmag = exact(x, dout, dres, w, eps)
    off = (got_dx.double() - dx).abs()
    assert bool((off <= U[got_dx.dtype] * dx.abs() + K * E * mag + TINY[got_dx.dtype]).all()), off.max()
    off = (got_dw.double() - dw).abs()
    k = K + x.shape[0] / 32 + 64
    assert bool((off <= U[got_dw.dtype] * dw.abs() + k * E * wmag + TINY[got_dw.dtype]).all()), off.max()


# every lane mapping's last and first width, widths off the 8-element grid and
# both sides of the register-resident kernels' range
WIDTHS = [1, 7, 8, 9, 64, 128, 129, 250, 256, 257, 512, 520, 1000, 1024, 1025, 2048, 2056, 4096, 4097, 4104, 5120, 6144,
          6145, 8192, 8200, 12001, 16384, 16392, 32768, 32769]


@pytest.mark.parametrize("hidden", WIDTHS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_matches_the_formula(ops, hidden, dtype):
    for rows, residual in ((1, True), (37, False), (300, True)):
        x, dout, dres, w = make(rows, hidden, dtype, hidden + rows, residual)
        dx, dw = ops.rms_norm_backward(dout, x, w, EPS, dresidual=dres)
        assert dx.dtype == dtype and dw.dtype == dtype
        check(dx, dw, x, dout, dres, w)


@pytest.mark.parametrize("rows,hidden", [(5000, 128), (20000, 64), (2500, 4096), (1500, 8192)])
def test_more_rows_than_workgroups(ops, rows, hidden):
    x, dout, dres, w = make(rows, hidden, torch.bfloat16, 5)
    dx, dw = ops.rms_norm_backward(dout, x, w, EPS, dresidual=dres)
    check(dx, dw, x, dout, dres, w)


@pytest.mark.parametrize("hidden,pad,offset", [(4096, 8, 0), (4096, 7, 1), (1001, 24, 3), (128, 128, 0), (20, 1, 5)])
def test_strided_and_misaligned_rows(ops, hidden, pad, offset):
    for dtype in (torch.bfloat16, torch.float16):
        x, dout, dres, w = make(70, hidden, dtype, 11, True, pad, offset)
        dx = torch.zeros(70 * (hidden + 3) + 1, device=DEV, dtype=dtype)[1:].view(70, hidden + 3)[:, :hidden]
        dw = torch.empty(hidden, device=DEV, dtype=torch.float32)
        ops.rms_norm_backward_out(dx, dw, dout, x, w, EPS, dresidual=dres)
        check(dx, dw, x, dout, dres, w)
        # the elements between the rows are left as they were
        store = torch.as_strided(dx, (70, hidden + 3), (hidden + 3, 1))
        assert not bool(store[:-1, hidden:].any())


def test_another_stream_and_misplaced_outputs(ops):
    x, dout, dres, w = make(300, 2048, torch.bfloat16, 4)
    want = ops.rms_norm_backward(dout, x, w, EPS, dresidual=dres)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.rms_norm_backward(dout, x, w, EPS, dresidual=dres)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    store = torch.zeros(300 * 2048 + 1, device=DEV, dtype=torch.bfloat16)
    for dx, dw in ((store[1:].view(300, 2048), store[:2048]), (x, x[0]), (dout, w)):
        with pytest.raises(RuntimeError):
            ops.rms_norm_backward_out(dx, dw, dout, x, w, EPS)
    shifted = torch.as_strided(dout, (299, 2048), (2048, 1), 2048)   # dout's rows, one further
    with pytest.raises(RuntimeError):
        ops.rms_norm_backward_out(shifted, torch.empty_like(w), dout[:299], x[:299], w, EPS)


def test_past_the_cached_size(ops):
    """More than 2^24 elements take the non-temporal loads: the same bits row by row."""
    x, dout, dres, w = make(4200, 4096, torch.bfloat16, 6)
    dx, dw = ops.rms_norm_backward(dout, x, w, EPS, dresidual=dres)
    check(dx, dw, x, dout, dres, w)
    part, _ = ops.rms_norm_backward(dout[4000:], x[4000:], w, EPS, dresidual=dres[4000:])
    assert torch.equal(part, dx[4000:])


@pytest.mark.parametrize("hidden", [9, 128, 4096, 4097, 40000])
def test_in_place_on_each_row_tensor(ops, hidden):
    x, dout, dres, w = make(50, hidden, torch.bfloat16, 3)
    want_dx, want_dw = ops.rms_norm_backward(dout, x, w, EPS, dresidual=dres)
    for which in range(3):
        t = [x.clone(), dout.clone(), dres.clone()]
        dw = torch.empty_like(want_dw)
        ops.rms_norm_backward_out(t[which], dw, t[1], t[0], w, EPS, dresidual=t[2])
        assert torch.equal(t[which], want_dx) and torch.equal(dw, want_dw)


def test_leading_dimensions_and_no_rows(ops):
    x, dout, dres, w = make(24, 256, torch.bfloat16, 9)
    want = ops.rms_norm_backward(dout, x, w, EPS)
    got = ops.rms_norm_backward(dout.reshape(2, 3, 4, 256), x.reshape(2, 3, 4, 256), w, EPS)
    assert torch.equal(got[0].reshape(24, 256), want[0]) and torch.equal(got[1], want[1])
    dx, dw = ops.rms_norm_backward(dout[:0], x[:0], w, EPS)
    assert dx.shape == (0, 256) and not bool(dw.any())


def test_rows_of_zeros_and_special_values(ops):
    x, dout, dres, w = make(6, 512, torch.bfloat16, 21)
    x[1] = 0
    dout[2] = 0
    dx, dw = ops.rms_norm_backward(dout, x, w, EPS, dresidual=dres)
    check(dx, dw, x, dout, dres, w)
    assert torch.equal(dx[2], dres[2])
    x[3, 5] = float("nan")
    dx, dw = ops.rms_norm_backward(dout, x, w, EPS, dresidual=dres)
    bad = torch.isnan(dx).all(1)
    assert bad.tolist() == [False, False, False, True, False, False]
    assert bool(torch.isnan(dw).all())


def test_agrees_with_differences_of_the_formula(ops):
    """A directional difference of the normalised rows' weighted sum in
    binary64 against the gradients: central differences of step h are off by
    O(h^2); the 16-bit gradients by u of the terms' magnitudes."""
    x, dout, _, w = make(4, 96, torch.bfloat16, 31, residual=False)
    dx, dw = ops.rms_norm_backward(dout, x, w, EPS)
    g = torch.Generator(device=DEV).manual_seed(1)
    vx = torch.randn(x.shape, generator=g, device=DEV, dtype=torch.float64)
    vw = torch.randn(w.shape, generator=g, device=DEV, dtype=torch.float64)

    def value(t):
        s, ww = x.double() + t * vx, w.double() + t * vw
        return (dout.double() * ww * s * (s.pow(2).mean(1, keepdim=True) + EPS).rsqrt()).sum()
    h = 1e-4
    slope = (value(h) - value(-h)) / (2 * h)
    parts = (dx.double() * vx).sum() + (dw.double() * vw).sum()
    bound = 2.0 ** -8 * ((dx.double() * vx).abs().sum() + (dw.double() * vw).abs().sum())
    assert abs(slope - parts) <= bound + 1e-5 * abs(slope)


@pytest.mark.parametrize("rows,hidden", [(300, 4096), (40000, 128), (6, 40000)])
def test_bits_repeat_and_a_graph_replays_them(ops, rows, hidden):
    x, dout, dres, w = make(rows, hidden, torch.bfloat16, 13)
    want = ops.rms_norm_backward(dout, x, w, EPS, dresidual=dres)
    dx, dw = torch.empty_like(want[0]), torch.empty_like(want[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            ops.rms_norm_backward_out(dx, dw, dout, x, w, EPS, dresidual=dres)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        dx.zero_(), dw.zero_()
        dout.mul_(1.0 if i < 2 else -1.0)
        want = ops.rms_norm_backward(dout, x, w, EPS, dresidual=dres)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dx, want[0]) and torch.equal(dw, want[1])
