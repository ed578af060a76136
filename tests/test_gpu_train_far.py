"""The training operators on tensors whose offsets pass 32 bits, and at the
widest rows and the largest vocabulary that they take.  Bounds:
tests/test_gpu_loss.py, tests/test_gpu_norm_backward.py, tests/test_gpu_grad_norm.py."""
import pytest
import torch

from test_gpu_grad_norm import check_clipped, check_norm
from test_gpu_loss import E, check_backward, check_forward, k_of, make
from test_gpu_norm_backward import EPS, K, U, check as check_norm_backward, exact

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "the gpu tests need a HIP device"
    import hp_rms_norm_amd
    return hp_rms_norm_amd


@pytest.mark.parametrize("rows,hidden", [(530000, 4096), (540000, 4097), (33600000, 64)])
def test_norm_gradient_of_more_than_2_31_elements(ops, rows, hidden):
    """Rows at both ends in full, all of dweight against sums a block of rows at
    a time."""
    g = torch.Generator(device=DEV).manual_seed(rows)
    x, dout = (torch.randn((rows, hidden), generator=g, device=DEV, dtype=BF) for _ in range(2))
    w = (1 + 0.1 * torch.randn(hidden, generator=g, device=DEV)).to(BF)
    dw = torch.empty(hidden, device=DEV)
    dx = torch.empty_like(x)
    ops.rms_norm_backward_out(dx, dw, dout, x, w, EPS, dresidual=dout)
    want, size = (torch.zeros(hidden, device=DEV, dtype=torch.float64) for _ in range(2))
    for at in range(0, rows, 1 << 27 >> hidden.bit_length()):
        part = slice(at, at + (1 << 27 >> hidden.bit_length()))
        dxe, mag, dwe, wmag = exact(x[part], dout[part], dout[part], w)
        off = (dx[part].double() - dxe).abs()
        assert bool((off <= U[BF] * dxe.abs() + K * E * mag).all())
        want += dwe
        size += wmag
    # a lane adds the rows of its group one by one: at least 256 groups on the device
    steps = rows / 256 + K + 64
    assert bool(((dw.double() - want).abs() <= 2.0 ** -24 * want.abs() + steps * E * size).all())


def test_norm_gradient_of_far_apart_and_of_the_widest_rows(ops):
    g = torch.Generator(device=DEV).manual_seed(1)
    stores = [torch.zeros((2300, 1 << 20), device=DEV, dtype=BF) for _ in range(3)]
    x, dout, dx = (s[:, 7:7 + 520] for s in stores)
    x.copy_(torch.randn((2300, 520), generator=g, device=DEV))
    dout.copy_(torch.randn((2300, 520), generator=g, device=DEV))
    w = (1 + 0.1 * torch.randn(520, generator=g, device=DEV)).to(BF)
    dw = torch.empty_like(w)
    ops.rms_norm_backward_out(dx, dw, dout, x, w, EPS)
    check_norm_backward(dx, dw, x, dout, None, w)
    assert not bool(stores[2][:, :7].any()) and not bool(stores[2][:, 527:].any())
    del stores, x, dout, dx
    x, dout = (torch.randn((3, 1 << 24), generator=g, device=DEV).to(BF) for _ in range(2))
    w = (1 + 0.1 * torch.randn(1 << 24, generator=g, device=DEV)).to(BF)
    dx, dw = ops.rms_norm_backward(dout, x, w, EPS)
    dxe, mag, dwe, wmag = exact(x, dout, None, w)
    # a lane adds 65536 elements of its row
    assert bool(((dx.double() - dxe).abs() <= U[BF] * dxe.abs() + 65600 * E * mag).all())
    assert bool(((dw.double() - dwe).abs() <= U[BF] * dwe.abs() + 65600 * E * wmag).all())


def test_loss_of_far_apart_rows(ops):
    """hidden, dhidden, weight and dweight with 2^20 and 2^21 elements from row to
    row (the weight read in place at that stride), and one element more (packed)."""
    for hs, wst, offset in ((1 << 20, 1 << 21, 8), ((1 << 20) + 1, (1 << 21) + 1, 3)):
        rows, hidden, vocab = 2100, 72, 1100
        h0, w0, t, dloss = make(rows, hidden, vocab, BF, 6, 0.2)
        sh, sdh = (torch.zeros(rows * hs, device=DEV, dtype=BF).view(rows, hs) for _ in range(2))
        sw, sdw = (torch.zeros(vocab * wst, device=DEV, dtype=BF).view(vocab, wst) for _ in range(2))
        h, dh = (s[:, offset:offset + hidden] for s in (sh, sdh))
        w, dw = (s[:, offset:offset + hidden] for s in (sw, sdw))
        h.copy_(h0)
        w.copy_(w0)
        loss, lse = ops.linear_cross_entropy(h, w, t)
        check_forward(loss, lse, h0, w0, t)
        ops.linear_cross_entropy_backward_out(dh, dw, dloss, h, w, t, lse)
        check_backward(dh.contiguous(), dw.contiguous(), h0, w0, t, dloss)
        for s, n in ((sdh, hidden), (sdw, hidden)):  # between the rows nothing is written
            assert not bool(s[:, :offset].any()) and not bool(s[:, offset + n:].any())


@pytest.mark.parametrize("hidden", [1 << 20, (1 << 20) - 1])
def test_loss_of_the_widest_rows(ops, hidden):
    """Bounds of 2^20 terms a logit, so logits that are small for their terms."""
    for rows in (2, 70):
        h, w, t, dloss = make(rows, hidden, 150, BF, 7, spread=0.01)
        loss, lse = ops.linear_cross_entropy(h, w, t)
        check_forward(loss, lse, h, w, t)
        dh, dw = ops.linear_cross_entropy_backward(dloss, h, w, t, lse)
        check_backward(dh, dw, h, w, t, dloss)


def test_loss_of_the_largest_vocabulary(ops):
    """2^28 entries: 2^21 tiles of one launch, 512 pieces of the gradient.  The
    sum of a row joins 2^21 tiles, 256 lanes apart, each step off by at most 3 e."""
    rows, hidden, vocab = 3, 8, 1 << 28
    g = torch.Generator(device=DEV).manual_seed(8)
    w = torch.randn((vocab, hidden), generator=g, device=DEV, dtype=BF) * 0.5
    h = torch.randn((rows, hidden), generator=g, device=DEV).to(BF)
    t = torch.tensor([vocab - 1, -100, 12345], device=DEV)
    dloss = torch.tensor([1.0, 3.0, 0.5], device=DEV)
    loss, lse = ops.linear_cross_entropy(h, w, t)
    dh, dw = ops.linear_cross_entropy_backward(dloss, h, w, t, lse)
    at, hd = torch.tensor([0, 2], device=DEV), h[[0, 2]].double()
    total, size = (torch.zeros(2, device=DEV, dtype=torch.float64) for _ in range(2))
    for part in w.split(1 << 24):
        total += torch.exp(hd @ part.double().t()).sum(1)
        size = torch.maximum(size, (hd.abs() @ part.double().abs().t()).amax(1))
    want = total.log()
    dz = k_of(hidden) * E * size
    off = dz + ((1 << 21) / 256 + 128) * 3 * E + 2.0 ** -16 + E * want.abs()
    assert float(lse[1]) == 0.0 and float(loss[1]) == 0.0 and not bool(dh[1].any())
    assert bool(((lse[at].double() - want).abs() <= off).all())
    z = (hd * w[t[at]].double()).sum(1)
    assert bool(((loss[at].double() - (want - z)).abs() <= off + dz + E * (want - z).abs()).all())
    # p = exp(z - lse) is off by a factor of dz and of the lse's own error
    u, gl = U[BF], dloss[at].double()[:, None]
    want_dh, bound_dh = (torch.zeros((2, hidden), device=DEV, dtype=torch.float64) for _ in range(2))
    for v in range(0, vocab, 1 << 24):
        part = w[v:v + (1 << 24)].double()
        p = torch.exp(hd @ part.t() - want[:, None])
        d = p.clone()
        here = (t[at] >= v) & (t[at] < v + (1 << 24))
        for i in here.nonzero()[:, 0].tolist():
            d[i, t[at][i] - v] -= 1.0
        d *= gl
        db = u * d.abs() + p * gl * (2 * dz + 2 * off)[:, None] + 2.0 ** -126
        want_dh += torch.stack([(row[:, None] * part).sum(0) for row in d])
        bound_dh += torch.stack([(row[:, None] * part.abs()).sum(0) for row in db + k_of(vocab) * E * d.abs()])
        want_dw = d.t() @ hd
        bound = (db + k_of(2) * E * d.abs()).t() @ hd.abs() + u * want_dw.abs()
        assert bool(((dw[v:v + (1 << 24)].double() - want_dw).abs() <= bound * (1 + u)).all())
    assert bool(((dh[at].double() - want_dh).abs() <= (bound_dh + u * want_dh.abs()) * (1 + u)).all())


def test_gradients_of_more_than_2_31_elements(ops):
    g = torch.Generator(device=DEV).manual_seed(9)
    big = torch.randn((1 << 31) + 12345, generator=g, device=DEV, dtype=BF)
    grads = [big, torch.randn(77, generator=g, device=DEV)]
    total = sum(float(part.double().pow(2).sum()) for v in grads for part in v.split(1 << 28)) ** 0.5
    norm = ops.grad_norm(grads)
    assert abs(float(norm) - total) <= (2.0 ** -24 + 2.0 ** -40) * total
    wide = [torch.empty(v.shape, device=DEV) for v in grads]
    ops.clip_grad_norm_out(wide, grads, 0.25 * total)
    factor = 0.25 * total / (total + 1e-6)
    for o, v in zip(wide, grads):
        for a, b in zip(o.split(1 << 28), v.split(1 << 28)):
            x = b.double() * factor
            assert bool(((a.double() - x).abs() <= (2.0 ** -24 + 2.0 ** -22) * x.abs()).all())
    del wide
    ends = [big[:1000].clone(), big[-20000:].clone()]
    ops.clip_grad_norm_(grads, 0.25 * total)
    for part, was in zip((big[:1000], big[-20000:]), ends):
        x = was.double() * factor
        assert bool(((part.double() - x).abs() <= (U[BF] + 2.0 ** -22) * x.abs()).all())
    check_norm(ops.grad_norm(grads[1:]), grads[1:])
    before = [grads[1].clone()]
    ops.clip_grad_norm_(grads[1:], 0.1)
    check_clipped(grads[1:], before, 0.1)
