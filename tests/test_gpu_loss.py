"""Softmax cross entropy under a vocabulary projection and its gradient, on
the GPU, against the formulas in binary64.

Bounds, with e = 2^-24, u half a step of the 16-bit type (bf16 2^-8, fp16
2^-11) and A = |hidden| |weight|^T. A product over n terms is summed 32 terms
at a time, each step off by at most a few e of the magnitudes so far:
K(n) = 2 (n / 32 + 32).

  z     K(hidden) e A =: dz
  lse   max over the row of dz, and 2^-16 for at most 2000 sequential additions of
        exponentials (3 e each for the exponential and the sum's step)
  loss  the two together
  gradient entries, exactly d = (p - onehot) g: rounding to 16 bits u |d|; p's
        own error p (2 dz + 2^-16); with the largest |g| scaled to 2^14,
        in float16 half the smallest subnormal, 2^-25 2^-14 max|g|; and 2^-126 |g|
        where p lies below binary32's normal numbers (its exponential may be 0:
        at a logit 88 under the row's lse p is 2^-127, and exact p goes down to
        2^-430 in the most peaked case)
  dhidden  sum over v of those times |weight|, K(vocab) e |d| |weight|, and u of itself
  dweight  the same with |hidden| and K(rows)
"""
import pytest
import torch

from hp_rms_norm_amd import abi

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
E = 2.0 ** -24
IGNORE = -100


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "the gpu tests need a HIP device"
    import hp_rms_norm_amd
    return hp_rms_norm_amd


def k_of(n):
    return 2 * (n / 32 + 32)


def matrix(rows, cols, dtype, g, pad=0, offset=0, scale=1.0):
    store = (torch.randn(rows * (cols + pad) + offset, generator=g, device=DEV) * scale).to(dtype)
    return store[offset:].view(rows, cols + pad)[:, :cols]


def make(rows, hidden, vocab, dtype, seed, ignored=0.0, pad=0, offset=0, spread=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    h = matrix(rows, hidden, dtype, g, pad, offset)
    w = matrix(vocab, hidden, dtype, g, pad, offset, spread / hidden ** 0.5)
    t = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    t = torch.where(torch.rand(rows, generator=g, device=DEV) < ignored, IGNORE, t)
    dloss = torch.rand(rows, generator=g, device=DEV) + 0.1
    return h, w, t, dloss


def exact(h, w, t, ignore=IGNORE):
    """Of the rows that count: (which, logits, lse, their bound)."""
    kept = t != ignore
    hd, wd = h[kept].double(), w.double()
    z = hd @ wd.t()
    dz = k_of(h.shape[1]) * E * (hd.abs() @ wd.abs().t())
    return kept, z, torch.logsumexp(z, 1), dz


def check_forward(loss, lse, h, w, t, ignore=IGNORE):
    kept, z, want, dz = exact(h, w, t, ignore)
    assert not bool(loss[~kept].any()) and not bool(lse[~kept].any())
    lse_bound = (dz.amax(1) if z.numel() else want) + 2.0 ** -16 + E * want.abs()
    assert bool(((lse[kept].double() - want).abs() <= lse_bound).all())
    at = t[kept][:, None]
    want_loss = want - z.gather(1, at)[:, 0]
    bound = lse_bound + dz.gather(1, at)[:, 0] + E * want_loss.abs()
    assert bool(((loss[kept].double() - want_loss).abs() <= bound).all())


def check_backward(dh, dw, h, w, t, dloss, ignore=IGNORE):
    u, tiny = U[h.dtype], TINY[h.dtype]
    kept, z, lse, dz = exact(h, w, t, ignore)
    assert not bool(dh[~kept].any())
    g = dloss[kept].double()[:, None]
    p = torch.exp(z - lse[:, None])
    d = p.clone()
    d[torch.arange(len(d), device=DEV), t[kept]] -= 1.0
    d *= g
    floor = max(tiny * 2.0 ** -14, 2.0 ** -126) * float(g.abs().max()) if g.numel() else 0.0
    db = u * d.abs() + p * g.abs() * (2 * dz.amax(1, keepdim=True) + 2.0 ** -16) + floor
    hd, wd = h[kept].double(), w.double()
    want = d @ wd
    bound = (db + k_of(w.shape[0]) * E * d.abs()) @ wd.abs() + u * want.abs() + tiny
    assert bool(((dh[kept].double() - want).abs() <= bound * (1 + u)).all())
    want = d.t() @ hd
    bound = (db + k_of(len(d)) * E * d.abs()).t() @ hd.abs() + u * want.abs() + tiny
    assert bool(((dw.double() - want).abs() <= bound * (1 + u)).all())


def run(ops, h, w, t, dloss, ignore=IGNORE):
    loss, lse = ops.linear_cross_entropy(h, w, t, ignore_index=ignore)
    check_forward(loss, lse, h, w, t, ignore)
    dh, dw = ops.linear_cross_entropy_backward(dloss, h, w, t, lse, ignore_index=ignore)
    check_backward(dh, dw, h, w, t, dloss, ignore)
    return loss, lse, dh, dw


SIZES = [(1, 64, 1), (1, 1, 2), (1, 128, 1000), (2, 8, 127), (3, 9, 129), (17, 33, 128), (16, 64, 256), (33, 96, 513),
         (64, 128, 300), (65, 200, 1023), (127, 512, 640), (128, 136, 1500), (129, 64, 2049), (200, 1000, 777),
         (256, 256, 1024), (257, 320, 1281), (300, 72, 5000), (511, 1024, 512), (700, 264, 3333)]


@pytest.mark.parametrize("rows,hidden,vocab", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_matches_the_formulas(ops, rows, hidden, vocab, dtype):
    run(ops, *make(rows, hidden, vocab, dtype, rows + hidden + vocab))


@pytest.mark.parametrize("rows,hidden,vocab", [(40, 64, 300), (300, 128, 700), (1200, 256, 900)])
@pytest.mark.parametrize("ignored", [0.1, 0.5, 0.97])
def test_ignored_rows(ops, rows, hidden, vocab, ignored):
    """Whatever the ignored rows and their dloss hold: they are not read."""
    h, w, t, dloss = make(rows, hidden, vocab, torch.bfloat16, rows, ignored)
    t[0], t[1], t[-1] = IGNORE, 3, IGNORE
    want = run(ops, h, w, t, dloss)
    h[t == IGNORE] = float("nan")
    h[0] = float("inf")
    dloss[t == IGNORE] = float("nan")
    got = run(ops, h, w, t, dloss)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_all_rows_ignored_and_no_rows(ops):
    h, w, t, dloss = make(100, 64, 300, torch.bfloat16, 1)
    t.fill_(IGNORE)
    _, _, dh, dw = run(ops, h, w, t, dloss)
    assert not bool(dh.any()) and not bool(dw.any())
    loss, lse = ops.linear_cross_entropy(h[:0], w, t[:0])
    assert loss.shape == (0,) and lse.shape == (0,)
    dh, dw = ops.linear_cross_entropy_backward(dloss[:0], h[:0], w, t[:0], lse)
    assert dh.shape == (0, 64) and not bool(dw.any())


@pytest.mark.parametrize("hidden", [64, 65])
def test_no_rows_need_no_tensors_but_dweight(ops, hidden):
    dw = torch.ones((300, hidden), dtype=torch.bfloat16, device="cuda")
    size = abi.linear_cross_entropy_backward_workspace(0, hidden, 300)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    abi.linear_cross_entropy_backward(0, dw.data_ptr(), 0, 0, 0, 0, 0, ws.data_ptr(), size, 0, hidden, 300, hidden,
                                      hidden, hidden, hidden, IGNORE, abi.DTYPE_BF16,
                                      torch.cuda.current_stream().cuda_stream)
    assert not bool(dw.any())


def test_other_ignore_index_and_targets_out_of_range(ops):
    h, w, t, dloss = make(50, 64, 300, torch.bfloat16, 2)
    t[5] = t[7] = 17
    run(ops, h, w, t, dloss, ignore=17)
    t[9], t[11] = 300, -5
    loss, lse = ops.linear_cross_entropy(h, w, t, ignore_index=17)
    assert torch.isnan(loss).nonzero()[:, 0].tolist() == [9, 11] and bool(torch.isfinite(lse).all())
    dh, dw = ops.linear_cross_entropy_backward(dloss, h, w, t, lse, ignore_index=17)
    assert torch.isnan(dh).all(1).nonzero()[:, 0].tolist() == [9, 11] and bool(torch.isnan(dw).all())


@pytest.mark.parametrize("hidden,pad,offset", [(128, 8, 0), (128, 0, 8), (128, 3, 1), (100, 4, 4), (65, 0, 0), (64, 64, 0)])
def test_strided_and_misaligned_rows(ops, hidden, pad, offset):
    for rows, dtype in ((70, torch.bfloat16), (400, torch.float16)):
        h, w, t, dloss = make(rows, hidden, 600, dtype, 7, 0.2, pad, offset)
        loss, lse = ops.linear_cross_entropy(h, w, t)
        check_forward(loss, lse, h, w, t)
        stores = [torch.zeros(n * (hidden + 5) + 1, device=DEV, dtype=dtype) for n in (rows, 600)]
        dh, dw = (s[1:].view(-1, hidden + 5)[:, :hidden] for s in stores)
        ops.linear_cross_entropy_backward_out(dh, dw, dloss, h, w, t, lse)
        check_backward(dh, dw, h, w, t, dloss)
        for s in stores:  # between the rows nothing is written
            assert not bool(s[0]) and not bool(s[1:].view(-1, hidden + 5)[:, hidden:].any())


def test_leading_dimensions(ops):
    h, w, t, dloss = make(60, 64, 500, torch.bfloat16, 8, 0.3)
    loss, lse, dh, dw = run(ops, h, w, t, dloss)
    h3, t3, d3 = h.view(3, 20, 64), t.view(3, 20), dloss.view(3, 20)
    loss3, lse3 = ops.linear_cross_entropy(h3, w, t3)
    dh3, dw3 = ops.linear_cross_entropy_backward(d3, h3, w, t3, lse3)
    assert torch.equal(loss3.view(-1), loss) and torch.equal(dh3.view(60, 64), dh) and torch.equal(dw3, dw)


@pytest.mark.parametrize("spread", [0.01, 30.0, 300.0])
def test_flat_and_peaked_distributions(ops, spread):
    for dtype in (torch.bfloat16, torch.float16):
        run(ops, *make(150, 128, 2000, dtype, 4, spread=spread))


def test_not_finite_logits(ops):
    h, w, t, dloss = make(20, 64, 300, torch.bfloat16, 5)
    h[3, 1] = float("nan")
    loss, lse = ops.linear_cross_entropy(h, w, t)
    assert torch.isnan(loss).nonzero()[:, 0].tolist() == [3]
    dh, dw = ops.linear_cross_entropy_backward(dloss, h, w, t, lse)
    assert torch.isnan(dh).all(1).nonzero()[:, 0].tolist() == [3] and bool(torch.isnan(dw).all())
    # logits of -inf leave the others' loss as it is without them
    h, w, t, dloss = make(20, 64, 300, torch.bfloat16, 6)
    h[:, 0] = 1.0
    w[130:290, 0] = float("-inf")
    t %= 130
    loss, lse = ops.linear_cross_entropy(h, w, t)
    rest = torch.cat([w[:130], w[290:]])
    check_forward(loss, lse, h, rest, t)


def test_many_pieces_of_the_vocabulary(ops):
    """More than 2^27 entries of dz: several pieces, the last one short."""
    run(ops, *make(2100, 64, 130001, torch.bfloat16, 9, 0.02))


def test_more_rows_than_one_forward_launch(ops):
    h, w, t, _ = make(33000, 16, 200, torch.bfloat16, 10, 0.3)
    loss, lse = ops.linear_cross_entropy(h, w, t)
    check_forward(loss, lse, h, w, t)


@pytest.mark.parametrize("scale", [1e-30, 3e-6, 4096.0])
def test_scale_of_the_incoming_gradient(ops, scale):
    """bfloat16 gradients are proportional to dloss, exactly for powers of two."""
    h, w, t, dloss = make(90, 128, 700, torch.bfloat16, 11)
    _, lse = ops.linear_cross_entropy(h, w, t)
    dloss = dloss * scale
    dh, dw = ops.linear_cross_entropy_backward(dloss, h, w, t, lse)
    check_backward(dh, dw, h, w, t, dloss)
    dh2, dw2 = ops.linear_cross_entropy_backward(dloss * 0.25, h, w, t, lse)
    assert torch.equal(dh2, dh * 0.25) and torch.equal(dw2, dw * 0.25)
    dh0, dw0 = ops.linear_cross_entropy_backward(torch.zeros_like(dloss), h, w, t, lse)
    assert not bool(dh0.any()) and not bool(dw0.any())


def test_scalar_dloss_expands(ops):
    h, w, t, _ = make(30, 64, 200, torch.bfloat16, 12)
    _, lse = ops.linear_cross_entropy(h, w, t)
    one = ops.linear_cross_entropy_backward(torch.tensor(0.5, device=DEV), h, w, t, lse)
    all_ = ops.linear_cross_entropy_backward(torch.full((30,), 0.5, device=DEV), h, w, t, lse)
    assert all(torch.equal(a, b) for a, b in zip(one, all_))


def test_agrees_with_differences_of_the_loss(ops):
    """The gradients along a direction against central differences of the
    mean loss in binary64; the bound sums the entries' half steps (twice: dz's
    rounding and the outputs')."""
    h, w, t, _ = make(12, 32, 60, torch.bfloat16, 13)
    _, lse = ops.linear_cross_entropy(h, w, t)
    dh, dw = ops.linear_cross_entropy_backward(torch.tensor(1 / 12, device=DEV), h, w, t, lse)
    g = torch.Generator(device=DEV).manual_seed(2)
    vh = torch.randn(h.shape, generator=g, device=DEV, dtype=torch.float64)
    vw = torch.randn(w.shape, generator=g, device=DEV, dtype=torch.float64)

    def value(s):
        z = (h.double() + s * vh) @ (w.double() + s * vw).t()
        return (torch.logsumexp(z, 1) - z.gather(1, t[:, None])[:, 0]).mean()
    step = 1e-5
    slope = (value(step) - value(-step)) / (2 * step)
    parts = (dh.double() * vh).sum() + (dw.double() * vw).sum()
    bound = 2 * 2.0 ** -8 * ((dh.double() * vh).abs().sum() + (dw.double() * vw).abs().sum())
    assert abs(slope - parts) <= bound + 1e-6


@pytest.mark.parametrize("rows", [1, 40, 700])
def test_bits_repeat_and_a_graph_replays_them(ops, rows):
    h, w, t, dloss = make(rows, 256, 3000, torch.bfloat16, 14)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            loss, lse = ops.linear_cross_entropy(h, w, t)
            dh, dw = ops.linear_cross_entropy_backward(dloss, h, w, t, lse)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        # other targets, and other rows without a loss, at each replay
        t.copy_((t + 7 * i).remainder(3000))
        if rows > 1:
            t[i] = IGNORE
        want = ops.linear_cross_entropy(h, w, t)
        want += ops.linear_cross_entropy_backward(dloss, h, w, t, want[1])
        for o in (loss, lse, dh, dw):
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((loss, lse, dh, dw), want))


def test_two_streams_at_once(ops):
    a, b = make(300, 128, 3000, torch.bfloat16, 15), make(300, 128, 3000, torch.bfloat16, 16)
    want = [run(ops, *a), run(ops, *b)]
    torch.cuda.synchronize()
    got = []
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for s, (h, w, t, dloss) in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                loss, lse = ops.linear_cross_entropy(h, w, t)
                got.append((loss, lse) + ops.linear_cross_entropy_backward(dloss, h, w, t, lse))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(x, y) for x, y in zip(g, want[i % 2]))


def test_batch_invariant_mode_fixes_a_rows_bits(ops):
    """With the mode on, a row's loss and lse are the same bits in calls of any
    row count, at any place among the rows."""
    h, w, t, _ = make(700, 192, 5000, torch.bfloat16, 17)
    previous = ops.set_batch_invariant(True)
    try:
        loss, lse = ops.linear_cross_entropy(h, w, t)
        check_forward(loss, lse, h, w, t)
        for rows in (1, 5, 16, 17, 64, 65, 128, 129, 300):
            for at in (0, 700 - rows):
                a, b = ops.linear_cross_entropy(h[at:at + rows], w, t[at:at + rows])
                assert torch.equal(a, loss[at:at + rows]) and torch.equal(b, lse[at:at + rows])
        keep = torch.arange(700, device=DEV) % 3 == 0
        a, b = ops.linear_cross_entropy(h, w, torch.where(keep, t, IGNORE))
        assert torch.equal(a[keep], loss[keep]) and torch.equal(b[keep], lse[keep])
    finally:
        ops.set_batch_invariant(previous)


SHAPES = [(12, 300, 700), (40, 512, 3000), (100, 264, 9000), (100, 128, 70000), (200, 128, 70000), (300, 384, 2000),
          (900, 128, 70000), (1500, 64, 200), (2000, 200, 1100), (700, 520, 300)]


@pytest.mark.parametrize("rows,hidden,vocab", SHAPES)
def test_every_tile_shape(ops, rows, hidden, vocab):
    """Row counts and vocabularies on both sides of the tile rules, and counts
    of listed rows below the call's rows (fewer row tiles, more splits)."""
    for ignored in (0.0, 0.6):
        run(ops, *make(rows, hidden, vocab, torch.bfloat16, rows + vocab, ignored))


FEW = [(1, 2600, 1000), (16, 6400, 4096), (7, 1537, 333), (3, 64, 4096), (9, 72, 4097), (5, 264, 5000),
       (16, 1600, 30001), (16, 128, 70000), (17, 1600, 500), (40, 128, 70000)]


@pytest.mark.parametrize("rows,hidden,vocab", FEW)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_few_rows(ops, rows, hidden, vocab, dtype):
    """Up to 64 rows: the tiles whose waves share the sum (whole turns, ends
    inside a turn, fewer slices than waves) and their neighbours."""
    for ignored in (0.0, 0.6):
        run(ops, *make(rows, hidden, vocab, dtype, rows + hidden, ignored))


def test_weight_rows_in_a_wider_store_with_other_values_around(ops):
    """What lies between and around the weight's rows is not part of it: NaN
    there changes nothing (in place and packed)."""
    for hidden, pad in ((96, 8), (104, 24), (64, 64), (100, 5)):
        h, w, t, dloss = make(80, hidden, 513, torch.bfloat16, 18)
        want = run(ops, h, w, t, dloss)
        store = torch.full((515, hidden + pad), float("nan"), device=DEV, dtype=torch.bfloat16)
        view = store[1:514, :hidden]
        view.copy_(w)
        loss, lse = ops.linear_cross_entropy(h, view, t)
        dh, dw = ops.linear_cross_entropy_backward(dloss, h, view, t, lse)
        assert torch.equal(loss, want[0]) and torch.equal(lse, want[1])
        assert torch.equal(dh, want[2]) and torch.equal(dw, want[3])
