"""Calls of the training operators that their documentation allows, beside
the ordinary ones: the mode that changes between a workspace's query and the
call, and gradients in the layouts that torch's engine hands on.  Bounds:
tests/test_gpu_loss.py, tests/test_gpu_norm_backward.py."""
import pytest
import torch

from hp_rms_norm_amd import abi
from test_gpu_loss import E, check_backward, check_forward, k_of, make
from test_gpu_norm_backward import check as check_norm_backward

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "the gpu tests need a HIP device"
    import hp_rms_norm_amd
    return hp_rms_norm_amd


@pytest.mark.parametrize("rows,hidden,vocab", [(1, 64, 300), (17, 128, 5000), (100, 65, 9000)])
def test_the_mode_changes_between_a_workspace_and_its_call(ops, rows, hidden, vocab):
    h, w, t, dloss = make(rows, hidden, vocab, torch.bfloat16, rows)
    stream = torch.cuda.current_stream().cuda_stream
    previous = ops.set_batch_invariant(False)
    try:
        for mode in (False, True):
            ops.set_batch_invariant(mode)
            n = abi.linear_cross_entropy_workspace(rows, hidden, vocab, w.data_ptr(), hidden)
            m = abi.linear_cross_entropy_backward_workspace(rows, hidden, vocab, w.data_ptr(), hidden)
            ws = torch.empty(max(n, m), dtype=torch.uint8, device=DEV)
            ops.set_batch_invariant(not mode)
            loss, lse = torch.empty(rows, device=DEV), torch.empty(rows, device=DEV)
            abi.linear_cross_entropy(loss.data_ptr(), lse.data_ptr(), h.data_ptr(), w.data_ptr(), t.data_ptr(),
                                     ws.data_ptr(), n, rows, hidden, vocab, hidden, hidden, -100, abi.DTYPE_BF16,
                                     stream)
            dh, dw = torch.empty_like(h), torch.empty_like(w)
            abi.linear_cross_entropy_backward(dh.data_ptr(), dw.data_ptr(), dloss.data_ptr(), h.data_ptr(),
                                              w.data_ptr(), t.data_ptr(), lse.data_ptr(), ws.data_ptr(), m, rows,
                                              hidden, vocab, hidden, hidden, hidden, hidden, -100, abi.DTYPE_BF16,
                                              stream)
            check_forward(loss, lse, h, w, t)
            check_backward(dh, dw, h, w, t, dloss)
            want = ops.linear_cross_entropy(h, w, t)
            assert torch.equal(loss, want[0]) and torch.equal(lse, want[1])
    finally:
        ops.set_batch_invariant(previous)


class AddNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ops, x, r, w):
        n, s = ops.fused_add_rms_norm(x, r, w, 1e-6)
        ctx.ops = ops
        ctx.save_for_backward(s, w)
        return n, s

    @staticmethod
    def backward(ctx, dn, ds):
        s, w = ctx.saved_tensors
        ctx.ops.seen.append((dn, ds))
        d, dw = ctx.ops.rms_norm_backward(dn, s, w, 1e-6, dresidual=ds)
        return None, d, d, dw


class Recorder:
    def __init__(self, ops):
        self.seen = []
        self.fused_add_rms_norm, self.rms_norm_backward = ops.fused_add_rms_norm, ops.rms_norm_backward


@pytest.mark.parametrize("hidden", [64, 96, 1000])
def test_gradients_as_the_engine_hands_them_on(ops, hidden):
    """Expanded gradients (of a sum) and permuted ones (of a consumer that
    transposed the output) of both outputs, against the formula with the same
    gradients written out; and nothing of what the engine holds is changed."""
    g = torch.Generator(device=DEV).manual_seed(hidden)
    x, r = (torch.randn((6, 10, hidden), generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    w = (1 + 0.1 * torch.randn(hidden, generator=g, device=DEV)).to(torch.bfloat16)
    c = torch.randn((10, 6, hidden), generator=g, device=DEV).to(torch.bfloat16)
    for value in (lambda n, s: n.sum() + s.sum(),
                  lambda n, s: (n.transpose(0, 1) * c).sum() + s.sum(),
                  lambda n, s: n[:, :, :1].sum() + (s.permute(2, 1, 0) * c.permute(2, 0, 1)).sum()):
        rec = Recorder(ops)
        leaves = [v.clone().requires_grad_() for v in (x, r, w)]
        n, s = AddNorm.apply(rec, *leaves)
        value(n, s).backward()
        ((dn, ds),) = rec.seen
        flat = [v.detach().contiguous().view(60, hidden) for v in (s, dn, ds)]
        check_norm_backward(leaves[0].grad.view(60, hidden), leaves[2].grad, flat[0], flat[1], flat[2], w)
        assert torch.equal(leaves[0].grad, leaves[1].grad)


def test_more_tiles_than_one_launch_holds(ops):
    """16384 rows of 2^25 + 1 vocabulary entries are 2^23 tiles of 512 lanes and
    more: 2^32 work-items.  A row's sum joins 131073 tiles, 16 lanes apart, each
    addition off by at most 3 e (its exponential and its step), besides what
    test_gpu_loss.py's bound counts."""
    rows, hidden, vocab = 16384, 64, (1 << 25) + 1
    g = torch.Generator(device=DEV).manual_seed(5)
    w = torch.randn((vocab, hidden), generator=g, device=DEV, dtype=torch.bfloat16) * 0.25
    h = torch.randn((rows, hidden), generator=g, device=DEV, dtype=torch.bfloat16)
    t = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    t[-2], t[5] = vocab - 1, -100
    loss, lse = ops.linear_cross_entropy(h, w, t)
    at = torch.tensor([0, 1, 5, 300, 16127, 16128, 16129, rows - 2, rows - 1], device=DEV)
    total, size = (torch.zeros(len(at), device=DEV, dtype=torch.float64) for _ in range(2))
    for part in w.split(1 << 22):
        total += torch.exp(h[at].double() @ part.double().t()).sum(1)
        size = torch.maximum(size, (h[at].double().abs() @ part.double().abs().t()).amax(1))
    want = torch.where(t[at] == -100, 0.0, total.log())
    bound = k_of(hidden) * E * size + 2.0 ** -16 + (131073 / 16 + 128) * 3 * E + E * want.abs()
    assert bool(((lse[at].double() - want).abs() <= bound).all())
    z = (h[at].double() * w[t[at].clamp(min=0)].double()).sum(1)
    want = torch.where(t[at] == -100, 0.0, want - z)
    assert bool(((loss[at].double() - want).abs() <= 2 * bound + E * want.abs()).all())
    assert bool(torch.isfinite(loss).all())


def test_torch_compile_with_the_training_operators(ops):
    """torch.compile (aot_eager: no codegen, fullgraph) traces the operators
    through their Meta kernels and functionalises what they write, the list of
    clip_grad_norm_ too: every output and every tensor written in place is the
    eager call's, bit for bit."""
    h, w, t, _ = make(40, 128, 300, torch.bfloat16, 30, 0.2)
    g = torch.Generator(device=DEV).manual_seed(31)
    r, dr = (torch.randn((40, 128), generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    nw = (1 + 0.1 * torch.randn(128, generator=g, device=DEV)).to(torch.bfloat16)
    bias = torch.randn(77, generator=g, device=DEV)

    def f(h, r, nw, w, t, dr, bias):
        n, s = ops.fused_add_rms_norm(h, r, nw, 1e-6)
        loss, lse = ops.linear_cross_entropy(n, w, t)
        dn, dw = ops.linear_cross_entropy_backward(torch.full((), 0.03125, device=DEV), n, w, t, lse)
        dx, dnw = ops.rms_norm_backward(dn, s, nw, 1e-6, dresidual=dr.expand(40, 128))
        into, dnw32 = torch.empty_like(dn), torch.empty(128, device=DEV)
        ops.rms_norm_backward_out(into, dnw32, dn, s, nw, 1e-6)
        loss2, lse2 = torch.empty_like(loss), torch.empty_like(lse)
        ops.linear_cross_entropy_out(loss2, lse2, n, w, t)
        dn2, dw2 = torch.empty_like(dn), torch.empty_like(dw)
        ops.linear_cross_entropy_backward_out(dn2, dw2, loss * 0.5, n, w, t, lse)
        db = bias * 0.5
        grads = [dw, dnw, db]
        plain = ops.grad_norm(grads)
        wide = [torch.empty(v.shape, device=DEV) for v in grads]
        copied = ops.clip_grad_norm_out(wide, grads, 0.25)
        clipped = ops.clip_grad_norm_(grads, 0.25)
        again = ops.clip_grad_norm_([bias], 0.5)  # an input of the traced function, in place
        return (loss, lse, dx, into, dnw32, loss2, lse2, dn2, dw2, plain, copied, clipped, again, *grads, *wide)

    args = (h, r, nw, w, t, dr[:1])
    b1, b2 = bias.clone(), bias.clone()
    want = f(*args, b1)
    got = torch.compile(f, backend="aot_eager", fullgraph=True)(*args, b2)
    torch.cuda.synchronize()
    assert torch.equal(b1, b2) and not torch.equal(b1, bias)
    for i, (a, b) in enumerate(zip(got, want)):
        assert a.dtype == b.dtype and a.shape == b.shape, i
        assert torch.equal(a, b), f"output {i} differs"


def test_opcheck_of_the_training_operators(ops):
    """torch's own check of schemas (what is written and what is not), Meta
    kernels and functionalisation."""
    h, w, t, dloss = make(12, 64, 100, torch.bfloat16, 32, 0.2)
    loss, lse = ops.linear_cross_entropy(h, w, t)
    nw = torch.ones(64, device=DEV, dtype=torch.bfloat16)
    o = torch.ops.hp_rms_norm
    grads = [torch.randn(5, device=DEV), torch.randn((3, 4), device=DEV).to(torch.float16)]
    norm = torch.empty((), device=DEV)
    for op, args in (
            (o.rms_norm_backward, (torch.empty_like(h), torch.empty_like(nw), h.clone(), h, nw, None, 1e-6)),
            (o.linear_cross_entropy, (loss.clone(), lse.clone(), h, w, t, -100)),
            (o.linear_cross_entropy_backward,
             (torch.empty_like(h), torch.empty_like(w), dloss, h, w, t, lse, -100)),
            (o.grad_norm, (norm, grads)),
            (o.clip_grad_norm_, (norm, [v.clone() for v in grads], 0.5)),
            (o.clip_grad_norm_out, (norm, [torch.empty_like(v) for v in grads], grads, 0.5))):
        torch.library.opcheck(op.default, args, test_utils=("test_schema", "test_faketensor", "test_aot_dispatch_static"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_gradients_of_many_rows_in_many_pieces(ops, dtype):
    """33000 rows: dz goes in pieces of 3840 vocabulary entries, and dhidden's
    shares run over 129 row tiles; an odd width and padded rows."""
    h, w, t, dloss = make(33000, 72, 9001, dtype, 40, 0.1, pad=3, offset=1)
    loss, lse = ops.linear_cross_entropy(h, w, t)
    check_forward(loss, lse, h, w, t)
    dh, dw = ops.linear_cross_entropy_backward(dloss, h, w, t, lse)
    check_backward(dh, dw, h, w, t, dloss)


def test_gradients_of_the_most_rows(ops):
    """2^22 rows, where the offsets into the turned rows come closest to 2^31
    bytes, in two pieces of the vocabulary; dhidden is looked at in some rows,
    dweight whole."""
    rows, hidden, vocab = 1 << 22, 40, 1100
    h, w, t, dloss = make(rows, hidden, vocab, torch.bfloat16, 41, 0.05)
    loss, lse = ops.linear_cross_entropy(h, w, t)
    dh, dw = ops.linear_cross_entropy_backward(dloss, h, w, t, lse)
    want_dw, bound_dw = (torch.zeros((vocab, hidden), device=DEV, dtype=torch.float64) for _ in range(2))
    wd, u = w.double(), 2.0 ** -8
    for at in torch.arange(rows, device=DEV).split(1 << 17):
        check_forward(loss[at], lse[at], h[at], w, t[at])
        kept = t[at] != -100
        hd, g, to = h[at][kept].double(), dloss[at][kept].double()[:, None], t[at][kept]
        z = hd @ wd.t()
        p = torch.softmax(z, 1)
        d = p.clone()
        d[torch.arange(len(d), device=DEV), to] -= 1.0
        d *= g
        dz = k_of(hidden) * E * (hd.abs() @ wd.abs().t()).amax(1, keepdim=True)
        db = u * d.abs() + p * g.abs() * (2 * dz + 2.0 ** -16)
        off = (dh[at][kept].double() - d @ wd).abs()
        assert bool((off <= ((db + k_of(vocab) * E * d.abs()) @ wd.abs() + u * (d @ wd).abs()) * (1 + u)).all())
        assert not bool(dh[at][~kept].any())
        want_dw += d.t() @ hd
        bound_dw += (db + k_of(rows) * E * d.abs()).t() @ hd.abs()
    assert bool(((dw.double() - want_dw).abs() <= (bound_dw + u * want_dw.abs()) * (1 + u)).all())


def test_float16_rows_of_very_different_dloss(ops):
    """One scale serves all rows, the one that takes the largest |dloss| to 2^14:
    an entry of dz is off by half a step of float16 or by 2^-39 of the largest
    |dloss|, whichever is more.  With dloss down to 2^-24 of the largest that
    is the bound, and with one row a call each row has half a step."""
    h, w, t, _ = make(60, 96, 700, torch.float16, 42)
    g = torch.Generator(device=DEV).manual_seed(43)
    dloss = 256.0 * torch.exp2(-torch.randint(0, 25, (60,), generator=g, device=DEV).float())
    dloss[0] = 256.0
    loss, lse = ops.linear_cross_entropy(h, w, t)
    dh, dw = ops.linear_cross_entropy_backward(dloss, h, w, t, lse)
    check_backward(dh, dw, h, w, t, dloss)
    for i in range(0, 60, 7):
        dh1, dw1 = ops.linear_cross_entropy_backward(dloss[i:i + 1], h[i:i + 1], w, t[i:i + 1], lse[i:i + 1])
        check_backward(dh1, dw1, h[i:i + 1], w, t[i:i + 1], dloss[i:i + 1])
