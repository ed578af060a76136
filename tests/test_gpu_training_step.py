"""One training step around the framework's norms, as a user puts it together:
two fused add + norm layers, the loss of the last one's rows under a
vocabulary projection, the gradients back through all of it, clipping by
their norm; and the same through torch.autograd.Function, and in a graph.

Against binary64 autograd of the formulas: on the way from the inputs to a
gradient at most 8 tensors are rounded to 16 bits (two residuals, two normed
outputs, dz, and three gradients), each by at most u = half a step relative to
its values; the norms' and softmax's Jacobians carry a relative error on with
a factor of at most about 2, so 16 u in the 2-norm bounds the sum.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1e-6
IGNORE = -100
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "the gpu tests need a HIP device"
    import hp_rms_norm_amd
    return hp_rms_norm_amd


def make(rows, hidden, vocab, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x, r = (torch.randn((rows, hidden), generator=g, device=DEV).to(dtype) for _ in range(2))
    w1, w2 = ((1 + 0.1 * torch.randn(hidden, generator=g, device=DEV)).to(dtype) for _ in range(2))
    head = (torch.randn((vocab, hidden), generator=g, device=DEV) * 2 / hidden ** 0.5).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    t[:: 5] = IGNORE
    return x, r, w1, w2, head, t


def step(ops, x, r, w1, w2, head, t, max_norm):
    """(loss, norm, gradients of x (and r), w1, w2, head), the last three clipped."""
    n1, r1 = ops.fused_add_rms_norm(x, r, w1, EPS)
    n2, r2 = ops.fused_add_rms_norm(n1, r1, w2, EPS)
    loss, lse = ops.linear_cross_entropy(n2, head, t, IGNORE)
    kept = (t != IGNORE).sum()
    dn2, dhead = ops.linear_cross_entropy_backward((1.0 / kept).float(), n2, head, t, lse, IGNORE)
    dr2, dw2 = ops.rms_norm_backward(dn2, r2, w2, EPS)          # of n1, and of r1 along the stream
    dx, dw1 = ops.rms_norm_backward(dr2, r1, w1, EPS, dresidual=dr2)
    grads = [dw1, dw2, dhead]
    norm = ops.clip_grad_norm_(grads, max_norm)
    return loss.sum() / kept, norm, dx, grads


def exact(x, r, w1, w2, head, t, max_norm):
    p = [v.double().requires_grad_() for v in (x, r, w1, w2, head)]

    def norm(s, w):
        return s * (s.pow(2).mean(1, keepdim=True) + EPS).rsqrt() * w
    r1 = p[0] + p[1]
    n1 = norm(r1, p[2])
    z = norm(n1 + r1, p[3]) @ p[4].t()
    kept = t != IGNORE
    z, at = z[kept], t[kept]
    loss = (torch.logsumexp(z, 1) - z.gather(1, at[:, None])[:, 0]).mean()
    loss.backward()
    grads = [v.grad for v in p[2:]]
    total = sum(float(v.pow(2).sum()) for v in grads) ** 0.5
    factor = min(1.0, max_norm / (total + 1e-6))
    return loss.detach(), total, p[0].grad, p[1].grad, [v * factor for v in grads]


def near(a, b, tol):
    off, size = (a.double() - b).norm(), b.norm()
    assert off <= tol * size, (float(off), float(size))


@pytest.mark.parametrize("rows,hidden,vocab,dtype", [(64, 256, 1000, torch.bfloat16), (300, 512, 3000, torch.float16),
                                                     (33, 136, 517, torch.bfloat16)])
def test_step_matches_autograd_of_the_formulas(ops, rows, hidden, vocab, dtype):
    args = make(rows, hidden, vocab, dtype, rows)
    loss, norm, dx, grads = step(ops, *args, 0.05)
    want_loss, want_norm, want_dx, want_dr, want = exact(*args, 0.05)
    tol = 16 * U[dtype]
    near(loss, want_loss, tol)
    assert abs(float(norm) - want_norm) <= tol * want_norm
    near(dx, want_dx, tol)
    near(dx, want_dr, tol)  # input and residual share one gradient
    for got, w in zip(grads, want):
        near(got, w, tol)


class AddNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ops, x, r, w):
        n, s = ops.fused_add_rms_norm(x, r, w, EPS)
        ctx.ops = ops
        ctx.save_for_backward(s, w)
        return n, s

    @staticmethod
    def backward(ctx, dn, ds):
        s, w = ctx.saved_tensors
        d, dw = ctx.ops.rms_norm_backward(dn, s, w, EPS, dresidual=ds)
        return None, d, d, dw


class HeadLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ops, h, head, t):
        loss, lse = ops.linear_cross_entropy(h, head, t, IGNORE)
        ctx.ops = ops
        ctx.save_for_backward(h, head, t, lse)
        return loss

    @staticmethod
    def backward(ctx, dloss):
        dh, dhead = ctx.ops.linear_cross_entropy_backward(dloss, *ctx.saved_tensors, IGNORE)
        return None, dh, dhead, None


def test_through_autograd_functions(ops):
    """The gradients of the same step through torch's engine, which hands the
    backward calls expanded (stride 0) and accumulated gradients."""
    x, r, w1, w2, head, t = make(64, 256, 1000, torch.bfloat16, 3)
    leaves = [v.clone().requires_grad_() for v in (x, r, w1, w2, head)]
    n1, r1 = AddNorm.apply(ops, leaves[0], leaves[1], leaves[2])
    n2, _ = AddNorm.apply(ops, n1, r1, leaves[3])
    (HeadLoss.apply(ops, n2, leaves[4], t).sum() / (t != IGNORE).sum()).backward()
    norm = ops.clip_grad_norm_([v.grad for v in leaves[2:]], 0.05)
    _, want_norm, dx, grads = step(ops, x, r, w1, w2, head, t, 0.05)
    assert torch.equal(leaves[0].grad, dx) and torch.equal(leaves[1].grad, dx)
    assert torch.equal(norm, want_norm)
    for v, want in zip(leaves[2:], grads):
        assert torch.equal(v.grad, want)


def test_step_in_a_graph(ops):
    """Captured whole and replayed on changing rows and targets, between eager
    steps, with a second graph of the same operators alive."""
    args = make(130, 256, 1500, torch.bfloat16, 5)
    other = make(20, 256, 700, torch.bfloat16, 6)
    step(ops, *args, 0.05), step(ops, *other, 0.05)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for a in (args, other):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            with torch.cuda.graph(graph, stream=side):
                outs.append(step(ops, *a, 0.05))
        torch.cuda.current_stream().wait_stream(side)
        graphs.append(graph)
    for i in range(4):
        for a in (args, other):
            a[0].mul_(-1.0 if i % 2 else 1.0)
            a[5].copy_(a[5].roll(i))
        want = [step(ops, *a, 0.05) for a in (args, other)]
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for got, w in zip(outs, want):
            assert all(torch.equal(p, q) for p, q in zip(got[:3], w[:3]))
            assert all(torch.equal(p, q) for p, q in zip(got[3], w[3]))
