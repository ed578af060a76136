"""The block-edge, 8-bit linear and log probability operators as they are used: in
a chain while serving, in a training step through torch's engine, captured into
graphs, on two streams at once, under torch.compile.  Bounds: tests/
test_gpu_norm_add.py, tests/test_gpu_int8_linear.py, tests/test_gpu_log_probs.py."""
import pytest
import torch

import test_gpu_int8_linear as lin
import test_gpu_log_probs as lp
import test_gpu_norm_add as edge
from hp_rms_norm_amd import abi

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16
EPS = 1e-6


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "the gpu tests need a HIP device"
    import hp_rms_norm_amd
    return hp_rms_norm_amd


def int8_weight(outer, inner, g):
    w = torch.randint(-127, 128, (outer, inner), generator=g, device=DEV, dtype=torch.int8)
    return w, (0.5 + torch.rand(outer, generator=g, device=DEV)) * (0.03 / 127)


@pytest.mark.parametrize("rows", [1, 7, 300])
def test_serving_chain(ops, rows):
    """Two blocks of a model in 8 bits: norms around them, products, and the
    answers' log probabilities; each stage against its formula on what the one
    before gave, and the whole in a graph that is replayed with other inputs."""
    hidden, inner, vocab = 512, 1408, 2000
    g = torch.Generator(device=DEV).manual_seed(rows)
    up, up_scale = int8_weight(inner, hidden, g)
    down, down_scale = int8_weight(hidden, inner, g)
    head, head_scale = int8_weight(vocab, hidden, g)
    c = edge.Case(1, rows, hidden, BF, rows, "channel", True, 0.8)
    one = torch.ones(inner, device=DEV, dtype=BF)
    zero = torch.zeros((1, rows, inner), device=DEV, dtype=BF)
    tokens = torch.randint(0, vocab, (1, rows), generator=g, device=DEV)

    def chain():
        got = [ops.norm_add_rms_norm_int8(c.x, c.s, c.p, c.w, EPS, gate=c.gate, residual_scale=0.8)]
        q, scale, res = got[-1]
        got.append(ops.int8_linear(q, scale, up, up_scale))
        got.append(ops.fused_add_rms_norm_int8(got[-1], zero.clone(), one, EPS))
        got.append(ops.int8_linear(*got[-1], down, down_scale))
        got.append(ops.norm_add_rms_norm_int8(got[-1], res, None, c.w, EPS))
        got.append(ops.int8_linear(got[-1][0], got[-1][1], head, head_scale, dtype=torch.float16))
        got.append(ops.token_log_probs(got[-1], tokens, top=5))
        return got

    got = chain()
    q, scale, res = got[0]
    c.check_residual(res)
    out, res2 = c.forward(ops)
    assert torch.equal(res, res2) and torch.equal(q, edge.quantised(out)[0])
    lin.check(got[1][0], q[0], scale[0], up, up_scale, None)
    lin.check(got[3][0], got[2][0][0], got[2][1][0], down, down_scale, None)
    lin.check(got[5][0], got[4][0][0], got[4][1][0], head, head_scale, None)
    lp.check([v[0] for v in got[6]], got[5][0], tokens[0], 5)

    flat = lambda v: [v] if isinstance(v, torch.Tensor) else [t for x in v for t in flat(x)]  # noqa: E731
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain()
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        held = chain()
    for seed in (1, 2, 3, 4):
        c.x.copy_(torch.randn(c.shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV))
        tokens.copy_((tokens + 7 * seed) % vocab)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(flat(held), flat(chain())):
            assert torch.equal(a, b)


class Edge(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ops, seen, x, s, p, w, gate):
        out, res = ops.norm_add_rms_norm(x, s, p, w, EPS, gate=gate, residual_scale=0.9)
        ctx.ops, ctx.seen = ops, seen
        ctx.save_for_backward(x, res, p, w, gate)
        return out, res

    @staticmethod
    def backward(ctx, dout, dres):
        x, res, p, w, gate = ctx.saved_tensors
        got = ctx.ops.norm_add_rms_norm_backward(dout, x, res, p, w, EPS, gate=gate, residual_scale=0.9,
                                                 dresidual=dres)
        ctx.seen.append((got, res, dout, dres))
        return (None, None) + tuple(got)


class LogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ops, seen, z, t):
        log_prob, entropy, lse, _, _ = ops.token_log_probs(z, t)
        ctx.ops, ctx.seen = ops, seen
        ctx.save_for_backward(z, t, lse, entropy)
        return log_prob, entropy

    @staticmethod
    def backward(ctx, dlog_prob, dentropy):
        z, t, lse, entropy = ctx.saved_tensors
        d = ctx.ops.token_log_probs_backward(dlog_prob, z, t, lse, entropy=entropy, dentropy=dentropy)
        ctx.seen.append((d, z, t, dlog_prob, dentropy))
        return None, None, d, None


@pytest.mark.parametrize("gate", ["channel", "sequence", "element"])
def test_training_step_through_the_engine(ops, gate):
    """Two block edges and a policy-gradient loss with an entropy bonus, with
    gradients as the engine hands them on (expanded, summed); each operator's
    gradient against its formula for what it was given."""
    c = edge.Case(3, 10, 256, BF, 31, gate, True, 0.9)
    g = torch.Generator(device=DEV).manual_seed(32)
    head = torch.randn((256, 700), generator=g, device=DEV).to(BF) * 0.1
    t = torch.randint(0, 700, (3, 10), generator=g, device=DEV)
    t[1, 4] = -100
    adv = torch.randn((3, 10), generator=g, device=DEV)
    leaves = [v.detach().clone().requires_grad_() for v in (c.x, c.s, c.p, c.w, c.gate)]
    x, s, p, w, gt = leaves
    edges, losses = [], []
    out, res = Edge.apply(ops, edges, x, s, p, w, gt)
    out2, res2 = Edge.apply(ops, edges, torch.tanh(out), res, p, w, gt)
    log_prob, entropy = LogProbs.apply(ops, losses, (out2.float() @ head.float()).to(BF), t)
    loss = -(adv * log_prob).mean() - 0.01 * entropy.sum() + 1e-3 * res2.float().square().mean()
    loss.backward()
    assert all(v.grad is not None and bool(torch.isfinite(v.grad).all()) for v in leaves)
    d, z, tt, dlog_prob, dentropy = losses[0]
    lp.check_backward(d.reshape(30, 700), z.reshape(30, 700), tt.reshape(30), dlog_prob.reshape(30).contiguous(),
                      dentropy.expand(3, 10).reshape(30).contiguous())
    for i, (got, r, dout, dres) in enumerate(edges):  # the second edge's comes first
        at = edge.Case(3, 10, 256, BF, 31, gate, True, 0.9)
        if i == 0:
            at.x = torch.tanh(out.detach())
        edge.check_backward(at, got, r, dout.contiguous(), dres.contiguous())
    # the leaves' gradients are the two edges' sums, added by the engine in 16 bits
    total = edges[0][0][2].double() + edges[1][0][2].double()
    assert bool(((p.grad.double() - total).abs() <= 2.0 ** -8 * total.abs()).all())


@pytest.mark.parametrize("gate,post", [("sequence", True), ("element", True), ("channel", False), ("none", True)])
def test_captured_gradients(ops, gate, post):
    c = edge.Case(4, 30, 1000, BF, 7, gate, post, 0.7)
    z, t = lp.make(50, 3001, torch.float16, 8, 0.0, 0.1)
    gh = torch.linspace(-1, 1, 50, device=DEV)
    dout, dres = c.rows_of(4, 30), c.rows_of(4, 30)

    def step():
        out, res = c.forward(ops)
        got = list(ops.norm_add_rms_norm_backward(dout, c.x, res, c.p, c.w, EPS, gate=c.gate, residual_scale=0.7,
                                                  dresidual=dres))
        log_prob, entropy, lse, _, _ = ops.token_log_probs(z, t)
        d = ops.token_log_probs_backward(log_prob, z, t, lse, entropy=entropy, dentropy=gh)
        return [out, res, log_prob, entropy, d] + [v for v in got if v is not None]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (1, 2, 3, 4):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        c.x.copy_(torch.randn(c.shape, generator=gen, device=DEV))
        dout.copy_(torch.randn(c.shape, generator=gen, device=DEV))
        z.copy_(torch.randn(z.shape, generator=gen, device=DEV) * 3)
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(held, step())):
            assert torch.equal(a, b), i


def test_two_streams_at_once(ops):
    """Calls of every operator on two streams at the same time: each has its own
    workspace, and gets what it gets alone."""
    cases = [edge.Case(2, 400, 4096, BF, 40 + i, "sequence") for i in range(2)]
    logits = [lp.make(64, 70001, BF, 50 + i) for i in range(2)]
    int8 = [lin.make(40, 16384, 2048, 60 + i) for i in range(2)]

    def call(i):
        c, (z, t), (x, sx, w, sw, _) = cases[i], logits[i], int8[i]
        out, res = c.forward(ops)
        got = ops.norm_add_rms_norm_backward(out, c.x, res, c.p, c.w, EPS, gate=c.gate)
        lps = ops.token_log_probs(z, t, top=9)
        return [out, res, *got, *lps, ops.int8_linear(x, sx, w, sw),
                ops.token_log_probs_backward(lps[0], z, t, lps[2], entropy=lps[1], dentropy=lps[0])]

    want = [call(0), call(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(3):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(call(i))
    torch.cuda.synchronize()
    for i in (0, 1):
        for again in got[i]:
            for a, b in zip(again, want[i]):
                assert torch.equal(a, b)


def test_misplaced_outputs(ops):
    c = edge.Case(1, 20, 256, BF, 9, "element")
    x, s, gate = (v.contiguous() for v in (c.x, c.s, c.gate))
    new = lambda: torch.empty_like(x)  # noqa: E731
    store = torch.zeros(20 * 256 + 256, device=DEV, dtype=BF)
    shifted = store[256:].view(1, 20, 256)
    for out, res, a in ((s, new(), x), (new(), x, x), (gate, new(), x), (new(), gate, x),
                        (store[:-256].view(1, 20, 256), new(), shifted)):
        with pytest.raises(RuntimeError):
            ops.norm_add_rms_norm_out(out, res, a, s, c.p, c.w, EPS, gate=gate)
    same = new()
    with pytest.raises(RuntimeError):
        ops.norm_add_rms_norm_out(same, same, x, s, c.p, c.w, EPS)
    dw, dp, dg = torch.empty_like(c.w), torch.empty_like(c.w), new()
    for di, dr, w1, w2, g1 in ((same, same, dw, dp, dg), (new(), new(), dw, dw, dg), (new(), new(), c.w, dp, dg),
                               (new(), new(), x[0, 0], dp, dg), (new(), new(), dw, dp, x), (gate, new(), dw, dp, dg)):
        with pytest.raises(RuntimeError):
            ops.norm_add_rms_norm_backward_out(di, dr, w2, w1, g1, x, x, s, c.p, c.w, EPS, gate)
    z, t = lp.make(6, 64, torch.float32, 1)
    o = [torch.empty(6, device=DEV) for _ in range(3)]
    top, at = torch.empty((6, 2), device=DEV), torch.empty((6, 2), device=DEV, dtype=torch.int64)
    with pytest.raises(RuntimeError):
        ops.token_log_probs_out(o[0], o[0], o[2], top, at, z, t)
    with pytest.raises(RuntimeError):
        ops.token_log_probs_out(z.view(-1)[:6], o[1], o[2], top, at, z, t)
    with pytest.raises(RuntimeError):
        ops.token_log_probs_backward_out(z.view(-1)[:5 * 64].view(5, 64), o[0][:5], z.view(-1)[64:].view(5, 64), t[:5],
                                         o[2][:5])
    xi, sx, w, sw, _ = lin.make(8, 64, 32, 1)
    with pytest.raises(RuntimeError):
        ops.int8_linear_out(w.view(-1).view(BF)[:8 * 32].view(8, 32), xi, sx, w, sw)


@pytest.mark.parametrize("rows", [1, 3, 40])
def test_the_mode_changes_between_a_workspace_and_its_call(ops, rows):
    z, t = lp.make(rows, 90000, torch.float32, rows)
    stream = torch.cuda.current_stream().cuda_stream
    previous = ops.set_batch_invariant(False)
    try:
        for mode in (False, True):
            ops.set_batch_invariant(mode)
            n = abi.token_log_probs_workspace(rows, 90000, 6, abi.DTYPE_FP32)
            ws = torch.empty(n, dtype=torch.uint8, device=DEV)
            ops.set_batch_invariant(not mode)
            o = [torch.empty(rows, device=DEV) for _ in range(3)]
            o += [torch.empty((rows, 6), device=DEV), torch.empty((rows, 6), device=DEV, dtype=torch.int64)]
            abi.token_log_probs(*(v.data_ptr() for v in o), z.data_ptr(), t.data_ptr(), ws.data_ptr(), n, rows, 90000, 6,
                                90000, -100, abi.DTYPE_FP32, stream)
            lp.check(o, z, t, 6)
            for a, b in zip(o, ops.token_log_probs(z, t, top=6)):
                assert torch.equal(a, b)
    finally:
        ops.set_batch_invariant(previous)


def test_torch_compile(ops):
    """aot_eager, fullgraph: traced through the Meta kernels and functionalised."""
    c = edge.Case(2, 12, 128, BF, 3, "sequence", True, 0.8)
    w8, w8s = int8_weight(300, 128, torch.Generator(device=DEV).manual_seed(4))
    t = torch.arange(24, device=DEV).view(2, 12)

    def f(x, s, p, w, gate, w8, w8s, t):
        out, res = ops.norm_add_rms_norm(x, s, p, w, 1e-6, gate=gate, residual_scale=0.8)
        q, scale, res8 = ops.norm_add_rms_norm_int8(x, res, None, w, 1e-6)
        s2 = s.clone()
        q2, scale2 = ops.fused_add_rms_norm_int8(x, s2, w, 1e-6)
        z = ops.int8_linear(q, scale, w8, w8s)
        log_prob, entropy, lse, top, at = ops.token_log_probs(z, t, top=3)
        dz = ops.token_log_probs_backward(log_prob, z, t, lse, entropy=entropy, dentropy=entropy)
        grads = ops.norm_add_rms_norm_backward(out, x, res, p, w, 1e-6, gate=gate, residual_scale=0.8)
        plain = ops.norm_add_rms_norm_backward(out, x, res, None, w, 1e-6)
        into = [torch.empty_like(x), torch.empty_like(x), torch.empty_like(w), torch.empty(128, device=x.device)]
        ops.norm_add_rms_norm_backward_out(into[0], into[1], into[2], into[3], None, out, x, res, p, w, 1e-6)
        return (out, res, q, scale, res8, s2, q2, scale2, z, log_prob, entropy, lse, top, at, dz, *grads, plain[0],
                plain[1], plain[3], *into)

    args = (c.x, c.s, c.p, c.w, c.gate, w8, w8s, t)
    want = f(*args)
    got = torch.compile(f, backend="aot_eager", fullgraph=True)(*args)
    torch.cuda.synchronize()
    for i, (a, b) in enumerate(zip(got, want)):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b), i


def test_opcheck(ops):
    c = edge.Case(2, 3, 64, BF, 3, "sequence")
    o = torch.ops.hp_rms_norm
    e = lambda v: torch.empty_like(v)  # noqa: E731
    q, scale = torch.empty(c.shape, device=DEV, dtype=torch.int8), torch.empty((2, 3, 1), device=DEV)
    x, sx, w, sw, b = lin.make(4, 32, 10, 1)
    z, t = lp.make(4, 50, torch.float32, 1)
    f = [torch.empty(4, device=DEV) for _ in range(3)]
    log_prob, entropy, lse, top, at = ops.token_log_probs(z, t, top=2)
    for op, args in (
            (o.norm_add_rms_norm, (e(c.x), e(c.x), c.x, c.p, c.w, c.s, c.gate, 0.5, 1e-6)),
            (o.norm_add_rms_norm, (e(c.x), e(c.x), c.x, None, c.w, c.s, None, 0.5, 1e-6)),
            (o.norm_add_rms_norm_int8, (q, scale, e(c.x), c.x, c.p, c.w, c.s, c.gate, 0.5, 1e-6)),
            (o.norm_add_rms_norm_backward, (e(c.x), e(c.x), e(c.p), e(c.w), e(c.gate), c.x.clone(), None, c.x, c.s,
                                            c.p, c.w, c.gate, 0.5, 1e-6)),
            (o.norm_add_rms_norm_backward, (e(c.x), e(c.x), None, e(c.w), None, c.x.clone(), c.s.clone(), c.x, c.s,
                                            None, c.w, None, 0.5, 1e-6)),
            (o.int8_linear, (torch.empty((4, 10), device=DEV, dtype=BF), x, sx, w, sw, b.to(BF))),
            (o.token_log_probs, (*f, e(top), e(at), z, t, -100)),
            (o.token_log_probs_backward, (e(z), log_prob, entropy, z, t, lse, entropy, -100)),
            (o.token_log_probs_backward, (e(z), log_prob, None, z, t, lse, None, -100))):
        torch.library.opcheck(op.default, args, test_utils=("test_schema", "test_faketensor", "test_aot_dispatch_static"))
