"""The block-edge, 8-bit linear and log probability operators on tensors whose
offsets pass 32 bits.  Bounds as in the operators' own tests."""
import pytest
import torch

import test_gpu_int8_linear as lin
import test_gpu_log_probs as lp
import test_gpu_norm_add as edge

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16
EPS = 1e-6


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "the gpu tests need a HIP device"
    import hp_rms_norm_amd
    return hp_rms_norm_amd


class Part:
    """Some rows of a long case, as tests/test_gpu_norm_add.py checks them."""

    def __init__(self, c, at):
        self.dtype, self.scale, self.hidden, self.p, self.w = c.dtype, c.scale, c.hidden, c.p, c.w
        self.x, self.s = c.x[:, at], c.s[:, at]
        self.shape = tuple(self.x.shape)
        self.gate = None if c.gate is None else c.gate[:, at] if c.gate.dim() == 3 and c.gate.shape[1] > 1 else c.gate
    check_residual, check_out = edge.Case.check_residual, edge.Case.check_out


@pytest.mark.parametrize("rows,hidden,gate", [(530000, 4096, "element"), (540000, 4097, "none"),
                                              (33600000, 64, "channel"), (130000, 16600, "none")])
def test_edges_of_more_than_2_31_elements(ops, rows, hidden, gate):
    c = edge.Case(1, 8, hidden, BF, 1, gate, True, 0.75)
    g = torch.Generator(device=DEV).manual_seed(rows)
    c.shape = (1, rows, hidden)
    c.x, c.s = (torch.randn(c.shape, generator=g, device=DEV, dtype=BF) for _ in range(2))
    if gate == "element":
        c.gate = torch.rand(c.shape, generator=g, device=DEV, dtype=BF)
    out, res = c.forward(ops)
    ends = [slice(0, 50), slice(rows // 2, rows // 2 + 50), slice(rows - 50, rows)]
    for at in ends:
        part = Part(c, at)
        part.check_residual(res[:, at])
        part.check_out(out[:, at], res[:, at])
    q, scale, _ = ops.norm_add_rms_norm_int8(c.x, c.s, c.p, c.w, EPS, gate=c.gate, residual_scale=0.75)
    for at in ends:
        want = edge.quantised(out[:, at])
        assert torch.equal(q[:, at], want[0]) and torch.equal(scale[:, at], want[1])
    del q, scale
    di, dr, dp, dw, dg = ops.norm_add_rms_norm_backward(out, c.x, res, c.p, c.w, EPS, gate=c.gate,
                                                        residual_scale=0.75, dresidual=c.s)
    # a part's rows alone give the same rows; the columns' sums, a block of rows at a time
    sums = [torch.zeros(hidden, device=DEV, dtype=torch.float64) for _ in range(4)]
    for at in range(0, rows, 1 << 27 >> hidden.bit_length()):
        rows_at = slice(at, at + (1 << 27 >> hidden.bit_length()))
        h, d = res[:, rows_at].double(), out[:, rows_at].double()
        r = (h.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
        t = d * h * r
        sums[0] += t.sum((0, 1))
        sums[1] += t.abs().sum((0, 1))
    steps = rows / 256 + 4 * edge.k_of(hidden) + 128
    off = (dw.double() - sums[0]).abs()
    assert bool((off <= 2.0 ** -8 * sums[0].abs() + steps * edge.E * sums[1]).all())
    for at in ends:
        part = Part(c, at)
        got = ops.norm_add_rms_norm_backward(out[:, at], part.x, res[:, at], c.p, c.w, EPS, gate=part.gate,
                                             residual_scale=0.75, dresidual=part.s)
        edge.check_backward(part, got, res[:, at], out[:, at], part.s)
        assert torch.equal(got[0], di[:, at]) and torch.equal(got[1], dr[:, at])
        if gate == "element":
            assert torch.equal(got[4], dg[:, at])


@pytest.mark.parametrize("rows,inner,outer", [(600000, 4096, 64), (3, 4096, 600000), (1, 8192, 300000),
                                              (70000, 64, 40000), (600000, 4001, 40)])
def test_products_of_more_than_2_31_elements(ops, rows, inner, outer):
    x, scale, w, weight_scale, bias = lin.make(rows, inner, outer, 3)
    out = ops.int8_linear(x, scale, w, weight_scale, bias=bias.to(BF))
    rs = sorted({0, 1, rows // 2, rows - 2, rows - 1} & set(range(rows)))
    os_ = sorted({0, 5, outer // 2, outer - 2, outer - 1} & set(range(outer)))
    for at in (rs, list(range(rows))[-300:]):
        at = torch.tensor(at, device=DEV)
        cols = torch.tensor(os_ if outer > 1000 else list(range(outer)), device=DEV)
        lin.check(out[at][:, cols], x[at], scale[at], w[cols], weight_scale[cols], bias.to(BF)[cols])


@pytest.mark.parametrize("rows,vocab,dtype,pad", [(40000, 131072, BF, 0), (70000, 50001, BF, 3),
                                                  (2200, 1 << 20, torch.float32, 0), (300, 1000, BF, 16000000)])
def test_logits_of_more_than_2_31_elements(ops, rows, vocab, dtype, pad):
    store = torch.empty(rows * (vocab + pad), device=DEV, dtype=dtype).view(rows, vocab + pad)
    z = store[:, :vocab]
    g = torch.Generator(device=DEV).manual_seed(vocab)
    for at in range(0, rows, 1000):
        z[at:at + 1000] = torch.randn(z[at:at + 1000].shape, generator=g, device=DEV, dtype=dtype) * 3
    t = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    t[7] = -100
    got = ops.token_log_probs(z, t, top=4)
    adv = torch.randn(rows, generator=g, device=DEV)
    d = ops.token_log_probs_backward(adv, z, t, got[2], entropy=got[1], dentropy=adv)
    at = torch.tensor([0, 1, 7, rows // 2, rows - 2, rows - 1], device=DEV)
    lp.check([v[at] for v in got], z[at], t[at], 4)
    lp.check_backward(d[at], z[at], t[at], adv[at], adv[at])
    assert bool(torch.isfinite(got[0]).all())


@pytest.mark.parametrize("groups,length,hidden,gate,lanes", [
    (1, 530000, 4096, "element", 512), (1, 540000, 4097, "none", 256), (1, 33600000, 64, "channel", 16384),
    (2, 525000, 2048, "sequence", 1024), (1, 130000, 16600, "none", 64)])
def test_column_sums_of_more_than_2_31_elements(ops, groups, length, hidden, gate, lanes):
    """The weights' gradients and a shared gate's over all rows.  The gradients
    that reach the edge follow its own tensors, so a column's terms have one
    sign nearly throughout (for each gate) and none may be missing.  `lanes` lanes share the
    rows of a column on 256 CUs: each adds rows / lanes terms, and 16 + 32
    partial sums of up to 32 row groups are joined."""
    c = edge.Case(groups, 8, hidden, BF, 1, gate, True, 0.75)
    rows = groups * length
    g = torch.Generator(device=DEV).manual_seed(rows)
    c.shape = (groups, length, hidden)
    c.x, c.s = (torch.randn(c.shape, generator=g, device=DEV, dtype=BF) for _ in range(2))
    if gate == "element":
        c.gate = torch.rand(c.shape, generator=g, device=DEV, dtype=BF)
    out, res = c.forward(ops)
    di, dr = torch.empty_like(c.x), torch.empty_like(c.x)
    dw, dp = torch.empty(hidden, device=DEV), torch.empty(hidden, device=DEV)
    dg = None if c.gate is None else torch.empty_like(c.gate)
    ops.norm_add_rms_norm_backward_out(di, dr, dp, dw, dg, out, c.x, res, c.p, c.w, EPS, c.gate, 0.75, c.x)
    del di, dr
    sums = torch.zeros((6, groups, hidden), device=DEV, dtype=torch.float64)
    block = 1 << 27 >> hidden.bit_length()
    for at in range(0, length, max(1, block // groups)):
        part = slice(at, at + max(1, block // groups))
        x, h, d = c.x[:, part].double(), res[:, part].double(), out[:, part].double()
        r = (h.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
        w = d * c.w.double()
        dh = r * w - h * r ** 3 * (w * h).mean(-1, keepdim=True) + x
        size = (r * w).abs() + h.abs() * r ** 3 * (w * h).abs().mean(-1, keepdim=True) + x.abs()
        t = d * h * r
        nx = x * (x.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
        by = 1.0 if c.gate is None else (c.gate[:, part] if gate == "element" else c.gate).double()
        n = nx * c.p.double()
        for i, v in enumerate((t, t.abs(), by * dh * nx, (by * size * nx).abs(), dh * n, (size * n).abs())):
            sums[i] += v.sum(1)
    steps = rows / lanes + 16 + 32 + 32 + 4 * edge.k_of(hidden)
    checks = [(dw, sums[0].sum(0), sums[1].sum(0)), (dp, sums[2].sum(0), sums[3].sum(0))]
    if gate == "channel":
        checks.append((dg, sums[4].sum(0), sums[5].sum(0)))
    elif gate == "sequence":
        checks.append((dg[:, 0], sums[4], sums[5]))
    for got, want, size in checks:
        u = edge.U[got.dtype]
        assert float((want.abs() / size).median()) > 0.1  # (or the bound would say little)
        off = (got.double() - want).abs()
        assert bool((off <= u * want.abs() + steps * edge.E * (1 + u) * size).all()), (off / size).max()
