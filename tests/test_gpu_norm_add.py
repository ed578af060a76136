"""The edge between two blocks (norm, gate, scaled residual, norm) and its
gradient on the GPU, against their formulas in binary64.

Bounds, element by element, with u half a step of the output type (bf16 2^-8,
fp16 2^-11 relative to the value, fp32 2^-24) and e = 2^-24.  A row's sums run
over at most 32 elements a lane and 12 joining steps (16 more for the rows that
take passes, per 4096 elements), each step off by at most e of the sum of
magnitudes, and the products, square roots and divisions by a few e more; K = 64
covers one norm and what hangs on it, 2 K the gradient's second one.

    |residual_out - exact| <= u |exact| + K e (|scale * residual| + |gate * n|)
    |out - exact|          <= u |exact| + K e |exact|, exact from the residual_out that came back

and half the smallest subnormal in float16.  The 8-bit output is held to the
16-bit one bit by bit.  In the gradient each sum of products is off by at most
its steps times e of the sum of magnitudes (`mag` below); a column's terms are
added over at most rows / workgroups in a lane, then over the workgroups.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}
E, K, EPS = 2.0 ** -24, 64, 1e-6
DTYPES = [torch.bfloat16, torch.float16]
IDS = ["bf16", "fp16"]
GATES = ["none", "channel", "sequence", "element"]


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "the gpu tests need a HIP device"
    import hp_rms_norm_amd
    return hp_rms_norm_amd


def k_of(hidden):
    return K + hidden / 4096 * 16


class Case:
    """Inputs of [groups, length, hidden], as views of wider rows that start
    `offset` elements in, and their exact results."""

    def __init__(self, groups, length, hidden, dtype, seed, gate="none", post=True, scale=1.0, pad=0, offset=0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.shape, self.dtype, self.scale, self.hidden = (groups, length, hidden), dtype, scale, hidden

        def rows_of(*lead, mean=0.0):
            n = 1
            for v in lead:
                n *= v
            store = (mean + torch.randn(n * (hidden + pad) + offset, generator=g, device=DEV)).to(dtype)
            return store[offset:].view(*lead, hidden + pad)[..., :hidden]
        self.rows_of = rows_of
        self.x, self.s = rows_of(groups, length), rows_of(groups, length)
        self.w, self.p = (1 + 0.1 * torch.randn((2, hidden + offset), generator=g, device=DEV)).to(dtype)[:, offset:]
        if not post:
            self.p = None
        lead = {"none": None, "channel": (), "sequence": (groups, 1), "element": (groups, length)}[gate]
        self.gate = None if lead is None else rows_of(*lead, mean=0.5)

    def forward(self, ops):
        return ops.norm_add_rms_norm(self.x, self.s, self.p, self.w, EPS, gate=self.gate, residual_scale=self.scale)

    def check_residual(self, got):
        n = self.x.double()
        if self.p is not None:
            n = n * (n.pow(2).mean(-1, keepdim=True) + EPS).rsqrt() * self.p.double()
        if self.gate is not None:
            n = n * self.gate.double()
        r = self.scale * self.s.double()
        off = (got.double() - (r + n)).abs()
        u = U[self.dtype]
        assert bool((off <= u * (r + n).abs() + k_of(self.hidden) * E * (1 + u) * (r.abs() + n.abs())
                     + TINY[self.dtype]).all()), off.max()

    def check_out(self, got, residual_out):
        h = residual_out.double()
        y = h * (h.pow(2).mean(-1, keepdim=True) + EPS).rsqrt() * self.w.double()
        off = (got.double() - y).abs()
        u = U[self.dtype]
        assert bool((off <= u * y.abs() + k_of(self.hidden) * E * (1 + u) * y.abs() + TINY[self.dtype]).all()), off.max()


def quantised(y):
    """The 8-bit integers and scales of 16-bit rows, operation by operation in
    binary32 as documented; the quotients in binary64 and rounded, which gives
    binary32's (torch divides by a number as it multiplies by its inverse)."""
    scale = torch.clamp((y.double().abs().amax(-1, keepdim=True) / 127.0).float(), min=2.0 ** -126)
    inverse = (1.0 / scale.double()).float()
    return torch.clamp(torch.round(y.float() * inverse), -127, 127).to(torch.int8), scale


# every lane mapping's last and first width, widths off the 8-element grid and
# both sides of the register-resident kernels' range
WIDTHS = [1, 7, 8, 9, 64, 128, 129, 250, 256, 257, 512, 520, 1000, 1024, 1025, 2048, 2056, 4096, 4097, 4104, 5120, 6144,
          6145, 8192, 8200, 12001, 16384, 16385, 16392, 32768, 32769]


@pytest.mark.parametrize("hidden", WIDTHS)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_forward_matches_the_formula(ops, hidden, dtype):
    for i, (groups, length, gate, post, scale) in enumerate((
            (1, 1, "none", True, 1.0), (3, 11, "sequence", True, 0.25), (1, 37, "channel", False, 1.4),
            (5, 4, "element", True, 0.7), (2, 20, "none", False, 1.0))):
        c = Case(groups, length, hidden, dtype, hidden + i, gate, post, scale)
        out, res = c.forward(ops)
        assert out.dtype == res.dtype == dtype and out.shape == res.shape == c.shape
        c.check_residual(res)
        c.check_out(out, res)
        q, qs, qres = ops.norm_add_rms_norm_int8(c.x, c.s, c.p, c.w, EPS, gate=c.gate, residual_scale=scale)
        assert q.dtype == torch.int8 and qs.shape == (groups, length, 1)
        assert torch.equal(qres, res)
        want, want_scale = quantised(out)
        assert torch.equal(qs, want_scale) and torch.equal(q, want)


@pytest.mark.parametrize("hidden", [64, 129, 4096, 5003])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_the_plain_add_with_an_8_bit_output(ops, hidden, dtype):
    """hp_rms_norm_int8 is hp_rms_norm with its output quantised: the residual
    exactly, the output to what a step of the 16-bit output (whose sum may be
    in another order) and half a step of the integers allow."""
    c = Case(1, 50, hidden, dtype, hidden, post=False)
    want, want_res = ops.fused_add_rms_norm(c.x, c.s, c.w, EPS)
    s = c.s.clone()
    q, scale = ops.fused_add_rms_norm_int8(c.x, s, c.w, EPS)
    assert torch.equal(s, want_res) and q.shape == c.shape and scale.shape == (1, 50, 1)
    off = (q.double() * scale.double() - want.double()).abs()
    assert bool((off <= scale.double() * (0.5 + 127 * 4 * E) + 2 * U[dtype] * want.double().abs() + TINY[dtype]).all())
    assert bool((q.abs().amax(-1) == 127).all())
    s2 = c.s.clone()
    q2, scale2 = torch.empty_like(q), torch.empty_like(scale)
    ops.hp_rms_norm_int8(q2, scale2, c.x, c.w, s2, EPS)
    assert torch.equal(q2, q) and torch.equal(scale2, scale) and torch.equal(s2, s)


@pytest.mark.parametrize("hidden,pad,offset", [(4096, 8, 0), (4096, 7, 1), (1001, 24, 3), (128, 128, 0), (20, 1, 5),
                                               (33000, 3, 1)])
def test_strided_and_misaligned_rows(ops, hidden, pad, offset):
    for dtype in DTYPES:
        c = Case(2, 35, hidden, dtype, 11, "sequence", True, 0.5, pad, offset)

        def room(dtype):
            return torch.zeros(70 * (hidden + 3) + 1, device=DEV, dtype=dtype)[1:].view(2, 35, hidden + 3)
        stores = [room(dtype), room(dtype)]
        out, res = (v[..., :hidden] for v in stores)
        ops.norm_add_rms_norm_out(out, res, c.x, c.s, c.p, c.w, EPS, gate=c.gate, residual_scale=0.5)
        c.check_residual(res)
        c.check_out(out, res)
        q8, r8 = room(torch.int8), room(dtype)
        scale = torch.empty(70, device=DEV)
        ops.norm_add_rms_norm_int8_out(q8[..., :hidden], scale, r8[..., :hidden], c.x, c.s, c.p, c.w, EPS, gate=c.gate,
                                       residual_scale=0.5)
        want, want_scale = quantised(out)
        assert torch.equal(q8[..., :hidden], want) and torch.equal(scale, want_scale.view(-1))
        assert torch.equal(r8[..., :hidden], res)
        for v in stores + [q8, r8]:  # what lies between the rows is left as it was
            assert not bool(v[..., hidden:].any())


@pytest.mark.parametrize("hidden", [9, 1001, 4096, 4097, 20000, 33000])
def test_in_place(ops, hidden):
    for gate, post in (("none", True), ("element", False)):
        c = Case(3, 40, hidden, torch.bfloat16, 3, gate, post, 0.9)
        want = c.forward(ops)
        x, s = c.x.clone(), c.s.clone()
        ops.norm_add_rms_norm_out(x, s, x, s, c.p, c.w, EPS, gate=c.gate, residual_scale=0.9)
        assert torch.equal(x, want[0]) and torch.equal(s, want[1])


def test_rows_do_not_depend_on_the_others(ops):
    """In either mode: the shape follows from the width alone."""
    for hidden in (128, 4096, 5003):
        c = Case(1, 700, hidden, torch.bfloat16, 8, "element")
        out, res = c.forward(ops)
        for at in (0, 1, 333, 699):
            one = slice(at, at + 1)
            o, r = ops.norm_add_rms_norm(c.x[:, one], c.s[:, one], c.p, c.w, EPS, gate=c.gate[:, one])
            assert torch.equal(o, out[:, one]) and torch.equal(r, res[:, one])


def test_special_rows(ops):
    """Zeros, infinities and NaN stay in their rows; a row of zeros has a zero
    output and the smallest scale; a row that holds NaN or infinity has that as
    its scale and zeros as integers."""
    for hidden in (64, 1001, 4096, 20000, 33000):
        c = Case(1, 9, hidden, torch.bfloat16, 5)
        x, s = c.x.clone(), c.s.clone()
        x[0, 2], s[0, 2] = 0.0, 0.0
        s[0, 4, hidden - 1] = float("nan")
        s[0, 5, 3] = float("inf")
        x[0, 6, hidden // 2] = float("nan")
        q, scale, res = ops.norm_add_rms_norm_int8(x, s, c.p, c.w, EPS)
        out, res2 = ops.norm_add_rms_norm(x, s, c.p, c.w, EPS)
        fine = [0, 1, 3, 7, 8]
        want, want_scale = quantised(out)
        assert torch.equal(q[:, fine], want[:, fine]) and torch.equal(scale[:, fine], want_scale[:, fine])
        assert not bool(out[0, 2].any()) and not bool(q[0, 2].any()) and float(scale[0, 2]) == 2.0 ** -126
        for row in (4, 5, 6):
            assert not bool(torch.isfinite(scale[0, row]).any()) and not bool(q[0, row].any())
        assert bool(torch.isnan(out[0, [4, 6]]).all()) and bool(torch.isnan(out[0, 5, 3]))
        assert bool(torch.isfinite(out[:, fine]).all()) and bool(torch.isfinite(res[:, fine]).all())
        assert torch.equal(torch.isnan(res), torch.isnan(res2))


# ---- the gradient ---------------------------------------------------------------------------
def check_backward(c, got, res, dout, dres):
    """`got`: the backward call's five; `res`: the updated residual it was given."""
    dinput, dresidual_in, dpost, dweight, dgate = got
    u, tiny = U[c.dtype], TINY[c.dtype]
    k = 2 * k_of(c.hidden)
    rows = c.shape[0] * c.shape[1]
    cols = k + rows / 32 + 64
    h, d, w = res.double(), dout.double(), c.w.double()
    r = (h.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
    g = d * w
    dh = r * g - h * r ** 3 * (g * h).mean(-1, keepdim=True)
    mag = (r * g).abs() + h.abs() * r ** 3 * (g * h).abs().mean(-1, keepdim=True)
    if dres is not None:
        dh, mag = dh + dres.double(), mag + dres.double().abs()

    def near(got, want, size, steps):
        v = U[got.dtype]
        off = (got.double() - want).abs()
        assert bool((off <= v * want.abs() + steps * E * (1 + v) * size + TINY[got.dtype]).all()), off.max()

    near(dresidual_in, c.scale * dh, abs(c.scale) * mag, k)
    t = d * h * r
    near(dweight, t.sum((0, 1)), t.abs().sum((0, 1)), cols)
    n, a, amag = c.x.double(), dh, mag
    if c.p is not None:
        q = (n.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
        n = n * q * c.p.double()
    if c.gate is not None:
        gate = c.gate.double()
        a, amag = a * gate, amag * gate.abs()
        near(dgate, (dh * n).sum_to_size(gate.shape), (mag * n.abs()).sum_to_size(gate.shape), cols)
    else:
        assert dgate is None
    if c.p is None:
        assert dpost is None
        near(dinput, a, amag, k)
        return
    x, p = c.x.double(), c.p.double()
    near(dpost, (a * x * q).sum((0, 1)), (amag * (x * q).abs()).sum((0, 1)), cols)
    dx = q * a * p - x * q ** 3 * (a * p * x).mean(-1, keepdim=True)
    size = q * amag * p.abs() + x.abs() * q ** 3 * (amag * (p * x).abs()).mean(-1, keepdim=True)
    near(dinput, dx, size, k)


def run_backward(ops, c, residual=True):
    _, res = c.forward(ops)
    dout = c.rows_of(*c.shape[:2])
    dres = c.rows_of(*c.shape[:2]) if residual else None
    got = ops.norm_add_rms_norm_backward(dout, c.x, res, c.p, c.w, EPS, gate=c.gate, residual_scale=c.scale,
                                         dresidual=dres)
    return got, res, dout, dres


@pytest.mark.parametrize("hidden", WIDTHS)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_gradient_matches_the_formula(ops, hidden, dtype):
    for i, (groups, length, gate, post, scale, residual) in enumerate((
            (1, 1, "none", True, 1.0, True), (3, 11, "sequence", True, 0.25, False),
            (1, 37, "channel", False, 1.4, True), (5, 4, "element", True, 0.7, True),
            (2, 150, "sequence", False, 1.0, True), (1, 290, "channel", True, 0.5, False),
            (2, 20, "none", False, 1.0, False), (9, 5, "element", False, 1.0, True))):
        c = Case(groups, length, hidden, dtype, 100 + hidden + i, gate, post, scale)
        got, res, dout, dres = run_backward(ops, c, residual)
        check_backward(c, got, res, dout, dres)


@pytest.mark.parametrize("groups,length,hidden", [
    (1, 5000, 128), (1, 20000, 64), (1, 2500, 4096), (1, 1500, 8192), (700, 3, 4096), (2000, 7, 96), (300, 9, 1000),
    (255, 8, 6144), (3, 700, 5003), (40, 60, 2048), (1300, 2, 512), (70, 5, 16384)])
@pytest.mark.parametrize("gate", GATES)
def test_more_rows_or_gates_than_workgroups(ops, groups, length, hidden, gate):
    c = Case(groups, length, hidden, torch.bfloat16, 6, gate, True, 0.8)
    got, res, dout, dres = run_backward(ops, c)
    check_backward(c, got, res, dout, dres)


@pytest.mark.parametrize("hidden,pad,offset", [(4096, 8, 0), (4096, 7, 1), (1001, 24, 3), (128, 128, 0), (20, 1, 5),
                                               (17000, 3, 1)])
@pytest.mark.parametrize("gate", ["sequence", "element"])
def test_gradient_of_strided_and_misaligned_rows(ops, hidden, pad, offset, gate):
    c = Case(2, 35, hidden, torch.float16, 12, gate, True, 0.5, pad, offset)
    _, res = c.forward(ops)
    dout, dres = c.rows_of(2, 35), c.rows_of(2, 35)

    def room(*lead):
        n = 1
        for v in lead:
            n *= v
        return torch.zeros(n * (hidden + 3) + 1, device=DEV, dtype=torch.float16)[1:].view(*lead, hidden + 3)
    stores = [room(2, 35), room(2, 35), room(*c.gate.shape[:2])]
    di, dr, dg = (v[..., :hidden] for v in stores)
    dw, dp = torch.empty(hidden, device=DEV), torch.empty(hidden, device=DEV)
    ops.norm_add_rms_norm_backward_out(di, dr, dp, dw, dg, dout, c.x, res, c.p, c.w, EPS, c.gate, 0.5, dres)
    check_backward(c, (di, dr, dp, dw, dg), res, dout, dres)
    for v in stores:
        assert not bool(v[..., hidden:].any())


@pytest.mark.parametrize("hidden", [9, 1001, 4096, 4097, 16384, 17000])
def test_gradient_in_place(ops, hidden):
    c = Case(4, 60, hidden, torch.bfloat16, 13, "element", True, 0.9)
    want, res, dout, dres = run_backward(ops, c)
    for pick in ((0, 1), (1, 2), (2, 3), (3, 0)):
        held = [dout.clone(), dres.clone(), c.x.clone(), res.clone()]
        gate = c.gate.clone()
        di, dr = held[pick[0]], held[pick[1]]
        dw, dp = torch.empty_like(c.w), torch.empty_like(c.w)
        ops.norm_add_rms_norm_backward_out(di, dr, dp, dw, gate, held[0], held[2], held[3], c.p, c.w, EPS, gate, 0.9,
                                           held[1])
        for a, b in zip((di, dr, dp, dw, gate), want):
            assert torch.equal(a, b)


def test_no_rows(ops):
    for shape, gate in (((0, 7, 64), (64,)), ((3, 0, 64), (3, 1, 64)), ((3, 0, 64), None)):
        e = torch.empty(shape, device=DEV, dtype=torch.bfloat16)
        w = torch.ones(64, device=DEV, dtype=torch.bfloat16)
        g = None if gate is None else torch.ones(gate, device=DEV, dtype=torch.bfloat16)
        out, res = ops.norm_add_rms_norm(e, e, w, w, EPS, gate=g)
        assert out.shape == res.shape == shape
        q, scale, _ = ops.norm_add_rms_norm_int8(e, e, w, w, EPS, gate=g)
        assert q.shape == shape and scale.shape == shape[:-1] + (1,)
        torch.full((1 << 16,), 3.0, device=DEV)  # what the allocator hands out next is not zero
        _, _, dp, dw, dg = ops.norm_add_rms_norm_backward(e, e, e, w, w, EPS, gate=g)
        assert not bool(dp.any()) and not bool(dw.any()) and (g is None or not bool(dg.any()))


def test_gradient_against_differences(ops):
    """Central differences of a binary64 model of the forward call, along a
    random direction of every input: the gradients' inner product with the
    direction.  Each gradient element is off by its rounding (u of itself) and
    far less, the difference's own error is below 1e-7 of the terms'
    magnitudes."""
    c = Case(3, 17, 200, torch.float16, 21, "sequence", True, 0.7)
    got, res, dout, dres = run_backward(ops, c)
    g = torch.Generator(device=DEV).manual_seed(22)

    def model(x, s, p, w, gate):
        n = x * (x.pow(2).mean(-1, keepdim=True) + EPS).rsqrt() * p
        h = c.scale * s + gate * n
        y = h * (h.pow(2).mean(-1, keepdim=True) + EPS).rsqrt() * w
        return (y * dout.double()).sum() + (h * dres.double()).sum()
    # the residual is such that the stored one is exact: h = res
    n = c.x.double() * (c.x.double().pow(2).mean(-1, keepdim=True) + EPS).rsqrt() * c.p.double()
    at = [c.x.double(), (res.double() - c.gate.double() * n) / c.scale, c.p.double(), c.w.double(), c.gate.double()]
    grads = [got[0], got[1], got[2], got[3], got[4]]
    for i, (v, d) in enumerate(zip(at, grads)):
        way = torch.randn(v.shape, generator=g, device=DEV, dtype=torch.float64)
        step = 1e-5
        up, down = list(at), list(at)
        up[i], down[i] = v + step * way, v - step * way
        slope = (model(*up) - model(*down)) / (2 * step)
        size = (d.double() * way).abs().sum()
        assert abs(float((d.double() * way).sum() - slope)) <= float((U[c.dtype] + 1e-4) * size)


@pytest.mark.parametrize("hidden", [1, 7, 9, 1001, 4096, 16384, 16385, 33000])
@pytest.mark.parametrize("gate", ["channel", "sequence", "element"])
@pytest.mark.parametrize("post", [True, False])
def test_gradient_of_one_row_in_place_of_its_gate(ops, hidden, gate, post):
    """One row has a gate of its own, whichever shape the gate has."""
    c = Case(1, 1, hidden, torch.bfloat16, 14, gate, post, 0.9)
    want, res, dout, dres = run_backward(ops, c)
    check_backward(c, want, res, dout, dres)
    held = c.gate.clone()
    di, dr, dw = torch.empty_like(c.x), torch.empty_like(c.x), torch.empty_like(c.w)
    dp = torch.empty_like(c.p) if post else None
    ops.norm_add_rms_norm_backward_out(di, dr, dp, dw, held, dout, c.x, res, c.p, c.w, EPS, held, 0.9, dres)
    for a, b in zip((di, dr, dp, dw, held), want):
        assert (a is None and b is None) or torch.equal(a, b)


# the last vector of a row overlaps the one before, in elements hidden - 8 ... hidden / 8 * 8 - 1
OVERLAPPED = [9, 121, 250, 257, 505, 1001, 2047, 4097, 5003, 8187, 12001, 16383, 17001, 32761]


def alike(got, want):
    """The same infinities and NaN, and elsewhere the same numbers up to roundings."""
    u = U[got.dtype]
    off = (got.double() - want).abs()
    same = (got.double() == want) | (torch.isnan(got) & torch.isnan(want))
    return bool((same | (torch.isfinite(want) & (off <= (u + 2 * k_of(want.shape[-1]) * E) * want.abs()
                                                 + TINY[got.dtype]))).all())


@pytest.mark.parametrize("hidden", OVERLAPPED)
@pytest.mark.parametrize("where", ["gate", "gate of a row", "post_weight", "weight"])
def test_infinities_where_a_rows_vectors_overlap(ops, hidden, where):
    """An infinity in the gate or a weight makes its own element infinite, the
    others 0 (its mean square is infinite) and no more than that NaN."""
    for at in (hidden - 8, hidden // 8 * 8 - 1):
        c = Case(1, 6, hidden, torch.bfloat16, 15, "element" if where == "gate of a row" else "channel", True, 0.5)
        if where == "post_weight":
            c.p[at] = float("inf")
        elif where == "weight":
            c.w[at] = float("inf")
        else:
            c.gate.view(-1, hidden)[-1, at] = -float("inf")
        out, res = c.forward(ops)
        x, gate = c.x.double(), c.gate.double()
        n = gate * (x * (x.pow(2).mean(-1, keepdim=True) + EPS).rsqrt() * c.p.double())
        want = c.scale * c.s.double() + n
        assert torch.equal(torch.isinf(res), torch.isinf(want)) and not bool(torch.isnan(res).any())
        assert torch.equal(res[torch.isinf(want)].double(), want[torch.isinf(want)])
        h = res.double()
        y = h * (h.pow(2).mean(-1, keepdim=True) + EPS).rsqrt() * c.w.double()
        assert alike(out, y)
        q, scale, qres = ops.norm_add_rms_norm_int8(c.x, c.s, c.p, c.w, EPS, gate=c.gate, residual_scale=c.scale)
        assert torch.equal(qres, res)
        top = out.abs().amax(-1, keepdim=True).double()  # NaN where a row has one
        bad = ~torch.isfinite(top)
        assert alike(scale[bad], top[bad]) and not bool(q.masked_select(bad).any())
        fine = ~bad.view(-1)
        want_q, want_scale = quantised(out[:, fine])
        assert torch.equal(q[:, fine], want_q) and torch.equal(scale[:, fine], want_scale)


@pytest.mark.parametrize("hidden", [9, 40, 257, 1001, 2048, 4097, 5003, 5120, 12001, 33000])
def test_8_bit_rows_whose_mean_square_is_lost(ops, hidden):
    """Without eps, a row too small to be squared in binary32 has an infinite
    output where it is not 0, and that is its scale."""
    c = Case(1, 4, hidden, torch.bfloat16, 17, post=False)
    x, s = torch.zeros_like(c.x), c.s.clone()
    s[0, 1] = torch.where(s[0, 1] >= 0, 1e-30, -1e-30).to(torch.bfloat16)
    q, scale, res = ops.norm_add_rms_norm_int8(x, s, None, c.w, 0.0)
    out, _ = ops.norm_add_rms_norm(x, s, None, c.w, 0.0)
    assert torch.equal(res, s) and bool(torch.isinf(out[0, 1]).all())
    assert float(scale[0, 1]) == float("inf") and not bool(q[0, 1].any())
    fine = [0, 2, 3]
    want, want_scale = quantised(out[:, fine])
    assert torch.equal(q[:, fine], want) and torch.equal(scale[:, fine], want_scale)


@pytest.mark.parametrize("hidden", [h for h in OVERLAPPED if h != 32761])
@pytest.mark.parametrize("where", ["gate of a row", "gate", "post_weight", "weight"])
@pytest.mark.parametrize("post", [True, False])
def test_gradient_of_infinities_where_a_rows_vectors_overlap(ops, hidden, where, post):
    """Infinities and NaN as the formula has them; what it leaves finite is what
    it is without the infinity, bit by bit."""
    if where == "post_weight" and not post:
        return
    for at in (hidden - 8, hidden // 8 * 8 - 1):
        c = Case(1, 6, hidden, torch.bfloat16, 16, "element" if where == "gate of a row" else "channel", post, 0.5)
        c.p = None if c.p is None else c.p.clone()
        base, res, dout, dres = run_backward(ops, c)
        if where == "post_weight":
            c.p[at] = float("inf")
        elif where == "weight":
            c.w[at] = float("inf")
        else:
            c.gate.view(-1, hidden)[-1, at] = -float("inf")
        got = ops.norm_add_rms_norm_backward(dout, c.x, res, c.p, c.w, EPS, gate=c.gate, residual_scale=c.scale,
                                             dresidual=dres)
        h, d, x, gate = res.double(), dout.double(), c.x.double(), c.gate.double()
        r = (h.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
        g = d * c.w.double()
        dh = r * g - h * (r ** 3 * (g * h).mean(-1, keepdim=True)) + dres.double()
        a, n, dpost = gate * dh, x, None
        dx = a
        if post:
            q = (x.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
            n = x * q * c.p.double()
            dpost = (a * x * q).sum((0, 1))
            a = a * c.p.double()
            dx = q * a - x * (q ** 3 * (a * x).mean(-1, keepdim=True))
        wants = (dx, c.scale * dh, dpost, (d * h * r).sum((0, 1)), (dh * n).sum_to_size(gate.shape))
        for name, v, want, b in zip(("dinput", "dresidual_in", "dpost", "dweight", "dgate"), got, wants, base):
            if want is None:
                assert v is None
                continue
            fine = torch.isfinite(want)
            assert torch.equal(v[fine], b[fine]), name
            if v.shape == c.shape:
                inf = torch.isinf(want)
                assert torch.equal(torch.isnan(v), torch.isnan(want)) and torch.equal(v[inf].double(), want[inf]), name
            else:  # a factor that rows share multiplies their sum: infinite where the sum of products is NaN
                assert not bool(torch.isfinite(v[~fine]).any()), name


@pytest.mark.parametrize("hidden", [7, 64, 129, 512, 1000, 2048, 4096, 5003, 8192, 12001, 16384, 17000])
@pytest.mark.parametrize("gate", GATES)
def test_rows_of_the_gradient_do_not_depend_on_the_others(ops, hidden, gate):
    """A row alone, whose gate is then one for all rows and one for each alike,
    among few and among many."""
    for dtype in DTYPES:
        for post in (True, False):
            c = Case(1, 240, hidden, dtype, 18, gate, post, 0.7)
            want, res, dout, dres = run_backward(ops, c)
            for at in [slice(i, i + 1) for i in range(0, 240, 6)] + [slice(3, 5), slice(100, 160)]:
                g = c.gate[:, at] if gate == "element" else c.gate
                got = ops.norm_add_rms_norm_backward(dout[:, at], c.x[:, at], res[:, at], c.p, c.w, EPS, gate=g,
                                                     residual_scale=0.7, dresidual=dres[:, at])
                assert torch.equal(got[0], want[0][:, at]) and torch.equal(got[1], want[1][:, at])
                if gate == "element":
                    assert torch.equal(got[4], want[4][:, at])
