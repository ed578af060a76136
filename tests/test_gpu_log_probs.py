"""Log probabilities of given tokens, entropy, alternatives and their gradient
on the GPU against binary64.

Bounds, with e = 2^-24: an exponential's argument is off by 2 e of itself, which
moves the exponential by less than 1 e of the largest one, its own error is
within 2 e, and a sum of positive terms is off by at most e a step: at most 128
terms a lane, 6 joining steps, as many again over the parts of a row.  With K =
256 a row's sum of exponentials is off by at most K e of itself, the weighted
sum likewise, so

    |lse - exact|       <= K e + 4 e |exact|
    |log_prob - exact|  <= K e + 4 e (|z| + |lse|)
    |entropy - exact|   <= 3 K e (1 + exact)

and a probability in the gradient by K e + 4 e (|lse| + |z - lse|) of itself.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -149}
E, K = 2.0 ** -24, 256
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = ["bf16", "fp16", "fp32"]
INF = float("inf")


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "the gpu tests need a HIP device"
    import hp_rms_norm_amd
    return hp_rms_norm_amd


def make(rows, vocab, dtype, seed, masked=0.0, ignored=0.0, pad=0, offset=0, spread=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    store = (spread * torch.randn(rows * (vocab + pad) + offset, generator=g, device=DEV)).to(dtype)
    z = store[offset:].view(rows, vocab + pad)[:, :vocab]
    if masked:
        z.masked_fill_(torch.rand((rows, vocab), generator=g, device=DEV) < masked, -INF)
    t = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    t[torch.rand(rows, generator=g, device=DEV) < ignored] = -100
    return z, t


def exact(z, t):
    """lse, log_prob, entropy of rows that have a finite value; relative to the
    largest logit, beside which binary64 too may lose the sum's logarithm."""
    z = z.double()
    m = z.amax(1)
    d = z - m[:, None]
    log_s = d.exp().sum(1).log()
    lse = m + log_s
    log_p = d - log_s[:, None]
    p = log_p.exp()
    entropy = -torch.where(p > 0, p * log_p, 0.0).sum(1)
    return lse, log_p.gather(1, t[:, None])[:, 0], entropy


def equal_or_near(got, want, bound):
    # a value past binary32's range rounds to infinity (bfloat16's and binary32's
    # largest minus their lowest)
    same = (got == want.float()) | (torch.isnan(got) & torch.isnan(want))
    return bool((same | ((got.double() - want).abs() <= bound)).all())


def check(got, z, t, top):
    log_prob, entropy, lse, top_log_prob, top_index = got
    kept = t != -100
    for v in (log_prob, entropy, lse):
        assert not bool(v[~kept].any())
    assert not bool(top_log_prob[~kept].any()) and bool((top_index[~kept] == -1).all())
    z, t = z[kept], t[kept]
    want_lse, want_log_prob, want_entropy = exact(z, t)
    at = z.double().gather(1, t[:, None])[:, 0]
    assert equal_or_near(lse[kept], want_lse, K * E + 4 * E * want_lse.abs())
    assert equal_or_near(log_prob[kept], want_log_prob, K * E + 4 * E * (at.abs() + want_lse.abs()))
    assert equal_or_near(entropy[kept], want_entropy, 3 * K * E * (1 + want_entropy))
    if top:
        order = torch.sort(z.double(), dim=1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(top_index[kept], order)
        v = z.double().gather(1, order)
        assert equal_or_near(top_log_prob[kept], v - want_lse[:, None],
                             K * E + 4 * E * (v.abs() + want_lse.abs()[:, None]))


# one element, both sides of a vector, of a step, of a part in either width, of 64 parts
VOCABS = [1, 2, 3, 7, 8, 9, 64, 255, 256, 257, 511, 513, 1000, 4095, 4096, 4097, 8191, 8192, 8193, 16385, 50001, 131072]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_matches_the_formula(ops, vocab, dtype):
    for i, (rows, top, masked, ignored, pad, offset) in enumerate((
            (1, 0, 0.0, 0.0, 0, 0), (5, 1, 0.0, 0.3, 3, 1), (33, 20, 0.5, 0.1, 0, 0), (7, 64, 0.0, 0.0, 13, 5))):
        top = min(top, vocab)
        z, t = make(rows, vocab, dtype, vocab + i, 0.0 if vocab < 9 else masked, ignored, pad, offset)
        if masked:
            z[:, 0] = 1.0  # no row is without a value
        got = ops.token_log_probs(z, t, top=top)
        assert got[0].shape == (rows,) and got[3].shape == got[4].shape == (rows, top)
        check(got, z, t, top)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("vocab", [600000, 1 << 20])
def test_the_largest_vocabularies(ops, vocab, dtype):
    z, t = make(3, vocab, dtype, 7)
    t[-1] = vocab - 1
    check(ops.token_log_probs(z, t, top=64), z, t, 64)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("vocab", [65, 1000, 9001, 40000])
def test_equal_values_go_by_the_lower_index(ops, vocab, dtype):
    """Few distinct values, one value, values in ascending and descending order,
    zeros of both signs, fewer allowed tokens than alternatives."""
    g = torch.Generator(device=DEV).manual_seed(vocab)
    z = torch.randint(-3, 4, (8, vocab), generator=g, device=DEV).to(dtype)
    z[1] = 2.5
    z[2] = torch.linspace(-4, 4, vocab, device=DEV).to(dtype)
    z[3] = torch.linspace(4, -4, vocab, device=DEV).to(dtype)
    z[4] = torch.where(torch.rand(vocab, generator=g, device=DEV) < 0.5, 0.0, -0.0).to(dtype)
    z[5] = -INF
    z[5, [vocab - 1, 17, 40]] = torch.tensor([1.0, 3.0, 1.0], device=DEV, dtype=dtype)
    z[6] = torch.finfo(dtype).min  # masks of the type's lowest value
    z[6, 33] = -2.0
    z[7] = torch.finfo(dtype).max
    z[7, 5:9] = torch.finfo(dtype).min
    t = torch.tensor([0, 1, 2, 3, 4, 17, 33, 7], device=DEV)
    for top in (1, 5, 64):
        check(ops.token_log_probs(z, t, top=top), z, t, top)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("top", [2, 19, 20, 21, 32, 33, 50, 63, 64])
def test_where_the_largest_values_lie(ops, top, dtype):
    """Spread out, neighbours in few lanes, in one wave, at a row's end, all
    negative, and one lane's apart from the others; few rows and many."""
    for rows, vocab in ((6, 2000), (6, 50001), (600, 9001)):
        z, t = make(rows, vocab, dtype, top)
        z[1::6, 100:100 + top] += 30.0
        z[2::6, :512] += 20.0
        z[3::6, vocab - top + 1:] += 25.0
        z[4::6] -= 40.0
        z[5::6, ::2048] += 30.0
        check(ops.token_log_probs(z, t, top=top), z, t, top)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("vocab", [3, 700, 20000])
def test_rows_without_a_value_and_values_that_are_not_numbers(ops, vocab, dtype):
    z, t = make(6, vocab, dtype, 3)
    t = torch.full((6,), 1, device=DEV)
    z[1] = -INF
    z[2, vocab - 1] = float("nan")
    z[3, 2] = INF
    z[4, 1] = -INF  # the given token is forbidden
    t[5] = vocab    # out of range
    top = min(3, vocab)
    log_prob, entropy, lse, top_log_prob, top_index = ops.token_log_probs(z, t, top=top)
    fine = torch.tensor([0, 4], device=DEV)
    check([v[fine] for v in (log_prob, entropy, lse, top_log_prob, top_index)], z[fine], t[fine], top)
    assert float(log_prob[1]) == float(lse[1]) == -INF and float(entropy[1]) == 0.0
    assert bool((top_log_prob[1] == -INF).all()) and top_index[1].tolist() == list(range(top))
    assert bool(torch.isnan(lse[[2, 3]]).all()) and bool(torch.isnan(log_prob[[2, 3, 5]]).all())
    assert int(top_index[2, 0]) == vocab - 1 and int(top_index[3, 0]) == 2
    assert float(log_prob[4]) == -INF and bool(torch.isfinite(lse[5]))
    g = torch.ones(6, device=DEV)
    d = ops.token_log_probs_backward(g, z, t, lse, entropy=entropy, dentropy=0.5 * g)
    assert not bool(d[1].any()) and bool(torch.isnan(d[[2, 3, 5]]).all())
    check_backward(d[fine], z[fine], t[fine], g[fine], 0.5 * g[fine])
    allowed = z[4] > -INF
    assert float(d[4, 1]) == 1.0 and not bool(d[4][~allowed][1:].any())


def test_ignored_rows_are_not_read(ops):
    z, t = make(9, 5000, torch.bfloat16, 12)
    want = ops.token_log_probs(z, t, top=4)
    z2, t2 = z.clone(), t.clone()
    z2[[2, 7]] = float("nan")
    t2[[2, 7]] = -7
    got = ops.token_log_probs(z2, t2, top=4, ignore_index=-7)
    keep = [i for i in range(9) if i not in (2, 7)]
    for a, b in zip(got, want):
        assert torch.equal(a[keep], b[keep])
    d = ops.token_log_probs_backward(torch.full((9,), float("nan"), device=DEV), z2, t2, got[2], ignore_index=-7)
    assert not bool(d[[2, 7]].any())


# ---- the gradient ---------------------------------------------------------------------------
def check_backward(d, z, t, g, gh):
    kept = t != -100
    assert not bool(d[~kept].any())
    z, t, d, g = z[kept].double(), t[kept], d[kept], g[kept].double()[:, None]
    gh = torch.zeros_like(g) if gh is None else gh[kept].double()[:, None]
    lse = torch.logsumexp(z, 1, keepdim=True)
    log_p = z - lse
    p = log_p.exp()
    log_p = torch.where(p > 0, log_p, 0.0)
    entropy = -(p * log_p).sum(1, keepdim=True)
    own = torch.zeros_like(p).scatter_(1, t[:, None], 1.0)
    want = g * (own - p) - gh * p * (log_p + entropy)
    rel = K * E + 4 * E * (lse.abs() + log_p.abs())
    size = p * (g.abs() + gh.abs() * (log_p.abs() + entropy))
    bound = U[d.dtype] * want.abs() + (1 + U[d.dtype]) * (
        (rel + 4 * E) * size + gh.abs() * p * (rel + 3 * K * E * (1 + entropy)) + E * g.abs() * own) + TINY[d.dtype]
    # what lies below 2^-200 of a probability is 0
    off = (d.double() - want).abs()
    assert bool((off <= bound + 2.0 ** -190 * (g.abs() + gh.abs())).all()), off.max()


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_gradient_matches_the_formula(ops, vocab, dtype):
    for i, (rows, masked, ignored, pad, offset, bonus) in enumerate((
            (1, 0.0, 0.0, 0, 0, True), (5, 0.0, 0.3, 3, 1, False), (19, 0.5, 0.1, 0, 0, True))):
        z, t = make(rows, vocab, dtype, 50 + vocab + i, 0.0 if vocab < 9 else masked, ignored, pad, offset)
        if masked:
            z[:, 0] = 1.0
        g = torch.randn(rows, device=DEV, generator=torch.Generator(device=DEV).manual_seed(i))
        gh = 0.3 * g.flip(0) if bonus else None
        _, entropy, lse, _, _ = ops.token_log_probs(z, t)
        d = ops.token_log_probs_backward(g, z, t, lse, entropy=entropy if bonus else None, dentropy=gh)
        assert d.dtype == dtype and d.is_contiguous()
        check_backward(d, z, t, g, gh)


@pytest.mark.parametrize("vocab,pad,offset", [(1000, 24, 0), (1001, 7, 1), (3, 1, 1)])
def test_gradient_into_strided_rows_and_in_place(ops, vocab, pad, offset):
    for dtype in DTYPES:
        z, t = make(12, vocab, dtype, 4, 0.0, 0.2, pad, offset)
        g = torch.linspace(-1, 1, 12, device=DEV)
        _, entropy, lse, _, _ = ops.token_log_probs(z, t)
        store = torch.zeros(12 * (vocab + 3) + 1, device=DEV, dtype=dtype)[1:].view(12, vocab + 3)
        ops.token_log_probs_backward_out(store[:, :vocab], g, z, t, lse, entropy, g)
        check_backward(store[:, :vocab], z, t, g, g)
        assert not bool(store[:, vocab:].any())
        want = store[:, :vocab].clone()
        between = torch.as_strided(z, (11, pad), (vocab + pad, 1), z.storage_offset() + vocab).clone()
        ops.token_log_probs_backward_out(z, g, z, t, lse, entropy, g)
        assert torch.equal(z, want)
        assert torch.equal(torch.as_strided(z, (11, pad), (vocab + pad, 1), z.storage_offset() + vocab), between)


def test_gradient_against_differences(ops):
    """Central differences in binary64 of a weighted sum of both outputs along a
    random direction."""
    z, t = make(11, 777, torch.float32, 9)
    gen = torch.Generator(device=DEV).manual_seed(10)
    g, gh = torch.randn((2, 11), generator=gen, device=DEV)
    _, entropy, lse, _, _ = ops.token_log_probs(z, t)
    d = ops.token_log_probs_backward(g, z, t, lse, entropy=entropy, dentropy=gh).double()
    way = torch.randn((11, 777), generator=gen, device=DEV, dtype=torch.float64)

    def value(v):
        _, log_prob, h = exact(v, t)
        return (log_prob * g.double() + h * gh.double()).sum()
    step = 1e-5
    slope = (value(z.double() + step * way) - value(z.double() - step * way)) / (2 * step)
    size = float((d * way).abs().sum())
    assert abs(float((d * way).sum() - slope)) <= 1e-5 * size + 1e-7


def test_more_rows_than_one_launch_takes(ops):
    """The partial results of 2^18 rows with 64 alternatives exceed a launch's
    share of the workspace; with rows of whole 16 bytes a row's bits depend on
    no other."""
    z, t = make(1 << 18, 64, torch.bfloat16, 5, 0.0, 0.01)
    got = ops.token_log_probs(z, t, top=64)
    check(got, z, t, 64)
    at = torch.tensor([0, 131071, 131072, (1 << 18) - 1], device=DEV)
    for a, b in zip(ops.token_log_probs(z[at], t[at], top=64), got):
        assert torch.equal(a, b[at])


@pytest.mark.parametrize("vocab,dtype", [(300, torch.bfloat16), (20000, torch.float32), (131072, torch.float16),
                                         (300001, torch.bfloat16)])
def test_batch_invariant_mode(ops, vocab, dtype):
    """In the mode a row's bits depend on no other row (at one address modulo 16
    bytes, where its vectors are cut); out of it the results are
    right with any number of rows, few of which are cut into more parts."""
    z, t = make(600, vocab, dtype, 8, 0.0, 0.1)
    previous = ops.set_batch_invariant(True)
    try:
        whole = ops.token_log_probs(z, t, top=7)
        for at in (slice(0, 1), slice(5, 12), slice(100, 300), slice(599, 600)):
            for a, b in zip(ops.token_log_probs(z[at], t[at], top=7), whole):
                assert torch.equal(a, b[at])
    finally:
        ops.set_batch_invariant(previous)
    for rows in (1, 2, 9, 40, 150):
        check(ops.token_log_probs(z[:rows], t[:rows], top=7), z[:rows], t[:rows], 7)


def test_values_in_particular_places(ops):
    """Rows whose largest values stand close together, in one lane's vectors, or
    reach the bound in numbers: in each the list or the way without it serves."""
    for dtype in DTYPES:
        n = 4 if dtype == torch.float32 else 8  # of a vector
        z, t = make(12, 33000, dtype, 15, spread=0.5)
        z[0, -200:] += 9.0                     # at the end
        z[1, :200] += 9.0                      # at the beginning
        z[2, 1000:1000 + 256 * n * 8:256 * n] += 9.0  # one lane's vectors
        z[3, 512 * n:513 * n] += 9.0           # one vector
        z[4] = z[4].round()                    # thousands of equal values
        z[5, ::3] = 4.0                        # a third of the row
        z[6] = -INF
        z[6, 30000:30040] = 1.5                # fewer allowed than alternatives
        z[7] = -INF
        z[7, ::700] = torch.arange(48, device=DEV).to(dtype)
        z[8, :600] = 9.0                       # more equal values than a list holds
        z[9] = z[9].abs()
        t[6], t[7] = 30001, 700
        for top in (1, 20, 47, 64):
            check(ops.token_log_probs(z, t, top=top), z, t, top)
            check(ops.token_log_probs(z[4:9], t[4:9], top=top), z[4:9], t[4:9], top)


def test_leading_dimensions_and_no_rows(ops):
    z, t = make(12, 300, torch.float16, 6)
    want = ops.token_log_probs(z, t, top=2)
    got = ops.token_log_probs(z.view(3, 4, 300), t.view(3, 4), top=2)
    assert got[4].shape == (3, 4, 2)
    for a, b in zip(got, want):
        assert torch.equal(a.reshape(b.shape), b)
    d = ops.token_log_probs_backward(torch.full((), -1.0, device=DEV), z.view(3, 4, 300), t.view(3, 4), got[2])
    check_backward(d.view(12, 300), z, t, torch.full((12,), -1.0, device=DEV), None)
    got = ops.token_log_probs(z[:0], t[:0], top=2)
    assert got[0].shape == (0,) and got[4].shape == (0, 2)
    assert ops.token_log_probs_backward(torch.empty(0, device=DEV), z[:0], t[:0], got[2]).shape == (0, 300)


@pytest.mark.parametrize("pad", [0, 1])
@pytest.mark.parametrize("vocab,dtype", [
    (32767, torch.bfloat16), (32768, torch.bfloat16), (50001, torch.bfloat16), (65535, torch.float16),
    (65536, torch.bfloat16), (131071, torch.float16), (131072, torch.bfloat16), (32767, torch.float32),
    (131072, torch.float32), (1001, torch.bfloat16), (77, torch.float32)])
def test_batch_invariant_mode_at_any_address(ops, vocab, dtype, pad):
    """In the mode a row's bits depend on neither the other rows nor on where the
    row lies: rows of odd strides alone, among others and copied to other
    addresses.  The vocabularies are those whose rows fill their parts to the
    last step, where a few bytes more would change the parts."""
    z, t = make(24, vocab, dtype, 8, 0.0, 0.1, pad)
    moved = make(24, vocab, dtype, 9, 0.0, 0.0, 4, 3)[0]
    moved.copy_(z)
    previous = ops.set_batch_invariant(True)
    try:
        whole = ops.token_log_probs(z, t, top=7)
        check(whole, z, t, 7)
        for rows in (z, moved):
            for at in (slice(0, 24), slice(0, 1), slice(8, 9), slice(3, 9), slice(23, 24)):
                for a, b in zip(ops.token_log_probs(rows[at], t[at], top=7), whole):
                    assert torch.equal(a, b[at])
    finally:
        ops.set_batch_invariant(previous)
