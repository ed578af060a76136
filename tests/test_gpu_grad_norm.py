"""The norm of a list of gradients and clipping by it, on the GPU.

Squares are exact in binary64 and their sum is off by at most n 2^-53 of
itself, so the float32 norm is within one rounding (2^-24) and 2^-40 of the
exact one, and an output within half a step of its type of g * factor, with
factor off by 2^-23 (its own rounding and the product's).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "the gpu tests need a HIP device"
    import hp_rms_norm_amd
    return hp_rms_norm_amd


def make(counts, dtypes, seed, scale=1.0, offset=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [(torch.randn(n + offset, generator=g, device=DEV) * scale).to(dtypes[i % len(dtypes)])[offset:]
            for i, n in enumerate(counts)]


def exact_norm(grads):
    return sum(float(t.double().pow(2).sum()) for t in grads) ** 0.5


def check_norm(norm, grads):
    want = exact_norm(grads)
    assert norm.dtype == torch.float32 and norm.dim() == 0
    assert abs(float(norm.double()) - want) <= (2.0 ** -24 + 2.0 ** -40) * want


def check_clipped(outs, grads, max_norm):
    factor = min(1.0, max_norm / (exact_norm(grads) + 1e-6))
    for o, t in zip(outs, grads):
        want = t.double() * factor
        bound = (U[o.dtype] + 2.0 ** -22) * want.abs() + TINY[o.dtype]
        assert bool(((o.double() - want).abs() <= bound).all())


COUNTS = [[1], [0, 5], [7, 8, 9], [8191, 8192, 8193], [100003], [3] * 95, [3] * 96, [17] * 97, [5, 0] * 150, [40000] * 200,
          [1 << 20, 3, 1 << 20]]


@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: f"{len(c)}x{c[0]}")
@pytest.mark.parametrize("dtypes", [[d] for d in DTYPES] + [DTYPES], ids=["bf16", "fp16", "fp32", "mixed"])
def test_norm_and_clipping(ops, counts, dtypes):
    grads = make(counts, dtypes, len(counts) + counts[0])
    before = [t.clone() for t in grads]
    check_norm(ops.grad_norm(grads), grads)
    limit = 0.3 * exact_norm(grads)
    outs = [torch.full_like(t, 9.0) for t in grads]
    wide = [torch.full(t.shape, 9.0, device=DEV) for t in grads]
    check_norm(ops.clip_grad_norm_out(outs, grads, limit), grads)
    check_clipped(outs, grads, limit)
    ops.clip_grad_norm_out(wide, grads, limit)
    check_clipped(wide, grads, limit)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    check_norm(ops.clip_grad_norm_(grads, limit), before)
    assert all(torch.equal(a, b) for a, b in zip(grads, outs))


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp16", "fp32"])
def test_below_the_limit_nothing_changes(ops, dtype):
    grads = make([1000, 9, 70000], [dtype], 3)
    before = [t.clone() for t in grads]
    ops.clip_grad_norm_(grads, 2 * exact_norm(grads))
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    outs = [torch.zeros_like(t) for t in grads]
    ops.clip_grad_norm_out(outs, grads, float("inf"))
    assert all(torch.equal(a, b) for a, b in zip(outs, before))


@pytest.mark.parametrize("offset", [1, 3])
def test_misaligned_tensors_and_their_neighbours(ops, offset):
    for dtype in DTYPES:
        grads = make([1000, 8192 * 3 + 5], [dtype], 17, offset=offset)
        stores = [torch.full((t.numel() + 2,), 5.0, device=DEV, dtype=dtype) for t in grads]
        outs = [s[1:-1] for s in stores]
        limit = 0.5 * exact_norm(grads)
        ops.clip_grad_norm_out(outs, grads, limit)
        check_clipped(outs, grads, limit)
        assert all(float(s[0]) == 5.0 and float(s[-1]) == 5.0 for s in stores)


def test_large_and_tiny_values(ops):
    """bfloat16 and float32 squares leave binary32's range both ways."""
    for scale in (1e25, 1e-25):
        grads = make([5000, 33], [torch.bfloat16, torch.float32], 4, scale)
        check_norm(ops.grad_norm(grads), grads)
    grads = [torch.full((4096,), 3e38, device=DEV)]
    assert float(ops.grad_norm(grads)) == float("inf")  # 1.9e40: past float32
    outs = [torch.empty_like(grads[0])]
    ops.clip_grad_norm_out(outs, grads, 1.0)            # the factor comes from the binary64 norm
    check_clipped(outs, grads, 1.0)


def test_tensors_without_elements(ops):
    empty = [torch.empty(0, device=DEV), torch.empty((3, 0), device=DEV, dtype=torch.bfloat16)]
    assert float(ops.grad_norm(empty)) == 0.0 and float(ops.clip_grad_norm_(empty, 1.0)) == 0.0
    grads = empty + make([10], [torch.float32], 2)
    check_norm(ops.grad_norm(grads), grads)


def test_shared_memory_is_refused_before_anything_is_written(ops):
    base = make([100], [torch.float32], 2)[0]
    before = base.clone()
    for call in (lambda: ops.clip_grad_norm_([base, base], 0.1),
                 lambda: ops.clip_grad_norm_([base[:60], base[40:]], 0.1),
                 lambda: ops.clip_grad_norm_out([base[:50], torch.empty(50, device=DEV)], [base[50:], base[:50]], 0.1),
                 lambda: ops.clip_grad_norm_out([base[1:51]], [base[:50]], 0.1)):
        with pytest.raises(RuntimeError, match="share"):
            call()
    assert torch.equal(base, before)
    # reading one tensor twice, into two others, is fine
    outs = [torch.empty(100, device=DEV), torch.empty(100, device=DEV)]
    ops.clip_grad_norm_out(outs, [base, base], 0.1)
    check_clipped(outs, [base, base], 0.1)


def test_a_list_past_the_folded_sums(ops):
    """More than 2^25 elements: longer units, and the sums added by a kernel of
    their own; in place and into other tensors, clipped and not."""
    grads = make([(1 << 25) + 77, 12345, 1 << 20], [torch.bfloat16, torch.float32], 20)
    norm = exact_norm(grads)
    outs = [torch.empty_like(t) for t in grads]
    check_norm(ops.clip_grad_norm_out(outs, grads, 0.25 * norm), grads)
    check_clipped(outs, grads, 0.25 * norm)
    before = [t.clone() for t in grads]
    ops.clip_grad_norm_(grads, 2 * norm)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    ops.clip_grad_norm_(grads, 0.25 * norm)
    assert all(torch.equal(a, b) for a, b in zip(grads, outs))


def test_not_finite(ops):
    for bad, factor in ((float("nan"), float("nan")), (float("inf"), 0.0)):
        grads = make([100, 100], [torch.float32], 8)
        grads[1][7] = bad
        before = [t.clone() for t in grads]
        norm = ops.clip_grad_norm_(grads, 1.0)
        assert torch.equal(torch.isnan(norm), torch.isnan(torch.tensor(bad, device=DEV)))
        for got, was in zip(grads, before):
            assert torch.equal(torch.nan_to_num(got, nan=7.0), torch.nan_to_num(was * factor, nan=7.0))


def test_dense_tensors_in_other_orders_and_repeated_reads(ops):
    base = make([64 * 48], [torch.bfloat16], 6)[0].view(64, 48)
    grads = [base.t(), base[:32]]
    check_norm(ops.grad_norm(grads), [base, base[:32]])
    check_norm(ops.grad_norm([base, base]), [base, base])
    out = torch.empty(64, 48, device=DEV, dtype=torch.bfloat16).t()
    ops.clip_grad_norm_out([out], [base.t()], 1.0)
    check_clipped([out], [base.t()], 1.0)


def test_bits_repeat_and_a_graph_replays_them(ops):
    grads = make([40000] * 100 + [3], [torch.bfloat16, torch.float32], 12)
    outs = [torch.empty_like(t) for t in grads]
    norm = torch.empty((), device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            norm = ops.clip_grad_norm_out(outs, grads, 5.0)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        grads[3].mul_(2.0 if i == 2 else 1.0)
        want_outs = [torch.empty_like(t) for t in grads]
        want = ops.clip_grad_norm_out(want_outs, grads, 5.0)
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(outs, want_outs))
