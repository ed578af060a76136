"""What the training operators refuse, on the CPU: the torch layer's checks
with meta tensors and the C ABI's with addresses that are never read."""
import ctypes

import pytest
import torch

from hp_rms_norm_amd import abi, ops

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def t(*shape, dtype=BF):
    return torch.empty(shape, dtype=dtype, device="meta")


def ids(*shape, dtype=torch.int64):
    return torch.empty(shape, dtype=dtype, device="meta")


def backward(dinput=None, dweight=None, dout=None, input=None, weight=None, dresidual=None, eps=1e-6):
    pick = lambda v, d: d if v is None else v  # noqa: E731
    return ops.rms_norm_backward_out(pick(dinput, t(4, 64)), pick(dweight, t(64)), pick(dout, t(4, 64)),
                                     pick(input, t(4, 64)), pick(weight, t(64)), eps, dresidual=dresidual)


def test_backward_accepts():
    assert backward() is None
    assert backward(dweight=t(64, dtype=F32), dresidual=t(4, 64)) is None
    dx, dw = ops.rms_norm_backward(t(2, 3, 64, dtype=F16), t(2, 3, 64, dtype=F16), t(64, dtype=F16), 1e-6)
    assert dx.shape == (2, 3, 64) and dw.shape == (64,) and dw.dtype == F16
    assert ops.rms_norm_backward(t(4, 0), t(4, 0), t(0), 1e-6)[0].shape == (4, 0)


@pytest.mark.parametrize("kw,msg", [
    (dict(input=t(64), dout=t(64), dinput=t(64)), r"input.dim\(\) >= 2"),
    (dict(weight=t(1, 64)), r"weight.dim\(\) == 1"),
    (dict(weight=t(32)), r"input.size\(-1\) == hidden_dim"),
    (dict(weight=t(64, dtype=F16)), r"weight.dtype\(\) == input.dtype\(\)"),
    (dict(weight=t(128)[::2]), r"weight.stride\(0\) == 1"),
    (dict(dweight=t(32)), "dweight must be shaped like weight"),
    (dict(dweight=t(64, dtype=F16)), r"dweight.dtype\(\) must be"),
    (dict(dout=t(5, 64)), "must be shaped like input"),
    (dict(dresidual=t(1, 64)), "must be shaped like input"),
    (dict(dout=t(4, 64, dtype=F16)), r"must have input.dtype\(\)"),
    (dict(dinput=t(64, 4).t()), "rows must be contiguous"),
    (dict(input=t(4, 64, dtype=F32), dout=t(4, 64, dtype=F32)), "dtype must be kFloat16 or kBFloat16"),
    (dict(dinput=t(1, 64).expand(4, 64)), "overlap"),
])
def test_backward_refuses(kw, msg):
    with pytest.raises(RuntimeError, match=msg):
        backward(**kw)


def loss(loss=None, lse=None, hidden=None, weight=None, target=None):
    pick = lambda v, d: d if v is None else v  # noqa: E731
    return ops.linear_cross_entropy_out(pick(loss, t(4, dtype=F32)), pick(lse, t(4, dtype=F32)),
                                        pick(hidden, t(4, 64)), pick(weight, t(100, 64)), pick(target, ids(4)))


def test_loss_accepts():
    assert loss() is None
    a, b = ops.linear_cross_entropy(t(2, 3, 64, dtype=F16), t(9, 64, dtype=F16), ids(2, 3))
    assert a.shape == b.shape == (2, 3) and a.dtype == b.dtype == F32
    dh, dw = ops.linear_cross_entropy_backward(t(dtype=F32), t(2, 3, 64), t(9, 64), ids(2, 3), t(2, 3, dtype=F32))
    assert dh.shape == (2, 3, 64) and dw.shape == (9, 64)


@pytest.mark.parametrize("kw,msg", [
    (dict(hidden=t(64)), r"hidden.dim\(\) >= 2"),
    (dict(weight=t(64)), r"weight.dim\(\) == 2"),
    (dict(weight=t(100, 32)), r"hidden.size\(-1\) == weight.size\(1\)"),
    (dict(weight=t(0, 64)), "at least one element"),
    (dict(weight=t(64, 100).t()), r"weight.stride\(1\) == 1"),
    (dict(weight=t(1, 64).expand(100, 64)), "rows of the tensor overlap"),
    (dict(weight=t(100, 64, dtype=F16)), r"weight.dtype\(\) == hidden.dtype\(\)"),
    (dict(hidden=t(4, 64, dtype=F32), weight=t(100, 64, dtype=F32)), "dtype must be kFloat16 or kBFloat16"),
    (dict(target=ids(4, dtype=torch.int32)), r"target.dtype\(\) == int64"),
    (dict(target=ids(5)), "one element per row"),
    (dict(target=ids(8)[::2]), "target must be contiguous"),
    (dict(loss=t(4)), "must be float32"),
    (dict(lse=t(4, 1, dtype=F32)), "must be shaped like target"),
    (dict(lse=t(8, dtype=F32)[::2]), "must be contiguous"),
])
def test_loss_refuses(kw, msg):
    with pytest.raises(RuntimeError, match=msg):
        loss(**kw)


@pytest.mark.parametrize("kw,msg", [
    (dict(dhidden=t(5, 64)), "dhidden must be shaped like hidden"),
    (dict(dweight=t(100, 63)), "dweight must be shaped like weight"),
    (dict(dweight=t(100, 64, dtype=F32)), r"must have hidden.dtype\(\)"),
    (dict(dweight=t(64, 100).t()), "rows must be contiguous"),
    (dict(dloss=t(4)), "must be float32"),
    (dict(lse=t(5, dtype=F32)), "must be shaped like target"),
])
def test_loss_backward_refuses(kw, msg):
    a = dict(dhidden=t(4, 64), dweight=t(100, 64), dloss=t(4, dtype=F32), lse=t(4, dtype=F32))
    a.update(kw)
    with pytest.raises(RuntimeError, match=msg):
        ops.linear_cross_entropy_backward_out(a["dhidden"], a["dweight"], a["dloss"], t(4, 64), t(100, 64), ids(4),
                                              a["lse"])


def test_clip_accepts():
    assert ops.grad_norm([t(4, 5), t(3, dtype=F32)]).shape == ()
    assert ops.clip_grad_norm_([t(4, 5)], 1.0).dtype == F32
    assert ops.clip_grad_norm_out([t(4, 5, dtype=F32)], [t(4, 5)], 1.0).shape == ()


@pytest.mark.parametrize("fn,msg", [
    (lambda: ops.grad_norm([]), None),
    (lambda: ops.grad_norm([t(4, dtype=torch.float64)]), "bfloat16, float16 or float32"),
    (lambda: ops.grad_norm([t(4, 8)[:, ::2]]), "dense"),
    (lambda: ops.clip_grad_norm_([t(1, 4).expand(3, 4)], 1.0), "dense"),
    (lambda: ops.clip_grad_norm_out([t(4)], [t(4), t(4)], 1.0), "one tensor per gradient"),
    (lambda: ops.clip_grad_norm_out([t(5)], [t(4)], 1.0), r"shaped like grads\[i\]"),
    (lambda: ops.clip_grad_norm_out([t(4, 5)], [t(5, 4).t()], 1.0), r"laid out like grads\[i\]"),
    (lambda: ops.clip_grad_norm_out([t(4, dtype=F16)], [t(4)], 1.0), r"grads\[i\].dtype\(\) or float32"),
    (lambda: ops.clip_grad_norm_out([t(4)], [t(4, dtype=F32)], 1.0), r"grads\[i\].dtype\(\) or float32"),
])
def test_clip_refuses(fn, msg):
    with pytest.raises(RuntimeError, match=msg):
        fn()


def test_no_cpu_fallback():
    x, w = torch.zeros(2, 8, dtype=BF), torch.ones(8, dtype=BF)
    for call in (lambda: ops.rms_norm_backward(x, x, w, 1e-6),
                 lambda: ops.linear_cross_entropy(x, torch.zeros(3, 8, dtype=BF), torch.zeros(2, dtype=torch.int64)),
                 lambda: ops.grad_norm([x]), lambda: ops.clip_grad_norm_([x], 1.0)):
        with pytest.raises(NotImplementedError):
            call()


# ---- the C ABI ---------------------------------------------------------------------------
def test_workspace_sizes():
    assert abi.rmsnorm_backward_workspace(0, 4096) == 0
    assert abi.rmsnorm_backward_workspace(1, 4096) == 4096 * 4
    assert abi.rmsnorm_backward_workspace(8192, 4096) <= 1024 * 4096 * 4
    small = abi.linear_cross_entropy_workspace(1, 4096, 131072)
    assert small < abi.linear_cross_entropy_workspace(4096, 4096, 131072) < 100 << 20
    assert abi.linear_cross_entropy_backward_workspace(4096, 4096, 131072) < 1 << 30
    assert abi.linear_cross_entropy_backward_workspace(0, 64, 100) > 0
    assert abi.grad_norm_workspace([]) >= 16
    assert abi.grad_norm_workspace([1 << 33]) < 1 << 20
    for call in (lambda: abi.rmsnorm_backward_workspace(-1, 64), lambda: abi.rmsnorm_backward_workspace(1, 0),
                 lambda: abi.rmsnorm_backward_workspace(1, (1 << 24) + 1),
                 lambda: abi.linear_cross_entropy_workspace(-1, 64, 64),
                 lambda: abi.linear_cross_entropy_workspace((1 << 22) + 1, 64, 64),
                 lambda: abi.linear_cross_entropy_backward_workspace(1, 64, 0),
                 lambda: abi.linear_cross_entropy_backward_workspace(1, 64, (1 << 28) + 1),
                 lambda: abi.grad_norm_workspace([-1]), lambda: abi.grad_norm_workspace([1 << 43])):
        with pytest.raises(abi.HprmsError):
            call()


def norm_backward(**kw):
    a = dict(dinput=0x1000, dweight=0x2000, dout=0x3000, input=0x4000, weight=0x5000, dres=0, ws=0x10000,
             ws_size=1 << 30, rows=4, hidden=64, s0=64, s1=64, s2=64, s3=64, dtype=0, wdtype=0, eps=1e-6)
    a.update(kw)
    return abi.lib().hprms_rmsnorm_backward(*a.values(), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=2), "dtype"), (dict(wdtype=1), "dweight_dtype"), (dict(rows=-1), "rows"), (dict(hidden=0), "hidden"),
    (dict(s0=63), "strides"), (dict(s1=1), "strides"), (dict(dres=0x6000, s3=2), "strides"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(dinput=0), "null"), (dict(dweight=0), "null"), (dict(weight=0), "null"),
    (dict(dout=0x3001), "aligned"), (dict(wdtype=2, dweight=0x2002), "aligned"), (dict(ws=0), "workspace"),
    (dict(ws_size=10), "workspace"), (dict(ws=0x10008), "workspace"),
])
def test_norm_backward_abi_refuses(kw, msg):
    assert norm_backward(**kw) == abi.HPRMS_E_INVALID
    assert msg in abi.last_error()


def test_norm_backward_abi_ranges():
    assert norm_backward(hidden=(1 << 24) + 8, s0=1 << 25, s1=1 << 25, s2=1 << 25) == abi.HPRMS_E_RANGE
    assert norm_backward(rows=1 << 16, s1=1 << 40) == abi.HPRMS_E_RANGE


def loss_abi(**kw):
    a = dict(loss=0x1000, lse=0x2000, hidden=0x3000, weight=0x4000, target=0x5000, ws=0x10000, ws_size=1 << 30, rows=4,
             width=64, vocab=100, hs=64, wst=64, ignore=-100, dtype=0)
    a.update(kw)
    return abi.lib().hprms_linear_cross_entropy(*a.values(), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=2), "dtype"), (dict(rows=-1), "rows"), (dict(width=0), "hidden"), (dict(vocab=0), "vocab"),
    (dict(hs=63), "strides"), (dict(wst=1), "strides"), (dict(loss=0), "null"), (dict(lse=0x2002), "misaligned"),
    (dict(hidden=0), "null"), (dict(target=0x5004), "aligned"), (dict(weight=0x4001), "aligned"),
    (dict(ws=0x10010), "workspace"), (dict(ws_size=100), "workspace"),
])
def test_loss_abi_refuses(kw, msg):
    assert loss_abi(**kw) == abi.HPRMS_E_INVALID
    assert msg in abi.last_error()


def test_loss_abi_ranges_and_no_rows():
    assert loss_abi(rows=(1 << 22) + 1) == abi.HPRMS_E_RANGE
    assert loss_abi(vocab=1 << 20, wst=1 << 40) == abi.HPRMS_E_RANGE
    assert loss_abi(rows=0, loss=0, lse=0, hidden=0, weight=0, target=0, ws=0) == abi.HPRMS_OK


def loss_backward_abi(**kw):
    a = dict(dhidden=0x1000, dweight=0x2000, dloss=0x3000, hidden=0x4000, weight=0x5000, target=0x6000, lse=0x7000,
             ws=0x10000, ws_size=1 << 30, rows=4, width=64, vocab=100, dhs=64, dws=64, hs=64, wst=64, ignore=-100,
             dtype=0)
    a.update(kw)
    return abi.lib().hprms_linear_cross_entropy_backward(*a.values(), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=7), "dtype"), (dict(dhs=63), "strides"), (dict(dws=63), "strides"), (dict(dweight=0), "null"),
    (dict(dhidden=0), "null"), (dict(dloss=0), "null"), (dict(lse=0), "null"), (dict(dloss=0x3002), "aligned"),
    (dict(dhidden=0x1001), "aligned"), (dict(ws=0), "workspace"), (dict(ws_size=1000), "workspace"),
])
def test_loss_backward_abi_refuses(kw, msg):
    assert loss_backward_abi(**kw) == abi.HPRMS_E_INVALID
    assert msg in abi.last_error()


@pytest.mark.parametrize("kw,msg", [
    (dict(norm=0), "norm"), (dict(ptrs=[0x1000, 0]), "null tensor pointer"), (dict(dtypes=[0, 3]), "dtype"),
    (dict(ptrs=[0x1000, 0x2001]), "aligned"), (dict(dtypes=[2, 0], ptrs=[0x1002, 0x2000]), "aligned"),
    (dict(counts=[4, -1]), "elements"), (dict(ws=0), "workspace"), (dict(ws_size=8), "workspace"),
])
def test_grad_norm_abi_refuses(kw, msg):
    a = dict(norm=0x100, ptrs=[0x1000, 0x2000], dtypes=[0, 0], counts=[4, 4], ws=0x10000, ws_size=1 << 20)
    a.update(kw)
    with pytest.raises(abi.HprmsError, match=msg):
        abi.grad_norm(a["norm"], a["ptrs"], a["dtypes"], a["counts"], a["ws"], a["ws_size"])


def test_clip_abi_refuses():
    call = lambda od=(0,), limit=1.0, out=0x3000: abi.clip_grad_norm(  # noqa: E731
        0x100, [out], od, [0x1000], [0], [4], limit, 0x10000, 1 << 20)
    for kw, msg in ((dict(limit=-1.0), "max_norm"), (dict(limit=float("nan")), "max_norm"), (dict(od=(1,)), "output 0"),
                    (dict(out=0), "null"), (dict(out=0x3002, od=(2,)), "aligned")):
        with pytest.raises(abi.HprmsError, match=msg):
            call(**kw)
    L = abi.lib()
    assert L.hprms_grad_norm(0x100, None, None, None, 2, 0x10000, 1 << 20, None) == abi.HPRMS_E_INVALID
    assert L.hprms_grad_norm(0x100, None, None, None, -1, 0x10000, 1 << 20, None) == abi.HPRMS_E_INVALID
    n = (ctypes.c_int64 * 1)(4)
    assert L.hprms_clip_grad_norm(0x100, None, None, None, None, n, 1, 1.0, 0x10000, 1 << 20, None) == \
        abi.HPRMS_E_INVALID


def test_clip_abi_refuses_an_output_of_another_dtype_on_its_gradient():
    for dtype in (0, 1):
        with pytest.raises(abi.HprmsError, match="output 1 lies on its gradient"):
            abi.clip_grad_norm(0x100, [0x3000, 0x1000], [2, 2], [0x2000, 0x1000], [dtype] * 2, [4, 4], 1.0, 0x10000,
                               1 << 20)
