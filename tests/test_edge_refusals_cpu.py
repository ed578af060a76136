"""What the block-edge, 8-bit linear and log probability operators refuse, on the
CPU: the torch layer's checks with meta tensors and the C ABI's with addresses
that are never read."""
import pytest
import torch

from hp_rms_norm_amd import abi, ops

BF, F16, F32, I8, I64 = torch.bfloat16, torch.float16, torch.float32, torch.int8, torch.int64


def t(*shape, dtype=BF):
    return torch.empty(shape, dtype=dtype, device="meta")


def pick(kw, **defaults):
    return [kw[k] if k in kw else v for k, v in defaults.items()]


def edge(**kw):
    out, res, x, s, p, w, gate = pick(kw, out=t(2, 3, 64), residual_out=t(2, 3, 64), input=t(2, 3, 64),
                                      residual=t(2, 3, 64), post_weight=t(64), weight=t(64), gate=None)
    return ops.norm_add_rms_norm_out(out, res, x, s, p, w, 1e-6, gate=gate)


def edge8(**kw):
    out, scale, res, x = pick(kw, out=t(2, 3, 64, dtype=I8), scale=t(2, 3, 1, dtype=F32), residual_out=t(2, 3, 64),
                              input=t(2, 3, 64))
    return ops.norm_add_rms_norm_int8_out(out, scale, res, x, t(2, 3, 64), t(64), t(64), 1e-6)


def test_edge_accepts():
    for gate in (None, t(64), t(2, 1, 64), t(2, 3, 64), t(1, 1, 64)):
        assert edge(gate=gate) is None
    assert edge(post_weight=None) is None
    assert edge8() is None and edge8(scale=t(6, dtype=F32)) is None
    out, res = ops.norm_add_rms_norm(t(4, 64), t(4, 64), None, t(64), 1e-6)
    assert out.shape == res.shape == (4, 64)
    q, scale, res = ops.norm_add_rms_norm_int8(t(2, 3, 64), t(2, 3, 64), t(64), t(64), 1e-6)
    assert q.dtype == I8 and scale.shape == (2, 3, 1) and res.dtype == BF
    q, scale = ops.fused_add_rms_norm_int8(t(4, 64, dtype=F16), t(4, 64, dtype=F16), t(64, dtype=F16), 1e-6)
    assert q.shape == (4, 64) and scale.shape == (4, 1)
    got = ops.norm_add_rms_norm_backward(t(2, 3, 64), t(2, 3, 64), t(2, 3, 64), t(64), t(64), 1e-6, gate=t(2, 1, 64))
    assert [v.shape for v in got] == [(2, 3, 64), (2, 3, 64), (64,), (64,), (2, 1, 64)]
    got = ops.norm_add_rms_norm_backward(t(4, 64), t(4, 64), t(4, 64), None, t(64), 1e-6)
    assert got[2] is None and got[4] is None
    # gradients as the engine hands them on
    ops.norm_add_rms_norm_backward(t(1, 1).expand(4, 64), t(4, 64), t(4, 64), None, t(64), 1e-6,
                                   dresidual=t(64, 4).t())


@pytest.mark.parametrize("kw,msg", [
    (dict(input=t(64)), r"input.dim\(\) >= 2"),
    (dict(weight=t(1, 64)), r"weight.dim\(\) == 1"),
    (dict(weight=t(32)), r"input.size\(-1\) == hidden_dim"),
    (dict(weight=t(64, dtype=F16)), r"weight.dtype\(\) == input.dtype\(\)"),
    (dict(post_weight=t(63)), "post_weight must be shaped like weight"),
    (dict(post_weight=t(128)[::2]), "weights must be contiguous"),
    (dict(post_weight=t(64, dtype=F32)), r"weight.dtype\(\) == input.dtype\(\)"),
    (dict(residual=t(3, 2, 64)), "residual must be shaped like input"),
    (dict(residual=t(2, 3, 64, dtype=F16)), r"residual.dtype\(\) == input.dtype\(\)"),
    (dict(residual=t(2, 3, 128)[..., ::2]), "rows must be contiguous"),
    (dict(out=t(2, 3, 63)), "out must be shaped like input"),
    (dict(out=t(2, 3, 64, dtype=I8)), r"out.dtype\(\) must be"),
    (dict(residual_out=t(2, 3, 64, dtype=F32)), r"residual_out.dtype\(\) must be"),
    (dict(out=t(1, 1, 64).expand(2, 3, 64)), "overlap"),
    (dict(gate=t(3, 64)), r"gate.dim\(\) must be"),
    (dict(gate=t(32)), r"gate.size\(-1\) == hidden_dim"),
    (dict(gate=t(2, 3, 1)), r"gate.size\(-1\) == hidden_dim"),
    (dict(gate=t(1, 3, 64)), "leading sizes"),
    (dict(gate=t(2, 2, 64)), "leading sizes"),
    (dict(gate=t(64, dtype=F32)), r"gate.dtype\(\) == input.dtype\(\)"),
    (dict(gate=t(2, 1, 128)[..., ::2]), r"gate.stride\(-1\) == 1"),
    (dict(input=t(2, 3, 64, dtype=F32), residual=t(2, 3, 64, dtype=F32)), "dtype must be kFloat16 or kBFloat16"),
])
def test_edge_refuses(kw, msg):
    with pytest.raises(RuntimeError, match=msg):
        edge(**kw)


@pytest.mark.parametrize("kw,msg", [
    (dict(out=t(2, 3, 64)), r"out.dtype\(\) must be"),
    (dict(scale=t(5, dtype=F32)), "number of rows"),
    (dict(scale=t(2, 3, 1)), r"scale.dtype\(\) == float32"),
    (dict(scale=t(12, dtype=F32)[::2]), "scale must be contiguous"),
])
def test_edge8_refuses(kw, msg):
    with pytest.raises(RuntimeError, match=msg):
        edge8(**kw)


def edge_backward(**kw):
    a = pick(kw, dinput=t(2, 3, 64), dresidual_in=t(2, 3, 64), dpost_weight=t(64), dweight=t(64),
             dgate=t(2, 1, 64), dout=t(2, 3, 64), input=t(2, 3, 64), residual=t(2, 3, 64), post_weight=t(64),
             weight=t(64))
    gate, dres = pick(kw, gate=t(2, 1, 64), dresidual=None)
    return ops.norm_add_rms_norm_backward_out(*a, 1e-6, gate, 1.0, dres)


@pytest.mark.parametrize("kw,msg", [
    (dict(dinput=t(2, 3, 32)), "dinput must be shaped like input"),
    (dict(dresidual_in=t(2, 3, 64, dtype=F32)), r"dresidual_in.dtype\(\) must be"),
    (dict(dout=t(6, 64)), "dout must be shaped like input"),
    (dict(dresidual=t(2, 3, 64, dtype=F16)), r"dresidual.dtype\(\) must be"),
    (dict(dweight=t(32)), "must be shaped like weight"),
    (dict(dpost_weight=t(64, dtype=F16)), r"dweight.dtype\(\) must be"),
    (dict(dpost_weight=None), "dpost_weight must come with post_weight"),
    (dict(post_weight=None), "dpost_weight must come with post_weight"),
    (dict(dgate=None), "dgate must come with gate"),
    (dict(gate=None), "dgate must come with gate"),
    (dict(dgate=t(64)), "dgate must be shaped like gate"),
    (dict(dgate=t(2, 1, 64, dtype=F32)), r"gate.dtype\(\) == input.dtype\(\)"),
])
def test_edge_backward_refuses(kw, msg):
    assert edge_backward() is None and edge_backward(dweight=t(64, dtype=F32)) is None
    with pytest.raises(RuntimeError, match=msg):
        edge_backward(**kw)


def linear(**kw):
    out, x, s, w, ws, b = pick(kw, out=t(2, 3, 40), input=t(2, 3, 64, dtype=I8), scale=t(2, 3, 1, dtype=F32),
                               weight=t(40, 64, dtype=I8), weight_scale=t(40, dtype=F32), bias=None)
    return ops.int8_linear_out(out, x, s, w, ws, bias=b)


def test_linear_accepts():
    assert linear() is None and linear(bias=t(40)) is None and linear(weight_scale=t(40, 1, dtype=F32)) is None
    out = ops.int8_linear(t(5, 64, dtype=I8), t(5, dtype=F32), t(7, 64, dtype=I8), t(7, dtype=F32), dtype=F16)
    assert out.shape == (5, 7) and out.dtype == F16


@pytest.mark.parametrize("kw,msg", [
    (dict(input=t(64, dtype=I8)), r"input.dim\(\) >= 2"),
    (dict(weight=t(64, dtype=I8)), r"weight.dim\(\) == 2"),
    (dict(input=t(2, 3, 64)), "must be int8"),
    (dict(weight=t(40, 64, dtype=torch.uint8)), "must be int8"),
    (dict(weight=t(40, 63, dtype=I8)), r"input.size\(-1\) == weight.size\(1\)"),
    (dict(weight=t(64, 40, dtype=I8).t()), "rows must be contiguous"),
    (dict(out=t(2, 3, 41)), "one row of"),
    (dict(out=t(6, 40)), "one row of"),
    (dict(out=t(2, 3, 40, dtype=F32)), "dtype must be kFloat16 or kBFloat16"),
    (dict(scale=t(5, dtype=F32)), "one contiguous element per row"),
    (dict(scale=t(2, 3, 1)), "must be float32"),
    (dict(weight_scale=t(41, dtype=F32)), "one contiguous element per row of weight"),
    (dict(weight_scale=t(80, dtype=F32)[::2]), "one contiguous element per row of weight"),
    (dict(bias=t(39)), "bias must hold"),
    (dict(bias=t(40, dtype=F16)), r"bias.dtype\(\) == out.dtype\(\)"),
])
def test_linear_refuses(kw, msg):
    with pytest.raises(RuntimeError, match=msg):
        linear(**kw)


def log_probs(**kw):
    a = pick(kw, log_prob=t(4, dtype=F32), entropy=t(4, dtype=F32), lse=t(4, dtype=F32),
             top_log_prob=t(4, 5, dtype=F32), top_index=t(4, 5, dtype=I64), logits=t(4, 100), tokens=t(4, dtype=I64))
    return ops.token_log_probs_out(*a)


def test_log_probs_accept():
    assert log_probs() is None and log_probs(logits=t(4, 100, dtype=F32)) is None
    got = ops.token_log_probs(t(2, 3, 50, dtype=F16), t(2, 3, dtype=I64), top=2)
    assert [v.shape for v in got] == [(2, 3)] * 3 + [(2, 3, 2)] * 2 and got[4].dtype == I64
    d = ops.token_log_probs_backward(t(1, dtype=F32), t(4, 50), t(4, dtype=I64), t(4, dtype=F32))
    assert d.shape == (4, 50) and d.dtype == BF


@pytest.mark.parametrize("kw,msg", [
    (dict(logits=t(100)), r"logits.dim\(\) >= 2"),
    (dict(logits=t(4, 100, dtype=torch.float64)), "bfloat16, float16 or float32"),
    (dict(logits=t(100, 4).t()), r"logits.stride\(-1\) == 1"),
    (dict(logits=t(4, 0)), "at least one element"),
    (dict(logits=t(1, 100).expand(4, 100)), "overlap"),
    (dict(logits=t(4, 4), tokens=t(4, dtype=I64)), "no more than the vocabulary"),
    (dict(tokens=t(4, dtype=torch.int32)), r"tokens.dtype\(\) == int64"),
    (dict(tokens=t(5, dtype=I64)), "tokens must have one element per row"),
    (dict(tokens=t(8, dtype=I64)[::2]), "tokens must be contiguous"),
    (dict(lse=t(4)), "must be float32"),
    (dict(entropy=t(4, 1, dtype=F32)), "must be shaped like tokens"),
    (dict(top_index=t(4, 5, dtype=torch.int32)), r"top_index.dtype\(\) == int64"),
    (dict(top_log_prob=t(4, 6, dtype=F32)), "must be shaped like tokens"),
    (dict(top_log_prob=t(4, 65, dtype=F32), top_index=t(4, 65, dtype=I64)), "at most 64"),
])
def test_log_probs_refuse(kw, msg):
    with pytest.raises(RuntimeError, match=msg):
        log_probs(**kw)


def log_probs_backward(**kw):
    d, g, z, ids, lse, entropy, gh = pick(kw, dlogits=t(4, 100), dlog_prob=t(4, dtype=F32), logits=t(4, 100),
                                          tokens=t(4, dtype=I64), lse=t(4, dtype=F32), entropy=t(4, dtype=F32),
                                          dentropy=t(4, dtype=F32))
    return ops.token_log_probs_backward_out(d, g, z, ids, lse, entropy, gh)


@pytest.mark.parametrize("kw,msg", [
    (dict(dlogits=t(4, 101)), "dlogits must be shaped like logits"),
    (dict(dlogits=t(4, 100, dtype=F32)), r"dlogits.dtype\(\) == logits.dtype\(\)"),
    (dict(dlog_prob=t(4)), "must be float32"),
    (dict(dentropy=t(5, dtype=F32)), "must be shaped like tokens"),
    (dict(entropy=None), "dentropy needs"),
    (dict(lse=t(8, dtype=F32)[::2]), "must be contiguous"),
])
def test_log_probs_backward_refuse(kw, msg):
    assert log_probs_backward() is None and log_probs_backward(entropy=None, dentropy=None) is None
    with pytest.raises(RuntimeError, match=msg):
        log_probs_backward(**kw)


def test_no_cpu_fallback():
    x, w = torch.zeros(2, 8, dtype=BF), torch.ones(8, dtype=BF)
    q, s = torch.zeros(2, 8, dtype=I8), torch.ones(2)
    z, ids = torch.zeros(2, 8), torch.zeros(2, dtype=I64)
    for call in (lambda: ops.norm_add_rms_norm(x, x, w, w, 1e-6), lambda: ops.norm_add_rms_norm_int8(x, x, w, w, 1e-6),
                 lambda: ops.fused_add_rms_norm_int8(x, x, w, 1e-6),
                 lambda: ops.norm_add_rms_norm_backward(x, x, x, w, w, 1e-6), lambda: ops.int8_linear(q, s, q, s),
                 lambda: ops.token_log_probs(z, ids), lambda: ops.token_log_probs_backward(s, z, ids, s)):
        with pytest.raises(NotImplementedError):
            call()


# ---- the C ABI ---------------------------------------------------------------------------
def test_workspace_sizes():
    n = abi.norm_add_rmsnorm_backward_workspace
    assert n(0, 4096, 0) == 0 and n(1, 4096, 0) == 2 * 4096 * 4
    assert n(8192, 4096, 1) <= 3 * 1024 * 4096 * 4 and n(8192, 4096, 8192) == n(8192, 4096, 0)
    i = abi.int8_linear_workspace
    assert i(0, 64, 64) == 0 and i(5, 64, 64) == 0 and i(5, 63, 64, input_stride=64, weight_stride=64) >= 69 * 64
    assert i(5, 64, 64, weight_ptr=8) >= 64 * 64 and i(5, 64, 64, input_stride=72) >= 5 * 64
    p = abi.token_log_probs_workspace
    assert p(0, 100, 5, 0) == 0 and p(1, 200000, 0, 0) >= 16 and p(1 << 30, 131072, 64, 2) <= (1 << 26) + 4096
    for call in (lambda: n(-1, 64, 0), lambda: n(1, 0, 0), lambda: n(1, (1 << 24) + 1, 0), lambda: n(6, 64, 4),
                 lambda: n(6, 64, -1), lambda: n(1 << 31, 64, 0), lambda: i(-1, 64, 64), lambda: i(1, 0, 64),
                 lambda: i(1, 64, 0), lambda: i(1, 131072, 64), lambda: i((1 << 24) + 1, 64, 64),
                 lambda: i(1 << 24, 64, 1 << 14), lambda: p(-1, 64, 0, 0), lambda: p(1, 0, 0, 0),
                 lambda: p(1, (1 << 20) + 1, 0, 0), lambda: p(1, 64, 65, 0), lambda: p(1, 5, 6, 0),
                 lambda: p(1, 64, -1, 0), lambda: p(1, 64, 0, 3)):
        with pytest.raises(abi.HprmsError):
            call()


def edge_abi(fn="hprms_norm_add_rmsnorm", **kw):
    a = dict(out=0x1000, res_out=0x2000, input=0x3000, post=0x4000, weight=0x5000, residual=0x6000, gate=0, rows=4,
             hidden=64, rpg=1, s0=64, s1=64, s2=64, s3=64, s4=64, dtype=0, scale=1.0, eps=1e-6)
    if fn.endswith("int8"):
        a = dict(out=a.pop("out"), sc=0x7000, **a)
    a.update(kw)
    return getattr(abi.lib(), fn)(*a.values(), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=2), "dtype"), (dict(rows=-1), "rows"), (dict(hidden=0), "hidden"), (dict(s0=63), "strides"),
    (dict(s1=1), "strides"), (dict(s2=63), "strides"), (dict(s3=63), "strides"), (dict(gate=0x8000, s4=3), "strides"),
    (dict(gate=0x8000, rpg=0), "rows_per_gate"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(scale=float("inf")), "residual_scale"), (dict(out=0), "null"), (dict(res_out=0), "null"),
    (dict(input=0), "null"), (dict(weight=0), "null"), (dict(residual=0), "null"), (dict(post=0x4001), "aligned"),
    (dict(gate=0x8001), "aligned"), (dict(out=0x2000), "alias"), (dict(out=0x6000), "alias"),
    (dict(res_out=0x3000), "alias"),
])
def test_edge_abi_refuses(kw, msg):
    assert edge_abi(**kw) == abi.HPRMS_E_INVALID
    assert msg in abi.last_error()


def test_edge_abi_ranges_and_no_rows():
    assert edge_abi(hidden=(1 << 24) + 8, **{f"s{i}": 1 << 25 for i in range(5)}) == abi.HPRMS_E_RANGE
    assert edge_abi(rows=1 << 16, s2=1 << 40) == abi.HPRMS_E_RANGE
    assert edge_abi(rows=1 << 31) == abi.HPRMS_E_RANGE
    assert edge_abi(rows=0, out=0, res_out=0, input=0, weight=0, residual=0) == abi.HPRMS_OK
    assert edge_abi("hprms_norm_add_rmsnorm_int8", sc=0) == abi.HPRMS_E_INVALID and "null" in abi.last_error()
    assert edge_abi("hprms_norm_add_rmsnorm_int8", sc=0x7002) == abi.HPRMS_E_INVALID and "aligned" in abi.last_error()
    assert edge_abi("hprms_norm_add_rmsnorm_int8", out=0x3000) == abi.HPRMS_E_INVALID and "alias" in abi.last_error()


def edge_backward_abi(**kw):
    a = dict(di=0x1000, dr=0x2000, dp=0x3000, dw=0x4000, dg=0, dout=0x5000, dres=0, input=0x6000, residual=0x7000,
             post=0x8000, weight=0x9000, gate=0, ws=0x10000, ws_size=1 << 30, rows=4, hidden=64, gates=0, s0=64, s1=64,
             s2=64, s3=64, s4=64, s5=64, s6=64, s7=64, dtype=0, dpt=0, dwt=0, scale=1.0, eps=1e-6)
    a.update(kw)
    return abi.lib().hprms_norm_add_rmsnorm_backward(*a.values(), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=2), "dtype"), (dict(dwt=1), "dweight_dtype"), (dict(dpt=1), "dpost_weight_dtype"),
    (dict(rows=-1), "rows"), (dict(hidden=0), "hidden"), (dict(s0=63), "strides"), (dict(s1=63), "strides"),
    (dict(s3=63), "strides"), (dict(dres=0xa000, s4=2), "strides"), (dict(s5=63), "strides"),
    (dict(s6=63), "strides"), (dict(gate=0xb000, dg=0xc000, gates=2, s7=1), "strides"),
    (dict(gate=0xb000, dg=0xc000, gates=3), "divide"), (dict(gate=0xb000, dg=0xc000, gates=0), "gate_rows"),
    (dict(gate=0xb000, gates=2), "null"), (dict(eps=-1.0), "eps"), (dict(scale=float("nan")), "residual_scale"),
    (dict(dw=0), "null"), (dict(dp=0), "null"), (dict(di=0), "null"), (dict(dr=0), "null"), (dict(dout=0), "null"),
    (dict(residual=0), "null"), (dict(input=0x6001), "aligned"), (dict(dwt=2, dw=0x4002), "aligned"),
    (dict(dr=0x1000), "alias"), (dict(ws=0), "workspace"), (dict(ws=0x10008), "workspace"),
    (dict(ws_size=100), "workspace"),
])
def test_edge_backward_abi_refuses(kw, msg):
    assert edge_backward_abi(**kw) == abi.HPRMS_E_INVALID
    assert msg in abi.last_error()


def linear_abi(**kw):
    a = dict(out=0x1000, input=0x2000, scale=0x3000, weight=0x4000, wscale=0x5000, bias=0, ws=0, ws_size=0, rows=4,
             inner=64, outer=40, s0=40, s1=64, s2=64, dtype=0)
    a.update(kw)
    return abi.lib().hprms_int8_linear(*a.values(), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=2), "dtype"), (dict(rows=-1), "rows"), (dict(inner=0), "inner"), (dict(outer=0), "outer"),
    (dict(s0=39), "strides"), (dict(s1=63), "strides"), (dict(s2=63), "strides"), (dict(out=0), "null"),
    (dict(input=0), "null"), (dict(scale=0), "null"), (dict(weight=0), "null"), (dict(wscale=0), "null"),
    (dict(out=0x1001), "aligned"), (dict(scale=0x3002), "aligned"), (dict(wscale=0x5001), "aligned"),
    (dict(bias=0x6001), "aligned"), (dict(weight=0x4008), "workspace"), (dict(s1=65), "workspace"),
    (dict(inner=63), "workspace"), (dict(weight=0x4008, ws=0x10010, ws_size=1 << 20), "workspace"),
    (dict(weight=0x4008, ws=0x10000, ws_size=100), "workspace"),
])
def test_linear_abi_refuses(kw, msg):
    assert linear_abi(**kw) == abi.HPRMS_E_INVALID
    assert msg in abi.last_error()


def test_linear_abi_ranges_and_no_rows():
    assert linear_abi(inner=131072, s1=131072, s2=131072) == abi.HPRMS_E_RANGE
    assert linear_abi(rows=1 << 20, s1=1 << 40) == abi.HPRMS_E_RANGE
    assert linear_abi(rows=0, out=0, input=0, scale=0, weight=0, wscale=0) == abi.HPRMS_OK


def log_probs_abi(**kw):
    a = dict(lp=0x1000, h=0x2000, lse=0x3000, tl=0x4000, ti=0x5000, logits=0x6000, tokens=0x7000, ws=0x10000,
             ws_size=1 << 30, rows=4, vocab=100, top=5, stride=100, ignore=-100, dtype=0)
    a.update(kw)
    return abi.lib().hprms_token_log_probs(*a.values(), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=3), "dtype"), (dict(rows=-1), "rows"), (dict(vocab=0), "vocab"), (dict(top=65), "top"),
    (dict(vocab=4, stride=4), "top"), (dict(stride=99), "strides"), (dict(lp=0), "null"), (dict(h=0), "null"),
    (dict(lse=0), "null"), (dict(tl=0), "null"), (dict(ti=0), "null"), (dict(logits=0), "null"),
    (dict(tokens=0), "null"), (dict(dtype=2, logits=0x6002), "aligned"), (dict(tokens=0x7004), "aligned"),
    (dict(ti=0x5004), "aligned"), (dict(ws=0, vocab=200000, stride=200000), "workspace"),
    (dict(ws=0x10008, vocab=200000, stride=200000), "workspace"),
    (dict(ws_size=100, vocab=200000, stride=200000), "workspace"),
])
def test_log_probs_abi_refuses(kw, msg):
    assert log_probs_abi(**kw) == abi.HPRMS_E_INVALID
    assert msg in abi.last_error()


def log_probs_backward_abi(**kw):
    a = dict(d=0x1000, g=0x2000, gh=0x3000, logits=0x4000, tokens=0x5000, lse=0x6000, h=0x7000, rows=4, vocab=100,
             s0=100, s1=100, ignore=-100, dtype=0)
    a.update(kw)
    return abi.lib().hprms_token_log_probs_backward(*a.values(), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=-1), "dtype"), (dict(rows=-1), "rows"), (dict(s0=99), "strides"), (dict(s1=99), "strides"),
    (dict(d=0), "null"), (dict(g=0), "null"), (dict(lse=0), "null"), (dict(h=0), "null"), (dict(d=0x1001), "aligned"),
    (dict(gh=0x3002), "aligned"),
])
def test_log_probs_backward_abi_refuses(kw, msg):
    assert log_probs_backward_abi(**kw) == abi.HPRMS_E_INVALID
    assert msg in abi.last_error()


def test_log_probs_abi_ranges_and_no_rows():
    assert log_probs_abi(vocab=(1 << 20) + 1, stride=1 << 21) == abi.HPRMS_E_RANGE
    assert log_probs_abi(rows=1 << 20, stride=1 << 40) == abi.HPRMS_E_RANGE
    assert log_probs_backward_abi(rows=1 << 20, s0=1 << 40) == abi.HPRMS_E_RANGE
    assert log_probs_abi(rows=0, lp=0, h=0, lse=0, tl=0, ti=0, logits=0, tokens=0, ws=0) == abi.HPRMS_OK
    assert log_probs_backward_abi(rows=0, d=0, g=0, logits=0, tokens=0, lse=0) == abi.HPRMS_OK


def test_in_place_with_other_strides():
    """A tensor in another's place has its row stride too: the rows of one would lie
    on others' of the other."""
    for kw in (dict(out=0x3000, s0=72), dict(res_out=0x6000, s1=72)):
        assert edge_abi(**kw) == abi.HPRMS_E_INVALID and "strides" in abi.last_error()
    assert edge_abi("hprms_norm_add_rmsnorm_int8", res_out=0x6000, s3=72) == abi.HPRMS_E_INVALID
    assert "strides" in abi.last_error()
    for out, stride in (("di", "s0"), ("dr", "s1")):
        for at in (0x5000, 0x6000, 0x7000, 0xa000):  # dout, input, residual, dresidual
            assert edge_backward_abi(dres=0xa000, **{out: at, stride: 72}) == abi.HPRMS_E_INVALID
            assert "equal row strides" in abi.last_error()
    assert edge_backward_abi(gate=0xb000, dg=0xb000, gates=4, s2=72) == abi.HPRMS_E_INVALID
    assert "equal row strides" in abi.last_error()
    assert log_probs_backward_abi(d=0x4000, s0=108) == abi.HPRMS_E_INVALID
    assert "equal row strides" in abi.last_error()


@pytest.mark.parametrize("gates", [1, 2])
def test_dgate_in_place_of_a_shared_gate(gates):
    assert edge_backward_abi(gate=0xb000, dg=0xb000, gates=gates) == abi.HPRMS_E_INVALID
    assert "rows share" in abi.last_error()
