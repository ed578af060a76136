"""The calls by which the speed of the training operators is judged.

Around the fused norm a training step needs three things: the norm's gradient,
the loss of the normed rows under a vocabulary projection with its gradient,
and the norm of all gradients with clipping by it.  ``listed()`` gives the
named cases, ``draw()`` more of the same ranges: 1 to 8192 rows of 64 to 16384
elements (per-head norms up to 262144 rows), vocabularies of 1000 to 131072,
lists of 1 to 56 gradients of up to 2^29 elements together, bfloat16, float16
and (gradients) float32.
"""
import math

import torch

own = False  # run() makes the framework's calls where this is true, else the plain form

EPS = 1e-6
IGNORE = -100
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

# Ops and the entry point each stands for:
#   norm_backward  rms_norm_backward: the gradient of rms_norm and of the fused
#                  add + norm (`residual`: the residual stream's own gradient
#                  joins the sum)
#   loss           linear_cross_entropy: per-row losses and log-sum-exps
#   loss_train     linear_cross_entropy, then linear_cross_entropy_backward
#   clip           clip_grad_norm_out: clipped copies of the gradients
#   clip_          clip_grad_norm_, in place, on gradients whose norm is below
#                  the limit, as most steps of a training run have them (so
#                  each pass meets the same values)
#   norm_of_grads  grad_norm


def listed():
    return [
        # a fine-tuning micro-batch's last tokens: launch and host cost
        dict(name="norm_backward_few", op="norm_backward", rows=32, hidden=4096, dtype="bf16", residual=True),
        # one layer's norm in a pre-training step of 8192 tokens
        dict(name="norm_backward", op="norm_backward", rows=8192, hidden=4096, dtype="bf16", residual=True),
        # an odd width in float16, ragged rows, the first norm of a stack (no residual gradient)
        dict(name="norm_backward_odd", op="norm_backward", rows=2999, hidden=4097, dtype="fp16", residual=False),
        # per-head norm of the queries: 4096 tokens x 32 heads of 128
        dict(name="norm_backward_head", op="norm_backward", rows=131072, hidden=128, dtype="bf16", residual=False),
        # the log-probability of one sampled token
        dict(name="loss_one", op="loss", rows=1, hidden=4096, vocab=131072, dtype="bf16", ignored=0.0),
        # scoring a ragged chunk, odd vocabulary
        dict(name="loss_ragged", op="loss", rows=777, hidden=5120, vocab=50001, dtype="fp16", ignored=0.1),
        # a fine-tuning micro-batch: half of the rows are prompt tokens, which carry no loss
        dict(name="loss_train_prompts", op="loss_train", rows=1000, hidden=2048, vocab=32000, dtype="bf16", ignored=0.5),
        # a pre-training micro-batch
        dict(name="loss_train", op="loss_train", rows=4096, hidden=4096, vocab=131072, dtype="bf16", ignored=0.0),
        # low-rank adapters' gradients: 56 small tensors
        dict(name="clip_adapters", op="clip", layers=28, width=0, rank=16, dtype="bf16"),
        # 4 layers of a 4096-wide model, bfloat16 gradients
        dict(name="clip_layers", op="clip", layers=4, width=4096, rank=0, dtype="bf16"),
        # 1 layer's float32 gradients below the limit, in place
        dict(name="clip_below", op="clip_", layers=1, width=4096, rank=0, dtype="fp32"),
        # monitoring the norm of a narrow model's gradients
        dict(name="norm_of_grads", op="norm_of_grads", layers=6, width=1000, rank=0, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm_backward"] * 4 + ["loss"] * 3 + ["loss_train"] * 4 + ["clip", "clip", "clip_", "norm_of_grads"])
    case = dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if op == "norm_backward":
        case["residual"] = rng.random() < 0.5
        if rng.random() < 0.2:  # per-head rows
            case.update(rows=_log_int(rng, 64, 262144), hidden=rng.choice([64, 96, 128, 192, 256]))
        else:
            hidden = 128 * _log_int(rng, 1, 128) if rng.random() < 0.7 else _log_int(rng, 64, 16384)
            case.update(rows=_log_int(rng, 1, min(8192, 8192 * 4096 // hidden)), hidden=hidden)
    elif op in ("loss", "loss_train"):
        hidden = 64 * _log_int(rng, 4, 128) if rng.random() < 0.8 else _log_int(rng, 200, 5000)
        vocab = _log_int(rng, 1000, 131072)
        most = min(8192, 4096 * 4096 * 131072 // (hidden * vocab))
        case.update(rows=_log_int(rng, 1, most), hidden=hidden, vocab=vocab,
                    ignored=rng.choice([0.0, 0.0, 0.1, 0.5, 0.9]))
    else:
        case["dtype"] = rng.choice(["bf16", "fp16", "fp32"])
        if rng.random() < 0.3:
            case.update(layers=rng.randint(1, 28), width=0, rank=rng.randint(1, 64))
        else:
            case.update(layers=rng.randint(1, 6), width=_log_int(rng, 100, 3000), rank=0)
    return case


def _grad_shapes(case):
    """The shapes of a list of gradients: of `layers` pairs of low-rank
    adapters of a 4096-wide model, or of `layers` transformer layers of `width`."""
    if case["width"] == 0:
        return [s for _ in range(case["layers"]) for s in ((case["rank"], 4096), (4096, case["rank"]))]
    h, f = case["width"], case["width"] * 7 // 2
    layer = [(h,), (h, h), (h // 4, h), (h // 4, h), (h, h), (h,), (f, h), (f, h), (h, f)]
    return layer * case["layers"]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 29)


def prepare(case, seed):
    g, dtype, dev = _generator(seed), DTYPES[case["dtype"]], "cuda"
    state = {"case": dict(case)}
    if case["op"] == "norm_backward":
        shape = (case["rows"], case["hidden"])
        # the normed rows have the residual stream's few large channels
        x = torch.randn(shape, generator=g, device=dev)
        x *= torch.where(torch.rand(shape[1], generator=g, device=dev) < 0.01, 20.0, 1.0)
        state["input"] = x.to(dtype)
        state["weight"] = (1.0 + 0.1 * torch.randn(shape[1], generator=g, device=dev)).to(dtype)
        state["dout"] = torch.randn(shape, generator=g, device=dev).to(dtype)
        state["dresidual"] = torch.randn(shape, generator=g, device=dev).to(dtype) if case["residual"] else None
    elif case["op"] in ("loss", "loss_train"):
        rows, hidden, vocab = case["rows"], case["hidden"], case["vocab"]
        weight = torch.randn((vocab, hidden), generator=g, device=dev, dtype=dtype) * 0.02
        target = torch.randint(0, vocab, (rows,), generator=g, device=dev)
        # normed rows that know their target more or less well
        aim = weight[target].float()
        aim *= 12.0 * torch.rand((rows, 1), generator=g, device=dev) / aim.norm(dim=1, keepdim=True).square()
        state["hidden"] = (torch.randn((rows, hidden), generator=g, device=dev) + aim).to(dtype)
        state["weight"] = weight
        keep = torch.rand(rows, generator=g, device=dev) >= case["ignored"]
        keep[0] = True
        state["target"] = torch.where(keep, target, IGNORE)
        # the gradient of the mean over the kept rows, in float16 with a loss scale
        scale = 1024.0 if case["dtype"] == "fp16" else 1.0
        state["dloss"] = (scale / keep.sum()).float().expand(rows).contiguous()
    else:
        state["grads"] = [torch.randn(s, generator=g, device=dev, dtype=dtype) * 1e-2 for s in _grad_shapes(case)]
        count = sum(t.numel() for t in state["grads"])
        # a limit below the norm, or above it
        state["max_norm"] = 1e-2 * math.sqrt(count) * (0.37 if case["op"] == "clip" else 2.0)
        if case["op"] == "clip":
            state["outs"] = [torch.empty_like(t) for t in state["grads"]]
    return state


def _norm_backward_plain(s):
    x, w, dout = s["input"].float(), s["weight"].float(), s["dout"].float()
    rstd = torch.rsqrt(x.square().mean(dim=1, keepdim=True) + EPS)
    n = x * rstd
    dn = dout * w
    dx = rstd * (dn - n * (dn * n).mean(dim=1, keepdim=True))
    if s["dresidual"] is not None:
        dx = dx + s["dresidual"].float()
    return dx.to(s["input"].dtype), (dout * n).sum(dim=0).to(s["weight"].dtype)


def _loss_plain(s):
    """(loss, lse, logits): both zero in rows without a target."""
    logits = s["hidden"].float() @ s["weight"].float().t()
    top = logits.amax(dim=1)
    lse = top + torch.log(torch.exp(logits - top[:, None]).sum(dim=1))
    kept = s["target"] != IGNORE
    at = torch.where(kept, s["target"], 0)
    loss = lse - logits.gather(1, at[:, None])[:, 0]
    return torch.where(kept, loss, 0.0), torch.where(kept, lse, 0.0), logits


def _loss_backward_plain(s, lse, logits):
    kept = (s["target"] != IGNORE)[:, None]
    at = torch.where(kept, s["target"][:, None], 0)
    p = torch.exp(logits - lse[:, None])
    p = torch.where(kept, p.scatter_add(1, at, torch.full_like(lse, -1.0)[:, None]) * s["dloss"][:, None], 0.0)
    dhidden = p @ s["weight"].float()
    dweight = p.t() @ s["hidden"].float()
    return dhidden.to(s["hidden"].dtype), dweight.to(s["weight"].dtype)


def _norm_plain(grads):
    return torch.stack([t.float().square().sum(dtype=torch.float64) for t in grads]).sum().sqrt()


def _plain(s):
    op = s["case"]["op"]
    if op == "norm_backward":
        dx, dw = _norm_backward_plain(s)
        return {"dinput": dx, "dweight": dw}
    if op == "loss":
        loss, lse, _ = _loss_plain(s)
        return {"loss": loss, "lse": lse}
    if op == "loss_train":
        loss, lse, logits = _loss_plain(s)
        dhidden, dweight = _loss_backward_plain(s, lse, logits)
        return {"loss": loss, "lse": lse, "dhidden": dhidden, "dweight": dweight}
    norm = _norm_plain(s["grads"])
    if op == "norm_of_grads":
        return {"norm": norm.float()}
    factor = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0).float()
    outs = s["outs"] if op == "clip" else s["grads"]
    return {"norm": norm.float(), "grads": [o.copy_(t.float() * factor) for o, t in zip(outs, s["grads"])]}


def _own(s):
    import hp_rms_norm_amd as hp
    op = s["case"]["op"]
    if op == "norm_backward":
        dx, dw = hp.rms_norm_backward(s["dout"], s["input"], s["weight"], EPS, dresidual=s["dresidual"])
        return {"dinput": dx, "dweight": dw}
    if op == "loss":
        loss, lse = hp.linear_cross_entropy(s["hidden"], s["weight"], s["target"], ignore_index=IGNORE)
        return {"loss": loss, "lse": lse}
    if op == "loss_train":
        loss, lse = hp.linear_cross_entropy(s["hidden"], s["weight"], s["target"], ignore_index=IGNORE)
        dhidden, dweight = hp.linear_cross_entropy_backward(s["dloss"], s["hidden"], s["weight"], s["target"], lse,
                                                            ignore_index=IGNORE)
        return {"loss": loss, "lse": lse, "dhidden": dhidden, "dweight": dweight}
    if op == "norm_of_grads":
        return {"norm": hp.grad_norm(s["grads"])}
    if op == "clip":
        return {"norm": hp.clip_grad_norm_out(s["outs"], s["grads"], s["max_norm"]), "grads": s["outs"]}
    return {"norm": hp.clip_grad_norm_(s["grads"], s["max_norm"]), "grads": s["grads"]}


def run(state):
    return _own(state) if own else _plain(state)


def exact(case, seed):
    """The definitions in 64 bits: the norm's gradient through the Jacobian of
    x / sqrt(mean(x^2) + eps), the loss through log_softmax-free sums per block
    of rows."""
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm_backward":
        x, gw = s["input"].double(), s["dout"].double() * s["weight"].double()
        ms = (x * x).sum(dim=1, keepdim=True) / x.shape[1] + EPS
        dx = gw / ms.sqrt() - x * ((gw * x).sum(dim=1, keepdim=True) / (x.shape[1] * ms * ms.sqrt()))
        if s["dresidual"] is not None:
            dx += s["dresidual"].double()
        return {"dinput": dx, "dweight": (s["dout"].double() * x / ms.sqrt()).sum(dim=0)}
    if op in ("loss", "loss_train"):
        w = s["weight"].double()
        rows = case["rows"]
        loss = torch.zeros(rows, dtype=torch.float64, device=w.device)
        lse = torch.zeros_like(loss)
        dhidden = torch.zeros((rows, case["hidden"]), dtype=torch.float64, device=w.device)
        dweight = torch.zeros_like(w) if op == "loss_train" else None
        kept = (s["target"] != IGNORE).nonzero()[:, 0]
        for at in kept.split(1024):
            h, t = s["hidden"][at].double(), s["target"][at]
            z = h @ w.T
            shift = z.max(dim=1).values
            e = torch.exp(z - shift[:, None])
            total = e.sum(dim=1)
            lse[at] = shift + total.log()
            loss[at] = lse[at] - z[torch.arange(len(at), device=w.device), t]
            if op == "loss_train":
                d = e / total[:, None]
                d[torch.arange(len(at), device=w.device), t] -= 1.0
                d *= s["dloss"][at].double()[:, None]
                dhidden[at] = d @ w
                dweight += d.T @ h
        if op == "loss":
            return {"loss": loss, "lse": lse}
        return {"loss": loss, "lse": lse, "dhidden": dhidden, "dweight": dweight}
    total = math.sqrt(sum(float(t.double().pow(2).sum()) for t in s["grads"]))
    norm = torch.tensor(total, dtype=torch.float64)
    if op == "norm_of_grads":
        return {"norm": norm}
    factor = min(1.0, s["max_norm"] / (total + 1e-6))
    return {"norm": norm, "grads": [t.double() * factor for t in s["grads"]]}


def work(case):
    """Bytes: each input read once and each output written once (a clipped
    gradient is read for the norm and again for the product, which needs the
    norm of all).  Operations: of the matrix products, one multiplication and
    one addition a term; a gradient needs the logits' product again, unless
    they were kept, which the operator's purpose rules out."""
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm_backward":
        n, h = case["rows"] * case["hidden"], case["hidden"]
        return {"bytes": n * size * (4 if case["residual"] else 3) + 2 * h * size, "flops": 12 * n}
    if case["op"] in ("loss", "loss_train"):
        kept = max(1, round(case["rows"] * (1.0 - case["ignored"])))
        product = 2 * kept * case["hidden"] * case["vocab"]
        nbytes = (kept + case["vocab"]) * case["hidden"] * size + case["rows"] * 16
        if case["op"] == "loss":
            return {"bytes": nbytes, "flops": product}
        return {"bytes": 3 * nbytes, "flops": 4 * product}
    n = sum(math.prod(s) for s in _grad_shapes(case))
    return {"bytes": n * size * (3 if case["op"] == "clip" else 1), "flops": n * (3 if case["op"] == "clip" else 2)}
