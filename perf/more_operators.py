"""The calls by which the speed of the block-edge, 8-bit and scoring operators is judged.

From a block's output to the next product and, behind the last block, to the
answer's probabilities: the norms on both sides of a block joined with its gate
and the residual's scale (and their gradient), the product of 8-bit integer
rows and weights that takes the quantised rows, and the log probabilities of
given tokens with the entropy and the most likely alternatives (and their
gradient).  ``listed()`` gives the named cases, ``draw()`` more of the same
ranges: 1 to 8192 rows of 64 to 16384 elements, products of 1 to 8192 rows with
128 to 16384 features on both sides, vocabularies of 1000 to 131072.
"""
import math

import torch

own = False  # run() makes the framework's calls where this is true, else the plain form

EPS = 1e-6
IGNORE = -100
FLT_MIN = 2.0 ** -126
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

# Ops and the entry points each stands for:
#   norm_add           norm_add_rms_norm, or (out "int8") norm_add_rms_norm_int8
#   norm_add_backward  norm_add_rms_norm_backward
#   int8_linear        int8_linear
#   log_probs          token_log_probs
#   log_probs_train    token_log_probs, then token_log_probs_backward
#
# `gate`: none, one for each channel, for each sequence and channel (`groups`
# sequences of equal length), or for each element.  `post`: the block's output
# is normed before it is added.


def listed():
    return [
        # one new token at a block's edge while decoding: launch and host cost
        dict(name="norm_add_token", op="norm_add", rows=1, hidden=4096, dtype="bf16", gate="none", groups=1, post=True,
             scale=1.0, out="same"),
        # four conditioned sequences of 2048, each with a gate of its own
        dict(name="norm_add_gated", op="norm_add", rows=8192, hidden=4096, dtype="bf16", gate="sequence", groups=4,
             post=True, scale=0.5, out="same"),
        # a prompt's chunk on its way into an 8-bit product
        dict(name="norm_add_int8", op="norm_add", rows=4096, hidden=8192, dtype="bf16", gate="none", groups=1, post=True,
             scale=1.0, out="int8"),
        # an odd width in float16, ragged rows, a gate that is an activation, no norm of the block's output
        dict(name="norm_add_odd", op="norm_add", rows=1777, hidden=2999, dtype="fp16", gate="element", groups=1,
             post=False, scale=0.7, out="same"),
        # a pre-training step's block edge with a learned gate for each channel
        dict(name="norm_add_backward", op="norm_add_backward", rows=8192, hidden=4096, dtype="bf16", gate="channel",
             groups=1, post=True, scale=1.0, residual=True),
        # a fine-tuning micro-batch, odd in both sizes, gated element by element, nothing else reads the residual
        dict(name="norm_add_backward_odd", op="norm_add_backward", rows=1021, hidden=5003, dtype="fp16", gate="element",
             groups=1, post=True, scale=0.7, residual=False),
        # one new token through a feed-forward layer's first product: the weight's bytes
        dict(name="int8_linear_token", op="int8_linear", rows=1, inner=4096, outer=14336, dtype="bf16", bias=False),
        # a decoding batch through an attention layer's projection: a small weight
        dict(name="int8_linear_batch", op="int8_linear", rows=48, inner=4096, outer=4096, dtype="bf16", bias=True),
        # a prompt of 8192 tokens: the matrix cores
        dict(name="int8_linear", op="int8_linear", rows=8192, inner=4096, outer=14336, dtype="bf16", bias=False),
        # one decoding step's answers for 32 requests, some words forbidden, with their 20 most likely alternatives
        dict(name="log_probs_step", op="log_probs", rows=32, vocab=131072, dtype="fp32", top=20, masked=0.3, ignored=0.0,
             pad=0),
        # a prompt scored token by token, rows of an odd vocabulary in a padded buffer
        dict(name="log_probs_prompt", op="log_probs", rows=4096, vocab=50001, dtype="bf16", top=5, masked=0.0,
             ignored=0.1, pad=47),
        # a policy-gradient step with an entropy bonus
        dict(name="log_probs_train", op="log_probs_train", rows=4096, vocab=131072, dtype="bf16", top=0, masked=0.0,
             ignored=0.3, pad=0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm_add"] * 3 + ["norm_add_backward"] * 3 + ["int8_linear"] * 3 + ["log_probs"] * 2 +
                    ["log_probs_train"])
    case = dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if op in ("norm_add", "norm_add_backward"):
        hidden = 128 * _log_int(rng, 1, 128) if rng.random() < 0.7 else _log_int(rng, 64, 16384)
        gate = rng.choice(["none", "channel", "sequence", "element"])
        groups = _log_int(rng, 2, 64) if gate == "sequence" else 1
        rows = _log_int(rng, 1, min(8192, 8192 * 4096 // hidden) // groups) * groups
        case.update(rows=rows, hidden=hidden, gate=gate, groups=groups, post=rng.random() < 0.7,
                    scale=rng.choice([1.0, 0.25, 0.7, 1.4]))
        if op == "norm_add":
            case["out"] = rng.choice(["same", "int8"])
        else:
            case["residual"] = rng.random() < 0.7
    elif op == "int8_linear":
        sizes = [128 * _log_int(rng, 1, 128) if rng.random() < 0.8 else _log_int(rng, 100, 10000) for _ in range(2)]
        most = min(8192, 8192 * 4096 * 14336 // (sizes[0] * sizes[1]))
        case.update(rows=_log_int(rng, 1, most), inner=sizes[0], outer=sizes[1], bias=rng.random() < 0.4)
    else:
        case["dtype"] = rng.choice(["bf16", "fp16", "fp32"])
        vocab = _log_int(rng, 1000, 131072)
        size = 2 if case["dtype"] == "fp32" else 1
        case.update(rows=_log_int(rng, 1, min(8192, 2048 * 131072 // (vocab * size))), vocab=vocab,
                    top=rng.choice([0, 1, 5, 20]) if op == "log_probs" else 0,
                    masked=rng.choice([0.0, 0.0, 0.5]), ignored=rng.choice([0.0, 0.1, 0.5]),
                    pad=rng.choice([0, 0, rng.randint(1, 127)]))
    return case


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 31)


def prepare(case, seed):
    g, dtype, dev = _generator(seed), DTYPES[case["dtype"]], "cuda"
    op, state = case["op"], {"case": dict(case)}

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev)

    if op in ("norm_add", "norm_add_backward"):
        rows, hidden, groups = case["rows"], case["hidden"], case["groups"]
        shape = (groups, rows // groups, hidden)
        # a few large channels, as the residual stream of a trained model has
        large = torch.where(torch.rand(hidden, generator=g, device=dev) < 0.01, 20.0, 1.0)
        state["input"] = (normal(*shape) * 0.3).to(dtype)
        residual = (normal(*shape) * large).to(dtype)
        state["weight"] = (1.0 + 0.1 * normal(hidden)).to(dtype)
        state["post_weight"] = (1.0 + 0.1 * normal(hidden)).to(dtype) if case["post"] else None
        gates = {"none": None, "channel": (hidden,), "sequence": (groups, 1, hidden), "element": shape}[case["gate"]]
        state["gate"] = torch.sigmoid(normal(*gates)).to(dtype) if gates else None
        if op == "norm_add":
            state["residual"] = residual
            if case["out"] == "int8":
                state["values"] = torch.empty_like(residual)
        else:
            # the gradient's call has the forward call's updated residual
            state["residual"] = _joined(dict(state, residual=residual))
            state["dout"] = normal(*shape).to(dtype)
            state["dresidual"] = normal(*shape).to(dtype) if case["residual"] else None
    elif op == "int8_linear":
        rows, inner, outer = case["rows"], case["inner"], case["outer"]
        # quantised normal rows: each row's largest magnitude is 127
        state["input"] = (normal(rows, inner) * 32.0).round_().clamp_(-127, 127).to(torch.int8)
        state["weight"] = (normal(outer, inner) * 32.0).round_().clamp_(-127, 127).to(torch.int8)
        state["scale"] = (0.5 + torch.rand((rows, 1), generator=g, device=dev)) / 32.0
        state["weight_scale"] = (0.5 + torch.rand(outer, generator=g, device=dev)) * (0.02 / 32.0)
        state["bias"] = normal(outer).to(dtype) if case["bias"] else None
    else:
        rows, vocab = case["rows"], case["vocab"]
        buffer = torch.empty((rows, vocab + case["pad"]), dtype=dtype, device=dev)
        buffer.normal_(0.0, 2.0, generator=g)
        logits = buffer[:, :vocab]
        tokens = torch.randint(0, vocab, (rows,), generator=g, device=dev)
        # answers that the model expects more or less
        at = torch.arange(rows, device=dev)
        logits[at, tokens] = (normal(rows) * 4.0 + 8.0).to(dtype)
        if case["masked"]:
            keep = torch.rand(vocab, generator=g, device=dev) >= case["masked"]
            own_token = logits[at, tokens]
            logits.masked_fill_(~keep, -math.inf)
            logits[at, tokens] = own_token
        keep = torch.rand(rows, generator=g, device=dev) >= case["ignored"]
        keep[0] = True
        state["logits"], state["tokens"] = logits, torch.where(keep, tokens, IGNORE)
        if op == "log_probs_train":
            # advantages over the number of tokens, and an entropy bonus
            state["dlog_prob"] = -normal(rows) / rows
            state["dentropy"] = torch.full((rows,), -0.01 / rows, device=dev)
    return state


# ---- the norms on both sides of a block ----------------------------------------------------
def _normed(x):
    return x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + EPS)


def _joined(s):
    """The updated residual, in its type: what the next norm reads."""
    n = s["input"].float()
    if s["post_weight"] is not None:
        n = _normed(n) * s["post_weight"].float()
    if s["gate"] is not None:
        n = n * s["gate"].float()
    return (s["residual"].float() * s["case"]["scale"] + n).to(s["input"].dtype)


def _norm_add_plain(s):
    h = _joined(s)
    y = (_normed(h.float()) * s["weight"].float()).to(h.dtype)
    if s["case"]["out"] == "same":
        return {"out": y, "residual": h}
    y = y.float()
    scale = torch.clamp(y.abs().amax(dim=-1, keepdim=True) / 127.0, min=FLT_MIN)
    q = torch.clamp(torch.round(y * (1.0 / scale)), -127, 127).to(torch.int8)
    return {"out": torch.mul(q, scale, out=s["values"]), "scale": scale, "residual": h}


def _norm_add_backward_plain(s):
    h, dy = s["residual"].float(), s["dout"].float()
    dtype = s["input"].dtype
    r = torch.rsqrt(h.square().mean(dim=-1, keepdim=True) + EPS)
    n = h * r
    g = dy * s["weight"].float()
    dh = r * (g - n * (g * n).mean(dim=-1, keepdim=True))
    if s["dresidual"] is not None:
        dh = dh + s["dresidual"].float()
    out = {"dweight": (dy * n).sum(dim=(0, 1)).to(dtype), "dresidual": (dh * s["case"]["scale"]).to(dtype)}
    x = s["input"].float()
    a = dh if s["gate"] is None else dh * s["gate"].float()  # the gradient of what is gated
    b = x
    if s["post_weight"] is not None:
        w = s["post_weight"].float()
        rx = torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + EPS)
        nx = x * rx
        b = nx * w
        out["dpost_weight"] = (a * nx).sum(dim=(0, 1)).to(dtype)
        a = a * w
        a = rx * (a - nx * (a * nx).mean(dim=-1, keepdim=True))
    out["dinput"] = a.to(dtype)
    if s["gate"] is not None:
        out["dgate"] = (dh * b).sum_to_size(s["gate"].shape).to(dtype)
    return out


# ---- the product of 8-bit integers -----------------------------------------------------------
def _int8_linear_plain(s):
    y = (s["input"].float() @ s["weight"].float().t()) * s["scale"] * s["weight_scale"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return {"out": y.to(DTYPES[s["case"]["dtype"]])}


# ---- log probabilities -------------------------------------------------------------------------
def _log_probs_plain(s):
    z, kept = s["logits"].float(), s["tokens"] != IGNORE
    top = z.amax(dim=1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(dim=1, keepdim=True)
    lse = top + torch.log(total)
    below = torch.where(e > 0, e * (top - z), 0.0).sum(dim=1, keepdim=True)
    entropy = torch.where(kept, (torch.log(total) + below / total)[:, 0], 0.0)
    at = torch.where(kept, s["tokens"], 0)
    log_prob = torch.where(kept, (z.gather(1, at[:, None]) - lse)[:, 0], 0.0)
    out = {"log_prob": log_prob, "entropy": entropy, "lse": torch.where(kept, lse[:, 0], 0.0)}
    if s["case"]["top"]:
        # the largest of whole keys: the value's order above, the lower index first below
        bits = (z + 0.0).view(torch.int32)
        key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * 2 ** 32
        key += 2 ** 32 - 1 - torch.arange(z.shape[1], device=z.device)
        best = 2 ** 32 - 1 - (torch.topk(key, s["case"]["top"], dim=1).values & (2 ** 32 - 1))
        out["top_log_prob"] = torch.where(kept[:, None], z.gather(1, best) - lse, 0.0)
        out["top_index"] = torch.where(kept[:, None], best, -1)
    return out


def _log_probs_backward_plain(s, lse, entropy):
    z, kept = s["logits"].float(), (s["tokens"] != IGNORE)[:, None]
    at = torch.where(kept, s["tokens"][:, None], 0)
    log_p = z - lse[:, None]
    p = torch.exp(log_p)
    d = torch.where(p > 0, p * (log_p + entropy[:, None]), 0.0) * -s["dentropy"][:, None]
    d -= p * s["dlog_prob"][:, None]
    d.scatter_add_(1, at, s["dlog_prob"][:, None])
    return torch.where(kept, d, 0.0).to(s["logits"].dtype)


def _plain(s):
    op = s["case"]["op"]
    if op == "norm_add":
        return _norm_add_plain(s)
    if op == "norm_add_backward":
        return _norm_add_backward_plain(s)
    if op == "int8_linear":
        return _int8_linear_plain(s)
    out = _log_probs_plain(s)
    if op == "log_probs_train":
        out["dlogits"] = _log_probs_backward_plain(s, out["lse"], out["entropy"])
    return out


def _own(s):
    import hp_rms_norm_amd as hp
    case = s["case"]
    op = case["op"]
    if op == "norm_add":
        args = (s["input"], s["residual"], s["post_weight"], s["weight"], EPS)
        if case["out"] == "same":
            out, residual = hp.norm_add_rms_norm(*args, gate=s["gate"], residual_scale=case["scale"])
            return {"out": out, "residual": residual}
        q, scale, residual = hp.norm_add_rms_norm_int8(*args, gate=s["gate"], residual_scale=case["scale"])
        return {"out": torch.mul(q, scale, out=s["values"]), "scale": scale, "residual": residual}
    if op == "norm_add_backward":
        names = ("dinput", "dresidual", "dpost_weight", "dweight", "dgate")
        got = hp.norm_add_rms_norm_backward(s["dout"], s["input"], s["residual"], s["post_weight"], s["weight"], EPS,
                                            gate=s["gate"], residual_scale=case["scale"], dresidual=s["dresidual"])
        return {k: v for k, v in zip(names, got) if v is not None}
    if op == "int8_linear":
        return {"out": hp.int8_linear(s["input"], s["scale"], s["weight"], s["weight_scale"], bias=s["bias"],
                                      dtype=DTYPES[case["dtype"]])}
    log_prob, entropy, lse, top_log_prob, top_index = hp.token_log_probs(s["logits"], s["tokens"], top=case["top"],
                                                                         ignore_index=IGNORE)
    out = {"log_prob": log_prob, "entropy": entropy, "lse": lse}
    if case["top"]:
        out.update(top_log_prob=top_log_prob, top_index=top_index)
    if op == "log_probs_train":
        out["dlogits"] = hp.token_log_probs_backward(s["dlog_prob"], s["logits"], s["tokens"], lse, entropy=entropy,
                                                     dentropy=s["dentropy"], ignore_index=IGNORE)
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ---- the definitions in 64 bits ----------------------------------------------------------------
def _exact_norm_add(s):
    case, dtype = s["case"], s["input"].dtype
    add = s["input"].double()
    if case["post"]:
        add = add / (add.pow(2).sum(-1, keepdim=True) / case["hidden"] + EPS).sqrt() * s["post_weight"].double()
    if s["gate"] is not None:
        add = add * s["gate"].double()
    h = add + case["scale"] * s["residual"].double()
    stored = h.to(dtype).double()  # the updated residual, which the second norm reads, is in the tensors' type
    y = stored / (stored.pow(2).sum(-1, keepdim=True) / case["hidden"] + EPS).sqrt() * s["weight"].double()
    if case["out"] == "same":
        return {"out": y, "residual": h}
    y = y.to(dtype).double()  # likewise what is quantised
    scale = (y.abs().max(-1, keepdim=True).values / 127).clamp(min=FLT_MIN)
    return {"out": (y / scale).round().clamp(-127, 127) * scale, "scale": scale, "residual": h}


def _exact_norm_add_backward(s):
    """Through the Jacobian of v / sqrt(mean(v^2) + eps) of both norms."""
    width = s["case"]["hidden"]

    def through(v, g):
        ms = v.pow(2).sum(-1, keepdim=True) / width + EPS
        return g / ms.sqrt() - v * ((g * v).sum(-1, keepdim=True) / (width * ms * ms.sqrt())), v / ms.sqrt()

    dy = s["dout"].double()
    dh, n = through(s["residual"].double(), dy * s["weight"].double())
    if s["dresidual"] is not None:
        dh += s["dresidual"].double()
    out = {"dresidual": s["case"]["scale"] * dh, "dweight": (dy * n).flatten(0, 1).sum(0)}
    added, x = s["input"].double(), s["input"].double()
    gated = dh if s["gate"] is None else s["gate"].double() * dh
    out["dinput"] = gated
    if s["post_weight"] is not None:
        w = s["post_weight"].double()
        out["dinput"], nx = through(x, gated * w)
        out["dpost_weight"] = (gated * nx).flatten(0, 1).sum(0)
        added = nx * w
    if s["gate"] is not None:
        dgate = dh * added
        if s["case"]["gate"] == "sequence":
            dgate = dgate.sum(1, keepdim=True)
        elif s["case"]["gate"] == "channel":
            dgate = dgate.sum(0).sum(0)
        out["dgate"] = dgate
    return out


def _exact_log_probs(s):
    """Row blocks through log_softmax's definition and a stable sort."""
    tokens, logits, top = s["tokens"], s["logits"], s["case"]["top"]
    rows, dev = tokens.numel(), tokens.device
    out = {k: torch.zeros(rows, dtype=torch.float64, device=dev) for k in ("log_prob", "entropy", "lse")}
    if top:
        out["top_log_prob"] = torch.zeros((rows, top), dtype=torch.float64, device=dev)
        out["top_index"] = torch.full((rows, top), -1, dtype=torch.int64, device=dev)
    if s["case"]["op"] == "log_probs_train":
        out["dlogits"] = torch.zeros(logits.shape, dtype=torch.float64, device=dev)
    for at in (tokens != IGNORE).nonzero()[:, 0].split(512):
        z = logits[at].double()
        lse = torch.logsumexp(z, dim=1)
        log_p = z - lse[:, None]
        p = log_p.exp()
        finite = torch.where(p > 0, log_p, 0.0)
        entropy = -(p * finite).sum(1)
        own_token = torch.nn.functional.one_hot(tokens[at], logits.shape[1]).bool()
        out["lse"][at], out["entropy"][at] = lse, entropy
        out["log_prob"][at] = log_p[own_token]
        if top:
            order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :top]
            out["top_index"][at], out["top_log_prob"][at] = order, log_p.gather(1, order)
        if "dlogits" in out:
            out["dlogits"][at] = (s["dlog_prob"][at].double()[:, None] * (own_token.double() - p)
                                  - s["dentropy"][at].double()[:, None] * p * (finite + entropy[:, None]))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm_add":
        return _exact_norm_add(s)
    if case["op"] == "norm_add_backward":
        return _exact_norm_add_backward(s)
    if case["op"] == "int8_linear":
        y = torch.mm(s["input"].double(), s["weight"].double().T)
        y *= s["weight_scale"].double()[None, :]
        y *= s["scale"].double()
        return {"out": y if s["bias"] is None else y + s["bias"].double()}
    return _exact_log_probs(s)


def work(case):
    """Bytes: each input read once and each output written once; a loss's
    gradient reads the logits again, since what it needs of all of a row is
    known at the row's end.  Operations: of the product one multiplication and
    one addition a term, elsewhere about what the formulas hold."""
    op = case["op"]
    size = 4 if case["dtype"] == "fp32" else 2
    if op in ("norm_add", "norm_add_backward"):
        n, h = case["rows"] * case["hidden"], case["hidden"]
        gates = {"none": 0, "channel": h, "sequence": case["groups"] * h, "element": n}[case["gate"]]
        weights = h * (2 if case["post"] else 1)
        if op == "norm_add":
            out = n * size if case["out"] == "same" else n + case["rows"] * 4
            return {"bytes": (3 * n + gates + weights) * size + out, "flops": 12 * n}
        return {"bytes": (n * (6 if case["residual"] else 5) + 2 * gates + 2 * weights) * size, "flops": 30 * n}
    if op == "int8_linear":
        rows, inner, outer = case["rows"], case["inner"], case["outer"]
        nbytes = (rows + outer) * inner + rows * outer * 2 + (rows + outer) * 4 + (outer * 2 if case["bias"] else 0)
        return {"bytes": nbytes, "flops": 2 * rows * inner * outer}
    kept = max(1, round(case["rows"] * (1.0 - case["ignored"])))
    n = kept * case["vocab"]
    nbytes = n * size + case["rows"] * (20 + 12 * case["top"])
    if op == "log_probs":
        return {"bytes": nbytes, "flops": 5 * n}
    return {"bytes": 2 * n * size + case["rows"] * (case["vocab"] * size + 40), "flops": 12 * n}
