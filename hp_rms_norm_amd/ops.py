"""Python surface of the ops; the first two are drop-ins for the reference's
``hp_rms_norm.ops`` (hp_rms_norm/ops.py:4-24): same names, positional
argument order, in-place semantics and ``None`` return."""
import torch

__all__ = ["hp_rms_norm", "relu", "relu_max0", "rms_norm", "fused_add_rms_norm", "fused_add_rms_norm_out",
           "hp_rms_norm_fp8", "fused_add_rms_norm_fp8", "hp_rms_norm_fp8_ub", "hp_rms_norm_fp8_static",
           "fused_add_rms_norm_fp8_static",
           "hp_rms_norm_fp8_group", "fused_add_rms_norm_fp8_group",
           "reduce_add_rms_norm", "hp_rms_norm_mx",
           "fused_add_rms_norm_mxfp8", "fused_add_rms_norm_mxfp4", "MXFP8", "MXFP4",
           "rms_norm_backward", "rms_norm_backward_out", "linear_cross_entropy", "linear_cross_entropy_out",
           "linear_cross_entropy_backward", "linear_cross_entropy_backward_out",
           "grad_norm", "clip_grad_norm_", "clip_grad_norm_out",
           "norm_add_rms_norm", "norm_add_rms_norm_out", "norm_add_rms_norm_int8", "norm_add_rms_norm_int8_out",
           "hp_rms_norm_int8", "fused_add_rms_norm_int8",
           "norm_add_rms_norm_backward", "norm_add_rms_norm_backward_out",
           "int8_linear", "int8_linear_out",
           "token_log_probs", "token_log_probs_out", "token_log_probs_backward", "token_log_probs_backward_out",
           "set_batch_invariant", "batch_invariant"]

MXFP8, MXFP4 = 0, 1  # element formats of the OCP MX output


def hp_rms_norm(input, weight, residual, eps):
    """Fused residual-add + RMSNorm, in place (reference: hp_rms_norm/ops.py:4-15).

    ``residual <- input + residual`` (rounded to the tensor dtype) and
    ``input <- rms_norm(input + residual) * weight`` with fp32 accumulation.
    Tensors: ``input``/``residual`` [..., H] bf16 or fp16 on a HIP device,
    ``weight`` [H] of the same dtype.  Returns None.
    """
    torch.ops.hp_rms_norm.rms_norm.default(input, weight, residual, eps)


def relu(output, input):
    """The reference's "relu" (hp_rms_norm/ops.py:17-24): its kernel is an
    identity copy (activation_kernels.cuh:99-119), so ``output <- input``."""
    torch.ops.hp_rms_norm.relu.default(output, input)


def relu_max0(output, input):
    """A true ReLU on the same streamer: ``output <- max(input, 0)``,
    matching ``torch.relu`` (-0 and NaN pass through).  No reference counterpart."""
    torch.ops.hp_rms_norm.relu_max0.default(output, input)


def rms_norm(output, input, weight, eps):
    """Plain RMSNorm without a residual stream: ``output <- rms_norm(input) *
    weight``; ``output`` may be ``input``.  No reference counterpart."""
    torch.ops.hp_rms_norm.rms_norm_plain.default(output, input, weight, eps)


def fused_add_rms_norm_out(out, residual_out, input, weight, residual, eps):
    """Out-of-place ``hp_rms_norm``: ``residual_out <- input + residual`` and
    ``out <- rms_norm(residual_out) * weight``; ``input`` and ``residual`` are
    only read.  ``out`` may be ``input`` and ``residual_out`` may be
    ``residual``.  The same kernel as the in-place op (2 reads and 2 writes
    per element).  No reference counterpart."""
    torch.ops.hp_rms_norm.rms_norm_out.default(out, residual_out, input, weight, residual, eps)


def fused_add_rms_norm(input, residual, weight, eps):
    """Allocating out-of-place form of ``hp_rms_norm``: returns ``(normed,
    input + residual)`` as new tensors and leaves the arguments untouched."""
    out = torch.empty_like(input)
    res = torch.empty_like(residual)
    torch.ops.hp_rms_norm.rms_norm_out.default(out, res, input, weight, residual, eps)
    return out, res


def hp_rms_norm_fp8(output, scale, input, weight, residual, eps):
    """Fused residual-add + RMSNorm with an FP8 output, dynamic per row:
    ``residual <- input + residual`` in place; with ``y`` the op's 16-bit
    output, ``scale[r] = max(amax|y[r]| / 448, FLT_MIN)`` and ``output[r] =
    float8_e4m3fn(clamp(y[r] * (1 / scale[r]), -448, 448))``.  ``input`` is
    only read.  ``output``: float8_e4m3fn, same shape as ``input``; ``scale``:
    float32 with one element per row.  No reference counterpart."""
    torch.ops.hp_rms_norm.rms_norm_fp8_quant.default(output, scale, input, weight, residual, eps)


def fused_add_rms_norm_fp8(input, residual, weight, eps, scale_ub=None):
    """Allocating form of ``hp_rms_norm_fp8``: returns ``(q, scale)`` with
    ``q`` float8_e4m3fn shaped like ``input`` and ``scale`` float32 of shape
    ``input.shape[:-1] + (1,)``; ``residual`` is updated in place.
    ``scale_ub``: an optional one-element float32 device tensor bounding each
    row's maximum (``hp_rms_norm_fp8_ub``)."""
    q = torch.empty(input.shape, dtype=torch.float8_e4m3fn, device=input.device)
    scale = torch.empty(input.shape[:-1] + (1,), dtype=torch.float32, device=input.device)
    if scale_ub is None:
        torch.ops.hp_rms_norm.rms_norm_fp8_quant.default(q, scale, input, weight, residual, eps)
    else:
        torch.ops.hp_rms_norm.rms_norm_fp8_quant_ub.default(q, scale, input, weight, residual, scale_ub, eps)
    return q, scale


def hp_rms_norm_fp8_ub(output, scale, input, weight, residual, scale_ub, eps):
    """``hp_rms_norm_fp8`` with an upper bound on each row's maximum (the
    activation scale bound of FP8 row-wise checkpoints): ``scale = max(min(
    amax|y|, scale_ub) / 448, FLT_MIN)``, ``output`` as before with that
    scale.  ``scale_ub``: one float32 on the device, read by the kernel; a
    row holding NaN keeps a NaN scale.  No reference counterpart."""
    torch.ops.hp_rms_norm.rms_norm_fp8_quant_ub.default(output, scale, input, weight, residual, scale_ub, eps)


def hp_rms_norm_fp8_static(output, scale, input, weight, residual, eps):
    """Fused residual-add + RMSNorm with an FP8 output and one given scale for
    every row (static per-tensor quantisation): ``residual <- input +
    residual`` in place; with ``y`` the op's 16-bit output, ``output =
    float8_e4m3fn(clamp(y * (1 / scale), -448, 448))``.  ``scale``: a float32
    tensor of one element on the device, only read; ``input`` is only read.
    No reference counterpart."""
    torch.ops.hp_rms_norm.rms_norm_fp8_static_quant.default(output, scale, input, weight, residual, eps)


def fused_add_rms_norm_fp8_static(input, residual, weight, scale, eps):
    """Allocating form of ``hp_rms_norm_fp8_static``: returns ``q``
    (float8_e4m3fn shaped like ``input``); ``residual`` is updated in place."""
    q = torch.empty(input.shape, dtype=torch.float8_e4m3fn, device=input.device)
    torch.ops.hp_rms_norm.rms_norm_fp8_static_quant.default(q, scale, input, weight, residual, eps)
    return q


def hp_rms_norm_fp8_group(output, scales, input, weight, residual, eps):
    """Fused residual-add + RMSNorm with an FP8 output and one float32 scale
    per 128 consecutive elements of a row (per-token-group quantisation, 1 x
    128 groups): ``residual <- input + residual`` in place; with ``y`` the op's
    16-bit output, per group ``scales = max(amax|y| / 448, FLT_MIN)`` and
    ``output = float8_e4m3fn(clamp(y * (1 / scales), -448, 448))``.
    ``output``: float8_e4m3fn shaped like ``input``; ``scales``: float32
    ``[..., H // 128]`` with any strides under which its leading dimensions
    flatten to one row stride and no two elements share memory: rows of
    scales, or the column-major (token-minor) layout that some block-scaled
    GEMMs read, e.g. ``torch.empty(H // 128, T).t()``.  ``input`` is only
    read.  Needs ``H % 128 == 0``.  No reference counterpart."""
    torch.ops.hp_rms_norm.rms_norm_fp8_group_quant.default(output, scales, input, weight, residual, eps)


def fused_add_rms_norm_fp8_group(input, residual, weight, eps, column_major_scales=False, scale_row_align=1):
    """Allocating form of ``hp_rms_norm_fp8_group``: returns ``(q, scales)``;
    ``residual`` is updated in place.  ``column_major_scales``: the scales are
    laid out token-minor (element ``(t, g)`` at ``g * T' + t``, where ``T'``
    is the token count rounded up to a multiple of ``scale_row_align``, e.g.
    4 for 16-byte aligned columns); the returned tensor is the ``[..., H //
    128]`` view of that storage."""
    q = torch.empty(input.shape, dtype=torch.float8_e4m3fn, device=input.device)
    groups = input.shape[-1] // 128
    if column_major_scales:
        tokens = input.numel() // input.shape[-1] if input.shape[-1] else 0
        padded = -(-tokens // scale_row_align) * scale_row_align
        store = torch.empty(groups, padded, dtype=torch.float32, device=input.device)
        scales = store[:, :tokens].t().view(input.shape[:-1] + (groups,))
    else:
        scales = torch.empty(input.shape[:-1] + (groups,), dtype=torch.float32, device=input.device)
    torch.ops.hp_rms_norm.rms_norm_fp8_group_quant.default(q, scales, input, weight, residual, eps)
    return q, scales


def reduce_add_rms_norm(out, parts, weight, residual, eps):
    """Partial sums fused with ``hp_rms_norm``: with ``a = sum(parts)`` added
    in fp32 in list order and rounded once to the tensor dtype,
    ``residual <- a + residual`` in place and ``out <- rms_norm(residual) *
    weight``.  ``parts``: 1 to 8 tensors shaped like ``residual`` that share one
    row stride (the buffers of a tensor-parallel all-reduce); they are only
    read, and ``out`` may be one of them.  With one part this is
    ``hp_rms_norm`` writing its output to ``out``.  No reference counterpart."""
    torch.ops.hp_rms_norm.reduce_add_rms_norm.default(out, list(parts), weight, residual, eps)


def hp_rms_norm_mx(output, scales, input, weight, residual, eps, format):
    """Fused residual-add + RMSNorm with an OCP MX block-scaled output
    (``format`` MXFP8: E4M3 elements, MXFP4: E2M1 elements two per byte, even
    element in the low nibble).  ``residual <- input + residual`` in place;
    with ``y`` the op's 16-bit output, each block of 32 consecutive elements
    of a row gets ``scales = floor(log2(max|y|)) - emax`` as an E8M0 byte
    (emax 8 / 2; 0xFF for a block holding NaN or inf) and ``output = y / 2^s``
    rounded to nearest even, saturated.  ``output``: ``[..., H]``
    float8_e4m3fn (MXFP8) or ``[..., H // 2]`` float4_e2m1fn_x2 (MXFP4), or
    uint8; ``scales``: ``[..., H // 32]`` float8_e8m0fnu or uint8.  ``input``
    is only read.  Needs ``H % 32 == 0``.  No reference counterpart."""
    torch.ops.hp_rms_norm.rms_norm_mx_quant.default(output, scales, input, weight, residual, format, eps)


def _mx_alloc(input, format):
    h = input.shape[-1]
    if format == MXFP8:
        q = torch.empty(input.shape, dtype=torch.float8_e4m3fn, device=input.device)
    else:
        q = torch.empty(input.shape[:-1] + (h // 2,), dtype=torch.float4_e2m1fn_x2, device=input.device)
    scales = torch.empty(input.shape[:-1] + (h // 32,), dtype=torch.float8_e8m0fnu, device=input.device)
    return q, scales


def fused_add_rms_norm_mxfp8(input, residual, weight, eps):
    """Allocating MXFP8 form of ``hp_rms_norm_mx``: returns ``(q, scales)``;
    ``residual`` is updated in place."""
    q, scales = _mx_alloc(input, MXFP8)
    hp_rms_norm_mx(q, scales, input, weight, residual, eps, MXFP8)
    return q, scales


def fused_add_rms_norm_mxfp4(input, residual, weight, eps):
    """Allocating MXFP4 form of ``hp_rms_norm_mx``: returns ``(q, scales)``
    with ``q`` packed two E2M1 codes per byte; ``residual`` is updated in place."""
    q, scales = _mx_alloc(input, MXFP4)
    hp_rms_norm_mx(q, scales, input, weight, residual, eps, MXFP4)
    return q, scales


def rms_norm_backward_out(dinput, dweight, dout, input, weight, eps, dresidual=None):
    """Gradient of ``rms_norm`` and of ``hp_rms_norm`` / ``fused_add_rms_norm``
    into given tensors.  ``input`` is what was normalised -- for the fused op
    the updated residual -- and ``dout`` the gradient of the normalised output.
    With ``r = rsqrt(mean(input^2) + eps)``: ``dinput <- r * (dout * weight) -
    input * (r^3 * mean(dout * weight * input))``, plus ``dresidual`` (the
    gradient that reaches the updated residual by its other uses) if given;
    ``dweight <- sum over rows of dout * input * r``, in ``weight``'s dtype or
    float32.  Sums are fp32, each output is rounded once.  The fused op's
    input and residual both have the gradient ``dinput``.  ``dinput`` may be
    ``dout``, ``dresidual`` or ``input``.  No reference counterpart."""
    torch.ops.hp_rms_norm.rms_norm_backward.default(dinput, dweight, dout, input, weight, dresidual, eps)


def _rows(t):
    """``t`` if its rows can be read in place, else a contiguous copy."""
    if t.is_contiguous():
        return t
    if t.dim() >= 2 and t.stride(-1) == 1 and t.stride(-2) >= t.size(-1) and all(
            t.stride(i) == t.stride(i + 1) * t.size(i + 1) for i in range(t.dim() - 2)):
        return t
    return t.contiguous()


def rms_norm_backward(dout, input, weight, eps, dresidual=None):
    """Allocating form of ``rms_norm_backward_out``: returns ``(dinput,
    dweight)`` in the shapes and dtypes of ``input`` and ``weight``.  ``dout``
    and ``dresidual`` may have any strides, as torch's engine hands them on
    (expanded by a sum, permuted by a consumer): rows that cannot be read in
    place are copied first."""
    dout = _rows(dout)
    if dresidual is not None:
        dresidual = _rows(dresidual)
    dinput, dweight = torch.empty_like(input), torch.empty_like(weight)
    torch.ops.hp_rms_norm.rms_norm_backward.default(dinput, dweight, dout, input, weight, dresidual, eps)
    return dinput, dweight


def linear_cross_entropy_out(loss, lse, hidden, weight, target, ignore_index=-100):
    """Softmax cross entropy of ``hidden`` rows under a vocabulary projection,
    without keeping the logits ``z = hidden @ weight.T``: ``lse <-
    logsumexp(z)`` and ``loss <- lse - z[target]`` per row.  ``hidden``: [..., H]
    bf16 or fp16; ``weight``: [V, H] of the same dtype; ``target``: int64
    [...], contiguous; ``loss`` and ``lse``: float32 like ``target``.  Products and sums
    are fp32.  Rows whose target is ``ignore_index`` get 0 and 0 and are never
    read (padding may hold anything); another target outside ``[0, V)`` gives
    a NaN loss.  No reference counterpart."""
    torch.ops.hp_rms_norm.linear_cross_entropy.default(loss, lse, hidden, weight, target, ignore_index)


def linear_cross_entropy(hidden, weight, target, ignore_index=-100):
    """Allocating form of ``linear_cross_entropy_out``: returns ``(loss,
    lse)``, float32 per row; the backward call takes ``lse``."""
    loss = torch.empty(target.shape, dtype=torch.float32, device=target.device)
    lse = torch.empty_like(loss)
    torch.ops.hp_rms_norm.linear_cross_entropy.default(loss, lse, hidden, weight, target, ignore_index)
    return loss, lse


def linear_cross_entropy_backward_out(dhidden, dweight, dloss, hidden, weight, target, lse, ignore_index=-100):
    """Gradient of ``linear_cross_entropy`` into given tensors: with ``dz =
    (exp(z - lse) - onehot(target)) * dloss``, ``dhidden <- dz @ weight`` and
    ``dweight <- dz.T @ hidden``.  ``lse`` is the forward call's, ``dloss``
    the gradient of each row's loss (float32 like ``target``; for a mean over
    n rows, 1 / n each).  The logits are computed again, a piece of the
    vocabulary at a time; ``dz`` is rounded to the tensors' dtype (in fp16 its
    entries are off by half a step or by 2^-39 of the call's largest
    ``|dloss|``, whichever is more: rows whose ``dloss`` is 2^16 or more below
    the largest are more precise in bf16, or in a call of their own), sums are
    fp32 and each output is rounded once.  Ignored rows get a zero
    ``dhidden`` and no part in ``dweight``; an out-of-range target makes the
    gradients NaN.  No reference counterpart."""
    torch.ops.hp_rms_norm.linear_cross_entropy_backward.default(dhidden, dweight, dloss, hidden, weight, target, lse,
                                                                ignore_index)


def linear_cross_entropy_backward(dloss, hidden, weight, target, lse, ignore_index=-100):
    """Allocating form of ``linear_cross_entropy_backward_out``: returns
    ``(dhidden, dweight)``.  ``dloss`` may be any float32 tensor that expands
    to ``target``'s shape (a scalar for a sum or mean of the losses)."""
    dhidden, dweight = torch.empty_like(hidden), torch.empty_like(weight)
    torch.ops.hp_rms_norm.linear_cross_entropy_backward.default(
        dhidden, dweight, dloss.expand(target.shape).contiguous(), hidden, weight, target, lse, ignore_index)
    return dhidden, dweight


def grad_norm(grads):
    """The 2-norm of all elements of ``grads`` (a sequence of bf16, fp16 or
    fp32 tensors on one device, dense in memory in any dimension order) as a
    float32 scalar on the device; squares are summed in fp64 in a fixed order.
    An empty sequence raises RuntimeError: it names no device.  No reference
    counterpart."""
    grads = list(grads)
    norm = torch.empty((), dtype=torch.float32, device=grads[0].device if grads else None)
    torch.ops.hp_rms_norm.grad_norm.default(norm, grads)
    return norm


def clip_grad_norm_(grads, max_norm):
    """Scales ``grads`` in place by ``min(1, max_norm / (norm + 1e-6))`` with
    ``norm = grad_norm(grads)`` (the rule of ``torch.nn.utils.
    clip_grad_norm_``), and returns ``norm``.  Nothing waits for the device:
    where the norm is below the limit the second pass ends at once.  No two
    tensors may share memory.  No reference counterpart."""
    grads = list(grads)
    norm = torch.empty((), dtype=torch.float32, device=grads[0].device if grads else None)
    torch.ops.hp_rms_norm.clip_grad_norm_.default(norm, grads, max_norm)
    return norm


def clip_grad_norm_out(outs, grads, max_norm):
    """``clip_grad_norm_`` into other tensors: ``outs[i] <- grads[i] *
    factor``, each shaped and laid out like its gradient, of its dtype or
    float32 (an optimizer's master gradients); ``outs[i]`` may be
    ``grads[i]``.  Returns the norm."""
    outs, grads = list(outs), list(grads)
    norm = torch.empty((), dtype=torch.float32, device=grads[0].device if grads else None)
    torch.ops.hp_rms_norm.clip_grad_norm_out.default(norm, outs, grads, max_norm)
    return norm


def norm_add_rms_norm_out(out, residual_out, input, residual, post_weight, weight, eps, gate=None,
                          residual_scale=1.0):
    """The edge between two blocks in one pass: the norm behind a block, its
    gate, the scaled residual and the norm before the next block.  ``n =
    rms_norm(input) * post_weight`` (``post_weight`` None: ``n = input``);
    ``residual_out <- residual_scale * residual + gate * n`` (rounded to the
    tensor dtype); ``out <- rms_norm(residual_out) * weight``.  Sums are fp32;
    both norms take ``eps``.  ``input``, ``residual``: [..., H] bf16 or fp16;
    the weights: [H]; ``gate``: None, [H] (one for each channel), or of as many
    dimensions as ``input`` with its leading sizes up to some dimension and 1
    from there on, e.g. [B, 1, H] (one for each sequence) or [B, S, H].  Apply
    the gate's own activation (a sigmoid, a tanh) before.  ``out`` may be
    ``input`` and ``residual_out`` may be ``residual``.  No reference
    counterpart."""
    torch.ops.hp_rms_norm.norm_add_rms_norm.default(out, residual_out, input, post_weight, weight, residual, gate,
                                                    residual_scale, eps)


def norm_add_rms_norm(input, residual, post_weight, weight, eps, gate=None, residual_scale=1.0):
    """Allocating form of ``norm_add_rms_norm_out``: returns ``(out,
    residual_out)`` and leaves the arguments untouched."""
    out, residual_out = torch.empty_like(input), torch.empty_like(residual)
    norm_add_rms_norm_out(out, residual_out, input, residual, post_weight, weight, eps, gate, residual_scale)
    return out, residual_out


def norm_add_rms_norm_int8_out(output, scale, residual_out, input, residual, post_weight, weight, eps, gate=None,
                               residual_scale=1.0):
    """``norm_add_rms_norm_out`` with an 8-bit integer output, dynamic per row:
    with ``y`` the 16-bit output, ``scale[r] = max(amax|y[r]| / 127, FLT_MIN)``
    and ``output[r] = round(clamp(y[r] * (1 / scale[r]), -127, 127))`` (ties to
    even), what ``int8_linear`` takes.  ``output``: int8, shaped like
    ``input``; ``scale``: float32 with one element per row.  A row that holds
    NaN or infinity has that as its scale and zeros as elements.
    ``residual_out`` may be ``residual``.  No reference counterpart."""
    torch.ops.hp_rms_norm.norm_add_rms_norm_int8.default(output, scale, residual_out, input, post_weight, weight,
                                                         residual, gate, residual_scale, eps)


def _int8_rows(input):
    return torch.empty_like(input, dtype=torch.int8), input.new_empty(input.shape[:-1] + (1,), dtype=torch.float32)


def norm_add_rms_norm_int8(input, residual, post_weight, weight, eps, gate=None, residual_scale=1.0):
    """Allocating form of ``norm_add_rms_norm_int8_out``: returns ``(q, scale,
    residual_out)`` with ``scale`` of shape ``input.shape[:-1] + (1,)``, and
    leaves the arguments untouched."""
    q, scale = _int8_rows(input)
    residual_out = torch.empty_like(residual)
    norm_add_rms_norm_int8_out(q, scale, residual_out, input, residual, post_weight, weight, eps, gate,
                               residual_scale)
    return q, scale, residual_out


def hp_rms_norm_int8(output, scale, input, weight, residual, eps):
    """``hp_rms_norm_fp8`` with 8-bit integers: ``residual <- input +
    residual`` in place and ``output``, ``scale`` as for
    ``norm_add_rms_norm_int8_out``.  ``input`` is only read.  No reference
    counterpart."""
    torch.ops.hp_rms_norm.norm_add_rms_norm_int8.default(output, scale, residual, input, None, weight, residual, None,
                                                         1.0, eps)


def fused_add_rms_norm_int8(input, residual, weight, eps):
    """Allocating form of ``hp_rms_norm_int8``: returns ``(q, scale)`` with
    ``q`` int8 shaped like ``input`` and ``scale`` float32 of shape
    ``input.shape[:-1] + (1,)``; ``residual`` is updated in place."""
    q, scale = _int8_rows(input)
    hp_rms_norm_int8(q, scale, input, weight, residual, eps)
    return q, scale


def norm_add_rms_norm_backward_out(dinput, dresidual_in, dpost_weight, dweight, dgate, dout, input, residual,
                                   post_weight, weight, eps, gate=None, residual_scale=1.0, dresidual=None):
    """Gradient of ``norm_add_rms_norm`` into given tensors.  ``residual`` is
    the forward call's ``residual_out``, ``dout`` the gradient of its ``out``
    and ``dresidual`` (or None) that of ``residual_out`` by its other uses.
    With ``r`` and ``q`` the reciprocal roots of the mean squares of
    ``residual`` and ``input``: ``dh = r * (dout * weight) - residual * (r^3 *
    mean(dout * weight * residual)) + dresidual``; ``dresidual_in <-
    residual_scale * dh``; ``dweight <- sum over rows of dout * residual * r``;
    ``dgate <- dh * n``, summed over the rows that share a gate;
    ``dpost_weight <- sum over rows of gate * dh * input * q``; ``dinput`` the
    gradient of ``input`` by the first norm.  ``dpost_weight`` and ``dgate``
    are None without ``post_weight`` and ``gate``; ``dweight`` and
    ``dpost_weight`` may be float32.  Sums are fp32, each output is rounded
    once.  ``dinput`` and ``dresidual_in`` may each be one of ``dout``,
    ``dresidual``, ``input`` and ``residual`` (not the same).  No reference
    counterpart."""
    torch.ops.hp_rms_norm.norm_add_rms_norm_backward.default(
        dinput, dresidual_in, dpost_weight, dweight, dgate, dout, dresidual, input, residual, post_weight, weight,
        gate, residual_scale, eps)


def norm_add_rms_norm_backward(dout, input, residual, post_weight, weight, eps, gate=None, residual_scale=1.0,
                               dresidual=None):
    """Allocating form of ``norm_add_rms_norm_backward_out``: returns
    ``(dinput, dresidual_in, dpost_weight, dweight, dgate)``, None for what
    there is not.  ``dout`` and ``dresidual`` may have any strides, as for
    ``rms_norm_backward``."""
    dout = _rows(dout)
    if dresidual is not None:
        dresidual = _rows(dresidual)
    dinput, dresidual_in, dweight = torch.empty_like(input), torch.empty_like(residual), torch.empty_like(weight)
    dpost_weight = None if post_weight is None else torch.empty_like(post_weight)
    dgate = None if gate is None else torch.empty_like(gate)
    norm_add_rms_norm_backward_out(dinput, dresidual_in, dpost_weight, dweight, dgate, dout, input, residual,
                                   post_weight, weight, eps, gate, residual_scale, dresidual)
    return dinput, dresidual_in, dpost_weight, dweight, dgate


def int8_linear_out(out, input, scale, weight, weight_scale, bias=None):
    """The product of 8-bit integer rows and weights, each row of both with a
    scale: ``out <- (input @ weight.T) * scale * weight_scale + bias``.
    ``input``: [..., K] int8 (as ``fused_add_rms_norm_int8`` gives it) with
    ``scale`` float32, one element per row; ``weight``: [N, K] int8 with
    ``weight_scale`` float32, one element per row; ``bias``: [N] of ``out``'s
    dtype or None; ``out``: [..., N] bf16 or fp16.  Sums are exact integers (K
    up to 131071), rounded to fp32 and scaled, and ``out`` is rounded once, so
    a row's bits do not depend on the other rows.  Operands whose rows are not
    whole 16 bytes at 16-byte boundaries are copied by each call: lay a weight
    out with K % 16 == 0.  No reference counterpart."""
    torch.ops.hp_rms_norm.int8_linear.default(out, input, scale, weight, weight_scale, bias)


def int8_linear(input, scale, weight, weight_scale, bias=None, dtype=torch.bfloat16):
    """Allocating form of ``int8_linear_out``: returns ``out`` of ``dtype``
    (bf16 or fp16)."""
    out = input.new_empty(input.shape[:-1] + (weight.shape[0],), dtype=dtype)
    torch.ops.hp_rms_norm.int8_linear.default(out, input, scale, weight, weight_scale, bias)
    return out


def token_log_probs_out(log_prob, entropy, lse, top_log_prob, top_index, logits, tokens, ignore_index=-100):
    """Log probabilities of given tokens under rows of logits, with the entropy
    and the most likely alternatives: ``lse <- logsumexp(logits)``, ``log_prob
    <- logits[token] - lse``, ``entropy <- -sum(p * log(p))``, ``top_index <-``
    the largest logits, equal ones by the lower index, and ``top_log_prob <-``
    theirs minus ``lse``.  ``logits``: [..., V] bf16, fp16 or fp32 (V up to
    2^20); ``tokens``: int64 [...], contiguous; ``log_prob``, ``entropy`` and
    ``lse``: float32 like ``tokens``; ``top_log_prob`` and ``top_index``:
    float32 and int64 [..., k], k from 0 to 64.  Rows whose token is
    ``ignore_index`` get zeros (and index -1) and are never read; another token
    outside ``[0, V)`` gives a NaN ``log_prob``.  Logits of -inf (forbidden
    tokens) have probability 0; a row of nothing else has entropy 0 and log
    probabilities of -inf.  NaN or +inf makes a row's ``lse`` NaN; NaN ranks
    first.  A row's last bits follow the row count and the row's address, in
    batch-invariant mode neither.  No reference counterpart."""
    torch.ops.hp_rms_norm.token_log_probs.default(log_prob, entropy, lse, top_log_prob, top_index, logits, tokens,
                                                  ignore_index)


def token_log_probs(logits, tokens, top=0, ignore_index=-100):
    """Allocating form of ``token_log_probs_out`` with ``top`` alternatives:
    returns ``(log_prob, entropy, lse, top_log_prob, top_index)``; the backward
    call takes ``lse`` and ``entropy``."""
    log_prob = torch.empty_like(tokens, dtype=torch.float32)
    entropy, lse = torch.empty_like(log_prob), torch.empty_like(log_prob)
    shape = (*tokens.shape, top)
    top_log_prob, top_index = log_prob.new_empty(shape), tokens.new_empty(shape)
    token_log_probs_out(log_prob, entropy, lse, top_log_prob, top_index, logits, tokens, ignore_index)
    return log_prob, entropy, lse, top_log_prob, top_index


def token_log_probs_backward_out(dlogits, dlog_prob, logits, tokens, lse, entropy=None, dentropy=None,
                                 ignore_index=-100):
    """Gradient of ``token_log_probs``' ``log_prob`` and ``entropy``: with ``p =
    exp(logits - lse)``, ``dlogits <- dlog_prob * (onehot(token) - p) - dentropy
    * p * (log(p) + entropy)``.  ``lse`` and ``entropy`` are the forward
    call's, ``dlog_prob`` and ``dentropy`` (or None) float32 like ``tokens``.
    Ignored rows and rows of nothing but -inf get zeros; a token out of range
    makes its row NaN.  A probability p is off by up to ``2^-16 + 2^-22 (|lse|
    + |log p|)`` of itself, as ``lse`` is float32: a row masked with the
    dtype's lowest value throughout needs an ignored token.  ``dlogits`` may
    be ``logits``.  No reference counterpart."""
    torch.ops.hp_rms_norm.token_log_probs_backward.default(dlogits, dlog_prob, dentropy, logits, tokens, lse,
                                                           entropy, ignore_index)


def token_log_probs_backward(dlog_prob, logits, tokens, lse, entropy=None, dentropy=None, ignore_index=-100):
    """Allocating form of ``token_log_probs_backward_out``: returns
    ``dlogits``.  ``dlog_prob`` and ``dentropy`` may be any float32 tensors
    that expand to ``tokens``' shape."""
    dlogits = torch.empty_like(logits)
    if dentropy is not None:
        dentropy = dentropy.expand(tokens.shape).contiguous()
    token_log_probs_backward_out(dlogits, dlog_prob.expand(tokens.shape).contiguous(), logits, tokens, lse, entropy,
                                 dentropy, ignore_index)
    return dlogits


def set_batch_invariant(enable):
    """Process-wide: with ``enable`` true every call chooses its kernel shape by
    the width (and dtype, form and layout) alone, as the reference's launcher
    does (hp_rms_norm/csrc/cuda/hp_rms_norm.cuh:562-618), so a row's output
    bits do not depend on how many rows the call holds; calls with few rows
    run slower.  By default the row count also picks the shape, and the same
    row can come out one ulp apart between calls of different row counts.
    Returns the previous setting.  ``HPRMS_BATCH_INVARIANT=1`` in the
    environment turns it on until set.  No reference counterpart."""
    from . import _C
    return _C.set_batch_invariant(bool(enable))


def batch_invariant():
    """The current batch-invariant setting (see ``set_batch_invariant``)."""
    from . import _C
    return _C.batch_invariant()

