"""Pure-PyTorch fp32 reference implementations of every HIP op.

These are the numerics oracles: each GPU kernel test compares the HIP op
against the matching function here (run in fp32), per the test strategy
SURVEY.md §4. They also serve as the CPU execution path (no GPU available).
"""

import torch
import torch.nn.functional as F

ACTS = {
    "none": lambda x: x,
    "relu": F.relu,
    "silu": F.silu,
}


def bn_act_forward(x, weight, bias, running_mean, running_var, training, momentum, eps, act="silu"):
    """BatchNorm2d (+ activation) exactly as torch — the semantics the fused
    HIP kernel must reproduce (fp32 stats, biased batch var for normalize,
    unbiased var into running stats — torch.nn.BatchNorm2d contract)."""
    y = F.batch_norm(x, running_mean, running_var, weight, bias, training, momentum, eps)
    return ACTS[act](y)


def group_norm_act_forward(x, num_groups, weight, bias, eps, act="silu", residual=None,
                           drop_path=None):
    """GroupNorm + activation, * drop_path by image, + residual, computed in
    fp32 at least and rounded once to x's type."""
    wide = torch.promote_types(x.dtype, torch.float32)
    n, c = x.shape[:2]
    v = x.to(wide).reshape(n, num_groups, -1)
    if v.numel() > 0:
        v = v - v.mean(dim=2, keepdim=True)
        v = v * torch.rsqrt((v * v).mean(dim=2, keepdim=True) + eps)
    y = v.reshape(x.shape)
    if weight is not None:
        y = y * weight.to(wide).view(1, c, 1, 1)
    if bias is not None:
        y = y + bias.to(wide).view(1, c, 1, 1)
    y = ACTS[act](y)
    if drop_path is not None:
        y = y * drop_path.to(wide).view(-1, 1, 1, 1)
    if residual is not None:
        y = y + residual.to(wide)
    return y.to(x.dtype)


def topk_logits_forward(logits, k, temperature=1.0):
    """(values, indices, rest) of functional.topk_logits, by a stable sort."""
    logits = logits.detach()
    wide = torch.promote_types(logits.dtype, torch.float32)
    values, indices = torch.sort(logits, dim=-1, descending=True, stable=True)
    values, indices = values[..., :k].contiguous(), indices[..., :k].contiguous()
    left = (logits.to(wide) / temperature).scatter(-1, indices, float("-inf"))
    rest = torch.logsumexp(left, dim=-1)
    return values, indices.masked_fill(values == float("-inf"), -1), rest.to(
        torch.promote_types(torch.float32, rest.dtype))


def distill_topk_forward(logits, values, indices, rest=None, temperature=1.0):
    """The rows' losses of functional.distill_topk, in fp32 at least."""
    wide = torch.promote_types(logits.dtype, torch.float32)
    inf = float("inf")
    shape, classes, k = logits.shape[:-1], logits.shape[-1], values.shape[-1]
    z = logits.to(wide).reshape(-1, classes) / temperature
    at = indices.reshape(-1, k).long()
    slot = (at >= 0) & (at < classes)
    bad = (at >= classes).any(dim=1)
    at = torch.where(slot, at, 0)
    u = (values.to(wide).reshape(-1, k) / temperature).masked_fill(~slot, -inf)
    left = torch.full_like(z[:, 0].detach(), -inf) if rest is None else rest.to(wide).reshape(-1)
    u = torch.cat([u, left[:, None]], dim=1)
    teaches = (u != -inf).any(dim=1)
    # what such a row holds must not reach its gradient either
    z = torch.where((teaches | bad)[:, None], z, 0.0)
    q = torch.softmax(torch.where(teaches[:, None], u, 0.0), dim=1)
    named = torch.zeros(z.shape, device=z.device, dtype=wide)
    named = named.scatter_add_(1, at, slot.to(wide)) > 0
    # where the teacher leaves the rest nothing its sum has no part in the loss
    counts = (q[:, -1:] > 0) & named & teaches[:, None]
    others = z.masked_fill(counts, -inf)

    # both sums about their largest: the gradient of logsumexp takes exp(z - its
    # result), which far from 0 is rounded to steps of more than one
    def largest(v):
        top = v.detach().amax(dim=1, keepdim=True)
        return torch.where(top.isfinite(), top, 0.0)

    top, top_rest = largest(z), largest(others)
    near = z - top
    log_rest = torch.logsumexp(others - top_rest, dim=1, keepdim=True) + (top_rest - top)
    log_p = torch.cat([near.gather(1, at), log_rest], dim=1) - torch.logsumexp(
        near, dim=1, keepdim=True)
    # q log q - q log p, with 0 for q = 0
    loss = torch.where(q == 0, 0.0, torch.xlogy(q, q) - q * log_p).sum(dim=1)
    loss = torch.where(teaches | bad, loss, 0.0)
    # loss and gradient alike
    loss = loss * torch.where(bad, float("nan"), 1.0)
    return loss.reshape(shape)


def se_forward(x, w_reduce, b_reduce, w_expand, b_expand, act="silu", gate="sigmoid"):
    """Squeeze-excite chain: global-avg-pool -> 1x1 reduce -> act -> 1x1
    expand -> sigmoid gate -> broadcast multiply
    (reference efficientnet_blocks.py:93-110)."""
    s = x.mean(dim=(2, 3), keepdim=True)
    s = F.conv2d(s, w_reduce, b_reduce)
    s = ACTS[act](s)
    s = F.conv2d(s, w_expand, b_expand)
    assert gate == "sigmoid"
    return x * torch.sigmoid(s)


def global_avg_pool(x):
    return x.mean(dim=(2, 3))


def rmsprop_tf_step(p, grad, square_avg, momentum_buffer, lr, alpha, eps, momentum, weight_decay,
                    decoupled_decay=False, lr_in_momentum=True):
    """One RMSpropTF update, TF semantics (reference rmsprop_tf.py:80-120):
    square_avg initialized to ONES by the optimizer, eps added INSIDE the
    sqrt, LR folded into the momentum buffer."""
    if weight_decay != 0:
        if decoupled_decay:
            p.add_(p, alpha=-weight_decay)
        else:
            grad = grad.add(p, alpha=weight_decay)
    one_minus_alpha = 1.0 - alpha
    square_avg.add_(grad.pow(2) - square_avg, alpha=one_minus_alpha)
    avg = square_avg.add(eps).sqrt_()
    if momentum > 0:
        if lr_in_momentum:
            momentum_buffer.mul_(momentum).addcdiv_(grad, avg, value=lr)
            p.add_(-momentum_buffer)
        else:
            momentum_buffer.mul_(momentum).addcdiv_(grad, avg)
            p.add_(momentum_buffer, alpha=-lr)
    else:
        p.addcdiv_(grad, avg, value=-lr)


def adamw_step(p, grad, exp_avg, exp_avg_sq, step, lr, beta1, beta2, eps, weight_decay):
    """Decoupled AdamW update (torch semantics)."""
    p.mul_(1 - lr * weight_decay)
    exp_avg.mul_(beta1).add_(grad, alpha=1 - beta1)
    exp_avg_sq.mul_(beta2).addcmul_(grad, grad, value=1 - beta2)
    bias_c1 = 1 - beta1 ** step
    bias_c2 = 1 - beta2 ** step
    denom = (exp_avg_sq / bias_c2).sqrt_().add_(eps)
    p.addcdiv_(exp_avg, denom, value=-lr / bias_c1)


def ema_update(ema_p, model_p, decay):
    """EMA: ema = ema*d + m*(1-d) (reference timm/utils.py:329-340)."""
    ema_p.mul_(decay).add_(model_p.to(ema_p.dtype), alpha=1.0 - decay)


def normalize_uint8(x_u8, mean, std, out_dtype=torch.float32):
    """Prefetcher device op: uint8 (N,C,H,W) -> float, (x - mean)/std with
    (1,C,1,1) broadcast (reference loader.py:246-253)."""
    x = x_u8.to(out_dtype)
    return (x - mean.to(out_dtype)) / std.to(out_dtype)
