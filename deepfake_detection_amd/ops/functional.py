"""Dispatch layer: model blocks call these; on ROCm devices they run the
hand-written gfx950 HIP kernels, on CPU the PyTorch reference path.

The HIP path is NOT optional on a GPU machine: if a CUDA(ROCm) tensor
arrives and the extension is missing, we raise (see ops/extension.py).
"""

import torch
import torch.nn.functional as F

from . import reference
from .extension import gpu_ops_required, load_extension

_FUSED_ACTS = ("none", "relu", "silu")


def fusable_bn(bn) -> bool:
    """True only for a plain ``nn.BatchNorm2d`` (exact type).

    Subclasses (SplitBatchNorm2d, SyncBatchNorm, ...) override ``forward``
    with semantics the fused kernel does not implement — an isinstance
    check would silently bypass them (aux-BN stats never updated), so the
    fused path requires the exact base type.
    """
    import torch.nn as nn

    return type(bn) is nn.BatchNorm2d


def act_name_of(module) -> str:
    """Map an activation module instance to a fused-kernel act name."""
    import torch.nn as nn

    from ..models import layers as L

    if module is None or isinstance(module, nn.Identity):
        return "none"
    if isinstance(module, (nn.SiLU, L.Swish)):
        return "silu"
    if isinstance(module, (nn.ReLU, nn.ReLU6)):
        return "relu"
    return "other"


def bn_act(x, bn, act: str = "silu", residual=None, drop_path_mask=None):
    """BatchNorm2d + activation (+ optional fused drop_path scale and
    residual add), fused on GPU (HIP kernel, NHWC, bf16 I/O, fp32 stats —
    SURVEY.md §2.6 items 5 and 7), torch ops on CPU.

    drop_path_mask: fp32 [B] per-sample 0-or-1/keep values (stochastic
    depth, reference drop.py:84-100), applied to the BN+act output before
    the residual add. A GroupNorm2d in bn's place runs as group_norm_act."""
    if not fusable_bn(bn):
        if fusable_gn(bn) and act in _FUSED_ACTS:
            bn.check_spread(x)
            return group_norm_act(x, bn, act, residual, drop_path_mask)
        # Subclass with its own semantics (SplitBatchNorm2d, SyncBatchNorm...):
        # module dispatch, then the named activation.
        y = bn(x)
        if act == "silu":
            y = F.silu(y)
        elif act == "relu":
            y = F.relu(y)
        if drop_path_mask is not None:
            y = y * drop_path_mask.to(y.dtype).view(-1, 1, 1, 1)
        if residual is not None:
            y = y + residual
        return y
    if x.is_cuda and gpu_ops_required() and act in _FUSED_ACTS:
        from .bn_act import fused_bn_act

        # the kernel requires fp32 BN params/stats. A .half()'ed model (the
        # reference's model_half.pth.tar inference path, test.py:44-47)
        # carries fp16 BN params: cast read-only copies for EVAL (no
        # write-back of running stats); a halved model in TRAINING falls
        # through to the torch path below.
        w, b = bn.weight, bn.bias
        rm, rv = bn.running_mean, bn.running_var
        halved = any(t is not None and t.dtype != torch.float32
                     for t in (w, rm, rv))
        use_fused = True
        if halved:
            if bn.training:
                use_fused = False  # halved training: eager fallback below
            else:
                w = w.float() if w is not None else w
                b = b.float() if b is not None else b
                rm = rm.float() if rm is not None else rm
                rv = rv.float() if rv is not None else rv
        if use_fused:
            # producer-fused BN stats: the conv kernel that wrote x may have
            # attached bucketed per-channel (sum, sumsq) partials
            stats = None
            attached = getattr(x, "_dfd_bn_stats", None)
            if attached is not None and bn.training:
                buckets, m, c = attached
                if c == x.shape[1] and m == x.shape[0] * x.shape[2] * x.shape[3]:
                    stats = buckets
            return fused_bn_act(
                x, w, b, rm, rv,
                bn.training, bn.momentum, bn.eps, act, residual, stats,
                drop_path_mask,
            )
    y = F.batch_norm(
        x, bn.running_mean, bn.running_var, bn.weight, bn.bias,
        bn.training, bn.momentum if bn.momentum is not None else 0.1, bn.eps,
    )
    if act == "silu":
        y = F.silu(y)
    elif act == "relu":
        y = F.relu(y)
    if drop_path_mask is not None:
        y = y * drop_path_mask.to(y.dtype).view(-1, 1, 1, 1)
    if residual is not None:
        y = y + residual
    return y


def fusable_gn(norm) -> bool:
    """True for GroupNorm2d, whose forward is the fused op itself; subclasses
    and other group norms keep their own forward."""
    from ..models.layers_extra import GroupNorm2d

    return type(norm) is GroupNorm2d


def fusable_norm(norm) -> bool:
    """True for the norms that bn_act runs fused with its activation."""
    return fusable_bn(norm) or fusable_gn(norm)


def group_norm_act(x, gn, act: str = "silu", residual=None, drop_path_mask=None):
    """GroupNorm + activation (+ fused drop_path scale and residual add) of a
    [B, C, H, W] image batch: act(gn(x)) * drop_path_mask + residual.

    The statistics are of one image each, so neither the batch's size nor the
    other images change an image's result, in training and in eval alike.
    GPU: HIP kernels (ops/hip/group_norm.hip), channels_last in and out (other
    layouts are copied), fp32/bf16/fp16, statistics and parameter gradients in
    fp32; differentiable once, in x, the parameters and residual; at most 2^18
    channels, 2^14 in a group. CPU: torch ops of the same result.

    gn: an ``nn.GroupNorm`` (its num_groups, eps, weight and bias are used).
    act: "silu", "relu" or "none". drop_path_mask: [B] per-sample 0-or-1/keep
    values, without a gradient, as bn_act takes them.
    """
    if act not in _FUSED_ACTS:
        raise ValueError(f"group_norm_act: act must be one of {_FUSED_ACTS}, got {act!r}")
    if x.dim() != 4:
        raise ValueError(f"group_norm_act: [B, C, H, W] expected, got {tuple(x.shape)}")
    if x.shape[1] != gn.num_channels:
        raise ValueError(f"group_norm_act: {gn.num_channels} channels expected, "
                         f"got {x.shape[1]}")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"group_norm_act: residual must be {tuple(x.shape)}, "
                         f"got {tuple(residual.shape)}")
    if drop_path_mask is not None and drop_path_mask.shape != x.shape[:1]:
        raise ValueError(f"group_norm_act: drop_path_mask must be ({x.shape[0]},), "
                         f"got {tuple(drop_path_mask.shape)}")
    if x.is_cuda and gpu_ops_required():
        return load_extension().group_norm_act(
            x, gn.weight, gn.bias, gn.num_groups, gn.eps, act, residual, drop_path_mask)
    return reference.group_norm_act_forward(
        x, gn.num_groups, gn.weight, gn.bias, gn.eps, act, residual, drop_path_mask)


_LOGIT_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_MAX_TOPK = 256
_MAX_DISTILL_CLASSES = 1 << 18


def _check_logits(op, logits, k, temperature):
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{op}: [..., classes] expected, got {tuple(logits.shape)}")
    if logits.is_cuda and logits.dtype not in _LOGIT_DTYPES:
        raise TypeError(f"{op}: float32, bfloat16 or float16 expected, got {logits.dtype}")
    if not logits.is_floating_point():
        raise TypeError(f"{op}: floating-point logits expected, got {logits.dtype}")
    if not 1 <= k <= _MAX_TOPK:
        raise ValueError(f"{op}: k must be in 1..{_MAX_TOPK}, got {k}")
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"{op}: temperature must be in 1e-6..1e6, got {temperature}")


def topk_logits(logits, k: int, temperature: float = 1.0):
    """A teacher's answer, short: the k largest logits of each row and what is
    left of it. Returns (values, indices, rest):

      values   [..., k]  the logits themselves, largest first, in logits' type
      indices  [..., k]  int64, their classes; equal logits by lowest class; -1
                         where the logit is -inf (a class that is switched off)
      rest     [...]     fp32, log(sum(exp(logit / temperature))) over the
                         classes that were not taken; -inf if none is left

    NaN counts as the largest value. logits: [..., classes], any row spacing;
    1 <= k <= 256 and no more than classes. No gradient: what a teacher says is
    given. GPU: one pass over the logits (ops/hip/distill.hip), fewer than
    2^31 - 4096 classes.
    """
    _check_logits("topk_logits", logits, k, temperature)
    if k > logits.shape[-1]:
        raise ValueError(f"topk_logits: k is {k}, of {logits.shape[-1]} classes")
    if logits.is_cuda and gpu_ops_required():
        return tuple(load_extension().topk_logits(logits, k, temperature))
    return reference.topk_logits_forward(logits, k, temperature)


def distill_topk(logits, values, indices, rest=None, temperature: float = 1.0):
    """Loss of a student's logits against a teacher's top logits, one fp32
    value for each row: the divergence KL(teacher || student) at the given
    temperature over the classes that the teacher names and, as one class more,
    all others together.

      logits   [..., classes] of the student, any row spacing, at most 2^18
               classes; fp32, bf16 or fp16; the gradient comes in their type
      values, indices, rest   as topk_logits gives them, at the same
               temperature; values of any of the three types, at most 256 slots.
               Without rest the teacher's answer is its named classes alone.

    A slot whose index is negative is empty. A row of empty slots without a
    finite rest teaches nothing: its loss and gradient are 0, whatever its
    logits hold. An index beyond the classes makes its row's loss and gradient
    NaN. If two slots name one class, each has its own term in the loss and their
    probabilities add up in the gradient. A class at -inf has student probability
    0; where the teacher gives it more, the loss is inf, as it is where a
    logarithm of a probability is beyond fp32. Any finite logits and masks are
    taken; a NaN or +inf among a row's logits leaves it no finite loss. The loss
    is not scaled by temperature^2. Differentiable once, in
    logits; the teacher's answer is given. GPU: one pass over the logits
    forward, one backward (ops/hip/distill.hip).
    """
    k = values.shape[-1] if values.dim() else 0
    _check_logits("distill_topk", logits, k, temperature)
    if logits.shape[-1] > _MAX_DISTILL_CLASSES:
        raise ValueError(f"distill_topk: at most {_MAX_DISTILL_CLASSES} classes, "
                         f"got {logits.shape[-1]}")
    if values.shape[:-1] != logits.shape[:-1]:
        raise ValueError(f"distill_topk: values must be [{logits.shape[:-1]}, k], "
                         f"got {tuple(values.shape)}")
    if indices.shape != values.shape:
        raise ValueError(f"distill_topk: indices must be {tuple(values.shape)}, "
                         f"got {tuple(indices.shape)}")
    if indices.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"distill_topk: int64 or int32 indices expected, got {indices.dtype}")
    if rest is not None and rest.shape != logits.shape[:-1]:
        raise ValueError(f"distill_topk: rest must be {tuple(logits.shape[:-1])}, "
                         f"got {tuple(rest.shape)}")
    for name, t in (("values", values), ("rest", rest)):
        if t is None:
            continue
        if t.requires_grad:
            raise ValueError(f"distill_topk: {name} has no gradient: detach it")
        if not t.is_floating_point() or (t.is_cuda and t.dtype not in _LOGIT_DTYPES):
            raise TypeError(f"distill_topk: {name} must be float32, bfloat16 or float16, "
                            f"got {t.dtype}")
    if logits.is_cuda and gpu_ops_required():
        return load_extension().distill_topk(logits, values, indices, rest, temperature)
    return reference.distill_topk_forward(logits, values, indices, rest, temperature)


def se(x, conv_reduce, act_module, conv_expand):
    """Squeeze-excite chain (pool -> 1x1 -> act -> 1x1 -> sigmoid -> mul).

    GPU: fused HIP kernel chain (ops/hip/se.hip); CPU: reference path.
    Falls back to composable torch ops for non-silu/relu gates.
    """
    act = act_name_of(act_module)
    if x.is_cuda and gpu_ops_required() and act in _FUSED_ACTS:
        from .se import fused_se

        return fused_se(x, conv_reduce.weight, conv_reduce.bias,
                        conv_expand.weight, conv_expand.bias, act)
    s = x.mean(dim=(2, 3), keepdim=True)
    s = conv_reduce(s)
    s = act_module(s)
    s = conv_expand(s)
    return x * torch.sigmoid(s)


def global_avg_pool(x):
    """Global average pool NxCxHxW -> NxC (head pooling)."""
    if x.is_cuda and gpu_ops_required():
        from .pool import fused_global_avg_pool

        return fused_global_avg_pool(x)
    return x.mean(dim=(2, 3))
