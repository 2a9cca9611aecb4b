"""Group norm + activation: the op against its formulas in 64 bits, its
refusals, and the models that run it."""

import math

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from deepfake_detection_amd.models.layers_extra import GroupNorm2d, convert_groupnorm_model
from deepfake_detection_amd.ops import functional as O

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}

# (n, channels, groups, h, w)
SHAPES = [
    (2, 32, 4, 5, 7),      # 8 channels a group: a thread's vector is one group
    (3, 15, 5, 4, 3),      # odd channels: no vector loads
    (1, 12, 1, 1, 1),      # one pixel, one group
    (2, 6, 6, 9, 2),       # one channel a group
    (1, 408, 8, 10, 10),   # 51 channels a group: groups end inside vectors
    (2, 20, 4, 33, 31),    # vectors of 4
    (1, 480, 32, 13, 17),
    (5, 8, 2, 64, 65),     # more rows than a block takes at once
    (1, 2056, 8, 2, 3),    # more channels than a block takes at once
    (2, 16, 4, 190, 170),  # many chunks of rows
    (40, 64, 32, 3, 5),    # many images
    (2, 1, 1, 8, 9),
    (7, 56, 8, 37, 41),
    (1, 256, 4, 90, 91),   # fp32: fewer chunks of rows than were asked for
    (64, 160, 32, 19, 19),
    (3, 448, 32, 10, 10),
    (4, 336, 16, 38, 38),
    (2, 1300, 1, 9, 11),   # groups wider than a block's channels
    (1, 4096, 2, 23, 25),
    (1, 16400, 16, 2, 3),
    (66, 32, 4, 48, 48),   # bf16: a slab of nearly all of a block's LDS
    (3, 4, 4, 1, 1),       # one value a group
    (2, 274, 2, 60, 62),   # widths that 16 bytes do not divide: rows are folded
    (1, 33, 1, 120, 136),
    (2, 150, 6, 90, 98),
    (3, 11, 1, 130, 176),
    (1, 50, 5, 151, 149),  # and an odd number of rows, which cannot be
    (1, 16, 4, 270, 260),  # more rows than a slab's indexes take
]


def oracle(x, groups, weight, bias, eps, act, residual, drop, dy):
    """The formulas in 64 bits: y, the gradients, and for each the size of the
    terms that it is made of."""
    n, c, h, w = x.shape
    d = lambda t: None if t is None else t.detach().double().cpu()  # noqa: E731
    x, weight, bias, residual, drop, dy = map(d, (x, weight, bias, residual, drop, dy))
    per_c = lambda v: v.view(1, c, 1, 1)  # noqa: E731
    weight = torch.ones(c, dtype=torch.float64) if weight is None else weight
    bias = torch.zeros(c, dtype=torch.float64) if bias is None else bias
    keep = torch.ones(n, dtype=torch.float64) if drop is None else drop
    keep = keep.view(n, 1, 1, 1)
    m = c // groups * h * w

    def mean(v):
        v = v.reshape(n, groups, -1).sum(2, keepdim=True) / m
        return v.expand(n, groups, m).reshape(n, c, h, w)

    mu = mean(x)
    r = (mean((x - mu) ** 2) + eps).rsqrt()
    hat = (x - mu) * r
    z = hat * per_c(weight) + per_c(bias)
    sig = torch.sigmoid(z)
    a, da = {"none": (z, torch.ones_like(z)), "relu": (z.clamp(min=0), (z > 0).double()),
             "silu": (z * sig, sig * (1 + z * (1 - sig)))}[act]
    y = a * keep + (0 if residual is None else residual)
    # hat's own error does not shrink with it: the mean is a rounded sum of
    # values about mu, whose mean size E|x - mu| r <= sqrt(E(x - mu)^2) r <= 1
    # in hat's units, so hat is made of terms of 1 + |mu r| besides itself
    hat_size = hat.abs() + mu.abs() * r + 1
    # z is hat * weight + bias in 32 bits and act' <= 1.1
    y_size = hat_size * per_c(weight).abs() + per_c(bias).abs()
    y_size = (1 + z.abs()) * (y_size * keep + (0 if residual is None else residual.abs()))
    g = dy * keep * da
    gw = g * per_c(weight)
    big, small = mean(gw), mean(gw * hat)
    dx = r * (gw - big - hat * small)
    # g's own error: act'' <= 0.5, of a z that is y_size large
    g_size = g.abs() + (dy * keep).abs() * (1 + z.abs()) * (1 + y_size)
    if act == "relu":
        g_size = g.abs()
    dx_size = r * (g_size * per_c(weight).abs() + mean(g_size * per_c(weight).abs())
                   + hat_size * mean(g_size * per_c(weight).abs() * hat_size))
    return {
        "y": (y, y_size), "dx": (dx, dx_size),
        "dweight": ((g * hat).sum((0, 2, 3)),
                    (g_size * hat_size).sum((0, 2, 3))),
        "dbias": (g.sum((0, 2, 3)), g_size.sum((0, 2, 3))),
    }


def check(got, want, size, what):
    """Half a step of the type for the rounding of the result, and 32 roundings
    of 2^-24 of the terms that it is made of."""
    assert got.shape == want.shape
    step = torch.finfo(got.dtype).eps / 2
    off = (got.detach().double().cpu() - want).abs()
    # under a type's normal values its steps no longer shrink
    least = torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps
    allowed = step * want.abs() + 32 * 2.0 ** -24 * size + least
    worst = (off / allowed).max().item() if off.numel() else 0.0
    assert torch.isfinite(got).all() and worst <= 1, f"{what}: {worst:.3g} of what is allowed"


def make(shape, dtype, device, act, affine=True, tail=False, seed=0, offset=0.0):
    n, c, groups, h, w = shape
    g = torch.Generator().manual_seed(seed)
    cl = lambda v: v.to(device).contiguous(memory_format=torch.channels_last)  # noqa: E731
    rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = cl((rand(n, c, h, w) * (0.5 + torch.rand(1, c, 1, 1, generator=g))
            + rand(1, c, 1, 1) + offset).to(dtype))
    gn = nn.GroupNorm(groups, c, eps=1e-5, affine=affine).to(device)
    if affine:
        with torch.no_grad():
            gn.weight.copy_(torch.rand(c, generator=g) + 0.5)
            gn.bias.copy_(rand(c) * 0.5)
    dy = cl(rand(n, c, h, w).to(dtype))
    residual = cl(rand(n, c, h, w).to(dtype)) if tail else None
    drop = None
    if tail:
        drop = (torch.rand(n, generator=g) < 0.8).float().div(0.8).to(device)
    if act == "relu":
        # no value so near to the kink that 32 bits may see the other side of it
        ref = oracle(x, groups, gn.weight, gn.bias, gn.eps, "none", None, None, dy)
        z, size = ref["y"]
        near = z.abs() < 32 * 2.0 ** -24 * size
        assert near.float().mean() < 0.01
        dy = dy.masked_fill(near.to(device), 0.0)
    return x, gn, dy, residual, drop


def step(x, gn, act, dy, residual=None, drop=None):
    x = x.detach().requires_grad_()
    leaves = [x] + [p for p in (gn.weight, gn.bias) if p is not None]
    if residual is not None:
        residual = residual.detach().requires_grad_()
        leaves.append(residual)
    y = O.group_norm_act(x, gn, act, residual, drop)
    grads = list(torch.autograd.grad(y, leaves, dy))
    got = {"y": y, "dx": grads.pop(0)}
    if gn.weight is not None:
        got["dweight"], got["dbias"] = grads.pop(0), grads.pop(0)
    if residual is not None:
        got["dresidual"] = grads.pop(0)
    return got


def against_formulas(shape, dtype, device, act, **kw):
    x, gn, dy, residual, drop = make(shape, dtype, device, act, **kw)
    want = oracle(x, gn.num_groups, gn.weight, gn.bias, gn.eps, act, residual, drop, dy)
    got = step(x, gn, act, dy, residual, drop)
    assert got["y"].dtype == x.dtype and got["dx"].dtype == x.dtype
    if residual is not None:
        assert torch.equal(got.pop("dresidual"), dy)
    for name, v in got.items():
        check(v, *want[name], what=name)
    return got


# ---------------------------------------------------------------------------
# CPU
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("shape", SHAPES[:6], ids=str)
@pytest.mark.parametrize("act", ["silu", "relu", "none"])
def test_cpu_path_against_formulas(shape, act):
    against_formulas(shape, torch.float32, "cpu", act, tail=True)


def test_cpu_path_is_torchs_group_norm():
    x, gn, *_ = make((2, 24, 8, 6, 5), torch.float32, "cpu", "none")
    assert torch.allclose(O.group_norm_act(x, gn, "silu"), F.silu(gn(x)), atol=1e-5)


def test_gradient_against_differences():
    x, gn, *_ = make((2, 6, 3, 3, 2), torch.float64, "cpu", "none")
    gn = gn.double()
    x.requires_grad_()
    residual = torch.randn_like(x).requires_grad_()
    drop = torch.tensor([1.25, 0.0], dtype=torch.float64)
    assert torch.autograd.gradcheck(
        lambda x, w, b, r: O.group_norm_act(x, gn, "silu", r, drop),
        (x, gn.weight, gn.bias, residual))


def refusals(device):
    x, gn, *_ = make((2, 12, 3, 4, 4), torch.float32, device, "none")
    with pytest.raises(ValueError, match="act must be"):
        O.group_norm_act(x, gn, "gelu")
    with pytest.raises(ValueError, match=r"\[B, C, H, W\]"):
        O.group_norm_act(x[0], gn)
    with pytest.raises(ValueError, match="12 channels"):
        O.group_norm_act(x[:, :6], gn)
    with pytest.raises(ValueError, match="residual"):
        O.group_norm_act(x, gn, "none", x[:1])
    with pytest.raises(ValueError, match="drop_path_mask"):
        O.group_norm_act(x, gn, "none", None, torch.ones(3, device=device))


def test_refusals_cpu():
    refusals("cpu")


@pytest.mark.parametrize("width,groups", [(48, 16), (1632, 32), (56, 8), (7, 1), (32, 32)])
def test_group_count_divides_any_width(width, groups):
    assert GroupNorm2d(width).num_groups == groups
    assert GroupNorm2d(width, eps=1e-3, momentum=0.01).eps == 1e-3


def test_one_image_does_not_depend_on_its_batch():
    x, gn, *_ = make((4, 24, 8, 6, 5), torch.float32, "cpu", "none")
    alone = torch.cat([O.group_norm_act(x[i:i + 1], gn, "silu") for i in range(4)])
    # torch sums 90 values in another order for another batch: 32 roundings of
    # 2^-24 of values up to 5
    off = (O.group_norm_act(x, gn, "silu") - alone).abs().max()
    assert off <= 32 * 2.0 ** -24 * 5


@pytest.mark.parametrize("name", ["efficientnet_b0", "resnet18", "efficientnet_lite0"])
def test_converted_model_trains_alike_in_both_modes(name):
    import deepfake_detection_amd as dfd

    torch.manual_seed(0)
    model = dfd.create_model(name, num_classes=4)
    params = {k: v.clone() for k, v in model.named_parameters()}
    model = convert_groupnorm_model(model, 8)
    assert not any(isinstance(m, nn.BatchNorm2d) for m in model.modules())
    assert not any(getattr(m, "emit_bn_stats", False) for m in model.modules())
    assert {k for k, _ in model.named_parameters()} == set(params)
    assert all(torch.equal(v, params[k]) for k, v in model.named_parameters())
    x = torch.randn(2, 3, 64, 64)
    out = model.eval()(x)
    model.train()
    for m in model.modules():  # what else acts in training alone
        if hasattr(m, "drop_path_rate"):
            m.drop_path_rate = 0.0
    model.drop_rate = 0.0
    assert torch.allclose(model(x), out, atol=1e-5)
    model(x).sum().backward()
    assert all(p.grad is not None for p in model.parameters())


def test_model_built_with_group_norm():
    import deepfake_detection_amd as dfd

    model = dfd.create_model("efficientnet_b0", num_classes=4, norm_layer=GroupNorm2d)
    assert not any(isinstance(m, nn.BatchNorm2d) for m in model.modules())
    assert not any(getattr(m, "emit_bn_stats", False) for m in model.modules())
    assert model(torch.randn(1, 3, 64, 64)).shape == (1, 4)


def has_a_live_gradient(model, x):
    model.train()
    model(x).square().sum().backward()
    dead = [k for k, p in model.named_parameters() if not p.grad.abs().max() > 0]
    assert not dead, dead


@pytest.mark.parametrize("name", ["skresnet18", "skresnet50"])
def test_norms_of_pooled_features_keep_their_spread(name):
    """Pooled features have one value a channel: as many groups as channels
    would leave of them their bias alone."""
    import deepfake_detection_amd as dfd

    torch.manual_seed(0)
    x = torch.randn(2, 3, 64, 64)
    for groups in (32, 8):
        model = convert_groupnorm_model(dfd.create_model(name, num_classes=4), groups)
        assert not any(isinstance(m, nn.BatchNorm2d) for m in model.modules())
        has_a_live_gradient(model, x)
    model = dfd.create_model(name, num_classes=4, norm_layer=GroupNorm2d)
    assert not any(isinstance(m, nn.BatchNorm2d) for m in model.modules())
    has_a_live_gradient(model, x)


@pytest.mark.parametrize("name", ["efficientnet_b0", "resnet18", "efficientnet_lite0"])
def test_converted_model_has_a_live_gradient(name):
    import deepfake_detection_amd as dfd

    torch.manual_seed(0)
    model = convert_groupnorm_model(dfd.create_model(name, num_classes=4))
    has_a_live_gradient(model, torch.randn(2, 3, 64, 64))


def test_one_value_a_group_is_refused_in_training():
    norm = GroupNorm2d(32)
    x = torch.randn(2, 32, 1, 1)
    with pytest.raises(ValueError, match="one value"):
        norm(x)
    with pytest.raises(ValueError, match="one value"):
        O.bn_act(x, norm, "silu")
    assert torch.equal(norm.eval()(x), norm.bias.view(1, 32, 1, 1).expand(2, 32, 1, 1))
    assert GroupNorm2d(32)(torch.randn(2, 32, 1, 2)).abs().max() > 0
    assert GroupNorm2d(48)(torch.randn(2, 48, 1, 1)).abs().max() > 0


def test_relu6_keeps_its_bound():
    from deepfake_detection_amd.models.blocks import ConvBnAct

    block = ConvBnAct(3, 8, 3, act_layer=nn.ReLU6, norm_layer=GroupNorm2d)
    with torch.no_grad():
        block.bn1.weight.fill_(50.0)
    assert block(torch.randn(1, 3, 8, 8)).max() == 6.0


def test_train_runner_flag():
    from deepfake_detection_amd.runners.train import _parse_args

    args, _ = _parse_args(["--group-norm", "16"])
    assert args.group_norm == 16 and _parse_args([])[0].group_norm == 0


# ---------------------------------------------------------------------------
# GPU
# ---------------------------------------------------------------------------

@pytest.mark.gpu
def test_refusals_gpu():
    refusals("cuda")
    x, gn, *_ = make((2, 12, 3, 4, 4), torch.float32, "cuda", "none")
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        O.group_norm_act(x.double(), gn, "none")
    with pytest.raises(RuntimeError, match="device of x"):
        O.group_norm_act(x, gn, "none", x.cpu())
    with pytest.raises(RuntimeError, match="device of x"):
        O.group_norm_act(x, nn.GroupNorm(3, 12), "none")
    with pytest.raises(RuntimeError, match="no gradient"):
        O.group_norm_act(x, gn, "none", None, torch.ones(2, device="cuda", requires_grad=True))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["silu", "relu", "none"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_formulas(shape, act, dtype):
    against_formulas(shape, TYPES[dtype], "cuda", act)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_tail_against_formulas(shape, dtype):
    against_formulas(shape, TYPES[dtype], "cuda", "none", tail=True)
    against_formulas(shape, TYPES[dtype], "cuda", "silu", tail=True, affine=False)


# many images of few rows: slabs of few threads, and the parameters' gradients
# in slices of images
MANY = [
    (2100, 256, 32, 1, 2),
    (1030, 256, 32, 7, 7),
    (513, 48, 16, 2, 3),   # one image in the last slice
    (600, 36, 4, 3, 1),
    (17000, 8, 1, 1, 1),   # more slices than 64 of 256 images
    (512, 40, 8, 5, 1),
    (520, 64, 2, 52, 50),  # and with streaming
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", MANY, ids=str)
def test_many_images(shape, dtype):
    against_formulas(shape, TYPES[dtype], "cuda", "silu", tail=True)


@pytest.mark.gpu
def test_too_large_is_refused():
    gn = nn.GroupNorm(1, 40960).cuda()
    with pytest.raises(RuntimeError, match="channels in a group"):
        O.group_norm_act(torch.zeros(1, 40960, 1, 1, device="cuda"), gn, "none")
    gn = nn.GroupNorm(4, 8).cuda()
    x = torch.zeros(2 ** 26, 8, 1, 1, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad(), pytest.raises(RuntimeError, match="too large for one launch"):
        O.group_norm_act(x, gn, "none")


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [SHAPES[7], SHAPES[9], SHAPES[4]], ids=str)
def test_large_common_offset(shape):
    """A mean 1000 times the spread: a sum of squares in 32 bits would keep
    nothing of the variance."""
    against_formulas(shape, torch.float32, "cuda", "none", offset=1000.0)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[6]], ids=str)
def test_other_layouts(shape):
    """NCHW tensors, a slice of a batch and an expanded upstream gradient give
    what their channels-last copies give."""
    x, gn, dy, residual, drop = make(shape, torch.bfloat16, "cuda", "silu", tail=True)
    want = step(x, gn, "silu", dy, residual, drop)
    got = step(x.contiguous(), gn, "silu", dy.contiguous(), residual.contiguous(), drop)
    for k in want:
        assert torch.equal(got[k], want[k]), k
    assert got["y"].is_contiguous(memory_format=torch.channels_last)
    ones = torch.ones((), device="cuda", dtype=torch.bfloat16)
    a = step(x, gn, "silu", ones.expand_as(x))
    b = step(x, gn, "silu", torch.ones_like(x))
    for k in a:
        assert torch.equal(a[k], b[k]), k


@pytest.mark.gpu
def test_unaligned_tensors():
    """Data that begins at an odd element takes narrower loads."""
    n, c, g, h, w = 2, 24, 4, 5, 6
    x, gn, dy, *_ = make((n, c, g, h, w), torch.bfloat16, "cuda", "none")
    flat = torch.empty(x.numel() + 1, device="cuda", dtype=x.dtype)
    odd = flat[1:].view(n, h, w, c).permute(0, 3, 1, 2)
    odd.copy_(x)
    want = oracle(x, g, gn.weight, gn.bias, gn.eps, "silu", None, None, dy)
    got = step(odd, gn, "silu", dy)
    for name, v in got.items():
        check(v, *want[name], what=name)


@pytest.mark.gpu
@pytest.mark.parametrize("pdtype", [torch.float16, torch.bfloat16])
def test_halved_parameters(pdtype):
    """A halved model's parameters are read as they are; their gradients come
    in their type."""
    x, gn, dy, *_ = make((2, 24, 4, 9, 7), pdtype, "cuda", "none")
    gn = gn.to(pdtype)
    want = oracle(x, 4, gn.weight, gn.bias, gn.eps, "silu", None, None, dy)
    got = step(x, gn, "silu", dy)
    assert got["dweight"].dtype == pdtype
    for name, v in got.items():
        check(v, *want[name], what=name)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 8, 3, 3), (2, 8, 0, 3)])
def test_empty(shape):
    gn = nn.GroupNorm(4, 8).cuda()
    x = torch.zeros(shape, device="cuda", requires_grad=True)
    y = O.group_norm_act(x, gn, "silu")
    dx, dw, db = torch.autograd.grad(y, (x, gn.weight, gn.bias), torch.zeros_like(y))
    assert y.shape == x.shape and dx.shape == x.shape
    assert not dw.any() and not db.any()


@pytest.mark.gpu
def test_constant_and_nonfinite_groups_stay_apart():
    """A group without spread is its bias; NaN and infinities reach their own
    group and no other, nor another image."""
    x, gn, *_ = make((3, 16, 4, 11, 13), torch.float32, "cuda", "none")
    clean = O.group_norm_act(x, gn, "silu")
    x = x.clone()
    x[0, 0:4] = 3.0
    x[1, 5, 2, 2] = float("nan")
    x[2, 15, 0, 0] = float("inf")
    y = O.group_norm_act(x, gn, "silu")
    assert torch.allclose(y[0, 0:4], F.silu(gn.bias[:4]).view(4, 1, 1).expand(4, 11, 13),
                          rtol=1e-5, atol=1e-6)
    assert y[1, 4:8].isnan().all() and y[2, 12:16].isnan().any()
    keep = torch.ones_like(y, dtype=torch.bool)
    keep[0, 0:4] = keep[1, 4:8] = keep[2, 12:16] = False
    assert torch.equal(y[keep], clean[keep])


@pytest.mark.gpu
def test_same_bits_every_time_and_on_another_stream():
    x, gn, dy, residual, drop = make((6, 48, 16, 75, 75), torch.bfloat16, "cuda", "silu", tail=True)
    want = step(x, gn, "silu", dy, residual, drop)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            got = step(x, gn, "silu", dy, residual, drop)
        again = step(x, gn, "silu", dy, residual, drop)  # both at once
        torch.cuda.synchronize()
        for k in want:
            assert torch.equal(got[k], want[k]) and torch.equal(again[k], want[k]), k


@pytest.mark.gpu
def test_only_the_gradients_that_are_asked_for():
    x, gn, dy, *_ = make((2, 24, 4, 9, 7), torch.bfloat16, "cuda", "none")
    want = step(x, gn, "silu", dy)
    (dw,) = torch.autograd.grad(O.group_norm_act(x, gn, "silu"), (gn.weight,), dy)
    assert torch.equal(dw, want["dweight"])
    gn.requires_grad_(False)
    x = x.detach().requires_grad_()
    (dx,) = torch.autograd.grad(O.group_norm_act(x, gn, "silu"), (x,), dy)
    assert torch.equal(dx, want["dx"])
    with torch.no_grad():
        assert torch.equal(O.group_norm_act(x, gn, "silu"), want["y"])


@pytest.mark.gpu
def test_gradients_of_gradients_are_refused():
    x, gn, dy, *_ = make((2, 8, 4, 3, 3), torch.float32, "cuda", "none")
    x.requires_grad_()
    with pytest.raises(RuntimeError, match="gradients of gradients"):
        torch.autograd.grad(O.group_norm_act(x, gn, "silu"), x, dy, create_graph=True)


@pytest.mark.gpu
def test_without_a_gradient():
    """The call that keeps nothing gives the bits of the one that does; forward
    derivatives are refused by both."""
    for shape in (SHAPES[4], SHAPES[9]):
        x, gn, dy, residual, drop = make(shape, torch.bfloat16, "cuda", "silu", tail=True)
        want = step(x, gn, "silu", dy, residual, drop)["y"]
        with torch.no_grad():
            assert torch.equal(O.group_norm_act(x, gn, "silu", residual, drop), want)
        gn.requires_grad_(False)
        got = O.group_norm_act(x, gn, "silu", residual, drop)
        assert torch.equal(got, want) and not got.requires_grad
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(x, dy)
            with pytest.raises((RuntimeError, NotImplementedError)):
                O.group_norm_act(dual, gn, "silu")


@pytest.mark.gpu
def test_captured_and_replayed():
    """Two graphs of the op, replayed in turn with new inputs between eager
    calls, give the eager results."""
    cases = [make(s, torch.bfloat16, "cuda", "silu", tail=True, seed=i)
             for i, s in enumerate([(3, 48, 16, 40, 40), (2, 408, 8, 10, 10)])]
    graphs = []
    for x, gn, dy, residual, drop in cases:
        step(x, gn, "silu", dy, residual, drop)
    torch.cuda.synchronize()
    for x, gn, dy, residual, drop in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step(x, gn, "silu", dy, residual, drop)
        graphs.append((graph, got))
    for turn in range(3):
        for x, *_ in cases:
            x.mul_(1.5).add_(0.25)
        for graph, _ in graphs:
            graph.replay()
        for (graph, got), (x, gn, dy, residual, drop) in zip(graphs, cases):
            want = step(x, gn, "silu", dy, residual, drop)
            torch.cuda.synchronize()
            for k in want:
                assert torch.equal(got[k], want[k]), (turn, k)


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """More than 2^31 values: the last images are as right as the first."""
    n, c, h, w = 9, 256, 1000, 1000
    x = torch.empty(n, h, w, c, device="cuda", dtype=torch.bfloat16)
    image = torch.randn(h, w, c, device="cuda", dtype=torch.bfloat16)
    for i in range(n):
        x[i] = image
    gn = nn.GroupNorm(32, c).cuda()
    y = O.group_norm_act(x.permute(0, 3, 1, 2), gn, "silu")
    one = O.group_norm_act(image[None].permute(0, 3, 1, 2), gn, "silu")
    assert x.numel() > 2 ** 31
    # an image alone is summed in other chunks: 32 roundings of 2^-24 of sums
    # over values of size one, then at most one step of bf16
    for i in (0, n - 1):
        off = (y[i].float() - one[0].float()).abs()
        assert (off <= 2.0 ** -7 * one[0].float().abs() + 1e-5).all()


@pytest.mark.gpu
def test_backward_offsets_beyond_32_bits():
    """The backward pass makes offsets of its own: the gradients of equal images
    are those of one alone, and the parameters' are as many times its sums."""
    n, c, h, w = 9, 256, 1000, 1000
    gen = torch.Generator(device="cuda").manual_seed(2)
    image, up = (torch.randn(1, h, w, c, device="cuda", generator=gen).bfloat16().permute(0, 3, 1, 2)
                 for _ in range(2))
    gn = nn.GroupNorm(32, c).cuda()
    one = step(image, gn, "silu", up)
    x = image.expand(n, c, h, w).contiguous(memory_format=torch.channels_last)
    assert x.numel() > 2 ** 31
    got = step(x, gn, "silu", up.expand(n, c, h, w))
    # Nine images: a thread adds up 10^6 rows / 8 at a time / 228 chunks = 549
    # values, then come 3 steps of joins, 228 chunks / 16 and 9 images: less than
    # 600 roundings of 2^-24 of the sum of magnitudes. One image, in 2048 chunks:
    # less than 150. |g| <= 1.1 |dy|, so a group's means of g and g h, with mean
    # |g h| < 1, are within slack each, and |h| < 7 of a normal distribution.
    slack = 768 * 2.0 ** -24
    for i in (0, n // 2, n - 1):
        off = (got["dx"][i].float() - one["dx"][0].float()).abs()
        assert (off <= 2.0 ** -7 * one["dx"][0].float().abs() + 8 * slack).all()
    size = (up[0].float() * image[0].float()).abs().sum((1, 2)) * 1.1
    assert ((got["dweight"] - n * one["dweight"]).abs() <= slack * n * size).all()
    assert ((got["dbias"] - n * one["dbias"]).abs() <= slack * n * 1.1 * up[0].float().abs().sum((1, 2))).all()


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["efficientnet_b0", "resnet18"])
def test_model_step_against_cpu(name):
    """A converted model's forward and gradients in fp32, GPU against CPU."""
    import deepfake_detection_amd as dfd

    torch.manual_seed(0)
    model = convert_groupnorm_model(dfd.create_model(name, num_classes=4))
    model.eval()
    x = torch.randn(2, 3, 64, 64)
    want = model(x)
    want.square().sum().backward()
    grads = {k: p.grad.clone() for k, p in model.named_parameters()}
    model.zero_grad()
    model = model.cuda().to(memory_format=torch.channels_last)
    got = model(x.cuda().contiguous(memory_format=torch.channels_last))
    got.square().sum().backward()
    # some 250 layers of products of up to 1152 terms in 32 bits
    assert torch.allclose(got.cpu(), want, rtol=1e-3, atol=1e-4)
    for k, p in model.named_parameters():
        a, b = p.grad.cpu(), grads[k]
        assert (a - b).norm() <= 5e-3 * b.norm() + 1e-5, k


@pytest.mark.gpu
def test_model_with_norms_of_pooled_features_against_cpu():
    test_model_step_against_cpu("skresnet18")
