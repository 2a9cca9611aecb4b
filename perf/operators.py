"""Cases of the framework's operators for small-batch training and distillation.

Three operators, each in its plain form (elementary torch operations in 32
bits) and, where ``own`` is true, through the framework's entry points:

  norm     group normalization with an activation over channels-last images,
           forward alone or with its backward pass
  topk     the k largest logits of each row and the log-sum-exp of the others
  distill  the loss of a student's logits against such a teacher's answer, with
           its gradient
"""

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # serving one image: the widest expansion of EfficientNet-B4 at 299 px
        # (1632 channels on 10x10), 51 channels a group
        _norm("norm one image", 1, 1632, 32, 10, 10, "fp16", "silu", train=False),
        # a serving batch through the head of the 12-channel 600 px model
        _norm("norm serving batch", 32, 256, 32, 19, 19, "fp16", "silu", train=False),
        # that model's training batch of 26, a depthwise layer of stage 3
        # (15 channels a group)
        _norm("norm train expand", 26, 480, 32, 75, 75, "bf16", "silu", train=True),
        # the tail of a residual block: no activation, stochastic depth, skip
        _norm("norm train tail", 64, 160, 32, 19, 19, "bf16", "none", train=True, tail=True),
        # the stem of the 12-channel 600 px model: the largest activation it has
        _norm("norm train stem", 26, 256, 32, 300, 300, "bf16", "silu", train=True),
        # fp32 training without autocast on odd sizes
        _norm("norm train fp32", 7, 56, 8, 37, 41, "fp32", "relu", train=True),
        # a teacher of 1000 classes answering a serving batch
        _topk("topk 1000 classes", 32, 1000, 5, 1.0, "fp16"),
        # a teacher with a long head over a training batch
        _topk("topk long head", 4096, 65536, 64, 2.0, "bf16"),
        # the two-class detector at its training batch
        _distill("distill two classes", 26, 2, 2, 2.0, "fp32", tail=False),
        # a 1000-class student at the benchmark's batch
        _distill("distill 1000 classes", 1536, 1000, 20, 4.0, "bf16", tail=True),
        # a long head over a large batch
        _distill("distill long head", 8192, 32000, 64, 2.0, "bf16", tail=True),
        # an odd number of classes in fp32, many teacher slots
        _distill("distill odd fp32", 513, 49999, 100, 1.0, "fp32", tail=True),
    ]


def draw(rng):
    def spread(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(["norm", "norm", "topk", "distill"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "norm":
        groups = rng.choice([1, 4, 8, 16, 32])
        c = groups * spread(1, max(1, 1632 // groups))
        h = spread(1, 300)
        w = max(1, min(300, h + rng.randint(-3, 3)))
        most = 1.5e8  # values of one tensor
        n = min(spread(1, 64), max(1, int(most // (c * h * w))))
        while n * c * h * w > most:
            h, w = max(1, h // 2), max(1, w // 2)
        # fewer values in a group say nothing: their norm is all but their signs
        while groups > 1 and c // groups * h * w < 64:
            groups //= 2
        if c // groups * h * w < 64:
            h = w = 8
        train = rng.random() < 0.7
        return _norm(None, n, c, groups, h, w, dtype, rng.choice(["silu", "relu", "none"]),
                     train=train, tail=rng.random() < 0.3)
    v = spread(2, 65536)
    rows = min(spread(1, 8192), max(1, int(1.0e8 // v)))
    k = min(v, spread(1, 128))
    t = rng.choice([1.0, 2.0, 4.0])
    if kind == "topk":
        return _topk(None, rows, v, k, t, dtype)
    return _distill(None, rows, v, k, t, dtype, tail=rng.random() < 0.7)


def _named(name, case):
    return case if name is None else dict(case, name=name)


def _norm(name, n, c, groups, h, w, dtype, act, train, tail=False):
    return _named(name, {"op": "norm", "n": n, "c": c, "groups": groups, "h": h, "w": w,
                         "dtype": dtype, "act": act, "train": train, "tail": tail})


def _topk(name, rows, classes, k, t, dtype):
    return _named(name, {"op": "topk", "rows": rows, "classes": classes, "k": k, "t": t,
                         "dtype": dtype})


def _distill(name, rows, classes, k, t, dtype, tail):
    return _named(name, {"op": "distill", "rows": rows, "classes": classes, "k": k, "t": t,
                         "dtype": dtype, "tail": tail})


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _logits(rows, classes, t, gen):
    """A few classes stand out of each row, as a trained head gives them: at
    temperature ``t`` they hold a good part of the probability."""
    z = torch.randn(rows, classes, device="cuda", generator=gen) * 1.5
    count = min(8, classes)
    peaks = torch.randint(0, classes, (rows, 1), device="cuda", generator=gen)
    peaks = (peaks + torch.arange(count, device="cuda") * (classes // count)) % classes
    height = torch.rand(rows, count, device="cuda", generator=gen) + 0.5
    height *= t * math.log(classes + 2.0)
    return z.scatter_add_(1, peaks, height), peaks, height


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "norm":
        n, c, h, w = case["n"], case["c"], case["h"], case["w"]

        def image(scale, shift):
            v = torch.empty(n, h, w, c, device="cuda", dtype=dtype).normal_(generator=gen)
            return v.mul_(scale.to(dtype)).add_(shift.to(dtype)).permute(0, 3, 1, 2)

        def channels(lo, hi):
            return torch.rand(c, device="cuda", generator=gen) * (hi - lo) + lo

        zero = torch.zeros(c, device="cuda")
        s = {"x": image(channels(0.5, 2.0), channels(-1.0, 1.0))}
        norm = torch.nn.GroupNorm(case["groups"], c, eps=1e-5, device="cuda")
        with torch.no_grad():
            norm.weight.copy_(channels(0.5, 1.5))
            norm.bias.copy_(channels(-0.5, 0.5))
        s["norm"] = norm
        if case["tail"]:
            s["residual"] = image(zero + 1.0, zero)
            keep = 0.8
            s["drop"] = torch.floor(
                keep + torch.rand(n, device="cuda", generator=gen)).div_(keep)
        if case["train"]:
            s["dy"] = image(zero + 1.0, zero + 0.01)
            s["x"].requires_grad_()
        else:
            norm.requires_grad_(False)
    elif case["op"] == "topk":
        z = _logits(case["rows"], case["classes"], case["t"], gen)[0].to(dtype)
        # one row in sixteen has most of its classes switched off
        off = torch.rand(case["rows"], device="cuda", generator=gen) < 1 / 16
        off = off[:, None] & (torch.arange(case["classes"], device="cuda") >= case["k"] // 2)
        s = {"logits": z.masked_fill_(off, float("-inf"))}
    else:
        rows, k = case["rows"], case["k"]
        z, peaks, height = _logits(rows, case["classes"], case["t"], gen)
        # the teacher agrees with the student in part
        teacher = torch.randn(z.shape, device="cuda", generator=gen).mul_(case["t"]).add_(z, alpha=0.6)
        teacher.scatter_add_(1, peaks, height.flip(1) * 0.6)
        values, indices = teacher.to(dtype).topk(k, dim=1)
        s = {"logits": z.to(dtype).requires_grad_(), "values": values}
        # one row in sixteen has nothing to learn from: padding of the batch
        empty = torch.rand(rows, device="cuda", generator=gen) < 1 / 16
        s["indices"] = indices.masked_fill(empty[:, None], -1)
        if case["tail"]:
            rest = (teacher / case["t"]).scatter_(1, indices, float("-inf"))
            s["rest"] = rest.logsumexp(1).masked_fill_(empty, float("-inf"))
        # the mean over the rows; fp16 gradients come with a scale, as its
        # training gives them
        scale = 256.0 if case["dtype"] == "fp16" else 1.0 / rows
        s["upstream"] = (torch.rand(rows, device="cuda", generator=gen) + 0.5) * scale
    return dict(s, case=case)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(s):
    case = s["case"]
    if own:
        return _own(s, case)
    if case["op"] == "norm":
        return _plain_norm(s, case)
    if case["op"] == "topk":
        return _plain_topk(s["logits"], case["k"], case["t"])
    return _plain_distill(s, case)


def _own(s, case):
    from deepfake_detection_amd.ops import functional as O

    if case["op"] == "norm":
        y = O.group_norm_act(s["x"], s["norm"], case["act"], s.get("residual"), s.get("drop"))
        if not case["train"]:
            return {"y": y}
        norm = s["norm"]
        dx, dw, db = torch.autograd.grad(y, (s["x"], norm.weight, norm.bias), s["dy"])
        return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}
    if case["op"] == "topk":
        values, indices, rest = O.topk_logits(s["logits"], case["k"], case["t"])
        return {"values": values, "indices": indices, "rest": rest}
    loss = O.distill_topk(s["logits"], s["values"], s["indices"], s.get("rest"), case["t"])
    (grad,) = torch.autograd.grad(loss, s["logits"], s["upstream"])
    return {"loss": loss.detach(), "grad": grad}


@torch.no_grad()
def _plain_norm(s, case):
    x = s["x"]
    n, c, h, w = x.shape
    g = case["groups"]
    nhwc = (n, h * w, g, c // g)
    xf = x.permute(0, 2, 3, 1).float().reshape(nhwc)
    weight = s["norm"].weight.reshape(1, 1, g, c // g)
    bias = s["norm"].bias.reshape(1, 1, g, c // g)
    centred = xf - xf.mean(dim=(1, 3), keepdim=True)
    rstd = 1.0 / torch.sqrt((centred * centred).mean(dim=(1, 3), keepdim=True) + s["norm"].eps)
    hat = centred * rstd
    z = hat * weight + bias

    def images(v):
        return v.reshape(n, h, w, c).to(x.dtype).permute(0, 3, 1, 2)

    scale = s["drop"].reshape(n, 1, 1, 1) if "drop" in s else 1.0
    sig = 1.0 / (1.0 + torch.exp(-z)) if case["act"] == "silu" else (z > 0).float()
    y = (z if case["act"] == "none" else z * sig) * scale
    if "residual" in s:
        y = y + s["residual"].permute(0, 2, 3, 1).float().reshape(nhwc)
    y = images(y)
    if not case["train"]:
        return {"y": y}
    dz = s["dy"].permute(0, 2, 3, 1).float().reshape(nhwc) * scale
    if case["act"] == "silu":
        dz = dz * (sig * (1.0 + z * (1.0 - sig)))
    elif case["act"] == "relu":
        dz = dz * sig
    dbias = dz.sum(dim=(0, 1), dtype=torch.float64).float().reshape(c)
    dweight = (dz * hat).sum(dim=(0, 1), dtype=torch.float64).float().reshape(c)
    dh = dz * weight
    dx = rstd * (dh - dh.mean(dim=(1, 3), keepdim=True)
                 - hat * (dh * hat).mean(dim=(1, 3), keepdim=True))
    return {"y": y, "dx": images(dx), "dweight": dweight, "dbias": dbias}


@torch.no_grad()
def _plain_topk(logits, k, t):
    values, indices = torch.sort(logits, dim=1, descending=True, stable=True)
    values, indices = values[:, :k].clone(), indices[:, :k].clone()
    rest = (logits.float() / t).scatter(1, indices, float("-inf"))
    top = rest.amax(dim=1, keepdim=True).clamp(min=-1e30)
    rest = torch.log(torch.exp(rest - top).sum(dim=1)) + top[:, 0]
    indices[values == float("-inf")] = -1
    return {"values": values, "indices": indices, "rest": rest}


@torch.no_grad()
def _plain_distill(s, case):
    z = s["logits"].float() / case["t"]
    slot = s["indices"] >= 0
    at = s["indices"].clamp(min=0)
    u = (s["values"].float() / case["t"]).masked_fill(~slot, float("-inf"))
    rest = s["rest"] if "rest" in s else torch.full_like(u[:, 0], float("-inf"))
    u = torch.cat([u, rest[:, None]], dim=1)
    teaches = u.amax(dim=1) > float("-inf")
    q = torch.exp(u - u.amax(dim=1, keepdim=True).clamp(min=-1e30))
    q = q / q.sum(dim=1, keepdim=True).clamp(min=1e-30)

    # a class that a slot names counts in none of the rest's sums
    named = torch.zeros(z.shape, device=z.device, dtype=torch.bool)
    named[torch.arange(z.shape[0], device=z.device)[:, None].expand_as(at)[slot], at[slot]] = True
    others = z.masked_fill(named, float("-inf"))
    top, top_r = z.amax(dim=1, keepdim=True), others.amax(dim=1, keepdim=True).clamp(min=-1e30)
    e, e_r = torch.exp(z - top), torch.exp(others - top_r)
    total, total_r = e.sum(dim=1, keepdim=True), e_r.sum(dim=1, keepdim=True)
    # the terms all but cancel where the two answers agree: they are summed in 64 bits
    log_p = torch.cat([z.gather(1, at) - top, top_r.double() - top + torch.log(total_r.double())], dim=1)
    term = torch.where(q > 0, q * (torch.log(q.double()) - log_p + torch.log(total.double())), 0.0)
    loss = term.sum(dim=1).float()
    q_r = q[:, -1:]
    target = torch.where(q_r > 0, e_r / total_r * q_r, 0.0)
    target.scatter_add_(1, at, torch.where(slot, q[:, :-1], 0.0))
    grad = (e / total - target) * (s["upstream"] / case["t"])[:, None]
    grad[~teaches] = 0.0
    return {"loss": torch.where(teaches, loss, 0.0), "grad": grad.to(s["logits"].dtype)}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(s, case)
    if case["op"] == "topk":
        t = s["logits"].detach().double()
        values, indices = t.topk(case["k"], dim=1)
        # which of equal logits are taken does not change the sum of the others
        rest = (t / case["t"]).scatter(1, indices, float("-inf")).logsumexp(dim=1)
        return {"values": values, "indices": None, "rest": rest}
    return _exact_distill(s, case)


def _exact_norm(s, case):
    """The norm image by image, and its gradients by differentiation."""
    x, norm = s["x"].detach(), s["norm"]
    weight = norm.weight.detach().double().requires_grad_(case["train"])
    bias = norm.bias.detach().double().requires_grad_(case["train"])
    ys, dxs, dws, dbs = [], [], 0.0, 0.0
    for i in range(case["n"]):
        xi = x[i].double().requires_grad_(case["train"])
        groups = xi.unflatten(0, (case["groups"], -1)).flatten(1)
        var, mean = torch.var_mean(groups, dim=1, correction=0, keepdim=True)
        hat = ((groups - mean) / (var + norm.eps).sqrt()).reshape(xi.shape)
        y = hat * weight[:, None, None] + bias[:, None, None]
        if case["act"] == "silu":
            y = y * y.sigmoid()
        elif case["act"] == "relu":
            y = y.clamp(min=0)
        if case["tail"]:
            y = y * s["drop"][i].double() + s["residual"][i].double()
        if case["train"]:
            dx, dw, db = torch.autograd.grad(y, (xi, weight, bias), s["dy"][i].double())
            dxs.append(dx)
            dws, dbs = dws + dw, dbs + db
        ys.append(y.detach())

    def images(v):
        # as `run` lays them out: stacked in the order of their channels last
        return torch.stack([i.permute(1, 2, 0) for i in v]).permute(0, 3, 1, 2)

    if not case["train"]:
        return {"y": images(ys)}
    return {"y": images(ys), "dx": images(dxs), "dweight": dws, "dbias": dbs}


def _exact_distill(s, case):
    """The divergence of the two answers over the named classes and one class
    of all others, and its gradient by differentiation, some rows at a time."""
    losses, grads = [], []
    for a in range(0, case["rows"], 1024):
        b = slice(a, a + 1024)
        z = s["logits"][b].detach().double().requires_grad_()
        slot = s["indices"][b] >= 0
        at = s["indices"][b].clamp(min=0)
        v = (s["values"][b].double() / case["t"]).masked_fill(~slot, float("-inf"))
        rest = s["rest"][b, None].double() if case["tail"] else torch.full_like(v[:, :1], float("-inf"))
        v = torch.cat([v, rest], dim=1)
        teaches = (v > float("-inf")).any(dim=1)
        q = v[teaches].softmax(dim=1)
        named = torch.zeros_like(z).scatter_(1, at, slot.double()) > 0
        scaled = z / case["t"]
        log_all = scaled.logsumexp(dim=1, keepdim=True)
        log_top = scaled.gather(1, at) - log_all
        used = q[:, -1] > 0
        log_rest = torch.zeros_like(log_all)
        pick = teaches.nonzero()[:, 0][used]
        log_rest = log_rest.index_put(
            (pick,), scaled[pick].masked_fill(named[pick], float("-inf"))
            .logsumexp(dim=1, keepdim=True) - log_all[pick])
        log_p = torch.cat([log_top, log_rest], dim=1)[teaches]
        loss = torch.zeros_like(z[:, 0])
        loss = loss.index_put((teaches,), (q.xlogy(q) - q * log_p).sum(dim=1))
        (dz,) = torch.autograd.grad(loss, z, s["upstream"][b].double())
        losses.append(loss.detach())
        grads.append(dz)
    return {"loss": torch.cat(losses), "grad": torch.cat(grads)}


def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] == "norm":
        values = case["n"] * case["c"] * case["h"] * case["w"]
        tensors = 2 + (1 if case["tail"] else 0) + (2 if case["train"] else 0)
        params = 4 * case["c"] * (4 if case["train"] else 2)
        return {"bytes": values * size * tensors + params,
                "flops": values * (30 if case["train"] else 12)}
    values = case["rows"] * case["classes"]
    answer = case["rows"] * case["k"] * (size + 8)
    if case["op"] == "topk":
        return {"bytes": values * size + answer + 4 * case["rows"], "flops": values * 6}
    return {"bytes": values * size * 2 + answer + 12 * case["rows"], "flops": values * 14}
