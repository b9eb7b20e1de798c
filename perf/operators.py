"""Operators of a training step that does without BatchNorm's batch, without a logit matrix and without Adam's second
moment: group normalisation with its activation on channels-last maps, the softmax cross entropy of a linear classifier
over a large label set, and the orthogonalisation of weight updates by Newton-Schulz products.

Each case is one call of one operator, with its gradients where the case trains.  ``own`` selects between the plain torch
form of the operators and this package's kernels.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
IGNORE = -100
NS_COEFFS = (3.4445, -4.7750, 2.0315)
NS_EPS = 1e-7
GN_EPS = 1e-5


# ------------------------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------------------------
def _gn(name, shape, groups, act, dtype, train, residual=False):
    return {"name": name, "op": "group_norm", "shape": "x".join(map(str, shape)), "groups": groups, "act": act,
            "dtype": dtype, "train": train, "residual": residual}


def _ce(name, rows, k, classes, dtype, wdtype, train, smoothing=0.0, ignored=0.0, bias=True):
    return {"name": name, "op": "linear_ce", "rows": rows, "k": k, "classes": classes, "dtype": dtype,
            "wdtype": wdtype, "train": train, "smoothing": smoothing, "ignored": ignored, "bias": bias}


def _ns(name, shapes, dtype, rank):
    return {"name": name, "op": "newton_schulz", "shapes": " ".join(f"{m}x{n}" for m, n in shapes), "dtype": dtype,
            "rank": rank}


def _resnet50_matrices():
    """[Co, Ci*kh*kw] of the bottleneck trunk's convolutions behind the stem."""
    out, inp = [], 64
    for planes, blocks in zip((64, 128, 256, 512), (3, 4, 6, 3)):
        for b in range(blocks):
            out += [(planes, inp), (planes, 9 * planes), (4 * planes, planes)]
            if b == 0:
                out.append((4 * planes, inp))
            inp = 4 * planes
    return out


def listed():
    return [
        # one clip's last feature maps while serving: a handful of frames, where only latency counts
        _gn("gn_serve_2x7x7x512", (2, 1, 7, 7, 512), 32, "relu", "bf16", False),
        # the first bottleneck stage of a trunk trained with normalisation per frame, 8 clips of 16 frames (training cases
        # take the smooth activations: next to ReLU's corner one unit in the last place decides about a whole gradient)
        _gn("gn_train_128x56x56x256", (128, 1, 56, 56, 256), 32, "silu", "bf16", True),
        # a clip normalised over time and space on the exact path, odd extents, groups of 3 channels, a shortcut
        _gn("gn_train_f32_3x5x27x29x72", (3, 5, 27, 29, 72), 24, "silu", "f32", True, residual=True),
        # the end of a residual block while evaluating: shortcut and ReLU with the normalisation
        _gn("gn_eval_64x28x28x512", (64, 1, 28, 28, 512), 32, "relu", "bf16", False, residual=True),
        # the action head itself: one batch of clips, 101 classes, fp32 master weights
        _ce("ce_train_32x256x101", 32, 256, 101, "bf16", "f32", True),
        # every frame of a batch labelled out of a codebook of visual tokens, part of the frames unlabelled
        _ce("ce_train_4096x768x16384", 4096, 768, 16384, "bf16", "f32", True, ignored=0.25),
        # the largest label set, weights kept in bf16
        _ce("ce_train_8192x1024x65536", 8192, 1024, 65536, "bf16", "bf16", True, bias=False),
        # exact path: odd sizes, label smoothing, ignored rows
        _ce("ce_train_f32_1003x327x10007", 1003, 327, 10007, "f32", "f32", True, smoothing=0.1, ignored=0.1),
        # validation loss of every sample over a large label set: forward only
        _ce("ce_eval_2048x512x20011", 2048, 512, 20011, "bf16", "bf16", False),
        # the four convolutions of the small frame encoder
        _ns("ns_encoder_4", [(32, 75), (64, 288), (128, 576), (256, 1152)], "f32", 0.25),
        # all convolutions of a ResNet-50 trunk in one optimizer step
        _ns("ns_resnet50_52", _resnet50_matrices(), "f32", 0.25),
        # one large square matrix, update in bf16
        _ns("ns_4096x4096", [(4096, 4096)], "bf16", 0.25),
    ]


def _logint(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("group_norm", "linear_ce", "newton_schulz"))
    if op == "group_norm":
        cpg = rng.choice((1, 2, 3, 4, 8, 8, 16, 16, 24, 32, 64))
        groups = _logint(rng, 1, 64)
        while (cpg * groups) % 8:
            groups += 1
        c = cpg * groups
        n = _logint(rng, 1, 256)
        d = rng.choice((1, 1, 1, _logint(rng, 2, 16)))
        h, w = _logint(rng, 1, 112), _logint(rng, 1, 112)
        while n * d * h * w * c > 100_000_000:
            if n > 1:
                n = (n + 1) // 2
            elif d > 1:
                d = (d + 1) // 2
            else:
                h, w = (h + 1) // 2, (w + 1) // 2
        train = rng.random() < 0.6
        return {"op": op, "shape": f"{n}x{d}x{h}x{w}x{c}", "groups": groups,
                "act": rng.choice(("none", "silu", "gelu") if train else ("none", "relu", "silu", "gelu")),
                "dtype": rng.choice(("bf16", "bf16", "f32")), "train": train, "residual": rng.random() < 0.4}
    if op == "linear_ce":
        rows, k, classes = _logint(rng, 1, 16384), _logint(rng, 8, 2048), _logint(rng, 2, 65536)
        while rows * k * classes > 8192 * 1024 * 32768:
            rows = (rows + 1) // 2
        dtype = rng.choice(("bf16", "bf16", "f32"))
        if dtype == "f32":
            while rows * k * classes > 8192 * 1024 * 8192:
                rows = (rows + 1) // 2
        return {"op": op, "rows": rows, "k": k, "classes": classes, "dtype": dtype,
                "wdtype": "f32" if dtype == "f32" else rng.choice(("bf16", "f32")), "train": rng.random() < 0.7,
                "smoothing": rng.choice((0.0, 0.0, 0.1)), "ignored": rng.choice((0.0, 0.0, 0.2, 0.9)),
                "bias": rng.random() < 0.7}
    count = rng.choice((1, 1, 2, 5, 16))
    shapes, budget = [], 4096 ** 3 // count
    for _ in range(count):
        m, n = _logint(rng, 1, 4096), _logint(rng, 1, 8192)
        while min(m, n) ** 2 * max(m, n) > budget:
            m, n = (m + 1) // 2, (n + 1) // 2
        shapes.append((m, n))
    return {"op": op, "shapes": " ".join(f"{m}x{n}" for m, n in shapes), "dtype": rng.choice(("f32", "f32", "bf16")),
            "rank": rng.choice((0.1, 0.25, 1.0))}


# ------------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------------
def _dims(text):
    return tuple(int(v) for v in text.split("x"))


def _shapes(case):
    return [_dims(s) for s in case["shapes"].split()]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device=dev, generator=gen)

    st = {"case": case, "op": case["op"]}
    if case["op"] == "group_norm":
        # what a convolution hands over: channels of their own mean and spread
        shape = _dims(case["shape"])
        c = shape[-1]
        x = randn(*shape).mul_(0.5 + randn(c).abs_()).add_(randn(c)).to(dt)
        gn = torch.nn.GroupNorm(case["groups"], c, eps=GN_EPS, device=dev)
        with torch.no_grad():
            gn.weight.copy_(1 + 0.2 * randn(c))
            gn.bias.copy_(0.2 * randn(c))
        st["gn"] = gn
        st["x"] = x.requires_grad_(case["train"])
        st["residual"] = randn(*shape).to(dt).requires_grad_(case["train"]) if case["residual"] else None
        st["dy"] = randn(*shape).to(dt) if case["train"] else None
    elif case["op"] == "linear_ce":
        rows, k, classes = case["rows"], case["k"], case["classes"]
        x = randn(rows, k).to(dt)
        # weights as a bf16 checkpoint holds them on the bf16 path, whatever type keeps them
        w = (randn(classes, k) * (2.5 / math.sqrt(k))).to(dt).to(DTYPES[case["wdtype"]])
        st["weight"] = torch.nn.Parameter(w, requires_grad=case["train"])
        st["bias"] = torch.nn.Parameter(randn(classes).to(DTYPES[case["wdtype"]]),
                                        requires_grad=case["train"]) if case["bias"] else None
        # frequent and rare labels
        u = torch.rand(rows, device=dev, generator=gen)
        target = (classes * u * u).long().clamp_(0, classes - 1)
        if case["ignored"] > 0:
            drop = torch.rand(rows, device=dev, generator=gen) < case["ignored"]
            target = torch.where(drop, torch.full_like(target, IGNORE), target)
        st["x"] = x.requires_grad_(case["train"])
        st["target"] = target
    else:
        # a momentum of gradients: a few strong directions over a floor of noise, at a gradient's size
        mats = []
        for m, n in _shapes(case):
            r = max(1, int(case["rank"] * min(m, n)))
            strong = randn(m, r).mul_(torch.logspace(0, -2, r, device=dev)) @ randn(r, n)
            mats.append((1e-3 * (strong + 0.1 * randn(m, n))).to(dt))
        st["mats"] = mats
    return st


# ------------------------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------------------------
def run(state):
    op = state["op"]
    if op == "group_norm":
        return _run_group_norm(state)
    if op == "linear_ce":
        return _run_linear_ce(state)
    return _run_newton_schulz(state)


def _run_group_norm(st):
    case, gn, x, res = st["case"], st["gn"], st["x"], st["residual"]
    if own:
        from video_classification_amd import ops
        if not case["train"]:
            with torch.no_grad():
                return {"y": ops.group_norm(x, gn, act=case["act"], residual=res)}
        x.grad = gn.weight.grad = gn.bias.grad = None
        if res is not None:
            res.grad = None
        y = ops.group_norm(x, gn, act=case["act"], residual=res)
        y.backward(st["dy"])
        out = {"y": y.detach(), "dx": x.grad, "dweight": gn.weight.grad, "dbias": gn.bias.grad}
        if res is not None:
            out["dresidual"] = res.grad
        return out
    with torch.no_grad():
        return _plain_group_norm(x, gn.weight, gn.bias, gn.num_groups, gn.eps, case["act"], res, st["dy"])


def _plain_group_norm(x, gamma, beta, groups, eps, act, res, dy):
    n, c = x.shape[0], x.shape[-1]
    xg = x.float().view(n, -1, groups, c // groups)
    mean = xg.mean(dim=(1, 3), keepdim=True)
    d = xg - mean
    rstd = torch.rsqrt((d * d).mean(dim=(1, 3), keepdim=True) + eps)
    xhat = (d * rstd).view(n, -1, c)
    z = xhat * gamma + beta
    if res is not None:
        z = z + res.float().view(z.shape)
    if act == "relu":
        y, slope = z.clamp_min(0), (z > 0).float()
    elif act == "silu":
        s = 1 / (1 + torch.exp(-z))
        y, slope = z * s, s * (1 + z * (1 - s))
    elif act == "gelu":
        phi = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
        y, slope = z * phi, phi + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    else:
        y, slope = z, None
    out = {"y": y.to(x.dtype).view(x.shape)}
    if dy is None:
        return out
    dz = dy.float().view(z.shape)
    if slope is not None:
        dz = dz * slope
    dxhat = (dz * gamma).view(xg.shape)
    xh = xhat.view(xg.shape)
    m1 = dxhat.mean(dim=(1, 3), keepdim=True)
    m2 = (dxhat * xh).mean(dim=(1, 3), keepdim=True)
    dx = rstd * (dxhat - m1 - xh * m2)
    out["dx"] = dx.to(x.dtype).view(x.shape)
    out["dweight"] = (dz * xhat).sum(dim=(0, 1))
    out["dbias"] = dz.sum(dim=(0, 1))
    if res is not None:
        out["dresidual"] = dz.to(res.dtype).view(x.shape)
    return out


def _run_linear_ce(st):
    case, x, w, b, target = st["case"], st["x"], st["weight"], st["bias"], st["target"]
    if own:
        from video_classification_amd import ops
        if not case["train"]:
            with torch.no_grad():
                return {"loss": ops.linear_cross_entropy(x, w, b, target, ignore_index=IGNORE,
                                                         label_smoothing=case["smoothing"], reduction="none")}
        x.grad = w.grad = None
        if b is not None:
            b.grad = None
        loss = ops.linear_cross_entropy(x, w, b, target, ignore_index=IGNORE, label_smoothing=case["smoothing"])
        loss.backward()
        out = {"loss": loss.detach(), "dx": x.grad, "dweight": w.grad}
        if b is not None:
            out["dbias"] = b.grad
        return out
    with torch.no_grad():
        return _plain_linear_ce(x, w, b, target, case["smoothing"], case["train"])


def _plain_linear_ce(x, w, b, target, smoothing, train):
    xf, wf = x.float(), w.float()
    z = xf @ wf.t()
    if b is not None:
        z = z + b.float()
    classes = z.shape[1]
    keep = target != IGNORE
    t = torch.where(keep, target, torch.zeros_like(target))
    top = z.max(dim=1, keepdim=True).values
    p = torch.exp(z - top)
    total = p.sum(dim=1, keepdim=True)
    lse = (top + torch.log(total)).squeeze(1)
    row = lse - (1 - smoothing) * z.gather(1, t[:, None]).squeeze(1)
    if smoothing > 0:
        row = row - smoothing * z.mean(dim=1)
    if not train:
        return {"loss": torch.where(keep, row, torch.zeros_like(row))}
    scale = keep.float() / keep.sum().clamp_min(1).float()
    out = {"loss": (row * scale).sum()}
    p = p.div_(total)
    rows = torch.arange(p.shape[0], device=p.device)
    p[rows, t] -= 1 - smoothing
    if smoothing > 0:
        p -= smoothing / classes
    p *= scale[:, None]
    out["dx"] = (p @ wf).to(x.dtype)
    out["dweight"] = (p.t() @ xf).to(w.dtype)
    if b is not None:
        out["dbias"] = p.sum(dim=0).to(b.dtype)
    return out


def _run_newton_schulz(st):
    if own:
        from video_classification_amd import ops
        return ops.newton_schulz(st["mats"], steps=5, coeffs=NS_COEFFS, eps=NS_EPS)
    return [_plain_newton_schulz(g) for g in st["mats"]]


def _plain_newton_schulz(g, steps=5):
    a, b, c = NS_COEFFS
    x = g.float()
    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.t()
    x = x / ((x * x).sum().sqrt() + NS_EPS)
    for _ in range(steps):
        s = x @ x.t()
        x = a * x + (b * s + c * (s @ s)) @ x
    if tall:
        x = x.t()
    return x.to(g.dtype).contiguous()


# ------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------------------------
def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "group_norm":
        shape = _dims(case["shape"])
        elems = math.prod(shape)
        maps = 2 + int(case["residual"])                 # x, y, the shortcut
        if case["train"]:
            maps += 2 + int(case["residual"])            # dy, dx, the shortcut's gradient
        params = shape[-1] * 4 * (4 if case["train"] else 2)
        return {"bytes": maps * elems * size + params, "flops": elems * (20 if case["train"] else 8)}
    if case["op"] == "linear_ce":
        rows, k, classes = case["rows"], case["k"], case["classes"]
        wsize = 2 if case["wdtype"] == "bf16" else 4
        params = classes * (k + int(case["bias"])) * wsize
        both = 2 if case["train"] else 1
        return {"bytes": both * (rows * k * size + params) + rows * 8 + (4 if case["train"] else 4 * rows),
                "flops": (6 if case["train"] else 2) * rows * k * classes}
    total = flops = 0
    for m, n in _shapes(case):
        s, l = min(m, n), max(m, n)
        total += 2 * m * n * size
        flops += 5 * (s * s * l + s * s * s + 2 * s * s * l)   # the two symmetric products need half of theirs
    return {"bytes": total, "flops": flops}


# ------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    with torch.enable_grad():
        if case["op"] == "group_norm":
            return _exact_group_norm(st)
        if case["op"] == "linear_ce":
            return _exact_linear_ce(st)
    return [_exact_newton_schulz(g) for g in st["mats"]]


def _exact_group_norm(st):
    case, gn = st["case"], st["gn"]
    train = case["train"]
    x = st["x"].detach().double().requires_grad_(train)
    gamma = gn.weight.detach().double().requires_grad_(train)
    beta = gn.bias.detach().double().requires_grad_(train)
    res = None if st["residual"] is None else st["residual"].detach().double().requires_grad_(train)
    n, c = x.shape[0], x.shape[-1]
    u = x.reshape(n, -1, c).transpose(1, 2).reshape(n * gn.num_groups, -1)
    var, mean = torch.var_mean(u, dim=1, correction=0, keepdim=True)
    u = ((u - mean) / (var + gn.eps).sqrt()).reshape(n, c, -1).transpose(1, 2).reshape(x.shape)
    y = u * gamma + beta
    if res is not None:
        y = y + res
    if case["act"] == "relu":
        y = torch.relu(y)
    elif case["act"] == "silu":
        y = y * torch.sigmoid(y)
    elif case["act"] == "gelu":
        y = y * torch.special.ndtr(y)
    out = {"y": y.detach()}
    if train:
        leaves = [x, gamma, beta] + ([res] if res is not None else [])
        grads = torch.autograd.grad(y, leaves, st["dy"].double())
        out.update(zip(("dx", "dweight", "dbias", "dresidual"), grads))
    return out


def _exact_linear_ce(st):
    case = st["case"]
    train = case["train"]
    x = st["x"].detach().double().requires_grad_(train)
    w = st["weight"].detach().double().requires_grad_(train)
    b = None if st["bias"] is None else st["bias"].detach().double().requires_grad_(train)
    target = st["target"]
    rows = (target != IGNORE).nonzero().squeeze(1)
    logp = x[rows] @ w.t()
    if b is not None:
        logp = logp + b
    logp = torch.log_softmax(logp, dim=1)
    eps = case["smoothing"]
    loss = -(1 - eps) * logp.gather(1, target[rows][:, None]).squeeze(1)
    if eps > 0:
        loss = loss - eps * logp.mean(dim=1)
    if not train:
        every = torch.zeros(target.shape, device=x.device, dtype=torch.float64)
        return {"loss": every.index_copy(0, rows, loss)}
    loss = loss.sum() / max(1, rows.numel())
    leaves = [x, w] + ([b] if b is not None else [])
    return {"loss": loss.detach(), **dict(zip(("dx", "dweight", "dbias"), torch.autograd.grad(loss, leaves)))}


def _exact_newton_schulz(g):
    a, b, c = NS_COEFFS
    x = g.double()
    x = x / (torch.linalg.vector_norm(x) + NS_EPS)
    for _ in range(5):
        # the same polynomial from either side: the smaller Gram matrix
        if x.shape[0] <= x.shape[1]:
            s = torch.mm(x, x.t())
            p = torch.addmm(b * s, s, s, alpha=c)
            x = torch.addmm(x, p, x, beta=a)
        else:
            s = torch.mm(x.t(), x)
            p = torch.addmm(b * s, s, s, alpha=c)
            x = torch.addmm(x, x, p, beta=a)
    return x
