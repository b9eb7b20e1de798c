"""ops.linear_cross_entropy against the definition in 64 bits, its masks and refusals.

Tolerances.  A logit is a sum of K products in fp32, joined 32 at a time (a unit in the last place, 2^-23, per join and
three joins per 32 products of two-term operands): dz = ((3K/32 + 4) 2^-23 + 2^-21) S with S = sum |x||w| + |b|; the 2^-21
is the two-term form itself.  exp(z - lse) is then off by 2 dz + 2^-20 relative.  A gradient sums d = p - onehot over
rows or classes: the error of p, plus the rounding of d to its terms (2^-12 or 2^-22 of the value) and the joins of that
sum, each weighted by |W| or |x|.  The result's own type adds half a step."""
import pytest
import torch
import torch.nn as nn

U = 2.0 ** -24
TYPES = {"f32": (torch.float32, torch.float32), "mixed": (torch.bfloat16, torch.float32),
         "bf16": (torch.bfloat16, torch.bfloat16)}


def half(dt):
    return torch.finfo(dt).eps / 2


def make(N, K, V, types, seed=0, bias=True, ignored=0.0, spread=2.0, dev="cuda"):
    xd, wd = TYPES[types]
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, K, generator=g).to(xd)
    w = (torch.randn(V, K, generator=g) * spread / K ** 0.5).to(xd).to(wd)
    b = torch.randn(V, generator=g).to(wd) if bias else None
    t = torch.randint(0, V, (N,), generator=g)
    if ignored:
        t[torch.rand(N, generator=g) < ignored] = -100
    par = lambda p: nn.Parameter(p.to(dev)) if p is not None else None
    return x.to(dev), par(w), par(b), t.to(dev)


def reference(x, w, b, t, eps, weight):
    """Row losses, gradients for the row weights `weight`, and error bounds, all in float64 on the tensors' device."""
    x, w = x.detach().double(), w.detach().double()
    bias = b.detach().double() if b is not None else torch.zeros(w.shape[0], device=x.device, dtype=torch.float64)
    N, K, V = x.shape[0], x.shape[1], w.shape[0]
    keep = t != -100
    x = torch.where(keep[:, None], x, torch.zeros_like(x))
    z = x @ w.t() + bias
    lse = torch.logsumexp(z, dim=1)
    tt = torch.where(keep, t, torch.zeros_like(t))
    rows = lse - (1 - eps) * z.gather(1, tt[:, None])[:, 0]
    if eps:
        rows = rows - eps * z.mean(1)
    rows = torch.where(keep, rows, torch.zeros_like(rows))
    p = torch.exp(z - lse[:, None])
    d = p - eps / V
    d[torch.arange(N, device=x.device), tt] -= 1 - eps
    r = torch.where(keep, weight.double(), torch.zeros_like(rows))
    d, p = d * r[:, None], p * r.abs()[:, None]
    S = x.abs() @ w.abs().t() + bias.abs().clamp_max(1e30)
    dz = ((3 * K / 32 + 4) * 2.0 ** -23 + 2.0 ** -21) * float(S.max())
    return dict(rows=rows, lse=lse, z=z, d=d, p=p, dz=dz, dx=d @ w, dw=d.t() @ x, db=d.sum(0), x=x, w=w)


# A term of 11 bits rounds by up to half a step, 2^-11 of a value just above a power of two (torch.finfo(torch.float16).eps / 2);
# over many rows the roundings average out and 2^-12 holds, over the few that a mask leaves it need not.
FEW_ROWS = 2.0 ** -11


def check(ref, types, rows=None, dx=None, dw=None, db=None, extra=0.0, one_term=2.0 ** -12):
    xd, wd = TYPES[types]
    dz = ref["dz"] + extra
    N, V = ref["d"].shape
    if rows is not None:
        err = (rows.double() - ref["rows"]).abs()
        assert (err <= 4 * dz + 2.0 ** -20 * (1 + ref["lse"].abs().clamp_max(1e30))).all(), float(err.max())
    ep = 2 * dz + 2.0 ** -20
    for got, want, A, P, M, dt, length in ((dx, ref["dx"], ref["d"].abs(), ref["p"], ref["w"].abs(), xd, V),
                                           (dw, ref["dw"], ref["d"].abs().t(), ref["p"].t(), ref["x"].abs(), wd, N)):
        if got is None:
            continue
        term = 2.0 ** -22 if dt == torch.float32 else one_term
        tol = (term + 2.0 ** -21 + (3 * length / 32 + 8) * 2.0 ** -23) * (A @ M) + ep * (P @ M)
        if got is dx and extra:
            tol = tol + 2.0 ** -12 * (A @ M)  # the weight's own single term
        err = (got.double() - want).abs()
        assert (err <= tol + half(dt) * want.abs() + 1e-37).all(), float((err - tol - half(dt) * want.abs()).max())
    if db is not None:
        tol = ep * ref["p"].sum(0) + (N / 16 + 16) * U * ref["d"].abs().sum(0)
        err = (db.double() - ref["db"]).abs()
        assert (err <= tol + half(wd) * ref["db"].abs() + 1e-37).all(), float((err - tol).max())


SHAPES = [(1, 8, 2), (1, 1, 1), (3, 5, 7), (32, 256, 101), (130, 64, 129), (257, 100, 300), (64, 72, 2001), (1000, 40, 130),
          (128, 128, 128), (129, 65, 1), (5, 520, 4099), (700, 33, 1025)]


@pytest.mark.gpu
@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("bias,eps,ignored", [(True, 0.0, 0.0), (False, 0.1, 0.3)])
@pytest.mark.parametrize("N,K,V", SHAPES)
def test_mean(cuda, types, bias, eps, ignored, N, K, V):
    from video_classification_amd import ops
    x, w, b, t = make(N, K, V, types, bias=bias, ignored=ignored)
    xg = x.clone().requires_grad_(True)
    stats = {}
    loss = ops.linear_cross_entropy(xg, w, b, t, label_smoothing=eps, stats=stats)
    loss.backward()
    count = max(1, int((t != -100).sum()))
    ref = reference(x, w, b, t, eps, torch.full((N,), 1.0 / count, device=x.device))
    want = float(ref["rows"].sum() / count)
    assert abs(loss.item() - want) <= 4 * ref["dz"] + 2.0 ** -20 * (1 + float(ref["lse"].abs().max()))
    check(ref, types, None, xg.grad, w.grad, b.grad if bias else None)
    assert xg.grad.dtype == x.dtype and w.grad.dtype == w.dtype
    assert (xg.grad[t == -100] == 0).all()
    top = ref["z"].max(1).values
    picked = ref["z"].gather(1, stats["pred"][:, None])[:, 0]
    assert (top - picked <= 2 * ref["dz"]).all()
    assert int(stats["correct"]) == int(((stats["pred"] == t) & (t != -100)).sum())


@pytest.mark.gpu
@pytest.mark.parametrize("types", list(TYPES))
def test_rows_and_sum(cuda, types):
    from video_classification_amd import ops
    x, w, b, t = make(150, 96, 333, types, ignored=0.2)
    g = torch.randn(150, generator=torch.Generator().manual_seed(5)).cuda() * 3e-3
    xg = x.clone().requires_grad_(True)
    rows = ops.linear_cross_entropy(xg, w, b, t, reduction="none")
    assert rows.shape == (150,) and (rows[t == -100] == 0).all()
    rows.backward(g)
    ref = reference(x, w, b, t, 0.0, g)
    check(ref, types, rows.detach(), xg.grad, w.grad, b.grad)
    w.grad = b.grad = xg.grad = None
    loss = ops.linear_cross_entropy(xg.view(10, 15, 96), w, b, t.view(10, 15), reduction="sum")
    (loss * 0.25).backward()
    ref = reference(x, w, b, t, 0.0, torch.full((150,), 0.25, device=x.device))
    assert abs(loss.item() - float(ref["rows"].sum())) <= 150 * (4 * ref["dz"] + 2.0 ** -20 * (1 + float(ref["lse"].abs().max())))
    check(ref, types, None, xg.grad, w.grad, b.grad)


@pytest.mark.gpu
@pytest.mark.parametrize("types,N,K,V", [("bf16", 4096, 64, 13001), ("mixed", 3000, 48, 13000), ("f32", 2000, 40, 13100)])
def test_pieces_of_the_classes(cuda, types, N, K, V):
    from video_classification_amd import ops
    x, w, b, t = make(N, K, V, types)
    xg = x.clone().requires_grad_(True)
    loss = ops.linear_cross_entropy(xg, w, b, t)
    loss.backward()
    ref = reference(x, w, b, t, 0.0, torch.full((N,), 1.0 / N, device=x.device))
    assert abs(loss.item() - float(ref["rows"].mean())) <= 4 * ref["dz"] + 2.0 ** -20 * (1 + float(ref["lse"].abs().max()))
    check(ref, types, None, xg.grad, w.grad, b.grad)


@pytest.mark.gpu
def test_master_weights_beyond_bf16(cuda):
    """bf16 rows against fp32 weights that bf16 cannot hold: the weight's single fp16 term is off by 2^-12 of the value."""
    from video_classification_amd import ops
    x, w, b, t = make(200, 128, 500, "mixed")
    with torch.no_grad():
        w.mul_(1.2345)
    xg = x.clone().requires_grad_(True)
    ops.linear_cross_entropy(xg, w, b, t, reduction="sum").backward()
    ref = reference(x, w, b, t, 0.0, torch.ones(200, device=x.device))
    check(ref, "mixed", None, xg.grad, w.grad, b.grad, extra=2.0 ** -12 * float((ref["x"].abs() @ ref["w"].abs().t()).max()))


@pytest.mark.gpu
@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("xs,ws", [(1e-6, 1e3), (1e8, 1e-9), (1e-20, 1e20)])
def test_magnitudes(cuda, types, xs, ws):
    """Operands far from 1: the scales follow their magnitudes."""
    from video_classification_amd import ops
    x, w, b, t = make(70, 64, 150, types)
    x = (x.float() * xs).to(x.dtype)
    with torch.no_grad():
        w.copy_((w.float() * ws).to(TYPES[types][0]).to(w.dtype))
    xg = x.clone().requires_grad_(True)
    ops.linear_cross_entropy(xg, w, b, t).backward()
    ref = reference(x, w, b, t, 0.0, torch.full((70,), 1 / 70, device=x.device))
    check(ref, types, None, xg.grad, w.grad, b.grad)


@pytest.mark.gpu
@pytest.mark.parametrize("types", list(TYPES))
def test_ignored_rows_may_hold_anything(cuda, types):
    from video_classification_amd import ops
    x, w, b, t = make(200, 64, 150, types, ignored=0.4)
    bad = x.clone()
    drop = (t == -100).nonzero()[:, 0]
    bad[drop[0]], bad[drop[1]], bad[drop[2]] = float("nan"), float("inf"), torch.finfo(x.dtype).min
    outs = []
    for src in (x, bad):
        w.grad = b.grad = None
        xg = src.clone().requires_grad_(True)
        loss = ops.linear_cross_entropy(xg, w, b, t, label_smoothing=0.1)
        loss.backward()
        outs.append((loss.detach(), xg.grad, w.grad, b.grad))
    for a, c in zip(*outs):
        assert torch.isfinite(a).all() and torch.equal(a, c)
    # nothing counts: loss 0, gradients 0
    w.grad = b.grad = None
    xg = bad.clone().requires_grad_(True)
    loss = ops.linear_cross_entropy(xg, w, b, torch.full_like(t, -100))
    loss.backward()
    assert loss.item() == 0 and not xg.grad.any() and not w.grad.any() and not b.grad.any()


@pytest.mark.gpu
@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("low", [float("-inf"), "lowest"])
def test_classes_masked_by_the_bias(cuda, types, low):
    from video_classification_amd import ops
    x, w, b, t = make(150, 64, 400, types)
    low = float(torch.finfo(b.dtype).min) if low == "lowest" else low
    with torch.no_grad():
        b[128:300] = low
    t = torch.where((t >= 128) & (t < 300), t % 128, t)  # targets are live classes
    xg = x.clone().requires_grad_(True)
    rows = ops.linear_cross_entropy(xg, w, b, t, reduction="none")
    rows.sum().backward()
    live = torch.cat([torch.arange(128), torch.arange(300, 400)]).cuda()
    tl = torch.where(t >= 300, t - 172, t)
    ref = reference(x, w[live], b[live], tl, 0.0, torch.ones(150, device=x.device))
    check(ref, types, rows.detach(), xg.grad, w.grad[live], b.grad[live])
    assert not w.grad[128:300].any() and not b.grad[128:300].any()


@pytest.mark.gpu
def test_bad_values_show(cuda):
    """A target outside the classes and a NaN in a row that counts make the loss NaN and touch nothing out of bounds."""
    from video_classification_amd import ops
    x, w, b, t = make(64, 32, 40, "f32")
    for v in (40, -1, 2 ** 40, -2 ** 40):
        bad = t.clone()
        bad[5] = v
        rows = ops.linear_cross_entropy(x, w, b, bad, reduction="none")
        assert torch.isnan(rows[5]) and torch.isfinite(rows[:5]).all() and torch.isfinite(rows[6:]).all()
        xg = x.clone().requires_grad_(True)
        ops.linear_cross_entropy(xg, w, b, bad).backward()
        assert torch.isnan(xg.grad[5]).all() and torch.isfinite(xg.grad[6:]).all()
    x[7, 3] = float("nan")
    rows = ops.linear_cross_entropy(x, w, b, t, reduction="none")
    assert torch.isnan(rows[7]) and torch.isfinite(rows[:7]).all() and torch.isfinite(rows[8:]).all()


@pytest.mark.gpu
def test_gradient_against_differences(cuda):
    from video_classification_amd import ops
    x, w, b, t = make(40, 24, 60, "f32", ignored=0.2)
    g = torch.Generator().manual_seed(1)
    vx, vw, vb = (torch.randn(s.shape, generator=g).cuda().double() for s in (x, w, b))
    one = torch.ones(40, device=x.device)
    f = lambda h: reference_sum(x.double() + h * vx, w.detach().double() + h * vw, b.detach().double() + h * vb, t)
    h = 1e-5
    want = (f(h) - f(-h)) / (2 * h)
    xg = x.clone().requires_grad_(True)
    ops.linear_cross_entropy(xg, w, b, t, label_smoothing=0.1, reduction="sum").backward()
    parts = [(xg.grad.double() * vx).sum(), (w.grad.double() * vw).sum(), (b.grad.double() * vb).sum()]
    scale = sum(float((p.grad.double() * v).abs().sum()) for p, v in ((xg, vx), (w, vw), (b, vb)))
    assert abs(float(sum(parts)) - want) <= 1e-5 * scale and one.numel() == 40


def reference_sum(x, w, b, t, eps=0.1):
    return float(reference(x, w, b, t, eps, torch.ones(x.shape[0], device=x.device))["rows"].sum())


@pytest.mark.gpu
def test_views_accumulation_repeatability_and_stream(cuda):
    from video_classification_amd import ops
    x, w, b, t = make(100, 64, 300, "mixed")
    want = ops.linear_cross_entropy(x, w, b, t).detach()
    wide = torch.zeros(100, 130, device=cuda, dtype=x.dtype)
    wide[:, 1:65] = x
    assert torch.equal(ops.linear_cross_entropy(wide[:, 1:65], w, b, t).detach(), want)
    wt = w.detach().t().contiguous().t()
    assert not wt.is_contiguous() and torch.equal(ops.linear_cross_entropy(x, wt, b, t), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = ops.linear_cross_entropy(x, w, b, t).detach()
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(other, want)
    ops.linear_cross_entropy(x, w, b, t).backward()  # x needs no gradient: only the parameters'
    once = w.grad.clone(), b.grad.clone()
    ops.linear_cross_entropy(x, w, b, t).backward()
    assert torch.equal(w.grad, 2 * once[0]) and torch.equal(b.grad, 2 * once[1])
    # agrees with the operators it stands in for (a linear layer in bf16 and the loss of its logits)
    lin = nn.Linear(64, 300).cuda()
    with torch.no_grad():
        lin.weight.copy_(w)
        lin.bias.copy_(b)
    z = ops.linear(x, lin.weight, lin.bias, out_f32=True)[:, :300]
    assert abs(ops.cross_entropy(z, t).item() - want.item()) < 1e-3


@pytest.mark.gpu
def test_captured_step_replays(cuda):
    from video_classification_amd import ops
    x, w, b, t = make(300, 96, 500, "mixed", ignored=0.1)
    w.grad, b.grad = torch.zeros_like(w), torch.zeros_like(b)

    def step():
        w.grad.zero_()
        b.grad.zero_()
        xi = x.detach().requires_grad_(True)
        loss = ops.linear_cross_entropy(xi, w, b, t)
        return [loss.detach(), torch.autograd.grad(loss, xi)[0]]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        nx, _, _, nt = make(300, 96, 500, "mixed", ignored=0.3 * k, seed=20 + k)
        x.copy_(nx)
        t.copy_(nt)
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in out] + [w.grad.clone(), b.grad.clone()]
        want = step() + [w.grad.clone(), b.grad.clone()]
        for a, c in zip(got, want):
            assert torch.equal(a, c)


@pytest.mark.gpu
def test_refusals(cuda):
    from video_classification_amd import ops
    x, w, b, t = make(6, 16, 20, "f32")
    ce = ops.linear_cross_entropy
    with pytest.raises(TypeError, match="float32 weights"):
        ce(x, w.detach().bfloat16(), None, t)
    with pytest.raises(TypeError):
        ce(x.half(), w, b, t)
    with pytest.raises(RuntimeError, match="bias"):
        ce(x, w, b[:5], t)
    with pytest.raises(RuntimeError, match="bias"):
        ce(x, w, b.detach().bfloat16(), t)
    with pytest.raises(RuntimeError, match="rows"):
        ce(x[:, :8], w, b, t)
    with pytest.raises(RuntimeError, match="target"):
        ce(x, w, b, t[:5])
    with pytest.raises(RuntimeError, match="target"):
        ce(x, w, b, t.int())
    with pytest.raises(ValueError, match="label_smoothing"):
        ce(x, w, b, t, label_smoothing=1.5)
    with pytest.raises(ValueError, match="reduction"):
        ce(x, w, b, t, reduction="max")
    with pytest.raises(RuntimeError, match="tensors on"):
        ce(x, w, b, t.cpu())
    xe = x[:0].requires_grad_(True)
    empty = ce(xe, w, b, t[:0])
    assert empty.item() == 0
    empty.backward()
    assert xe.grad.shape == (0, 16) and w.grad is None


def test_refuses_cpu_and_bad_abi_arguments():
    from video_classification_amd import _lib as L
    from video_classification_amd import ops
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.linear_cross_entropy(torch.zeros(2, 8), torch.zeros(4, 8), None, torch.zeros(2, dtype=torch.int64))
    assert L.query("vc_linear_ce_bytes", 0, 1, 1, 0, 4, 8) == -1
    assert L.query("vc_linear_ce_bytes", 0, 0, 1, 2, 4, 8) == -1
    assert L.query("vc_linear_ce_bytes", 3, 1, 1, 2, 4, 8) == -1
    for what in (0, 1, 2):
        assert L.query("vc_linear_ce_bytes", what, 1, 0, 2, 4, 8) > 0
    null = L.ptr(None)

    def fwd(xd, wd, n, v, k, smooth=0.0):
        L.call("vc_linear_ce_fwd", xd, wd, null, null, null, null, L.i64(-100), float(smooth), 1, null, null, null, null, null,
               null, n, v, k, null)

    for args, code in (((0, 1, 2, 4, 8), -4), ((5, 1, 2, 4, 8), -2), ((1, 1, 0, 4, 8), -1), ((1, 1, 2, 4, 1 << 21), -1),
                       ((1, 1, 2, 4, 8), -4), ((1, 1, 2, 4, 8, 2.0), -4)):
        with pytest.raises(RuntimeError, match=f"status {code}"):
            fwd(*args)


def test_plan_covers_every_size():
    """Workspace sizes are positive and grow with the sizes (the pieces keep the gradient buffers bounded)."""
    from video_classification_amd import _lib as L
    for n, v, k in ((1, 1, 1), (16384, 65536, 2048), (4096, 13001, 64), (1 << 22, 7, 8), (3, 1 << 22, 8)):
        sizes = [L.query("vc_linear_ce_bytes", what, 1, 1, n, v, k) for what in (0, 1, 2)]
        assert all(s > 0 for s in sizes)
        assert sizes[0] >= 2 * (n + v) * k
    small = L.query("vc_linear_ce_bytes", 2, 1, 1, 8192, 65536, 64)
    assert small < (8192 + 65536) * 64 * 2 + (400 << 20)


@pytest.mark.gpu
def test_backward_passes_of_two_streams_follow_each_other(cuda):
    """Forward calls on two streams write the same parameter gradients: the second pass waits for the first."""
    from video_classification_amd import ops
    x, w, b, t = make(1000, 256, 5000, "mixed")
    ops.linear_cross_entropy(x, w, b, t).backward()
    once = [p.grad.clone() for p in (w, b)]
    w.grad = b.grad = None
    main, streams, losses = torch.cuda.current_stream(), [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        s.wait_stream(main)
        with torch.cuda.stream(s):
            losses.append(ops.linear_cross_entropy(x, w, b, t))
    torch.autograd.backward(losses)
    for p, a in zip((w, b), once):
        assert torch.equal(p.grad, 2 * a)


@pytest.mark.gpu
def test_computed_weights_sizes_and_empty_batches(cuda):
    from video_classification_amd import ops
    x, w, b, t = make(6, 16, 20, "f32")
    ce = ops.linear_cross_entropy
    with pytest.raises(RuntimeError, match="must be leaves"):
        ce(x, w * 2, b, t)
    with pytest.raises(RuntimeError, match="must be leaves"):
        ce(x, w, b + 1, t)
    with torch.no_grad():
        ce(x, w * 2, b + 1, t)
    n = (1 << 22) + 1
    with pytest.raises(RuntimeError, match="exceed"):
        ce(x[:1].expand(n, 16), w, b, t[:1].expand(n))
    with pytest.raises(RuntimeError, match="exceed"):
        ce(x[:, :1].expand(6, (1 << 20) + 1), w[:, :1].detach().expand(20, (1 << 20) + 1), b, t)
    with pytest.raises(ValueError, match="int64"):
        ce(x, w, b, t, ignore_index=1 << 64)
    for reduction in ("mean", "sum", "none"):  # nothing but the parameters needs gradients, and there are no rows
        loss = ce(x[:0], w, b, t[:0], reduction=reduction)
        assert loss.shape == ((0,) if reduction == "none" else ())
        loss.sum().backward()
        assert w.grad is None


@pytest.mark.gpu
@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("N,K,V,share", [(700, 72, 300, 0.85), (5000, 40, 130, 0.5), (4300, 64, 13001, 0.97), (130, 33, 50, 0.99),
                                         (300, 64, 257, 1.0), (9000, 16, 20, 0.3)])
def test_many_ignored_rows(cuda, types, N, K, V, share):
    """Most rows, whole tiles of them, or all: what is left is packed and comes back to its place."""
    from video_classification_amd import ops
    x, w, b, t = make(N, K, V, types, seed=3)
    drop = torch.rand(N, generator=torch.Generator().manual_seed(5)) < share
    t[drop.to(cuda)] = -100
    xg = x.clone().requires_grad_(True)
    xg.data[t == -100] = float("nan")  # never read
    stats = {}
    count = int((t != -100).sum())
    g = torch.randn(N, generator=torch.Generator().manual_seed(6)).to(cuda)
    rows = ops.linear_cross_entropy(xg, w, b, t, reduction="none", stats=stats)
    rows.backward(g)
    ref = reference(x, w, b, t, 0.0, g)
    check(ref, types, rows.detach(), xg.grad, w.grad, b.grad, one_term=FEW_ROWS)
    assert (xg.grad[t == -100] == 0).all() and (rows[t == -100] == 0).all() and (stats["pred"][t == -100] == 0).all()
    assert int(stats["correct"]) == int(((stats["pred"] == t) & (t != -100)).sum())
    xg.grad, w.grad, b.grad = None, None, None
    loss = ops.linear_cross_entropy(xg, w, b, t)
    loss.backward()
    ref = reference(x, w, b, t, 0.0, torch.full((N,), 1.0 / max(1, count), device=cuda))
    assert abs(loss.item() - float(ref["rows"].sum() / max(1, count))) <= 4 * ref["dz"] + 2.0 ** -20 * (1 + float(ref["lse"].abs().max()))
    check(ref, types, None, xg.grad, w.grad, b.grad, one_term=FEW_ROWS)
    if not count:
        assert not w.grad.any() and not b.grad.any()


@pytest.mark.gpu
def test_slices_of_few_rows(cuda):
    """dx is summed over more slices of the classes the fewer rows count; from all rows to one, in one buffer."""
    from video_classification_amd import ops
    x, w, b, t = make(1500, 130, 16500, "bf16", seed=9)
    for count in (1500, 1100, 700, 300, 129, 128, 1):
        tt = t.clone()
        tt[torch.randperm(1500, generator=torch.Generator().manual_seed(count))[count:].to(cuda)] = -100
        xg = x.clone().requires_grad_(True)
        ops.linear_cross_entropy(xg, w.detach(), b.detach(), tt, reduction="sum").backward()
        check(reference(x, w, b, tt, 0.0, torch.ones(1500, device=cuda)), "bf16", dx=xg.grad, one_term=FEW_ROWS)
        assert (xg.grad[tt == -100] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("types,N,K,V,eps", [("bf16", 300, 64, 257, 0.0), ("bf16", 1, 128, 1, 0.0), ("bf16", 777, 192, 2100, 0.2),
                                             ("bf16", 300, 72, 257, 0.1), ("mixed", 300, 64, 257, 0.0), ("f32", 90, 64, 300, 0.1)])
def test_without_gradients(cuda, types, N, K, V, eps):
    """A call that keeps nothing for a backward pass: bf16 operands with K a multiple of 64 are multiplied as they are."""
    from video_classification_amd import ops
    x, w, b, t = make(N, K, V, types, seed=12, ignored=0.4 if N > 1 else 0.0)
    x[t == -100] = float("inf")
    ref = reference(x, w, b, t, eps, torch.ones(N, device=cuda))
    count = max(1, int((t != -100).sum()))
    with torch.no_grad():
        stats = {}
        rows = ops.linear_cross_entropy(x, w, b, t, label_smoothing=eps, reduction="none", stats=stats)
        mean = ops.linear_cross_entropy(x, w, b, t, label_smoothing=eps)
        off = torch.empty(V * K + 1, device=cuda, dtype=w.dtype)[1:].view(V, K)  # a weight and rows off the 16-byte grid
        off.copy_(w)
        offx = torch.empty(N * K + 1, device=cuda, dtype=x.dtype)[1:].view(N, K)
        offx.copy_(x)
        shifted = ops.linear_cross_entropy(offx, off, b, t, label_smoothing=eps, reduction="none")
        moved, still = (ops.linear_cross_entropy(v, w, b, t, label_smoothing=eps, reduction="none") for v in (offx, x))
        bare = ops.linear_cross_entropy(x, w, None, t, reduction="sum")
    check(ref, types, rows)
    check(ref, types, shifted)
    assert torch.equal(moved, still)
    assert abs(mean.item() - float(ref["rows"].sum() / count)) <= 4 * ref["dz"] + 2.0 ** -20 * (1 + float(ref["lse"].abs().max()))
    live = t != -100
    top, picked = ref["z"].max(1).values, ref["z"].gather(1, stats["pred"][:, None])[:, 0]
    assert (top - picked <= 2 * ref["dz"])[live].all() and (stats["pred"][~live] == 0).all()
    assert int(stats["correct"]) == int(((stats["pred"] == t) & live).sum())
    plain = reference(x, w, None, t, 0.0, torch.ones(N, device=cuda))
    assert abs(bare.item() - float(plain["rows"].sum())) <= N * (4 * plain["dz"] + 2.0 ** -20 * (1 + float(plain["lse"].abs().max())))


@pytest.mark.gpu
def test_bf16_without_gradients_keeps_the_whole_range(cuda):
    """Rows of very different magnitude do not take precision from each other where bf16 operands are used as they are."""
    from video_classification_amd import ops
    x, w, b, t = make(200, 64, 300, "bf16", seed=13)
    want = torch.nn.functional.cross_entropy(x.double() @ w.detach().double().t() + b.detach().double(), t, reduction="none")
    big = x.clone()
    big[7] = 3e38
    with torch.no_grad():
        got = ops.linear_cross_entropy(big, w, b, t, reduction="none")
        alone = ops.linear_cross_entropy(x, w, b, t, reduction="none")
    keep = torch.arange(200, device=cuda) != 7
    assert torch.equal(got[keep], alone[keep])
    assert float((got.double() - want)[keep].abs().max()) < 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("types,N,K,V", [("bf16", 1500, 128, 9000), ("mixed", 260, 72, 300), ("f32", 300, 40, 700)])
def test_replays_follow_the_rows_that_count(cuda, types, N, K, V):
    """How many rows count is read on the device: one captured step serves every mask, from none to all rows."""
    from video_classification_amd import ops
    x, w, b, t = make(N, K, V, types, seed=21)
    xs, ts = x.clone().requires_grad_(True), t.clone()
    w.grad, b.grad, xs.grad = torch.zeros_like(w), torch.zeros_like(b), torch.zeros_like(xs)

    def step():
        for g in (w.grad, b.grad, xs.grad):
            g.zero_()
        loss = ops.linear_cross_entropy(xs, w, b, ts)
        loss.backward()
        with torch.no_grad():
            rows = ops.linear_cross_entropy(xs, w, b, ts, reduction="none")
        return loss.detach(), rows

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, rows = step()
    for k, share in enumerate((0.0, 0.9, 0.5, 1.0, 0.0, 0.3)):
        drop = torch.rand(N, generator=torch.Generator().manual_seed(k)) < share
        ts.copy_(torch.where(drop.to(cuda), torch.full_like(t, -100), t.roll(k)))
        graph.replay()
        torch.cuda.synchronize()
        got = [loss.clone(), rows.clone(), xs.grad.clone(), w.grad.clone(), b.grad.clone()]
        want = step()
        want = [want[0], want[1], xs.grad, w.grad, b.grad]
        for g, e in zip(got, want):
            assert torch.equal(g, e)


@pytest.mark.gpu
@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("e", [0, 12, 40])
def test_ties_of_large_logits(cuda, types, e):
    """Logits that are whole multiples of 2^e, so that from e = 12 on a row's probability falls in equal shares on the classes that
    tie for its maximum: the maximum takes nothing from the sum, however large it is.

    Every product and every logit is exact; the maximum and the target's logit meet a rounding each on their way through
    log2 (2^-22 of the larger with the factors'), the shares the error of exp2 and log2 (2^-20)."""
    from video_classification_amd import ops
    xd, wd = TYPES[types]
    N, K, V = 96, 32, 160
    g = torch.Generator().manual_seed(3)
    x = (torch.randint(-3, 4, (N, K), generator=g) * 2.0 ** (e // 2)).to(xd).cuda()
    w = torch.randint(-2, 3, (V, K), generator=g) * 2.0 ** (e - e // 2)
    w[80:] = w[:80]  # every maximum is met twice
    w = nn.Parameter(w.to(wd).cuda())
    t = torch.randint(0, V, (N,), generator=g).cuda()
    x64, w64 = x.double(), w.detach().double()
    z = x64 @ w64.t()
    p = torch.softmax(z, dim=1)
    d = p.clone()
    d[torch.arange(N), t] -= 1
    xg = x.clone().requires_grad_(True)
    rows = ops.linear_cross_entropy(xg, w, None, t, reduction="none")
    rows.sum().backward()
    want = torch.nn.functional.cross_entropy(z, t, reduction="none")
    assert ((rows.double() - want).abs() <= 2.0 ** -20 + 2.0 ** -22 * (z.max(1).values.abs() + z[torch.arange(N), t].abs())).all()
    # a share's error: 2^-20, and where the shares are unequal (e = 0) that of the logits in log2, 2^-22 of the largest
    share = p * (2.0 ** -20 + (2.0 ** -21 * float(z.abs().max()) if e == 0 else 0.0))
    for got, want, A, M, P, dt, n in ((xg.grad, d @ w64, d.abs(), w64.abs(), share, xd, V),
                                      (w.grad, d.t() @ x64, d.abs().t(), x64.abs(), share.t(), wd, N)):
        term = (2.0 ** -22 if dt == torch.float32 else FEW_ROWS) + 2.0 ** -21 + (3 * n / 32 + 8) * 2.0 ** -23
        # fp16's smallest step is 2^-24 and d is scaled by 2^15: whatever the terms, half a step is 2^-40
        floor = 2.0 ** -40 * (torch.ones_like(A) @ M)
        assert ((got.double() - want).abs() <= term * (A @ M) + P @ M + floor + half(dt) * want.abs()).all()


def check_each(types, x, w, b, t, rows, dx, dw, db, weight, skip=()):
    """Like `check`, with every logit's own error bound: rows and classes of any magnitude side by side.  skip: rows whose
    logits overflow, with weight 0."""
    xd, wd = TYPES[types]
    N, V, K = x.shape[0], w.shape[0], x.shape[1]
    live = torch.ones(N, dtype=torch.bool, device=x.device)
    live[list(skip)] = False
    x64, w64 = x.double() * live[:, None], w.detach().double()
    z, S = x64 @ w64.t() + b.detach().double(), x64.abs() @ w64.abs().t() + b.detach().double().abs()
    lse = torch.logsumexp(z, dim=1)
    p = torch.exp(z - lse[:, None])
    dz = ((3 * K / 32 + 4) * 2.0 ** -23 + 2.0 ** -21) * S
    mid = (p * dz).sum(1)
    at = torch.arange(N, device=x.device)
    want = lse - z[at, t]
    tol = 2 * (mid + dz[at, t]) + 2.0 ** -20 * (1 + lse.abs() + want.abs())
    err = (rows.double() - want).abs()
    assert (err <= tol)[live].all(), float((err - tol)[live].max())
    d = p.clone()
    d[at, t] -= 1
    # fp16's smallest step is 2^-24 and d is scaled by 2^15: half a step is 2^-40 of the row's weight (of the largest one where
    # they are within 2^16 of each other), or all of a smaller value
    size = (weight * live).abs()
    unit = size if size[size > 0].min() < 2.0 ** -16 * size.max() else size.max().expand(N)
    floor = torch.minimum(d.abs() * size[:, None], 2.0 ** -40 * unit[:, None])
    d = d * (weight * live)[:, None]
    off = (2 * p * (1 - p).clamp_min(0) * (dz + mid[:, None]) + 2.0 ** -20 * p) * size[:, None]
    for got, want, A, F, M, P, dt, length in ((dx, d @ w64, d.abs(), floor, w64.abs(), off, xd, V),
                                              (dw, d.t() @ x64, d.abs().t(), floor.t(), x64.abs(), off.t(), wd, N)):
        # joins of a sum: of 32 fp16 products each, or (rows of their own scale) one rounding per fp32 product
        term = (2.0 ** -22 if dt == torch.float32 else FEW_ROWS) + 2.0 ** -21 + (length + 8) * 2.0 ** -23
        tol = term * (A @ M) + F @ M + P @ M + half(dt) * want.abs() + 1e-37
        err = (got.double() - want).abs()
        assert (err <= tol).all(), float((err / tol).max())
    tol = off.sum(0) + (N / 16 + 16) * U * d.abs().sum(0) + half(wd) * d.sum(0).abs() + 1e-37
    assert ((db.double() - d.sum(0)).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("N,K,V", [(200, 64, 300), (77, 72, 130), (1500, 40, 700)])
@pytest.mark.parametrize("where", ["row", "class", "both", "near", "small row", "overflow"])
def test_magnitudes_of_rows_and_classes_side_by_side(cuda, types, N, K, V, where):
    """One row of x, or one class's weights, far larger than the others takes no precision from them, with gradients as
    without."""
    from video_classification_amd import ops
    x, w, b, t = make(N, K, V, types, seed=13)
    weight = torch.ones(N, device=cuda, dtype=torch.float64)
    with torch.no_grad():
        if where in ("row", "both"):
            x[7] *= 2.0 ** 40
        if where in ("class", "both"):
            w[11] *= 2.0 ** 40
        if where == "near":  # within one scale's reach
            x[7] *= 2.0 ** 14
            w[11] *= 2.0 ** 14
        if where == "small row":
            x[:-1] *= 2.0 ** 60
            w.mul_(2.0 ** -60)
        if where == "overflow":
            x[7], weight[7] = 3e38, 0.0
    xg = x.clone().requires_grad_(True)
    rows = ops.linear_cross_entropy(xg, w, b, t, reduction="none")
    rows.backward(weight.float())
    check_each(types, x, w, b, t, rows.detach(), xg.grad, w.grad, b.grad, weight, skip=[7] if where == "overflow" else [])
    with torch.no_grad():
        again = ops.linear_cross_entropy(x, w, b, t, reduction="none")
    keep = torch.ones(N, dtype=torch.bool, device=cuda)
    keep[7] = where != "overflow"
    scale = (rows.detach().abs() + again.abs())[keep]
    assert ((rows.detach() - again).abs()[keep] <= 2.0 ** -10 * (1 + scale)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("types,N,K,V", [("bf16", 3000, 64, 13001), ("f32", 200, 520, 4099)])
def test_magnitudes_in_pieces_and_slices(cuda, types, N, K, V):
    """The same where the classes come in pieces and the reductions in slices, next to a call without such rows."""
    from video_classification_amd import ops
    x, w, b, t = make(N, K, V, types, seed=14)
    one = torch.ones(N, device=cuda, dtype=torch.float64)
    for scale in (2.0 ** 40, 1.0):
        with torch.no_grad():
            big, wide = x.clone(), nn.Parameter(w.detach().clone())
            big[7] *= scale
            wide[11] *= scale
        b.grad = None
        xg = big.clone().requires_grad_(True)
        rows = ops.linear_cross_entropy(xg, wide, b, t, reduction="none")
        rows.sum().backward()
        check_each(types, big, wide, b, t, rows.detach(), xg.grad, wide.grad, b.grad, one)


@pytest.mark.gpu
def test_replays_follow_the_magnitudes(cuda):
    """Whether rows have scales of their own is found on the device: one captured step serves both."""
    from video_classification_amd import ops
    x, w, b, t = make(300, 96, 500, "bf16", seed=15)
    xs = x.clone().requires_grad_(True)
    w.grad, b.grad, xs.grad = torch.zeros_like(w), torch.zeros_like(b), torch.zeros_like(xs)

    def step():
        for g in (w.grad, b.grad, xs.grad):
            g.zero_()
        loss = ops.linear_cross_entropy(xs, w, b, t)
        loss.backward()
        return loss.detach()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step()
    for k in (0, 40, 0, 30, 0):
        with torch.no_grad():
            xs.copy_(x)
            xs[3] *= 2.0 ** k
        graph.replay()
        torch.cuda.synchronize()
        got = [loss.clone(), xs.grad.clone(), w.grad.clone(), b.grad.clone()]
        for g, e in zip(got, [step(), xs.grad, w.grad, b.grad]):
            assert torch.equal(g, e)


@pytest.mark.gpu
@pytest.mark.parametrize("types", list(TYPES))
def test_bias_gradient_of_many_rows(cuda, types):
    """Rows that are all alike: every tile of 128 rows has the sums of a call of 128 rows, bit for bit, and 10000 of them add
    nothing but the rounding of the result, and of the tile's sum in the smaller call's own type."""
    from video_classification_amd import ops
    grads = []
    for n in (128, 1280000):
        x, t = torch.zeros(n, 8, device=cuda, dtype=TYPES[types][0]), torch.zeros(n, dtype=torch.int64, device=cuda)
        w = nn.Parameter(torch.zeros(3, 8, device=cuda, dtype=TYPES[types][1]))
        b = nn.Parameter(torch.tensor([0.5, 0.1, -0.3], device=cuda).to(w.dtype))
        ops.linear_cross_entropy(x, w, b, t, reduction="sum").backward()
        grads.append(b.grad.double())
    want = 10000 * grads[0]
    assert ((grads[1] - want).abs() <= 2 * half(TYPES[types][1]) * want.abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("xs,ws,gs", [(2.0 ** -112, 2.0 ** 112, 1 / 3), (2.0 ** 112, 2.0 ** -112, 1 / 3), (2.0 ** -60, 2.0 ** 60, 2.0 ** -60 / 3),
                                      (1.0, 1.0, 2.0 ** -100 / 3)])
@pytest.mark.parametrize("N,K,V", [(70, 64, 150), (20, 520, 4099)])
def test_gradients_of_tiny_magnitude(cuda, types, xs, ws, gs, N, K, V):
    """Gradients close to the smallest normal number keep their relative accuracy: operands scaled by powers of two give the
    gradients of the unscaled ones, scaled."""
    from video_classification_amd import ops
    x, w, b, t = make(N, K, V, types, seed=16)
    ref = reference(x, w, b, t, 0.0, torch.full((N,), 1 / 3, device=x.device))
    x = x * xs
    with torch.no_grad():
        w.mul_(ws)
    xg = x.clone().requires_grad_(True)
    loss = ops.linear_cross_entropy(xg, w, b, t, reduction="sum")
    (loss * torch.tensor(gs, device=cuda)).backward()
    up = 3 * gs  # exact: gs is the float next to a power of two over three, and so is 1 / 3
    got = []
    for p, want, scale in ((xg, ref["dx"], ws * up), (w, ref["dw"], xs * up), (b, ref["db"], up)):
        # below 2^-126 a type has steps of 2^-126 eps: half of one belongs to the result's rounding
        half_step = 2.0 ** -126 * half(p.dtype) / scale
        g = p.grad.double() / scale
        got.append(g + (want - g).clamp(-half_step, half_step))
    check(ref, types, None, *got, one_term=FEW_ROWS)


def test_refuses_what_no_launch_can_hold():
    """A launch has fewer than 2^32 threads: sizes beyond that are refused before the first one, with a reason."""
    from video_classification_amd import _lib as L, ops
    for n, v, k, why in ((1 << 20, 1 << 18, 64, "tiles of logits"), (1 << 22, 1 << 22, 8, "tiles of logits"),
                         (1 << 17, 1 << 19, 1 << 17, "pieces of 512"), (1 << 20, 7, 1 << 15, "pieces of 512")):
        for what in (0, 1, 2, 4):
            assert L.query("vc_linear_ce_bytes", what, 1, 1, n, v, k) == -1
            with pytest.raises(RuntimeError, match=why):
                ops._size("vc_linear_ce_bytes", what, 1, 1, n, v, k)
    assert ops._size("vc_linear_ce_bytes", 0, 1, 1, (1 << 20) - 128, 1 << 18, 64) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("N,K,V", [(200, 64, 300), (1500, 40, 700), (90, 520, 4099)])
@pytest.mark.parametrize("e", [10, 40, -140])
def test_upstream_gradients_side_by_side(cuda, types, N, K, V, e):
    """One row's upstream gradient 2^e times the others', and one of zero: no row's gradient takes precision from another."""
    from video_classification_amd import ops
    x, w, b, t = make(N, K, V, types, seed=17)
    weight = torch.full((N,), -1 / 3, device=cuda)
    weight[7], weight[20] = 2.0 ** e, 0.0
    xg = x.clone().requires_grad_(True)
    rows = ops.linear_cross_entropy(xg, w, b, t, reduction="none")
    rows.backward(weight)
    check_each(types, x, w, b, t, rows.detach(), xg.grad, w.grad, b.grad, weight.double())
    assert not xg.grad[20].any()


@pytest.mark.gpu
@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("N,K,V", [(50, 64, 300), (70, 40, 128), (3, 8, 5)])
def test_nothing_left_by_lowest_values(cuda, types, N, K, V):
    """Every class at the type's lowest value: next to it no logit counts, the probabilities are all 1 / V; with a single class
    beside it that one takes all, and a target among the masked ones has a finite loss."""
    from video_classification_amd import ops
    x, w, b, t = make(N, K, V, types, seed=18)
    low = torch.finfo(b.dtype).min
    x64, w64 = x.double(), w.detach().double()
    at = torch.arange(N, device=cuda)
    for spared in (None, 2):
        with torch.no_grad():
            b.fill_(low)
            if spared is not None:
                b[spared] = 0.25
        w.grad = b.grad = None
        xg = x.clone().requires_grad_(True)
        stats = {}
        rows = ops.linear_cross_entropy(xg, w, b, t, reduction="none", stats=stats)
        rows.sum().backward()
        p = torch.full((N, V), 1.0 / V, device=cuda, dtype=torch.float64)
        if spared is None:
            assert ((rows.double() - torch.log(torch.tensor(float(V)))).abs() <= 2.0 ** -20 * 6).all()
        else:
            p.zero_()
            p[:, spared] = 1
            masked = t != spared
            assert torch.isfinite(rows).all() and (rows[masked] > 2e38).all() and (rows[~masked].abs() <= 2.0 ** -20).all()
        assert (stats["pred"] == (0 if spared is None else spared)).all()
        d = p.clone()
        d[at, t] -= 1
        off = 2.0 ** -20 * p
        for got, want, A, M, P, dt, n in ((xg.grad, d @ w64, d.abs(), w64.abs(), off, xg.dtype, V),
                                          (w.grad, d.t() @ x64, d.abs().t(), x64.abs(), off.t(), w.dtype, N)):
            term = (2.0 ** -22 if dt == torch.float32 else FEW_ROWS) + 2.0 ** -21 + (3 * n / 32 + 8) * 2.0 ** -23
            assert ((got.double() - want).abs() <= term * (A @ M) + P @ M + half(dt) * want.abs()).all()
        assert ((b.grad.double() - d.sum(0)).abs() <= off.sum(0) + (N / 16 + 16) * U * d.abs().sum(0) + half(b.dtype) * d.sum(0).abs()).all()
        with torch.no_grad():
            assert torch.allclose(ops.linear_cross_entropy(x, w, b, t, reduction="none"), rows.detach(), rtol=1e-6, atol=1e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("N,K,V", [(1, 1 << 18, 3), (2, 100001, 1), (3, 4096, 130), (200, 64, 150)])
def test_no_row_counts(cuda, types, N, K, V):
    """Every row ignored: no product is worked, whatever is not there is not read, and loss and gradients are zeros."""
    from video_classification_amd import ops
    x, w, b, t = make(N, K, V, types, seed=19)
    t = torch.full_like(t, -100)
    for reduction in ("mean", "sum", "none"):
        w.grad = b.grad = None
        xg = x.clone().requires_grad_(True)
        stats = {}
        loss = ops.linear_cross_entropy(xg, w, b, t, reduction=reduction, label_smoothing=0.1, stats=stats)
        loss.sum().backward()
        with torch.no_grad():
            again = ops.linear_cross_entropy(x, w, b, t, reduction=reduction)
        for v in (loss.detach(), again, xg.grad, w.grad, b.grad, stats["pred"], stats["correct"]):
            assert not v.any() and torch.isfinite(v.double()).all()
