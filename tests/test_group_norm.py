"""ops.group_norm against the definition in 64 bits, its refusals, and the guard that keeps a capture away from leaves of
a live eager graph.

Tolerances.  u = 2^-24 is half a step of fp32.  A normalised value carries the rounding of the mean, r u with r = |mean| /
spread, and a handful of roundings of its own; sums over R rows are joined pairwise over at most 64 consecutive rows.  A
bf16 result adds half a step, 2^-8 of the value."""
import types

import pytest
import torch
import torch.nn as nn

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def act64(z, act):
    if act == "relu":
        return torch.relu(z)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    return z


def ref64(x, gn, act, res):
    """The definition in float64 (also on autograd): x [N, ..., C]."""
    N, C = x.shape[0], x.shape[-1]
    u = x.reshape(N, -1, gn.num_groups, C // gn.num_groups)
    mu = u.mean(dim=(1, 3), keepdim=True)
    var = ((u - mu) ** 2).mean(dim=(1, 3), keepdim=True)
    z = ((u - mu) / torch.sqrt(var + gn.eps)).reshape(x.shape)
    if gn.weight is not None:
        z = z * gn.weight.double() + gn.bias.double()
    if res is not None:
        z = z + res
    sd = torch.sqrt(var + gn.eps).detach()
    return act64(z, act), float((mu.detach().abs() / sd).max()), float(1 / sd.min()), z


def make(shape, groups, dt, seed=0, shift=0.5, affine=True):
    g = torch.Generator().manual_seed(seed)
    C = shape[-1]
    x = (torch.randn(*shape, generator=g) * (0.5 + torch.rand(C, generator=g)) + shift).to(dt)
    gn = nn.GroupNorm(groups, C, affine=affine)
    if affine:
        with torch.no_grad():
            gn.weight.copy_(1 + 0.3 * torch.randn(C, generator=g))
            gn.bias.copy_(0.3 * torch.randn(C, generator=g))
    res = torch.randn(*shape, generator=g).to(dt)
    dy = torch.randn(*shape, generator=g).to(dt)
    return x, gn, res, dy


SHAPES = [((2, 1, 7, 7, 64), 8), ((1, 3, 5, 9, 24), 8), ((3, 1, 33, 17, 40), 5), ((2, 1, 1, 1, 32), 4), ((5, 16), 16),
          ((2, 37, 7), 7), ((2, 11, 30), 5), ((1, 5000, 8), 1), ((2, 3, 2304), 2), ((1, 1), 1), ((4, 1, 56, 56, 32), 4),
          ((1, 2, 4104), 3), ((130, 9, 16), 2), ((2, 700, 256), 32), ((2, 1, 57, 55, 128), 1), ((3, 200, 8), 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("act,use_res", [("none", False), ("relu", True), ("silu", False), ("silu", True), ("gelu", True)])
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_forward_backward(cuda, dt, act, use_res, shape, groups):
    from video_classification_amd import ops
    x, gn, res, dy = make(shape, groups, DT[dt])
    res = res if use_res else None
    x64 = x.double().requires_grad_(True)
    r64 = res.double().requires_grad_(True) if use_res else None
    gr = nn.GroupNorm(groups, shape[-1]).double()
    gr.load_state_dict(gn.state_dict())
    y64, r, rstd, z64 = ref64(x64, gr, act, r64)
    if act == "relu":
        # the kernels decide on z, rounded differently: keep the gradient away from the corner
        near = z64.detach().abs() < 1e-3
        dy = torch.where(near, torch.zeros_like(dy), dy)
    y64.backward(dy.double())
    gn.to(cuda)
    xm = x.to(cuda).requires_grad_(True)
    rm = res.to(cuda).requires_grad_(True) if use_res else None
    y = ops.group_norm(xm, gn, act, rm)
    assert y.shape == x.shape and y.dtype == x.dtype
    y.backward(dy.to(cuda))
    half = U if dt == "f32" else 2.0 ** -8
    zmax = float(z64.detach().abs().max()) + 1
    dzmax = float(dy.abs().max()) * 1.2 * 2
    step = U * (64 + 8 * r)
    for got, want, scale in ((y.detach(), y64.detach(), zmax), (xm.grad, x64.grad, rstd * dzmax * zmax)):
        err = (got.cpu().double() - want).abs()
        assert (err <= half * want.abs() + step * scale).all(), float((err - half * want.abs()).max() / scale)
    if use_res:
        err = (rm.grad.cpu().double() - r64.grad).abs()
        assert (err <= half * r64.grad.abs() + step * dzmax * zmax).all()
    rows = x.numel() // shape[-1]
    for got, want in ((gn.weight.grad, gr.weight.grad), (gn.bias.grad, gr.bias.grad)):
        assert (got.cpu().double() - want).abs().max() <= step * rows * dzmax * zmax / min(rows, 16) ** 0.5


@pytest.mark.gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("shape,groups", [((2, 1, 20, 20, 64), 8), ((2, 333, 24), 8)])
@pytest.mark.parametrize("shift", [1000.0, -40.0])
def test_large_mean_does_not_cancel(cuda, dt, shape, groups, shift):
    from video_classification_amd import ops
    x, gn, _, _ = make(shape, groups, DT[dt], shift=shift)
    y64, r, _, z = ref64(x.double(), nn.GroupNorm(groups, shape[-1]), "none", None)
    with torch.no_grad():
        y = ops.group_norm(x.to(cuda), nn.GroupNorm(groups, shape[-1]).to(cuda))
    half = U if dt == "f32" else 2.0 ** -8
    assert ((y.cpu().double() - y64).abs() <= half * y64.abs() + U * (64 + 8 * r) * float(z.detach().abs().max())).all()


@pytest.mark.gpu
def test_gradient_against_differences(cuda):
    """Directional derivative of the float64 definition by central differences, against the kernels' gradients."""
    from video_classification_amd import ops
    x, gn, res, dy = make((2, 1, 6, 5, 24), 6, torch.float32, seed=3)
    g = torch.Generator().manual_seed(9)
    v = torch.randn(x.shape, generator=g).double()
    f = lambda t: (ref64(x.double() + t * v, gn.double(), "silu", res.double())[0] * dy.double()).sum()
    h = 1e-5
    want = float((f(h) - f(-h)) / (2 * h))
    gn.float().to(cuda)
    xm = x.to(cuda).requires_grad_(True)
    ops.group_norm(xm, gn, "silu", res.to(cuda)).backward(dy.to(cuda))
    got = float((xm.grad.cpu().double() * v).sum())
    assert abs(got - want) <= 1e-5 * float((xm.grad.cpu().double() * v).abs().sum())


@pytest.mark.gpu
def test_views_streams_accumulation_and_no_affine(cuda):
    from video_classification_amd import ops
    x, gn, _, dy = make((3, 1, 9, 8, 32), 4, torch.bfloat16)
    gn.to(cuda)
    xc = x.to(cuda)
    want = ops.group_norm(xc, gn, "gelu")
    # a transposed view and a view whose memory starts off the 16-byte grid
    t = xc.permute(0, 3, 1, 2, 4).contiguous().permute(0, 2, 3, 1, 4)
    assert not t.is_contiguous() and torch.equal(ops.group_norm(t, gn, "gelu"), want)
    flat = torch.empty(xc.numel() + 1, device=cuda, dtype=xc.dtype)
    off = flat[1:].view(xc.shape)
    off.copy_(xc)
    assert off.data_ptr() % 16 != 0
    assert (ops.group_norm(off, gn, "gelu").float() - want.float()).abs().max() <= 2 * 2.0 ** -8 * want.float().abs().max()
    # the current stream is the one that is used
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = ops.group_norm(xc, gn, "gelu")
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(other, want)
    # only parameters need gradients; they add up over calls, and repeat bit for bit
    dyc = dy.to(cuda)
    ops.group_norm(xc, gn, "gelu").backward(dyc)
    once = [gn.weight.grad.clone(), gn.bias.grad.clone()]
    ops.group_norm(xc, gn, "gelu").backward(dyc)
    for a, p in zip(once, (gn.weight, gn.bias)):
        assert torch.equal(p.grad, 2 * a)
    bare = nn.GroupNorm(4, 32, affine=False)
    y64 = ref64(x.double(), bare, "none", None)[0]
    y = ops.group_norm(xc, bare)
    assert y.grad_fn is None and ((y.cpu().double() - y64).abs() <= 2.0 ** -8 * y64.abs() + 1e-5).all()


@pytest.mark.gpu
def test_nan_and_inf_stay_in_their_sample(cuda):
    from video_classification_amd import ops
    x, gn, _, _ = make((4, 30, 32), 4, torch.float32)
    gn.to(cuda)
    clean = ops.group_norm(x.to(cuda), gn, "relu")
    x[1, 3, 2], x[2, 0, 8] = float("nan"), float("inf")
    y = ops.group_norm(x.to(cuda), gn, "relu")
    assert torch.isnan(y[1, :, :8]).all() and torch.isnan(y[2, :, 8:16]).all()
    for i, c in ((0, slice(0, 32)), (3, slice(0, 32)), (1, slice(8, 32)), (2, slice(16, 32)), (2, slice(0, 8))):
        assert torch.equal(y[i][:, c], clean[i][:, c])


@pytest.mark.gpu
def test_captured_forward_and_backward_replay(cuda):
    from video_classification_amd import ops
    x, gn, res, dy = make((4, 1, 12, 12, 64), 8, torch.bfloat16)
    gn.to(cuda)
    for p in gn.parameters():
        p.grad = torch.zeros_like(p)
    xs, rs, dys = x.to(cuda), res.to(cuda), dy.to(cuda)

    def step():
        for p in gn.parameters():
            p.grad.zero_()
        xi, ri = xs.detach().requires_grad_(True), rs.detach().requires_grad_(True)
        y = ops.group_norm(xi, gn, "silu", ri)
        return [y.detach(), *torch.autograd.grad(y, (xi, ri), dys)]

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
        xs.copy_(make((4, 1, 12, 12, 64), 8, torch.bfloat16, seed=10 + k)[0])
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out] + [p.grad.clone() for p in gn.parameters()]
        want = step() + [p.grad.clone() for p in gn.parameters()]
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_refusals(cuda):
    from video_classification_amd import ops
    gn = nn.GroupNorm(4, 32).to(cuda)
    x = torch.zeros(2, 3, 32, device=cuda)
    with pytest.raises(ValueError, match="act must be"):
        ops.group_norm(x, gn, act="tanh")
    with pytest.raises(RuntimeError, match="does not end in 32"):
        ops.group_norm(x[..., :24], gn)
    with pytest.raises(RuntimeError, match="residual"):
        ops.group_norm(x, gn, residual=x[:1])
    with pytest.raises(RuntimeError, match="residual"):
        ops.group_norm(x, gn, residual=x.bfloat16())
    with pytest.raises(TypeError):
        ops.group_norm(x.half(), gn)
    with pytest.raises(TypeError, match="float32"):
        ops.group_norm(x, nn.GroupNorm(4, 32).to(cuda).bfloat16())
    with pytest.raises(RuntimeError, match="tensors on"):
        ops.group_norm(x, nn.GroupNorm(4, 32))
    assert ops.group_norm(x[:0], gn).shape == (0, 3, 32)
    xg = x.clone().requires_grad_(True)
    g = torch.autograd.grad(ops.group_norm(xg, gn).sum(), xg, create_graph=True)[0]
    assert not g.requires_grad or pytest.raises(RuntimeError, torch.autograd.grad, g.sum(), xg)


def test_refuses_cpu_and_bad_abi_arguments():
    from video_classification_amd import _lib as L
    from video_classification_amd import ops
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.group_norm(torch.zeros(2, 3, 32), nn.GroupNorm(4, 32))
    null = L.ptr(None)
    args = (null, null, null, null, null, null, null, null)
    for dims, code in (((2, 3, 30, 4), -1), ((0, 3, 32, 4), -1), ((2, 0, 32, 4), -1), ((70000, 3, 32, 4), -1),
                       ((2, 3, 32, 4), -4)):
        with pytest.raises(RuntimeError, match=f"status {code}"):
            L.call("vc_group_norm_fwd", 1, *args, *dims, 1e-5, 0, null)
    with pytest.raises(RuntimeError, match="status -2"):
        L.call("vc_group_norm_fwd", 7, *args, 2, 3, 32, 4, 1e-5, 0, null)
    with pytest.raises(RuntimeError, match="unknown activation"):
        L.call("vc_group_norm_fwd", 1, *args, 2, 3, 32, 4, 1e-5, 9, null)
    assert L.query("vc_group_norm_workspace_floats", 0, 3, 32, 4) == 0
    assert L.query("vc_group_norm_workspace_floats", 2, 3, 32, 4) >= 2 * (2 * 32 + 2 * 32 + 8)


def test_leaf_guard(monkeypatch):
    """A leaf met eagerly may not be met by a capture while that eager graph lives; afterwards it may."""
    from video_classification_amd import ops
    x = torch.zeros(3, requires_grad=True)
    alive = x * 2
    ops._leaf_guard("op", x, None)
    monkeypatch.setattr(ops, "_capturing", lambda t: True)
    with pytest.raises(RuntimeError, match="eager graph is still alive"):
        ops._leaf_guard("op", x)
    ops._leaf_guard("op", x.detach().requires_grad_(True))
    with torch.no_grad():
        ops._leaf_guard("op", x)
    del alive
    ops._leaf_guard("op", x)


def test_anchor_only_for_parameters_alone():
    from video_classification_amd import ops
    p, x = nn.Parameter(torch.zeros(2)), torch.zeros(2)
    assert ops._anchor((x, None), (p, None)).requires_grad
    assert ops._anchor((x.requires_grad_(True),), (p,)) is None
    assert ops._anchor((torch.zeros(2),), (types.SimpleNamespace(requires_grad=False),)) is None
    with torch.no_grad():
        assert ops._anchor((torch.zeros(2),), (p,)) is None


@pytest.mark.gpu
def test_more_samples_than_one_launch_takes(cuda):
    """65535 samples go into one call of the library; more of them are the same as two calls that add up."""
    from video_classification_amd import ops
    N, cut = 70001, 65535
    x, gn, res, dy = (t.to(cuda) for t in make((N, 3, 16), 4, torch.float32))
    got = []
    for parts in (((0, N),), ((0, cut), (cut, N))):
        gn.zero_grad()
        row = []
        for a, b in parts:
            xs, rs = x[a:b].clone().requires_grad_(True), res[a:b].clone().requires_grad_(True)
            y = ops.group_norm(xs, gn, "silu", rs)
            y.backward(dy[a:b])
            row.append((y.detach(), xs.grad, rs.grad))
        got.append([torch.cat(c) for c in zip(*row)] + [gn.weight.grad.clone(), gn.bias.grad.clone()])
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert (got[0][0][cut:].double() - act64(ref64(x[cut:].double(), gn, "none", res[cut:].double())[3], "silu")).abs().max() < 1e-4


@pytest.mark.gpu
def test_backward_passes_of_two_streams_follow_each_other(cuda):
    """Forward calls on two streams write the same parameter gradients: the second pass waits for the first."""
    from video_classification_amd import ops
    x, gn, _, dy = (t.to(cuda) for t in make((64, 1, 56, 56, 64), 8, torch.bfloat16))
    ops.group_norm(x, gn, "relu").backward(dy)
    once = [p.grad.clone() for p in gn.parameters()]
    gn.zero_grad()
    main, streams, ys = torch.cuda.current_stream(), [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        s.wait_stream(main)
        with torch.cuda.stream(s):
            ys.append(ops.group_norm(x, gn, "relu"))
    torch.autograd.backward(ys, [dy, dy])
    for p, a in zip(gn.parameters(), once):
        assert torch.equal(p.grad, 2 * a)
    ops.group_norm(x, gn, "relu").backward(dy)  # and the default stream after them
    for p, a in zip(gn.parameters(), once):
        assert torch.equal(p.grad, 2 * a + a)


@pytest.mark.gpu
def test_refuses_computed_parameters_and_sizes(cuda):
    from video_classification_amd import ops
    x = torch.zeros(2, 3, 32, device=cuda)
    w = torch.ones(32, device=cuda, requires_grad=True)
    gn = types.SimpleNamespace(num_groups=4, num_channels=32, eps=1e-5, weight=w * 2, bias=None)
    with pytest.raises(RuntimeError, match="must be leaves"):
        ops.group_norm(x, gn)
    with torch.no_grad():
        assert ops.group_norm(x, gn).shape == x.shape
    wide = types.SimpleNamespace(num_groups=1, num_channels=(1 << 20) + 8, eps=1e-5, weight=None, bias=None)
    with pytest.raises(RuntimeError, match="exceed"):
        ops.group_norm(torch.zeros(1, 1, device=cuda).expand(1, (1 << 20) + 8), wide)
    gn.weight, gn.num_groups, gn.num_channels = None, 1, 1
    with pytest.raises(RuntimeError, match="exceed"):
        ops.group_norm(torch.zeros(1, 1, 1, device=cuda).expand(1, (1 << 32) + 1, 1), gn)


def test_runs_of_samples_cover_them_once():
    from video_classification_amd import ops
    for n in (1, 65535, 65536, 131070, 200000):
        runs = list(ops._gn_runs(n, 24))
        assert sum(k for _, k, _ in runs) == n and all(0 < k <= 65535 and o == 24 * a for a, k, o in runs)
        assert [a for a, _, _ in runs] == [sum(k for _, k, _ in runs[:i]) for i in range(len(runs))]


@pytest.mark.gpu
def test_parameter_gradients_of_many_samples(cuda):
    """One value per sample and channel, 65535 times the same: the join of the samples adds nothing but the rounding of its
    result (half a step, 2^-24), and of the two runs' sums where the gradients are added to."""
    from video_classification_amd import ops
    N, C = 65535, 16
    gn = nn.GroupNorm(2, C).to(cuda)
    x = torch.arange(C, device=cuda, dtype=torch.float32).repeat(N, 1)
    dy = torch.full((N, C), 0.1, device=cuda)
    for times in (1, 2):
        ops.group_norm(x, gn).backward(dy)
        want = times * N * dy[0].double()
        assert ((gn.bias.grad.double() - want).abs() <= times * U * want).all()
        xh = ops.group_norm(x[:1], nn.GroupNorm(2, C, affine=False)).double()[0]
        want = times * N * dy[0].double() * xh
        # dy * xhat is rounded once per sample, the same way in each
        assert ((gn.weight.grad.double() - want).abs() <= (times + 2) * U * want.abs()).all()


@pytest.mark.gpu
def test_more_slabs_than_a_launch_holds(cuda):
    """65535 rows of 16384 channels are 33 million slabs of 256 threads: the two-pass form takes them."""
    from video_classification_amd import ops
    N, C, G = 65535, 16384, 512
    gn = nn.GroupNorm(G, C).to(cuda)
    x = torch.empty(N, C, device=cuda).uniform_(-1, 3)
    pick = torch.tensor([0, 1, 777, N // 2, N - 2, N - 1], device=cuda)
    xg = x.requires_grad_(True)
    y = ops.group_norm(xg, gn, "relu")
    x64 = x.detach()[pick].double().requires_grad_(True)
    want = torch.relu(torch.nn.functional.group_norm(x64, G, eps=gn.eps))
    assert (y.detach()[pick].double() - want).abs().max() < 1e-5
    y.backward(torch.ones((), device=cuda).expand_as(y))
    want.backward(torch.ones_like(want))
    # next to the corner of ReLU a rounding decides about a whole gradient; elsewhere the norm's gradient holds to 1e-5
    err = (xg.grad[pick].double() - x64.grad).abs()
    assert float((err > 1e-4).double().mean()) < 1e-3


# Groups of 1 to 64 channels in slabs of one group and of several, as wide as a line (many samples) or narrowed (few), with the
# register counts of every size of the one-pass kernels; the layers of a ResNet trunk with 32 groups.
SLABS = [((300, 49, 64), 64), ((300, 49, 64), 32), ((300, 49, 64), 16), ((300, 49, 64), 8), ((300, 9, 128), 4),
         ((40, 9, 256), 16), ((16, 25, 1024), 32), ((8, 16, 2048), 32), ((2, 49, 512), 8), ((1, 120, 64), 1),
         ((1, 510, 64), 1), ((1, 1020, 32), 1), ((1, 9001, 8), 1), ((1, 9001, 8), 4), ((1, 9001, 8), 8), ((2, 4500, 16), 1),
         ((1, 3000, 32), 1), ((1, 1700, 64), 1), ((2, 1, 56, 56, 256), 32), ((3, 1, 28, 28, 512), 32), ((4, 1, 14, 14, 1024), 32),
         ((5, 1, 7, 7, 2048), 32), ((270, 768), 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("act,use_res", [("none", False), ("relu", True), ("silu", True), ("gelu", False)])
@pytest.mark.parametrize("shape,groups", SLABS)
def test_slabs(cuda, dt, act, use_res, shape, groups):
    test_forward_backward(cuda, dt, act, use_res, shape, groups)
