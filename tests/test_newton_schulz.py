"""ops.newton_schulz against the definition in 64 bits, and its refusals.

Tolerance.  A step stores X, S and P in 22 bits and sums K-term products in fp32, whose roundings of random sign grow with
sqrt(K): a relative perturbation of at most (4 + 3 sqrt(K) / 16) 2^-22 of |X_k|_F per step.  What step k perturbs is
amplified by at most `slope` (the polynomial's slope at 0, its largest) per step that is left, so the result is off by at most
sum_k slope^(steps - k) (4 + ...) 2^-22 |X_k|_F in the Frobenius norm, and by half a step of its own type."""
import pytest
import torch

C = (3.4445, -4.7750, 2.0315)
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def reference(g, steps=5, coeffs=C, eps=1e-7):
    x = g.double()
    x = x / (x.norm() + eps)
    per = [coeffs] * steps if not isinstance(coeffs[0], tuple) else coeffs
    norms = [float(x.norm())]
    for a, b, c in per:
        s = x @ x.t() if x.shape[0] <= x.shape[1] else x.t() @ x
        p = b * s + c * (s @ s)
        x = a * x + (p @ x if x.shape[0] <= x.shape[1] else x @ p)
        norms.append(float(x.norm()))
    return x, norms


def close(got, g, steps=5, coeffs=C, eps=1e-7):
    want, norms = reference(g.cpu(), steps, coeffs, eps)
    slope = max(1.0, max(abs(c[0]) for c in ([coeffs] if not isinstance(coeffs[0], tuple) else coeffs)))
    unit = (4 + 3 * max(g.shape) ** 0.5 / 16) * 2.0 ** -22
    tol = sum(slope ** (steps - k) * unit * n for k, n in enumerate(norms))
    err = (got.cpu().double() - want).norm()
    assert float(err) <= tol + torch.finfo(got.dtype).eps / 2 * float(want.norm()) + 1e-40, (float(err), tol)
    return want


def gaussian(m, n, seed=0):
    return torch.randn(m, n, generator=torch.Generator().manual_seed(seed))


def low_rank(m, n, seed=0):
    r = max(1, min(m, n) // 8)
    return gaussian(m, r, seed) @ gaussian(r, n, seed + 1) + 0.01 * gaussian(m, n, seed + 2)


SHAPES = [(1, 1), (1, 7), (7, 1), (3, 3), (64, 64), (75, 32), (32, 75), (64, 576), (130, 257), (257, 130), (128, 128),
          (129, 127), (300, 1000), (1000, 5), (2, 2050)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("kind", [gaussian, low_rank])
@pytest.mark.parametrize("m,n", SHAPES)
def test_shapes(cuda, dt, kind, m, n):
    from video_classification_amd import ops
    g = kind(m, n).to(DT[dt]).to(cuda)
    keep = g.clone()
    out = ops.newton_schulz(g)
    assert out.shape == g.shape and out.dtype == g.dtype and torch.equal(g, keep)
    close(out, g)


@pytest.mark.gpu
def test_singular_values_reach_one(cuda):
    from video_classification_amd import ops
    s = torch.linalg.svdvals(ops.newton_schulz(gaussian(96, 200).to(cuda)).cpu().double())
    assert 0.6 < float(s.min()) and float(s.max()) < 1.25


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-30, 1e-12, 3e-7, 1e-3, 1e4, 1e18, 1e30])
def test_scales(cuda, scale):
    """eps matters only next to it, and no size over- or underflows on the way."""
    from video_classification_amd import ops
    g = (gaussian(60, 90).double() * scale).float().to(cuda)
    close(ops.newton_schulz(g), g)
    close(ops.newton_schulz(g, eps=0.0), g, eps=0.0)


@pytest.mark.gpu
def test_many_matrices_share_a_call(cuda):
    from video_classification_amd import ops
    shapes = [(3 + 7 * i % 90, 5 + 11 * i % 140) for i in range(70)]
    mats = [gaussian(m, n, i).to(cuda) for i, (m, n) in enumerate(shapes)]
    outs = ops.newton_schulz(mats)
    assert isinstance(outs, list)
    for o, g in zip(outs, mats):
        close(o, g)
        assert torch.equal(o, ops.newton_schulz(g))  # alone or in company, bit for bit
    batch = torch.stack([gaussian(33, 20, 100 + i) for i in range(130)]).view(2, 65, 33, 20).to(cuda)
    out = ops.newton_schulz((batch,))
    assert isinstance(out, tuple) and out[0].shape == batch.shape
    for i in (0, 64, 65, 129):
        close(out[0].view(130, 33, 20)[i], batch.view(130, 33, 20)[i])


@pytest.mark.gpu
def test_views_streams_and_empty(cuda):
    from video_classification_amd import ops
    g = gaussian(70, 150).to(cuda)
    want = ops.newton_schulz(g)
    t = g.t().contiguous().t()
    assert not t.is_contiguous() and torch.equal(ops.newton_schulz(t), want)
    wide = torch.zeros(70, 160, device=cuda)
    wide[:, 3:153] = g
    assert torch.equal(ops.newton_schulz(wide[:, 3:153]), want)
    flat = torch.empty(70 * 150 + 1, device=cuda)
    flat[1:] = g.reshape(-1)
    assert torch.equal(ops.newton_schulz(flat[1:].view(70, 150)), want)
    # the other orientation is the same matrix transposed, to the last bit
    assert torch.equal(ops.newton_schulz(g.t().contiguous()), want.t())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = ops.newton_schulz(g)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(other, want)
    assert ops.newton_schulz([]) == []
    e = ops.newton_schulz([g[:0], g, torch.zeros(0, 3, 4, device=cuda)])
    assert e[0].shape == (0, 150) and e[2].shape == (0, 3, 4) and torch.equal(e[1], want)


@pytest.mark.gpu
def test_coefficients_and_steps(cuda):
    from video_classification_amd import ops
    g = gaussian(50, 120).to(cuda)
    for steps, coeffs in ((0, C), (1, C), (2, C), (7, C), (12, (1.5, -0.5, 0.0)),
                          (3, [(4.0, -6.0, 2.5), (3.0, -3.5, 1.5), (1.875, -1.25, 0.375)])):
        close(ops.newton_schulz(g, steps=steps, coeffs=coeffs), g, steps, coeffs)


@pytest.mark.gpu
def test_zero_nan_and_inf(cuda):
    from video_classification_amd import ops
    z, g = torch.zeros(20, 30, device=cuda), gaussian(40, 30).to(cuda)
    bad, inf = g.clone(), g.clone()
    bad[3, 4], inf[0, 0] = float("nan"), float("inf")
    out = ops.newton_schulz([z, bad, g, inf])
    assert not out[0].any() and torch.isnan(out[1]).all() and torch.isnan(out[3]).all()
    close(out[2], g)


@pytest.mark.gpu
def test_captured_call_replays(cuda):
    from video_classification_amd import ops
    mats = [gaussian(64, 100).to(cuda), gaussian(150, 40).to(cuda)]
    ops.newton_schulz(mats)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.newton_schulz(mats)
    for k in range(3):
        mats[0].copy_(gaussian(64, 100, 5 + k))
        mats[1].copy_(low_rank(150, 40, 5 + k))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        for a, b in zip(got, ops.newton_schulz(mats)):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_refusals_on_the_device(cuda):
    from video_classification_amd import ops
    g = gaussian(4, 5).to(cuda)
    with pytest.raises(TypeError):
        ops.newton_schulz(g.half())
    with pytest.raises(TypeError, match="in one call"):
        ops.newton_schulz([g, g.bfloat16()])
    with pytest.raises(RuntimeError, match="two dimensions"):
        ops.newton_schulz(g[0])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.newton_schulz([g, g.cpu()])
    assert not ops.newton_schulz(g.requires_grad_(True)).requires_grad


def test_refusals():
    from video_classification_amd import _lib as L
    from video_classification_amd import ops
    g = torch.zeros(3, 4)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.newton_schulz(g)
    for kw, what in ((dict(steps=-1), "steps"), (dict(steps=65), "steps"), (dict(eps=-1.0), "eps"),
                     (dict(steps=2, coeffs=[C]), "coeffs"), (dict(coeffs=[(1.0, 2.0)] * 5), "coeffs"),
                     (dict(coeffs=(30.0, 1.0, 1.0)), "grow")):
        with pytest.raises(ValueError, match=what):
            ops.newton_schulz(g, **kw)
    null = L.ptr(None)
    one, two = L.int_array([3]), L.int_array([4])
    pa = L.ptr_array([0])

    def call(dtype=0, count=1, rows=one, steps=5, cap=1.2, gain=500.0, pmax=3.0, ws=null):
        L.call("vc_newton_schulz", dtype, count, pa, pa, rows, two, steps, L.float_array([0.0] * 15), L.f64(1e-7), float(cap),
               float(gain), float(pmax), ws, null)

    for kw, code in ((dict(dtype=3), -2), (dict(count=0), -4), (dict(rows=L.int_array([0])), -1),
                     (dict(rows=L.int_array([1 << 21])), -1), (dict(), -4)):
        with pytest.raises(RuntimeError, match=f"status {code}"):
            call(**kw)
    assert L.query("vc_newton_schulz_bytes", 0, one, two) == -1
    assert L.query("vc_newton_schulz_bytes", 1, one, two) > 0


def test_bounds_of_the_coefficients():
    from video_classification_amd import ops
    cap, gain, pmax = ops._ns_bounds((C,) * 5)
    assert 1.202 < cap < 1.24 and 484 < gain < 496 and 2.80 < pmax < 2.95
    cap, gain, _ = ops._ns_bounds(((1.5, -0.5, 0.0),) * 5)
    assert cap == pytest.approx(1.02) and 7.5 < gain < 7.8


@pytest.mark.gpu
def test_refuses_shared_memory_in_place(cuda):
    from video_classification_amd import ops
    buf = torch.randn(3 * 20, 30, generator=torch.Generator().manual_seed(0)).to(cuda)
    a, b = buf[:20], buf[20:40]
    for pair in ([a, a], [a, buf[19:39]], [buf, b]):
        with pytest.raises(RuntimeError, match="share no memory"):
            ops.newton_schulz(pair, inplace=True)
    want = ops.newton_schulz([a, a, b])  # out of place the same matrix may come twice
    assert torch.equal(want[0], want[1])
    ops.newton_schulz([b, a], inplace=True)  # neighbours share nothing
    assert torch.equal(a, want[0]) and torch.equal(b, want[2])
    with pytest.raises(RuntimeError, match="exceed"):
        ops.newton_schulz(buf[:1, :1].expand(2, (1 << 20) + 1))


def test_disjoint():
    from video_classification_amd import ops
    buf = torch.zeros(4, 6)
    ops._disjoint("op", [buf[2:], buf[:2], buf[:0]])
    for pair in ([buf, buf], [buf[:3], buf[2:]], [buf, buf[1:2]]):
        with pytest.raises(RuntimeError, match="share no memory"):
            ops._disjoint("op", pair)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", list(DT))
def test_large_tiles(cuda, dt):
    """A call with enough work for the large tiles: odd shapes, tall and wide, whole and cut reductions beside a big matrix."""
    from video_classification_amd import ops
    shapes = [(2053, 2100), (130, 257), (257, 130), (129, 127), (300, 1000), (700, 64), (40, 2050), (64, 576), (384, 384)]
    mats = [gaussian(m, n, i).to(DT[dt]).to(cuda) for i, (m, n) in enumerate(shapes)]
    outs = ops.newton_schulz(mats)
    for o, g in zip(outs[1:], mats[1:]):
        close(o, g)
    want, norms = reference(mats[0])
    unit = (4 + 3 * 2100 ** 0.5 / 16) * 2.0 ** -22
    tol = sum(C[0] ** (5 - k) * unit * float(n) for k, n in enumerate(norms)) + torch.finfo(DT[dt]).eps / 2 * float(want.norm())
    assert float((outs[0].double() - want).norm()) <= tol


@pytest.mark.gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("m,n", [(4033, 4040), (4100, 4000)])
def test_last_round_of_a_large_matrix(cuda, dt, m, n):
    """More than 512 tiles of a symmetric product: those of the last round are cut along the reduction, the others are whole."""
    from video_classification_amd import ops
    g = gaussian(m, n, 5).to(DT[dt]).to(cuda)
    out = ops.newton_schulz(g)
    want, norms = reference(g)
    unit = (4 + 3 * max(m, n) ** 0.5 / 16) * 2.0 ** -22
    tol = sum(C[0] ** (5 - k) * unit * float(v) for k, v in enumerate(norms)) + torch.finfo(DT[dt]).eps / 2 * float(want.norm())
    assert float((out.double() - want).norm()) <= tol
    # every entry, for a wrong tile could hide in the norm of them all: 485 times a step's 16 x 2^-22 is 2^-9, the result's own
    # rounding another 2^-9, relative to entries of the largest's size
    assert float((out.double() - want).abs().max()) <= 2.0 ** -7 * float(want.abs().max())
    assert torch.equal(out, ops.newton_schulz(g))


@pytest.mark.gpu
def test_bits_repeat_for_the_same_set(cuda):
    """The same matrices in the same call give the same bits, cut reductions or not; in other company the reductions may be cut
    elsewhere, and the results agree within the tolerance only."""
    from video_classification_amd import ops
    shapes = [(64, 576), (128, 1152), (256, 2304), (512, 4608), (512, 512), (1000, 64)]
    mats = [gaussian(m, n, i).to(cuda) for i, (m, n) in enumerate(shapes)]
    first, second = ops.newton_schulz(mats), ops.newton_schulz(mats)
    for a, b, g in zip(first, second, mats):
        assert torch.equal(a, b)
        close(a, g)
        close(ops.newton_schulz(g), g)
