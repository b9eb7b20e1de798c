"""Forward-mode derivatives: the operators that bypass autograd where no gradient is needed refuse dual tensors instead of
dropping their tangents.  Runs on the CPU: the refusal comes before any launch."""
import pytest
import torch
import torch.autograd.forward_ad as fwd
import torch.nn as nn


@pytest.fixture
def ops(monkeypatch):
    from video_classification_amd import ops
    monkeypatch.setattr(ops, "_require_cuda", lambda t, what: None)

    def fast(name, *args):
        raise AssertionError(f"{name} launched")

    monkeypatch.setattr(ops.L, "fast", fast)
    monkeypatch.setattr(ops.L, "call", fast)
    monkeypatch.setattr(ops, "_on", lambda device: ops._HERE)
    return ops


def calls(ops):
    torch.manual_seed(0)
    gn, frozen = nn.GroupNorm(4, 16), nn.GroupNorm(4, 16).requires_grad_(False)
    w, b, t = torch.randn(5, 16), torch.randn(5), torch.tensor([0, 1, 4])
    return [
        ("trainable group norm", lambda x: ops.group_norm(x, gn)),
        ("frozen group norm", lambda x: ops.group_norm(x, frozen)),
        ("residual", lambda x: ops.group_norm(torch.zeros(3, 16), frozen, "relu", x)),
        ("loss", lambda x: ops.linear_cross_entropy(x, w, b, t)),
        ("loss of its weight", lambda x: ops.linear_cross_entropy(torch.zeros(3, 16), x, None, torch.tensor([0, 1, 2]))),
        ("orthogonalisation", lambda x: ops.newton_schulz(x)),
    ]


@pytest.mark.parametrize("which", range(6))
@pytest.mark.parametrize("grad", [True, False])
def test_dual_tensors_are_refused(ops, which, grad):
    what, call = calls(ops)[which]
    with torch.set_grad_enabled(grad), fwd.dual_level():
        x = fwd.make_dual(torch.randn(3, 16), torch.randn(3, 16))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(x)


@pytest.mark.parametrize("which", [1, 3, 5])
def test_transforms_are_refused(ops, which):
    what, call = calls(ops)[which]
    with pytest.raises(RuntimeError):
        torch.func.jvp(call, (torch.randn(3, 16),), (torch.randn(3, 16),))


@pytest.mark.parametrize("which", [1, 3])
def test_plain_tensors_inside_a_level_reach_the_kernels(ops, which):
    what, call = calls(ops)[which]
    with fwd.dual_level(), pytest.raises(AssertionError, match="launched"):
        call(torch.randn(3, 16))
