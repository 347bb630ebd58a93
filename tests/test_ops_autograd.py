"""The operators' forward functions beside torch's autograd: a gradient is never lost silently."""
import pytest
import torch

from nnv_b200 import ops


@pytest.mark.parametrize("which", [0, 1, 2])
def test_tensors_that_require_a_gradient_are_refused(which):
    x, s, o = (torch.zeros(n, dtype=torch.float32) for n in ((4, 8), 8, 8))
    (x, s, o)[which].requires_grad_()
    with pytest.raises(ValueError, match="autograd"):
        ops.layer_norm(x, s, o)
    q, k, v = (torch.zeros(2, 3, 4, 8) for _ in range(3))
    (q, k, v)[which].requires_grad_()
    with pytest.raises(ValueError, match="autograd"):
        ops.cross_attention(q, k, v)
    with torch.no_grad(), pytest.raises(ValueError, match="no CPU path"):        # past the check
        ops.cross_attention(q, k, v)


@pytest.mark.gpu
def test_under_no_grad_and_with_explicit_gradients():
    x = torch.randn(5, 16, device="cuda", requires_grad=True)
    w = torch.nn.Parameter(torch.randn(16, device="cuda"))
    q = torch.randn(2, 3, 4, 16, device="cuda", requires_grad=True)
    with torch.no_grad():
        y, mean, rstd = ops.layer_norm(x, w, None, return_stats=True)
        out, lse = ops.cross_attention(q, q, q, return_lse=True)
    assert torch.equal(y, ops.layer_norm(x.detach(), w.detach()))
    grads = (*ops.layer_norm_backward(y, x, w, mean, rstd), *ops.cross_attention_backward(out, q, q, q, out, lse))
    assert not any(g.requires_grad for g in grads)
