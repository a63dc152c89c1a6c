"""GPU tests of the class losses at the edges of what they take: infinite and
lowest table entries, infinite and vanishing upstream gradients, saved-tensor
hooks, forward mode, long sums, and float32 results held to float32's own
rounding (test_gpu_class_losses.py has the definition over all shapes)."""
import pytest
import torch

from tests.test_gpu_class_losses import BF16, DTYPES, F16, F32, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,V,D,dtype", [
    (300, 37, 0, F32), (20, 1500, 0, BF16), (300, 20, 4, F32), (300, 1003, 72, BF16),
    (100, 1003, 72, F16), (300, 203, 40, F32), (3, 500, 64, BF16), (17000, 9, 100, F32)])
@pytest.mark.parametrize("form", ["offset", "strided"])
def test_saved_tensor_hooks(n, V, D, dtype, form):
    """What the backward gets back from a hook may lie anywhere: off every
    alignment, or with other strides."""
    from gs_voxelizer_b200 import losses
    fn = losses.linear_cross_entropy if D else losses.softmax_cross_entropy
    data, labels = make(n, V, D, dtype, 54, ignored=0.2, garbage=False)
    leaves = [t.requires_grad_(True) for t in data]
    want = torch.autograd.grad(fn(*leaves, labels), leaves)

    def unpack(t):
        if form == "offset":
            flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
            flat[1:] = t.reshape(-1)
            return flat[1:].view(t.shape)
        return torch.stack([t, t], -1)[..., 0]

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), unpack):
        loss = fn(*leaves, labels)
    got = torch.autograd.grad(loss, leaves, retain_graph=True)
    again = torch.autograd.grad(loss, leaves)
    for a, b, c, t in zip(got, again, want, leaves):
        assert torch.equal(a, b)
        # (where a row's words begin decides the order of its sums)
        tol = 2.0 ** {F32: -20, BF16: -7, F16: -10}[dtype]
        assert torch.allclose(a.float(), c.float(), rtol=tol, atol=tol * float(c.abs().max()))
