"""What programs may hand the training operators beside ordinary tensors: nodes called directly, hooks, dual numbers, copies and
saved states of optimizers, values at the ends of their types. Refused before any device work, or computed by the formulas."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEVICE = 'cuda:0'


def test_embedding_node_checks_its_upstream():
    """A node called directly passes autograd's own checks by: shapes and devices that the kernels would read past are refused."""
    import efgs
    indices = torch.randint(0, 9, (5, 3), device=DEVICE)
    table = torch.randn(9, 4, device=DEVICE, requires_grad=True)
    out = efgs.embedding(indices, table)
    for upstream in (torch.ones(5, 2, 4, device=DEVICE), torch.ones(15, 4, device=DEVICE), torch.ones(1, device=DEVICE), torch.ones(5, 3, 5, device=DEVICE)):
        with pytest.raises(ValueError, match="the output's shape"):
            out.grad_fn(upstream)
    with pytest.raises(ValueError, match="on the gradient's device"):
        out.grad_fn(torch.ones(5, 3, 4))
    with pytest.raises(ValueError, match='float32, bfloat16 or float16'):
        out.grad_fn(torch.ones(5, 3, 4, device=DEVICE, dtype=torch.float64))
    got = out.grad_fn(torch.ones(5, 3, 4, device=DEVICE))
    got = got[0] if isinstance(got, tuple) else got
    assert torch.equal(got, torch.bincount(indices.reshape(-1), minlength=9).float()[:, None].expand(9, 4))


def test_embedding_node_checks_what_hooks_give_back():
    """Hooks on saved tensors that return the indices on the host, or as floats, are refused; in other strides they are read right."""
    import efgs
    indices = torch.randint(0, 9, (6, 5), device=DEVICE)
    table = torch.randn(9, 4, device=DEVICE, requires_grad=True)
    upstream = torch.randn(6, 5, 4, device=DEVICE)
    want = torch.autograd.grad(efgs.embedding(indices, table), table, upstream)[0]
    for unpack in (lambda x: x.cpu(), lambda x: x.float(), lambda x: x.short()):
        with torch.autograd.graph.saved_tensors_hooks(lambda x: x, unpack):
            out = efgs.embedding(indices, table)
        with pytest.raises(ValueError, match='indices'):
            out.backward(upstream)
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda x: x.t().contiguous().t()):
        out = efgs.embedding(indices, table)
    assert torch.equal(torch.autograd.grad(out, table, upstream)[0], want)


@pytest.mark.parametrize('requires_grad', [False, True])
@pytest.mark.parametrize('grad_mode', [False, True])
def test_embedding_of_a_dual_number_is_refused(requires_grad, grad_mode):
    """There is no forward-mode derivative: an error, as the rasterizer's, and no result without a tangent."""
    import efgs
    from torch.autograd import forward_ad
    indices = torch.randint(0, 9, (5,), device=DEVICE)
    table = torch.randn(9, 4, device=DEVICE, requires_grad=requires_grad)
    with torch.set_grad_enabled(grad_mode), forward_ad.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError)):
            efgs.embedding(indices, forward_ad.make_dual(table, torch.ones_like(table)))
        assert efgs.embedding(indices, table).shape == (5, 4)
