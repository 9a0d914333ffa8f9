"""CudaArray around torch tensors: from_torch keeps the memory, not the tensor
object, and to_torch returns a view of its own."""
import pytest

import phptensors as P

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def test_views_are_their_own_objects():
    t = torch.randn(6, 16, device="cuda")
    a = P.CudaArray.from_torch(t)
    v = a.to_torch()
    assert v is not t and v.data_ptr() == t.data_ptr()
    v.unsqueeze_(0)
    v.requires_grad_()
    assert list(t.shape) == [6, 16] and not t.requires_grad
    assert list(a.to_torch().shape) == [6, 16] and not a.to_torch().requires_grad
    y = a.layer_norm()                       # and a result's
    v = y.to_torch().unsqueeze_(0).requires_grad_()
    assert list(y.to_torch().shape) == [6, 16] and not y.to_torch().requires_grad
    v.data[0, 0, 0] = 5.0                    # the memory is shared
    assert y.to_torch()[0, 0] == 5.0
    a.to_torch()[1, 2] = 7.0
    assert t[1, 2] == 7.0


def test_a_tensor_that_changes_after_it_was_wrapped():
    """`tensor.data = ...` (a module's .to() or .half()) and in-place changes of
    its shape leave the array on the memory and the shape it was given."""
    t = torch.nn.Parameter(torch.randn(6, 16, device="cuda"), requires_grad=False)
    first = t.detach().clone()
    at = t.data_ptr()
    a = P.CudaArray.from_torch(t)
    t.data = torch.zeros(6, 16, device="cuda")
    assert a.to_torch().data_ptr() == at and torch.equal(a.to_torch(), first)
    assert torch.equal(a.layer_norm().to_torch(), P.CudaArray.from_torch(first).layer_norm().to_torch())
    b = torch.randn(2, 3, 5, device="cuda")
    a = P.CudaArray.from_torch(b)
    b.transpose_(0, 2)
    assert a.getShape() == [2, 3, 5] and list(a.to_torch().shape) == [2, 3, 5]
    assert torch.equal(a.to_torch(), b.transpose(0, 2))


def test_a_tensor_of_a_graph():
    """What autograd knows of a wrapped tensor reaches the view, as before."""
    t = torch.randn(4, 8, device="cuda", requires_grad=True)
    v = P.CudaArray.from_torch(t).to_torch()
    assert v.requires_grad
    v.sum().backward()
    assert torch.equal(t.grad, torch.ones_like(t))
    with torch.no_grad():
        assert torch.equal(P.CudaArray.from_torch(t).transpose().to_torch(), t.t())


def test_slices_and_offsets():
    base = torch.randn(10, 12, device="cuda").bfloat16()
    a = P.CudaArray.from_torch(base[2:7, 1:9])
    assert torch.equal(a.to_torch(), base[2:7, 1:9]) and a.getStrides() == [12, 1]
    assert torch.equal(a.transpose().to_torch(), base[2:7, 1:9].t())
    assert a.view([3], [12], 5).to_torch().data_ptr() == base.data_ptr() + 10
