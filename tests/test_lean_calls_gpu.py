"""Calls of the memory-lean operators that their documentation allows: fp32 operands with a bf16 bias, a backward
pass that runs twice, an input or bias that changes after the forward."""
import pytest
import torch

from vodascheduler_amd.ops.act8 import linear_act8
from vodascheduler_amd.ops.linear_xent import linear_cross_entropy

import test_act8_gpu as A
import test_linear_xent_gpu as X

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float32]


@pytest.mark.parametrize("rows", [20, 700])
def test_fp32_with_a_bf16_bias(rows):
    x, w, b, y = X._inputs(rows, 72, 300, 290, torch.float32, bias=True)
    _, grads = X._check(x, w, b.detach().bfloat16().requires_grad_(), y, 290)
    assert grads[2].dtype == torch.bfloat16
    x, w, b, dy = A._inputs(rows, 72, 48, torch.float32, bias=True)
    assert A._check(x, w, b.detach().bfloat16().requires_grad_(), dy, "gelu")[3].dtype == torch.bfloat16


@pytest.mark.parametrize("dtype", TYPES)
def test_the_backward_twice(dtype):
    x, w, b, y = X._inputs(200, 72, 300, 290, dtype, bias=True)
    loss = linear_cross_entropy(x, w, y, b, 290)[0]
    first, second = (torch.autograd.grad(loss, (x, w, b), retain_graph=True) for _ in range(2))
    assert all(torch.equal(p, q) for p, q in zip(first, second))
    x, w, b, dy = A._inputs(200, 72, 48, dtype, bias=True)
    for act in (None, "gelu"):
        out = linear_act8(x, w, b, act)
        first, second = (torch.autograd.grad(out, (x, w, b), dy, retain_graph=True) for _ in range(2))
        assert all(torch.equal(p, q) for p, q in zip(first, second))


@pytest.mark.parametrize("dtype", TYPES)
def test_what_changes_between_forward_and_backward(dtype):
    """Of the input and the bias the operators keep their own copies; a weight that changed is an error."""
    x, w, b, y = X._inputs(200, 72, 300, 290, dtype, bias=True)
    want = torch.autograd.grad(linear_cross_entropy(x, w, y, b, 290)[0], (x, w, b))
    loss = linear_cross_entropy(x, w, y, b, 290)[0]
    keep = y.clone()
    with torch.no_grad():
        x.zero_(), b.zero_(), y.zero_()
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(loss, (x, w, b)), want))
    loss = linear_cross_entropy(x, w, keep, b, 290)[0]
    with torch.no_grad():
        w.zero_()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, (x, w, b))
    x, w, b, dy = A._inputs(200, 72, 48, dtype, bias=True)
    want = torch.autograd.grad(linear_act8(x, w, b, "gelu"), (x, w, b), dy)
    out = linear_act8(x, w, b, "gelu")
    with torch.no_grad():
        x.zero_(), b.zero_()
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(out, (x, w, b), dy), want))
    out = linear_act8(x, w, b, "gelu")
    with torch.no_grad():
        w.zero_()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out, (x, w, b), dy)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_batch_no_row_of_which_is_labelled_onto_flat_gradients(dtype):
    """Nothing is added, and the engine is told all the same."""
    from vodascheduler_amd.utils.flat import FlatGroup, grad_of

    for rows in (20, 700):
        x, w, b, y = X._inputs(rows, 72, 300, 290, dtype, bias=True)
        w, b = torch.nn.Parameter(w.detach()), torch.nn.Parameter(b.detach())
        group = FlatGroup([w, b])  # noqa: F841  (owns the gradients)
        seen = []
        for t in (w, b):
            t._voda_grad_ready = lambda q: seen.append(q)
            grad_of(t).fill_(0.5)
        loss, correct, n = linear_cross_entropy(x, w, torch.full_like(y, -100), b, 290)
        loss.backward()
        assert float(loss.detach()) == 0.0 and int(correct) == int(n) == 0 and len(seen) == 2
        assert float(x.grad.abs().max()) == 0.0
        assert all(torch.equal(grad_of(t), torch.full_like(grad_of(t), 0.5)) for t in (w, b))
