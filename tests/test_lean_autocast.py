"""ops/act8.py and ops/linear_xent.py under autocast on the CPU: fp32 operands are computed in fp32, as on the
GPU, and bf16 weights take the input in their type."""
import pytest
import torch

from vodascheduler_amd.ops.act8 import linear_act8
from vodascheduler_amd.ops.linear_xent import linear_cross_entropy


def _inputs(dtype):
    g = torch.Generator().manual_seed(0)
    x, w, b = (torch.randn(*s, generator=g).to(dtype).requires_grad_() for s in ((12, 40), (30, 40), (30,)))
    return x, w, b, torch.randint(0, 30, (12,), generator=g)


def _layer(autocast, x, w, b, act):
    with torch.autocast("cpu", dtype=torch.bfloat16, enabled=autocast):
        y = linear_act8(x, w, b, act)
    return (y.detach(), *torch.autograd.grad(y.float().square().sum(), (x, w, b)))


def _loss(autocast, x, w, b, labels):
    with torch.autocast("cpu", dtype=torch.bfloat16, enabled=autocast):
        loss, correct, n = linear_cross_entropy(x, w, labels, b)
    return (loss.detach(), correct, n, *torch.autograd.grad(loss, (x, w, b)))


@pytest.mark.parametrize("rows", [12, 0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_same_bits_under_autocast(dtype, rows):
    x, w, b, labels = _inputs(dtype)
    x, labels = x.detach()[:rows].requires_grad_(), labels[:rows]
    for run, more in ((_layer, (None,)), (_layer, ("gelu",)), (_loss, (labels,))):
        want, got = run(False, x, w, b, *more), run(True, x, w, b, *more)
        for o, r in zip(got, want):
            assert o.dtype == r.dtype and torch.equal(o, r)


def test_an_fp32_input_of_bf16_weights():
    x, w, b, labels = _inputs(torch.bfloat16)
    wide = x.detach().float().requires_grad_()
    for run, more in ((_layer, (None,)), (_loss, (labels,))):
        want, got = run(False, x, w, b, *more), run(True, wide, w, b, *more)
        assert all(torch.equal(o.float(), r.float()) for o, r in zip(got, want))
