"""rotary_embed under autograd.  The map is linear and its gradient is its transpose, so both are held to the
64-bit formula within the bounds of test_rotary_gpu, and to differences of the map itself: for a linear map
(f(x + d) - f(x - d)) / 2 is f(d) but for the roundings of 32 bits: two of x +- d, three in each map on terms of
twice max |x|, three in the gradient, under 2^-20 of |w| max (|x| + 1) together."""
from __future__ import annotations

import pytest
import torch

from qwen_mla_vllm_b200 import ops  # noqa: F401
from qwen_mla_vllm_b200.rotary import rotary_embed, rotary_steps
from test_rotary_gpu import check, expect

pytestmark = pytest.mark.gpu
CASES = [(5, 3, 40, 32, 3, 1, 1.0), (130, 24, 232, 58, 0, 4, 1.3), (7, 2, 64, 64, 0, 1, 1.0)]  # tokens, heads, dim, rot, start, blocks, scale


def case(dev, tokens, heads, dim, rot, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x, w = (torch.randn(tokens, heads, dim, generator=g).to(dtype).to(dev) for _ in range(2))
    pos = torch.randint(-50, 100000, (tokens,), generator=g).to(dev)
    return x, w, pos, rotary_steps(rot, 1e4, device=dev)[0]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,heads,dim,rot,start,blocks,scale", CASES)
def test_the_gradient_is_the_transpose(cuda_device, tokens, heads, dim, rot, start, blocks, scale, dtype, interleaved):
    x, w, pos, steps = case(cuda_device, tokens, heads, dim, rot, dtype)
    how = dict(start=start, blocks=blocks, interleaved=interleaved, scale=scale)
    x.requires_grad_()
    for adjoint in (False, True):
        y = rotary_embed(x, pos, steps, adjoint=adjoint, **how)
        assert y.requires_grad
        check(y.detach(), *expect(x, pos, steps, start, blocks, interleaved, adjoint, scale), dtype)
        gx, = torch.autograd.grad(y, x, w)
        check(gx, *expect(w, pos, steps, start, blocks, interleaved, not adjoint, scale), dtype)


@pytest.mark.parametrize("interleaved", [False, True])
def test_the_gradient_against_differences(cuda_device, interleaved):
    x, w, pos, steps = case(cuda_device, 6, 2, 40, 32, torch.float32)
    how = dict(start=4, interleaved=interleaved)
    xr = x.clone().requires_grad_()
    gx, = torch.autograd.grad(rotary_embed(xr, pos, steps, **how), xr, w)
    for k in range(40):  # one dim of every token and head at a time
        d = torch.zeros_like(x)
        d[..., k] = 1.0
        diff = (rotary_embed(x + d, pos, steps, **how).double() - rotary_embed(x - d, pos, steps, **how).double()) / 2
        got, want = (w.double() * diff).sum(-1), gx[..., k].double()
        assert ((got - want).abs() <= 2.0**-20 * (w.abs().double() * (x.abs() + 1).amax(-1, keepdim=True)).sum(-1)).all()


@pytest.mark.parametrize("op", [False, True])
def test_the_gradient_has_a_gradient(cuda_device, op):
    x, w, pos, steps = case(cuda_device, 9, 3, 64, 58, torch.float32)
    x.requires_grad_(), w.requires_grad_()
    y = torch.ops.qmla.rotary(x, pos, steps, 2, 1, False, 1.0, False) if op else rotary_embed(x, pos, steps, start=2)
    gx, = torch.autograd.grad(y, x, w, create_graph=True)
    v = torch.randn(x.shape, generator=torch.Generator().manual_seed(5)).to(cuda_device)
    gw, = torch.autograd.grad(gx, w, v)  # the map itself, of v
    check(gw, *expect(v, pos, steps, 2, 1, False), torch.float32)


def test_expanded_gradients_and_two_dims(cuda_device):
    x, _, pos, steps = case(cuda_device, 9, 3, 64, 64, torch.float32)
    x.requires_grad_()
    rotary_embed(x, pos, steps).sum().backward()  # a gradient with strides of zero
    check(x.grad, *expect(torch.ones_like(x), pos, steps, 0, 1, False, True), torch.float32)
    z = x.detach()[:, 0].clone().requires_grad_()
    rotary_embed(z, pos, steps).sum().backward()
    check(z.grad[:, None], *expect(torch.ones_like(z)[:, None], pos, steps, 0, 1, False, True), torch.float32)


def test_out_stays_outside(cuda_device):
    x, _, pos, steps = case(cuda_device, 9, 3, 64, 64, torch.float32)
    want = rotary_embed(x, pos, steps)
    assert not want.requires_grad
    x.requires_grad_()
    with pytest.raises(RuntimeError):
        rotary_embed(x, pos, steps, out=torch.empty_like(x))
    with torch.no_grad():
        out = torch.empty_like(x)
        assert torch.equal(rotary_embed(x, pos, steps, out=out), want)
        assert torch.equal(rotary_embed(x, pos, steps), want)
