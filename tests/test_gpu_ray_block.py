"""The residual block that runs the block operators together (ray_block.py) against torch autograd."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def reference(block, x, region, live):
    """The block in float64 with autograd, from the 16-bit copies of the weights.  live: which hidden units
    of which rows the block found positive (one within rounding of zero may fall on either side, and its
    gradient with it)."""
    p = {k: (block.w16[k] if k in block.w16 else block.params[k]).double().requires_grad_() for k in block.params}
    xr = x.double().requires_grad_()
    b, s, d = x.shape
    norm = lambda v, g: v / (v.square().mean(-1, keepdim=True) + 1e-6).sqrt() * g  # noqa: E731
    q = norm(xr, p["g1"]) @ p["w_in"][0].t()
    a = torch.sigmoid(q[..., :d])
    c = (1 - a) * q[..., d:]
    state, mix = torch.zeros(b, d, dtype=torch.float64, device=x.device), []
    for t in range(s - 1, -1, -1):
        state = a[:, t] * state + c[:, t]
        mix.append(state)
    h = (torch.stack(mix[::-1], 1) + xr).reshape(b * s, d)
    y = norm(h, p["g2"])
    o = torch.zeros_like(h)
    for e in range(block.experts):
        rows = torch.nonzero(region == e)[:, 0]
        o = o.index_add(0, rows, ((y[rows] @ p["w1"][e].t()) * live[rows]) @ p["w2"][e].t())
    return (h + o).view(b, s, d), xr, p


def rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    return float((a - b).norm() / b.norm())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_block_matches_autograd(dtype):
    import ffn_ops
    from ray_block import RayBlock, regions
    g = torch.Generator().manual_seed(3)
    b, s, d, side = 24, 33, 48, 2
    block = RayBlock(d, 80, side ** 3, dtype=dtype, seed=4)
    x, dout = torch.randn(b, s, d, generator=g).to(dtype).cuda(), torch.randn(b, s, d, generator=g).to(dtype).cuda()
    pts = torch.rand(b * s, 3, generator=g).cuda()
    pts[:, 0] *= 0.45                          # half of the regions have no samples
    region = regions(pts, (0.0, 0.0, 0.0), (1.0, 1.0, 1.0), side)
    out, saved = block.forward(x, region)
    dx, grads = block.backward(dout, saved)
    a, back = saved[-1], saved[9]
    want, xr, p = reference(block, x, region, (a > 0)[back])
    want.backward(dout.double())
    # about ten roundings to the 16-bit type lie between input and output, and as many on the way back
    unit = 2.0 ** -8 if dtype is torch.bfloat16 else 2.0 ** -11
    assert rel(out, want) < 5 * unit
    assert rel(dx, xr.grad) < 8 * unit
    for k in grads:
        assert rel(grads[k].view_as(p[k]), p[k].grad) < 8 * unit, k
    assert bool((grads["w1"][4:] == 0).all()) and bool((grads["w2"][4:] == 0).all())
    served = block.serve(x, region)
    assert rel(served, want) < 2.0 ** -4       # one product in e4m3: 2^-4 of a value at most, less over a sum
    assert ffn_ops.status() == 0


def test_example_trains():
    from ray_block import example
    losses, _ = example(rays=64, samples=32, steps=40)
    assert losses[-1] < 0.5 * losses[0]
