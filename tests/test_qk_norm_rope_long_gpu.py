"""Norm with rotation at lengths where every warp has many tasks: stages filled again and again, remainders, heads apart.

Tolerances of results and of gradients of operands are those of test_qk_norm_rope_gpu.py.  A weight's gradient goes through fewer
additions than it has rows: a lane's own rows one after the other, three shuffles, two warps, a 32nd of the blocks, five shuffles."""

import math

import pytest
import torch

import draft_reference as T

pytestmark = pytest.mark.gpu

_HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
_F = 2.0 ** -24
_H, _HK = 32, 8
_BLOCKS = 6                                                                    # of an SM, at most
_WARPS = {"forward": 4, "backward": 2}                                         # of a block


def _tiny(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 1e-37


def _tables(p, d):
    a = torch.arange(p, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
    return a.cos().float(), a.sin().float()


def _warps(way):
    return torch.cuda.get_device_properties(0).multi_processor_count * _BLOCKS * _WARPS[way]


def _tasks(tokens, d, size):
    """Tasks that a warp has, forward and backward: steps of 512 / d rows, two (fp32 one) or four (two) of them a task."""
    step = 512 // d
    steps = {"forward": 1 if size == 4 else 2, "backward": 2 if size == 4 else 4}
    return {way: tokens * (_H + _HK) // (step * s) // _warps(way) for way, s in steps.items()}


def _laid(x, heads_outside):
    """[T, H, D] as views of one buffer with other things around: heads of a token side by side, or tokens of a head."""
    t, h, d = x.shape
    if heads_outside:
        buf = torch.full((h, t + 3, d), 7.0, dtype=x.dtype, device="cuda")
        view = buf[:, 3:].transpose(0, 1)
    else:
        buf = torch.full((t, h + 2, d), 7.0, dtype=x.dtype, device="cuda")
        view = buf[:, 1:h + 1]
    view.copy_(x)
    return view


def _rows_a_lane(rows, d, dtype, heads):
    """Rows that one lane of the backward pass adds at most: its operand's blocks are shared out by tasks, of `steps` rows a lane."""
    steps, step = (2 if dtype == torch.float32 else 4), 512 // d
    share = heads / (_H + _HK)
    warps = max(2, math.floor(_warps("backward") / 3 * share))                 # three blocks an SM at least fit their stages, rounded down
    return (math.ceil(rows / (step * steps) / warps) + 2) * steps


@pytest.mark.parametrize("heads_outside", [False, True])
@pytest.mark.parametrize("d,tokens", [(128, 4003), (256, 4001)])
@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32), (torch.float32, torch.float32)])
def test_every_row_of_many_tasks(dtype, wdtype, d, tokens, heads_outside):
    import sageattention_b200.nvfp4 as nv
    assert min(_tasks(tokens, d, torch.finfo(dtype).bits // 8).values()) >= 4
    g = torch.Generator(device="cuda").manual_seed(tokens)
    ops = [torch.randn(tokens, n, d, generator=g, device="cuda") * torch.exp(torch.randn(tokens, n, 1, generator=g, device="cuda")) for n in (_H, _HK)]
    q, k = (_laid(x.to(dtype), heads_outside) for x in ops)
    gq, gk = (_laid(torch.randn(tokens, n, d, generator=g, device="cuda").to(dtype), heads_outside) for n in (_H, _HK))
    wq, wk = (1 + 0.5 * torch.randn(2, d, generator=g, device="cuda")).to(wdtype)
    cos, sin = _tables(700, d)
    inside = torch.randint(700, (tokens,), generator=g, device="cuda")
    out = torch.rand(tokens, generator=g, device="cuda") < 0.03
    out[-1] = out[0] = True
    for pos in (inside.int(), torch.where(out, torch.randint(-9, 0, (tokens,), generator=g, device="cuda") + 709 * (inside % 2), inside)):
        there = (pos >= 0) & (pos < 700)
        leaves = [x.detach().requires_grad_(True) for x in (q, k, wq, wk)]
        res = nv.qk_norm_rope(*leaves, cos, sin, pos)
        grads = torch.autograd.grad(res, leaves, (gq, gk))
        at = pos.long().clamp(0, 699)
        c, s = cos.double()[at][:, None], sin.double()[at][:, None]
        for i, (x, w, gr) in enumerate(((q, wq, gq), (k, wk, gk))):
            y, dx, dw = res[i].detach(), grads[i], grads[2 + i]
            assert bool(torch.isnan(y[~there]).all()) and bool(torch.isnan(dx[~there]).all())
            want, n, _ = T.norm_rope(x.double(), w.double(), c, s, 1e-6)
            tol = 24 * _F * T.turned_size(n * w.double(), c, s) + _HALF_STEP[dtype] * want.abs() + _tiny(dtype)
            assert bool(((y.double() - want).abs() <= tol)[there].all())
            want, want_w, back, n, r = T.norm_rope_grads(x.double(), w.double(), c, s, 1e-6, gr.double())
            size = T.turned_size(gr.double(), c, s)
            part = (size * w.double().abs() * n.abs()).mean(-1, keepdim=True)
            tol = 48 * _F * r * (size * w.double().abs() + n.abs() * part) + _HALF_STEP[dtype] * want.abs() + _tiny(dtype)
            assert bool(((dx.double() - want).abs() <= tol)[there].all())
            if bool(there.all()):
                depth = _rows_a_lane(x.numel() // d, d, dtype, x.shape[1]) + 3 + 2 + math.ceil(_warps("backward") / 2 / 32) + 5
                tol = (depth + 48) * _F * (size * n.abs()).flatten(0, -2).sum(0) + _HALF_STEP[wdtype] * want_w.abs() + _tiny(wdtype)
                off = (dw.double() - want_w).abs()
                assert bool((off <= tol).all()), float((off / tol).max())
            else:
                assert bool(torch.isnan(dw).all())


@pytest.mark.parametrize("d,dtype,tokens,h,hk", [(128, torch.bfloat16, 4003, 32, 8), (128, torch.float16, 4097, 32, 8), (256, torch.bfloat16, 4001, 16, 4),
                                                 (128, torch.float32, 3999, 32, 8), (256, torch.float16, 2501, 7, 3), (128, torch.bfloat16, 5003, 5, 1),
                                                 (128, torch.bfloat16, 9001, 1, 1), (256, torch.float32, 1501, 16, 4)])
@pytest.mark.parametrize("heads_outside", [False, True])
def test_every_row_counts_once_in_the_weights(d, dtype, tokens, h, hk, heads_outside):
    """Rows of +-1 with cos 1 and sin 0, eps 0: n is x times the device's 1 / sqrt(1), off by two steps (2^-22) at most, and g' is g.  With g of -1,
    0 and 1 a sum is a whole number N; what is computed is off by less than a half, so that a row lost or taken twice shows in
    every column that its g has a value in."""
    import sageattention_b200.nvfp4 as nv
    g = torch.Generator(device="cuda").manual_seed(tokens + h)
    sign = lambda n: (torch.randint(0, 2, (tokens, n, d), generator=g, device="cuda") * 2 - 1).to(dtype)

    def few(n):
        there = torch.rand(tokens, n, d, generator=g, device="cuda") < 0.03
        return sign(n) * there.scatter(2, torch.randint(d, (tokens, n, 1), generator=g, device="cuda"), True)

    q, k, gq, gk = (_laid(x, heads_outside) for x in (sign(h), sign(hk), few(h), few(hk)))
    w = torch.ones(d, device="cuda")
    cos, sin = torch.ones(tokens, d // 2, device="cuda"), torch.zeros(tokens, d // 2, device="cuda")
    leaves = [x.detach().requires_grad_(True) for x in (q, k, w, w.clone())]
    grads = torch.autograd.grad(nv.qk_norm_rope(*leaves, cos, sin, eps=0.0), leaves, (gq, gk))
    for x, gr, dw in ((q, gq, grads[2]), (k, gk, grads[3])):
        assert bool((gr != 0).any(-1).all())                                   # every row would be missed
        want, size = ((y.double()).sum((0, 1)) for y in (gr.double() * x.double(), gr.double().abs()))
        # a term: those and a rounding, 5 2^-24; additions as many as rows of a lane and the tree above them, at most 200 in all
        assert float(size.max()) * 210 * _F < 0.25
        assert bool(((dw.double() - want).abs() < 0.25).all())
