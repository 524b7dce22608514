"""Paths between blocks whose scales are no powers of two: every code that moves is the one rounding of the value it stood for."""

import numpy as np
import pytest
import torch

import paged_reference as R
from test_paged_cache_gpu import _i32, _nv

pytestmark = pytest.mark.gpu


def _pairs(count, seed):
    """(scale it comes from, scale it goes to): quotients that bring some code to, or by less than a float's step beside, the border
    between two codes."""
    g = np.random.default_rng(seed)
    out = []
    while len(out) < count:
        code = float(g.integers(8, 16)) * 2.0 ** float(g.integers(-3, 5))
        border = (2.0 * float(g.integers(8, 16)) + 1.0) * 2.0 ** float(g.integers(-3, 3))
        now = np.float32(g.uniform(1.0, 2.0) * 2.0 ** float(g.integers(-20, 20)))
        near = np.float32(border * float(now) / code)
        for _ in range(int(g.integers(0, 3))):
            near = np.nextafter(near, np.float32(np.inf if g.random() < 0.5 else 0.0))
        out.append((float(near), float(now)))
    return out


def _rounded(x, s, now):
    """x s is exact in 64 bits; a quotient of such lengths that is no border is further from one than its rounding to 53 bits."""
    return R.nearest_e4m3((x * s) / now)


@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("seed", range(4))
def test_unequal_scales_that_are_no_powers_of_two(seed, d):
    hk, block = 40, 16
    codes = (torch.arange(hk * block * d) * 37 % 256).to(torch.uint8).view(hk, block, d)           # all of them in every token
    caches, scales, wants = [], [], []
    for which in (0, 1):
        pairs = _pairs(hk, 10 * seed + which)
        c = torch.stack([codes, codes.flip(-1)]).view(torch.float8_e4m3fn).cuda()
        s = torch.tensor([[now for _, now in pairs], [come for come, _ in pairs]])
        # tokens 1 .. 14 of block 0 come from block 1; its token 0 stays
        x, sd = c.cpu().double(), s.double()
        come, was = sd[1][:, None, None], sd[0][:, None, None]
        moved = x[1][:, 1:15]
        top = torch.nan_to_num((moved * come).abs(), nan=0.0).amax((1, 2))
        now = torch.where(sd[1] > sd[0], torch.maximum(sd[0], R.scale_of(top)), sd[0])
        want, new = x.clone(), now[:, None, None]
        want[0][:, 1:15] = _rounded(moved, come, new)
        want[0][:, :1] = torch.where(new == was, x[0][:, :1], _rounded(x[0][:, :1], was, new))
        wants.append((want, now))
        caches.append(c)
        scales.append(s.cuda())
    grown = sum(int((now != s[0].cpu().double()).sum()) for (_, now), s in zip(wants, scales))
    assert 0 < grown < 2 * hk                                                  # both ways
    path = [0] + list(range(17, 31))
    keep = _nv().paged_kv_keep_path(_i32(path + [-1] * 17), _i32([15]), _i32([0, 32]), _i32([32]), torch.tensor([[0, 1]], dtype=torch.int32).cuda(),
                                    *caches, *scales)
    assert keep.tolist() == [15]
    for c, s, (want, now) in zip(caches, scales, wants):
        got = c.cpu().double()
        assert torch.equal(s[0].cpu().double(), now)
        rows = [slice(0, 15), slice(0, block)]                                 # what lies behind the path in its block is no token
        for b in (0, 1):
            x, y = got[b][:, rows[b]], want[b][:, rows[b]]
            assert torch.equal(torch.isnan(x), torch.isnan(y)) and torch.equal(torch.nan_to_num(x), torch.nan_to_num(y))


def test_scales_far_apart():
    """Quotients outside the floats: zeros stay zeros, the rest saturates or vanishes."""
    hk, block, d = 4, 16, 128
    codes = (torch.arange(hk * block * d) * 37 % 256).to(torch.uint8).view(hk, block, d)
    c = [torch.stack([codes, codes.flip(-1)]).view(torch.float8_e4m3fn).cuda() for _ in (0, 1)]
    come = torch.tensor([1.5e-38, 3e-44, 1.3e38, 1.7])
    was = torch.tensor([1.1e30, 1.3e-39, 1.2e38, 1.9e-20])
    s = [torch.stack([was, come]).cuda() for _ in (0, 1)]
    before = c[0].cpu().double()
    keep = _nv().paged_kv_keep_path(_i32([0, 17] + [-1] * 30), _i32([2]), _i32([0, 32]), _i32([32]), torch.tensor([[0, 1]], dtype=torch.int32).cuda(), *c, *s)
    assert keep.tolist() == [2]
    for x, y in zip(c, s):
        now = y[0].cpu().double()
        assert bool((now >= was.double()).all()) and torch.equal(now[:2], was[:2].double())
        want = _rounded(before[1][:, 1], come.double()[:, None], now[:, None])
        got = x.cpu().double()[0][:, 1]
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
