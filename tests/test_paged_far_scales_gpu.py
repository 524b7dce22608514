"""Attention over the paged 8-bit KV cache where the scales of neighbouring blocks lie far apart, with a row count for each of its
kernels: what a row does not see, or gives no weight, leaves its result alone."""

import math

import pytest
import torch

import paged_reference as R
from test_paged_cache_gpu import _HALF_STEP, _cache, _i32, _key_scales, _nv, _table

pytestmark = pytest.mark.gpu


def _near(got, lse, q, k, v, vscale, limits, scaling, g, odd=False):
    """Rows of one request against 64 bits; row i sees the first limits[i] keys, and only those count here.

    With A = sum p |v| and S = scaling * max sum |q| |k|: products of exact halves summed in fp32 put a score off by
    S (D + 8) 2^-23; it is brought to units of log2 and to the exponent of its V scale in fp32, whose values reach
    S + L (L the largest |log2 vscale|): 2^-21 (1 + S + L); exp2 and sums (keys + 8) 2^-23.  A weight is a half, 2^-11 of
    itself; the result is rounded once.  Halves end at 2^-24: a weight is held times 2^3 or more relative to W and is off by 2^-28 W at
    most, with codes of at most 448 a value by 2^-28 W 448 keys.  W is the largest p vs of a key, or of 128 keys the largest p times the
    largest vs where these are within 2^16 of each other.  K and V are exact where scales are powers of two; another scale is rounded
    to eleven bits and its products with codes are (2^-11 each): 2^-10 of a score's terms and of A."""
    qd = q.cpu().double()
    n = max([0, *limits])
    k, v, vscale = k[:, :n], v[:, :n], vscale[:, :n].double()
    want, want_lse = R.attend(qd, k, v, limits, scaling, g)
    size, _ = R.attend(qd, k, v.abs(), limits, scaling, g)
    seen = (torch.arange(n) < torch.tensor(limits)[:, None])[:, None]                                   # [rows, 1, keys]
    terms = torch.einsum("nhd,hsd->nhs", qd.abs(), k.abs().repeat_interleave(g, 0)) * abs(scaling)
    top = torch.where(seen, terms, 0.0).amax(2) if n else torch.zeros(want_lse.shape).double()
    scales = torch.where(seen, vscale.repeat_interleave(g, 0)[None], 0.0)
    logs = torch.where(scales > 0, torch.log2(scales.clamp(min=1e-300)).abs(), 0.0)
    far = logs.amax(2) if n else torch.zeros(want_lse.shape).double()
    delta = top * (q.shape[2] + 8) * 2.0 ** -23 + (n + 8) * 2.0 ** -23 + 2.0 ** -21 * (1 + top + far) + (2.0 ** -10 * top if odd else 0.0)
    two = q.dtype == torch.float32
    weight = 2.0 ** -21 if two else 2.0 ** -11
    tol = size * (2 * delta + weight + (2.0 ** -10 if odd else 0.0))[..., None] + want.abs() * _HALF_STEP[q.dtype] + 1e-30
    if n:
        p = torch.exp(torch.einsum("nhd,hsd->nhs", qd, k.repeat_interleave(g, 0)) * scaling - want_lse[..., None])
        p = torch.where(seen, p, 0.0)
        groups = lambda x: torch.nn.functional.pad(x, (0, -n % 128)).unflatten(-1, (-1, 128)).amax(-1)
        w = torch.minimum(groups(p) * groups(scales), 2.0 ** 16 * groups(p * scales)).amax(2)
        tol = tol + (2.0 ** -28 * 448 * n * w)[..., None]
    if q.dtype == torch.float16:
        tol = tol + 2.0 ** -25                                       # subnormals
    off = (got.cpu().double() - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())
    none = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse.cpu()), none)
    d = (lse.cpu().double() - want_lse)[~none].abs()
    assert bool((d <= (delta + 2.0 ** -22 * want_lse.abs())[~none]).all())


# (new tokens, D, dtype): 4 query rows a token, so few rows, one group of 128, two groups of 128
_FEW = [(3, 128, torch.bfloat16), (3, 256, torch.float16), (3, 128, torch.float32)]
_MANY = [(20, 128, torch.bfloat16), (60, 128, torch.float16), (20, 256, torch.bfloat16), (60, 256, torch.float16)]


class _One:
    """One request of `new` tokens behind `held`: blocks of 16, two KV heads of four query heads."""

    def __init__(self, new, held, d, dtype, seed):
        self.total, self.block = held + new, 16
        self.new, self.held, self.d = new, held, d
        blocks = -(-self.total // 16) + 2
        self.k, self.ks = _cache(blocks, 2, 16, d, seed, 0.0)
        self.v, self.vs = _cache(blocks, 2, 16, d, seed + 50, 0.0)
        self.table = _table([self.total], 16, blocks, seed)
        self.q = torch.randn(new, 8, d, generator=torch.Generator().manual_seed(seed + 7)).to(dtype)
        self.scaling = d ** -0.5

    def block_of(self, position):
        return int(self.table[0, position // 16])

    def run(self):
        return _nv().fp8_paged_attention(self.q.cuda(), _i32([0, self.new]), self.k.cuda(), self.v.cuda(), self.ks.cuda(), self.vs.cuda(),
                                         self.table.cuda(), _i32([self.total]), self.scaling, 4, return_lse=True)

    def check(self, out, lse, rows=None, odd=False):
        """The first `rows` tokens."""
        rows = self.new if rows is None else rows
        kk, vv = (R.gather(c, s, self.table[0], self.total, 16) for c, s in ((self.k, self.ks), (self.v, self.vs)))
        _near(out[:rows], lse[:rows], self.q[:rows], kk, vv, _key_scales(self.vs, self.table[0], self.total, 16),
              [self.held + 1 + i for i in range(rows)], self.scaling, 4, odd=odd)


@pytest.mark.parametrize("far", [10, 20, 40])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("new,d,dtype", _FEW + _MANY)
def test_later_keys_of_a_larger_scale_leave_earlier_tokens_alone(new, d, dtype, which, far):
    """The last blocks of the request have a scale 2^far above the others; tokens in front of them do not see them, but their keys
    are among the same 128."""
    held, at = {3: (78, 80), 20: (70, 80), 60: (70, 112)}[new]
    x = _One(new, held, d, dtype, 3)
    for position in range(at, x.total, 16):
        (x.ks if which == "k" else x.vs)[x.block_of(position)] *= 2.0 ** far
    out, lse = x.run()
    x.check(out, lse, rows=at - held)


@pytest.mark.parametrize("new,d,dtype", _FEW + _MANY)
@pytest.mark.parametrize("which", ["values", "keys", "both", "zeros", "smallest", "odd"])
def test_scales_of_a_tile_far_apart(which, new, d, dtype):
    x = _One(new, 300, d, dtype, 5)
    g = torch.Generator().manual_seed(9)
    powers = lambda lo, hi: torch.exp2(torch.randint(lo, hi, x.vs.shape, generator=g).float())
    if which in ("values", "both"):
        x.vs = powers(-60, 60) if dtype != torch.float16 else powers(-60, 4)
    if which in ("keys", "both"):
        x.ks = torch.where(torch.rand(x.ks.shape, generator=g) < 0.5, 2.0 ** -6, powers(-60, -7))
    if which == "zeros":
        x.vs = torch.where(torch.rand(x.vs.shape, generator=g) < 0.5, 0.0, 2.0 ** -6)
        x.ks = torch.where(torch.rand(x.ks.shape, generator=g) < 0.5, 0.0, 2.0 ** -6)
    if which == "smallest":
        x.vs, x.ks = torch.full(x.vs.shape, 2.0 ** -110), torch.full(x.ks.shape, 2.0 ** -110)
    if which == "odd":
        x.vs = torch.rand(x.vs.shape, generator=g) * 3e-3 + 1e-5
        x.ks = torch.rand(x.ks.shape, generator=g) * 1e-2
    x.check(*x.run(), odd=which == "odd")


@pytest.mark.parametrize("position", [0, 100, 140])
@pytest.mark.parametrize("new,d,dtype", [m for m in _FEW + _MANY if m[2] != torch.float16])
def test_large_values_without_weight_do_not_count(new, d, dtype, position):
    """Keys with scores of about -300 whose values are 2^106 times those of the others."""
    x = _One(new, 300, d, dtype, 7)
    b = x.block_of(position)
    x.q[..., 0] = 8.0 * (d / 128) ** 0.5
    raw = x.k.view(torch.uint8)
    raw[:, :, :, 0] = 0
    raw[b, :, :, 0] = torch.tensor([-448.0]).to(torch.float8_e4m3fn).view(torch.uint8).item()
    x.ks[b], x.vs[b] = 1.0, 2.0 ** 100
    raw[b, :, :, 1:] = 0
    x.check(*x.run())


@pytest.mark.parametrize("most,d,dtype", [(9, 128, torch.bfloat16), (60, 128, torch.float16), (12, 256, torch.bfloat16), (4, 128, torch.float32)])
def test_far_scales_in_long_shares(most, d, dtype):
    """So much work that a CTA goes through many key tiles of a unit: most tiles hold blocks of all scales, some of one."""
    g = torch.Generator().manual_seed(most)
    block, requests, hk, h = 64, 24, 4, 32
    new = [most] * requests
    held = torch.randint(1500, 3000, (requests,), generator=g).tolist()
    total = [a + b for a, b in zip(new, held)]
    blocks = sum(-(-n // block) for n in total) + 1
    k, ks = _cache(blocks, hk, block, d, 1, 0.0)
    v, vs = _cache(blocks, hk, block, d, 2, 0.0)
    far = torch.rand(ks.shape, generator=g)
    ks = torch.where(far < 0.3, ks * torch.exp2(torch.randint(-60, 1, ks.shape, generator=g).float()), ks)
    low = -60 if dtype != torch.float16 else -20
    vs = torch.where(far > 0.7, vs * torch.exp2(torch.randint(low, 1 - low if dtype != torch.float16 else 1, vs.shape, generator=g).float()), vs)
    table = _table(total, block, blocks, 3)
    starts = [i * most for i in range(requests + 1)]
    q = torch.randn(starts[-1], h, d, generator=g).to(dtype)
    out, lse = _nv().fp8_paged_attention(q.cuda(), _i32(starts), k.cuda(), v.cuda(), ks.cuda(), vs.cuda(), table.cuda(), _i32(total), d ** -0.5,
                                         h // hk, return_lse=True)
    for r in (0, 7, 23):
        a, b = starts[r], starts[r + 1]
        kk, vv = R.gather(k, ks, table[r], total[r], block), R.gather(v, vs, table[r], total[r], block)
        _near(out[a:b], lse[a:b], q[a:b], kk, vv, _key_scales(vs, table[r], total[r], block), [held[r] + 1 + i for i in range(most)], d ** -0.5,
              h // hk)


@pytest.mark.parametrize("new,d,dtype", [m for m in _FEW + _MANY if m[2] != torch.float16])
def test_large_factors_of_products_that_are_zero(new, d, dtype):
    """q and K of 2^100 in channels of their own: every score is 0, although the product of their scales is above fp32."""
    x = _One(new, 90, d, dtype, 11)
    x.q = torch.zeros_like(x.q)
    x.q[..., 3] = 2.0 ** 100
    raw = x.k.view(torch.uint8)
    raw[:, :, :, 3] = 0
    x.ks[:] = 2.0 ** 100
    out, lse = x.run()
    vv = R.gather(x.v, x.vs, x.table[0], x.total, 16)
    for i in range(new):
        n = x.held + 1 + i
        want = vv[:, :n].mean(1).repeat_interleave(4, 0)
        # weights are equal powers of two, V exact: fp32 sums of n values, the sum of weights and its reciprocal, one rounding
        tol = vv[:, :n].abs().mean(1).repeat_interleave(4, 0) * (n + 8) * 2.0 ** -22 + want.abs() * _HALF_STEP[dtype] + 1e-30
        assert bool(((out[i].cpu().double() - want).abs() <= tol).all())
        assert bool(((lse[i].cpu().double() - math.log(n)).abs() <= 2.0 ** -20 * math.log(n)).all())
