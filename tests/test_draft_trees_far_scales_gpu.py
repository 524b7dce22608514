"""Attention of trees and of any bits where the scales of neighbouring blocks lie far apart: the many-row kernel brings such keys
together one by one, and its masks are sixteen keys wide there."""

import math

import pytest
import torch

import paged_reference as R
from test_draft_trees_gpu import _parents, _random_mask, _seen_of, _starts
from test_paged_cache_gpu import _HALF_STEP, _cache, _chunk, _i32, _key_scales, _nv, _table

pytestmark = pytest.mark.gpu


def _near(got, lse, q, k, v, vscale, seen, scaling, g):
    """A token [H, D] against 64 bits; `seen` [keys]: the keys that it sees.

    With A = sum p |v| and S = scaling * max sum |q| |k|: products of exact halves summed in fp32 put a score off by S (D + 8) 2^-23
    (fp32 queries are two halves); it is brought to units of log2 and to the exponent of its V scale in fp32, whose values reach S + L
    (L the largest |log2 vscale|): 2^-21 (1 + S + L); exp2 and sums (keys + 8) 2^-23.  A weight is a half, 2^-11 of itself (two of them
    2^-21); the result is rounded once.  Halves end at 2^-24: a weight is held times 2^3 or more relative to W and is off by 2^-28 W
    at most, with codes of at most 448 a value by 2^-28 W 448 keys.  W is the largest p times the largest scale of 128 keys, hidden ones
    among them, as long as these are within 2^16 of each other, else the largest p vs of a key times 2^16."""
    n = seen.shape[0]
    if not seen.any():
        assert bool((got == 0).all()) and bool((lse == -math.inf).all())
        return
    qd = q.cpu().double()
    heads = lambda x: x.repeat_interleave(g, 0)
    s = torch.einsum("hd,hsd->hs", qd, heads(k)) * scaling
    s = torch.where(seen, s, -math.inf)
    want_lse = torch.logsumexp(s, 1)
    p = torch.exp(s - want_lse[:, None])
    want, size = (torch.einsum("hs,hsd->hd", p, heads(x)) for x in (v, v.abs()))
    terms = torch.einsum("hd,hsd->hs", qd.abs(), heads(k.abs())) * abs(scaling)
    top = torch.where(seen, terms, 0.0).amax(1)
    scales = heads(vscale.double())
    far = torch.where(seen & (scales > 0), torch.log2(scales.clamp(min=1e-300)).abs(), 0.0).amax(1)
    delta = top * (q.shape[1] + 8) * 2.0 ** -23 + (n + 8) * 2.0 ** -23 + 2.0 ** -21 * (1 + top + far)
    tol = size * (2 * delta + (2.0 ** -21 if q.dtype == torch.float32 else 2.0 ** -11))[:, None] + want.abs() * _HALF_STEP[q.dtype] + 1e-30
    groups = lambda x: torch.nn.functional.pad(x, (0, -n % 128)).unflatten(-1, (-1, 128)).amax(-1)
    w = torch.minimum(groups(p) * groups(scales), 2.0 ** 16 * groups(p * scales)).amax(1)
    tol = tol + (2.0 ** -28 * 448 * n * w)[:, None] + (2.0 ** -25 if q.dtype == torch.float16 else 0.0)
    off = (got.cpu().double() - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())
    assert bool(((lse.cpu().double() - want_lse).abs() <= delta + 2.0 ** -22 * want_lse.abs()).all())


def _case(new, held, d, dtype, block, mask, which, seed, check, h=8, hk=2, behind=2):
    """Blocks whose scales are 2^-60 to 2^60 of each other (values of fp16 results below 2^4), those of `which`."""
    total = [a + b for a, b in zip(new, held)]
    blocks = sum(-(-n // block) for n in total) + 2
    k, ks = _cache(blocks, hk, block, d, seed, 0.0)
    v, vs = _cache(blocks, hk, block, d, seed + 50, 0.0)
    g = torch.Generator().manual_seed(seed)
    powers = lambda lo, hi: torch.exp2(torch.randint(lo, hi, vs.shape, generator=g).float())
    if which in ("values", "both"):
        vs = powers(-60, 60 if dtype != torch.float16 else 4)
    if which in ("keys", "both"):
        ks = torch.where(torch.rand(ks.shape, generator=g) < 0.5, 2.0 ** -6, powers(-60, -7))
    table, starts = _table(total, block, blocks, seed), _starts(new)
    q = torch.randn(starts[-1] + behind, h, d, generator=g).to(dtype)
    out, lse = _nv().fp8_paged_tree_attention(q.cuda(), _i32(starts), mask.cuda(), k.cuda(), v.cuda(), ks.cuda(), vs.cuda(), table.cuda(),
                                              _i32(total), d ** -0.5, h // hk, return_lse=True)
    for r, n in enumerate(new):
        if n == 0:
            continue
        kk, vv = R.gather(k, ks, table[r], total[r], block), R.gather(v, vs, table[r], total[r], block)
        scales = _key_scales(vs, table[r], total[r], block)
        seen = _seen_of(mask[starts[r]:starts[r + 1]].tolist(), n, total[r])
        for i in sorted({x % n for x in check}):
            t = starts[r] + i
            _near(out[t], lse[t], q[t], kk, vv, scales, seen[i], d ** -0.5, h // hk)
    assert bool((out[starts[-1]:] == 0).all()) and bool((lse[starts[-1]:] == -math.inf).all())


# trees that lie across the borders of 16 and of 128 keys, contexts that end on them and none
_SIZES = [([20, 33, 25], [119, 0, 240]), ([64, 60, 70], [100, 128, 0]), ([130, 40, 0, 90], [60, 250, 9, 127])]
_CHECK = (0, 1, 7, 8, 9, 15, 16, 17, 31, 32, 40, 63, 64, 100, 129)


@pytest.mark.parametrize("which", ["values", "keys", "both"])
@pytest.mark.parametrize("d,dtype", [(128, torch.bfloat16), (128, torch.float16), (256, torch.bfloat16), (256, torch.float16)])
@pytest.mark.parametrize("new,held", _SIZES)
def test_any_bits(new, held, d, dtype, which):
    """Bits of every kind: of tokens that are not there, none, all; and rows with fewer words than the request has tokens."""
    assert _chunk(dtype, d, sum(new) + 2, 4, len(new))
    words = 1 if max(new) > 100 else 2
    _case(new, held, d, dtype, 16, _random_mask(sum(new) + 2, words, 3), which, 3, _CHECK)


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("d,dtype", [(128, torch.bfloat16), (256, torch.float16)])
@pytest.mark.parametrize("new,held", _SIZES)
def test_trees(new, held, d, dtype, block):
    parents, total = _parents(new, 5), [a + b for a, b in zip(new, held)]
    mask, _ = _nv().draft_tree(_i32(parents + [0] * 2), _i32(_starts(new)), _i32(total), max(new))
    _case(new, held, d, dtype, block, mask.cpu(), "both", 7, _CHECK)


@pytest.mark.parametrize("new,held,d,dtype", [([3, 2, 1], [125, 0, 40], 128, torch.bfloat16), ([8, 6, 7], [250, 120, 0], 128, torch.float16),
                                              ([3, 4, 2], [126, 0, 300], 256, torch.float16), ([3, 4, 2], [126, 0, 300], 128, torch.float32)])
def test_few_rows(new, held, d, dtype):
    """The other kernel, whose rows are relative to a key's own."""
    assert not _chunk(dtype, d, sum(new) + 2, 4, len(new))
    _case(new, held, d, dtype, 16, _random_mask(sum(new) + 2, 1, 3), "both", 9, range(8))
