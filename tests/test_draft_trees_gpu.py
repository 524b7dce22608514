"""Trees of drafts over the paged 8-bit cache against the 64-bit reference of draft_reference.py: tables, verification and moved
codes exactly, attention within what its roundings can add up to (as for causal attention, test_paged_cache_gpu.py)."""

import math

import numpy as np
import pytest
import torch

import draft_reference as T
import paged_reference as R
from test_paged_cache_gpu import _as_values, _cache, _chunk, _close, _empty_cache, _i32, _key_scales, _nv, _spoil, _table

pytestmark = pytest.mark.gpu


def _starts(new):
    out = [0]
    for n in new:
        out.append(out[-1] + n)
    return out


def _parents(new, seed, branch=3):
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in new:
        out += [-1 if i == 0 else max(0, i - 1 - int(torch.randint(2 * branch, (1,), generator=g))) for i in range(n)]
    return out


# ------------------------------------------------------------------------------------------------ tables
@pytest.mark.parametrize("most", [1, 8, 64, 65, 300, 1024])
def test_tables_of_trees(most):
    new = [5, 0, 1, 64, 65, 300, 0, 129, 2]
    g = torch.Generator().manual_seed(most)
    parents = _parents(new, most)
    for i in torch.randint(len(parents), (40,), generator=g).tolist():
        parents[i] = int(torch.randint(-3, 400, (1,), generator=g))           # roots inside, and what names no earlier node
    parents[-1] = 2 ** 31 - 1
    starts, tokens = _starts(new), sum(new) + 7
    lengths = [n + int(torch.randint(0, 5000, (1,), generator=g)) for n in new]
    lengths[3] = 10                                                            # fewer keys than nodes
    mask, positions = _nv().draft_tree(_i32(parents + [0] * 7), _i32(starts), _i32(lengths), most)
    count = -(-most // 64)
    assert mask.shape == (tokens, count) and mask.dtype == torch.int64 and positions.dtype == torch.int32
    for r, n in enumerate(new):
        a, b = starts[r], starts[r + 1]
        seen, depth = T.tree(parents[a:b], most)
        assert mask[a:b].tolist() == T.words(seen, count)
        assert positions[a:b].tolist() == [max(0, lengths[r] - n + d) for d in depth]
    assert not mask[starts[-1]:].any() and not positions[starts[-1]:].any()


def test_tables_of_a_long_chain_and_of_nothing():
    n = 1024
    mask, positions = _nv().draft_tree(_i32([i - 1 for i in range(n)]), _i32([0, n]), _i32([n + 3]), n)
    assert mask.tolist() == T.words(torch.ones(n, n).tril().bool(), 16) and positions.tolist() == list(range(3, n + 3))
    mask, positions = _nv().draft_tree(_i32([]), _i32([0, 0]), _i32([9]), 5)
    assert mask.shape == (0, 1) and positions.shape == (0,)
    for cu in ([0, 100, 200], [-5, 6, 12], [8, 3, 12], [12, 12, 12], [3, 6, 9], [2 ** 31 - 1, -2 ** 31, 0]):
        _nv().draft_tree(_i32([0] * 12), _i32(cu), _i32([20, 20]), 64)
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------------ attention
def _seen_of(words, n, length):
    """[n, length]: what the tokens of one request see, from their rows of words."""
    bits = torch.tensor([[(int(w) >> j) & 1 for w in row for j in range(64)] for row in words], dtype=torch.bool).view(len(words), -1)
    out = torch.zeros(n, max(length, 0), dtype=torch.bool)
    for j in range(n):
        key = length - n + j
        if 0 <= key and j < bits.shape[1]:
            out[:, key] = bits[:, j]
    out[:, :max(0, length - n)] = True
    return out


def _tree_case(new, held, h, hk, d, block, dtype, mask, seed=0, behind=0, spread=2.0, spoil=True, check=None):
    total = [a + b for a, b in zip(new, held)]
    blocks = sum(-(-n // block) for n in total) + 2
    k, ks = _cache(blocks, hk, block, d, seed, spread)
    v, vs = _cache(blocks, hk, block, d, seed + 50, spread)
    table = _table(total, block, blocks, seed)
    if spoil:
        _spoil(k, ks, table, total, block)
        _spoil(v, vs, table, total, block)
    starts = _starts(new)
    tokens = starts[-1] + behind
    q = torch.randn(tokens, h, d, generator=torch.Generator().manual_seed(seed + 7)).to(dtype)
    out, lse = _nv().fp8_paged_tree_attention(q.cuda(), _i32(starts), mask.cuda(), k.cuda(), v.cuda(), ks.cuda(), vs.cuda(), table.cuda(),
                                              _i32(total), d ** -0.5, h // hk, return_lse=True)
    assert out.shape == q.shape and out.dtype == dtype and lse.shape == (tokens, h)
    for r, n in enumerate(new):
        kk, vv = R.gather(k, ks, table[r], total[r], block), R.gather(v, vs, table[r], total[r], block)
        scales = _key_scales(vs, table[r], total[r], block)
        seen = _seen_of(mask[starts[r]:starts[r + 1]].tolist(), n, total[r]) if n else None
        for i in range(n) if check is None else sorted({x % n for x in check}) if n else ():
            t = starts[r] + i
            _close(out[t:t + 1], lse[t:t + 1], q[t:t + 1], kk, vv, scales, [total[r]], d ** -0.5, h // hk, hidden=~seen[i],
                   chunk=_chunk(dtype, d, tokens, h // hk, len(new)))
    assert bool((out[starts[-1]:] == 0).all()) and bool((lse[starts[-1]:] == -math.inf).all())
    return out, lse


def _random_mask(tokens, count, seed):
    """Any bits: also of tokens behind, of none, and of those that are not there."""
    g = torch.Generator().manual_seed(seed)
    mask = torch.randint(-2 ** 63, 2 ** 63 - 1, (tokens, count), generator=g)
    mask[torch.rand(tokens, generator=g) < 0.2] = 0
    mask[torch.rand(tokens, generator=g) < 0.1] = -1
    return mask


_NEW, _HELD = [1, 0, 5, 17, 33, 1, 64], [0, 9, 40, 100, 0, 300, 65]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("h,hk,d,block", [(4, 1, 128, 16), (8, 2, 128, 64), (6, 2, 256, 32), (16, 1, 128, 128)])
def test_attention_of_any_bits(h, hk, d, block, dtype):
    _tree_case(_NEW, _HELD, h, hk, d, block, dtype, _random_mask(sum(_NEW) + 3, 1, h), seed=h, behind=3, check=(0, 1, 4, 16, 31, 40, 63))


# few rows a request (8, 16, 24, 32 of them), then the other kernel's 128 and 256, and those at D 256
@pytest.mark.parametrize("new,held,h,hk,d,dtype", [([2, 1, 2], [500, 40, 127], 4, 1, 128, torch.bfloat16), ([4, 4], [260, 0], 8, 2, 128, torch.float16),
                                                   ([6, 5], [123, 511], 4, 1, 128, torch.bfloat16), ([8, 8], [700, 120], 4, 1, 128, torch.bfloat16),
                                                   ([26, 30], [1000, 3], 4, 1, 128, torch.bfloat16), ([64, 40], [130, 600], 8, 2, 128, torch.float16),
                                                   ([3, 4], [300, 17], 16, 4, 256, torch.float16), ([40, 12], [200, 511], 8, 2, 256, torch.bfloat16),
                                                   ([100, 130], [60, 0], 8, 2, 128, torch.bfloat16), ([70, 66], [10, 300], 4, 1, 256, torch.float16)])
@pytest.mark.parametrize("block", [16, 64])
def test_trees_through_every_kernel(new, held, h, hk, d, dtype, block):
    parents = _parents(new, 5)
    total = [a + b for a, b in zip(new, held)]
    mask, _ = _nv().draft_tree(_i32(parents), _i32(_starts(new)), _i32(total), max(new))
    _tree_case(new, held, h, hk, d, block, dtype, mask.cpu(), seed=3, check=(0, 1, 2, 7, 33, 63, 64, 99, 129))


@pytest.mark.parametrize("h,hk,d,most,dtype", [(32, 8, 128, 2, torch.bfloat16), (32, 8, 128, 30, torch.float16), (16, 4, 256, 8, torch.float16),
                                               (32, 8, 128, 4, torch.float32)])
def test_long_shares_of_trees(h, hk, d, most, dtype):
    """So much work that a block of threads goes through many key tiles of a unit and through several units, which are cut."""
    g = torch.Generator().manual_seed(h + most)
    new = torch.randint(1, most + 1, (40,), generator=g).tolist()
    held = torch.randint(1000, 3001, (40,), generator=g).tolist()
    total = [a + b for a, b in zip(new, held)]
    mask, _ = _nv().draft_tree(_i32(_parents(new, 2)), _i32(_starts(new)), _i32(total), most)
    _tree_case(new[:40], held, h, hk, d, 64, dtype, mask.cpu(), seed=1, spoil=False, check=(0, most - 1))


@pytest.mark.parametrize("new,d,dtype", [([20, 9, 12], 128, torch.bfloat16), ([60, 0, 40], 128, torch.float16), ([11, 40, 7], 256, torch.bfloat16),
                                         ([4, 3, 4], 128, torch.float32)])
def test_words_more_and_fewer_than_tokens(new, d, dtype):
    _tree_case(new, [30, 10, 70], 4, 2, d, 16, dtype, _random_mask(sum(new), 3, 1), seed=2)
    long = [n + 60 for n in new]
    _tree_case(long, [30, 0, 70], 4, 2, d, 16, dtype, _random_mask(sum(long), 1, 1), seed=2, check=(0, 5, 62, 63, 64, 65, 99))


def test_a_chain_is_causal_attention():
    """Scales far apart too, where the many-row kernel brings keys together one by one."""
    nv, block = _nv(), 16
    for d, new, dtype, spread in ((128, [40, 70, 3], torch.bfloat16, 2.0), (128, [40, 70, 3], torch.float16, 14.0), (256, [20, 64, 1], torch.bfloat16, 14.0),
                                  (128, [2, 1, 2], torch.bfloat16, 14.0)):
        total = [n + x for n, x in zip(new, (100, 7, 300))]
        blocks = sum(-(-n // block) for n in total)
        k, ks = _cache(blocks, 2, block, d, 3, 0.0)
        v, vs = _cache(blocks, 2, block, d, 4, 0.0)
        g = torch.Generator().manual_seed(1)
        ks, vs = (s * torch.exp2((spread * torch.randn(s.shape, generator=g)).round().clamp(-40, 4)) for s in (ks, vs))
        table, starts = _table(total, block, blocks, 1).cuda(), _i32(_starts(new))
        q = torch.randn(sum(new), 8, d, generator=g).to(dtype).cuda()
        parents = _i32([i - 1 for n in new for i in range(n)])
        mask, positions = nv.draft_tree(parents, starts, _i32(total), max(new))
        assert positions.tolist() == [t - n + i for n, t in zip(new, total) for i in range(n)]
        args = (k.cuda(), v.cuda(), ks.cuda(), vs.cuda(), table, _i32(total), d ** -0.5, 4, True)
        a, la = nv.fp8_paged_tree_attention(q, starts, mask, *args)
        b, lb = nv.fp8_paged_attention(q, starts, *args)
        # Two roundings of weights to halves (2^-11) and of results each; a value is below 448 of the largest V scale
        size = 448 * float(vs.max())
        assert bool(((a.float() - b.float()).abs() <= 2.0 ** -7 * b.float().abs() + 2.0 ** -10 * size).all())
        assert bool(((la - lb).abs() <= 2.0 ** -18 * (1 + lb.abs())).all())


def test_a_token_that_sees_nothing_and_more_tokens_than_keys():
    block, nv = 16, _nv()
    for n, h, dtype in ((6, 4, torch.bfloat16), (40, 8, torch.bfloat16), (40, 8, torch.float16), (6, 4, torch.float32)):
        k, ks = _cache(8, 1, block, 128, 3)
        v, vs = _cache(8, 1, block, 128, 4)
        table = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32)
        q = torch.randn(2 * n, h, 128, generator=torch.Generator().manual_seed(1)).to(dtype)
        mask = torch.zeros(2 * n, 1, dtype=torch.int64)
        mask[1], mask[n + 1], mask[n + 2], mask[2] = 1 << 1, 1 << (n - 1), 1, 1 << (n - 1)
        out, lse = nv.fp8_paged_tree_attention(q.cuda(), _i32([0, n, 2 * n]), mask.cuda(), k.cuda(), v.cuda(), ks.cuda(), vs.cuda(), table.cuda(),
                                               _i32([n, 4]), 0.1, h, return_lse=True)
        for r, length in ((0, n), (1, 4)):
            kk, vv = R.gather(k, ks, table[r], length, block), R.gather(v, vs, table[r], length, block)
            seen = _seen_of(mask[r * n:r * n + n].tolist(), n, length)
            for i in range(n):
                t = r * n + i
                _close(out[t:t + 1], lse[t:t + 1], q[t:t + 1], kk, vv, _key_scales(vs, table[r], length, block), [length], 0.1, h,
                       hidden=~seen[i], chunk=_chunk(dtype, 128, 2 * n, h, 2))
                if not seen[i].any():
                    assert bool((out[t] == 0).all()) and bool((lse[t] == -math.inf).all())


# ------------------------------------------------------------------------------------------------ verification
def _rows(t, v, seed, peak=6.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(t, v, generator=g) * 2
    x.scatter_add_(1, torch.randint(v, (t, 4), generator=g), torch.full((t, 4), peak))
    return torch.softmax(x, 1)


def _check_verify(p, tokens, parents, starts, u, q=None, behind=0):
    """p, q, u on the CPU; tokens and parents lists; the last `behind` tokens are nobody's."""
    got = _nv().verify_drafts(p.cuda(), tokens.cuda(), _i32(parents), _i32(starts), u.cuda(), draft_probs=None if q is None else q.cuda())
    pd, qd, ud = p.double().numpy(), None if q is None else q.double().numpy(), u.double().numpy()
    accepted, count, after = [], [], []
    for a, b in zip(starts[:-1], starts[1:]):
        path, x = T.verify(pd[a:b], tokens[a:b].tolist(), parents[a:b], ud[a:b], None if q is None else qd[a:b])
        accepted += path + [-1] * (b - a - len(path))
        count.append(len(path))
        after.append(x)
    assert got.accepted.tolist() == accepted + [-1] * behind
    assert got.num_accepted.tolist() == count and got.next_tokens.tolist() == after
    assert got.accepted.dtype == got.num_accepted.dtype == torch.int32 and got.next_tokens.dtype == torch.int64
    return count


def _drafts(p, q, parents, starts, seed, likeliest=False):
    """Tokens drawn from their parent's row, or its likeliest ones."""
    g = torch.Generator().manual_seed(seed)
    tokens = torch.zeros(p.shape[0], dtype=torch.long)
    for a, b in zip(starts[:-1], starts[1:]):
        rank = {}
        for i in range(b - a):
            up = T.parent_of(i, parents[a:b])
            row = (p if q is None else q)[a + max(up, 0)].double()
            if likeliest:
                n = rank[up] = rank.get(up, -1) + 1
                tokens[a + i] = torch.topk(row, min(n + 1, len(row))).indices[-1]
            else:
                tokens[a + i] = torch.multinomial(row.clamp(min=0), 1, generator=g)
    return tokens


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("v", [1, 7, 130, 1001, 32000, 50001])
@pytest.mark.parametrize("drawn", [True, False])
def test_verification_is_the_definitions(v, drawn, dtype):
    new = [5, 1, 0, 12, 33, 2]
    starts, parents = _starts(new), _parents(new, v, branch=2)
    parents[-1] = -1                                                           # hangs on the context: never kept
    p = _rows(sum(new) + 2, v, 1).to(dtype)
    q = (0.6 * p.float() + 0.4 * _rows(sum(new) + 2, v, 2)).to(dtype) if drawn else None
    kept = 0
    for seed in range(3):
        tokens = _drafts(p, q, parents, starts, seed, likeliest=not drawn)
        u = torch.rand(sum(new) + 2, generator=torch.Generator().manual_seed(seed))
        kept += sum(_check_verify(p, tokens, parents + [0, 0], starts, u, q, behind=2))
    assert kept > 3 * 5 or v > 1001                                            # rows of many tokens are too flat for some seeds


@pytest.mark.parametrize("requests", [1, 19, 40, 75, 150, 400])
@pytest.mark.parametrize("drawn", [True, False])
def test_clusters_of_every_size(requests, drawn):
    new = [1 + (7 * i) % 5 for i in range(requests)]
    starts, parents = _starts(new), _parents(new, 3)
    p = _rows(sum(new), 3001, 5, peak=4.0)
    q = 0.5 * p + 0.5 * _rows(sum(new), 3001, 6) if drawn else None
    u = torch.rand(sum(new), generator=torch.Generator().manual_seed(requests))
    _check_verify(p, _drafts(p, q, parents, starts, 4, likeliest=not drawn).int(), parents, starts, u, q)


@pytest.mark.parametrize("drawn", [True, False])
def test_trees_of_about_a_warp(drawn):
    """One warp finds the siblings of up to 32 nodes, each thread those of its own behind that; tokens come again among them."""
    new = [31, 32, 33, 34, 32, 33, 32]
    g = torch.Generator().manual_seed(8)
    starts, total, v = _starts(new), sum(new), 11
    p, q = _rows(total, v, 3, peak=2.0), _rows(total, v, 4, peak=2.0) if drawn else None
    for near in (1, 2, 40):                                                    # chains, trees and shallow ones
        parents = [-1 if i == 0 else int(torch.randint(min(i, near), (1,), generator=g)) + max(0, i - near) * (near < 40)
                   for n in new for i in range(n)]
        for seed in range(4):
            tokens = torch.randint(-1, v, (total,), generator=g) if seed else _drafts(p, q, parents, starts, seed)
            _check_verify(p, tokens, parents, starts, torch.rand(total, generator=g) * (1.0 if seed < 3 else 0.2), q)


def test_long_chains_and_wide_trees():
    """Trees end with their 1024th token; children of one node in the hundreds, all of them rejected."""
    p = _rows(1100, 50, 1)
    u = torch.zeros(1100)
    tokens = torch.randint(50, (1100,), generator=torch.Generator().manual_seed(1))
    assert _check_verify(p, tokens, [i - 1 for i in range(1100)], [0, 1100], u) == [1024]
    assert _check_verify(p, tokens, [i - 1 for i in range(1100)], [0, 1100], u, p) == [1024]
    wide = [-1] + [0] * 299
    u = torch.rand(300, generator=torch.Generator().manual_seed(2))
    tokens = torch.arange(300) % 280                                           # the last ones again
    p = _rows(300, 2000, 3, peak=0.0)
    p[0, :280] *= 1e-6
    _check_verify(p, tokens, wide, [0, 300], u)
    q = torch.zeros(300, 2000)
    q[0, :280] = 1 / 280
    _check_verify(p, tokens, wide, [0, 300], u, q)


def test_rows_that_are_no_distribution_and_borders():
    nan, inf = math.nan, math.inf
    p = torch.tensor([[0.5, nan, 0.25, -1.0, 0.25], [0.0, 0.0, 0.0, 0.0, 0.0], [inf, 0.5, 0.0, 0.5, 0.0], [0.0, 0.0, 1.0, 0.0, 0.0]])
    q = torch.tensor([[0.5, 0.25, nan, 0.25, 0.0], [0.2] * 5, [0.5, 0.5, 0.0, 0.0, inf], [0.0, 0.0, 1.0, 0.0, 0.0]])
    for parents in ([-1, 0, 1, 2], [-1, 0, 0, 0], [-1, 0, 0, 2]):
        for ids in ([9, 0, 3, 2], [0, 2, 2, 2], [0, -1, 5, 2 ** 40], [1, 1, 0, 4]):
            for w in (0.0, 0.25, 0.5, 1 - 2.0 ** -24):
                for x in (0.0, 0.5, 1 - 2.0 ** -24):
                    u = torch.tensor([w, x, x, x])
                    tokens = torch.tensor(ids)
                    _check_verify(p, tokens, parents, [0, 4], u)
                    _check_verify(p, tokens, parents, [0, 4], u, q)
    # numbers outside [0, 1) leave nothing out of bounds
    for w in (1.0, 5.0, -1.0, nan, inf):
        for d in (None, q.cuda()):
            out = _nv().verify_drafts(p.cuda(), torch.tensor([0, 0, 3, 2]).cuda(), _i32([-1, 0, 1, 2]), _i32([0, 4]), torch.full((4,), w).cuda(), d)
            assert 0 <= int(out.next_tokens) < 5 and 1 <= int(out.num_accepted) <= 4


@pytest.mark.parametrize("v", [2, 40, 3000])
def test_drafts_that_leave_nothing(v):
    """Rows that sum to less than one, all of whose tokens are drafts and rejected: the next token is drawn from the row itself."""
    n = min(v, 60) + 1
    p = torch.zeros(n, v)
    p[:, :n - 1] = 0.01 + 0.3 * torch.rand(n, n - 1, generator=torch.Generator().manual_seed(v)) / n
    tokens = torch.arange(n) - 1
    for parents in ([-1] + [0] * (n - 1), [-1] + [0] * (n - 1 - n // 3) + [1] * (n // 3)):
        for w in (0.0, 0.3, 0.99):
            u = torch.full((n,), 1 - 2.0 ** -24)
            u[0] = w
            assert _check_verify(p, tokens, parents, [0, n], u) == [1]
            q = torch.full((n, v), 1.0)                                        # more than the target has, everywhere
            assert _check_verify(p, tokens, parents, [0, n], u, q) == [1]


def test_strided_rows_and_offsets_that_are_none():
    wide, other = _rows(9, 300, 1).cuda(), _rows(9, 300, 2).cuda()
    parents, starts = [-1, 0, 0, 1, -1, 0, 1, 1], [0, 4, 8]
    u = torch.rand(8, generator=torch.Generator().manual_seed(1))
    for dtype in (torch.float32, torch.bfloat16):
        a, b = wide.to(dtype), other.to(dtype)
        for p, q in ((a[1:, 3:104], b[:8, 2:103]), (a[:8, ::2][:, :101], b[:8].T.contiguous().T[:, 10:111])):
            tokens = _drafts(p.float().cpu(), q.float().cpu(), parents, starts, 1)
            got = _nv().verify_drafts(p, tokens.cuda(), _i32(parents), _i32(starts), u.cuda(), q)
            want = _nv().verify_drafts(p.contiguous(), tokens.cuda(), _i32(parents), _i32(starts), u.cuda(), q.contiguous())
            assert all(torch.equal(x, y) for x, y in zip(got, want))
            _check_verify(p.cpu(), tokens, parents, starts, u, q.cpu())
    for cu in ([0, 100, 200], [-5, 3, 8], [6, 3, 8], [8, 8, 8], [2 ** 31 - 1, -2 ** 31, 0]):
        _nv().verify_drafts(wide[:8], torch.zeros(8, dtype=torch.long, device="cuda"), _i32(parents), _i32(cu), u.cuda(), other[:8])
    empty = torch.empty(0, dtype=torch.long, device="cuda")
    none = _nv().verify_drafts(wide[:0], empty, empty.int(), _i32([0, 0, 0]), empty.float())
    assert none.num_accepted.tolist() == [0, 0] and none.next_tokens.tolist() == [-1, -1]


@pytest.mark.parametrize("kind", ["chain", "drawn", "likeliest"])
def test_what_is_kept_is_distributed_as_the_targets_own(kind):
    """First token of 40000 requests, over six tokens: each count within five standard deviations of its own."""
    n, v = 40000, 6
    g = torch.Generator().manual_seed(11)
    p = torch.tensor([0.35, 0.05, 0.25, 0.2, 0.05, 0.1])
    q = torch.tensor([0.1, 0.3, 0.2, 0.1, 0.2, 0.1])
    nodes = 2 if kind == "chain" else 4
    tokens = torch.zeros(n, nodes, dtype=torch.long)
    tokens[:, 1:] = torch.multinomial(q.expand(n, v), nodes - 1, replacement=True, generator=g) if kind != "likeliest" else torch.tensor([1, 0, 4])
    parents = torch.tensor([-1] + [0] * (nodes - 1)).repeat(n)
    got = _nv().verify_drafts(p.expand(n * nodes, v).cuda(), tokens.flatten().cuda(), parents.int().cuda(), (torch.arange(n + 1) * nodes).int().cuda(),
                              torch.rand(n * nodes, generator=g).cuda(), None if kind == "likeliest" else q.expand(n * nodes, v).cuda())
    second = got.accepted.view(n, nodes)[:, 1].cpu().long() if nodes > 1 else None
    first = torch.where(got.num_accepted.cpu() > 1, tokens.gather(1, second.clamp(min=0)[:, None])[:, 0], got.next_tokens.cpu())
    seen = torch.bincount(first, minlength=v).double() / n
    assert bool(((seen - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all()), seen


# ------------------------------------------------------------------------------------------------ the path moved together
def _check_keep(new, held, paths, hk, d, block, layers, seed=0, near=False, nan=False, table=None, behind=0, between=0):
    total = [a + b for a, b in zip(new, held)]
    blocks = sum(-(-n // block) for n in total) + 2
    table = _table(total, block, blocks, seed) if table is None else table
    starts = _starts(new)
    accepted = [x for n, path in zip(new, paths) for x in (list(path) + [-1] * n)[:n]] + [0] * behind
    caches, wants = [], []
    for which in (1, 2):
        parts = [_empty_cache(blocks, hk, block, d, seed + 10 * layer + which, between) for layer in range(layers)]
        flat = torch.stack([f for _, _, f in parts])
        if nan:
            flat[..., 5:hk * block * d:97] = 0xFF
        codes = flat[:, :, :hk * block * d].unflatten(2, (hk, block, d)).view(torch.float8_e4m3fn)
        scale = torch.stack([s for _, s, _ in parts])
        if near:
            scale.fill_(0.75)
        caches.append((codes, scale, flat, flat[:, :, hk * block * d:].clone()))
        values = [(_as_values(codes[layer]), scale[layer].cpu().double()) for layer in range(layers)]
        for x, s in values:
            for r, path in enumerate(paths):
                T.keep_path(list(path)[:new[r]], new[r], total[r], table[r], x, s, block)
        wants.append(values)
    (k, ks, _, _), (v, vs, _, _) = caches
    pick = (lambda x: x) if layers > 1 else (lambda x: x[0])
    keep = _nv().paged_kv_keep_path(_i32(accepted), _i32([len(x) for x in paths]), _i32(starts), _i32(total), table.cuda(), pick(k), pick(v),
                                    pick(ks), pick(vs))
    scratch = [torch.zeros(blocks, 1, block, 1, dtype=torch.float64), torch.ones(blocks, 1, dtype=torch.float64)]
    assert keep.tolist() == [T.keep_path(list(x)[:n], n, t, row, *(y.clone() for y in scratch), block) for x, n, t, row in zip(paths, new, total, table)]
    for values, (codes, scale, flat, gap) in zip(wants, caches):
        for layer, (x, s) in enumerate(values):
            got = _as_values(codes[layer])
            assert torch.equal(scale[layer].cpu().double(), s)
            assert torch.equal(torch.isnan(got), torch.isnan(x)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(x))
        assert torch.equal(flat[:, :, hk * block * d:], gap)


@pytest.mark.parametrize("hk,d,block,layers", [(1, 128, 16, 1), (3, 128, 64, 2), (2, 256, 32, 3), (1, 256, 128, 1), (8, 128, 16, 4)])
def test_moved_codes_are_the_definitions(hk, d, block, layers):
    new, held = [9, 0, 64, 5, 200, 30, 1], [0, 9, 40, 100, 63, 15, 30]
    g = torch.Generator().manual_seed(hk)
    paths = [sorted(torch.randperm(n, generator=g)[:max(1, n // 3)].tolist()) if n else [] for n in new]
    paths[0], paths[3] = [0, 2, 3, 8], [0, 1, 2]                               # nothing of the latter moves
    paths[4] = [0, 1] + sorted((torch.randperm(198, generator=g)[:150] + 2).tolist())
    _check_keep(new, held, paths, hk, d, block, layers, seed=block, behind=3, between=32)


def test_codes_that_are_nan_and_paths_that_are_none():
    new, held = [6, 20, 7, 8, 40, 3, 5], [13, 30, 1, 2, 3, 4, 16]
    paths = [[0, 3, 3, 5], [5, 2], [0, 9], [-1, 2], [2, 7, 30, 39, 40], [], [1, 2, 3, 4, 0, 0, 0]]
    _check_keep(new, held, paths, 2, 128, 16, 2, seed=3, nan=True)
    _check_keep(new, held, paths, 2, 128, 16, 1, seed=4, near=True)            # scales that are no powers of two, but the same


def test_blocks_that_are_none():
    new, held = [40, 30], [20, 3]
    total = [60, 33]
    table = _table(total, 16, 8, 1)
    table[0, 2], table[1, 0], table[1, 2] = -1, 8, 2 ** 31 - 1
    _check_keep(new, held, [[0, 5, 9, 13, 15, 33, 39], [1, 4, 20, 29]], 2, 128, 16, 2, seed=1, table=table)
    _check_keep(new, held, [[0, 5, 9, 13, 15, 33, 39], [1, 4, 20, 29]], 1, 256, 16, 1, seed=1, table=table[:, :2].contiguous())


def test_blocks_of_scale_zero():
    """Zeros that move to a block which was never written, and to one with a scale."""
    block, d = 16, 128
    k, ks, _ = _empty_cache(4, 2, block, d, 1)
    v, vs, _ = _empty_cache(4, 2, block, d, 2)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32)
    for c, s in ((k, ks), (v, vs)):
        s[0] = 0.0
        c.view(torch.uint8)[1] = 0                                             # 0 times any scale
        s[1] = 4.0
        s[3] = 0.0                                                             # and any codes times 0
    want = []
    for c, s in ((k, ks), (v, vs)):
        x, y = _as_values(c), s.cpu().double()
        for r in range(2):
            T.keep_path([0, 4, 7, 20], 24, 30, table[r], x, y, block)
        want.append((x, y))
    keep = _nv().paged_kv_keep_path(_i32(([0, 4, 7, 20] + [-1] * 20) * 2), _i32([4, 4]), _i32([0, 24, 48]), _i32([30, 30]), table.cuda(), k, v, ks, vs)
    assert keep.tolist() == [10, 10]
    for (x, y), c, s in zip(want, (k, v), (ks, vs)):
        assert torch.equal(_as_values(c), x) and torch.equal(s.cpu().double(), y)


def test_layers_inside_blocks():
    """[blocks, layers, ...] in memory: layers closer together than blocks."""
    k, ks, _ = _empty_cache(6 * 3, 2, 16, 128, 1)
    v, vs, _ = _empty_cache(6 * 3, 2, 16, 128, 2)
    ours = [x.unflatten(0, (6, 3)).transpose(0, 1) for x in (k, v, ks, vs)]
    plain = [x.contiguous() for x in ours]
    table = _table([40], 16, 6, 1)
    for x in (ours, plain):
        keep = _nv().paged_kv_keep_path(_i32([0, 4, 9] + [-1] * 27), _i32([3]), _i32([0, 30]), _i32([40]), table.cuda(), *x)
        assert keep.tolist() == [13]
    for a, b in zip(ours, plain):
        assert torch.equal(a.contiguous().view(torch.uint8), b.view(torch.uint8))


def test_layers_blocks_and_rows_past_32_bits():
    """Blocks half a gigabyte apart, layers 2.5: a path moved in both; rows of probabilities two gigabytes apart."""
    hk, block, d, apart, layer = 2, 16, 128, (1 << 29) + 4096, 5 << 29
    flat = torch.empty(layer + 5 * apart, dtype=torch.uint8, device="cuda")
    view = lambda at: flat.as_strided((2, 5, hk, block, d), (layer, apart, block * d, d, 1), at)
    small = [_empty_cache(2 * 5, hk, block, d, x) for x in (1, 2)]
    caches, scales = [view(0), view(1 << 20)], [x[1].view(2, 5, hk) for x in small]
    want = []
    for c, (codes, scale, _) in zip(caches, small):
        c.copy_(codes.view(torch.uint8).view(2, 5, hk, block, d))
        want.append([(_as_values(codes.view(2, 5, hk, block, d)[i]), scale.view(2, 5, hk)[i].cpu().double()) for i in (0, 1)])
    table = torch.tensor([[4, 0, 3], [2, 1, -1]], dtype=torch.int32)
    path, new, total = [0, 3, 20, 21, 29], [30, 25], [45, 32]
    for values in want:
        for x, y in values:
            for r in (0, 1):
                T.keep_path([a for a in path if a < new[r]], new[r], total[r], table[r], x, y, block)
    keep = _nv().paged_kv_keep_path(_i32(path + [-1] * 25 + path[:4] + [-1] * 21), _i32([5, 4]), _i32([0, 30, 55]), _i32(total), table.cuda(), *caches, *scales)
    assert keep.tolist() == [20, 11]
    for c, s, values in zip(caches, scales, want):
        for i, (x, y) in enumerate(values):
            assert torch.equal(c[i].contiguous().cpu().view(torch.float8_e4m3fn).double(), x) and torch.equal(s[i].cpu().double(), y)
    del flat, caches, view
    v, stride = 700, (1 << 29) + 5
    wide = torch.empty(5 * stride, device="cuda")
    p = wide.as_strided((5, v), (stride, 1), 3)
    p.copy_(_rows(5, v, 1).cuda())
    parents, u = [-1, 0, 1, 2, 3], torch.tensor([0.7, 1e-6, 1e-6, 1e-6, 1e-6])
    tokens = p.argmax(1).roll(1).cpu()
    got = _nv().verify_drafts(p, tokens.cuda(), _i32(parents), _i32([0, 5]), u.cuda())
    assert got.accepted.tolist() == [0, 1, 2, 3, 4]
    assert int(got.next_tokens) == T.verify(p.cpu().double().numpy(), tokens.tolist(), parents, u.double().numpy())[1]
    got = _nv().verify_drafts(p, tokens.cuda(), _i32(parents), _i32([0, 5]), u.cuda(), p)
    assert got.accepted.tolist() == [0, 1, 2, 3, 4]


# ------------------------------------------------------------------------------------------------ together
def _step(cache, layers, model, parents, tokens, u, cu_lens, most, g, scaling):
    """A step of drafted trees, as a server runs it; `model`: (query, key, value) of every layer, and the target's rows."""
    step = cache.reserve(cu_lens, tokens.shape[0])
    tree = cache.tree(parents, step.cu_seqlens, most)
    outs = []
    for layer in range(layers):
        q, k, v = model[layer]
        cache.write(layer, k, v, step.slot_map)
        outs.append(cache.attend_tree(layer, q, step.cu_seqlens, tree.tree_mask, scaling, g))
    got = _nv().verify_drafts(model[-1], tokens, parents, step.cu_seqlens, u)
    cache.keep_path(got.accepted, got.num_accepted, step.cu_seqlens)
    return step, tree, outs, got


def _state(cache):
    return [x.clone() for x in (cache.k, cache.v, cache.k_scale, cache.v_scale, cache.block_table, cache.lengths, cache.free_blocks, cache.free_count)]


def _filled(layers, held, seed):
    nv = _nv()
    cache = nv.FP8PagedKVCache(layers, 30, 2, 128, len(held), 200, "cuda", block_size=16)
    g = torch.Generator(device="cuda").manual_seed(seed)
    step = cache.reserve(_i32(held), sum(held))
    for layer in range(layers):
        kv = torch.randn(2, sum(held), 2, 128, generator=g, device="cuda").bfloat16()
        cache.write(layer, kv[0], kv[1], step.slot_map)
    return cache


def _inputs(layers, new, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = sum(new) + 4                                                           # a padded batch
    model = [tuple(2 * torch.randn(n, heads, 128, generator=g, device="cuda").bfloat16() for heads in (8, 2, 2)) for _ in range(layers)]
    p = torch.softmax(3 * torch.randn(n, 500, generator=g, device="cuda"), 1)
    parents = _parents(new, seed)
    starts = _starts(new)
    tokens = _drafts(p.cpu(), None, parents, starts, seed, likeliest=True)
    return [*model, p], _i32(parents + [0] * 4), tokens.cuda(), torch.rand(n, generator=g, device="cuda") * 0.6


def test_steps_of_trees_one_after_the_other():
    layers, held = 2, [40, 3, 15, 100]
    cache = _filled(layers, held, 1)
    length = list(held)
    for s, new in enumerate(([9, 12, 0, 30], [20, 1, 5, 7], [3, 16, 16, 2])):
        before = _state(cache)
        model, parents, tokens, u = _inputs(layers, new, 10 + s)
        step, tree, outs, got = _step(cache, layers, model, parents, tokens, u, _i32(new), 30, 4, 128 ** -0.5)
        assert int(step.shortage) == 0
        # the same tables and codes from the references, then the path moved in them
        table = before[4].cpu().clone()
        ref = dict(lengths=before[5].cpu().clone(), table=table, free=before[6].cpu().clone(), count=int(before[7]))
        slots, _, starts, _ = R.reserve(new, ref, tokens.shape[0], 16)
        for layer in range(layers):
            for which, name, scale in ((1, 0, 2), (2, 1, 3)):
                x, sc = _as_values(before[name][layer]), before[scale][layer].cpu().double()
                R.write(model[layer][which].cpu().double(), slots, x, sc, 16)
                if which == 1:
                    kk = x.clone(), sc.clone()
                else:
                    vv = x.clone(), sc.clone()
                for r, n in enumerate(new):
                    path = got.accepted[starts[r]:starts[r] + int(got.num_accepted[r])].tolist()
                    T.keep_path(path, n, length[r] + n, ref["table"][r], x, sc, 16)
                assert torch.equal((cache.k, cache.v)[which - 1][layer].cpu().double()[:, :, :, :], x)
                assert torch.equal((cache.k_scale, cache.v_scale)[which - 1][layer].cpu().double(), sc)
            for r, n in enumerate(new):
                seen, _ = T.tree(parents[starts[r]:starts[r + 1]].tolist(), 30)
                total = length[r] + n
                k1, v1 = (R.gather(c, sc, ref["table"][r], total, 16) for c, sc in (kk, vv))
                for i in sorted({0, n // 2, n - 1} & set(range(n))):
                    hidden = torch.cat([torch.zeros(length[r], dtype=torch.bool), ~seen[i]])
                    t = starts[r] + i
                    _close(outs[layer][t:t + 1], None, model[layer][0][t:t + 1], k1, v1, _key_scales(vv[1].float(), ref["table"][r], total, 16), [total],
                           128 ** -0.5, 4, hidden=hidden, chunk=_chunk(torch.bfloat16, 128, tokens.shape[0], 4, 4))
        length = [a + int(x) for a, x in zip(length, got.num_accepted)]
        R.trim(length, ref, 16)
        assert cache.lengths.tolist() == length and cache.block_table.tolist() == ref["table"].tolist()
        assert int(cache.free_count) == ref["count"] and cache.free_blocks[:ref["count"]].tolist() == ref["free"][:ref["count"]].tolist()


def test_a_step_that_does_not_fit_keeps_everything():
    cache = _filled(2, [40, 3, 15, 100], 1)
    before = _state(cache)
    model, parents, tokens, u = _inputs(2, [150, 150, 150, 90], 3)             # more blocks than there are
    step, tree, outs, got = _step(cache, 2, model, parents, tokens, u, _i32([150, 150, 150, 90]), 150, 4, 0.1)
    assert int(step.shortage) == 1 and not tree.tree_mask.any() and not tree.positions.any()
    assert all(not o.any() for o in outs)
    assert bool((got.accepted == -1).all()) and got.num_accepted.tolist() == [0] * 4 and got.next_tokens.tolist() == [-1] * 4
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(_state(cache), before))


def test_a_captured_step_of_trees():
    layers, new = 2, [9, 12, 0, 30]
    model, parents, tokens, u = _inputs(layers, new, 3)
    lens = _i32(new)

    def run(cache):
        step, tree, outs, got = _step(cache, layers, model, parents, tokens, u, lens, 30, 4, 128 ** -0.5)
        return [*step, *tree, *outs, *got]

    eager_cache = _filled(layers, [40, 3, 15, 100], 1)
    start = _state(eager_cache)
    eager = [x.clone() for x in run(eager_cache)]
    cache = _filled(layers, [40, 3, 15, 100], 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(cache)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run(cache)
    for _ in range(2):
        for x, y in zip((cache.k, cache.v, cache.k_scale, cache.v_scale, cache.block_table, cache.lengths, cache.free_blocks, cache.free_count), start):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager))
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(_state(cache), _state(eager_cache)))
    del graph


def test_calls_on_two_streams_at_once():
    sets = [_inputs(1, [9, 12, 3, 30], s) for s in (1, 2)]
    caches = [_filled(1, [40, 3, 15, 100], s) for s in (1, 2)]
    lens = _i32([9, 12, 3, 30])
    again = [_filled(1, [40, 3, 15, 100], s) for s in (1, 2)]
    want = [_step(c, 1, *i[:2], *i[2:], lens, 30, 4, 0.1) for c, i in zip(again, sets)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for st, c, i in zip(streams, caches, sets):
        with torch.cuda.stream(st):
            got.append(_step(c, 1, *i, lens, 30, 4, 0.1))
    torch.cuda.synchronize()
    for a, b, ca, cb in zip(got, want, caches, again):
        assert torch.equal(a[2][0], b[2][0]) and all(torch.equal(x, y) for x, y in zip(a[3], b[3]))
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(_state(ca), _state(cb)))


def test_registered_operators_give_the_same():
    import sageattention_b200.nvfp4.custom_ops  # noqa: F401
    ops, nv = torch.ops.sageattention_b200, _nv()
    model, parents, tokens, u = _inputs(1, [9, 12, 0, 30], 3)
    starts = _i32(_starts([9, 12, 0, 30]))
    cache = _filled(1, [60, 30, 15, 100], 1)
    mask, pos = ops.draft_tree(parents, starts, cache.lengths, 64)
    assert all(torch.equal(a, b) for a, b in zip((mask, pos), nv.draft_tree(parents, starts, cache.lengths, 64)))
    args = (cache.k[0], cache.v[0], cache.k_scale[0], cache.v_scale[0], cache.block_table, cache.lengths, 0.1, 4)
    assert all(torch.equal(a, b) for a, b in zip(ops.fp8_paged_tree_attention(model[0][0], starts, mask, *args),
                                                 nv.fp8_paged_tree_attention(model[0][0], starts, mask, *args, True)))
    got = ops.verify_drafts(model[-1], tokens, parents, starts, u, None)
    assert all(torch.equal(a, b) for a, b in zip(got, nv.verify_drafts(model[-1], tokens, parents, starts, u)))
    other = _filled(1, [60, 30, 15, 100], 1)
    keep = ops.paged_kv_keep_path(got[0], got[1], starts, cache.lengths, cache.block_table, cache.k, cache.v, cache.k_scale, cache.v_scale)
    assert torch.equal(keep, nv.paged_kv_keep_path(got[0], got[1], starts, other.lengths, other.block_table, other.k, other.v, other.k_scale, other.v_scale))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(_state(cache), _state(other)))


# ------------------------------------------------------------------------------------------------ refusals
def test_arguments_that_are_refused():
    nv = _nv()
    i64 = lambda *s: torch.zeros(*s, dtype=torch.int64, device="cuda")
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    for most in (0, 1025, -1):
        with pytest.raises(AssertionError, match="max_tokens"):
            nv.draft_tree(i(3), i(2), i(1), most)
    with pytest.raises(TypeError, match="parents"):
        nv.draft_tree(i64(3), i(2), i(1), 3)
    with pytest.raises(AssertionError, match="lengths"):
        nv.draft_tree(i(3), i(2), i(2), 3)
    with pytest.raises(AssertionError, match="cu_seqlens"):
        nv.draft_tree(i(3), i(1), i(0), 3)
    with pytest.raises(RuntimeError, match="no CPU path"):
        nv.draft_tree(i(3), i(2).cpu(), i(1), 3)
    c, s = torch.zeros(4, 1, 16, 128, dtype=torch.float8_e4m3fn, device="cuda"), torch.zeros(4, 1, device="cuda")
    q = torch.zeros(3, 2, 128, device="cuda")
    for bad, error in ((i(3, 1), TypeError), (i64(2, 1), AssertionError), (i64(3), AssertionError), (i64(3, 0), AssertionError),
                       (i64(3, 2)[:, :1], AssertionError)):
        with pytest.raises(error, match="tree_mask"):
            nv.fp8_paged_tree_attention(q, i(2), bad, c, c, s, s, i(1, 2), i(1), 1.0, 2)
    with pytest.raises(RuntimeError, match="scaling"):
        nv.fp8_paged_tree_attention(q, i(2), i64(3, 1), c, c, s, s, i(1, 2), i(1), math.inf, 2)
    p, u = torch.zeros(3, 9, device="cuda"), torch.zeros(3, device="cuda")
    with pytest.raises(TypeError, match="draft_probs"):
        nv.verify_drafts(p, i(3), i(3), i(2), u, p.half())
    with pytest.raises(AssertionError, match="draft_probs"):
        nv.verify_drafts(p, i(3), i(3), i(2), u, p[:, :8])
    with pytest.raises(TypeError, match="tokens"):
        nv.verify_drafts(p, u, i(3), i(2), u)
    with pytest.raises(TypeError, match="dtype"):
        nv.verify_drafts(p.double(), i(3), i(3), i(2), u)
    with pytest.raises(AssertionError, match="uniforms"):
        nv.verify_drafts(p, i(3), i(3), i(2), u[:2])
    with pytest.raises(ValueError, match="target_probs"):
        nv.verify_drafts(p[0], i(3), i(3), i(2), u)
    many, scales = c[None].repeat(2, 1, 1, 1, 1), s[None].repeat(2, 1, 1)
    args = (i(3), i(1), i(2), i(1), i(1, 2))
    for bad in ((many, c, scales, s), (many, many, s, s), (many, many[:1], scales, scales), (many, many, scales, scales[:1]),
                (many[0].expand(2, -1, -1, -1, -1), many, scales, scales), (many, many, scales[0].expand(2, -1, -1), scales)):
        with pytest.raises((AssertionError, ValueError)):
            nv.paged_kv_keep_path(*args, *bad)
    with pytest.raises(AssertionError, match="num_accepted"):
        nv.paged_kv_keep_path(i(3), i(2), *args[2:], c, c, s, s)
