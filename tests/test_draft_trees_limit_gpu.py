"""Trees that are larger than the step's max_tokens: what was attended without its ancestors is never kept."""

import pytest
import torch

import draft_reference as T
from test_draft_trees_gpu import _drafts, _filled, _i32, _nv, _parents, _rows, _starts

pytestmark = pytest.mark.gpu


def _cut(parents, starts, most):
    """Parents of the trees' first `most` nodes; the others hang on nothing."""
    out = list(parents)
    for a, b in zip(starts[:-1], starts[1:]):
        out[a + most:b] = [-1] * max(0, b - a - most)
    return out


@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("most", [1, 2, 9, 16, 31, 32, 33, 40, 64, 1024])
def test_nothing_behind_the_limit_is_kept(most, drawn):
    new = [20, 40, 33, 1, 0, 17, 64, 32]
    starts = _starts(new)
    for branch, seed in ((1, 1), (2, 2), (4, 3)):
        parents = [i - 1 for n in new for i in range(n)] if branch == 1 else _parents(new, seed, branch)
        p = _rows(sum(new), 300, seed)
        q = 0.7 * p + 0.3 * _rows(sum(new), 300, seed + 9) if drawn else None
        tokens = _drafts(p, q, parents, starts, seed, likeliest=not drawn)
        u = 0.2 * torch.rand(sum(new), generator=torch.Generator().manual_seed(seed))
        got = _nv().verify_drafts(p.cuda(), tokens.cuda(), _i32(parents), _i32(starts), u.cuda(), None if q is None else q.cuda(), most)
        cut = _cut(parents, starts, most)
        for r, (a, b) in enumerate(zip(starts[:-1], starts[1:])):
            path, x = T.verify(p[a:b].double().numpy(), tokens[a:b].tolist(), cut[a:b], u[a:b].double().numpy(),
                               None if q is None else q[a:b].double().numpy())
            assert got.accepted[a:b].tolist() == path + [-1] * (b - a - len(path))
            assert int(got.num_accepted[r]) == len(path) and int(got.next_tokens[r]) == x
            assert all(i < most for i in path)


def _chain_step(cache, lens, tokens, parents, inputs, probs, u, most):
    """A step of chains whose drafts all pass, as far as they may."""
    q, k, v = inputs
    step = cache.reserve(lens, tokens.shape[0])
    tree = cache.tree(parents, step.cu_seqlens, most)
    cache.write(0, k, v, step.slot_map)
    out = cache.attend_tree(0, q, step.cu_seqlens, tree.tree_mask, 0.1, 4)
    got = _nv().verify_drafts(probs, tokens, parents, step.cu_seqlens, u, max_tokens=most)
    cache.keep_path(got.accepted, got.num_accepted, step.cu_seqlens)
    return out, got, tree


def _chains(new, slots):
    """Chains: every token's row has the next token alone."""
    g = torch.Generator(device="cuda").manual_seed(4)
    inputs = [torch.randn(slots, heads, 128, generator=g, device="cuda").bfloat16() for heads in (8, 2, 2)]
    tokens = torch.arange(slots, device="cuda") % 50
    probs = torch.nn.functional.one_hot((tokens + 1) % 50, 50).float()
    parents = _i32([i - 1 for n in new for i in range(n)] + [0] * (slots - sum(new)))
    return tokens, parents, inputs, probs, torch.full((slots,), 0.5, device="cuda")


@pytest.mark.parametrize("most", [3, 10, 32])
def test_a_step_keeps_a_tree_as_far_as_it_was_attended(most):
    new, held = [40, 3, 12, 33], [40, 3, 15, 100]
    tokens, parents, inputs, probs, u = _chains(new, sum(new) + 4)
    cache, whole = _filled(1, held, 1), _filled(1, held, 1)
    out, got, _ = _chain_step(cache, _i32(new), tokens, parents, inputs, probs, u, most)
    want, full, _ = _chain_step(whole, _i32(new), tokens, parents, inputs, probs, u, 64)
    kept = [min(n, most) for n in new]
    assert got.num_accepted.tolist() == kept and full.num_accepted.tolist() == new
    assert cache.lengths.tolist() == [a + b for a, b in zip(held, kept)]
    for r, (a, n) in enumerate(zip(_starts(new), kept)):
        # what is kept was attended with all of its ancestors, and the token behind it comes from its own row
        assert torch.equal(out[a:a + n], want[a:a + n])
        assert int(got.next_tokens[r]) == (int(tokens[a + n - 1]) + 1) % 50
    if most < 33:
        assert not torch.equal(out[:40], want[:40])


def test_a_captured_step_that_meets_larger_trees():
    """max_tokens stays as it was captured; the trees' sizes are on the device."""
    small, large, held, slots = [5, 3, 8, 1], [40, 8, 2, 20], [40, 3, 15, 100], 80
    tokens, parents, inputs, probs, u = _chains(small, slots)
    lens = _i32(small)
    cache = _filled(1, held, 1)
    start = [x.clone() for x in (cache.k, cache.v, cache.k_scale, cache.v_scale, cache.block_table, cache.lengths, cache.free_blocks, cache.free_count)]
    state = lambda: (cache.k, cache.v, cache.k_scale, cache.v_scale, cache.block_table, cache.lengths, cache.free_blocks, cache.free_count)

    def back():
        for x, y in zip(state(), start):
            x.copy_(y)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _chain_step(cache, lens, tokens, parents, inputs, probs, u, 8)
    torch.cuda.current_stream().wait_stream(side)
    back()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, got, _ = _chain_step(cache, lens, tokens, parents, inputs, probs, u, 8)
    for new in (small, large):
        back()
        lens.copy_(_i32(new))
        parents.copy_(_i32([i - 1 for n in new for i in range(n)] + [0] * (slots - sum(new))))
        graph.replay()
        torch.cuda.synchronize()
        kept = [min(n, 8) for n in new]
        assert got.num_accepted.tolist() == kept and cache.lengths.tolist() == [a + b for a, b in zip(held, kept)]
    del graph


def test_limits_that_are_refused():
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    for most in (0, 1025, -1):
        with pytest.raises(AssertionError, match="max_tokens"):
            _nv().verify_drafts(torch.zeros(3, 9, device="cuda"), i(3), i(3), i(2), torch.zeros(3, device="cuda"), max_tokens=most)
    import sageattention_b200.nvfp4.custom_ops  # noqa: F401
    args = (torch.full((3, 9), 1 / 9, device="cuda"), i(3), _i32([-1, 0, 1]), _i32([0, 3]), torch.zeros(3, device="cuda"), None)
    assert torch.ops.sageattention_b200.verify_drafts(*args)[1].tolist() == [3]
    assert torch.ops.sageattention_b200.verify_drafts(*args, 2)[1].tolist() == [2]
