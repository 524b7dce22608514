"""What follows a kept draft is distributed as the target's own draws behind it, also where siblings in front of it were rejected."""

import pytest
import torch

pytestmark = pytest.mark.gpu

_V = 5
_FIRST = torch.tensor([0.35, 0.05, 0.25, 0.2, 0.15])
_FIRST_DRAFT = torch.tensor([0.1, 0.4, 0.2, 0.1, 0.2])


def _tables(seed):
    g = torch.Generator().manual_seed(seed)
    return torch.softmax(1.2 * torch.randn(_V, _V, generator=g), 1), torch.softmax(1.2 * torch.randn(_V, _V, generator=g), 1)


@pytest.mark.parametrize("kind", ["chain", "drawn", "likeliest"])
def test_the_second_token(kind):
    """120000 requests of trees of two levels, over five tokens: of those that keep a first draft t, the next token (a kept draft or
    the one that is drawn) is one of target[t]: each count within five standard deviations of its own, for every t, over all and over
    those where a sibling in front was rejected."""
    import sageattention_b200.nvfp4 as nv
    n = 120000
    g = torch.Generator().manual_seed(21)
    target, draft = _tables(3)
    chosen = kind == "likeliest"
    width, below = (1, 1) if kind == "chain" else (3, 2)
    # node 0, its children, their children
    parents = [-1] + [0] * width + [1 + i for i in range(width) for _ in range(below)]
    nodes = len(parents)
    tokens = torch.zeros(n, nodes, dtype=torch.long)
    if chosen:
        tokens[:, 1:1 + width] = torch.tensor([1, 3, 0])
        tokens[:, 1 + width:] = target.topk(2, 1).indices[tokens[:, 1:1 + width]].flatten(1)
    else:
        tokens[:, 1:1 + width] = torch.multinomial(_FIRST_DRAFT.expand(n, _V), width, replacement=True, generator=g)
        rows = draft[tokens[:, 1:1 + width]].flatten(0, 1)
        tokens[:, 1 + width:] = torch.multinomial(rows, below, replacement=True, generator=g).view(n, -1)
    p, q = target[tokens].clone(), draft[tokens].clone()
    p[:, 0], q[:, 0] = _FIRST, _FIRST_DRAFT
    got = nv.verify_drafts(p.flatten(0, 1).cuda(), tokens.flatten().cuda(), torch.tensor(parents, dtype=torch.int32).repeat(n).cuda(),
                           (torch.arange(n + 1) * nodes).int().cuda(), torch.rand(n * nodes, generator=g).cuda(),
                           None if chosen else q.flatten(0, 1).cuda())
    path, count, after = got.accepted.view(n, nodes).cpu().long(), got.num_accepted.cpu(), got.next_tokens.cpu()
    assert int(count.max()) == 3
    node = path[:, 1].clamp(min=0)
    first = tokens.gather(1, node[:, None])[:, 0]
    second = torch.where(count > 2, tokens.gather(1, path[:, 2].clamp(min=0)[:, None])[:, 0], after)
    kept = count > 1
    for where in [kept] + ([kept & (node > 1)] if width > 1 else []):
        met = 0
        for t in range(_V):
            mine = second[where & (first == t)]
            if mine.numel() < 500:
                continue
            met += 1
            seen, want = torch.bincount(mine, minlength=_V).double() / mine.numel(), target[t].double()
            assert bool(((seen - want).abs() <= 5 * (want * (1 - want) / mine.numel()).sqrt()).all()), (t, seen, want)
        assert met >= 2 and (met == _V or chosen or where is not kept)
