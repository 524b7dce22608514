"""What a caller may do with the results of the norm with rotation: change them in place, whatever their layout."""

import pytest
import torch

pytestmark = pytest.mark.gpu

_CALLS = ["entry", "registered"]
# [T, H, D]; [Z, H, S, D] with heads outside of tokens; the same as views of a projection; one head, one token
_LAYOUTS = {"tokens": lambda n: (20, n, 128), "heads": lambda n: (2, n, 20, 128), "views": lambda n: (2, 20, n, 128), "one": lambda n: (3, 1, 1, 128)}


def _call(kind):
    import sageattention_b200.nvfp4 as nv
    if kind == "entry":
        return nv.qk_norm_rope
    import sageattention_b200.nvfp4.custom_ops  # noqa: F401
    return lambda *x: torch.ops.sageattention_b200.qk_norm_rope(*x, None, 0, 1e-6)


def _operands(layout, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k = (torch.randn(_LAYOUTS[layout](n), generator=g, device="cuda") for n in (4, 2))
    if layout == "views":
        q, k = q.transpose(1, 2), k.transpose(1, 2)
    w = 1 + 0.1 * torch.randn(2, 128, generator=g, device="cuda")
    angle = torch.arange(20, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, 128, 2, device="cuda") / 128)
    return q, k, w[0].clone(), w[1].clone(), angle.cos(), angle.sin()


@pytest.mark.parametrize("kind", _CALLS)
@pytest.mark.parametrize("layout", list(_LAYOUTS))
def test_results_changed_in_place(layout, kind):
    """In the graph, and by a product with something that has a gradient of its own; the gradients are those of new tensors."""
    f, ops = _call(kind), _operands(layout)
    scale = torch.full((), 0.5, device="cuda")

    def grads(change):
        leaves = [x.detach().requires_grad_(True) for x in ops[:4]] + [scale.clone().requires_grad_(True)]
        q, k = f(*leaves[:4], *ops[4:])
        q, k = change(q, k, leaves[4])
        return q, k, torch.autograd.grad((q * q).sum() + (k * k).sum(), leaves)

    want = grads(lambda q, k, s: (q * s, k * 3.0))

    def change(q, k, s):
        q *= s
        k.mul_(3.0)
        return q, k

    got = grads(change)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert all(torch.equal(a, b) for a, b in zip(got[2], want[2]))


@pytest.mark.parametrize("kind", _CALLS)
@pytest.mark.parametrize("layout", list(_LAYOUTS))
def test_results_without_a_graph_are_changed_in_one(layout, kind):
    """Operands without gradients: a result is a plain tensor that may join a graph in place."""
    f, ops = _call(kind), _operands(layout)
    s = torch.full((), 0.5, device="cuda", requires_grad=True)
    (want,) = torch.autograd.grad((f(*ops)[0] * s).sum(), s)
    q, _ = f(*ops)
    q.mul_(s)
    assert torch.equal(torch.autograd.grad(q.sum(), s)[0], want)


@pytest.mark.parametrize("layout", list(_LAYOUTS))
def test_results_changed_where_nothing_is_recorded(layout):
    import sageattention_b200.nvfp4 as nv
    ops = _operands(layout)
    leaves = [x.detach().requires_grad_(True) for x in ops[:4]]
    q, k = nv.qk_norm_rope(*leaves, *ops[4:])
    with torch.no_grad():
        q.mul_(2.0)
    assert q.grad_fn is not None and k.grad_fn is not None
    want = torch.autograd.grad(nv.qk_norm_rope(*leaves, *ops[4:])[0].sum(), leaves[0])[0]
    assert torch.equal(torch.autograd.grad(q.sum(), leaves[0])[0], want)


@pytest.mark.parametrize("layout", list(_LAYOUTS))
def test_no_result_or_gradient_is_a_view(layout):
    import sageattention_b200.nvfp4 as nv
    ops = _operands(layout)
    leaves = [x.detach().requires_grad_(True) for x in ops[:4]]
    out = nv.qk_norm_rope(*leaves, *ops[4:])
    grads = torch.autograd.grad(out, leaves, [torch.ones_like(x) for x in out])
    for y, x in (*zip(out, ops), *zip(grads, ops)):
        assert y._base is None and y.shape == x.shape
        if layout != "one":
            assert y.stride() == x.stride()
    s = torch.full((), 0.5, device="cuda", requires_grad=True)
    assert (grads[0].mul_(s)).requires_grad


def test_no_tokens_as_views():
    import sageattention_b200.nvfp4 as nv
    _, _, wq, wk, cos, sin = _operands("views")
    x = torch.zeros(2, 0, 4, 128, device="cuda").transpose(1, 2).requires_grad_(True)
    q, k = nv.qk_norm_rope(x, x, wq, wk, cos, sin)
    assert q.shape == k.shape == (2, 4, 0, 128)
    (q.sum() + k.sum()).backward()
    assert x.grad.shape == x.shape
