"""Norm and rotation of queries and keys against their formulas in 64 bits, and their gradients against the formulas and against
differences.

Tolerances.  A row's sum of squares is 16 products a lane and at most four more additions of lanes, then rsqrt (2 ulp), so r is off by
at most 12 steps of 2^-24 relative (half of the sum's 20, and 2); the result has four more roundings in fp32 and one to its type:
(16 + 8) 2^-24 of what the rotation adds up, and half a step of the result (fp16: or of its subnormals, 2^-25).  A gradient of x adds
the mean of g' w n, whose error is at most 40 roundings of sum |g' w n| / D, and two more products.  A gradient of a weight sums
rows: at most one rounding a row and 48 for a product's own, of sum |g' n|."""

import pytest
import torch

import draft_reference as T

pytestmark = pytest.mark.gpu

_HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
_F = 2.0 ** -24


def _nv():
    import sageattention_b200.nvfp4 as nv
    return nv


def _tables(p, d, seed=None):
    """Angles of position and channel; with a seed, tables that are no rotation."""
    a = torch.arange(p, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    if seed is None:
        return a.cos().float(), a.sin().float()
    g = torch.Generator().manual_seed(seed)
    return torch.randn(p, d // 2, generator=g), torch.randn(p, d // 2, generator=g)


def _operands(shape_q, shape_k, dtype, wdtype, seed):
    g = torch.Generator().manual_seed(seed)
    d = shape_q[-1]
    q, k = (torch.randn(*s, generator=g) * torch.exp(torch.randn(*s[:-1], 1, generator=g)) for s in (shape_q, shape_k))
    wq, wk = 1 + 0.5 * torch.randn(2, d, generator=g)
    return q.to(dtype), k.to(dtype), wq.to(wdtype), wk.to(wdtype)


def _at(table, positions, dim):
    """Rows of a table broadcast to [T, H, D/2] or [Z, H, S, D/2]."""
    x = table.double()[positions.long()]
    return x[:, None] if dim == 3 else x if positions.dim() == 1 else x[:, None]


def _tiny(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 1e-37


def _check_forward(got, x, w, cos, sin, eps):
    want, n, _ = T.norm_rope(x.double(), w.double(), cos, sin, eps)
    tol = 24 * _F * T.turned_size(n * w.double(), cos, sin) + _HALF_STEP[x.dtype] * want.abs() + _tiny(x.dtype)
    off = (got.cpu().double() - want).abs()
    assert got.shape == x.shape and got.dtype == x.dtype
    assert bool((off <= tol).all()), float((off / tol).max())


def _check_backward(dx, dw, x, w, cos, sin, eps, g):
    want, want_w, back, n, r = T.norm_rope_grads(x.double(), w.double(), cos, sin, eps, g.double())
    size = T.turned_size(g.double(), cos, sin)                       # of g'
    part = (size * w.double().abs() * n.abs()).mean(-1, keepdim=True)
    tol = 48 * _F * r * (size * w.double().abs() + n.abs() * part) + _HALF_STEP[x.dtype] * want.abs() + _tiny(x.dtype)
    off = (dx.cpu().double() - want).abs()
    assert dx.shape == x.shape and dx.dtype == x.dtype
    assert bool((off <= tol).all()), float((off / tol).max())
    if dw is not None:
        rows = x.numel() // x.shape[-1]
        tol = (rows + 48) * _F * (size * n.abs()).flatten(0, -2).sum(0) + _HALF_STEP[w.dtype] * want_w.abs() + _tiny(w.dtype)
        off = (dw.cpu().double() - want_w).abs()
        assert dw.shape == w.shape and dw.dtype == w.dtype and bool((off <= tol).all()), float((off / tol).max())


_SIZES = [((1, 1, 128), 1), ((3, 4, 128), 1), ((33, 32, 128), 8), ((130, 7, 256), 1), ((5, 3, 256), 3), ((257, 40, 128), 5), ((64, 2, 256), 2)]


@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                          (torch.float16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("shape,hk", _SIZES)
def test_tokens_heads(shape, hk, dtype, wdtype):
    t, h, d = shape
    q, k, wq, wk = _operands(shape, (t, hk, d), dtype, wdtype, t)
    g = torch.Generator().manual_seed(t)
    pos = torch.randint(500, (t,), generator=g).int()
    cos, sin = _tables(500, d, seed=4 if t == 33 else None)
    c, s = _at(cos, pos, 3), _at(sin, pos, 3)
    leaves = [x.cuda().requires_grad_(True) for x in (q, k, wq, wk)]
    out = _nv().qk_norm_rope(*leaves, cos.cuda(), sin.cuda(), pos.cuda(), eps=1e-5)
    grads = [torch.randn(x.shape, generator=g).to(dtype) for x in (q, k)]
    dq, dk, dwq, dwk = torch.autograd.grad(out, leaves, [x.cuda() for x in grads])
    for y, dx, dw, x, w, gr in ((out[0], dq, dwq, q, wq, grads[0]), (out[1], dk, dwk, k, wk, grads[1])):
        _check_forward(y.detach(), x, w, c, s, 1e-5)
        _check_backward(dx, dw, x, w, c, s, 1e-5, gr)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("z,h,hk,s,d", [(1, 4, 2, 77, 128), (3, 8, 1, 130, 128), (2, 6, 6, 33, 256), (2, 1, 1, 1, 128)])
@pytest.mark.parametrize("inside", [True, False])
def test_batches(z, h, hk, s, d, dtype, inside):
    """Heads inside of tokens (a projection's view) or outside; positions of all entries, of each, or counted on."""
    q, k, wq, wk = _operands((z, h, s, d), (z, hk, s, d), dtype, dtype, s)
    lay = (lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)) if inside else (lambda x: x)
    cos, sin = _tables(300, d)
    g = torch.Generator().manual_seed(s)
    grads = [torch.randn(x.shape, generator=g).to(dtype) for x in (q, k)]
    own = torch.randint(300, (z, s), generator=g)
    for pos, pos0, given in ((torch.arange(s) + 11, 11, None), (torch.arange(s) + 5, 0, (torch.arange(s) + 5).int()), (own, 0, own)):
        leaves = [x.requires_grad_(True) for x in (lay(q.cuda()).detach(), lay(k.cuda()).detach(), wq.cuda().detach(), wk.cuda().detach())]
        out = _nv().qk_norm_rope(*leaves, cos.cuda(), sin.cuda(), None if given is None else given.cuda(), pos0)
        if h > 1 and s > 1:
            assert out[0].transpose(1, 2).is_contiguous() == inside
        res = torch.autograd.grad(out, leaves, [lay(x.cuda()) for x in grads])
        c, sn = _at(cos, pos, 4), _at(sin, pos, 4)
        for i, (x, w) in enumerate(((q, wq), (k, wk))):
            _check_forward(out[i].detach(), x.detach(), w, c, sn, 1e-6)
            _check_backward(res[i], res[2 + i], x.detach(), w, c, sn, 1e-6, grads[i])


@pytest.mark.parametrize("seed", range(40))
def test_any_heads_lengths_and_strides(seed):
    """Heads that fill a step and a task or do not, tokens apart, heads apart, gradients laid out otherwise than results."""
    g = torch.Generator().manual_seed(1000 + seed)
    pick = lambda *x: x[int(torch.randint(len(x), (1,), generator=g))]
    d, dtype, four = pick(128, 256), pick(torch.bfloat16, torch.float16, torch.float32), pick(True, False)
    hk, h = pick(1, 2, 3, 4, 5, 8), pick(1, 2, 3, 6, 7, 12, 17, 20, 33)
    z, s = (pick(1, 2, 3) if four else 1), pick(1, 2, 3, 15, 16, 17, 31, 64, 129, 300)
    w = pick(dtype, torch.float32)
    gap, lead = pick(0, 0, 1, 2), pick(0, 3)                                   # heads between heads, tokens in front

    def laid(x):                                                               # [Z, H, S, D]
        n = x.shape[1]
        if pick(True, False):                                                  # tokens outside
            buf = torch.zeros(z, s + lead, n * (1 + gap), d, dtype=dtype, device="cuda")
            view = buf[:, lead:, ::1 + gap].transpose(1, 2)
        else:
            buf = torch.zeros(z, n * (1 + gap), s + lead, d, dtype=dtype, device="cuda")
            view = buf[:, ::1 + gap, lead:]
        view.copy_(x)
        return view

    q, k, wq, wk = _operands((z, h, s, d), (z, hk, s, d), dtype, w, seed)
    cos, sin = _tables(400, d, seed=seed)
    pos = torch.randint(400, (z, s) if four else (s,), generator=g).int()
    c, sn = _at(cos, pos if four else pos[None], 4), _at(sin, pos if four else pos[None], 4)
    flat = (lambda x: x) if four else (lambda x: x[0].transpose(0, 1))         # [T, H, D]
    back = (lambda x: x) if four else (lambda x: x.transpose(0, 1)[None])
    leaves = [flat(laid(q)).detach().requires_grad_(True), flat(laid(k)).detach().requires_grad_(True),
              wq.cuda().requires_grad_(True), wk.cuda().requires_grad_(True)]
    out = _nv().qk_norm_rope(*leaves, cos.cuda(), sin.cuda(), pos.cuda())
    grads = [torch.randn(x.shape, generator=g).to(dtype) for x in (q, k)]
    res = torch.autograd.grad(out, leaves, [flat(laid(x)) for x in grads])
    for i, (x, wt) in enumerate(((q, wq), (k, wk))):
        _check_forward(back(out[i].detach()), x, wt, c, sn, 1e-6)
        _check_backward(back(res[i]), res[2 + i], x, wt, c, sn, 1e-6, grads[i])


def test_views_of_a_projection_unaligned_and_broadcast_operands():
    nv = _nv()
    g = torch.Generator().manual_seed(1)
    cos, sin = (x.cuda() for x in _tables(64, 128))
    w = (1 + 0.1 * torch.randn(128, generator=g)).bfloat16().cuda()
    pos = torch.randint(64, (50,), generator=g).int().cuda()
    x = torch.randn(50, 12 * 128 + 8, generator=g).bfloat16().cuda()
    for off in (0, 8, 3):                                                      # aligned, still aligned, not
        heads = x[:, off:off + 12 * 128 if off < 8 else None].unflatten(1, (12, 128))
        q, k = heads[:, :8], heads[:, 8:10]
        a = nv.qk_norm_rope(q, k, w, w, cos, sin, pos)
        b = nv.qk_norm_rope(q.contiguous(), k.contiguous(), w, w, cos, sin, pos)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and a[0].is_contiguous()
    # one row for all heads and tokens, and a gradient that is one value for all
    one = torch.randn(1, 1, 128, generator=g).cuda().requires_grad_(True)
    wf = torch.ones(128, device="cuda").requires_grad_(True)
    q, k = one.expand(50, 4, 128), one.expand(50, 2, 128)
    out = nv.qk_norm_rope(q, k, wf, wf, cos, sin, pos)
    (out[0].sum() + out[1].sum()).backward()
    y = one.detach().cpu().double().requires_grad_(True)
    u = torch.ones(128, dtype=torch.float64, requires_grad=True)
    c, s = _at(cos.cpu(), pos.cpu(), 3), _at(sin.cpu(), pos.cpu(), 3)
    (T.norm_rope(y.expand(50, 4, 128), u, c, s, 1e-6)[0].sum() + T.norm_rope(y.expand(50, 2, 128), u, c, s, 1e-6)[0].sum()).backward()
    # 300 rows of gradients of at most 2 r |w| and (a weight's) 2 |n| each, every one off by less than 48 + 48 roundings, and as many
    # again of the sums
    r, n = float(1 / y.detach().square().mean().sqrt()), float(y.detach().abs().max() / y.detach().square().mean().sqrt())
    assert float((one.grad.cpu().double() - y.grad).abs().max()) <= 300 * 2 * r * (1 + n * n) * (96 + 300) * _F
    assert float((wf.grad.cpu().double() - u.grad).abs().max()) <= 300 * 2 * n * (96 + 300) * _F


def test_rows_of_zeros_infinities_and_positions_outside():
    nv = _nv()
    cos, sin = (x.cuda() for x in _tables(10, 128))
    x = torch.randn(6, 4, 128, generator=torch.Generator().manual_seed(1)).cuda()
    x[1] = 0
    x[2, 1, 5], x[2, 2, 70] = float("inf"), float("nan")
    x[3] *= 1e-30
    w = torch.ones(128, device="cuda")
    pos = torch.tensor([0, 3, 9, 5, -1, 10], dtype=torch.int32, device="cuda")
    a = x.clone().requires_grad_(True)
    q, k = nv.qk_norm_rope(a, x, w, w, cos, sin, pos)
    assert bool((q[1] == 0).all()) and bool(torch.isnan(q[2, 1:3]).any(1).all()) and bool(torch.isfinite(q[2, [0, 3]]).all())
    assert bool(torch.isfinite(q[3]).all()) and bool(torch.isnan(q[4:]).all()) and torch.equal(torch.nan_to_num(q), torch.nan_to_num(k))
    far, _ = nv.qk_norm_rope(x, x, w, w, cos, sin, torch.tensor([0, 3, 9, 5, -1 - 2 ** 32, 2 ** 32], device="cuda"))
    assert torch.equal(torch.nan_to_num(far), torch.nan_to_num(q.detach()))
    (grad,) = torch.autograd.grad(q, a, torch.ones_like(q))
    assert bool(torch.isfinite(grad[[0, 1, 3]]).all()) and bool(torch.isfinite(grad[2, [0, 3]]).all()) and bool(torch.isnan(grad[4:]).all())


def test_rows_past_32_bits():
    """Tokens half a gigabyte apart, operands and gradients: the results of the same rows side by side."""
    nv = _nv()
    t, h, d, apart = 20, 5, 128, (1 << 28) + 8
    flat = torch.empty(t * apart, dtype=torch.bfloat16, device="cuda")
    view = lambda heads, at: flat.as_strided((t, heads, d), (apart, d, 1), at)
    g = torch.Generator(device="cuda").manual_seed(1)
    near = [torch.randn(t, n, d, generator=g, device="cuda").bfloat16() for n in (h, 2, h, 2)]
    far = [view(n, at) for n, at in ((h, 0), (2, 1024), (h, 4096), (2, 8192))]
    for a, b in zip(far, near):
        a.copy_(b)
    assert (t - 1) * apart > 1 << 32
    w = torch.ones(d, device="cuda")
    cos, sin = (x.cuda() for x in _tables(t, d))
    res = []
    for q, k, gq, gk in (near, far):
        leaves = [x.detach().requires_grad_(True) for x in (q, k, w, w)]
        out = nv.qk_norm_rope(*leaves, cos, sin)
        res.append([*(x.detach() for x in out), *torch.autograd.grad(out, leaves, (gq, gk))])
    assert all(torch.equal(a, b) for a, b in zip(*res))


def test_no_tokens():
    nv = _nv()
    cos, sin = (x.cuda() for x in _tables(10, 128))
    w = torch.ones(128, device="cuda", requires_grad=True)
    x = torch.zeros(0, 4, 128, device="cuda", requires_grad=True)
    q, k = nv.qk_norm_rope(x, x, w, w, cos, sin)
    assert q.shape == (0, 4, 128)
    (q.sum() + k.sum()).backward()
    assert x.grad.shape == x.shape and bool((w.grad == 0).all())


@pytest.mark.parametrize("d", [128, 256])
def test_gradients_are_slopes(d):
    """Along a random direction, the change of sum(g y) between two forward passes.  y is off by 32 2^-24 of its size (24 and
    its rounding), so a difference over 2 h by sum |g| |y| 32 2^-24 / h; the third derivative adds h^2: both sides are taken at h and 2 h, whose
    distance bounds it."""
    nv = _nv()
    g = torch.Generator(device="cuda").manual_seed(2)
    cos, sin = (x.cuda() for x in _tables(40, d))
    ops = [torch.randn(s, generator=g, device="cuda") for s in ((40, 6, d), (40, 2, d), (d,), (d,))]
    way = [torch.randn(x.shape, generator=g, device="cuda") for x in ops]
    gq, gk = (torch.randn(x.shape, generator=g, device="cuda") for x in ops[:2])

    def value(h):
        q, k = nv.qk_norm_rope(*(x + h * y for x, y in zip(ops, way)), cos, sin)
        return float((q.double() * gq).sum() + (k.double() * gk).sum()), float((q.double() * gq).abs().sum() + (k.double() * gk).abs().sum())

    leaves = [x.clone().requires_grad_(True) for x in ops]
    slopes = torch.autograd.grad(nv.qk_norm_rope(*leaves, cos, sin), leaves, (gq, gk))
    got = sum(float((a.double() * b).sum()) for a, b in zip(slopes, way))
    size = sum(float((a.double() * b).abs().sum()) for a, b in zip(slopes, way))
    h = 2.0 ** -9
    one, two = ((value(x)[0] - value(-x)[0]) / (2 * x) for x in (h, 2 * h))
    # the operands x + h y are rounded too: 2^-24 of x, through a slope
    noise = value(0)[1] * 33 * _F / h + size * 4 * _F / h
    assert abs(got - (4 * one - two) / 3) <= abs(one - two) + 2 * noise


def test_the_same_bits_every_time_and_in_a_graph():
    nv = _nv()
    q, k, wq, wk = (x.cuda().requires_grad_(True) for x in _operands((700, 8, 128), (700, 2, 128), torch.bfloat16, torch.float32, 3))
    cos, sin = (x.cuda() for x in _tables(700, 128))
    g = [torch.randn(x.shape, device="cuda").bfloat16() for x in (q, k)]

    def step():
        out = nv.qk_norm_rope(q, k, wq, wk, cos, sin)
        return (*(x.detach() for x in out), *torch.autograd.grad(out, (q, k, wq, wk), g))

    want = step()
    assert all(torch.equal(a, b) for a, b in zip(step(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for x in out:
        x.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    del graph


def test_parts_of_the_graph():
    """One result alone, weights without gradients, hooks, checkpoints; a second derivative is refused."""
    from torch.utils.checkpoint import checkpoint
    nv = _nv()
    q, k, wq, wk = (x.cuda() for x in _operands((9, 4, 128), (9, 2, 128), torch.float32, torch.float32, 3))
    cos, sin = (x.cuda() for x in _tables(9, 128))
    leaves = [x.clone().requires_grad_(True) for x in (q, k, wq, wk)]
    out = nv.qk_norm_rope(*leaves, cos, sin)
    g = [torch.randn_like(x) for x in out]
    want = torch.autograd.grad(out, leaves, g)
    only_q = torch.autograd.grad(nv.qk_norm_rope(*leaves, cos, sin)[0], leaves, g[0], allow_unused=True)
    assert torch.equal(only_q[0], want[0]) and torch.equal(only_q[2], want[2]) and only_q[1] is None and only_q[3] is None
    a, b = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
    assert all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(nv.qk_norm_rope(a, b, wq, wk, cos, sin), (a, b), g), want))
    w = wk.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(nv.qk_norm_rope(q, k, wq, w, cos, sin)[1], w, g[1])[0], want[3])
    again = checkpoint(lambda *x: nv.qk_norm_rope(*x, cos, sin), *leaves, use_reentrant=False)
    assert all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(again, leaves, g), want))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
        kept = nv.qk_norm_rope(*leaves, cos, sin)
    assert all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(kept, leaves, g), want))
    with pytest.raises((RuntimeError, NotImplementedError), match="create_graph"):
        torch.autograd.grad(nv.qk_norm_rope(*leaves, cos, sin), leaves, g, create_graph=True)
    with torch.no_grad():
        assert not nv.qk_norm_rope(*leaves, cos, sin)[0].requires_grad
    import sageattention_b200.nvfp4.custom_ops  # noqa: F401
    f = lambda *x: torch.ops.sageattention_b200.qk_norm_rope(*x, cos, sin, None, 0, 1e-6)
    for fn in (f, torch.compile(f, backend="aot_eager", fullgraph=True)):
        got = fn(*leaves)
        assert all(torch.equal(x, y) for x, y in zip(got, out))
        assert all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(got, leaves, g), want))


def test_arguments_that_are_refused():
    nv = _nv()
    cos, sin = (x.cuda() for x in _tables(9, 128))
    x, w = torch.zeros(9, 4, 128, device="cuda"), torch.ones(128, device="cuda")
    for args, error, match in (((x, x[:8], w, w, cos, sin), AssertionError, "query and key"), ((x, x[None], w, w, cos, sin), ValueError, "query and key"),
                               ((x, x.half(), w, w, cos, sin), TypeError, "dtype"), ((x, x, w[:64], w, cos, sin), AssertionError, "weight"),
                               ((x, x, w.half(), w.half(), cos, sin), TypeError, "weight"), ((x, x, w, w, cos[:, :32], sin), AssertionError, "cos"),
                               ((x, x, w, w, cos.half(), sin), AssertionError, "cos"), ((x, x, w, w, cos[:8], sin[:8]), AssertionError, "within"),
                               ((x[..., :64], x[..., :64], w, w, cos, sin), AssertionError, "128 or 256"),
                               ((x, x, w, w, cos, sin, torch.zeros(8, dtype=torch.int32, device="cuda")), AssertionError, "positions"),
                               ((x, x, w, w, cos, sin, torch.zeros(9, device="cuda")), TypeError, "positions"),
                               ((x, x, w, w, cos, sin, None, -1), AssertionError, "within"), ((x, x, w, w, cos, sin, None, 0, -1e-6), AssertionError, "eps"),
                               ((x, x, w, w.cpu(), cos, sin), RuntimeError, "CUDA"), ((x.cpu(), x, w, w, cos, sin), RuntimeError, "no CPU path"),
                               ((x.double(), x.double(), w, w, cos, sin), TypeError, "dtype")):
        with pytest.raises(error, match=match):
            nv.qk_norm_rope(*args)
    with pytest.raises(NotImplementedError, match="cos"):
        nv.qk_norm_rope(x, x, w, w, cos.clone().requires_grad_(True), sin)
