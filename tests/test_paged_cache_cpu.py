"""Paged 8-bit KV cache without a GPU: refusals of the C ABI and of the Python entries, and the rules the GPU tests compare
with (scales, rounding, tables)."""

import ctypes
import math
import os

import pytest
import torch

from paged_reference import nearest_e4m3, reserve, scale_of, trim, write


def _lib():
    from sageattention_b200 import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    return _lib.lib()


def test_rounding_of_the_reference_is_that_of_the_type():
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    every = every[torch.isfinite(every)].double()
    assert torch.equal(nearest_e4m3(every), every)
    x = torch.cat([every, (every[1:] + every[:-1]) / 2, torch.randn(4096, dtype=torch.float64) * 2.0 ** torch.randint(-9, 8, (4096,))])
    x = x.float().clamp(-448, 448)
    assert torch.equal(nearest_e4m3(x.double()).float(), x.to(torch.float8_e4m3fn).float())


def test_scales_are_the_smallest_powers_of_two():
    for amax in (1.0, 448.0, 448.5, 1.75, 1.7500001, 3e38, 1e-20, 0.0, 7.0 * 2.0 ** -30):
        s = scale_of(torch.tensor([amax], dtype=torch.float64))[0].item()
        assert math.frexp(s)[0] == 0.5 and (448 * s >= amax)
        assert s == 2.0 ** -110 or 448 * s / 2 < amax


def test_a_trim_undoes_a_reservation():
    g = torch.Generator().manual_seed(0)
    for _ in range(50):
        rows, block = int(torch.randint(1, 9, (1,), generator=g)), 16
        held = torch.randint(0, 80, (rows,), generator=g)
        new = torch.randint(0, 50, (rows,), generator=g)
        state = dict(lengths=held.clone(), table=torch.full((rows, 10), -1), free=torch.randperm(90, generator=g), count=90)
        empty = dict(state, lengths=torch.zeros_like(held))
        reserve(held, empty, 10 ** 6, block)
        before = {k: (v.clone() if torch.is_tensor(v) else v) for k, v in empty.items()}
        _, _, _, short = reserve(new, empty, 10 ** 6, block)
        assert short == 0
        trim(held, empty, block)
        assert all(torch.equal(before[k], empty[k]) if torch.is_tensor(before[k]) else before[k] == empty[k] for k in before)


def test_blocks_written_token_by_token_stay_near_the_one_shot_block():
    """A code that is rounded again when the scale grows is off by half a step of each rounding; only codes below
    2^-6 of the scale move at all."""
    x = torch.randn(16, 2, 128, generator=torch.Generator().manual_seed(3)).double()
    x *= torch.exp2(torch.arange(16).double() - 8)[:, None, None]
    one, one_s = torch.zeros(1, 2, 16, 128).double(), torch.zeros(1, 2).double()
    write(x, torch.arange(16), one, one_s, 16)
    many, many_s = torch.zeros(1, 2, 16, 128).double(), torch.zeros(1, 2).double()
    for t in range(16):
        write(x[t:t + 1], torch.tensor([t]), many, many_s, 16)
    assert torch.equal(one_s, many_s)
    diff = (one - many).abs()
    assert diff.max() <= 2.0 ** -9              # one step of the codes that move
    assert torch.equal(one[one.abs() >= 2.0 ** -5], many[one.abs() >= 2.0 ** -5])


def test_c_entries_refuse_bad_sizes():
    L = _lib()
    n = None
    assert L.nvfp4_paged_reserve(n, n, n, 1, n, n, 1, 1, 1, 24, 1, n, n, n, n, n, n) < 0 and b"block_size" in L.nvfp4_last_error()
    assert L.nvfp4_paged_reserve(n, n, n, 1, n, n, 0, 1, 1, 16, 1, n, n, n, n, n, n) < 0 and b"sizes" in L.nvfp4_last_error()
    assert L.nvfp4_paged_reserve(n, n, n, 1, n, n, 1, 1, 1, 16, -1, n, n, n, n, n, n) < 0 and b"slot" in L.nvfp4_last_error()
    assert L.nvfp4_paged_trim(n, n, n, 1, n, n, 1, 1, 1, 8, n, n) < 0 and b"block_size" in L.nvfp4_last_error()
    assert L.nvfp4_paged_trim(n, n, n, 1, n, n, 1 << 20, 1 << 20, 1, 16, n, n) < 0 and b"entries" in L.nvfp4_last_error()
    w = lambda **k: L.nvfp4_kv8_write(k.get("key", 0), 0, k.get("dt", 0), k.get("t", 1), 1, k.get("d", 128), k.get("st", 128), 128, 128,
                                      128, n, 0, 2048, 0, 2048, n, 1, n, 1, 1, k.get("bs", 16), n)
    for bad, text in ((dict(bs=17), b"block_size"), (dict(d=64), b"D must"), (dict(st=129), b"aligned"), (dict(key=2), b"aligned"),
                      (dict(t=-1), b"sizes"), (dict(dt=7), b"dtype")):
        assert w(**bad) < 0 and text in L.nvfp4_last_error(), bad
    assert w(t=0) == 0
    size = ctypes.c_size_t()
    plan = lambda dt, t, r, g, d: L.nvfp4_kv8_attention_plan(dt, t, r, g, d, 148, ctypes.byref(size))
    assert plan(0, 1, 1, 1, 96) < 0 and plan(0, 1, 0, 1, 128) < 0
    assert plan(0, 7, 7, 16, 128) == 0 and size.value == 2 * 148 * (2 * 16 * 130 * 4 + 16)
    assert plan(1, 80, 7, 4, 256) == 0 and size.value == 148 * (2 * 128 * 258 * 4 + 16)
    assert plan(2, 80, 7, 4, 256) == 0 and size.value == 2 * 148 * (2 * 16 * 258 * 4 + 16)
    a = lambda **k: L.nvfp4_kv8_attention(0, 0, 128, 128, k.get("cu", n), k.get("t", 1), k.get("kc", 0), 2048, 0, 2048, n, 1, n, 1, 1,
                                          k.get("bs", 16), n, 1, k.get("w", 1), n, 1, 1, k.get("g", 1), k.get("d", 128), 1.0, 0, n, 0,
                                          k.get("ws", 0), n, n)
    for bad, text in ((dict(bs=48), b"block_size"), (dict(d=80), b"D must"), (dict(t=2), b"cu_seqlens"), (dict(kc=8), b"aligned"),
                      (dict(g=0), b"sizes"), (dict(w=1 << 28), b"sizes"), (dict(t=-1, cu=16), b"sizes")):
        assert a(**bad) < 0 and text in L.nvfp4_last_error(), bad
    assert a(t=0, cu=16) == 0


def test_scaling_has_to_be_finite():
    L, n = _lib(), None
    for scaling in (math.inf, -math.inf, math.nan):
        assert L.nvfp4_kv8_attention(0, 0, 128, 128, 16, 0, 0, 2048, 0, 2048, n, 1, n, 1, 1, 16, n, 1, 1, n, 1, 1, 1, 128, scaling, 0, n, 0,
                                     0, n, n) < 0 and b"scaling" in L.nvfp4_last_error()


def test_python_entries_refuse_cpu_tensors():
    import sageattention_b200.nvfp4 as nv
    _lib()
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        nv.paged_kv_reserve(i(1), i(1), i(1, 1), i(1), i(1), 1, 16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        nv.paged_kv_trim(i(1), i(1), i(1, 1), i(1), i(1), 16)
    x = torch.zeros(1, 1, 128)
    c, s = torch.zeros(1, 1, 16, 128, dtype=torch.float8_e4m3fn), torch.zeros(1, 1)
    with pytest.raises(RuntimeError, match="no CPU path"):
        nv.fp8_kv_write(x, x, torch.zeros(1, dtype=torch.int64), c, c, s, s)
    with pytest.raises(RuntimeError, match="no CPU path"):
        nv.fp8_paged_decode(x[:, :, None], c, c, s, s, i(1, 1), i(1), 1.0)
    with pytest.raises(ValueError, match="cu_seqlens"):
        nv.fp8_paged_attention(x, None, c, c, s, s, i(1, 1), i(1), 1.0)
    with pytest.raises(AssertionError, match="block_size"):
        nv.FP8PagedKVCache(1, 4, 1, 128, 1, 64, "cpu", block_size=24)
    cache = nv.FP8PagedKVCache(2, 5, 3, 128, 2, 65, "cpu", block_size=32)
    assert cache.block_table.shape == (2, 3) and int(cache.free_count) == 5 and cache.free_blocks.tolist() == [4, 3, 2, 1, 0]
    assert cache.cache_bytes() == sum(t.numel() * t.element_size() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale))


def test_custom_ops_infer_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    import sageattention_b200.nvfp4.custom_ops  # noqa: F401  (registers the ops)
    ns = torch.ops.sageattention_b200
    with FakeTensorMode():
        i = lambda *s: torch.empty(*s, dtype=torch.int32)
        slots, pos, cu, short = ns.paged_kv_reserve(i(3), i(3), i(3, 9), i(20), i(1), 50, 16)
        assert slots.shape == (50,) and slots.dtype == torch.int64 and pos.shape == (50,) and cu.shape == (4,) and short.shape == (1,)
        assert {pos.dtype, cu.dtype, short.dtype} == {torch.int32}
        assert ns.paged_kv_trim(i(3), i(3), i(3, 9), i(20), i(1), 16) is None
        c, s = torch.empty(20, 2, 16, 128, dtype=torch.float8_e4m3fn), torch.empty(20, 2)
        x = torch.empty(50, 2, 128, dtype=torch.bfloat16)
        assert ns.fp8_kv_write(x, x, slots, c, c, s, s) is None
        q = torch.empty(3, 8, 1, 128, dtype=torch.bfloat16)
        out, lse = ns.fp8_paged_decode(q, c, c, s, s, i(3, 9), i(3), 0.1, 4)
        assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == (3, 8) and lse.dtype == torch.float32
        q = torch.empty(50, 8, 128, dtype=torch.float16)
        out, lse = ns.fp8_paged_attention(q, cu, c, c, s, s, i(3, 9), i(3), 0.1, 4)
        assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == (50, 8)


def _ends(segments, stages=2, per_tile=2):
    """The roles of the many-row kernel at D 128 as lists of (what is waited for, what is told); True if all come to their end.
    Segments are (tiles, rows above 128).  One converting group does K and V of tile after tile in two places; group g of two
    has every tile, or every other one; products are issued one after the other."""
    convert, issue, soft, done, jobs_of = [], [], [[], []], set(), []
    n = 0
    for at, (tiles, both) in enumerate(segments):
        jobs = [(tiles if both else (tiles + 1 - g) // 2) * per_tile for g in (0, 1)]
        steps = [(kind, g, j + ahead) for j in range(-2, max(jobs) + 1)
                 for kind, g, ahead in ((("pv", 0, 0), ("s", 0, 2), ("pv", 1, 0), ("s", 1, 2)) if both else
                                        (("pv", 0, 0), ("pv", 1, -1), ("s", 0, 2), ("s", 1, 1)))]
        for kind, g, j in steps:
            if 0 <= j < jobs[g]:
                tile = n + j // per_tile * (1 if both else 2) + (0 if both else g)
                told = [(kind, at, g, j)]
                if j % per_tile == per_tile - 1 and (not both or g == 1):
                    told.append((kind + " of", tile))
                issue.append(([("k", tile)] if kind == "s" else [("v", tile), ("p", at, g, j)], *told))
        for g in (0, 1):
            soft[g] += [([("s", at, g, j)], ("p", at, g, j)) for j in range(jobs[g])]
        jobs_of.append(jobs)
        n += tiles
    for t in range(n + 1):                                 # K of a tile, then V of the one before
        convert += [([("s of", t - stages)] if t >= stages else [], ("k", t))] if t < n else []
        convert += [([("pv of", t - 1 - stages)] if t > stages else [], ("v", t - 1))] if t else []
    assert len(issue) == 2 * sum(map(sum, jobs_of))
    roles = [convert, issue, *soft]
    moved = True
    while moved:
        moved = False
        for role in roles:
            while role and all(w in done for w in role[0][0]):
                done.update(role.pop(0)[1:])
                moved = True
    return not any(roles)


def test_no_role_of_the_many_row_kernel_waits_for_itself():
    gen = torch.Generator().manual_seed(0)
    for tiles in range(1, 40):
        assert _ends([(tiles, False)]) and _ends([(tiles, True)])
    for _ in range(300):
        size = torch.randint(1, 25, (5,), generator=gen).tolist()
        rows = (torch.rand(5, generator=gen) < 0.5).tolist()
        assert _ends(list(zip(size, rows)))
