"""Entries of drafted trees and of the norm with rotation, as far as they go without a GPU: refusals and shapes."""

import os

import pytest
import torch


def _lib():
    from sageattention_b200 import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    return _lib.lib()


def test_c_entries_refuse_what_they_cannot_do():
    L, n = _lib(), None
    bad = lambda rc, text: rc < 0 and text in L.nvfp4_last_error()
    for most in (0, 1025, -5):
        assert bad(L.nvfp4_draft_tree(n, n, n, 5, 1, most, n, n, n), b"max_tokens")
    assert bad(L.nvfp4_draft_tree(n, n, n, 5, 0, 8, n, n, n), b"sizes") and bad(L.nvfp4_draft_tree(n, n, n, -1, 1, 8, n, n, n), b"sizes")
    attention = lambda cu, mask, words, d=128, bs=16, scaling=1.0: L.nvfp4_kv8_tree_attention(
        0, 0, 128, 128, cu, 1, mask, words, 0, 2048, 0, 2048, n, 1, n, 1, 1, bs, n, 1, 1, n, 1, 1, 1, d, scaling, 0, n, 0, 0, n, n)
    assert bad(attention(n, 16, 1), b"cu_seqlens") and bad(attention(16, n, 1), b"tree_mask") and bad(attention(16, 16, 0), b"tree_words")
    assert bad(attention(16, 16, 1, d=64), b"kv8_tree_attention: D") and bad(attention(16, 16, 1, bs=24), b"block_size")
    assert bad(attention(16, 16, 1, scaling=float("inf")), b"scaling") and bad(attention(16, 16, 1), b"workspace too small")
    verify = lambda v=9, dt=2, t=4, r=1, p=0, q=n: L.nvfp4_verify_drafts(p, v, q, v, dt, v, n, 1, n, n, n, t, r, n, n, n, n)
    assert bad(verify(v=0), b"vocabulary") and bad(verify(r=0), b"sizes") and bad(verify(dt=7), b"dtype") and bad(verify(p=2), b"unaligned")
    assert bad(verify(dt=0, q=1), b"unaligned")
    keep = lambda d=128, bs=16, layers=1, hk=1, k=0, kb=2048, kl=0: L.nvfp4_paged_keep_path(
        n, n, n, 4, n, n, 1, 1, 1, k, kl, kb, 0, 0, 2048, n, 0, 1, n, 0, 1, layers, 1, hk, bs, d, n, n)
    assert bad(keep(d=64), b"D must") and bad(keep(bs=8), b"block_size") and bad(keep(k=8), b"aligned") and bad(keep(kb=2056), b"aligned")
    assert bad(keep(kl=4), b"aligned") and bad(keep(layers=-1), b"sizes") and bad(keep(layers=1 << 28), b"layers")
    import ctypes
    three = (ctypes.c_int64 * 3)(0, 128, 128)
    odd = (ctypes.c_int64 * 3)(0, 128, 129)
    norm = lambda d=128, dt=0, wdt=0, z=1, s=1, h=1, eps=1e-6, q=0, st=three, table=0: L.nvfp4_qk_norm_rope(
        q, st, 0, three, dt, z, s, h, 1, d, n, n, wdt, table, 0, 1, n, 0, 0, eps, 0, three, 0, three, n)
    assert bad(norm(d=64), b"D must") and bad(norm(dt=5), b"dtype") and bad(norm(wdt=1), b"weights") and bad(norm(h=0), b"sizes")
    assert bad(norm(eps=-1.0), b"eps") and bad(norm(q=8), b"aligned") and bad(norm(st=odd), b"aligned") and bad(norm(table=4), b"tables")
    assert bad(norm(z=1 << 20, s=1 << 20), b"tokens") and bad(norm(s=1 << 20, h=1 << 14), b"rows") and norm(s=0) == 0
    size = ctypes.c_size_t()
    assert L.nvfp4_qk_norm_rope_bwd_plan(256, 148, ctypes.byref(size)) == 0 and size.value > 0
    assert bad(L.nvfp4_qk_norm_rope_bwd_plan(64, 148, ctypes.byref(size)), b"D must")
    assert bad(L.nvfp4_qk_norm_rope_bwd(0, three, 0, three, 0, three, 0, three, 0, 1, 1, 1, 1, 128, n, n, 0, 0, 0, 1, n, 0, 0, 1e-6, 0, three,
                                        0, three, 16, n, n, 0, n, n), b"workspace")


def test_python_entries_refuse_cpu_tensors():
    import sageattention_b200.nvfp4 as nv
    _lib()
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    c, s, x = torch.zeros(1, 1, 16, 128, dtype=torch.float8_e4m3fn), torch.zeros(1, 1), torch.zeros(1, 1, 128)
    for call in (lambda: nv.draft_tree(i(1), i(2), i(1), 4),
                 lambda: nv.fp8_paged_tree_attention(x, i(2), i(1, 1).long(), c, c, s, s, i(1, 1), i(1), 1.0),
                 lambda: nv.verify_drafts(torch.zeros(1, 5), i(1), i(1), i(2), torch.zeros(1)),
                 lambda: nv.paged_kv_keep_path(i(1), i(1), i(2), i(1), i(1, 1), c, c, s, s),
                 lambda: nv.qk_norm_rope(x, x, torch.ones(128), torch.ones(128), torch.zeros(1, 64), torch.zeros(1, 64))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_custom_ops_infer_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    import sageattention_b200.nvfp4.custom_ops  # noqa: F401  (registers the ops)
    ns = torch.ops.sageattention_b200
    with FakeTensorMode():
        i = lambda *s: torch.empty(*s, dtype=torch.int32)
        mask, pos = ns.draft_tree(i(50), i(4), i(3), 65)
        assert mask.shape == (50, 2) and mask.dtype == torch.int64 and pos.shape == (50,) and pos.dtype == torch.int32
        c, s = torch.empty(20, 2, 16, 128, dtype=torch.float8_e4m3fn), torch.empty(20, 2)
        q = torch.empty(50, 8, 128, dtype=torch.float16)
        out, lse = ns.fp8_paged_tree_attention(q, i(4), mask, c, c, s, s, i(3, 9), i(3), 0.1, 4)
        assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == (50, 8)
        acc, num, nxt = ns.verify_drafts(torch.empty(50, 99), i(50), i(50), i(4), torch.empty(50), None)
        assert acc.shape == (50,) and num.shape == (3,) and nxt.shape == (3,) and nxt.dtype == torch.int64 and acc.dtype == num.dtype == torch.int32
        assert ns.paged_kv_keep_path(acc, num, i(4), i(3), i(3, 9), c, c, s, s).shape == (3,)
        w, t = torch.empty(128, dtype=torch.float16), torch.empty(60, 64)
        a, b = ns.qk_norm_rope(q, q[:, :2], w, w, t, t, i(50), 0, 1e-6)
        assert a.shape == q.shape and b.shape == (50, 2, 128) and a.dtype == q.dtype
        x = torch.empty(2, 30, 4, 128).transpose(1, 2)
        a, _ = ns.qk_norm_rope(x, x, torch.empty(128), torch.empty(128), t, t, None, 0, 1e-6)
        assert a.shape == x.shape and a.stride() == x.stride()


def test_waits_of_the_gradient_kernel_are_bounded_and_reported():
    """Its copies arrive on barriers: every wait is of the whole warp and gives up, and what gave up is told at the end."""
    import re
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sageattention_b200", "csrc")
    text = re.sub(r"//[^\n]*", "", open(os.path.join(csrc, "qknorm.cu")).read())
    start = text.index("qk_norm_rope_bwd_kernel(NormParams p)")
    body = text[start:re.compile(r"^}", re.M).search(text, start).start()]
    assert set(re.findall(r"\bmbar_\w*wait\w*", body)) == {"mbar_wait_warp"} and len(re.findall(r"&expired, \d+\)", body)) == 1
    assert re.search(r"__syncthreads\(\);\s*report_error\(&expired, p\.status\);\s*$", body)
    # copies into a stage are asked for when all lanes have read it
    assert body.rindex("__syncwarp();") < body.index("if (p.part != nullptr)")
