"""The limit of a tree's nodes in the verification, as far as it goes without a GPU."""

import os

import pytest
import torch


def test_c_entry_refuses_limits_out_of_range():
    from sageattention_b200 import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    L, n = _lib.lib(), None
    call = lambda most, v=9: L.nvfp4_verify_drafts_within(0, v, n, v, 2, v, n, 1, n, n, n, 4, 1, most, n, n, n, n)
    for most in (0, 1025, -5):
        assert call(most) < 0 and b"max_tokens" in L.nvfp4_last_error()
    assert call(1024, v=0) < 0 and b"vocabulary" in L.nvfp4_last_error()


def test_registered_operator_takes_it_or_not():
    from torch._subclasses.fake_tensor import FakeTensorMode

    import sageattention_b200.nvfp4.custom_ops  # noqa: F401
    ns = torch.ops.sageattention_b200
    with FakeTensorMode():
        i = lambda *s: torch.empty(*s, dtype=torch.int32)
        args = (torch.empty(50, 99), i(50), i(50), i(4), torch.empty(50), None)
        for more in ((), (64,)):
            assert [x.shape for x in ns.verify_drafts(*args, *more)] == [(50,), (3,), (3,)]
