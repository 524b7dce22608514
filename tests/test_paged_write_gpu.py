"""Writes into the paged 8-bit KV cache that are long enough for its wide windows: every type, head dim and block size, codes and
scales exactly those of the 64-bit reference."""

import pytest
import torch

from test_paged_cache_gpu import _check_write, _rows, _runs

pytestmark = pytest.mark.gpu


def _window_operands(tokens, hk):
    """Of 64 tokens; in units of an SM.  From two on the windows are wide, from sixteen on a block of threads has two operands."""
    return -(-tokens // 64) * 2 * hk / torch.cuda.get_device_properties(0).multi_processor_count


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_wide_windows(block, d, dtype):
    """Long and short runs that begin anywhere in a block and in a window, in blocks whose older scales are smaller or larger."""
    lens = [330, 1, 128, 5, 64, 127, 300, 17, 1, 1, 255, 63, 130]
    starts = [37, 15, 0, 127, 64, 1, 100, 31, 5, 63, 16, 65, 126]
    slots = _runs(lens, starts, block, 3, 150)
    hk = 8
    assert 2 <= _window_operands(len(slots), hk) < 16
    key, value = _rows((len(slots), hk, d), 5, dtype).cuda(), _rows((len(slots), hk, d), 6, dtype).cuda()
    _check_write(key, value, slots, block, d, hk, 150, between=16)


@pytest.mark.parametrize("d,block,dtype", [(128, 64, torch.bfloat16), (128, 128, torch.float16), (256, 32, torch.bfloat16), (256, 128, torch.float32),
                                           (128, 16, torch.float32)])
def test_two_operands_a_block_of_threads(d, block, dtype):
    """The second operand's values, maxima and scales go where the first one's were."""
    lens = [1400, 3, 900, 1, 1000, 130, 1500]
    starts = [37, 15, 0, 127, 64, 1, 100]
    blocks = sum(-(-(n + s) // block) for n, s in zip(lens, starts)) + 3
    slots = _runs(lens, starts, block, 4, blocks)
    hk = 16
    assert _window_operands(len(slots), hk) >= 16
    key, value = _rows((len(slots), hk, d), 7, dtype).cuda(), _rows((len(slots), hk, d), 8, dtype).cuda()
    _check_write(key, value, slots, block, d, hk, blocks)


@pytest.mark.parametrize("offset", [0, 1, 63, 64, 100, 126, 127])
def test_runs_that_begin_at_every_end_of_a_window_of_128(offset):
    """Tokens in front (of no slot) move the runs of 128-token blocks through the window; what is behind a run is another run's, or nobody's."""
    hk, d, block = 8, 128, 128
    slots = [-1] * offset + _runs([128, 128, 1, 129, 1, 127, 300, 700], [0, 0, 127, 127, 5, 1, 64, 3], block, 6, 20)
    assert 2 <= _window_operands(len(slots), hk) < 16
    key, value = _rows((len(slots), hk, d), 9, torch.bfloat16).cuda(), _rows((len(slots), hk, d), 10, torch.bfloat16).cuda()
    _check_write(key, value, slots, block, d, hk, 20)
