"""The demo's steps of drafted trees: it runs, and what it generates is what its own model chooses."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_trees_of_earlier_text():
    from sageattention_b200.nvfp4.demo_decode import lookup_tree
    assert lookup_tree([5]) == ([5], [-1])
    assert lookup_tree([1, 2, 3, 1]) == ([1, 2, 3, 1], [-1, 0, 1, 2])
    # two occurrences that go the same way for one token: 7 9 .. and 7 8 .., the latest first
    assert lookup_tree([4, 7, 8, 4, 7, 9, 4], branches=2, depth=2) == ([4, 7, 9, 8], [-1, 0, 1, 1])


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_generation_with_trees(temperature):
    from sageattention_b200.nvfp4 import demo_decode as D
    model = D.TinyGQADecoder(2, 256, 4, 2, 128, 64, torch.bfloat16, "cuda")
    prompt = torch.randint(0, 64, (3, 90), generator=torch.Generator().manual_seed(1)).cuda()
    first, kv = D.prefill(model, prompt)
    toks, steps, _, cache = D.generate_trees(model, prompt, kv, first, 40, 160, temperature)
    assert toks.shape == (3, 41) and 1 <= steps <= 40 and bool(((toks >= 0) & (toks < 64)).all())
    # the cache holds the prompt and what was kept but the last token
    held = cache.lengths.tolist()
    assert all(90 + 40 <= n <= 90 + 40 + 5 for n in held)
    blocks = [-(-n // 64) for n in held]
    assert int(cache.free_count) == cache.num_blocks - sum(blocks)
    assert [int((row >= 0).sum()) for row in cache.block_table] == blocks
    if temperature == 0.0:
        again, steps_again, _, _ = D.generate_trees(model, prompt, kv, first, 40, 160)
        assert torch.equal(toks, again) and steps == steps_again


def test_the_demo_reports_its_trees():
    from sageattention_b200.nvfp4 import demo_decode as D
    rep = D.main(["--layers", "2", "--hidden", "256", "--heads", "4", "--kv-heads", "2", "--vocab", "64", "--batch", "2", "--prompt", "70",
                  "--new", "12", "--window", "32"])
    assert set(rep["tree"]) == {"agreement", "ms_per_step", "steps", "tokens_per_step", "bytes"} and rep["tree"]["steps"] <= 12
