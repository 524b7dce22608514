"""The gradient kernel of the norm with rotation asks for copies into a stage when all lanes have read it."""

import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sageattention_b200", "csrc")


def _kernel():
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, "qknorm.cu")).read())
    start = text.index("qk_norm_rope_bwd_kernel(NormParams p)")
    return text[start:re.compile(r"^}", re.M).search(text, start).start()]


def _loop(body):
    """Statements of the loop over tasks, from its head to its closing brace."""
    head = body.index("for (uint32_t i = first; i < o.tasks; i += warps, ++n) {")
    depth, at = 0, body.index("{", head)
    for end in range(at, len(body)):
        depth += {"{": 1, "}": -1}.get(body[end], 0)
        if depth == 0:
            return body[at + 1:end]
    raise AssertionError("the loop does not end")


def _held(body):
    """Its last statement brings the warp together, behind all that reads the stage, and it asks for more only at its beginning."""
    loop = _loop(body)
    reads = max(loop.rindex(x) for x in (".load(row", "inside_s[warp][stage]", "place_s[warp][stage]", "cos.load(", "sin.load("))
    ends = re.search(r"\}\s*__syncwarp\(\);\s*$", loop)
    return ends is not None and reads < ends.start() and re.match(r"\s*ask\(\);", loop) is not None and loop.count("ask()") == 1


def test_a_stage_is_filled_again_when_all_lanes_have_read_it():
    body = _kernel()
    assert _held(body)
    loop = _loop(body)
    at = loop.rindex("__syncwarp();")
    assert not _held(body.replace(loop, loop[:at]))                            # without it the check fails
    assert not _held(body.replace(loop, loop[:at] + loop[at:] + "ask();"))
