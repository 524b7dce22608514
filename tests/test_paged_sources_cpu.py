"""Rules of the paged 8-bit KV cache that its sources show and no run does."""

import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sageattention_b200", "csrc")


def test_every_slot_that_is_looked_at_has_been_fetched():
    """The quantising write looks at the slot map as far as a run can reach, and at nothing that no thread has fetched."""
    text = open(os.path.join(CSRC, "paged.cu")).read()
    names = {n: int(re.search(rf"constexpr int {n} = (\d+);", text).group(1)) for n in ("kWriteThreads", "kMaxBlock")}
    windows = {int(w) for w in re.findall(r"launch_window<T, D, (\d+),", text)}
    assert windows == {16, 64, 128}
    for w in windows:
        span = eval(re.search(r"constexpr int kSpan = ([^;]+);", text).group(1), {}, dict(names, W=w))
        fetched = {t for t in range(names["kWriteThreads"]) if t <= span}              # slot of token t0 - 1 + t
        looked_at = {t + i for t in range(names["kWriteThreads"]) if t < span for i in (0, 1)}
        assert looked_at <= fetched, w
        # a run begins in the window's last token at the latest, and is a cache block at most
        assert span >= w - 1 + names["kMaxBlock"]


def test_every_function_of_the_headers_is_called():
    text = {f: open(os.path.join(root, f)).read() for root, _, files in os.walk(CSRC) for f in files if f.endswith((".cu", ".cuh"))}
    for header in ("kv8.cuh", "paged.cuh"):
        for name in re.findall(r"__forceinline__ [\w:<>* ]+? \*?(\w+)\(", text[header]):
            assert sum(len(re.findall(rf"\b{name}\b", re.sub(r"//[^\n]*", "", t))) for t in text.values()) > 1, name
