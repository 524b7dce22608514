"""Rules of the paged 8-bit KV cache that its sources show and no run does."""

import os
import random
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


def _all_end(segments, d):
    """All roles of the many-row kernel at head dim d as lists of (what is waited for, what is told); True if they come to their end.

    Segments are (tiles, rows above 128).  Besides codes, scores, weights and products (as the kernel issues them) these are the
    waits for a segment's query rows, for their place, for its result and for the result before it to have been read."""
    both_groups = d == 128
    stages, per_tile = (2, 2) if both_groups else (1, 1)
    groups = (0, 1) if both_groups else (0,)
    issue, load, soft, done, n = [], [], {g: [] for g in groups}, set(), 0
    last_result = {g: None for g in groups}
    for seg, (tiles, above) in enumerate(segments):
        both = both_groups and above
        turns = both_groups and not both
        jobs = {g: (tiles if not turns else (tiles + 1 - g) // 2) * per_tile for g in groups}
        steps = []
        for j in range(-2, jobs[0] + (1 if turns else 0)):
            steps += ([("pv", 0, j), ("pv", 1, j - 1), ("s", 0, j + 2), ("s", 1, j + 1)] if turns else
                      [x for g in groups for x in (("pv", g, j), ("s", g, j + 2))])
        steps = [(kind, g, j) for kind, g, j in steps if 0 <= j < jobs[g]]
        assert len(steps) == 2 * sum(jobs.values())
        last_s = max(i for i, x in enumerate(steps) if x[0] == "s")
        load.append(([("q free", seg - 1, g) for g in groups] + [("s last", seg - 1)] if seg else [], [("q", seg)]))
        issue.append(([("q", seg)], []))
        for i, (kind, g, j) in enumerate(steps):
            tile = n + (j // per_tile if not turns else j // per_tile * 2 + g)
            told = [(kind, seg, g, j)] + ([("s last", seg)] if i == last_s else [])
            if j % per_tile == per_tile - 1 and (not both or g == 1):
                told.append((kind + " of", tile))
            if kind == "pv" and j == jobs[g] - 1:
                told.append(("o", seg, g))
            wait = [("k", tile)] if kind == "s" else [("v", tile), ("p", seg, g, j)]
            if kind == "pv" and j == 0 and last_result[g] is not None:
                wait.append(("o free", last_result[g], g))
            issue.append((wait, told))
        for g in groups:
            soft[g].append(([("q", seg)], [] if turns else [("q free", seg, g)]))
            for j in range(jobs[g]):
                # a reference that moves waits for the product before
                soft[g].append(([("s", seg, g, j)] + ([("pv", seg, g, j - 1)] if j else []), [("p", seg, g, j)]))
            soft[g].append(([("o", seg, g)] if jobs[g] else [], [("met", seg, g)]))
            soft[g].append(([("met", seg, x) for x in groups] if turns else [],
                            ([("o free", seg, g)] if jobs[g] else []) + ([("q free", seg, g)] if turns else [])))
            if jobs[g]:
                last_result[g] = seg
        n += tiles
    place = lambda what, t: [(what, t - stages)] if t >= stages else []
    if both_groups:                                        # one converting group: K of a tile, then V of the one before
        convert = [[x for t in range(n + 1) for x in ([(place("s of", t), [("k", t)])] if t < n else []) +
                    ([(place("pv of", t - 1), [("v", t - 1)])] if t else [])]]
    else:                                                  # one each
        convert = [[(place("s of", t), [("k", t)]) for t in range(n)], [(place("pv of", t), [("v", t)]) for t in range(n)]]
    roles = [issue, load, *soft.values(), *convert]
    moved = True
    while moved:
        moved = False
        for role in roles:
            while role and all(w in done for w in role[0][0]):
                done.update(role.pop(0)[1])
                moved = True
    return not any(roles)


def test_no_role_of_the_many_row_kernel_waits_for_itself_at_either_head_dim():
    gen = random.Random(0)
    for d in (128, 256):
        for tiles in range(1, 40):
            for above in (False, True):
                assert _all_end([(tiles, above)], d), (d, tiles, above)
        for _ in range(300):
            segments = [(gen.choice([1, 1, 2, 3, gen.randint(1, 25)]), gen.random() < 0.5) for _ in range(6)]
            assert _all_end(segments, d), (d, segments)
