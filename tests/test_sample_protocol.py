"""What the CTAs of a row tell one another in csrc/sample.cu, on the host: how full the lists are. After a join of the cluster every warp of every CTA adds up all CTAs'
counts; CTA 0 then narrows its list without another join. In random order no warp may come out at another sum than the rest, whichever count the narrowing keeps: the
one that the source names is run, and a warp that goes on into a round which the others leave out would wait there for good."""
import os
import random
import re

import pytest

SOURCE = os.path.join(os.path.dirname(__file__), "..", "llamd_rs_b200", "csrc", "sample.cu")
LIST, RANKED = 1024, 256


def narrowing():
    """CTA 0's own part between the lists' joins: from where it pulls the others' lists to the next join."""
    text = re.sub(r"//[^\n]*", "", open(SOURCE).read())
    begin = text.index("pull();", text.index("while (n > kList)"))
    return text[begin:text.index("cluster.sync();", begin)]


def written(part):
    """The fields of the CTA's shared memory that this part of the kernel writes."""
    by_name = re.findall(r"\bsh\.(\w+)(?:\[[^\]]*\])?(?:\s*=\s*sh\.\w+(?:\[[^\]]*\])?)*\s*=(?!=)", part)
    chained = re.findall(r"=\s*sh\.(\w+)(?:\[[^\]]*\])?\s*=(?!=)", part)
    return set(by_name) | set(chained) | set(re.findall(r"atomic\w+\(&sh\.(\w+)", part))


def read_by_others():
    """The fields that CTAs read of one another behind the join in front of the narrowing: by in_all_lists."""
    text = open(SOURCE).read()
    begin = text.index("auto in_all_lists")
    return set(re.findall(r"\)->(\w+)", text[begin:text.index("};", begin)]))


class Row:
    """The lists' counts of a row's CTAs, and their warps from the join on: each reads all CTAs' counts, one after the other; CTA 0's go on to narrow its list."""

    def __init__(self, rng, ctas, warps, shared_count):
        self.rng, self.shared_count = rng, shared_count
        total = rng.randint(RANKED + 1, LIST)
        cuts = sorted(rng.randint(0, total) for _ in range(ctas - 1))
        self.n_list = [b - a for a, b in zip([0] + cuts, cuts + [total])]
        self.total, self.sums = total, {}
        self.pulled = 0  # warps of CTA 0 that have come to the CTA's own barrier
        self.warps = warps
        self.steps = [self.other(c, w) for c in range(1, ctas) for w in range(warps)] + [self.first(w) for w in range(warps)]

    def counts(self, who):
        n = 0
        for c in range(len(self.n_list)):
            n += self.n_list[c]
            yield
        self.sums[who] = n

    def other(self, c, w):
        yield from self.counts((c, w))

    def first(self, w):
        yield from self.counts((0, w))
        self.pulled += 1
        while self.pulled < self.warps:
            yield
        if w:
            return
        left = self.total
        while left > RANKED:  # a bin of what is left
            narrowed = max(1, left - self.rng.randint(1, left - 1))
            if self.shared_count:
                self.n_list[0] = 0
            for _ in range(narrowed):
                if self.shared_count:
                    self.n_list[0] += 1
                yield
            left = narrowed

    def run(self):
        live = [(step, 10.0 ** self.rng.uniform(-3, 0)) for step in self.steps]  # (some warps are late)
        while live:
            i = self.rng.choices(range(len(live)), [speed for _, speed in live])[0]
            try:
                next(live[i][0])
            except StopIteration:
                del live[i]
        return set(self.sums.values()) == {self.total}


@pytest.mark.parametrize("ctas", [2, 4, 8])
def test_counts_are_everybodys(ctas):
    shared = bool(written(narrowing()) & read_by_others())
    for seed in range(60):
        assert Row(random.Random(seed), ctas, 4, shared).run(), "a warp has read a count that the narrowing wrote"


def test_the_model_meets_the_mistake():
    """With one count for both a late warp reads the wrong one, and sums beyond a list's room are among them."""
    rows = [Row(random.Random(seed), 4, 4, True) for seed in range(400)]
    assert not all([row.run() for row in rows])
    assert any(n > LIST for row in rows for n in row.sums.values())


def test_fields_are_found():
    """The narrowing writes what it is known to write, and the reader of the source finds it."""
    assert {"hist", "bin", "before", "list"} <= written(narrowing())
    assert read_by_others() == {"n_list"}
    assert written("if (a) sh.x = sh.y[3] = 0; sh.z[i] = 1; b = sh.w == 2; atomicAdd(&sh.v, 1);") == {"x", "y", "z", "v"}
