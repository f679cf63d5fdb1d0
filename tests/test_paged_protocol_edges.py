"""The prompt attention's barriers (csrc/paged_prompt.cu) as test_paged_protocol.py has them, with what that model leaves out: weights that come in two
parts, loads that land some time after they are issued, the last block's V rows that the softmax clears in the loader's ring, the wait for every product
before the block ends, and blocks that give up at any wait."""
import random

import pytest

from test_paged_protocol import Model, Wrong


class GaveUp(Exception):
    pass


class Whole(Model):
    """pieces: (blocks of tile 0, of tile 1, whether the last block is ragged). fails: how likely a wait that is not met at once runs out."""

    def __init__(self, pieces, stages, queries, rng, fails=0.0):
        super().__init__([p[:2] for p in pieces], stages, queries, rng)
        self.ragged = [p[2] for p in pieces]
        self.fails, self.abort = fails, False
        self.flying, self.holds, self.cleared = [], {}, set()  # loads on their way; stage -> slot that lies there; (tile, slot)
        self.ended = 0

    def wait(self, bar, phase, bounded=True):
        while (self.phases.get(bar, 0) & 1) == (phase & 1):
            if bounded and (self.abort or self.rng.random() < self.fails):
                self.abort = True
                raise GaveUp
            yield bar, phase
        if not self.abort and self.phases.get(bar, 0) != phase + 1:
            raise Wrong(f"{bar}: phase {phase} taken for over at {self.phases.get(bar, 0)} completed")

    def tma(self):
        while True:
            if self.flying and self.rng.random() < 0.4:
                bar, slot = self.flying.pop(self.rng.randrange(len(self.flying)))
                if bar[0] == "full":
                    self.holds[bar[1]] = slot
                self.arrive(bar)
            yield len(self.flying)

    def tensor_pipe(self):
        while True:
            if self.pipe and self.rng.random() < 0.4:
                what, x = self.pipe.pop(0)
                if what == "product":
                    t, slot, ragged = x
                    if not self.abort and self.holds.get(slot % self.stages) != slot:
                        raise Wrong(f"a product of block {slot} finds {self.holds.get(slot % self.stages)}")
                    if not self.abort and ragged and (t, slot) not in self.cleared:
                        raise Wrong("a product of rows that are not cleared")
                    self.done[t] += 1
                else:
                    self.arrive((what, x))
            yield len(self.pipe)

    def load(self):
        slot = n_q = 0
        try:
            for blocks in self.pieces:
                for j in range(max(blocks)):
                    for kv in range(2):
                        if slot // self.stages:
                            yield from self.wait(("empty", slot % self.stages), slot // self.stages - 1)
                        self.flying.append((("full", slot % self.stages), slot))
                        slot += 1
                        if kv or j:
                            continue
                        for t in range(2):
                            if blocks[t]:
                                if n_q // self.queries:
                                    yield from self.wait(("q_empty", n_q % self.queries), n_q // self.queries - 1)
                                self.flying.append((("q_full", n_q % self.queries), n_q))
                                n_q += 1
        except GaveUp:
            pass
        self.ended += 1
        while self.ended < 4:  # (the block's barrier)
            yield self.ended
        if self.abort:
            for i in range(max(0, slot - self.stages), slot):
                yield from self.wait(("full", i % self.stages), i // self.stages, bounded=False)
            for i in range(max(0, n_q - self.queries), n_q):
                yield from self.wait(("q_full", i % self.queries), i // self.queries, bounded=False)
        if self.flying:
            raise Wrong("a load lands after the block has ended")

    def products(self):
        try:
            yield from self.all_products()
        except GaveUp:
            pass
        self.pipe.append(("drain", 0))
        yield from self.wait(("drain", 0), 0, bounded=False)
        if self.pipe:
            raise Wrong("a product, or its commit's arrival, after the block has ended")
        self.ended += 1

    def all_products(self):
        k, v, n_q, buf, n_s, n_o = 0, 1, 0, [0, 0], [0, 0], [0, 0]
        commit = lambda what, x: self.pipe.append((what, x))  # noqa: E731

        def begin(t, blocks):
            nonlocal n_q
            yield from self.wait(("full", k % self.stages), k // self.stages)
            yield from self.wait(("q_full", n_q % self.queries), n_q // self.queries)
            buf[t] = n_q % self.queries
            n_q += 1
            commit("s", t)
            if blocks == 1:
                commit("q_empty", buf[t])

        now = self.pieces[0]
        for t in range(2):
            if now[t]:
                yield from begin(t, now[t])
        if sum(now):
            commit("empty", k % self.stages)
        for n in range(len(self.pieces)):
            after = self.pieces[n + 1] if n + 1 < len(self.pieces) else (0, 0)
            most, begun = max(now), [False, False]
            for j in range(most):
                k += 2
                yield from self.wait(("full", v % self.stages), v // self.stages)
                if j + 1 < most:
                    yield from self.wait(("full", k % self.stages), k // self.stages)
                for t in range(2):
                    if j >= now[t]:
                        continue
                    if not j and n_o[t]:
                        yield from self.wait(("o_empty", t), n_o[t] - 1)
                    for part in range(2):
                        yield from self.wait((f"p{part}", t), n_s[t])
                        commit("product", (t, v, self.ragged[n] and j + 1 == most))
                    n_s[t] += 1
                    if j + 1 < now[t]:
                        commit("s", t)
                        if j + 2 == now[t]:
                            commit("q_empty", buf[t])
                    else:
                        commit("o_full", t)
                        n_o[t] += 1
                        if after[t] and j + 1 == most and (t == 0 or not after[0] or begun[0]):
                            yield from begin(t, after[t])
                            begun[t] = True
                commit("empty", v % self.stages)
                if j + 1 < most:
                    commit("empty", k % self.stages)
                v += 2
            for t in range(2):
                if after[t] and not begun[t]:
                    yield from begin(t, after[t])
            if sum(after):
                commit("empty", k % self.stages)
            now = after

    def clear(self, t, slot):
        """Zeros into V's rows behind the last position."""
        yield from self.wait(("full", slot % self.stages), slot // self.stages)
        if self.holds.get(slot % self.stages) != slot:
            raise Wrong(f"rows of block {self.holds.get(slot % self.stages)} cleared for those of {slot}")
        self.cleared.add((t, slot))

    def softmax(self, t):
        n_s = n_o = base = 0
        try:
            for n, blocks in enumerate(self.pieces):
                for j in range(blocks[t]):
                    yield from self.wait(("s", t), n_s)
                    if j and self.done[t] < 2 * n_s:
                        raise Wrong("O rescaled before its products")
                    if self.ragged[n] and j + 1 == max(blocks):
                        yield from self.clear(t, base + 2 * j + 1)
                    self.arrive(("p0", t))
                    yield "between", n_s
                    self.arrive(("p1", t))
                    n_s += 1
                if blocks[t]:
                    yield from self.wait(("o_full", t), n_o)
                    if self.done[t] < 2 * n_s:
                        raise Wrong("O read before its products")
                    n_o += 1
                    self.arrive(("o_empty", t))
                base += 2 * max(blocks)
        except GaveUp:
            pass
        self.ended += 1

    def run(self):
        alive = {"load": self.load(), "products": self.products(), "softmax 0": self.softmax(0), "softmax 1": self.softmax(1), "pipe": self.tensor_pipe(), "tma": self.tma()}
        where, idle = {}, 0
        while len(alive) > 2:
            moved = False
            for name in self.rng.sample(sorted(alive), len(alive)):
                if self.rng.random() < 0.3:
                    continue
                try:
                    at = next(alive[name])
                    moved |= where.get(name) != at
                    where[name] = at
                except StopIteration:
                    del alive[name]
                    moved = True
            idle = 0 if moved else idle + 1
            if idle > 600:
                raise Wrong(f"nothing moves: {where}")


def some_pieces(rng):
    pieces = []
    for _ in range(rng.randint(1, 8)):
        n = rng.randint(1, 4)
        pieces.append(rng.choice([(n, n), (n, n + 1), (n, 0), (0, n), (1, 0), (1, 1), (0, 0) if pieces else (1, 1)]) + (rng.random() < 0.6,))
    return pieces


@pytest.mark.parametrize("fails", [0.0, 0.003, 0.05])
@pytest.mark.parametrize("stages,queries", [(4, 3), (8, 4)])
def test_ragged_blocks_and_two_part_weights(stages, queries, fails):
    for seed in range(800):
        rng = random.Random(seed)
        Whole(some_pieces(rng), stages, queries, rng, fails).run()


def fails_somewhere(model, fails=0.0):
    with pytest.raises(Wrong):
        for seed in range(300):
            rng = random.Random(seed)
            model(some_pieces(rng), 4, 3, rng, fails).run()


def test_the_model_finds_rows_cleared_in_another_slot():
    class Shifted(Whole):
        def clear(self, t, slot):
            yield from super().clear(t, slot - 1)

    fails_somewhere(Shifted)


def test_the_model_finds_one_barrier_for_both_parts():
    class One(Whole):
        def wait(self, bar, phase, bounded=True):
            yield from super().wait(("p0", bar[1]) if bar[0] == "p1" else bar, phase, bounded)

        def arrive(self, bar):
            super().arrive(("p0", bar[1]) if bar[0] == "p1" else bar)

    fails_somewhere(One)


def test_the_model_finds_loads_that_outlive_the_block():
    """The loading warp looks for a failure when it has issued its own loads, not when all warps have ended."""
    class Early(Whole):
        def load(self):
            self.ended += 3
            yield from super().load()

    fails_somewhere(Early, 0.05)


def test_the_model_finds_a_block_that_does_not_wait_for_its_products():
    class Hasty(Whole):
        def products(self):
            yield from self.all_products()
            if self.pipe:
                raise Wrong("a product, or its commit's arrival, after the block has ended")
            self.ended += 1

    fails_somewhere(Hasty)
