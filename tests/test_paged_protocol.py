"""The barriers of the prompt attention (csrc/paged_prompt.cu) as a model on the host: the loading warp, the thread that issues the products, the tensor
pipe that finishes them in order, and each tile's softmax are coroutines over mbarriers, which know no more than the parity of
a phase. In random order, over random lists of pieces, no wait may pass before its phase or after the next, O may not be read or
rescaled before its products, and nothing may stand still."""
import random

import pytest


class Wrong(Exception):
    pass


class Model:
    def __init__(self, pieces, stages, queries, rng):
        self.pieces, self.stages, self.queries, self.rng = pieces, stages, queries, rng
        self.phases = {}                  # barrier -> phases completed
        self.pipe = []                    # commits on their way, in order
        self.issued, self.done = [0, 0], [0, 0]  # products into O, by tile

    def arrive(self, bar):
        self.phases[bar] = self.phases.get(bar, 0) + 1

    def wait(self, bar, phase):
        """As the device waits: until the parity of the phase under way is another than this one's."""
        while (self.phases.get(bar, 0) & 1) == (phase & 1):
            yield bar, phase
        if self.phases.get(bar, 0) != phase + 1:
            raise Wrong(f"{bar}: phase {phase} taken for over at {self.phases.get(bar, 0)} completed")

    def tensor_pipe(self):
        while True:
            if self.pipe and self.rng.random() < 0.4:
                what, x = self.pipe.pop(0)
                if what == "product":
                    self.done[x] += 1
                else:
                    self.arrive((what, x))
            yield len(self.pipe)

    def load(self):
        slot = n_q = 0
        for blocks in self.pieces:
            for j in range(max(blocks)):
                for kv in range(2):
                    if slot // self.stages:
                        yield from self.wait(("empty", slot % self.stages), slot // self.stages - 1)
                    self.arrive(("full", slot % self.stages))
                    slot += 1
                    if kv or j:
                        continue
                    for t in range(2):
                        if blocks[t]:
                            if n_q // self.queries:
                                yield from self.wait(("q_empty", n_q % self.queries), n_q // self.queries - 1)
                            self.arrive(("q_full", n_q % self.queries))
                            n_q += 1

    def products(self):
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
                    yield from self.wait(("p", t), n_s[t])
                    commit("product", t)
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

    def softmax(self, t):
        n_s = n_o = 0
        for blocks in self.pieces:
            for j in range(blocks[t]):
                yield from self.wait(("s", t), n_s)
                if j and self.done[t] < n_s:
                    raise Wrong("O rescaled before its products")
                self.arrive(("p", t))
                n_s += 1
            if blocks[t]:
                yield from self.wait(("o_full", t), n_o)
                if self.done[t] < n_s:
                    raise Wrong("O read before its products")
                n_o += 1
                self.arrive(("o_empty", t))

    def run(self):
        alive = {"load": self.load(), "products": self.products(), "softmax 0": self.softmax(0), "softmax 1": self.softmax(1), "pipe": self.tensor_pipe()}
        where, idle = {}, 0
        while len(alive) > 1:
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


@pytest.mark.parametrize("stages,queries", [(4, 3), (8, 4)])
def test_no_wait_is_early_late_or_for_good(stages, queries):
    for seed in range(1500):
        rng = random.Random(seed)
        pieces = []
        for _ in range(rng.randint(1, 8)):
            n = rng.randint(1, 4)
            # both tiles see the same blocks, the second one more, or only one of them has anything to do
            pieces.append(rng.choice([(n, n), (n, n + 1), (n, 0), (0, n), (1, 0), (1, 1), (0, 0) if pieces else (1, 1)]))
        Model(pieces, stages, queries, rng).run()


def test_the_model_finds_a_shared_barrier():
    """The same with one barrier for both tiles' S: the model has to see it."""
    class Shared(Model):
        def wait(self, bar, phase):
            yield from super().wait(("s", 0) if bar[0] == "s" else bar, phase)

        def arrive(self, bar):
            super().arrive(("s", 0) if bar[0] == "s" else bar)

    with pytest.raises(Wrong):
        for seed in range(50):
            Shared([(2, 2), (1, 0), (3, 3)], 4, 3, random.Random(seed)).run()
