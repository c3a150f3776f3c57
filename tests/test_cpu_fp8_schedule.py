"""The warps of the attention over 8-bit pages (pie_chunk_attn.cuh) hand pages, tiles, scores and scales to one another through mbarriers, whose waits know a round only by its parity.  Walked here:
every role as the kernel has it, in random order, over random sequences of pieces.  A wait that a round other than its own lets through, one that never ends, and a product that reads what
is not its own are found."""
import os
import random
import re

import pytest

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "proxy_inference_engine_b200", "csrc", "pie_chunk_attn.cuh")
PAIR, ONE, FEW = "pair", "one", "few"


def constants(D):
    with open(HEADER) as f:
        text = f.read()
    pick = lambda pattern: tuple(int(x) for x in re.search(pattern, text).groups())
    ring = dict(zip((64, 128), pick(r"int RING = D == 64 \? (\d+) : (\d+);")))[D]
    assert "PLACES = 2 * RING;" in text
    return ring, pick(r"kChunkScales = (\d+);")[0]


class Bar:
    def __init__(self, count):
        self.count, self.left, self.done = count, count, 0

    def arrive(self, n=1):
        assert self.left >= n, "more arrivals than the round has"
        self.left -= n
        if self.left == 0:
            self.left, self.done = self.count, self.done + 1


class Walk:
    def __init__(self, pieces, D, seed, weights_wait=True):
        self.rng, self.pieces = random.Random(seed), pieces
        self.R, self.SC = constants(D)
        self.PLACES, self.weights_wait = 2 * self.R, weights_wait
        bars = lambda n, count: [Bar(count) for _ in range(n)]
        self.q_full, self.q_empty = bars(2, 1), bars(2, 1)
        self.k_full, self.k_empty, self.v_full, self.v_empty = (bars(self.R, 1) for _ in range(4))
        self.s_full, self.p_full, self.o_full = bars(2, 1), bars(2, 4), bars(2, 1)
        self.f_full, self.f_empty = bars(self.PLACES, 1), bars(self.PLACES, 1)
        self.sc_full, self.sc_empty = bars(self.SC, 1), bars(self.SC, 4)
        self.fs_full, self.fp_full, self.fo_full = bars(4, 1), bars(2, 4), bars(2, 1)
        self.turn_free, self.qf_full, self.qf_empty = bars(2, 1), bars(2, 1), bars(2, 9)
        self.pipe, self.copies, self.at_sync, self.moves = [], [], 0, 0
        self.sync_round = 0
        self.place_in, self.q_in = [None] * self.PLACES, [None, None]   # places: those of V, then those of K; the two query tiles, the second of which is P's place too
        self.qf_in, self.scale_in, self.scores_in = [None, None], [None] * self.SC, [None] * 4

    # ---- waits: a generator yields what it waits for
    def wait(self, bar, round_, own=True):
        """For the end of round `round_` (from 0), known by its parity alone."""
        while (bar.done & 1) == (round_ & 1):
            yield
        assert not own or bar.done == round_ + 1, f"round {round_} was waited for, {bar.done} are done"

    def wait_free(self, bar, use):
        """For the place's use number `use`: the first is free."""
        if use > 0:
            yield from self.wait(bar, use - 1)
        else:
            assert bar.done == 0
            yield

    @staticmethod
    def ready(bar, round_):
        done = (bar.done & 1) != (round_ & 1)
        assert not done or bar.done == round_ + 1, f"round {round_} was asked for, {bar.done} are done"
        return done

    def sync(self):
        round_ = self.sync_round
        self.at_sync += 1
        if self.at_sync == 8:
            self.at_sync, self.sync_round = 0, self.sync_round + 1
        while self.sync_round == round_:
            yield

    # ---- roles
    def tma(self):
        cq, ck, cf, few = [0, 0], 0, 0, 0
        held, rounds = {}, {}

        def acquire(place):
            kind = held.pop(place, None)
            if kind:
                bar = self.f_empty[place] if kind == FEW else self.v_empty[place] if place < self.R else self.k_empty[place - self.R]
                yield from self.wait(bar, rounds.get((place, kind), 0))
                rounds[place, kind] = rounds.get((place, kind), 0) + 1

        def copy(bar, into, at, what):
            self.copies.append(lambda: (into.__setitem__(at, what), bar.arrive()))
        for n, p in enumerate(self.pieces):
            kind, tiles, cnt = p[:3]
            if kind == FEW and few > 1:
                yield from self.wait(self.turn_free[few & 1], (few >> 1) - 1)

            def fetch_q(g):
                if (cnt[g] if kind == PAIR else 0 if kind == FEW else 1 - g) == 0:
                    return
                yield from self.wait_free(self.q_empty[g], cq[g])
                cq[g] += 1
                if g and few > 0 and self.weights_wait:
                    yield from self.wait(self.turn_free[(few - 1) & 1], (few - 1) >> 1)
                copy(self.q_full[g], self.q_in, g, n)
            yield from fetch_q(0)
            for j in range(tiles):
                if kind == FEW:
                    place = cf % self.PLACES
                    yield from acquire(place)
                    held[place] = FEW
                    copy(self.f_full[place], self.place_in, place, (n, j))
                    cf += 1
                    continue
                i = ck % self.R
                yield from acquire(self.R + i)
                held[self.R + i] = PAIR
                copy(self.k_full[i], self.place_in, self.R + i, (n, j))
                if j == 0:
                    yield from fetch_q(1)
                yield from acquire(i)
                held[i] = PAIR
                copy(self.v_full[i], self.place_in, i, (n, j))
                ck += 1
            few += kind == FEW

    def scales(self):
        cf = 0
        for n, (kind, tiles, *_) in enumerate(self.pieces):
            for j in range(tiles if kind == FEW else 0):
                i = cf % self.SC
                yield from self.wait_free(self.sc_empty[i], cf // self.SC)
                cf += 1
                self.scale_in[i] = (n, j)
                yield
                self.sc_full[i].arrive()

    def queries(self):
        k = 0
        for n, (kind, *_) in enumerate(self.pieces):
            if kind == FEW:
                yield from self.wait_free(self.qf_empty[k & 1], k >> 1)
                self.qf_in[k & 1] = n
                yield
                self.qf_full[k & 1].arrive()
                k += 1

    def mma(self):
        c, cq, ck, cf, few, scored = [0, 0], [0, 0], 0, 0, 0, 0
        ahead = [False, False]

        def commit(bar):
            self.pipe.append(bar.arrive)

        def scores(n, g, tile, t, step):
            def run():
                assert self.place_in[self.R + t % self.R] == (n, step) and self.q_in[tile] == n, "scores of other operands"
            self.pipe.append(run)
            commit(self.s_full[g])

        def product(n, g, t, step):
            def run():
                assert self.place_in[t % self.R] == (n, step), "a product of other values"
            self.pipe.append(run)
            commit(self.o_full[g])

        def scores8(n, tile, which, step):
            def run():
                assert self.place_in[tile % self.PLACES] == (n, step) and self.qf_in[which] == n, "scores of other operands"
                assert self.scores_in[tile & 3] is None, "scores written over"
                self.scores_in[tile & 3] = (n, step)
            self.pipe.append(run)
            commit(self.fs_full[tile & 3])

        def product8(n, tile, step):
            def run():
                assert self.place_in[tile % self.PLACES] == (n, step) and self.q_in[1][tile & 1] == (n, step), "a product of other operands"
            self.pipe.append(run)
            commit(self.fo_full[tile & 1])
            commit(self.f_empty[tile % self.PLACES])

        def open_(n, p, g, t, q):
            kind, tiles, cnt = p[:3]
            pair = kind == PAIR
            tile, step = (g, 0) if pair else (0, g)
            yield from self.wait(self.q_full[tile], q[tile])
            yield from self.wait(self.k_full[(t + step) % self.R], (t + step) // self.R)
            scores(n, g, tile, t + step, step)
            if not pair:
                commit(self.k_empty[(t + step) % self.R])
            if (cnt[g] == 1) if pair else step == tiles - 1:
                commit(self.q_empty[tile])
        for n, p in enumerate(self.pieces):
            kind, tiles, cnt = p[:3]
            more = n + 1 < len(self.pieces)
            following = self.pieces[n + 1] if more else (None, 0, (0, 0))
            pair = kind == PAIR
            if kind == FEW:
                end_own = cf + tiles
                end_all = end_own + (following[1] if following[0] == FEW else 0)
                tile = cf
                while tile < end_own:
                    if scored < min(tile + 4, end_all):
                        own = scored < end_own
                        f, place = few + (not own), scored % self.PLACES
                        if self.ready(self.qf_full[f & 1], f >> 1) and self.ready(self.f_full[place], scored // self.PLACES):
                            scores8(n if own else n + 1, scored, f & 1, scored - (cf if own else end_own))
                            if scored + 1 == (end_own if own else end_all):
                                commit(self.qf_empty[f & 1])
                            scored += 1
                    if tile < scored and self.ready(self.fp_full[tile & 1], tile >> 1):
                        product8(n, tile, tile - cf)
                        if tile + 1 == end_own:
                            commit(self.turn_free[few & 1])
                        tile += 1
                    yield
                cf, few = end_own, few + 1
                continue
            tn = ck + tiles
            nq = [cq[0] + (cnt[0] > 0 if pair else 1), cq[1] + (pair and cnt[1] > 0)]
            for g in range(2):
                if cnt[g] > 0 and not ahead[g]:
                    yield from open_(n, p, g, ck, cq)
                ahead[g] = False

            def go_on(g):
                if more and following[0] != FEW and following[2][g] > 0 and (following[0] == PAIR or g == 0 or ahead[0]):
                    yield from open_(n + 1, following, g, tn, nq)
                    ahead[g] = True
            if pair:
                commit(self.k_empty[ck % self.R])
                for j in range(tiles):
                    t = ck + j
                    yield from self.wait(self.v_full[t % self.R], t // self.R)
                    if j + 1 < tiles:
                        yield from self.wait(self.k_full[(t + 1) % self.R], (t + 1) // self.R)
                    for g in range(2):
                        if j < cnt[g]:
                            yield from self.wait(self.p_full[g], c[g] + j)
                            product(n, g, t, j)
                            if j + 1 < cnt[g]:
                                scores(n, g, g, t + 1, j + 1)
                                if j + 2 == cnt[g]:
                                    commit(self.q_empty[g])
                            if j + 1 == cnt[g]:
                                yield from go_on(g)
                    commit(self.v_empty[t % self.R])
                    if j + 1 < tiles:
                        commit(self.k_empty[(t + 1) % self.R])
            else:
                for j in range(tiles):
                    t, g = ck + j, j & 1
                    yield from self.wait(self.v_full[t % self.R], t // self.R)
                    yield from self.wait(self.p_full[g], c[g] + (j >> 1))
                    product(n, g, t, j)
                    commit(self.v_empty[t % self.R])
                    if j + 2 < tiles:
                        yield from self.wait(self.k_full[(t + 2) % self.R], (t + 2) // self.R)
                        scores(n, g, 0, t + 2, j + 2)
                        commit(self.k_empty[(t + 2) % self.R])
                        if j + 3 == tiles:
                            commit(self.q_empty[0])
                    else:
                        yield from go_on(g)
            c = [c[0] + cnt[0], c[1] + cnt[1]]
            ck, cq = tn, nq

    def softmax(self, warp):
        g, quad = warp >> 2, warp & 3
        c, cf, few = [0, 0], 0, 0
        for n, (kind, tiles, cnt, cut) in enumerate(self.pieces):
            if kind == FEW:
                yield from self.wait(self.qf_full[few & 1], few >> 1)
                own = (g ^ cf) & 1
                cnt = [(tiles + 1 - (h ^ cf & 1)) // 2 for h in range(2)]
                for i in range(cnt[g]):
                    step = 2 * i + own
                    tile = cf + step
                    yield from self.wait(self.sc_full[tile % self.SC], tile // self.SC)
                    assert self.scale_in[tile % self.SC] == (n, step), "another tile's scales"
                    self.sc_empty[tile % self.SC].arrive()
                    yield from self.wait(self.fs_full[tile & 3], tile >> 2)
                    assert self.scores_in[tile & 3] == (n, step) and self.qf_in[few & 1] == n
                    if i > 0 and self.weights_wait:
                        yield from self.wait(self.fo_full[g], (tile >> 1) - 1)
                    self.q_in[1] = {**(self.q_in[1] if isinstance(self.q_in[1], dict) else {}), g: (n, step)}
                    if step == tiles - 1:   # values behind the last key
                        yield from self.wait(self.f_full[tile % self.PLACES], tile // self.PLACES)
                        assert self.place_in[tile % self.PLACES] == (n, step)
                    yield
                    if self.fp_full[g].left == 1:
                        self.scores_in[tile & 3] = None
                    self.fp_full[g].arrive()
                self.qf_empty[few & 1].arrive()
                few, cf = few + 1, cf + tiles
            else:
                for i in range(cnt[g]):
                    yield from self.wait(self.s_full[g], c[g] + i)
                    if i > 0 and self.rng.random() < 0.3:
                        yield from self.wait(self.o_full[g], c[g] + i - 1)
                    yield
                    self.p_full[g].arrive()
            if kind == FEW:
                if cnt[g]:
                    yield from self.wait(self.fo_full[g], (cf - tiles + 2 * cnt[g] - 2 + own) >> 1)
                yield from self.sync()
                assert all(self.fo_full[last & 1].done == (last >> 1) + 1 for last in range(cf - min(tiles, 2), cf))
                yield from self.sync()
            else:
                c = [c[0] + cnt[0], c[1] + cnt[1]]
                for h in (g,) if kind == PAIR else (0, 1):
                    if cnt[h] > 0:   # (the other group's: its own warps see to it, and all meet behind that)
                        yield from self.wait(self.o_full[h], c[h] - 1, own=h == g)
                if kind == ONE:
                    yield from self.sync()
                    assert all(self.o_full[h].done == c[h] for h in range(2))
            if cut:
                yield from self.sync()
                yield from self.sync()
            elif kind != PAIR:
                yield from self.sync()

    def go(self):
        roles = [self.tma(), self.scales(), self.queries(), self.mma()] + [self.softmax(w) for w in range(8)]
        pace = [self.rng.choice([1, 1, 1, 8, 40]) for _ in roles]
        pipe_pace, copy_pace = self.rng.choice([1, 3, 20]), self.rng.choice([1, 3, 20])
        idle = 0
        while roles:
            k = self.rng.randrange(len(roles) + 2)
            before = (len(roles), len(self.pipe), len(self.copies))
            if k == len(roles):
                if self.pipe and self.rng.random() < 1 / pipe_pace:
                    self.pipe.pop(0)()
            elif k == len(roles) + 1:
                if self.copies and self.rng.random() < 1 / copy_pace:
                    self.copies.pop(self.rng.randrange(len(self.copies)))()   # (copies land in any order)
            elif self.rng.random() < 1 / pace[k]:
                mark = self.mark()
                try:
                    next(roles[k])
                except StopIteration:
                    del roles[k], pace[k]
                if self.mark() != mark:
                    idle = 0
            idle = 0 if (len(roles), len(self.pipe), len(self.copies)) != before else idle + 1
            assert idle < 400 * 40 * 20, "nothing moves"

    def mark(self):
        return self.at_sync, self.sync_round, sum(b.done * 16 + b.left for bars in (self.p_full, self.fp_full, self.qf_full, self.qf_empty, self.sc_full, self.sc_empty) for b in bars)


def pieces_of(rng, count, most=6):
    got = []
    for _ in range(count):
        kind, n = rng.choice([PAIR, ONE, FEW, FEW]), rng.randint(1, most)
        cnt = (rng.choice([n, n, max(0, n - 1)]), n) if kind == PAIR else ((n + 1) // 2, n // 2)
        got.append((kind, n, cnt, rng.random() < 0.3))
    return got


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("seed", range(40))
def test_every_wait_ends_with_its_own_round(D, seed):
    rng = random.Random(1000 * D + seed)
    Walk(pieces_of(rng, rng.choice([1, 2, 3, 8, 20])), D, seed).go()


def test_the_walk_finds_what_would_break():
    """A query tile copied to where weights still lie, and weights written over that a product still reads."""
    for seed in range(30):
        rng = random.Random(seed)
        try:
            Walk(pieces_of(rng, 12), 128, seed, weights_wait=False).go()
        except (AssertionError, IndexError, TypeError):
            return
    assert False
