"""The warps of the stream of few rows (int8_few_kernel, pie_int8.cuh) that bring a tile's sums out, where a wait of one of them runs out: walked here in random order, with what the kernel's text says
that such a warp does.  Every warp comes to the kernel's end, and the workspace is at zero behind it."""
import os
import random
import re

import pytest

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "proxy_inference_engine_b200", "csrc", "pie_int8.cuh")


def role():
    """The text of the warps that take accumulators, without comments."""
    with open(HEADER) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    text = text[text.index("int8_few_kernel(const __grid_constant__"):]
    return text[text.index("if (warp < 4) {"):text.index("} else if (warp == T::W_TMA) {")]


class Launch:
    """CTAs with equal shares of a line of tiles, as the kernel cuts it.  expired: (CTA, warp, its n-th tile) of waits that run out."""

    def __init__(self, tiles, nk, ctas, expired, leaves, seed):
        self.rng, self.expired, self.leaves = random.Random(seed), expired, leaves
        self.tiles, self.nk, self.steps = tiles, nk, tiles * nk
        self.ctas = min(ctas, self.steps)
        self.sums, self.count = [[0] * 4 for _ in range(tiles)], [0] * tiles
        self.out = [[None] * 4 for _ in range(tiles)]
        self.at_bar, self.round, self.last = [0] * self.ctas, [0] * self.ctas, [False] * self.ctas
        self.aborted = [False] * self.ctas

    def bar(self, cta):
        mine = self.round[cta]
        self.at_bar[cta] += 1
        if self.at_bar[cta] == 4:
            self.at_bar[cta], self.round[cta] = 0, mine + 1
        while self.round[cta] == mine:
            yield

    def warp(self, cta, warp):
        lo, hi = cta * self.steps // self.ctas, (cta + 1) * self.steps // self.ctas
        t, k0, done, i, alive = lo // self.nk, lo % self.nk, 0, 0, True
        while done < hi - lo:
            n = min(self.nk - k0, hi - lo - done)
            done += n
            yield
            if (cta, warp, i) in self.expired:
                self.aborted[cta] = True
            # another warp's abort is seen, or the accumulator is there first
            if alive and self.aborted[cta]:
                alive = (cta, warp, i) not in self.expired and self.rng.random() < 0.5
            if not alive and self.leaves:
                return
            if n == self.nk:
                if alive:
                    self.out[t][warp] = n
            else:
                if alive:
                    self.sums[t][warp] += n
                parts = ((t + 1) * self.nk * self.ctas - 1) // self.steps - ((t * self.nk + 1) * self.ctas - 1) // self.steps + 1
                yield from self.bar(cta)
                if warp == 0:
                    before, self.count[t] = self.count[t], self.count[t] + 1
                    self.last[cta] = before == parts - 1
                    if self.last[cta]:
                        self.count[t] = 0
                yield from self.bar(cta)
                if self.last[cta]:
                    self.out[t][warp], self.sums[t][warp] = self.sums[t][warp], 0
            t, k0, i = t + 1, 0, i + 1

    def go(self):
        """Whether every warp came to its end."""
        warps = [self.warp(c, w) for c in range(self.ctas) for w in range(4)]
        idle = 0
        while warps and idle < 400 * len(warps):
            k = self.rng.randrange(len(warps))
            before = (sum(self.round), sum(self.at_bar))
            try:
                next(warps[k])
                idle = 0 if (sum(self.round), sum(self.at_bar)) != before else idle + 1
            except StopIteration:
                del warps[k]
                idle = 0
        return not warps


def launches(seed, leaves, expire=True):
    rng = random.Random(seed)
    tiles, nk, ctas = rng.choice([1, 2, 5, 32]), rng.choice([1, 3, 7, 32]), rng.choice([2, 5, 37])
    expired = {(rng.randrange(ctas), rng.randrange(4), rng.choice([0, 0, 1, 2])) for _ in range(rng.choice([1, 2, 9]))} if expire else ()
    return Launch(tiles, nk, ctas, expired, leaves, seed)


def test_a_warp_whose_wait_ran_out_does_not_leave():
    text = role()
    assert "gemm_wait_warp(smem_u32(&tfull_bar" in text
    assert not re.search(r"\b(break|return|continue|goto)\b", text)
    # barriers and counter stand under no condition but that of a tile in several shares
    shared = text[text.index("if (!whole) {"):]
    assert "alive" not in shared and shared.count("bar.sync 1, 128") == 2 and text.count("bar.sync 1, 128") == 2


@pytest.mark.parametrize("seed", range(200))
def test_every_warp_ends_and_the_workspace_is_left_at_zero(seed):
    at = launches(seed, leaves=bool(re.search(r"\b(break|return)\b", role())))
    assert at.go()
    assert not any(at.count) and not any(map(any, at.sums))


@pytest.mark.parametrize("seed", range(40))
def test_sums_are_whole_where_no_wait_runs_out(seed):
    at = launches(seed, leaves=False, expire=False)
    assert at.go() and not any(at.count) and not any(map(any, at.sums))
    assert all(n == at.nk for tile in at.out for n in tile)


def test_the_walk_finds_a_warp_that_leaves():
    """Others wait for it for good, or the workspace is left as it was."""
    ends = [launches(seed, leaves=True) for seed in range(200)]
    assert any(not at.go() for at in ends) and any(any(at.count) or any(map(any, at.sums)) for at in ends)
