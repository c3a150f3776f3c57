"""What the walk of the attention's waits over 8-bit pages (test_cpu_fp8_schedule.py) holds the kernel to is the kernel's own, and it finds each wait that is left out, each by itself and each
with the finding that it should be."""
import random
import re
import sys

import pytest

from test_cpu_fp8_schedule import HEADER, Walk, pieces_of


def source():
    with open(HEADER) as f:
        return f.read()


def test_the_walk_has_the_kernels_barriers():
    """Arrivals of a round, places, and how far scores are ahead."""
    text = re.sub(r"//[^\n]*", "", source())
    counts = dict(re.findall(r"mbar_init\(&(\w+)\[i\], (\d+)\);", text))
    walk = Walk([], 128, 0)
    for name in counts:
        assert {bar.count for bar in getattr(walk, name)} == {int(counts[name])}, name
    assert {"q_full", "q_empty", "s_full", "p_full", "o_full", "k_full", "k_empty", "v_full", "v_empty", "f_full", "f_empty", "sc_full", "sc_empty", "qf_full", "qf_empty", "turn_free", "fp_full",
            "fo_full", "fs_full"} == set(counts)
    declared = dict(re.findall(r"\b(fs_full|turn_free|qf_full|qf_empty|fp_full|fo_full)\[(\d)\]", text[text.index("__align__(8) uint64_t f_full["):]))
    for name, n in declared.items():
        assert len(getattr(walk, name)) == int(n), name
    assert "scored < min(tile + 4, end_all)" in text and "fs_full[tile & 3]" in text and "fs_full[tile & 3]), (tile >> 2) & 1" in text
    assert "turn_free[few_pieces & 1]), ((few_pieces >> 1) - 1) & 1" in text and "turn_free[(few_pieces - 1) & 1]), ((few_pieces - 1) >> 1) & 1" in text
    assert "fo_full[g]), ((tile >> 1) - 1) & 1" in text


class Without(Walk):
    """A walk whose waits of one kind are let through at once.  left_out(role, bar, round, locals of the role)."""

    def __init__(self, *args, left_out, **kw):
        super().__init__(*args, **kw)
        self.left_out = left_out

    def wait(self, bar, round_, own=True):
        frame = sys._getframe(1)
        if self.left_out(self, frame.f_code.co_name, bar, round_, frame.f_locals):
            return iter(())
        return super().wait(bar, round_, own)


def query_tile_over_weights(w, role, bar, round_, at):
    return role == "fetch_q" and bar in w.turn_free


def weights_over_weights(w, role, bar, round_, at):
    return role == "softmax" and bar in w.fo_full and round_ == (at["tile"] >> 1) - 1   # (not the wait behind the last tile)


def place_over_place(w, role, bar, round_, at):
    return role == "acquire" and bar in w.f_empty


def scores_before_their_tile(w, role, bar, round_, at):
    return role == "softmax" and bar in w.fs_full


def scales_before_they_are_there(w, role, bar, round_, at):
    return role == "softmax" and bar in w.sc_full


FAULTS = [(query_tile_over_weights, "other operands"), (weights_over_weights, "a product of other operands"), (place_over_place, "other operands"),
          (scores_before_their_tile, "assert (None == ("), (scales_before_they_are_there, "another tile's scales")]


@pytest.mark.parametrize("left_out,finding", FAULTS, ids=lambda v: getattr(v, "__name__", ""))
def test_a_wait_that_is_left_out_is_found(left_out, finding):
    found = set()
    for seed in range(60):
        try:
            Without(pieces_of(random.Random(seed), 12), 128, seed, left_out=left_out).go()
        except AssertionError as e:
            found.add(str(e))
            if finding in str(e):
                return
        except (TypeError, KeyError):   # (a query tile where weights were asked for; not what is looked for here)
            pass
    assert False, found


@pytest.mark.parametrize("seed", range(8))
def test_with_every_wait_the_walk_ends(seed):
    rng = random.Random(seed)
    Without(pieces_of(rng, 12), 128, seed, left_out=lambda *a: False).go()
