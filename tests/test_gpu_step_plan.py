"""ragged.StepPlan: rows, slots, block table, logit rows and attention's schedule, built on the device from the requests' lengths."""
import random

import pytest
import torch

import step_oracle as O

pytestmark = pytest.mark.gpu
ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
NAMES = ("row_starts", "contexts", "sequences", "positions", "slots", "block_table", "logit_rows", "logit_starts", "draft_tokens")


def case(new, cached, drafted=None, pad=0, pad_logits=0, heads=(32, 8), seed=0, table=False, spare=2):
    from proxy_inference_engine_b200.ragged import StepPlan
    rng = random.Random(seed)
    T, R = sum(new) + pad, sum((drafted[s] if drafted else 0) + 1 for s, n in enumerate(new) if n) + pad_logits
    T, R = max(T, 1), max(R, 1)
    counts = [O.need(n, c) for n, c in zip(new, cached)]
    width, n_pages = max(1, *counts) + (1 if seed % 2 else 0), sum(counts) + 3
    all_pages = rng.sample(range(n_pages), sum(counts))
    pages = [[all_pages.pop() for _ in range(k)] for k in counts]
    ids = [rng.randrange(1000) for _ in range(T)]
    if table:
        wide = torch.full((len(new), width + spare), 10 ** 6, dtype=torch.int32)      # what lies behind a request's pages is not looked at
        for s, p in enumerate(pages):
            wide[s, :len(p)] = torch.tensor(p, dtype=torch.int32)
        given = wide.cuda()[:, :width + 1]
    else:
        given = ints([p for mine in pages for p in mine])
    plan = StepPlan.build(ints(ids), ints(new), ints(cached), given, num_pages=n_pages, max_blocks=width, num_heads=heads[0], num_kv_heads=heads[1],
                          draft_lengths=None if drafted is None else ints(drafted), num_logits=R)
    return plan, O.plan(ids, new, cached, pages, width, drafted, T, R)


def agrees(plan, want):
    for name in NAMES:
        assert getattr(plan, name).tolist() == want[name], name
    plan.check()


def schedule_is_whole(plan):
    """Every key tile of every item is in one CTA's list, an item's pieces are in CTAs one behind the other and agree on how many they are, and a CTA has at most one piece that
    goes on from the CTA before and one that goes on in the next."""
    words, d = plan.words.tolist(), plan.dims
    at = plan.status.storage_offset() + 192
    ranges, base = words[at:at + 384], at + 384
    G = d.Hq // d.Hkv
    tile, starts, ctx = 128 // G, plan.row_starts.tolist(), plan.contexts.tolist()
    seen, opens, shares, plan_table = {}, set(), [], plan.block_table.tolist()
    for c in range(192):
        lo, hi = ranges[2 * c], ranges[2 * c + 1]
        assert 0 <= lo <= hi and (base + 12 * hi <= len(words) or lo == hi)
        cost = 0
        for i in range(lo, hi):
            row0, pos0, tokens, s, h, k0, k1, first, pieces, page0, page1 = words[base + 12 * i:base + 12 * i + 11]
            assert 0 <= k0 <= k1
            if k0 == k1:
                continue
            mine = plan_table[s][:(pos0 + tokens + 63) // 64]
            assert [page0, page1] == [mine[min(j, len(mine) - 1)] for j in (2 * k0, 2 * k0 + 1)]
            item = seen.setdefault((h, s, row0), [])
            item.append((k0, k1, c, first, pieces))
            cost += (k1 - k0) * (2 if tokens > tile else 1)
            assert 0 <= h < d.Hkv and (row0 - starts[s]) % (2 * tile) == 0 and pos0 == ctx[s] + row0 - starts[s]
            assert tokens == min(2 * tile, starts[s + 1] - row0) and k1 <= (pos0 + tokens + 127) // 128
            if pieces > 1 and c == first:
                assert c not in opens
                opens.add(c)
        shares.append(cost)
    for (h, s, row0), pieces in seen.items():
        tokens = min(2 * tile, starts[s + 1] - row0)
        assert [p[0] for p in pieces] == [0] + [p[1] for p in pieces[:-1]] and pieces[-1][1] == (ctx[s] + row0 - starts[s] + tokens + 127) // 128
        assert [p[2] for p in pieces] == list(range(pieces[0][2], pieces[0][2] + len(pieces)))
        assert all(p[3] == pieces[0][2] and p[4] == len(pieces) for p in pieces)
    assert len(seen) == d.Hkv * sum((starts[s + 1] - starts[s] + 2 * tile - 1) // (2 * tile) for s in range(d.requests))
    return shares


@pytest.mark.parametrize("table", [False, True])
@pytest.mark.parametrize("new,cached,drafted,pad", [
    ([1], [0], None, 0),
    ([5], [63], [4], 0),
    ([70, 1, 20], [0, 100, 64], None, 0),
    ([1, 4, 64, 65, 3], [64, 60, 0, 63, 1], [0, 3, 0, 0, 2], 0),
    ([0, 3, 0, 0, 7, 0], [10, 0, 0, 64, 129, 65], [0, 2, 0, 0, 6, 0], 0),       # requests that sit the step out, drafts up to all but one
    ([3, 2], [61, 7], [1, 0], 9),                                              # rows behind the last request's
    ([0, 0], [5, 0], None, 4),                                                 # nobody has anything
    ([513, 1, 700], [1000, 5000, 3], None, 3),
])
def test_arrays(new, cached, drafted, pad, table):
    plan, want = case(new, cached, drafted, pad, pad_logits=pad, seed=len(new), table=table)
    agrees(plan, want)
    schedule_is_whole(plan)


@pytest.mark.parametrize("requests", [2, 511, 512, 513, 1000, 4096])
def test_many_requests(requests):
    rng = random.Random(requests)
    new = [rng.choice([0, 1, 1, 1, 2, 6, 33]) for _ in range(requests)]
    cached = [rng.randint(0, 300) for _ in range(requests)]
    plan, want = case(new, cached, [max(0, min(n - 1, 5)) for n in new], pad=5, pad_logits=2, seed=requests)
    agrees(plan, want)
    schedule_is_whole(plan)


@pytest.mark.parametrize("heads", [(32, 8), (64, 8), (4, 4), (24, 8), (7, 1), (40, 1), (128, 1), (6, 2)])
def test_schedule_of_other_heads(heads):
    rng = random.Random(sum(heads))
    plan, want = case([300, 1, 4, 90, 1], [1000, 8191, 777, 0, 30000], heads=heads, seed=3)
    agrees(plan, want)
    schedule_is_whole(plan)


def test_the_shares_are_even():
    plan, _ = case([2048], [15000])
    shares = [c for c in schedule_is_whole(plan) if c]
    assert len(shares) >= 100 and max(shares) - min(shares) <= 2 * 16 + 8      # a cut moves by up to eight tiles of two; an item's constant, and a tile at either end
    plan, _ = case([1] * 32, [2000] * 32)
    shares = [c for c in schedule_is_whole(plan) if c]
    assert len(shares) >= 100 and max(shares) <= 1.15 * sum(shares) / len(shares) + 2 * 6 + 3


def _build(new, cached, pages, ids=None, blocks=4, num_pages=50, drafted=None, num_logits=None, T=12):
    from proxy_inference_engine_b200.ragged import StepPlan
    return StepPlan.build(ints(ids or list(range(T))), ints(new), ints(cached), pages if torch.is_tensor(pages) else ints(pages), num_pages=num_pages, max_blocks=blocks,
                          num_heads=8, num_kv_heads=2, draft_lengths=None if drafted is None else ints(drafted), num_logits=num_logits)


@pytest.mark.parametrize("text,kw", [
    ("negative", dict(new=[-1, 3], cached=[0, 0], pages=[1, 2])),
    ("negative", dict(new=[1, 3], cached=[-5, 0], pages=[1, 2])),
    ("longer than the step", dict(new=[13, 3], cached=[0, 0], pages=[1, 2])),
    ("longer than the step", dict(new=[1, 3], cached=[256, 0], pages=[1, 2, 3, 4, 5, 6])),
    ("longer than the step", dict(new=[2 ** 31 - 1, 3], cached=[2 ** 31 - 1, 0], pages=[1, 2])),
    ("more tokens than", dict(new=[9, 4], cached=[0, 0], pages=[1, 2])),
    ("more pages than", dict(new=[9, 3], cached=[60, 0], pages=[1, 2])),
    ("outside the pools", dict(new=[9, 3], cached=[0, 0], pages=[1, 50])),
    ("outside the pools", dict(new=[9, 3], cached=[0, 0], pages=[-1, 2])),
    ("not fewer than", dict(new=[9, 3], cached=[0, 0], pages=[1, 2], drafted=[0, 3])),
    ("not fewer than", dict(new=[9, 3], cached=[0, 0], pages=[1, 2], drafted=[-1, 0])),
    ("more logit rows", dict(new=[9, 3], cached=[0, 0], pages=[1, 2], drafted=[4, 2], num_logits=7)),
])
def test_what_does_not_fit_is_told_and_stays_in_bounds(text, kw):
    plan = _build(**kw)
    with pytest.raises(ValueError, match=text):
        plan.check()
    starts = plan.row_starts.tolist()
    assert starts == sorted(starts) and 0 <= starts[0] and starts[-1] <= 12
    assert all(-1 <= s < 50 * 64 for s in plan.slots.tolist()) and all(0 <= p < 50 for p in plan.block_table.flatten().tolist())
    assert all(0 <= r < 12 for r in plan.logit_rows.tolist()) and plan.logit_starts.tolist() == sorted(plan.logit_starts.tolist())
    assert plan.logit_starts.tolist()[-1] <= plan.dims.logit_rows
    schedule_is_whole(plan)


@pytest.mark.parametrize("rows", range(1, 9))
def test_logit_rows_that_do_not_fit_are_cut_off_at_the_end(rows):
    """What is left is what it would have been: a request's first drafts, judged in order, and none behind an unjudged one."""
    plan = _build([9, 3], [0, 0], [1, 2], drafted=[4, 2], num_logits=rows)
    assert plan.logit_rows.tolist() == [4, 5, 6, 7, 8, 9, 10, 11][:rows] and plan.logit_starts.tolist() == [0, min(rows, 5), rows if rows > 5 else min(rows, 5)]
    want = [5, 6, 7, 8, -1, 10, 11, -1][:rows]
    want[-1] = -1
    assert plan.draft_tokens.tolist() == want
    if rows < 8:
        with pytest.raises(ValueError, match="more logit rows"):
            plan.check()
    else:
        plan.check()


@pytest.mark.parametrize("new,drafted,rows,starts,tokens", [
    ([9, 4], [0, 2], [8, 10, 11], [0, 1, 3], [-1, 11, -1]),          # of 10, 11, 12: the last draft has no row
    ([9, 5], [0, 1], [8, 11], [0, 1, 2], [-1, -1]),                  # none of its drafts has
    ([9, 6], [3, 5], [5, 6, 7, 8, 9, 10, 11], [0, 4, 7], [6, 7, 8, -1, 10, 11, -1]),
])
def test_rows_that_do_not_fit_take_their_drafts_with_them(new, drafted, rows, starts, tokens):
    """What is left of a request judges the drafts that it would have, and no token that was not drafted."""
    plan = _build(new, [0, 0], [1, 2], drafted=drafted, num_logits=10)
    assert plan.logit_rows.tolist() == rows + [0] * (10 - len(rows)) and plan.logit_starts.tolist() == starts
    assert plan.draft_tokens.tolist() == tokens + [-1] * (10 - len(tokens)) and plan.row_starts.tolist() == [0, 9, 12]
    with pytest.raises(ValueError, match="more tokens than token_ids$"):
        plan.check()


def test_a_table_that_is_too_narrow():
    plan = _build([9, 3], [60, 0], ints([[1], [2]]))
    with pytest.raises(ValueError, match="more pages than"):
        plan.check()
    assert plan.slots.tolist()[:12] == [1 * 64 + 60, 1 * 64 + 61, 1 * 64 + 62, 1 * 64 + 63] + [-1] * 5 + [2 * 64, 2 * 64 + 1, 2 * 64 + 2]


def test_a_captured_plan_follows_its_lengths():
    from proxy_inference_engine_b200.ragged import StepPlan
    ids, new, cached, table = ints(list(range(40))), ints([1, 1, 1]), ints([5, 6, 7]), ints([[3, 4, 5], [6, 7, 8], [9, 10, 11]])
    build = lambda: StepPlan.build(ids, new, cached, table, num_pages=12, max_blocks=3, num_heads=8, num_kv_heads=2)
    build()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = build()
    for lens, ctx in (([1, 2, 3], [63, 64, 65]), ([0, 30, 10], [1, 150, 0]), ([1, 1, 1], [5, 6, 7])):
        new.copy_(ints(lens)), cached.copy_(ints(ctx))
        graph.replay()
        want = O.plan(list(range(40)), lens, ctx, table.tolist(), 3, T=40)
        agrees(plan, want)
        schedule_is_whole(plan)
