"""The operators of a ragged step beside its plan: rotation and cache write through the slot map, attention of every request's new tokens over its pages, drafted tokens
against the target's probabilities -- each against 64 bits, and all of them together."""
import math
import random

import pytest
import torch

import step_oracle as O

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
gen = lambda seed: torch.Generator(device="cuda").manual_seed(seed)
randn = lambda g, *s, std=1.0: (std * torch.randn(s, generator=g, device="cuda")).to(BF)
FREQS = lambda D: 500000.0 ** (torch.arange(0, D, 2, dtype=torch.float32, device="cuda") / D)


# ---------------------------------------------------------------------------------------------------- rotation and cache write
@pytest.mark.parametrize("D,Hq,Hkv,T,fused", [(64, 4, 2, 1, False), (128, 32, 8, 33, True), (64, 32, 8, 1030, True), (128, 5, 1, 7, False), (128, 64, 8, 1024, False)])
def test_rope_kv_slots(D, Hq, Hkv, T, fused):
    from proxy_inference_engine_b200 import ops
    g, n_pages = gen(T + D), T // 64 + 3
    if fused:
        q, k, v = (t.view(T, -1, D) for t in randn(g, T, (Hq + 2 * Hkv) * D).split([Hq * D, Hkv * D, Hkv * D], 1))
    else:
        q, k, v = randn(g, T, Hq, D), randn(g, T, Hkv, D), randn(g, T, Hkv, D)
    kp, vp = randn(g, n_pages, 64, Hkv, D), randn(g, n_pages, 64, Hkv, D)
    positions = torch.randint(0, 131072, (T,), generator=g, device="cuda").to(torch.int32)
    slots = torch.randperm(n_pages * 64, generator=g, device="cuda")[:T].to(torch.int32)
    positions[0], slots[T // 2] = 0, n_pages * 64 - 1 if (n_pages * 64 - 1) not in slots.tolist() else slots[T // 2]
    dead = [T - 1] if T > 2 else []
    if dead:
        slots[T - 1] = -1
        if T > 20:
            slots[11], dead = n_pages * 64, dead + [11]
    live = [t for t in range(T) if t not in dead]
    was_k, was_v = kp.clone(), vp.clone()
    got = ops.rope_kv_slots(q, k, v, FREQS(D), positions, slots, kp, vp)
    # half a step of bf16, and 3e-6 of sine and cosine (2 pi in two pieces, the approximation unit) and two fp32 products on either feature
    near = lambda got, x, want: bool(((got.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 4e-6 * x.cpu().double().abs().sum(-1, keepdim=True)).all())
    assert near(got[live], q[live], O.rope(q, positions, FREQS(D))[live]) and not got[dead].any()
    at = slots[live].long()
    assert near(kp.view(-1, Hkv, D)[at], k[live], O.rope(k, positions, FREQS(D))[live]) and torch.equal(vp.view(-1, Hkv, D)[at], v[live])
    rest = torch.ones(n_pages * 64, dtype=torch.bool, device="cuda")
    rest[at] = False
    for pool, was in ((kp, was_k), (vp, was_v)):
        assert torch.equal(pool.view(-1, Hkv, D)[rest], was.view(-1, Hkv, D)[rest])
    out = torch.full_like(got, 7.0)
    assert ops.rope_kv_slots(q, k, v, FREQS(D), positions, slots, kp, vp, out=out) is out
    assert torch.equal(out[live], got[live]) and bool((out[dead] == 7.0).all())


def test_rope_kv_slots_is_rope_kv_append():
    """Bit for bit, through a table of pages of one row each."""
    import ctypes as C
    from proxy_inference_engine_b200 import _lib, ops
    g, T, Hq, Hkv, D = gen(5), 37, 8, 2, 128
    qkv = randn(g, T, (Hq + 2 * Hkv) * D)
    positions = torch.randint(0, 4096, (T,), generator=g, device="cuda").to(torch.int32)
    table = torch.randint(0, 1, (T, 64), device="cuda", dtype=torch.int32)
    pages = torch.randperm(64, generator=g, device="cuda")[:T].to(torch.int32)
    table[torch.arange(T), (positions // 64).long()] = pages
    pools = [torch.zeros((64, 64, Hkv, D), dtype=BF, device="cuda") for _ in range(4)]
    q = torch.empty((T, Hq, D), dtype=BF, device="cuda")
    lay = ops.kv_layout(pools[0], table, 64)
    _lib.check(_lib.load().pie_rope_kv_append(q.data_ptr(), qkv.data_ptr(), pools[0].data_ptr(), pools[1].data_ptr(), C.byref(lay), positions.data_ptr(), FREQS(D).data_ptr(), T,
                                              Hq, Hkv, D, ops._stream()), "rope_kv_append")
    parts = (t.view(T, -1, D) for t in qkv.split([Hq * D, Hkv * D, Hkv * D], 1))
    got = ops.rope_kv_slots(*parts, FREQS(D), positions, pages * 64 + positions % 64, pools[2], pools[3])
    assert torch.equal(got, q) and torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])


# ---------------------------------------------------------------------------------------------------- attention
def attention_case(new, cached, Hq, Hkv, D, seed=0, pad=0, std=2.0, strided=False):
    """A plan and random queries over pools whose unused places hold NaN."""
    from proxy_inference_engine_b200.ragged import StepPlan
    rng, g = random.Random(seed), gen(seed)
    counts = [O.need(n, c) for n, c in zip(new, cached)]
    n_pages, T = sum(counts) + 2, sum(new) + pad
    order = rng.sample(range(n_pages), sum(counts))
    tables = [[order.pop() for _ in range(k)] for k in counts]
    plan = StepPlan.build(ints([0] * T), ints(new), ints(cached), ints([p for t in tables for p in t]), num_pages=n_pages, max_blocks=max(1, *counts), num_heads=Hq,
                          num_kv_heads=Hkv)
    k, v = randn(g, n_pages, 64, Hkv, D), randn(g, n_pages, 64, Hkv, D)
    used = torch.zeros(n_pages * 64, dtype=torch.bool)
    for n, c, t in zip(new, cached, tables):
        for i, p in enumerate(t):
            used[p * 64:p * 64 + max(0, min(64, n + c - 64 * i))] = True
    k.view(-1, Hkv, D)[~used.cuda()] = torch.nan
    v.view(-1, Hkv, D)[~used.cuda()] = torch.nan
    q = randn(g, T, Hq + (3 if strided else 0), D, std=std)[:, :Hq]
    return plan, q, k, v, tables


def attention_holds(got, q, k, v, new, cached, tables, scale):
    """A weight in [0, 1] is rounded to bf16 at most once (2^-8 of it), the result once; scores are sums of D products in fp32 (2^-24 D of the sum of
    |q k| scale, up to 2^-13 here, and so for the weights and for their sum), exponentials are off by a few 2^-22."""
    want, weight = O.attention(q, k, v, new, cached, tables, scale)
    T = sum(new)
    got = got.view(got.shape[0], *q.shape[1:]).cpu().double()
    off = (got[:T] - want[:T]).abs() - (2.0 ** -8 * want[:T].abs() + (2.0 ** -8 + 2.0 ** -12) * weight[:T])
    assert bool((off <= 0).all()), float(off.max())     # (a NaN is not below)


SHAPES = [
    ([1], [0]), ([1], [63]), ([1], [64]), ([1], [127]), ([1], [128]), ([2], [255]), ([5], [700]), ([64], [0]), ([65], [0]), ([33], [100]), ([130], [0]), ([300], [77]),
    ([1, 1, 1, 1], [0, 1, 300, 5000]), ([0, 3, 0, 70, 1, 0], [5, 60, 0, 1, 128, 0]), ([1, 6, 200, 1], [1000, 63, 300, 0]), ([700, 2], [513, 9000]),
]


@pytest.mark.parametrize("Hq,Hkv,D", [(4, 2, 64), (8, 2, 128), (32, 8, 128)])
@pytest.mark.parametrize("new,cached", SHAPES)
def test_chunk_attention(new, cached, Hq, Hkv, D):
    from proxy_inference_engine_b200 import ops
    plan, q, k, v, tables = attention_case(new, cached, Hq, Hkv, D, seed=len(new) + sum(new), strided=len(new) % 2 == 1)
    plan.check()
    got = ops.chunk_attention(q, k, v, plan, D ** -0.5)
    attention_holds(got, q, k, v, new, cached, tables, D ** -0.5)
    assert torch.equal(got, ops.chunk_attention(q, k, v, plan, D ** -0.5))      # whichever CTA comes last
    ops.check_pipeline()


@pytest.mark.parametrize("Hq,Hkv,D", [(1, 1, 64), (3, 1, 128), (24, 8, 64), (64, 8, 128), (7, 1, 64), (40, 1, 128), (128, 1, 64), (16, 16, 128)])
def test_chunk_attention_of_other_heads(Hq, Hkv, D):
    from proxy_inference_engine_b200 import ops
    # (long ones of two, three and more query tiles: items that are cut between key tiles)
    for new, cached in (([1, 45, 9, 4], [900, 30, 250, 2000]), ([3, 7, 40, 140 * Hkv // Hq + 1], [5000, 6001, 4000, 9000])):
        plan, q, k, v, tables = attention_case(new, cached, Hq, Hkv, D, seed=Hq)
        attention_holds(ops.chunk_attention(q, k, v, plan, D ** -0.5), q, k, v, new, cached, tables, D ** -0.5)
        ops.check_pipeline()


@pytest.mark.parametrize("seed", range(24))
def test_steps_of_all_kinds_of_requests(seed):
    """Single tokens, drafts, portions of every size and requests that sit the step out, in any order: a CTA turns from one kind of item to another."""
    from proxy_inference_engine_b200 import ops
    rng = random.Random(seed)
    D, Hkv, G = rng.choice([64, 128]), rng.choice([1, 2, 4]), rng.choice([1, 2, 3, 4, 8, 16])
    kinds = [lambda: 1, lambda: rng.randint(1, 8), lambda: rng.randint(9, 70), lambda: rng.randint(60, 300), lambda: 0]
    new = [rng.choice(kinds)() for _ in range(rng.randint(2, 14))] + [1]
    cached = [rng.choice([0, rng.randint(0, 200), rng.randint(0, 2500)]) for _ in new]
    plan, q, k, v, tables = attention_case(new, cached, Hkv * G, Hkv, D, seed=seed, pad=seed % 3, std=rng.choice([0.5, 2.0, 3.0]))
    got = ops.chunk_attention(q, k, v, plan, D ** -0.5)
    attention_holds(got, q, k, v, new, cached, tables, D ** -0.5)
    assert torch.equal(got, ops.chunk_attention(q, k, v, plan, D ** -0.5)) and not got[sum(new):].any()
    ops.check_pipeline()


@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 64), (8, 2, 128), (16, 2, 128), (3, 1, 64), (16, 1, 64), (48, 1, 128)])
@pytest.mark.parametrize("long", [False, True])
def test_an_answers_weights_hold_16_bits(Hq, Hkv, D, long):
    """Up to 64 rows (tokens x query heads of a key / value head; 48 at head size 128) have what a decode step's attention has: weights rounded to bf16 and what that
    leaves rounded again, 2^-16 of them, so that an answer does not depend on which of the two it is given."""
    from proxy_inference_engine_b200 import ops
    most = (64 if D == 64 else 48) * Hkv // Hq
    new = sorted({1, 1 + most // 3, most // 2 + 1, most})
    for cached in ([(9000, 4000, 63, 700)[i] if long else (0, 9, 64, 200)[i] for i in range(len(new))], [3000 if long else 30] * len(new)):
        plan, q, k, v, tables = attention_case(new, cached, Hq, Hkv, D, seed=Hq + D, std=0.7)
        got = ops.chunk_attention(q, k, v, plan, D ** -0.5)
        want, weight = O.attention(q, k, v, new, cached, tables, D ** -0.5)
        off = (got.view(want.shape).cpu().double() - want).abs() - (2.0 ** -8 * want.abs() + (2.0 ** -16 + 2.0 ** -12) * weight)      # (attention_holds', with 2^-16 for the weights)
        assert bool((off <= 0).all()), float(off.max())
        ops.check_pipeline()


@pytest.mark.parametrize("std", [0.0, 30.0])
def test_chunk_attention_of_flat_and_of_steep_scores(std):
    """All keys alike, and one key that takes all: the running maximum moves by hundreds."""
    from proxy_inference_engine_b200 import ops
    new, cached = [3, 140], [1000, 600]
    plan, q, k, v, tables = attention_case(new, cached, 8, 2, 128, seed=9, std=std)
    want, weight = O.attention(q, k, v, new, cached, tables, 128 ** -0.5)
    got = ops.chunk_attention(q, k, v, plan, 128 ** -0.5).view(want.shape).cpu().double()
    # scores of up to 30 * 4 * 128^0.5 = 1400: 1400 * 128 * 2^-24 = 0.011 in the exponent at the worst, on either side of a quotient
    assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + (0.022 if std else 2.0 ** -12)) * weight).all())
    ops.check_pipeline()


def test_rows_that_belong_to_nobody():
    from proxy_inference_engine_b200 import ops
    new, cached = [2, 0, 150], [70, 3, 0]
    plan, q, k, v, tables = attention_case(new, cached, 8, 2, 64, seed=4, pad=70)
    got = ops.chunk_attention(q, k, v, plan, 0.125)
    attention_holds(got, q, k, v, new, cached, tables, 0.125)
    assert not got[152:].any()
    out = torch.full((222, 512), 3.0, dtype=BF, device="cuda")
    assert ops.chunk_attention(q, k, v, plan, 0.125, out=out) is out
    assert torch.equal(out[:152], got[:152]) and bool((out[152:] == 3.0).all())
    nobody, q, k, v, _ = attention_case([0, 0], [5, 70], 8, 2, 64, pad=9)
    assert not ops.chunk_attention(q, k, v, nobody, 0.125).any()


def test_a_page_shared_by_two_requests():
    from proxy_inference_engine_b200 import ops
    from proxy_inference_engine_b200.ragged import StepPlan
    g = gen(8)
    k, v, q = randn(g, 5, 64, 2, 64), randn(g, 5, 64, 2, 64), randn(g, 21, 4, 64)
    tables, new, cached = [[2, 0], [2, 4]], [1, 20], [100, 64]
    plan = StepPlan.build(ints([0] * 21), ints(new), ints(cached), ints(tables), num_pages=5, max_blocks=2, num_heads=4, num_kv_heads=2)
    attention_holds(ops.chunk_attention(q, k, v, plan, 0.2), q, k, v, new, cached, tables, 0.2)


def test_pools_inside_larger_ones():
    """Keys and values beside each other in one allocation, heads apart."""
    from proxy_inference_engine_b200 import ops
    new, cached = [3, 90], [300, 40]
    plan, q, k, v, tables = attention_case(new, cached, 8, 2, 128, seed=6)
    both = torch.full((k.shape[0], 64, 5, 128), torch.nan, dtype=BF, device="cuda")
    both[:, :, 0:2], both[:, :, 2:4] = k, v
    assert torch.equal(ops.chunk_attention(q, both[:, :, 0:2], both[:, :, 2:4], plan, 0.1), ops.chunk_attention(q, k, v, plan, 0.1))


def test_rows_and_heads_that_lie_anywhere():
    """Queries, keys and values with heads outside rows, pools with heads outside pages."""
    from proxy_inference_engine_b200 import ops
    for D in (64, 128):
        new, cached, Hq, Hkv = [3, 90, 17], [300, 40, 0], 8, 2
        plan, q, k, v, tables = attention_case(new, cached, Hq, Hkv, D, seed=D)
        outside = lambda x, *order: x.permute(*order).contiguous().permute(*[order.index(i) for i in range(x.dim())])
        oq, ok, ov = outside(q, 1, 0, 2), outside(k, 2, 0, 1, 3), outside(v, 2, 0, 1, 3)
        assert oq.stride(1) > oq.stride(0) and ok.stride(2) > ok.stride(0)
        want = ops.chunk_attention(q, k, v, plan, D ** -0.5)
        attention_holds(want, q, k, v, new, cached, tables, D ** -0.5)
        assert torch.equal(ops.chunk_attention(oq, ok, ov, plan, D ** -0.5), want)
        g = gen(D)
        nk, nv = randn(g, 110, Hkv, D), randn(g, 110, Hkv, D)
        turned = ops.rope_kv_slots(q, nk, nv, FREQS(D), plan.positions, plan.slots, k, v)
        assert torch.equal(ops.rope_kv_slots(oq, outside(nk, 1, 0, 2), outside(nv, 1, 0, 2), FREQS(D), plan.positions, plan.slots, ok, ov), turned)
        assert torch.equal(ok.view(torch.int16), k.view(torch.int16)) and torch.equal(ov.view(torch.int16), v.view(torch.int16))
        ops.check_pipeline()


@pytest.mark.parametrize("D", [64, 128])
def test_more_pieces_than_a_cta_holds_at_once(D):
    """Seven hundred requests, a portion of a prompt among every few: some CTAs have more than 32 pieces, of all kinds."""
    from proxy_inference_engine_b200 import ops
    rng, Hkv = random.Random(D), 8
    new = [rng.choice([1, 1, 1, 1, 1, 1, 1, 2, 5, 70, 130, 300]) if s % 5 == 0 else 1 for s in range(700)]
    cached = [rng.choice([0, 1, 63, 64, 100, 127, 128]) for _ in new]
    plan, q, k, v, tables = attention_case(new, cached, Hkv, Hkv, D, seed=D)
    plan.check()
    at = plan.status.storage_offset() + 192
    ranges = plan.words[at:at + 384].view(192, 2)
    assert int((ranges[:, 1] - ranges[:, 0]).max()) > 34
    got = ops.chunk_attention(q, k, v, plan, D ** -0.5)
    attention_holds(got, q, k, v, new, cached, tables, D ** -0.5)
    assert torch.equal(got, ops.chunk_attention(q, k, v, plan, D ** -0.5))
    ops.check_pipeline()


def test_attention_on_two_streams_at_once():
    from proxy_inference_engine_b200 import ops
    cases = [attention_case([4, 1], [6000, 3000], 8, 2, 128, seed=s) for s in (1, 2)]
    want = [ops.chunk_attention(q, k, v, plan, 0.1) for plan, q, k, v, _ in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(20):
        for i, (stream, (plan, q, k, v, _)) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(stream):
                got[i].append(ops.chunk_attention(q, k, v, plan, 0.1))
    torch.cuda.synchronize()
    for mine, w in zip(got, want):
        assert all(torch.equal(x, w) for x in mine)


def test_what_other_requests_and_later_keys_hold_does_not_matter():
    """NaN and infinities in one request's keys and values stay its own, and in the keys of later new tokens they are masked."""
    from proxy_inference_engine_b200 import ops
    for new, cached in (([3, 40, 1], [200, 100, 300]), ([200, 300, 5], [0, 70, 10])):
        plan, q, k, v, tables = attention_case(new, cached, 8, 2, 128, seed=13)
        want = ops.chunk_attention(q, k, v, plan, 0.1)
        k2, v2 = k.clone(), v.clone()
        k2[tables[1]], v2[tables[1]] = torch.inf, torch.nan
        got = ops.chunk_attention(q, k2, v2, plan, 0.1)
        rest = list(range(new[0])) + list(range(new[0] + new[1], sum(new)))
        assert torch.equal(got[rest], want[rest]) and bool(torch.isnan(got[new[0]:new[0] + new[1]]).all())
        k2, last = k.clone(), cached[1] + new[1] - 1
        k2[tables[1][last // 64], last % 64] = torch.nan
        got = ops.chunk_attention(q, k2, v, plan, 0.1)
        but = [t for t in range(sum(new)) if t != new[0] + new[1] - 1]
        assert torch.equal(got[but], want[but]) and bool(torch.isnan(got[new[0] + new[1] - 1]).all())


def test_pages_behind_the_32_bit_offsets():
    """Pools of 2.6e9 elements: pages at either end."""
    from proxy_inference_engine_b200 import ops
    from proxy_inference_engine_b200.ragged import StepPlan
    g, n_pages, Hq, Hkv, D = gen(21), 40000, 32, 8, 128
    k_pool, v_pool = (torch.empty((n_pages, 64, Hkv, D), dtype=BF, device="cuda") for _ in range(2))
    tables, new, cached = [[39999, 3, 39990], [35000, 39998]], [5, 70], [130, 20]
    for t in tables:
        k_pool[t], v_pool[t] = randn(g, len(t), 64, Hkv, D), randn(g, len(t), 64, Hkv, D)
    plan = StepPlan.build(ints([0] * 75), ints(new), ints(cached), ints(sum(tables, [])), num_pages=n_pages, max_blocks=3, num_heads=Hq, num_kv_heads=Hkv)
    plan.check()
    q, k, v = randn(g, 75, Hq, D, std=2.0), randn(g, 75, Hkv, D), randn(g, 75, Hkv, D)
    turned = ops.rope_kv_slots(q, k, v, FREQS(D), plan.positions, plan.slots, k_pool, v_pool)
    at = plan.slots.long()
    assert torch.equal(v_pool.view(-1, Hkv, D)[at], v) and int(at.max()) * Hkv * D > 2 ** 31
    some = sorted(set(sum(tables, [])))
    small = [[some.index(p) for p in t] for t in tables]
    attention_holds(ops.chunk_attention(turned, k_pool, v_pool, plan, 0.1), turned, k_pool[some], v_pool[some], new, cached, small, 0.1)


def test_two_captured_graphs_at_once():
    """... of calls whose items are cut: neither counts in the other's workspace, nor in an eager call's."""
    from proxy_inference_engine_b200 import ops
    cases = [attention_case([4, 1], [6000, 3000], 8, 2, 128, seed=s) for s in (3, 4)]
    drafts = [verify_case([3, 4], 5000, 0.7, True, seed=s)[0] for s in (5, 6)]

    def run(i):
        plan, q, k, v, _ = cases[i]
        kw = dict(drafts[i])
        return (ops.chunk_attention(q, k, v, plan, 0.1), *ops.verify_draft(kw.pop("logits"), kw.pop("draft_tokens"), kw.pop("logit_starts"), max_draft=4, **kw))
    want = [run(0), run(1)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run(i))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        eager = run(0)
    torch.cuda.synchronize()
    for got, w in ((outs[0], want[0]), (outs[1], want[1]), (eager, want[0])):
        assert all(torch.equal(a, b) for a, b in zip(got, w))


# ---------------------------------------------------------------------------------------------------- verification
def verify_case(drafted, V, temp, model, seed=0, ld=None):
    g = gen(seed)
    starts = [0]
    for k in drafted:
        starts.append(starts[-1] + (k + 1 if k >= 0 else 0))      # -1: a request without rows
    R = max(1, starts[-1])
    logits = 2.5 * torch.randn((R, V), generator=g, device="cuda")
    logits.scatter_add_(1, torch.randint(0, V, (R, 1), generator=g, device="cuda"), 12 * torch.rand((R, 1), generator=g, device="cuda"))
    guess = (logits + 0.8 * torch.randn((R, V), generator=g, device="cuda")).to(BF) if model else None
    tokens = (guess.float() / temp).softmax(1).multinomial(1, generator=g)[:, 0] if model else torch.where(
        torch.rand(R, generator=g, device="cuda") < 0.8, logits.argmax(1), torch.randint(0, V, (R,), generator=g, device="cuda"))
    logits = logits.to(BF)
    if ld:
        wide = [None if t is None else torch.full((R, ld), 99.0, dtype=BF, device="cuda") for t in (logits, guess)]
        wide[0][:, :V] = logits
        if model:
            wide[1][:, :V] = guess
        logits, guess = wide[0][:, :V], None if guess is None else wide[1][:, :V]
    return dict(logits=logits, draft_tokens=tokens.to(torch.int32), logit_starts=ints(starts), temp=temp, draft_logits=guess,
                uniforms=torch.rand(R, generator=g, device="cuda") if temp else None, noise=torch.rand((len(drafted), V), generator=g, device="cuda") if temp else None), starts


def verified(kw, starts, most):
    from proxy_inference_engine_b200 import ops
    tokens, counts, logprobs = ops.verify_draft(kw["logits"], kw["draft_tokens"], kw["logit_starts"], max_draft=most, temp=kw["temp"], uniforms=kw["uniforms"], noise=kw["noise"],
                                                draft_logits=kw["draft_logits"])
    want = O.verify(kw["logits"], kw["draft_tokens"], starts, most, kw["temp"], kw["uniforms"], kw["noise"], kw["draft_logits"])
    tokens, counts, logprobs = tokens.tolist(), counts.tolist(), logprobs.tolist()
    # a logarithm of a sum of exponentials that are each off by 2^-21 or so, of arguments rounded in fp32, and a difference
    off = 4e-6 + 2.0 ** -22 * float(kw["logits"].float().nan_to_num(0, 0, 0).abs().max()) / (kw["temp"] or 1.0)
    surely = 0
    for t, c, lp, (wt, wlp, sure) in zip(tokens, counts, logprobs, want):
        assert t[c:] == [-1] * (most + 1 - c) and lp[c:] == [0.0] * (most + 1 - c)
        if sure:
            surely += 1
            assert t[:c] == wt and all(abs(a - b) <= off for a, b in zip(lp, wlp))
    assert surely >= 0.9 * len(want)
    return counts


@pytest.mark.parametrize("V,ld", [(640, None), (50257, None), (128256, None), (1001, 1016), (8, None), (1, None)])
@pytest.mark.parametrize("temp,model", [(0.0, False), (0.7, False), (1.0, True), (0.3, True)])
def test_verify_draft(V, ld, temp, model):
    drafted = [4, 0, 7, -1, 1, 2, 5, 7, 3]
    kw, starts = verify_case(drafted, V, temp, model, seed=V, ld=ld)
    counts = verified(kw, starts, 7)
    assert counts[3] == 0 and all(1 <= c <= k + 1 for c, k in zip(counts, drafted) if k >= 0)
    verified(kw, starts, 2)      # further drafts are not looked at


@pytest.mark.parametrize("S,K", [(1, 4), (1, 127), (300, 1), (64, 5)])
def test_verify_of_few_and_of_many(S, K):
    rng = random.Random(S)
    kw, starts = verify_case([K if S == 1 else rng.randint(0, K) for _ in range(S)], 4001, 0.9, True, seed=S)
    if S == 1 and K == 127:      # all of them accepted but the last: a draw below every quotient
        kw["uniforms"].zero_()
        kw["uniforms"][126] = 1.0 - 2.0 ** -24
    verified(kw, starts, K)


def test_the_same_draft_is_always_accepted():
    kw, starts = verify_case([5] * 8, 3001, 1.0, True, seed=3)
    kw["draft_logits"] = kw["logits"].clone()
    kw["uniforms"].fill_(1.0 - 2.0 ** -24)
    # q(x) u < p(x) with q = p in the same bits
    from proxy_inference_engine_b200 import ops
    counts = ops.verify_draft(kw["logits"], kw["draft_tokens"], kw["logit_starts"], max_draft=5, temp=1.0, uniforms=kw["uniforms"], noise=kw["noise"],
                              draft_logits=kw["draft_logits"])[1]
    assert counts.tolist() == [6] * 8


@pytest.mark.parametrize("temp,model", [(0.0, False), (0.8, False), (1.0, True)])
def test_rows_behind_the_last_request_judge_nothing(temp, model):
    """A captured step's room for logit rows is an upper bound: what the rows have that belong to nobody does not matter, NaN included, nor what lies there at a replay."""
    from proxy_inference_engine_b200 import ops
    drafted, V, room = [4, 0, 7, -1, 2], 128256, 68
    kw, starts = verify_case(drafted, V, temp, model, seed=51)
    live = starts[-1]
    kw["draft_tokens"][live - 1] = -1
    want = ops.verify_draft(max_draft=7, **kw)
    wide = dict(kw)
    for name in ("logits", "draft_logits", "uniforms"):
        if kw[name] is not None:
            wide[name] = torch.full((room, *kw[name].shape[1:]), torch.nan, dtype=kw[name].dtype, device="cuda")
            wide[name][:live] = kw[name]
    wide["draft_tokens"] = torch.full((room,), -1, dtype=torch.int32, device="cuda")
    wide["draft_tokens"][:live] = kw["draft_tokens"]
    bits = lambda got: [t.view(torch.int32) for t in got]
    assert all(torch.equal(a, b) for a, b in zip(bits(ops.verify_draft(max_draft=7, **wide)), bits(want)))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.verify_draft(max_draft=7, **wide)
    for fill, token in ((torch.nan, -1), (torch.inf, V - 1), (0.0, 1 << 30)):
        wide["logits"][live:], wide["draft_tokens"][live:] = fill, token
        for t in got:
            t.zero_()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(bits(got), bits(want)))


def test_ties_go_to_the_first():
    from proxy_inference_engine_b200 import ops
    logits = torch.zeros((4, 5000), dtype=BF, device="cuda")
    logits[:, 3000] = logits[:, 777] = 2.0
    logits[1, 10], logits[2] = -0.0, -torch.inf
    logits[2, 9], logits[2, 5], logits[3], logits[3, 40] = 0.0, -0.0, -1.0, -0.0
    got = ops.verify_draft(logits, ints([777, 777, 5, 0]), ints([0, 4]), max_draft=3)
    assert got[0].tolist() == [[777, 777, 5, 40]] and got[1].tolist() == [4]


def test_filters_and_rows_without_a_distribution():
    from proxy_inference_engine_b200 import ops
    V, inf = 3000, float("inf")
    kw, starts = verify_case([2] * 6, V, 0.8, True, seed=12)
    for t in (kw["logits"], kw["draft_logits"]):
        keep = torch.rand(t.shape, generator=gen(5), device="cuda") < 0.01
        keep[:, 17] = True
        t[~keep] = -inf                                       # a filter's work: the drafted token may be one that cannot be
    verified(kw, starts, 2)
    kw["logits"][0, 5], kw["logits"][3, 6], kw["logits"][6], kw["draft_logits"][9, 3] = float("nan"), inf, -inf, float("nan")
    kw["logits"][12:15] = -inf
    kw["logits"][12:15, 17] = 1.0                              # all of it on one token
    kw["draft_tokens"][12:15] = 17
    tokens, counts, logprobs = ops.verify_draft(kw["logits"], kw["draft_tokens"], kw["logit_starts"], max_draft=2, temp=0.8, uniforms=kw["uniforms"], noise=kw["noise"],
                                                draft_logits=kw["draft_logits"])
    tokens = tokens.tolist()
    assert counts.tolist()[:4] == [1, 1, 1, 1] and [t[0] for t in tokens[:3]] == [0, 0, 0] and tokens[4] == [17, 17, 17]
    assert all(0 <= x < V for x in tokens[3][:1]) and float(kw["logits"][9, tokens[3][0]]) > -inf
    assert torch.isnan(logprobs[0, 0]) and logprobs[4].tolist() == [0.0, 0.0, 0.0]
    greedy = torch.full((2, 64), -inf, dtype=BF, device="cuda")
    greedy[0, 3], greedy[0, 7] = float("nan"), 2.0
    assert ops.verify_draft(greedy, ints([7, 0]), ints([0, 2]), max_draft=1)[0].tolist() == [[7, 0]]


@pytest.mark.parametrize("model", [False, True])
def test_filters_of_the_lowest_value(model):
    """A filter that writes the type's lowest value leaves what one that writes -inf does, bit for bit; a row of nothing else is flat."""
    from proxy_inference_engine_b200 import ops
    V, low = 40000, torch.finfo(BF).min
    kw, starts = verify_case([3] * 8, V, 0.8, model, seed=21)
    keep = torch.rand(V, generator=gen(6), device="cuda") < 0.001
    keep[:100], keep[39000:] = False, False
    results = []
    for masked in (-torch.inf, low):
        given = {n: torch.where(keep, kw[n], torch.tensor(masked, dtype=BF, device="cuda")) for n in ("logits", "draft_logits") if kw[n] is not None}
        results.append(ops.verify_draft(max_draft=3, **{**kw, **given}))
    for a, b in zip(*results):
        assert torch.equal(a, b) and not bool(torch.isnan(a).any())
    assert bool(keep[results[0][0][results[0][0] >= 0].long()].all())
    kw["logits"].fill_(low)
    kw["uniforms"].fill_(1.0 - 2.0 ** -24)
    tokens, counts, logprobs = ops.verify_draft(max_draft=3, **kw)
    assert bool(((logprobs[:, 0] + math.log(V)).abs() <= 4e-6).all())
    if not model:   # every other token is as likely, so that the largest draw has it
        noise = kw["noise"].clone().scatter_(1, kw["draft_tokens"].view(8, 4)[:, :1].long(), 0.0)
        assert counts.tolist() == [1] * 8 and tokens[:, 0].tolist() == noise.argmax(1).tolist()


@pytest.mark.parametrize("temp,factor", [(1e-3, 1.0), (1e-8, 1.0), (1e-30, 1.0), (1e-42, 1.0), (1.0, 1e4), (1.0, 1e30), (0.7, 1e37)])
@pytest.mark.parametrize("model", [False, True])
def test_temperatures_near_0_and_logits_of_any_size_are_greedy(temp, factor, model):
    """One logit of each row is larger than the others by 2^-3 of itself at least: p is 1 there."""
    from proxy_inference_engine_b200 import ops
    kw, starts = verify_case([5] * 8, 9001, 1.0, model, seed=31)
    R = kw["logits"].shape[0]
    best = torch.randint(0, 9001, (R,), generator=gen(32), device="cuda")
    x = kw["logits"].float().clamp(-8, 8).scatter(1, best[:, None], 10.0)
    kw["logits"] = (x * factor).to(BF)
    kw["draft_tokens"] = torch.where(torch.rand(R, generator=gen(33), device="cuda") < 0.6, best, (best + 1) % 9001).to(torch.int32)
    if model:
        kw["draft_logits"] = (x.scatter(1, kw["draft_tokens"][:, None].long(), 13.0) * factor).to(BF)
    kw["temp"] = temp
    got = ops.verify_draft(max_draft=5, **kw)
    want = ops.verify_draft(kw["logits"], kw["draft_tokens"], kw["logit_starts"], max_draft=5)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert 0 < int((want[1] > 1).sum()) and bool((got[2] == 0).all())


@pytest.mark.parametrize("model", [False, True])
@pytest.mark.parametrize("native", [True, False])
def test_a_temperature_that_32_bits_do_not_hold_is_none_of_0(model, native, monkeypatch):
    """It is a draw at the lowest temperature there is, log-probabilities included, and not a greedy answer, whose log-probabilities are the model's own."""
    from proxy_inference_engine_b200 import ops
    if not native:
        monkeypatch.setattr(ops, "native_host", lambda: ops._NoHost)
    kw, _ = verify_case([5] * 4, 9001, 1.0, model, seed=41)
    want = ops.verify_draft(max_draft=5, **{**kw, "temp": 1e-42})
    for temp in (1e-50, 5e-324):
        assert all(torch.equal(a, b) for a, b in zip(ops.verify_draft(max_draft=5, **{**kw, "temp": temp}), want))


def test_tokens_outside_the_vocabulary_and_starts_outside_the_rows():
    from proxy_inference_engine_b200 import ops
    kw, starts = verify_case([2, 2, 2], 900, 0.8, False, seed=2)
    kw["draft_tokens"][0], kw["draft_tokens"][3], kw["uniforms"][:] = -1, 900, 0.0
    got = ops.verify_draft(kw["logits"], kw["draft_tokens"], kw["logit_starts"], max_draft=2, temp=0.8, uniforms=kw["uniforms"], noise=kw["noise"])
    assert got[1].tolist()[:2] == [1, 1] and got[1].tolist()[2] >= 1
    for bad in ([-5, 2, 100, 7], [9, 3, 3, 9], [0, 1 << 30, -(1 << 30), 2]):
        tokens, counts, _ = ops.verify_draft(kw["logits"], kw["draft_tokens"], ints(bad), max_draft=2, temp=0.8, uniforms=kw["uniforms"], noise=kw["noise"])
        assert all(0 <= c <= 3 for c in counts.tolist())


def test_one_workspace_for_calls_of_all_shapes():
    """What a call leaves in it does not reach the next one, whose counters lie where others' sums did; nor does what was there before the first."""
    from proxy_inference_engine_b200 import _lib, ops
    L, V = _lib.load(), 50000
    ptr = lambda t: None if t is None else t.data_ptr()

    def call(kw, S, R, ws):
        out = torch.full((S, 2), -7, dtype=torch.int32, device="cuda"), torch.full((S,), -7, dtype=torch.int32, device="cuda"), torch.full((S, 2), 9.0, device="cuda")
        _lib.check(L.pie_verify_draft(*map(ptr, out), ptr(kw["logits"]), ptr(kw["draft_logits"]), V, ptr(kw["draft_tokens"]), ptr(kw["logit_starts"]), S, R, V, 1, kw["temp"],
                                      ptr(kw["uniforms"]), ptr(kw["noise"]), ptr(ws), ws.numel(), ops._stream()), "verify_draft")
        return out
    most = L.pie_verify_workspace_bytes(300, 600, V)
    shared = torch.full((most,), 0x5A, dtype=torch.uint8, device="cuda")
    for S in (64, 65, 300, 1, 65):
        kw, _ = verify_case([1] * S, V, 0.8, True, seed=S)
        got, want = call(kw, S, 2 * S, shared), call(kw, S, 2 * S, torch.zeros_like(shared))
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and bool((got[1] > 0).all())
        assert all(torch.equal(a, b) for a, b in zip(got, ops.verify_draft(max_draft=1, **kw)))


def test_starts_that_do_not_rise_meet_no_other_calls_sums():
    """A row that is one request's last and lies within another: what a call before this one left of its draft's logits does not matter."""
    from proxy_inference_engine_b200 import ops
    kw, _ = verify_case([5], 9000, 0.8, True, seed=1)
    kw["logit_starts"], kw["noise"], kw["uniforms"] = ints([0, 3, 2, 6]), torch.rand((3, 9000), generator=gen(2), device="cuda"), torch.full((6,), 0.5, device="cuda")
    results = []
    for level in (0.0, 40.0):
        other, _ = verify_case([5], 9000, 0.8, True, seed=2)
        other["logit_starts"], other["noise"] = ints([0, 1, 2, 6]), torch.rand((3, 9000), generator=gen(3), device="cuda")
        other["draft_logits"].fill_(level)
        ops.verify_draft(max_draft=5, **other)
        results.append(ops.verify_draft(max_draft=5, **kw))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    assert results[0][1].tolist()[1:] == [0, 1]      # (and refuses its token)


def test_draws_follow_the_target():
    """Drafts from q, verified against p: the first token behind them is distributed as p.  4000 draws of 6 tokens: five standard deviations."""
    from proxy_inference_engine_b200 import ops
    S, V, g = 4000, 6, gen(77)
    p, q = torch.tensor([2.0, 1.0, 0.0, 0.5, -1.0, 1.5], device="cuda"), torch.tensor([0.0, 2.0, 1.0, 0.5, 0.0, -2.0], device="cuda")
    logits, guess = p.to(BF).expand(2 * S, V).contiguous(), q.to(BF).expand(2 * S, V).contiguous()
    drafted = guess[0].float().softmax(0).multinomial(2 * S, replacement=True, generator=g).to(torch.int32)
    for draft_logits, given in ((guess, drafted), (None, torch.full_like(drafted, 1))):
        tokens, counts, _ = ops.verify_draft(logits, given, torch.arange(0, 2 * S + 1, 2, device="cuda", dtype=torch.int32), max_draft=1, temp=1.0,
                                             uniforms=torch.rand(2 * S, generator=g, device="cuda"), noise=torch.rand((S, V), generator=g, device="cuda"), draft_logits=draft_logits)
        want = p.double().softmax(0).cpu()
        seen = torch.bincount(tokens[:, 0].long().cpu(), minlength=V).double() / S
        assert bool(((seen - want).abs() <= 5 * (want * (1 - want) / S).sqrt()).all())
        assert set(counts.tolist()) == {1, 2}


# ---------------------------------------------------------------------------------------------------- together
def _model(head_dim=64, n_pages=40, seed=5):
    from parity_util import tiny_args
    from proxy_inference_engine_b200.checkpoint import build_model, random_weights
    args = tiny_args(bits=4, head_dim=head_dim)
    w = random_weights(args, seed=seed, device="cuda", gen_device="cpu")
    mk = lambda: [tuple(torch.full((n_pages, 64, args.num_key_value_heads, args.head_dim), torch.nan, dtype=BF, device="cuda") for _ in range(2))
                  for _ in range(args.num_hidden_layers)]
    return args, w, build_model(args, w), mk


@pytest.mark.parametrize("head_dim", [64, 128])
def test_a_planned_step_is_the_ragged_step(head_dim):
    """The same logits as BatchDetails', whose rows each have a decode attention of their own, and as the oracle's."""
    import numpy as np
    from parity_util import make_oracle, rel_l2
    from proxy_inference_engine_b200.ragged import BatchDetails, StepPlan, ragged_step
    args, w, model, mk = _model(head_dim)
    rng = np.random.default_rng(0)
    seq = {s: rng.integers(0, args.vocab_size, n).tolist() for s, n in ((7, 70), (11, 101), (12, 84))}
    pages = {7: [3, 9], 11: [1, 0], 12: [30, 5]}
    old, new = mk(), mk()
    for k, v in old:
        k.zero_(), v.zero_()
    steps = [[(11, 0, 100), (12, 0, 64)], [(7, 0, 70), (11, 100, 101), (12, 64, 84)]]
    for step in steps:
        batch = BatchDetails.build([(s, seq[s][a:b], a, pages[s]) for s, a, b in step])
        want = ragged_step(model, batch, old, all_logits=True).float().cpu().numpy()
        plan = StepPlan.build(ints([t for s, a, b in step for t in seq[s][a:b]]), ints([b - a for s, a, b in step]), ints([a for s, a, b in step]),
                              ints([p for s, a, b in step for p in pages[s][:O.need(b - a, a)]]), num_pages=40, max_blocks=2, num_heads=args.num_attention_heads,
                              num_kv_heads=args.num_key_value_heads)
        plan.check()
        got = ragged_step(model, plan, new, all_logits=True).float().cpu().numpy()
        assert rel_l2(got, want) < 1e-2
        last = ragged_step(model, plan, new).float().cpu().numpy()
        assert last.shape[0] == len(step) and rel_l2(last, got[batch.last_token_rows().tolist()]) < 5e-3
    o = make_oracle(args, w)
    for row, (s, _, _) in zip(last, steps[-1]):
        lo = o(np.asarray([seq[s]], np.int32), o.make_cache(), last_only=True)[0, -1]
        assert rel_l2(row, lo) < 2e-2


def test_drafting_gives_the_text_that_decoding_gives():
    """Greedy speculative steps with good, bad and no drafts, lengths kept on the device: every token is the first largest logit of the 64-token-page cache's own
    model, or one that the model cannot tell from it (other row counts round other sums)."""
    import numpy as np
    from parity_util import make_oracle
    from proxy_inference_engine_b200.ragged import StepPlan, speculative_step
    args, w, model, mk = _model(64)
    pools, rng, S, K = mk(), random.Random(3), 3, 4
    prompts = [[rng.randrange(args.vocab_size) for _ in range(n)] for n in (61, 5, 130)]
    table = ints([[i * 8 + j for j in range(8)] for i in range(S)])
    plan_of = lambda ids, new, cached, drafted, R: StepPlan.build(ids, new, cached, table, num_pages=40, max_blocks=8, num_heads=args.num_attention_heads,
                                                                  num_kv_heads=args.num_key_value_heads, draft_lengths=drafted, num_logits=R)
    new, cached = ints([len(p) for p in prompts]), ints([0] * S)
    tokens, counts, _ = speculative_step(model, plan_of(ints(sum(prompts, [])), new, cached, None, S), pools, max_draft=0)
    cached, text = cached + new, [p + [t] for p, t in zip(prompts, tokens[:, 0].tolist())]
    o = make_oracle(args, w)
    truth = [list(t) for t in text]
    accepted = 0
    for step in range(6):
        drafts = []
        for s in range(S):      # the oracle's own continuation as a draft, spoilt at some place
            ids, mine = list(text[s]), []
            for _ in range((step + s) % (K + 1)):
                lo = o(np.asarray([ids], np.int32), o.make_cache(), last_only=True)[0, -1]
                mine.append(int(lo.argmax()))
                ids.append(mine[-1])
            if mine and rng.random() < 0.5:
                mine[rng.randrange(len(mine))] = rng.randrange(args.vocab_size)
            drafts.append(mine)
        ids = [t for s in range(S) for t in [text[s][-1]] + drafts[s]]
        drafted = ints([len(d) for d in drafts])
        plan = plan_of(ints(ids + [0] * 3), drafted + 1, cached, drafted, len(ids))
        tokens, counts, _ = speculative_step(model, plan, pools, max_draft=K)
        cached = cached + counts                                    # context + new - drafted + counts - 1
        plan.check()
        for s, (t, c) in enumerate(zip(tokens.tolist(), counts.tolist())):
            accepted += c - 1
            assert 1 <= c <= len(drafts[s]) + 1 and t[:c - 1] == drafts[s][:c - 1]
            text[s] += t[:c]
    assert accepted > 5
    for s in range(S):
        lo = o(np.asarray([text[s][:-1]], np.int32), o.make_cache())[0]
        for i in range(len(prompts[s]), len(text[s])):
            row = lo[i - 1]
            assert text[s][i] == int(row.argmax()) or row.max() - row[text[s][i]] < 2e-2 * np.abs(row).max()


def test_a_captured_step_runs_again_on_other_lengths():
    from proxy_inference_engine_b200.ragged import StepPlan, speculative_step
    args, w, model, mk = _model(128)
    pools, S, T, V = mk(), 2, 12, args.vocab_size
    g = gen(1)
    for k, v in pools:
        k.copy_(randn(g, *k.shape, std=0.5)), v.copy_(randn(g, *v.shape))
    ids, new, cached, drafted = ints([0] * T), ints([1, 1]), ints([10, 10]), ints([0, 0])
    table, uniforms, noise = ints([[3, 4, 5, 6], [7, 8, 9, 10]]), torch.rand(T, generator=g, device="cuda"), torch.rand((S, V), generator=g, device="cuda")

    def step():
        plan = StepPlan.build(ids, new, cached, table, num_pages=40, max_blocks=4, num_heads=args.num_attention_heads, num_kv_heads=args.num_key_value_heads, draft_lengths=drafted,
                              num_logits=T)
        return speculative_step(model, plan, pools, max_draft=4, temp=0.9, uniforms=uniforms, noise=noise)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    kept = [(k.clone(), v.clone()) for k, v in pools]
    restore = lambda: [t.copy_(t0) for pair, pair0 in zip(pools, kept) for t, t0 in zip(pair, pair0)]
    for lens, ctx, dr in (([3, 5], [60, 100], [2, 4]), ([0, 1], [7, 200], [0, 0]), ([5, 1], [130, 0], [4, 0])):
        for t, x in ((new, lens), (cached, ctx), (drafted, dr), (ids, [(7 * i + sum(ctx)) % V for i in range(T)])):
            t.copy_(ints(x))
        restore()
        graph.replay()
        got = [t.clone() for t in out]
        restore()
        want = step()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_the_native_host_form_is_the_python_one(monkeypatch):
    """The same bits, for tensors that the native form takes and for those it leaves: views, other strides, odd addresses."""
    from proxy_inference_engine_b200 import ops
    from proxy_inference_engine_b200.ragged import StepPlan
    assert ops.native_host() is not ops._NoHost
    g, Hq, Hkv, D, V = gen(2), 8, 2, 64, 1000
    lens = [ints([3, 0, 70]), ints([60, 5, 0]), ints([2, 0, 0])]
    ids, pages, wide = ints(list(range(73))), ints([4, 2, 3, 0, 1]), ints([[4, 2, 9, 9], [3, 9, 9, 9], [0, 1, 9, 9]])
    pool = lambda: (randn(gen(3), 6, 64, Hkv, D), randn(gen(4), 6, 64, Hkv, D))
    rows = randn(g, 73, Hq + 2 * Hkv, D)
    odd = torch.empty(73 * Hq * D + 1, dtype=BF, device="cuda")[1:].view(73, Hq, D)
    odd.copy_(rows[:, :Hq])
    logits, u, noise = randn(g, 6, V + 8), torch.rand(6, generator=g, device="cuda"), torch.rand((2, V), generator=g, device="cuda")
    guess, drafts, starts = randn(g, 6, V + 8), ints([5, 6, 7, 8, 9, 10]), ints([0, 2, 6])
    plain_q = rows[:, :Hq].contiguous()

    def everything():
        got = []
        for table in (pages, wide, wide[:, :2], wide.t().contiguous().t()):
            plan = StepPlan.build(ids, *lens[:2], table, num_pages=10, max_blocks=3, num_heads=Hq, num_kv_heads=Hkv, draft_lengths=lens[2], num_logits=5)
            got += [getattr(plan, n) for n in ("row_starts", "contexts", "sequences", "positions", "slots", "block_table", "logit_starts", "logit_rows", "draft_tokens")]
            plan = StepPlan.build(ids, *lens[:2], table, num_pages=6, max_blocks=3, num_heads=Hq, num_kv_heads=Hkv)
            for q in (plain_q, rows[:, :Hq], odd, rows[:, :1].expand(73, Hq, D)):
                k_pool, v_pool = pool()
                turned = ops.rope_kv_slots(q, rows[:, Hq:Hq + Hkv], rows[:, Hq + Hkv:], FREQS(D), plan.positions, plan.slots, k_pool, v_pool)
                got += [turned, k_pool, v_pool, ops.chunk_attention(q, k_pool, v_pool, plan, 0.2), ops.chunk_attention(q, k_pool, v_pool, plan, 0.2, out=torch.ones_like(turned).view(73, -1))]
        for x, q in ((logits[:, :V], guess[:, :V]), (logits[:, :V].contiguous(), guess[:, :V].contiguous()), (logits[:, :V].contiguous(), guess[:, :V]), (logits[:, 3:V + 3], None),
                     (logits[:, :V], None)):
            got += ops.verify_draft(x, drafts, starts, max_draft=3, temp=0.7, uniforms=u, noise=noise, draft_logits=q)
            got += ops.verify_draft(x, drafts, starts, max_draft=1)
        return got

    native = everything()
    monkeypatch.setattr(ops, "native_host", lambda: ops._NoHost)
    python = everything()
    assert len(native) == len(python)
    for i, (a, b) in enumerate(zip(native, python)):
        assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride() and torch.equal(a.view(torch.int16) if a.dtype == BF else a, b.view(torch.int16) if b.dtype == BF else b), i


@pytest.mark.parametrize("stride", [0, 1, 24])
def test_one_row_of_any_stride(stride):
    """The stride of a dimension of one is anything at all."""
    import dataclasses
    from proxy_inference_engine_b200 import ops
    from proxy_inference_engine_b200.ragged import StepPlan
    Hq, Hkv, D, V = 4, 2, 64, 4001
    pools = [torch.randn((4, 64, Hkv, D), generator=gen(1), device="cuda").to(BF) for _ in range(2)]
    q, k, v = (torch.randn((1, H, D), generator=gen(2), device="cuda").to(BF) for H in (Hq, Hkv, Hkv))
    freqs = torch.linspace(1.0, 9.0, D // 2, device="cuda")
    plan = StepPlan.build(ints([1]), ints([1]), ints([70]), ints([2, 1]), num_pages=4, max_blocks=2, num_heads=Hq, num_kv_heads=Hkv)
    odd = lambda x: x.as_strided(x.shape, (stride, *x.stride()[1:]))
    other = [p.clone() for p in pools]
    got = ops.rope_kv_slots(odd(q), odd(k), odd(v), freqs, plan.positions, plan.slots, *pools)
    want = ops.rope_kv_slots(q, k, v, freqs, plan.positions, plan.slots, *other)
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(pools, other))
    assert torch.equal(ops.chunk_attention(odd(q), *pools, plan, 0.125), ops.chunk_attention(q, *pools, plan, 0.125))
    x = torch.randn((1, V), generator=gen(3), device="cuda").to(BF)
    for a, b in zip(*(ops.verify_draft(t, ints([-1]), ints([0, 1]), max_draft=0) for t in (odd(x), x))):
        assert torch.equal(a, b)
    with pytest.raises(ValueError, match="plan.words"):
        ops.chunk_attention(q, *pools, dataclasses.replace(plan, words=plan.words[:-4].clone()), 0.125)


def test_a_planned_step_that_is_refused_writes_nothing():
    """A plan of other heads or pools, and pools of which the last layer's do not fit: the first layer's are left as they were."""
    from proxy_inference_engine_b200.ragged import StepPlan, ragged_step
    args, w, model, mk = _model(64)
    Hq, Hkv = args.num_attention_heads, args.num_key_value_heads
    plan_of = lambda pages, hq, hkv: StepPlan.build(ints([1]), ints([1]), ints([0]), ints([0]), num_pages=pages, max_blocks=1, num_heads=hq, num_kv_heads=hkv)
    pools = [tuple(torch.zeros_like(t) for t in pair) for pair in mk()]
    short, eights = [(k[:39], v[:39]) for k, v in pools], [((k,), (v,)) for k, v in pools]
    for plan, given, match in ((plan_of(39, Hq, Hkv), pools, "the plan is for"), (plan_of(40, 2 * Hq, Hkv), pools, "the plan is for"), (plan_of(40, Hq, Hq), pools, "the plan is for"),
                               (plan_of(40, Hq, Hkv), pools[:-1] + short[-1:], "the plan is for"), (plan_of(40, Hq, Hkv), pools[:-1] + eights[-1:], "8-bit"),
                               (plan_of(40, Hq, Hkv), pools[:-1] + [(pools[-1][0], pools[-1][1].float())], "bfloat16")):
        with pytest.raises(ValueError, match=match):
            ragged_step(model, plan, given)
    assert not any(bool(t.any()) for pair in pools for t in pair)
    ragged_step(model, plan_of(40, Hq, Hkv), pools)
    assert all(bool(t[0, 0].any()) for pair in pools for t in pair)


def test_a_planned_step_refuses():
    from proxy_inference_engine_b200.ragged import StepPlan, ragged_step
    args, w, model, mk = _model(64)
    plan = StepPlan.build(ints([1]), ints([1]), ints([0]), ints([0]), num_pages=40, max_blocks=1, num_heads=args.num_attention_heads, num_kv_heads=args.num_key_value_heads)
    pools = mk()
    with pytest.raises(ValueError, match="8-bit"):
        ragged_step(model, plan, [((k,), (v,)) for k, v in pools])
    with pytest.raises(ValueError, match="pools for"):
        ragged_step(model, plan, pools[:1])
    model.layers[0].self_attn.rope.traditional = True
    with pytest.raises(ValueError, match="by halves"):
        ragged_step(model, plan, pools)
