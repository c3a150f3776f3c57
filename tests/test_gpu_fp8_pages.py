"""A ragged step over a cache of 8 bits against plain arithmetic in 64 bits.

Tolerances.  Codes: a feature's code is the nearest of e4m3, half a step off: 2^-4 of it, or 2^-10 of the scale; values (and keys at angle 0) are coded from the numbers as they are,
so their codes and scales are equal.  Attention, as over 16-bit pages: the result's rounding 2^-8, the weights' 2^-8 (fp16's 2^-11 where a request has up to 32 rows), and 2^-12 of the weights
for the scores' sums in fp32, the exponentials and the row's sum."""
import random

import pytest
import torch

import step_oracle as O

pytestmark = pytest.mark.gpu
BF, F8, F64 = torch.bfloat16, torch.float8_e4m3fn, torch.float64
FREQS = lambda D: 500000.0 ** (torch.arange(0, D, 2, dtype=torch.float32, device="cuda") / D)
STILL = lambda D: torch.full((D // 2,), float("inf"), device="cuda")   # angle 0
ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, std=1.0):
    return (std * torch.randn(shape, generator=g, device="cuda")).to(BF)


def make_plan(new, cached, tables, n_pages, Hq, Hkv, pad=0):
    from proxy_inference_engine_b200.ragged import StepPlan
    T = max(1, sum(new) + pad)
    pages = [p for n, c, t in zip(new, cached, tables) for p in t[:O.need(n, c)]]
    return StepPlan.build(ints([0] * T), ints(new), ints(cached), ints(pages or [0]), num_pages=n_pages, max_blocks=max(1, max(O.need(n, c) for n, c in zip(new, cached))),
                          num_heads=Hq, num_kv_heads=Hkv)


def make_tables(new, cached, seed, spare=3):
    need = [O.need(n, c) for n, c in zip(new, cached)]
    n_pages = sum(need) + spare
    order = list(range(n_pages))
    random.Random(seed).shuffle(order)
    tables, at = [], 0
    for k in need:
        tables.append(order[at:at + k])
        at += k
    return tables, n_pages


def make_pools(g, n_pages, Hkv, D, std=1.0):
    """Codes of all sizes, e4m3's lowest among them, and scales that differ from page to page."""
    pools = []
    for s in (std, 0.6 * std):
        x = s * torch.randn((n_pages, Hkv, 64, D), generator=g, device="cuda")
        scales = torch.exp2(torch.randint(-9, -5, (n_pages, Hkv), generator=g, device="cuda").float())
        pools += [(x / scales[..., None, None]).clamp(-448, 448).to(F8), scales]
    return pools


def values(pool, scales):
    return pool.double() * scales.double()[..., None, None]


def raw(t):
    return t.view(torch.int8) if t.dtype == F8 else t.view(torch.int32) if t.dtype == torch.float32 else t.view(torch.int16)


def e4m3_scale(amax):
    """The lowest power of two with which amax is 448 or less (and 2^-60 at least), of float64."""
    return torch.exp2(torch.ceil(torch.log2(amax.clamp(min=448 * 2.0 ** -60) / 448)))


def write(pool, scales, x, new, cached, tables):
    """x [T, Hkv, D] of 64 bits to its pages, one at a time; all on the CPU."""
    row = 0
    for n, c, table in zip(new, cached, tables):
        at = c
        while at < c + n:
            to, page, lies = min(c + n, (at // 64 + 1) * 64), table[at // 64], at % 64
            rows = x[row + at - c:row + to - c].transpose(0, 1)
            scale = e4m3_scale(rows.abs().flatten(1).amax(1)).float()
            if lies:
                old = scales[page].clone()
                scale = torch.maximum(scale, old)
                pool[page, :, :lies] = (pool[page, :, :lies].float() * (old / scale)[:, None, None]).to(F8)
            pool[page, :, lies:lies + to - at] = (rows / scale.double()[:, None, None]).float().to(F8)
            scales[page] = scale
            at = to
        row += n


STEPS = [([1], [0]), ([1, 1, 1], [0, 63, 64]), ([5, 0, 70, 1], [3, 9, 40, 700]), ([64, 65, 128, 200], [0, 0, 64, 63]), ([0, 0, 3], [0, 5, 62]), ([1] * 300, [i * 7 % 200 for i in range(300)]),
         ([700, 1, 2], [130, 127, 126])]


@pytest.mark.parametrize("Hq,Hkv,D", [(4, 2, 64), (8, 2, 128), (32, 8, 128), (5, 1, 64)])
@pytest.mark.parametrize("new,cached", STEPS)
def test_rows_into_pages(new, cached, Hq, Hkv, D):
    """Codes, scales, what lay in the pages and what lies in others, bit for bit (keys at angle 0); then keys and queries at their own angles."""
    from proxy_inference_engine_b200 import ops
    g = gen(len(new) + D)
    tables, n_pages = make_tables(new, cached, D)
    plan = make_plan(new, cached, tables, n_pages, Hq, Hkv, pad=3)
    plan.check()
    T, live = sum(new) + 3, sum(new)
    sizes = torch.exp2(torch.randint(-3, 4, (T, 1, 1), generator=g, device="cuda").float()).to(BF)
    q, k, v = randn(g, T, Hq, D), randn(g, T, Hkv, D) * sizes, randn(g, T, Hkv, D) * sizes
    start = make_pools(g, n_pages, Hkv, D)
    got = [t.clone() for t in start]
    out = ops.rope_kv_fp8(q, k, v, STILL(D), plan, *got)
    want = [t.cpu().clone() for t in start]
    for (pool, scales), x in zip((want[:2], want[2:]), (k, v)):
        write(pool, scales, x[:live].cpu().double(), new, cached, tables)
    for a, b in zip(got, want):
        assert torch.equal(raw(a.cpu()), raw(b))
    assert torch.equal(out[:live], q[:live]) and not out[live:].any()

    got = [t.clone() for t in start]
    kept = torch.full((T, Hq, D), 7.0, dtype=BF, device="cuda")
    assert ops.rope_kv_fp8(q, k, v, FREQS(D), plan, *got, out=kept) is kept
    scratch = [torch.zeros((n_pages, 64, Hkv, D), dtype=BF, device="cuda") for _ in range(2)]
    turned = ops.rope_kv_slots(q, k, v, FREQS(D), plan.positions, plan.slots, *scratch)
    assert torch.equal(kept[:live], turned[:live]) and bool((kept[live:] == 7.0).all())
    for a, b in zip(got[2:], want[2:]):
        assert torch.equal(raw(a.cpu()), raw(b))
    exact = O.rope(k, plan.positions, FREQS(D))
    codes, scales = values(got[0], got[1]).cpu(), got[1].cpu().double()
    at, of = plan.slots.cpu()[:live].long(), start[1].cpu().double()
    mine = codes[at // 64, :, at % 64]
    # (a rotation is off by 1e-6 of the pair's size)
    pair = exact[:live].view(live, Hkv, 2, D // 2).square().sum(2, keepdim=True).sqrt().expand(-1, -1, 2, -1).reshape(live, Hkv, D)
    bound = torch.maximum(2.0 ** -4 * exact[:live].abs(), 2.0 ** -10 * scales[at // 64][..., None]) + 2e-6 * pair
    # a row that was coded before a later row of another step: none here, so that half a step is all
    assert bool(((mine - exact[:live]).abs() <= bound).all())
    # scales: those of the exact rotation, where its largest is not next to a border
    near = torch.zeros_like(of, dtype=torch.bool)
    row = 0
    for n, c, table in zip(new, cached, tables):
        for j in range(c // 64, O.need(n, c)) if n else ():
            lo, hi = max(c, 64 * j), min(c + n, 64 * j + 64)
            top = exact[row + lo - c:row + hi - c].abs().amax((0, 2))
            need = e4m3_scale(top)
            near[table[j]] = (top / need > 448 * (1 - 1e-5)) | (top / need < 224 * (1 + 1e-5))
            of[table[j]] = torch.maximum(need, of[table[j]]) if lo % 64 else need
        row += n
    assert bool(((scales == of) | near).all()) and float(near.double().mean()) < 0.05


def test_page_after_page_token_by_token():
    """What a hundred steps leave is what the plain form leaves; a scale grows, and begins anew with the page."""
    from proxy_inference_engine_b200 import ops
    g, Hkv, D = gen(3), 2, 64
    tables, n_pages = [[4, 0, 2], [1, 3, 5]], 6
    got = make_pools(g, n_pages, Hkv, D)
    want = [t.cpu().clone() for t in got]
    cached = [0, 60]
    rng = random.Random(1)
    for step in range(60):
        new = [rng.choice([1, 1, 1, 2, 5]), rng.choice([0, 1, 1, 3])]
        if max(c + n for c, n in zip(cached, new)) > 190:
            break
        T = sum(new)
        k, v = (randn(g, T, Hkv, D) * 2.0 ** rng.randint(-6, 6) for _ in range(2))
        ops.rope_kv_fp8(randn(g, T, 4, D), k, v, STILL(D), make_plan(new, cached, tables, n_pages, 4, Hkv), *got)
        for (pool, scales), x in zip((want[:2], want[2:]), (k, v)):
            write(pool, scales, x.cpu().double(), new, cached, tables)
        for a, b in zip(got, want):
            assert torch.equal(raw(a.cpu()), raw(b)), step
        # drafted tokens that were refused are written over
        cached = [c + max(0, n - (rng.random() < 0.3 and n > 1)) for c, n in zip(cached, new)]
    assert min(cached) > 70


def test_features_at_the_borders_of_scales():
    """448 2^n and its neighbours, the type's lowest and largest numbers, blocks of zeros, infinities and NaN."""
    from proxy_inference_engine_b200 import ops
    D, tops = 64, [448.0, 450.0, 446.0, 224.0, 226.0, 0.0, 2.0 ** -133, 448 * 2.0 ** -60, 450 * 2.0 ** -60, 1.0, 3.38e38, 1.75, 2.0]
    new, cached = [1] * (len(tops) + 3), [0] * (len(tops) + 3)
    tables, n_pages = make_tables(new, cached, 1)
    x = torch.zeros((len(new), 1, D), dtype=BF, device="cuda")
    for i, top in enumerate(tops):
        x[i, 0] = (torch.linspace(-1, 1, D) * top).to(BF).cuda()
    x[len(tops), 0, 5], x[len(tops) + 1, 0, 63], x[len(tops) + 2, 0, 0] = torch.inf, -torch.inf, torch.nan
    got = make_pools(gen(1), n_pages, 1, D)
    want = [t.cpu().clone() for t in got]
    plan = make_plan(new, cached, tables, n_pages, 1, 1)
    ops.rope_kv_fp8(x, x, x, STILL(D), plan, *got)
    write(want[2], want[3], x[:len(tops)].cpu().double(), new[:len(tops)], cached[:len(tops)], tables[:len(tops)])
    fine = [t[0] for t in tables[:len(tops)]]
    assert torch.equal(raw(got[2].cpu())[fine, :, 0], raw(want[2])[fine, :, 0]) and torch.equal(got[3].cpu()[fine], want[3][fine])
    rest = [t[0] for t in tables[len(tops):]]
    assert bool(got[3][rest].isnan().all())
    # such a block stays without numbers while it is written on, and begins anew with its first token
    y = torch.ones_like(x)
    ops.rope_kv_fp8(y, y, y, STILL(D), make_plan(new, [1] * len(new), tables, n_pages, 1, 1), *got)
    assert bool(got[3][rest].isnan().all()) and not bool(got[3][fine].isnan().any())
    ops.rope_kv_fp8(y, y, y, STILL(D), plan, *got)
    assert bool((got[3][rest] == 2.0 ** -8).all()) and bool((values(got[2], got[3])[rest, :, 0] == 1.0).all())


def attention_case(new, cached, Hq, Hkv, D, seed=0, pad=0, std=2.0):
    g = gen(seed)
    tables, n_pages = make_tables(new, cached, seed)
    plan = make_plan(new, cached, tables, n_pages, Hq, Hkv, pad)
    return plan, randn(g, max(1, sum(new) + pad), Hq, D, std=std), make_pools(g, n_pages, Hkv, D), tables


def attention_holds(got, q, pools, new, cached, tables, scale, slack=2.0 ** -12):
    Hq, D = q.shape[1:]
    Hkv = pools[0].shape[1]
    k, v = (values(*p).transpose(1, 2) for p in (pools[:2], pools[2:]))
    want, weight = O.attention(q[:sum(new)], k, v, new, cached, tables, scale)
    few = torch.tensor([n * (Hq // Hkv) <= 32 for n in new for _ in range(n)])[:, None, None]
    off = (got[:sum(new)].view(want.shape).cpu().double() - want).abs()
    bound = 2.0 ** -8 * want.abs() + (torch.where(few, 2.0 ** -11, 2.0 ** -8).double() + slack) * weight + 1e-37
    assert bool((off <= bound).all()), float((off - bound).max())


SHAPES = [([1], [0]), ([1], [63]), ([1], [64]), ([3], [200]), ([8, 1, 5], [900, 70, 0]), ([64, 1], [0, 129]), ([33, 40], [64, 500]), ([129], [1]), ([300, 2, 17], [100, 1000, 63]),
          ([700, 1, 1, 64], [30, 2000, 5, 300]), ([0, 4, 0], [7, 100, 0]), ([1] * 40, [i * 37 % 900 for i in range(40)]), ([1, 200], [9000, 20])]


@pytest.mark.parametrize("Hq,Hkv,D", [(4, 2, 64), (8, 2, 128), (32, 8, 128), (32, 8, 64)])
@pytest.mark.parametrize("new,cached", SHAPES)
def test_attention(new, cached, Hq, Hkv, D):
    from proxy_inference_engine_b200 import ops
    plan, q, pools, tables = attention_case(new, cached, Hq, Hkv, D, seed=len(new) + D, pad=2)
    got = ops.chunk_attention_fp8(q, *pools, plan, D ** -0.5)
    attention_holds(got, q, pools, new, cached, tables, D ** -0.5)
    assert not got[sum(new):].any()
    assert torch.equal(got, ops.chunk_attention_fp8(q, *pools, plan, D ** -0.5))
    ops.check_pipeline()


@pytest.mark.parametrize("seed", range(24))
def test_steps_of_all_kinds_of_requests(seed):
    """Few rows, one query tile and two of them, one behind the other in every order."""
    from proxy_inference_engine_b200 import ops
    rng = random.Random(seed)
    D, (Hq, Hkv) = rng.choice([64, 128]), rng.choice([(4, 2), (8, 2), (32, 8), (8, 8), (7, 1), (40, 1), (24, 8)])
    new = [rng.choice([1, 1, 2, 3, 4, 5, 8, 9, 16, 17, 33, 70, 130, 200, 0]) for _ in range(rng.choice([3, 12, 60]))]
    cached = [rng.choice([0, 1, 62, 63, 64, 65, 127, 128, 300, 1000, rng.randint(0, 2500)]) for _ in new]
    plan, q, pools, tables = attention_case(new, cached, Hq, Hkv, D, seed=seed, pad=rng.choice([0, 5]))
    got = ops.chunk_attention_fp8(q, *pools, plan, D ** -0.5)
    attention_holds(got, q, pools, new, cached, tables, D ** -0.5)
    assert not got[sum(new):].any()
    for _ in range(3):
        assert torch.equal(got, ops.chunk_attention_fp8(q, *pools, plan, D ** -0.5))
    ops.check_pipeline()


def test_rows_that_lie_anywhere_and_rows_of_nobody():
    from proxy_inference_engine_b200 import ops
    new, cached, Hq, Hkv = [3, 90, 0, 17], [300, 40, 9, 0], 8, 2
    outside = lambda x: x.permute(1, 0, 2).contiguous().permute(1, 0, 2)
    for D in (64, 128):
        plan, q, pools, tables = attention_case(new, cached, Hq, Hkv, D, seed=D, pad=7)
        want = ops.chunk_attention_fp8(q, *pools, plan, D ** -0.5)
        attention_holds(want, q, pools, new, cached, tables, D ** -0.5)
        assert torch.equal(ops.chunk_attention_fp8(outside(q), *pools, plan, D ** -0.5), want)
        out = torch.full_like(want, 3.0)
        assert ops.chunk_attention_fp8(q, *pools, plan, D ** -0.5, out=out) is out
        assert torch.equal(out[:110], want[:110]) and bool((out[110:] == 3.0).all()) and not want[110:].any()
        side = randn(gen(D), 117, (Hq + 2 * Hkv) * D)
        a, b, c = (t.view(117, -1, D) for t in side.split([Hq * D, Hkv * D, Hkv * D], 1))
        got = [[t.clone() for t in pools] for _ in range(3)]
        turned = ops.rope_kv_fp8(a, b, c, FREQS(D), plan, *got[0])
        assert torch.equal(ops.rope_kv_fp8(outside(a), outside(b), outside(c), FREQS(D), plan, *got[1]), turned)
        odd = torch.empty(a.numel() + 1, dtype=BF, device="cuda")[1:].view(a.shape).copy_(a)
        assert torch.equal(ops.rope_kv_fp8(odd, b, c, FREQS(D), plan, *got[2]), turned) and not turned[110:].any()
        for other in got[1:]:
            assert all(torch.equal(raw(x), raw(y)) for x, y in zip(got[0], other))
        ops.check_pipeline()


def test_what_lies_behind_the_last_token_does_not_matter():
    """Codes of NaN, scales of NaN and infinity in pages that no request has, and codes behind a request's last token; one request's NaN is its own."""
    from proxy_inference_engine_b200 import ops
    for new, cached in (([3, 40, 1], [200, 100, 301]), ([1, 5, 200], [30, 70, 10])):
        plan, q, pools, tables = attention_case(new, cached, 8, 2, 128, seed=13)
        want = ops.chunk_attention_fp8(q, *pools, plan, 0.1)
        p2 = [t.clone() for t in pools]
        spare = [i for i in range(len(p2[0])) if i not in sum(tables, [])]
        for i in (0, 2):
            raw(p2[i])[spare] = 0x7f
            p2[i + 1][spare] = torch.nan
            for n, c, t in zip(new, cached, tables):
                raw(p2[i])[t[-1], :, (n + c - 1) % 64 + 1:] = 0x7f if i else -1
        assert torch.equal(ops.chunk_attention_fp8(q, *p2, plan, 0.1), want)
        for i in (1, 3):
            p2 = [t.clone() for t in pools]
            p2[i][tables[1][0]] = torch.nan
            got = ops.chunk_attention_fp8(q, *p2, plan, 0.1)
            rest = list(range(new[0])) + list(range(new[0] + new[1], sum(new)))
            assert torch.equal(got[rest], want[rest]) and bool(torch.isnan(got[new[0]:new[0] + new[1]]).all())
    ops.check_pipeline()


@pytest.mark.parametrize("new", [[1], [4], [8], [30]])
def test_pages_of_very_different_scales(new):
    """Values a million million times larger in some pages than in others, which the rows do not attend to, and the other way round."""
    from proxy_inference_engine_b200 import ops
    cached, D, Hq, Hkv = [1000], 128, 8, 2
    for order in (1, -1):
        plan, q, pools, tables = attention_case(new, cached, Hq, Hkv, D, seed=3, std=0.5)
        for j, page in enumerate(tables[0]):
            pools[3][page] = 2.0 ** (-40 if (j // 5) % 2 == (order > 0) else 2)
            pools[1][page] = 2.0 ** -8 if j != 7 else 2.0 ** -5
        got = ops.chunk_attention_fp8(q, *pools, plan, D ** -0.5)
        attention_holds(got, q, pools, new, cached, tables, D ** -0.5)
    # one page takes all of the weight: its values, whatever the others' scales
    q[:], one = 1.0, 9
    raw(pools[0])[:], raw(pools[0])[tables[0][one]] = -72, 0x38   # codes of -1 and 1
    pools[1][:] = 8.0
    got = ops.chunk_attention_fp8(q, *pools, plan, D ** -0.5).view(-1, Hkv, Hq // Hkv, D).double()
    mean = values(pools[2], pools[3])[tables[0][one]].mean(1)[None, :, None]
    assert bool(((got - mean).abs() <= 2.0 ** -8 * mean.abs() + (2.0 ** -8 + 2.0 ** -12) * values(pools[2], pools[3])[tables[0][one]].abs().mean(1)[None, :, None]).all())


@pytest.mark.parametrize("new", [[1], [8], [30]])
def test_pages_that_nothing_was_written_to(new):
    """Codes of 0 and scale 0, as pools begin: keys and values of 0, alone and among others."""
    from proxy_inference_engine_b200 import ops
    cached, D, Hq, Hkv = [700], 128, 8, 2
    plan, q, pools, tables = attention_case(new, cached, Hq, Hkv, D, seed=5)
    for page in tables[0][2:5]:
        for pool in pools:
            raw(pool)[page] = 0
    attention_holds(ops.chunk_attention_fp8(q, *pools, plan, D ** -0.5), q, pools, new, cached, tables, D ** -0.5)
    for pool in pools:
        raw(pool)[:] = 0
    assert not ops.chunk_attention_fp8(q, *pools, plan, D ** -0.5).any()


@pytest.mark.parametrize("std", [0.0, 30.0])
def test_flat_and_steep_scores(std):
    from proxy_inference_engine_b200 import ops
    new, cached = [3, 140, 12], [1000, 600, 3000]
    plan, q, pools, tables = attention_case(new, cached, 8, 2, 128, seed=9, std=std)
    # scores of up to 30 * 4 * 128^0.5 = 1400: 1400 * 128 * 2^-24 = 0.011 in the exponent at the worst, on either side of a quotient; few rows' queries 2^-17 of the largest: as much again
    attention_holds(ops.chunk_attention_fp8(q, *pools, plan, 128 ** -0.5), q, pools, new, cached, tables, 128 ** -0.5, slack=0.044 if std else 2.0 ** -12)
    big = q * 2.0 ** 40
    same = [pools[0], pools[1] * 2.0 ** -40, pools[2], pools[3]]
    if not std:
        return
    attention_holds(ops.chunk_attention_fp8(big, *same, plan, 128 ** -0.5), big, same, new, cached, tables, 128 ** -0.5, slack=0.044)


@pytest.mark.parametrize("D", [64, 128])
def test_queries_of_all_sizes(D):
    """Down to bfloat16's lowest, each row with a power of two of its own; what is not finite makes its own row NaN and no other."""
    from proxy_inference_engine_b200 import ops
    new, cached, Hq, Hkv = [7, 1, 40, 8], [700, 3000, 100, 0], 8, 2
    plan, q, pools, tables = attention_case(new, cached, Hq, Hkv, D, seed=21)
    powers = torch.randint(-135, 1, (sum(new), Hq, 1), generator=gen(2), device="cuda").double()
    q = (q.double() * torch.exp2(powers)).to(BF)
    want = ops.chunk_attention_fp8(q, *pools, plan, D ** -0.5)
    attention_holds(want, q, pools, new, cached, tables, D ** -0.5)
    bad = q.clone()
    bad[2, 3, 5], bad[7, 0, D - 1], bad[50, 7, 0] = torch.nan, torch.inf, -torch.inf
    got = ops.chunk_attention_fp8(bad, *pools, plan, D ** -0.5).view(-1, Hq, D)
    for row, head in ((2, 3), (7, 0), (50, 7)):
        assert bool(got[row, head].isnan().all())
        got[row, head] = want.view(-1, Hq, D)[row, head]
    assert torch.equal(got.view(want.shape), want)
    ops.check_pipeline()


def test_two_streams_and_captured_graphs_at_once():
    from proxy_inference_engine_b200 import ops
    cases = [attention_case([4, 1, 70], [6000, 3000, 100], 8, 2, 128, seed=s) for s in (1, 2)]
    want = [ops.chunk_attention_fp8(q, *pools, plan, 0.1) for plan, q, pools, _ in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], [[], []]
    for _ in range(10):
        for i, (stream, (plan, q, pools, _)) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(stream):
                got[i].append(ops.chunk_attention_fp8(q, *pools, plan, 0.1))
    torch.cuda.synchronize()
    graphs = []
    for plan, q, pools, _ in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, ops.chunk_attention_fp8(q, *pools, plan, 0.1)))
    for _ in range(5):
        for stream, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i]) and torch.equal(graphs[i][1], want[i])
    ops.check_pipeline()


def test_pages_behind_the_32_bit_offsets():
    """Pools of 4.6e9 bytes: pages at either end, few rows and many."""
    from proxy_inference_engine_b200 import ops
    g, n_pages, Hq, Hkv, D = gen(21), 70000, 32, 8, 128
    pools = [torch.empty((n_pages, Hkv, 64, D), dtype=F8, device="cuda"), torch.full((n_pages, Hkv), torch.nan, device="cuda")] * 2
    pools = [pools[0], pools[1].clone(), torch.empty_like(pools[0]), pools[1].clone()]
    new, cached, tables = [5, 70], [100, 60], [[n_pages - 1, 3], [0, n_pages - 2, n_pages - 3]]
    plan = make_plan(new, cached, tables, n_pages, Hq, Hkv)
    for t in tables:
        for p in t:
            pools[0][p], pools[2][p] = (randn(g, Hkv, 64, D, std=100.0).clamp(-448, 448).to(F8) for _ in range(2))
            pools[1][p], pools[3][p] = 2.0 ** -7, 2.0 ** -8
    q, k, v = randn(g, 75, Hq, D), randn(g, 75, Hkv, D), randn(g, 75, Hkv, D)
    start = [{p: t[p].cpu().clone() for row in tables for p in row} for t in pools]
    ops.rope_kv_fp8(q, k, v, STILL(D), plan, *pools)
    at = plan.slots.long()
    for pool, scales, x in ((pools[0], pools[1], k), (pools[2], pools[3], v)):
        mine = pool[at // 64, :, at % 64].double() * scales[at // 64][..., None].double()
        assert bool(((mine - x.double()).abs() <= torch.maximum(2.0 ** -4 * x.double().abs(), 2.0 ** -10 * scales[at // 64][..., None].double())).all())
    got = ops.chunk_attention_fp8(q, *pools, plan, D ** -0.5)
    sub = {p: i for i, p in enumerate(sorted({p for t in tables for p in t}))}
    small = [t[sorted(sub)] for t in pools]
    attention_holds(got, q, small, new, cached, [[sub[p] for p in t] for t in tables], D ** -0.5)
    ops.check_pipeline()


def test_the_native_host_form_is_the_python_one(monkeypatch):
    from proxy_inference_engine_b200 import ops
    assert ops.native_host() is not ops._NoHost
    new, cached, Hq, Hkv, D = [3, 90, 17], [300, 40, 0], 8, 2, 64
    plan, q, pools, tables = attention_case(new, cached, Hq, Hkv, D, seed=1)
    g = gen(2)
    k, v, x = randn(g, 110, Hkv, D), randn(g, 110, Hkv, D), randn(g, 40, 512)
    weight, ws = ops.int8_rows(randn(g, 300, 512))
    norm, residual = randn(g, 512), randn(g, 40, 300)

    def everything():
        mine = [t.clone() for t in pools]
        codes, scales = ops.int8_rows(x, norm_weight=norm, eps=1e-6)
        return [ops.rope_kv_fp8(q, k, v, FREQS(D), plan, *mine), *map(raw, mine), ops.chunk_attention_fp8(q, *mine, plan, 0.125), codes, raw(scales),
                ops.int8_matmul(codes, scales, weight, ws, residual=residual), ops.int8_linear(x, weight, ws, norm_weight=norm, eps=1e-6, residual=residual),
                ops.int8_linear(x[::2, 16:272], *ops.int8_rows(randn(gen(5), 33, 256)))]
    native = everything()
    monkeypatch.setattr(ops, "native_host", lambda: ops._NoHost)
    for a, b in zip(native, everything()):
        assert torch.equal(a, b)


# ---------------------------------------------------------------------------------------------------- together
def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def _model(head_dim, seed=5):
    from parity_util import tiny_args
    from proxy_inference_engine_b200.checkpoint import build_model, random_weights
    args = tiny_args(bits=8, head_dim=head_dim)
    w = random_weights(args, seed=seed, device="cuda", gen_device="cpu")
    return args, w, build_model(args, w)


def _steps(args, steps, pages, seq, model, pools, n_pages=40):
    from proxy_inference_engine_b200.ragged import StepPlan, ragged_step
    out = []
    for step in steps:
        plan = StepPlan.build(ints([t for s, a, b in step for t in seq[s][a:b]]), ints([b - a for s, a, b in step]), ints([a for s, a, b in step]),
                              ints([p for s, a, b in step for p in pages[s][:O.need(b - a, a)]]), num_pages=n_pages, max_blocks=3, num_heads=args.num_attention_heads,
                              num_kv_heads=args.num_key_value_heads)
        plan.check()
        out.append(ragged_step(model, plan, pools, all_logits=True))
    return out


@pytest.mark.parametrize("head_dim", [64, 128])
def test_a_model_of_8_bits(head_dim):
    """Steps of a prompt, of its continuation and of single tokens: over 8-bit pages near the steps over 16-bit ones (a code is off by up to 2^-4 of a feature, 2^-6 of it on average), with
    linears of integers near those of the same weights (1 / 254 of a row's largest and of a channel's), and both together; the same bits again."""
    import random as rnd
    from proxy_inference_engine_b200 import nn
    from proxy_inference_engine_b200.ragged import fp8_pools
    args, w, model = _model(head_dim)
    r = rnd.Random(1)
    seq = {s: [r.randrange(args.vocab_size) for _ in range(n)] for s, n in ((7, 75), (11, 104), (12, 88))}
    pages = {7: [3, 9], 11: [1, 0], 12: [30, 5]}
    steps = [[(11, 0, 100), (12, 0, 64)], [(7, 0, 70), (11, 100, 101), (12, 64, 84)], [(7, 70, 71), (11, 101, 102), (12, 84, 88)]]
    wide = lambda: [tuple(torch.zeros((40, 64, args.num_key_value_heads, args.head_dim), dtype=BF, device="cuda") for _ in range(2)) for _ in range(args.num_hidden_layers)]
    want = _steps(args, steps, pages, seq, model, wide())
    eight = _steps(args, steps, pages, seq, model, fp8_pools(model, 40))
    assert all(rel(a, b) < 0.08 for a, b in zip(eight, want))
    assert all(torch.equal(a, b) for a, b in zip(eight, _steps(args, steps, pages, seq, model, fp8_pools(model, 40))))
    assert model.to_int8() is model and type(model.layers[0].mlp.up_proj) is nn.Int8Linear
    integers = _steps(args, steps, pages, seq, model, wide())
    both = _steps(args, steps, pages, seq, model, fp8_pools(model, 40))
    assert all(rel(a, b) < 0.05 for a, b in zip(integers, want)) and all(rel(a, b) < 0.1 for a, b in zip(both, want))
    # the model's other paths take such layers too
    x = torch.tensor([seq[11][:100]], dtype=torch.int32, device="cuda")
    assert rel(model(x)[0], integers[0][:100]) < 0.02


def test_drafting_over_8_bit_pages_in_a_captured_step():
    """Speculative steps on other lengths, captured once: the eager step's tokens, codes and scales."""
    from proxy_inference_engine_b200.ragged import StepPlan, fp8_pools, speculative_step
    args, w, model = _model(128)
    model.to_int8()
    pools, S, T, V = fp8_pools(model, 40), 2, 12, args.vocab_size
    g = gen(1)
    for pair in pools:
        for codes, scales in pair:
            codes.copy_((100 * torch.randn(codes.shape, generator=g, device="cuda")).clamp(-448, 448).to(F8))
            scales.copy_(torch.exp2(torch.randint(-9, -6, scales.shape, generator=g, device="cuda").float()))
    ids, new, cached, drafted = ints([0] * T), ints([1, 1]), ints([10, 10]), ints([0, 0])
    table, uniforms, noise = ints([[3, 4, 5, 6], [7, 8, 9, 10]]), torch.rand(T, generator=g, device="cuda"), torch.rand((S, V), generator=g, device="cuda")

    def step():
        plan = StepPlan.build(ids, new, cached, table, num_pages=40, max_blocks=4, num_heads=args.num_attention_heads, num_kv_heads=args.num_key_value_heads, draft_lengths=drafted,
                              num_logits=T)
        return speculative_step(model, plan, pools, max_draft=4, temp=0.9, uniforms=uniforms, noise=noise)
    flat = [t for pair in pools for both in pair for t in both]
    kept = [t.clone() for t in flat]
    restore = lambda: [t.copy_(t0) for t, t0 in zip(flat, kept)]
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for lens, ctx, dr in (([3, 5], [60, 100], [2, 4]), ([0, 1], [7, 200], [0, 0]), ([5, 1], [130, 0], [4, 0])):
        for t, x in ((new, lens), (cached, ctx), (drafted, dr), (ids, [(7 * i + sum(ctx)) % V for i in range(T)])):
            t.copy_(ints(x))
        restore()
        graph.replay()
        got = [t.clone() for t in out] + [t.clone() for t in flat]
        restore()
        want = list(step()) + flat
        for a, b in zip(got, want):
            assert torch.equal(raw(a) if a.dtype != torch.int32 else a, raw(b) if b.dtype != torch.int32 else b)


def test_a_planned_step_refuses_pools_that_do_not_fit():
    from proxy_inference_engine_b200.ragged import StepPlan, fp8_pools, ragged_step
    args, w, model = _model(64)
    pools = fp8_pools(model, 9)
    plan = StepPlan.build(ints([1]), ints([1]), ints([0]), ints([0]), num_pages=9, max_blocks=1, num_heads=args.num_attention_heads, num_kv_heads=args.num_key_value_heads)
    (k, ks), v = pools[-1]
    for bad in (((k[:8], ks), v), ((k, ks[:8]), v), ((k.transpose(1, 2), ks), v), ((k, ks.half()), v), ((raw(k), ks), v), ((k, ks), v[0]), ((k, ks, ks), v)):
        with pytest.raises(ValueError):
            ragged_step(model, plan, pools[:-1] + [bad])
    assert not any(bool(raw(t).any()) for pair in pools for both in pair for t in both)
    ragged_step(model, plan, pools)
