"""A ragged step over a cache of 8 bits against plain arithmetic in 64 bits.

Tolerances.  Codes: a feature's code is the nearest of e4m3, half a step off: 2^-4 of it, or 2^-10 of the scale; values (and keys at angle 0) are coded from the numbers as they are,
so their codes and scales are equal.  Attention, as over 16-bit pages: the result's rounding 2^-8, the weights' 2^-8 (fp16's 2^-11 where a request has up to 64 rows), and 2^-12 of the weights
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
    few = torch.tensor([n * (Hq // Hkv) <= 64 // (Hq // Hkv) * (Hq // Hkv) for n in new for _ in range(n)])[:, None, None]
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
