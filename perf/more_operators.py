"""The operators of a step served in 8 bits, at the sizes its users run: rows of activations as integers with a scale for each token, their products
with integer weights of a scale for each channel, and a paged cache of 8-bit keys and values with a scale for each page and head -- what is written to
it, and the attention of a ragged step over it.

Kinds (``case["kind"]``) and what one pass runs:
    rows    activations as int8 rows and a scale each (ops.int8_rows)
    linear  a linear layer of int8 weights: norm, rows, product, residual sum (ops.int8_linear)
    append  rotation of the step's queries and keys, keys and values written to 8-bit pages (ops.rope_kv_fp8)
    attend  causal attention of every request's new tokens over its 8-bit pages (ops.chunk_attention_fp8)

Definitions.  A row's scale is amax / 127 in 32 bits, its codes are x / scale rounded to the nearest (even).  A block of the cache is a page of 64 tokens of
one head: its scale is the lowest power of two, 2^-60 at least, with which every feature written since the page's first token is 448 or less, its codes are
float8 e4m3; where a new token needs a larger scale, the page's earlier codes are brought to it.

Sizes are those of the Llama presets (``checkpoint.LLAMA_PRESETS``) and of the tests' small model.  With ``own`` false a pass is the plain form:
elementary torch operations, requests padded to the longest of their kind.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BF16, F32, F64, I32, I8, F8 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.int8, torch.float8_e4m3fn
PAGE = 64
# query heads, key / value heads, head size
HEADS = {"1b": (32, 8, 64), "8b": (32, 8, 128), "70b": (64, 8, 128), "tiny": (4, 2, 64)}
# features in, features out
LINEARS = {"1b_up": (2048, 8192), "1b_down": (8192, 2048), "8b_qkv": (4096, 6144), "8b_o": (4096, 4096), "8b_up": (4096, 14336),
           "8b_gate_up": (4096, 28672), "8b_down": (14336, 4096), "70b_qkv": (8192, 10240), "70b_o": (8192, 8192), "tiny": (256, 512), "odd": (4112, 5003)}
VOCAB, MAX_POSITION, EPS = 128256, 131072, 1e-5


def listed():
    return [
        # eight answers' tokens as they go into a layer: all latency
        {"name": "rows_8b_8", "kind": "rows", "rows": 8, "features": 4096},
        # a prompt's portion in front of the widest matrix
        {"name": "rows_8b_8191", "kind": "rows", "rows": 8191, "features": 14336},
        # one answer: a stream of weights
        {"name": "linear_8b_down_1", "kind": "linear", "size": "8b_down", "rows": 1, "norm": False, "residual": True},
        # sixteen answers with drafted tokens
        {"name": "linear_8b_qkv_53", "kind": "linear", "size": "8b_qkv", "rows": 53, "norm": True, "residual": False},
        # a server's full step of answers
        {"name": "linear_8b_gate_up_212", "kind": "linear", "size": "8b_gate_up", "rows": 212, "norm": True, "residual": False},
        # a prompt's portion: the largest product
        {"name": "linear_8b_up_8191", "kind": "linear", "size": "8b_up", "rows": 8191, "norm": True, "residual": False},
        # a layer's rows of thirty-two answers, each into a page of its own
        {"name": "append_8b_32", "kind": "append", "size": "8b", "fused": False, "decodes": 32, "drafts": 0, "context": 3000, "prompts": 0, "tokens": 0, "behind": 0},
        # a layer's rows of an 8191-token portion, lying side by side as one projection wrote them
        {"name": "append_8b_8191", "kind": "append", "size": "8b", "fused": True, "decodes": 0, "drafts": 0, "context": 0, "prompts": 1, "tokens": 8191, "behind": 1000},
        # one answer with four drafted tokens in a long conversation: few rows, one long axis
        {"name": "attend_8b_draft_1", "kind": "attend", "size": "8b", "decodes": 1, "drafts": 4, "context": 9000, "prompts": 0, "tokens": 0, "behind": 0},
        # forty answers with up to five drafted tokens each
        {"name": "attend_8b_draft_40", "kind": "attend", "size": "8b", "decodes": 40, "drafts": 5, "context": 6000, "prompts": 0, "tokens": 0, "behind": 0},
        # portions of three prompts beside the next tokens of twenty-nine answers, head size 64
        {"name": "attend_1b_mixed_32", "kind": "attend", "size": "1b", "decodes": 29, "drafts": 0, "context": 1500, "prompts": 3, "tokens": 700, "behind": 500},
        # a portion of a long document behind what was read before
        {"name": "attend_8b_prompt_2048", "kind": "attend", "size": "8b", "decodes": 0, "drafts": 0, "context": 0, "prompts": 1, "tokens": 2048, "behind": 15000},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rows", "linear", "linear", "linear", "append", "append", "attend", "attend", "attend"])
    if kind == "rows":
        return {"kind": kind, "rows": _log_int(rng, 1, 8000), "features": 16 * _log_int(rng, 4, 896)}
    if kind == "linear":
        size = rng.choice(list(LINEARS))
        most = min(8191, 8191 * 4096 * 14336 // (LINEARS[size][0] * LINEARS[size][1]))
        return {"kind": kind, "size": size, "rows": _log_int(rng, 1, most), "norm": rng.choice([False, True]), "residual": rng.choice([False, True])}
    decodes = rng.choice([0, _log_int(rng, 1, 48)])
    prompts = rng.choice([0, 1, rng.randint(1, 4)]) if decodes else rng.randint(1, 4)
    case = {"kind": kind, "size": rng.choice(["1b", "8b", "8b", "70b", "tiny"]), "decodes": decodes, "drafts": rng.randint(0, 7),
            "context": _log_int(rng, 5, 60000 // max(8, decodes)), "prompts": prompts, "tokens": _log_int(rng, 8, 1600 // max(1, prompts)),
            "behind": rng.choice([0, _log_int(rng, 10, 4000)])}
    if kind == "append":
        case["fused"] = rng.choice([False, True])
    return case


# ---------------------------------------------------------------------------------------------------- inputs
def _lengths(case):
    """(new tokens, tokens in the cache, drafted ones among the new) of every request: answers first, then portions of prompts.  A case's own,
    whatever the seed, so that its work is known."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    got = []
    for _ in range(case["decodes"]):
        drafted = rng.randint(0, case["drafts"]) if case["decodes"] > 1 else case["drafts"]
        got.append((1 + drafted, rng.randint(case["context"] // 2, case["context"] * 3 // 2), drafted))
    for _ in range(case["prompts"]):
        if case["prompts"] + case["decodes"] == 1:
            got.append((case["tokens"], case["behind"], 0))
        else:
            got.append((rng.randint(max(1, case["tokens"] // 2), case["tokens"] * 3 // 2), rng.randint(0, 2 * case["behind"]), 0))
    return got


def _pages(lengths):
    return [(n + c + PAGE - 1) // PAGE for n, c, _ in lengths]


def _runs(lengths):
    """What a step writes, a page a time: (request, page of the request, tokens that lie in it already, first row of the step, rows)."""
    got, row = [], 0
    for s, (n, c, _) in enumerate(lengths):
        at = c
        while at < c + n:
            to = min(c + n, (at // PAGE + 1) * PAGE)
            got.append((s, at // PAGE, at % PAGE, row + at - c, to - at))
            at = to
        row += n
    return got


def _ints(values):
    return torch.tensor(values, dtype=I32, device="cuda")


def _normal(g, *shape, std=1.0):
    return (std * torch.randn(shape, generator=g, device="cuda")).to(BF16)


def _freqs(dim):
    return 500000.0 ** (torch.arange(0, dim, 2, dtype=F32, device="cuda") / dim)


def _activations(g, rows, features):
    """A residual stream's rows: another size for each token, some features much larger than the rest."""
    x = torch.randn((rows, features), generator=g, device="cuda") * torch.exp(0.5 * torch.randn((rows, 1), generator=g, device="cuda"))
    return (x * torch.where(torch.rand(features, generator=g, device="cuda") < 0.004, 12.0, 1.0)).to(BF16)


def _cache(g, pages, heads, dim, std):
    """A cache's pages as earlier steps left them: codes and a scale for each page and head."""
    x = std * torch.randn((pages, heads, PAGE, dim), generator=g, device="cuda")
    # (a page that is being filled has seen other tokens, so its scale is now and then a step lower or higher than the next token needs)
    scales = torch.exp2(torch.floor(torch.log2(x.abs().amax((2, 3)))) - 8 + torch.randint(0, 2, (pages, heads), generator=g, device="cuda"))
    return (x / scales[..., None, None]).clamp(-448, 448).to(F8), scales


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = {"kind": case["kind"]}
    if case["kind"] == "rows":
        state["x"] = _activations(g, case["rows"], case["features"])
        return state
    if case["kind"] == "linear":
        k, n = LINEARS[case["size"]]
        w = torch.randn((n, k), generator=g, device="cuda") * k ** -0.5 * torch.exp(0.3 * torch.randn((n, 1), generator=g, device="cuda"))
        scales = w.abs().amax(1) / 127
        state.update(x=_activations(g, case["rows"], k), weight=(w / scales[:, None]).round().to(I8), scales=scales,
                     norm=1 + _normal(g, k, std=0.1) if case["norm"] else None, residual=_normal(g, case["rows"], n) if case["residual"] else None)
        return state
    lengths = _lengths(case)
    hq, hkv, d = HEADS[case["size"]]
    rows, pages = sum(n for n, _, _ in lengths), _pages(lengths)
    n_pages = sum(pages) + 3
    ids = torch.randperm(n_pages, generator=g, device="cuda")[:sum(pages)]
    state.update(ids=torch.randint(0, VOCAB, (rows,), generator=g, device="cuda").to(I32), new=_ints([n for n, _, _ in lengths]), cached=_ints([c for _, c, _ in lengths]),
                 pages=ids.to(I32), n_pages=n_pages, width=max(pages), heads=hq, kv_heads=hkv)
    state["k_pool"], state["k_scales"] = _cache(g, n_pages, hkv, d, 1.0)
    state["v_pool"], state["v_scales"] = _cache(g, n_pages, hkv, d, 0.6)
    if case["kind"] == "attend":
        # queries of unit keys' scores with a spread of two, so that a row attends to some of its keys and not to all alike
        state.update(q=_normal(g, rows, hq, d, std=2.0), scale=d ** -0.5, groups=[_group(lengths, 0, case["decodes"]), _group(lengths, case["decodes"], len(lengths))])
    else:
        if case["fused"]:
            side = _normal(g, rows, (hq + 2 * hkv) * d)
            q, k, v = (t.view(rows, -1, d) for t in side.split([hq * d, hkv * d, hkv * d], 1))
        else:
            q, k, v = _normal(g, rows, hq, d), _normal(g, rows, hkv, d), _normal(g, rows, hkv, d)
        # where the step's rows go: pages written to, the tokens they hold already, the row that each of their places gets (the last: none)
        runs, firsts = _runs(lengths), [sum(pages[:s]) for s in range(len(pages))]
        places = torch.arange(PAGE, device="cuda")[None]
        before, first, count = (torch.tensor([r[i] for r in runs], device="cuda")[:, None] for i in (2, 3, 4))
        there = (places >= before) & (places < before + count)
        state.update(q=q, k=k, v=v, freqs=_freqs(d), positions=torch.cat([torch.arange(c, c + n) for n, c, _ in lengths]).to("cuda"), before=before,
                     written=ids[torch.tensor([firsts[r[0]] + r[1] for r in runs], device="cuda")], rows_of=torch.where(there, first + places - before, rows))
    if own:
        from proxy_inference_engine_b200.ragged import StepPlan

        state["plan"] = StepPlan.build(state["ids"], state["new"], state["cached"], state["pages"], num_pages=n_pages, max_blocks=state["width"], num_heads=hq, num_kv_heads=hkv)
    return state


def _group(lengths, first, last):
    """Requests first .. last - 1, as the plain form pads them: (first, how many, most new tokens, most pages)."""
    some = lengths[first:last]
    return first, len(some), max([n for n, _, _ in some], default=0), max(_pages(some), default=0)


# ---------------------------------------------------------------------------------------------------- one pass
def _codes(x):
    """(whole numbers as 32-bit floats, scales) of rows."""
    scales = x.abs().amax(1, keepdim=True) / 127
    return torch.where(scales > 0, (x / scales).round().clamp(-127, 127), 0.0), scales


def _run_rows(state):
    if own:
        from proxy_inference_engine_b200 import ops

        codes, scales = ops.int8_rows(state["x"])
        return {"codes": codes, "scales": scales}
    codes, scales = _codes(state["x"].float())
    return {"codes": codes.to(I8), "scales": scales[:, 0]}


def _run_linear(state):
    x, weight, scales, norm, residual = (state[n] for n in ("x", "weight", "scales", "norm", "residual"))
    if own:
        from proxy_inference_engine_b200 import ops

        return ops.int8_linear(x, weight, scales, norm_weight=norm, eps=EPS, residual=residual)
    x = x.float()
    if norm is not None:
        x = (x * (x.square().mean(1, keepdim=True) + EPS).rsqrt()).to(BF16).float()
        x = (x * norm.float()).to(BF16).float()
    codes, of = _codes(x)
    y = (torch.matmul(codes, weight.float().t()) * of * scales).to(BF16)
    return y if residual is None else (residual.float() + y.float()).to(BF16)


def _turn(x, cos, sin):
    a, b = x.float().chunk(2, -1)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _write(x, pool, scales, state):
    """Rows x [T, heads, features] into their pages."""
    pages, before, rows_of = state["written"], state["before"], state["rows_of"]
    new = torch.cat([x, torch.zeros_like(x[:1])])[rows_of].transpose(1, 2)
    amax = new.abs().amax((2, 3))
    mantissa, power = torch.frexp(amax)
    need = torch.exp2((power - 9 + (mantissa > 0.875)).clamp(min=-60).where(amax > 0, -60).float())
    had = torch.where(before > 0, scales[pages], 0.0)
    scale = torch.maximum(had, need)
    places = torch.arange(PAGE, device="cuda")[None]
    old = pool[pages].float()
    values = torch.where((places < before)[:, None, :, None], old * (had / scale)[..., None, None], old)
    values = torch.where((rows_of < len(x))[:, None, :, None], new / scale[..., None, None], values)
    pool[pages] = values.to(F8)
    scales[pages] = scale


def _run_append(state):
    q, k, v, freqs, positions, k_pool, v_pool = (state[n] for n in ("q", "k", "v", "freqs", "positions", "k_pool", "v_pool"))
    if own:
        from proxy_inference_engine_b200 import ops

        q = ops.rope_kv_fp8(q, k, v, freqs, state["plan"], k_pool, state["k_scales"], v_pool, state["v_scales"])
        return {"q": q, "k_pool": k_pool, "k_scales": state["k_scales"], "v_pool": v_pool, "v_scales": state["v_scales"]}
    # the angle is the product of two 32-bit numbers rounded to 32 bits, by definition; what is made of it is not
    angle = (positions.float()[:, None] * (1.0 / freqs)[None]).double()[:, None]
    cos, sin = angle.cos().float(), angle.sin().float()
    _write(_turn(k, cos, sin), k_pool, state["k_scales"], state)
    _write(v.float(), v_pool, state["v_scales"], state)
    return {"q": _turn(q, cos, sin).to(BF16), "k_pool": k_pool, "k_scales": state["k_scales"], "v_pool": v_pool, "v_scales": state["v_scales"]}


def _before(counts):
    """Sums of what comes before each, and the whole sum behind the last."""
    return torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), counts.long().cumsum(0)])


def _attend(state, starts, first_page, group, out):
    """The requests of a group, padded to its longest; rows that are padding go to a last row of out, which is dropped."""
    first, count, most, blocks = group
    if count == 0:
        return
    q, hq, hkv, d = state["q"], state["heads"], state["kv_heads"], state["q"].shape[2]
    mine = slice(first, first + count)
    new, cached = state["new"][mine].long(), state["cached"][mine].long()
    tokens, keys = torch.arange(most, device="cuda"), torch.arange(blocks * PAGE, device="cuda")
    rows = torch.where(tokens[None] < new[:, None], starts[mine][:, None] + tokens[None], len(q))
    pages = state["pages"].long()[(first_page[mine][:, None] + keys[None, ::PAGE] // PAGE).clamp(max=len(state["pages"]) - 1)]
    # [requests, heads, keys, features]
    k, v = ((state[n + "_pool"][pages].float() * state[n + "_scales"][pages][..., None, None]).transpose(1, 2).reshape(count, hkv, -1, d) for n in "kv")
    x = q[rows.clamp(max=len(q) - 1)].float().view(count, most, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(count, hkv, -1, d)
    scores = torch.matmul(x, k.transpose(2, 3)).mul_(state["scale"]).view(count, hkv, most, hq // hkv, -1)
    seen = keys[None, None] <= (cached[:, None] + tokens[None])[..., None]
    scores.masked_fill_(~seen[:, None, :, None], -math.inf)
    weights = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    weights = weights.div_(weights.sum(-1, keepdim=True)).view(count, hkv, -1, keys.numel())
    got = torch.matmul(weights, v).view(count, hkv, most, hq // hkv, d).permute(0, 2, 1, 3, 4)
    out[rows.view(-1)] = got.reshape(count * most, hq * d).to(BF16)


def _run_attend(state):
    if own:
        from proxy_inference_engine_b200 import ops

        return ops.chunk_attention_fp8(state["q"], state["k_pool"], state["k_scales"], state["v_pool"], state["v_scales"], state["plan"], state["scale"])
    starts = _before(state["new"])
    first_page = _before((state["new"] + state["cached"] + PAGE - 1) // PAGE)
    out = torch.empty((len(state["q"]) + 1, state["heads"] * state["q"].shape[2]), dtype=BF16, device="cuda")
    _attend(state, starts, first_page, state["groups"][0], out)
    _attend(state, starts, first_page, state["groups"][1], out)
    return out[:-1]


def run(state):
    if state["kind"] == "rows":
        return _run_rows(state)
    if state["kind"] == "linear":
        return _run_linear(state)
    if state["kind"] == "append":
        return _run_append(state)
    return _run_attend(state)


# ---------------------------------------------------------------------------------------------------- what it takes, and what comes out
def work(case):
    if case["kind"] == "rows":
        return {"bytes": 3 * case["rows"] * case["features"] + 4 * case["rows"], "flops": 2 * case["rows"] * case["features"]}
    if case["kind"] == "linear":
        m, (k, n) = case["rows"], LINEARS[case["size"]]
        return {"bytes": 2 * m * k + n * k + 4 * n + 2 * m * n * (2 if case["residual"] else 1) + (2 * k if case["norm"] else 0), "flops": 2 * m * n * k}
    lengths = _lengths(case)
    hq, hkv, d = HEADS[case["size"]]
    rows = sum(n for n, _, _ in lengths)
    if case["kind"] == "append":
        scales = 4 * 2 * hkv * sum(2 if r[2] else 1 for r in _runs(lengths))
        return {"bytes": rows * d * (4 * hq + 6 * hkv) + 8 * rows + scales + 2 * d, "flops": 3 * rows * (hq + hkv) * d}
    pairs = sum(n * c + n * (n + 1) // 2 for n, c, _ in lengths)
    read = 2 * hkv * (sum(n + c for n, c, _ in lengths) * d + 4 * sum(_pages(lengths)))
    return {"bytes": 4 * rows * hq * d + read + 4 * sum(_pages(lengths)), "flops": 4 * pairs * hq * d}


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "rows":
        return _exact_rows(state["x"].double())
    if case["kind"] == "linear":
        return _exact_linear(state)
    if case["kind"] == "append":
        return _exact_append(_lengths(case), state)
    return _exact_attend(_lengths(case), state)


def _exact_rows(x):
    top = torch.maximum(x.amax(1), -x.amin(1))
    return {"codes": torch.round(x * (127 / top)[:, None]).to(I8), "scales": top / 127}


def _exact_linear(state):
    x = state["x"].double()
    if state["norm"] is not None:
        # the norm's rows are of 16 bits, the product's with its weight too
        x = (x / torch.sqrt(EPS + torch.einsum("mk,mk->m", x, x) / x.shape[1])[:, None]).to(BF16).double()
        x = (x * state["norm"].double()).to(BF16).double()
    got = _exact_rows(x)
    y = got["codes"].double() @ (state["weight"].double() * state["scales"].double()[:, None]).T * got["scales"][:, None]
    return y if state["residual"] is None else y + state["residual"].double()


def _to_e4m3(x):
    """The nearest number of three bits behind the first, none finer than 2^-9; of two as near, the even one."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_append(lengths, state):
    """Page by page and head by head."""
    q, k, v = (state[n].double() for n in ("q", "k", "v"))
    angle = (state["positions"].float()[:, None] * state["freqs"].reciprocal()[None]).double()
    half = q.shape[2] // 2
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    turned = [torch.view_as_real(torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * turn) for x in (q, k)]
    q, k = (torch.cat([t[..., 0], t[..., 1]], -1) for t in turned)
    got = {"q": q}
    for name, x in (("k", k), ("v", v)):
        pool, scales = state[name + "_pool"].double(), state[name + "_scales"].double()
        for (_, _, lies, row, count), page in zip(_runs(lengths), state["written"].tolist()):
            new = x[row:row + count].transpose(0, 1)
            top = new.abs().flatten(1).amax(1)
            scale = torch.exp2(torch.ceil(torch.log2(top.clamp(min=448 * 2.0 ** -60) / 448)))
            if lies:
                scale = torch.maximum(scale, scales[page])
                pool[page, :, :lies] = _to_e4m3(pool[page, :, :lies] * (scales[page] / scale)[:, None, None])
            pool[page, :, lies:lies + count] = _to_e4m3(new / scale[:, None, None])
            scales[page] = scale
        got[name + "_pool"], got[name + "_scales"] = pool, scales
    return got


def _exact_attend(lengths, state):
    """Request by request and head by head."""
    hq, hkv, d = state["heads"], state["kv_heads"], state["q"].shape[2]
    out = torch.empty((len(state["q"]), hq, d), dtype=F64, device="cuda")
    row = page = 0
    for n, c, _ in lengths:
        mine = state["pages"].long()[page:page + (n + c + PAGE - 1) // PAGE]
        page += len(mine)
        beyond = torch.arange(n + c, device="cuda")[None] > torch.arange(c, c + n, device="cuda")[:, None]
        for h in range(hkv):
            k, v = ((state[x + "_pool"][mine, h].double() * state[x + "_scales"][mine, h].double()[:, None, None]).flatten(0, 1)[:n + c] for x in "kv")
            for i in range(h * hq // hkv, (h + 1) * hq // hkv):
                scores = state["scale"] * (state["q"][row:row + n, i].double() @ k.t())
                out[row:row + n, i] = scores.masked_fill_(beyond, -math.inf).softmax(1) @ v
        row += n
    return out.flatten(1)
