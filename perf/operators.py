"""The operators of a ragged step, at the sizes its users run: a step whose requests each bring another number of new tokens -- a
prompt's portion, the next token of an answer, or that token and some drafted ones -- over a paged cache.

Kinds (``case["kind"]``) and what one pass runs:
    plan    rows, positions, cache slots, block table and logit rows of a step, from the requests' lengths (ragged.StepPlan.build)
    rope    rotation of the step's queries and keys, and keys and values written to their cache slots (ops.rope_kv_slots)
    chunk   causal attention of every request's new tokens over its pages (ops.chunk_attention)
    verify  drafted tokens against the target's probabilities, and the token behind the accepted ones (ops.verify_draft)

Sizes are those of the Llama presets (``checkpoint.LLAMA_PRESETS``) and of the tests' small model.  With ``own`` false a pass is the plain
form: elementary torch operations, the requests padded to the longest of their kind.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
PAGE = 64
# query heads, key / value heads, head size
HEADS = {"1b": (32, 8, 64), "8b": (32, 8, 128), "70b": (64, 8, 128), "tiny": (4, 2, 64)}
VOCAB = {"llama": 128256, "small": 32000, "odd": 50257, "tiny": 640}
MAX_POSITION = 131072


def listed():
    return [
        # eight answers, a token each: the smallest step, all latency
        {"name": "plan_decode_8", "kind": "plan", "size": "8b", "decodes": 8, "drafts": 0, "context": 1000, "prompts": 0, "tokens": 0, "behind": 0},
        # a server's full step: two hundred answers with drafted tokens beside a dozen portions of prompts
        {"name": "plan_mixed_212", "kind": "plan", "size": "8b", "decodes": 200, "drafts": 5, "context": 3000, "prompts": 12, "tokens": 900, "behind": 1500},
        # a layer's rows of thirty-two answers
        {"name": "rope_8b_32", "kind": "rope", "size": "8b", "rows": 32, "fused": False},
        # a layer's rows of an 8191-token portion, lying side by side as one projection wrote them
        {"name": "rope_8b_8191", "kind": "rope", "size": "8b", "rows": 8191, "fused": True},
        # one answer with four drafted tokens in a long conversation: few rows, one long axis
        {"name": "chunk_8b_draft_1", "kind": "chunk", "size": "8b", "decodes": 1, "drafts": 4, "context": 9000, "prompts": 0, "tokens": 0, "behind": 0},
        # sixteen answers with up to five drafted tokens each
        {"name": "chunk_8b_draft_16", "kind": "chunk", "size": "8b", "decodes": 16, "drafts": 5, "context": 4000, "prompts": 0, "tokens": 0, "behind": 0},
        # portions of three prompts beside the next tokens of twenty-nine answers, head size 64
        {"name": "chunk_1b_mixed_32", "kind": "chunk", "size": "1b", "decodes": 29, "drafts": 0, "context": 1500, "prompts": 3, "tokens": 700, "behind": 500},
        # a portion of a long document behind what was read before: the largest call
        {"name": "chunk_8b_prompt_2048", "kind": "chunk", "size": "8b", "decodes": 0, "drafts": 0, "context": 0, "prompts": 1, "tokens": 2048, "behind": 15000},
        # one greedy answer, four drafted tokens
        {"name": "verify_greedy_1", "kind": "verify", "vocab": "llama", "sequences": 1, "drafts": 4, "temp": 0.0, "drafter": "lookup"},
        # sixteen greedy answers, seven drafted tokens each
        {"name": "verify_greedy_16", "kind": "verify", "vocab": "llama", "sequences": 16, "drafts": 7, "temp": 0.0, "drafter": "lookup"},
        # thirty-two sampled answers whose drafts were looked up in the prompt
        {"name": "verify_lookup_32", "kind": "verify", "vocab": "llama", "sequences": 32, "drafts": 5, "temp": 0.8, "drafter": "lookup"},
        # sixty-four sampled answers whose drafts a smaller model drew
        {"name": "verify_model_64", "kind": "verify", "vocab": "llama", "sequences": 64, "drafts": 5, "temp": 1.0, "drafter": "model"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "rope", "chunk", "chunk", "chunk", "verify", "verify"])
    size = rng.choice(["1b", "8b", "8b", "70b", "tiny"])
    if kind == "plan":
        return {"kind": kind, "size": size, "decodes": _log_int(rng, 1, 200), "drafts": rng.randint(0, 6), "context": _log_int(rng, 20, 4000),
                "prompts": rng.choice([0, _log_int(rng, 1, 12)]), "tokens": _log_int(rng, 10, 900), "behind": rng.choice([0, _log_int(rng, 10, 1500)])}
    if kind == "rope":
        return {"kind": kind, "size": size, "rows": _log_int(rng, 1, 4000), "fused": rng.choice([False, True])}
    if kind == "chunk":
        decodes = rng.choice([0, _log_int(rng, 1, 48)])
        prompts = rng.choice([0, 1, rng.randint(1, 4)]) if decodes else rng.randint(1, 4)
        return {"kind": kind, "size": size, "decodes": decodes, "drafts": rng.randint(0, 7), "context": _log_int(rng, 5, 60000 // max(8, decodes)),
                "prompts": prompts, "tokens": _log_int(rng, 8, 1600 // max(1, prompts)), "behind": rng.choice([0, _log_int(rng, 10, 4000)])}
    temp = rng.choice([0.0, 0.6, 1.0])
    return {"kind": kind, "vocab": rng.choice(list(VOCAB)), "sequences": _log_int(rng, 1, 48), "drafts": rng.randint(1, 7), "temp": temp,
            "drafter": "lookup" if temp == 0.0 else rng.choice(["lookup", "model"])}


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


def _drafted(case):
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    return [rng.randint(0, case["drafts"]) if case["sequences"] > 1 else case["drafts"] for _ in range(case["sequences"])]


def _pages(lengths):
    return [(n + c + PAGE - 1) // PAGE for n, c, _ in lengths]


def _ints(values):
    return torch.tensor(values, dtype=I32, device="cuda")


def _starts(counts):
    got = [0]
    for n in counts:
        got.append(got[-1] + n)
    return got


def _normal(g, *shape, std=1.0):
    return (std * torch.randn(shape, generator=g, device="cuda")).to(BF16)


def _freqs(dim):
    return 500000.0 ** (torch.arange(0, dim, 2, dtype=F32, device="cuda") / dim)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = {"kind": case["kind"]}
    if case["kind"] in ("plan", "chunk"):
        lengths = _lengths(case)
        hq, hkv, d = HEADS[case["size"]]
        pages = _pages(lengths)
        n_pages = sum(pages) + 3
        state.update(ids=torch.randint(0, VOCAB["llama"], (sum(n for n, _, _ in lengths),), generator=g, device="cuda").to(I32),
                     new=_ints([n for n, _, _ in lengths]), cached=_ints([c for _, c, _ in lengths]), drafted=_ints([k for _, _, k in lengths]),
                     pages=torch.randperm(n_pages, generator=g, device="cuda")[:sum(pages)].to(I32), n_pages=n_pages, width=max(pages),
                     logit_rows=sum(k + 1 for _, _, k in lengths), heads=hq, kv_heads=hkv)
        if case["kind"] == "chunk":
            # queries of unit keys' scores with a spread of two, so that a row attends to some of its keys and not to all alike
            state.update(q=_normal(g, len(state["ids"]), hq, d, std=2.0), k=_normal(g, n_pages, PAGE, hkv, d), v=_normal(g, n_pages, PAGE, hkv, d, std=0.6),
                         scale=d ** -0.5, groups=[_group(lengths, 0, case["decodes"]), _group(lengths, case["decodes"], len(lengths))])
            if own:
                state["plan"] = _plan(state)
    elif case["kind"] == "rope":
        hq, hkv, d = HEADS[case["size"]]
        rows, n_pages = case["rows"], case["rows"] // PAGE + 2
        if case["fused"]:
            side = _normal(g, rows, (hq + 2 * hkv) * d)
            q, k, v = (t.view(rows, -1, d) for t in side.split([hq * d, hkv * d, hkv * d], 1))
        else:
            q, k, v = _normal(g, rows, hq, d), _normal(g, rows, hkv, d), _normal(g, rows, hkv, d)
        state.update(q=q, k=k, v=v, freqs=_freqs(d), positions=torch.randint(0, MAX_POSITION, (rows,), generator=g, device="cuda").to(I32),
                     slots=torch.randperm(n_pages * PAGE, generator=g, device="cuda")[:rows].to(I32),
                     k_pool=_normal(g, n_pages, PAGE, hkv, d), v_pool=_normal(g, n_pages, PAGE, hkv, d))
    else:
        drafted, vocab = _drafted(case), VOCAB[case["vocab"]]
        starts = _starts([k + 1 for k in drafted])
        rows = starts[-1]
        logits = 2.5 * torch.randn((rows, vocab), generator=g, device="cuda")
        # a trained model is often sure of its token
        sure = torch.randint(0, vocab, (rows, 1), generator=g, device="cuda")
        logits.scatter_add_(1, sure, 6 + 8 * torch.rand((rows, 1), generator=g, device="cuda"))
        state.update(logits=logits.to(BF16), starts=_ints(starts), most=case["drafts"], temp=case["temp"], uniforms=None, noise=None, draft_logits=None)
        if case["drafter"] == "model":
            guess = logits + 0.7 * torch.randn((rows, vocab), generator=g, device="cuda")
            state["draft_logits"] = guess.to(BF16)
            race = torch.rand((rows, vocab), generator=g, device="cuda").log_().neg_()
            tokens = (state["draft_logits"].float() / case["temp"]).softmax(1).div_(race).argmax(1)
        else:
            tokens = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.8, logits.argmax(1), torch.randint(0, vocab, (rows,), generator=g, device="cuda"))
        state["tokens"] = tokens.to(I32)
        if case["temp"] > 0:
            state.update(uniforms=torch.rand(rows, generator=g, device="cuda"), noise=torch.rand((len(drafted), vocab), generator=g, device="cuda"))
    return state


def _group(lengths, first, last):
    """Requests first .. last - 1, as the plain form pads them: (first, how many, most new tokens, most pages)."""
    some = lengths[first:last]
    return first, len(some), max([n for n, _, _ in some], default=0), max(_pages(some), default=0)


# ---------------------------------------------------------------------------------------------------- one pass
def _plan(state):
    from proxy_inference_engine_b200.ragged import StepPlan

    return StepPlan.build(state["ids"], state["new"], state["cached"], state["pages"], num_pages=state["n_pages"], max_blocks=state["width"],
                          draft_lengths=state["drafted"], num_logits=state["logit_rows"], num_heads=state["heads"], num_kv_heads=state["kv_heads"])


def _before(counts):
    """Sums of what comes before each, and the whole sum behind the last."""
    return torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), counts.long().cumsum(0)])


def _run_plan(state):
    if own:
        p = _plan(state)
        return {"row_starts": p.row_starts, "sequences": p.sequences, "positions": p.positions, "slots": p.slots, "block_table": p.block_table,
                "logit_rows": p.logit_rows, "logit_starts": p.logit_starts, "draft_tokens": p.draft_tokens}
    new, cached, drafted, pages = state["new"].long(), state["cached"].long(), state["drafted"].long(), state["pages"].long()
    starts, logit_starts = _before(new), _before(drafted + 1)
    rows = torch.arange(len(state["ids"]), device="cuda")
    seq = (rows[:, None] >= starts[None, 1:]).sum(1)
    positions = cached[seq] + rows - starts[seq]
    need = (new + cached + PAGE - 1) // PAGE
    blocks, first = torch.arange(state["width"], device="cuda"), _before(need)[:-1]
    table = torch.where(blocks[None] < need[:, None], pages[(first[:, None] + blocks[None]).clamp(max=len(pages) - 1)], 0)
    slots = table[seq, positions // PAGE] * PAGE + positions % PAGE
    at = torch.arange(state["logit_rows"], device="cuda")
    of = (at[:, None] >= logit_starts[None, 1:]).sum(1)
    logit_rows = starts[of + 1] - logit_starts[of + 1] + at
    follows = state["ids"].long()[(logit_rows + 1).clamp(max=len(rows) - 1)]
    draft_tokens = torch.where(at + 1 < logit_starts[of + 1], follows, -1)
    got = {"row_starts": starts, "sequences": seq, "positions": positions, "slots": slots, "block_table": table, "logit_rows": logit_rows,
           "logit_starts": logit_starts, "draft_tokens": draft_tokens}
    return {name: t.to(I32) for name, t in got.items()}


def _turn(x, cos, sin):
    a, b = x.float().chunk(2, -1)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1).to(BF16)


def _run_rope(state):
    q, k, v, freqs, positions, slots, k_pool, v_pool = (state[n] for n in ("q", "k", "v", "freqs", "positions", "slots", "k_pool", "v_pool"))
    if own:
        from proxy_inference_engine_b200 import ops

        return {"q": ops.rope_kv_slots(q, k, v, freqs, positions, slots, k_pool, v_pool), "k_pool": k_pool, "v_pool": v_pool}
    # the angle is the product of two 32-bit numbers rounded to 32 bits, by definition; what is made of it is not
    angle = (positions.float()[:, None] * (1.0 / freqs)[None]).double()[:, None]
    cos, sin = angle.cos().float(), angle.sin().float()
    k_pool.view(-1, *k.shape[1:])[slots.long()] = _turn(k, cos, sin)
    v_pool.view(-1, *v.shape[1:])[slots.long()] = v
    return {"q": _turn(q, cos, sin), "k_pool": k_pool, "v_pool": v_pool}


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
    at = (first_page[mine][:, None] + keys[None, ::PAGE] // PAGE).clamp(max=len(state["pages"]) - 1)
    pages = state["pages"].long()[at]
    there = keys[None] < (new + cached)[:, None]
    k = state["k"][pages].view(count, -1, hkv, d).float()
    v = torch.where(there[..., None, None], state["v"][pages].view(count, -1, hkv, d).float(), 0.0)
    x = q[rows.clamp(max=len(q) - 1)].float().view(count, most, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(count, hkv, -1, d)
    scores = torch.matmul(x, k.permute(0, 2, 3, 1)).mul_(state["scale"]).view(count, hkv, most, hq // hkv, -1)
    seen = keys[None, None] <= (cached[:, None] + tokens[None])[..., None]
    scores.masked_fill_(~seen[:, None, :, None], -math.inf)
    weights = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    weights = weights.div_(weights.sum(-1, keepdim=True)).view(count, hkv, -1, keys.numel())
    got = torch.matmul(weights, v.permute(0, 2, 1, 3)).view(count, hkv, most, hq // hkv, d).permute(0, 2, 1, 3, 4)
    out[rows.view(-1)] = got.reshape(count * most, hq * d).to(BF16)


def _run_chunk(state):
    if own:
        from proxy_inference_engine_b200 import ops

        return ops.chunk_attention(state["q"], state["k"], state["v"], state["plan"], state["scale"])
    starts = _before(state["new"])
    first_page = _before((state["new"] + state["cached"] + PAGE - 1) // PAGE)
    out = torch.empty((len(state["q"]) + 1, state["heads"] * state["q"].shape[2]), dtype=BF16, device="cuda")
    _attend(state, starts, first_page, state["groups"][0], out)
    _attend(state, starts, first_page, state["groups"][1], out)
    return out[:-1]


def _first_largest(x):
    index = torch.arange(x.shape[-1], device="cuda")
    return torch.where(x == x.amax(-1, keepdim=True), index, x.shape[-1]).amin(-1)


def _run_verify(state):
    logits, tokens, starts, most, temp = (state[n] for n in ("logits", "tokens", "starts", "most", "temp"))
    if own:
        from proxy_inference_engine_b200 import ops

        got, counts, logprobs = ops.verify_draft(logits, tokens, starts, max_draft=most, temp=temp, uniforms=state["uniforms"], noise=state["noise"],
                                                 draft_logits=state["draft_logits"])
        return {"tokens": got, "counts": counts, "logprobs": logprobs}
    starts, place = starts.long(), torch.arange(most + 1, device="cuda")
    drafted = starts[1:] - starts[:-1] - 1
    rows = (starts[:-1, None] + place[None]).clamp(max=len(logits) - 1)
    given = tokens.long()[rows]
    # in 64 bits: a draw next to its border falls to one side or the other
    scaled = logits.double() / (temp if temp > 0 else 1.0)
    logp = scaled - scaled.logsumexp(1, keepdim=True)
    p_given = logp[rows, given]
    if temp == 0:
        accept = _first_largest(logits)[rows] == given
    elif state["draft_logits"] is None:
        accept = state["uniforms"].double()[rows] < p_given.exp()
    else:
        guess = state["draft_logits"].double() / temp
        logq = guess - guess.logsumexp(1, keepdim=True)
        accept = state["uniforms"].double()[rows] * logq[rows, given].exp() < p_given.exp()
    accepted = (accept & (place[None] < drafted[:, None])).long().cumprod(1).sum(1)
    last = starts[:-1] + accepted
    if temp == 0:
        emitted = _first_largest(logits[last])
    else:
        weight = p = logp[last].exp()
        refused = (accepted < drafted)[:, None]
        if state["draft_logits"] is None:
            weight = torch.where(refused & (torch.arange(logits.shape[1], device="cuda")[None] == tokens.long()[last][:, None]), 0.0, p)
        else:
            weight = torch.where(refused, (p - logq[last].exp()).clamp(min=0), p)
        weight = torch.where(weight.sum(1, keepdim=True) > 0, weight, p)
        emitted = _first_largest(weight / -state["noise"].double().log())
    taken = place[None] < accepted[:, None]
    behind = place[None] == accepted[:, None]
    got = torch.where(taken, given, torch.where(behind, emitted[:, None], -1))
    logprobs = torch.where(taken, p_given, torch.where(behind, logp[last, emitted][:, None], 0.0))
    return {"tokens": got.to(I32), "counts": (accepted + 1).to(I32), "logprobs": logprobs.float()}


def run(state):
    if state["kind"] == "plan":
        return _run_plan(state)
    if state["kind"] == "rope":
        return _run_rope(state)
    if state["kind"] == "chunk":
        return _run_chunk(state)
    return _run_verify(state)


# ---------------------------------------------------------------------------------------------------- what it takes, and what comes out
def work(case):
    if case["kind"] in ("plan", "chunk"):
        lengths = _lengths(case)
        rows, requests, pages = sum(n for n, _, _ in lengths), len(lengths), _pages(lengths)
        if case["kind"] == "plan":
            outs = rows * 3 + requests * max(pages) + 2 * (requests + 1) + 2 * sum(k + 1 for _, _, k in lengths)
            return {"bytes": 4 * (rows + 3 * requests + sum(pages) + outs), "flops": outs}
        hq, hkv, d = HEADS[case["size"]]
        pairs = sum(n * c + n * (n + 1) // 2 for n, c, _ in lengths)
        return {"bytes": 2 * (2 * rows * hq * d + 2 * sum(n + c for n, c, _ in lengths) * hkv * d) + 4 * sum(pages), "flops": 4 * pairs * hq * d}
    if case["kind"] == "rope":
        hq, hkv, d = HEADS[case["size"]]
        return {"bytes": 4 * case["rows"] * (hq + 2 * hkv) * d + 8 * case["rows"] + 2 * d, "flops": 3 * case["rows"] * (hq + hkv) * d}
    drafted, vocab = _drafted(case), VOCAB[case["vocab"]]
    rows = sum(drafted) + len(drafted)
    read = 2 * rows * vocab + (4 * len(drafted) * vocab if case["temp"] > 0 else 0) + (2 * sum(drafted) * vocab if case["drafter"] == "model" else 0)
    return {"bytes": read + 8 * rows + (8 * len(drafted) * (case["drafts"] + 1)), "flops": read}


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "plan":
        return _exact_plan(_lengths(case), state)
    if case["kind"] == "rope":
        return _exact_rope(state)
    if case["kind"] == "chunk":
        return _exact_chunk(_lengths(case), state)
    return _exact_verify(_drafted(case), state)


def _exact_plan(lengths, state):
    """Request by request, in whole numbers."""
    ids, pages = state["ids"].tolist(), state["pages"].tolist()
    got = {n: [] for n in ("row_starts", "sequences", "positions", "slots", "block_table", "logit_rows", "logit_starts", "draft_tokens")}
    row = page = 0
    for s, (n, c, k) in enumerate(lengths):
        mine = pages[page:page + (n + c + PAGE - 1) // PAGE]
        page += len(mine)
        got["row_starts"].append(row)
        got["logit_starts"].append(len(got["logit_rows"]))
        got["sequences"] += [s] * n
        got["positions"] += range(c, c + n)
        got["slots"] += [mine[p // PAGE] * PAGE + p % PAGE for p in range(c, c + n)]
        got["block_table"].append(mine + [0] * (state["width"] - len(mine)))
        row += n
        got["logit_rows"] += range(row - 1 - k, row)
        got["draft_tokens"] += ids[row - k:row] + [-1]
    got["row_starts"].append(row)
    got["logit_starts"].append(len(got["logit_rows"]))
    return {name: torch.tensor(v, dtype=I32) for name, v in got.items()}


def _exact_rope(state):
    q, k, v = (state[n].double() for n in ("q", "k", "v"))
    angle = (state["positions"].float()[:, None] * state["freqs"].reciprocal()[None]).double()
    half = q.shape[2] // 2
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    turned = [torch.view_as_real(torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * turn) for x in (q, k)]
    q, k = (torch.cat([t[..., 0], t[..., 1]], -1) for t in turned)
    k_pool, v_pool = state["k_pool"].double(), state["v_pool"].double()
    page, place = state["slots"].long() // PAGE, state["slots"].long() % PAGE
    k_pool[page, place], v_pool[page, place] = k, v
    return {"q": q, "k_pool": k_pool, "v_pool": v_pool}


def _exact_chunk(lengths, state):
    """Request by request and head by head."""
    hq, hkv, d = state["heads"], state["kv_heads"], state["q"].shape[2]
    out = torch.empty((len(state["q"]), hq, d), dtype=F64, device="cuda")
    row = page = 0
    for n, c, _ in lengths:
        mine = state["pages"].long()[page:page + (n + c + PAGE - 1) // PAGE]
        page += len(mine)
        beyond = torch.arange(n + c, device="cuda")[None] > torch.arange(c, c + n, device="cuda")[:, None]
        for h in range(hq):
            k, v = (state[name][mine, :, h * hkv // hq].double().flatten(0, 1)[:n + c] for name in "kv")
            scores = state["scale"] * (state["q"][row:row + n, h].double() @ k.t())
            out[row:row + n, h] = scores.masked_fill_(beyond, -math.inf).softmax(1) @ v
        row += n
    return out.flatten(1)


def _exact_verify(drafted, state):
    """Request by request, token by token."""
    temp, most = state["temp"], state["most"]
    tokens, row = [], 0
    logprobs = torch.zeros((len(drafted), most + 1), dtype=F64, device="cuda")
    given = state["tokens"].tolist()
    for s, k in enumerate(drafted):
        got = []
        for i in range(row, row + k + 1):
            logits, x = state["logits"][i].double(), given[i]
            logp = (logits / (temp or 1.0)).log_softmax(0)
            if temp == 0:
                best = int((logits == logits.max()).nonzero()[0])
                emit = None if i < row + k and best == x else best
            else:
                weight, emit = logp.exp(), None
                if i < row + k:
                    q = torch.zeros_like(weight)
                    if state["draft_logits"] is None:
                        q[x] = 1.0
                    else:
                        q = (state["draft_logits"][i].double() / temp).softmax(0)
                    refuse = not float(state["uniforms"][i].double() * q[x]) < float(weight[x])
                    left = torch.where(weight > q, weight - q, 0.0)
                    weight = left if float(left.max()) > 0 else weight
                if i == row + k or refuse:
                    emit = int((weight.log() - (-state["noise"][s].double().log()).log()).argmax())
            logprobs[s, len(got)] = logp[x if emit is None else emit]
            got.append(x if emit is None else emit)
            if emit is not None:
                break
        tokens.append(got)
        row += k + 1
    filled = [t + [-1] * (most + 1 - len(t)) for t in tokens]
    return {"tokens": torch.tensor(filled, dtype=I32), "counts": torch.tensor([len(t) for t in tokens], dtype=I32), "logprobs": logprobs}
