"""The operators of a ragged step in 64 bits, request by request (tests of ragged.StepPlan, ops.rope_kv_slots, ops.chunk_attention, ops.verify_draft)."""
from __future__ import annotations

import numpy as np
import torch

PAGE = 64


def need(n, c):
    return (n + c + PAGE - 1) // PAGE


def plan(ids, new, cached, pages, width, drafted=None, T=None, R=None):
    """pages: a list per request.  The arrays of StepPlan as lists, padded to T rows and R logit rows."""
    T, R = T or len(ids), R or len(new)
    got = {n: [] for n in ("row_starts", "contexts", "sequences", "positions", "slots", "block_table", "logit_rows", "logit_starts", "draft_tokens")}
    row = 0
    for s, (n, c) in enumerate(zip(new, cached)):
        k = drafted[s] if drafted and n else 0
        got["row_starts"].append(row)
        got["contexts"].append(c)
        got["logit_starts"].append(len(got["logit_rows"]))
        got["sequences"] += [s] * n
        got["positions"] += list(range(c, c + n))
        got["slots"] += [pages[s][p // PAGE] * PAGE + p % PAGE for p in range(c, c + n)]
        got["block_table"].append(pages[s][:need(n, c)] + [0] * (width - need(n, c)))
        row += n
        if n:
            got["logit_rows"] += list(range(row - 1 - k, row))
            got["draft_tokens"] += list(ids[row - k:row]) + [-1]
    got["row_starts"].append(row)
    got["logit_starts"].append(len(got["logit_rows"]))
    for name, fill, size in (("sequences", -1, T), ("positions", 0, T), ("slots", -1, T), ("logit_rows", 0, R), ("draft_tokens", -1, R)):
        got[name] += [fill] * (size - len(got[name]))
    return got


def rope(x, positions, freqs):
    """x [T, H, D] bf16 -> float64; the angle is a product of 32-bit numbers rounded to 32 bits."""
    angle = (positions.cpu().float()[:, None] * (1.0 / freqs.cpu().float())[None]).double()
    a, b = x.cpu().double().chunk(2, -1)
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def attention(q, k_pool, v_pool, new, cached, tables, scale):
    """(out, weight) [T, Hq, D] float64: softmax(scale q k) v over the keys 0 .. position of each row, and the same sum over |v|, which bounds what a rounding of
    the weights does."""
    q, T = q.cpu().double(), q.shape[0]
    Hq, D = q.shape[1:]
    Hkv = k_pool.shape[2]
    k_pool, v_pool = k_pool.cpu(), v_pool.cpu()
    out, weight = torch.zeros((T, Hq, D), dtype=torch.float64), torch.zeros((T, Hq, D), dtype=torch.float64)
    row = 0
    for n, c, table in zip(new, cached, tables):
        if n:
            at = torch.tensor(table[:need(n, c)])
            k = k_pool[at].reshape(-1, Hkv, D)[:n + c].double().repeat_interleave(Hq // Hkv, 1)
            v = v_pool[at].reshape(-1, Hkv, D)[:n + c].double().repeat_interleave(Hq // Hkv, 1)
            s = scale * torch.einsum("thd,jhd->htj", q[row:row + n], k)
            beyond = torch.arange(n + c)[None] > torch.arange(c, c + n)[:, None]
            p = s.masked_fill(beyond, -torch.inf).softmax(-1)
            out[row:row + n] = torch.einsum("htj,jhd->thd", p, v)
            weight[row:row + n] = torch.einsum("htj,jhd->thd", p, v.abs())
        row += n
    return out, weight


def verify(logits, draft_tokens, starts, most, temp, uniforms=None, noise=None, draft_logits=None):
    """(tokens, logprobs, sure) per request; sure: no decision of it lies within 1e-5 of its border (32 bits may fall to the other side of those)."""
    logits = logits.cpu().double().numpy()
    guess = None if draft_logits is None else draft_logits.cpu().double().numpy()
    given = draft_tokens.tolist()
    soft = lambda x: (lambda e: e / e.sum())(np.exp(x - x.max()))
    got = []
    for s in range(len(starts) - 1):
        tokens, logprobs, sure = [], [], True
        rows = list(range(starts[s], starts[s + 1]))[:most + 1]
        for r in rows:
            x, last = given[r], r == rows[-1]
            t = logits[r] / (temp or 1.0)
            with np.errstate(all="ignore"):
                p = soft(t)
                logp = t - t.max() - np.log(np.exp(t - t.max()).sum())
            real = 0 <= x < len(p)
            if temp == 0:
                best = int(np.nanargmax(np.where(np.isnan(logits[r]), -np.inf, logits[r])))
                emit = None if not last and best == x else best
            else:
                q = np.zeros_like(p) if guess is None else soft(guess[r] / temp)
                if guess is None and real:
                    q[x] = 1.0
                refuse = True
                if not last and real:
                    left, right = float(uniforms[r]) * q[x], p[x]
                    refuse = not left < right
                    sure = sure and (left == right == 0.0 or abs(left - right) > 1e-5 * max(left, right))
                emit = None
                if last or refuse:
                    w = p if last else np.maximum(p - q, 0.0)
                    if not (w > 0).any():
                        w = p
                    with np.errstate(all="ignore"):
                        race = w / -np.log(noise[s].cpu().double().numpy())
                    race[np.isnan(race)] = 0.0
                    emit = int(race.argmax())
                    if not (race > 0).any():
                        emit = 0
                    else:
                        two = np.partition(race, -2)[-2:] if len(race) > 1 else [0.0, race[0]]
                        # the weights of a refusal are differences: what 32 bits leave of them goes by what they were
                        sure = sure and two[1] - two[0] > 1e-5 * two[1] * (1.0 if last or guess is None else max(1.0, p[emit] / w[emit]))
            tokens.append(x if emit is None else emit)
            logprobs.append(logp[tokens[-1]])
            if emit is not None:
                break
        got.append((tokens, logprobs, sure))
    return got
