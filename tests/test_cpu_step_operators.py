"""What the operators of a ragged step refuse before anything is launched."""
import ctypes as C

import pytest
import torch

from proxy_inference_engine_b200 import _lib, ops
from proxy_inference_engine_b200.ragged import StepPlan

BF = torch.bfloat16
ints = lambda *v: torch.tensor(v, dtype=torch.int32)


def refuses(call, kw):
    """Without anything else wrong: tensors that are not on a CUDA device."""
    with pytest.raises(ValueError) as e:
        call(**kw)
    assert ("CUDA device" in str(e.value)) == (not kw), str(e.value)


def _dims(**kw):
    d = dict(requests=2, rows=10, logit_rows=2, blocks=4, pages=9, Hq=8, Hkv=2)
    d.update(kw)
    return _lib.StepDims(*d.values())


@pytest.mark.parametrize("kw", [dict(requests=0), dict(requests=4097), dict(rows=0), dict(rows=-1), dict(logit_rows=0), dict(blocks=0), dict(pages=0), dict(Hq=0), dict(Hkv=0),
                                dict(Hq=7), dict(Hq=258, Hkv=2), dict(pages=1 << 26), dict(blocks=1 << 26), dict(requests=4096, blocks=1 << 20)])
def test_dimensions(kw):
    L, d = _lib.load(), _dims(**kw)
    assert L.pie_step_plan_words(C.byref(d)) == 0 and L.pie_chunk_attn_workspace_bytes(C.byref(d), 64) == 0
    fake = C.c_void_p(0x1000)
    assert L.pie_step_plan_build(fake, C.byref(d), fake, fake, fake, None, fake, 4, 0, None) == 1
    assert L.pie_step_plan_offsets(C.byref(d), (C.c_longlong * 10)()) == 1


@pytest.mark.parametrize("blocks,fits", [((2 ** 31 - 1) // 64, False), ((2 ** 31 - 1025) // 64 + 1, False), ((2 ** 31 - 1025) // 64, True)])
def test_positions_leave_room_for_a_tile_behind_them(blocks, fits):
    """A request of as many keys as its row of the table holds: what is added to them -- a tile, an item's cost -- has to fit 32 bits."""
    assert (_lib.load().pie_step_plan_words(C.byref(_dims(blocks=blocks))) > 0) == fits
    assert not fits or blocks * 64 + 1024 <= 2 ** 31 - 1


def test_offsets_are_apart_and_aligned():
    L, d, at = _lib.load(), _dims(requests=3, rows=11, logit_rows=5), (C.c_longlong * 10)()
    assert L.pie_step_plan_offsets(C.byref(d), at) == 0
    sizes = [4, 3, 11, 11, 11, 12, 4, 5, 5, 192]
    assert all(a % 4 == 0 for a in at) and all(at[i] + sizes[i] <= at[i + 1] for i in range(9)) and at[9] + 192 < L.pie_step_plan_words(C.byref(d))


def test_null_and_alignment():
    L, d, fake = _lib.load(), _dims(), C.c_void_p(0x1000)
    n0 = L.pie_launch_count()
    assert L.pie_step_plan_build(None, C.byref(d), fake, fake, fake, None, fake, 4, 0, None) == 5
    assert L.pie_step_plan_build(C.c_void_p(0x1004), C.byref(d), fake, fake, fake, None, fake, 4, 0, None) == 6
    assert L.pie_step_plan_build(fake, C.byref(d), fake, fake, fake, None, fake, -1, 0, None) == 1
    kv, rows = _lib.KvLayout(0, 64, 128, None, 0, 64), _lib.HeadRows(0x1000, 0, 64, 512)
    off = _lib.HeadRows(0x1002, 0, 64, 512)
    rope = lambda q, D=64, n=3: L.pie_rope_kv_slots(fake, fake, fake, C.byref(kv), C.byref(q), C.byref(rows), C.byref(rows), fake, fake, fake, n, 4, 8, 2, D, 1, None)
    assert rope(off) == 6 and rope(rows, D=96) == 1 and rope(rows, n=-1) == 1 and rope(rows, n=0) == 0
    attn = lambda q, D=64, scale=1.0, ws=1 << 40: L.pie_chunk_attn(fake, C.byref(q), fake, fake, C.byref(kv), fake, C.byref(d), D, scale, 1, fake, ws, None)
    assert attn(off) == 6 and attn(rows, D=96) == 1 and attn(rows, scale=0.0) == 1 and attn(rows, scale=float("nan")) == 1 and attn(rows, ws=8) == 7
    ver = lambda **kw: L.pie_verify_draft(*{**dict(t=fake, c=fake, lp=fake, x=fake, g=None, ld=50, dt=fake, st=fake, S=2, R=6, V=50, K=3, temp=0.5, u=fake, no=fake, ws=fake,
                                                  nb=1 << 40, stream=None), **kw}.values())
    assert ver(t=None) == 5 and ver(u=None) == 5 and ver(ld=49) == 1 and ver(K=128) == 1 and ver(K=-1) == 1 and ver(temp=-1.0) == 1 and ver(temp=float("nan")) == 1
    assert ver(temp=0.0, g=fake) == 1 and ver(nb=8) == 7 and ver(R=0) == 1 and ver(S=0) == 0 and ver(temp=float("inf")) == 1
    assert L.pie_launch_count() == n0


def _plan(**kw):
    a = dict(token_ids=ints(1, 2, 3), input_lengths=ints(1, 2), context_lengths=ints(0, 5), pages=ints(1, 2), num_pages=4, max_blocks=2, num_heads=4, num_kv_heads=2)
    a.update(kw)
    return StepPlan.build(a.pop("token_ids"), a.pop("input_lengths"), a.pop("context_lengths"), a.pop("pages"), **a)


@pytest.mark.parametrize("kw", [
    dict(), dict(token_ids=torch.tensor([1, 2, 3])), dict(token_ids=ints()), dict(token_ids=ints(1, 2).view(1, 2)), dict(input_lengths=ints(1)), dict(context_lengths=ints(1)),
    dict(pages=torch.tensor([1, 2])), dict(pages=ints(1, 2, 3).view(3, 1)), dict(draft_lengths=ints(0)), dict(num_heads=3), dict(max_blocks=0), dict(num_pages=0), dict(num_logits=0),
    dict(num_pages=(1 << 32) + 4), dict(max_blocks=(1 << 32) + 2), dict(num_logits=(1 << 32) + 2), dict(num_heads=4.0), dict(input_lengths=torch.tensor([[1, 2], [3, 4]], dtype=torch.int32).t()[0])])
def test_plan_refuses(kw):
    refuses(_plan, kw)


def _rope(**kw):
    a = dict(q=torch.zeros((3, 4, 64), dtype=BF), k=torch.zeros((3, 2, 64), dtype=BF), v=torch.zeros((3, 2, 64), dtype=BF), freqs=torch.ones(32), positions=ints(0, 1, 2),
             slots=ints(0, 1, 2), kp=torch.zeros((2, 64, 2, 64), dtype=BF), vp=torch.zeros((2, 64, 2, 64), dtype=BF), out=None)
    a.update(kw)
    return ops.rope_kv_slots(*a.values())


@pytest.mark.parametrize("kw", [
    dict(), dict(q=torch.zeros((3, 4, 64))), dict(q=torch.zeros((2, 4, 64), dtype=BF)), dict(k=torch.zeros((3, 2, 128), dtype=BF)), dict(v=torch.zeros((3, 1, 64), dtype=BF)),
    dict(freqs=torch.ones(64)), dict(freqs=torch.ones(32).double()), dict(positions=torch.arange(3)), dict(slots=ints(0, 1)), dict(kp=torch.zeros((2, 32, 2, 64), dtype=BF)),
    dict(vp=torch.zeros((2, 64, 2, 64))), dict(kp=torch.zeros((2, 64, 64, 2), dtype=BF).transpose(2, 3)), dict(vp=torch.zeros((3, 64, 2, 64), dtype=BF)),
    dict(q=torch.zeros((3, 4, 96), dtype=BF), k=torch.zeros((3, 2, 96), dtype=BF), v=torch.zeros((3, 2, 96), dtype=BF)), dict(kp=torch.zeros((2, 64, 2, 72), dtype=BF)[..., :64]),
    dict(out=torch.zeros((3, 4, 64)))])
def test_rope_refuses(kw):
    refuses(_rope, kw)


class _Plan:
    dims, words = _lib.StepDims(2, 3, 2, 2, 2, 4, 2), ints(0)


def _chunk(**kw):
    a = dict(q=torch.zeros((3, 4, 64), dtype=BF), kp=torch.zeros((2, 64, 2, 64), dtype=BF), vp=torch.zeros((2, 64, 2, 64), dtype=BF), plan=_Plan, scale=1.0, out=None)
    a.update(kw)
    return ops.chunk_attention(*a.values())


@pytest.mark.parametrize("kw", [
    dict(), dict(q=torch.zeros((3, 4, 64))), dict(q=torch.zeros((4, 4, 64), dtype=BF)), dict(q=torch.zeros((3, 8, 64), dtype=BF)), dict(q=torch.zeros((3, 4, 128), dtype=BF)),
    dict(kp=torch.zeros((3, 64, 2, 64), dtype=BF), vp=torch.zeros((3, 64, 2, 64), dtype=BF)), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
    dict(out=torch.zeros((3, 4, 64), dtype=BF))])
def test_attention_refuses(kw):
    refuses(_chunk, kw)


def _verify(**kw):
    a = dict(logits=torch.zeros((6, 50), dtype=BF), tokens=ints(0, 1, 2, 3, 4, 5), starts=ints(0, 2, 6), max_draft=3, temp=0.5, uniforms=torch.zeros(6), noise=torch.zeros((2, 50)),
             draft_logits=None)
    a.update(kw)
    return ops.verify_draft(a.pop("logits"), a.pop("tokens"), a.pop("starts"), **a)


@pytest.mark.parametrize("kw", [
    dict(), dict(logits=torch.zeros((6, 50))), dict(logits=torch.zeros((6, 0), dtype=BF)), dict(tokens=ints(0)), dict(tokens=torch.arange(6)), dict(starts=ints(0)), dict(starts=torch.arange(3)),
    dict(max_draft=128), dict(max_draft=-1), dict(max_draft=2.0), dict(temp=-0.1), dict(temp=float("inf")), dict(temp=float("nan")), dict(uniforms=None), dict(noise=torch.zeros((6, 50))),
    dict(noise=torch.zeros((2, 50)).double()), dict(uniforms=torch.zeros(12)[::2]), dict(draft_logits=torch.zeros((6, 51), dtype=BF)), dict(draft_logits=torch.zeros((6, 50))),
    dict(temp=0.0, draft_logits=torch.zeros((6, 50), dtype=BF))])
def test_verify_refuses(kw):
    refuses(_verify, kw)
