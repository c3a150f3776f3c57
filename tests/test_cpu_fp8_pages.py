"""What the operators over 8-bit pages refuse before anything is launched."""
import ctypes as C

import pytest
import torch

from proxy_inference_engine_b200 import _lib, ops

BF, F8 = torch.bfloat16, torch.float8_e4m3fn
DIMS = dict(requests=2, rows=3, logit_rows=2, blocks=4, pages=5, Hq=8, Hkv=2)


class Plan:
    def __init__(self, **kw):
        self.dims = _lib.StepDims(*{**DIMS, **kw}.values())
        self.words = torch.zeros(_lib.load().pie_step_plan_words(C.byref(self.dims)), dtype=torch.int32)


def given(D=64, **kw):
    pool = lambda: torch.zeros((5, 2, 64, D), dtype=F8)
    got = dict(queries=torch.zeros((3, 8, D), dtype=BF), keys=torch.zeros((3, 2, D), dtype=BF), values=torch.zeros((3, 2, D), dtype=BF), freqs=torch.ones(D // 2), plan=Plan(),
               k_pool=pool(), k_scales=torch.ones((5, 2)), v_pool=pool(), v_scales=torch.ones((5, 2)))
    return {**got, **kw}


def refuses(call, changed, kw):
    """Without anything else wrong: tensors that are not on a CUDA device."""
    with pytest.raises(ValueError) as e:
        call(**kw)
    assert ("CUDA device" in str(e.value)) == (not changed), str(e.value)


POOLS = [dict(k_pool=torch.zeros((5, 2, 64, 64), dtype=torch.uint8)), dict(v_pool=torch.zeros((4, 2, 64, 64), dtype=F8)), dict(k_pool=torch.zeros((5, 64, 2, 64), dtype=F8)),
         dict(v_pool=torch.zeros((5, 2, 64, 128), dtype=F8)[..., :64]), dict(k_scales=torch.ones((5, 1))), dict(v_scales=torch.ones((2, 5)).t()), dict(k_scales=torch.ones((5, 2), dtype=BF)),
         dict(plan=Plan(rows=4)), dict(plan=Plan(Hq=4)), dict(plan=Plan(pages=6)), dict(plan=Plan(Hkv=4)), dict(out=torch.zeros((3, 8, 64)))]


@pytest.mark.parametrize("kw", [dict(), dict(queries=torch.zeros((3, 8, 64))), dict(keys=torch.zeros((3, 4, 64), dtype=BF)), dict(values=torch.zeros((2, 2, 64), dtype=BF)),
                                dict(freqs=torch.ones(64)), dict(freqs=torch.ones(32, dtype=BF)), *POOLS])
def test_rows_into_pages(kw):
    refuses(ops.rope_kv_fp8, kw, given(**kw))


def test_head_sizes():
    with pytest.raises(ValueError, match="head size"):
        ops.rope_kv_fp8(**given(96))


@pytest.mark.parametrize("kw", [dict(), dict(q=torch.zeros((3, 8, 64))), dict(q=torch.zeros((3, 8, 96), dtype=BF)), dict(q=torch.zeros((3, 512), dtype=BF)), dict(scale=0.0), dict(scale=float("nan")),
                                *POOLS])
def test_attention(kw):
    base = given()
    refuses(ops.chunk_attention_fp8, kw, {**dict(q=base["queries"], scale=0.1, **{n: base[n] for n in ("k_pool", "k_scales", "v_pool", "v_scales", "plan")}), **kw})


def test_c_calls():
    L, fake, odd, d = _lib.load(), C.c_void_p(0x1000), C.c_void_p(0x1008), _lib.StepDims(*DIMS.values())
    n0 = L.pie_launch_count()
    rows, off, half = _lib.HeadRows(0x1000, 0, 64, 512), _lib.HeadRows(0x1002, 0, 64, 512), _lib.HeadRows(0x1000, 0, 64, 500)
    rope = lambda q=rows, dims=d, D=64, pool=fake, scales=fake, out=fake: L.pie_rope_kv_fp8(out, pool, scales, fake, fake, C.byref(q), C.byref(rows), C.byref(rows), fake, C.byref(dims), fake, D, 1, None)
    assert rope(q=off) == 6 and rope(q=half) == 1 and rope(D=96) == 1 and rope(pool=None) == 5 and rope(scales=None) == 5 and rope(pool=odd) == 6 and rope(out=odd) == 6
    assert rope(dims=_lib.StepDims(0, 3, 2, 4, 5, 8, 2)) == 1
    need = L.pie_chunk_attn_fp8_workspace_bytes(C.byref(d), 64)
    attend = lambda D=64, scale=0.1, ws=fake, nb=need, pool=fake, scales=fake, dims=d: L.pie_chunk_attn_fp8(fake, C.byref(rows), pool, scales, fake, fake, fake, C.byref(dims), D, scale, 1, ws, nb, None)
    assert attend(D=80) == 1 and attend(scale=0.0) == 1 and attend(ws=None) == 7 and attend(nb=need - 1) == 7 and attend(pool=None) == 5 and attend(scales=None) == 5 and attend(pool=odd) == 6
    assert L.pie_launch_count() == n0


def test_room_for_pages_in_16_bits():
    """Where every request is of few rows, there is none; otherwise twice the pools."""
    L = _lib.load()
    of = lambda **kw: L.pie_chunk_attn_fp8_workspace_bytes(C.byref(_lib.StepDims(*{**DIMS, **kw}.values())), 128)
    few = of(rows=8)
    assert few == L.pie_chunk_attn_workspace_bytes(C.byref(_lib.StepDims(*DIMS.values())), 128) and of(rows=9) == few + 2 * 2 * 5 * 2 * 64 * 128
    assert of(requests=0) == 0 and L.pie_chunk_attn_fp8_workspace_bytes(C.byref(_lib.StepDims(*DIMS.values())), 96) == 0
