"""What products in 8-bit integers refuse before anything is launched."""
import ctypes as C

import pytest
import torch

from proxy_inference_engine_b200 import _lib, ops

BF, F32, I8 = torch.bfloat16, torch.float32, torch.int8


def refuses(call, changed, **kw):
    """Without anything else wrong: tensors that are not on a CUDA device."""
    with pytest.raises(ValueError) as e:
        call(**kw)
    assert ("CUDA device" in str(e.value)) == (not changed), str(e.value)


@pytest.mark.parametrize("kw", [dict(), dict(x=torch.zeros((3, 32), dtype=F32)), dict(x=torch.zeros((3, 40), dtype=BF)), dict(x=torch.zeros((3, 0), dtype=BF)),
                                dict(x=torch.tensor(1.0, dtype=BF)), dict(norm_weight=torch.ones(32)), dict(norm_weight=torch.ones(48, dtype=BF)),
                                dict(norm_weight=torch.ones((1, 32), dtype=BF))])
def test_rows(kw):
    refuses(ops.int8_rows, kw, **{**dict(x=torch.zeros((3, 32), dtype=BF)), **kw})


@pytest.mark.parametrize("kw", [dict(), dict(codes=torch.zeros((3, 32), dtype=torch.uint8)), dict(codes=torch.zeros((3, 40), dtype=I8)), dict(codes=torch.zeros((3, 0), dtype=I8)),
                                dict(scales=torch.zeros((3, 1))), dict(scales=torch.zeros(4)), dict(scales=torch.zeros(3, dtype=torch.float64)),
                                dict(weight=torch.zeros((5, 48), dtype=I8)), dict(weight=torch.zeros((5, 32), dtype=torch.uint8)), dict(weight=torch.zeros((32, 5), dtype=I8).t()),
                                dict(weight=torch.zeros(32, dtype=I8)), dict(weight_scales=torch.zeros(4)), dict(weight_scales=torch.zeros(10)[::2]),
                                dict(weight_scales=torch.zeros(5, dtype=BF)), dict(residual=torch.zeros((3, 6), dtype=BF)), dict(residual=torch.zeros((3, 5)))])
def test_product(kw):
    given = dict(codes=torch.zeros((3, 32), dtype=I8), scales=torch.zeros(3), weight=torch.zeros((5, 32), dtype=I8), weight_scales=torch.zeros(5))
    refuses(ops.int8_matmul, kw, **{**given, **kw})


def test_sums_that_do_not_fit():
    K = 131072
    with pytest.raises(ValueError, match="131072"):
        ops.int8_matmul(torch.zeros((1, K), dtype=I8), torch.zeros(1), torch.zeros((1, K), dtype=I8), torch.zeros(1))


@pytest.mark.parametrize("kw", [dict(), dict(x=torch.zeros((3, 32))), dict(norm_weight=torch.ones(31, dtype=BF)), dict(weight=torch.zeros((5, 16), dtype=I8)),
                                dict(weight_scales=torch.zeros(6)), dict(residual=torch.zeros((2, 5), dtype=BF))])
def test_linear(kw):
    given = dict(x=torch.zeros((3, 32), dtype=BF), weight=torch.zeros((5, 32), dtype=I8), weight_scales=torch.zeros(5))
    refuses(ops.int8_linear, kw, **{**given, **kw})


def test_c_calls():
    L, fake, odd = _lib.load(), C.c_void_p(0x1000), C.c_void_p(0x1008)
    n0 = L.pie_launch_count()
    rows = lambda codes=fake, x=fake, ld=32, n=3, K=32, norm=None: L.pie_int8_rows(codes, fake, x, ld, n, K, norm, 1e-5, None)
    assert rows(codes=None) == 5 and rows(x=None) == 5 and rows(x=odd) == 6 and rows(codes=odd) == 6 and rows(norm=odd) == 6
    assert rows(ld=33) == 1 and rows(ld=-32) == 1 and rows(n=-1) == 1 and rows(K=24) == 1 and rows(K=0) == 1 and rows(n=0) == 0
    mul = lambda y=fake, w=fake, M=3, N=5, K=32, ws=fake, nb=1 << 20: L.pie_int8_matmul(y, fake, fake, w, fake, None, M, N, K, ws, nb, None)
    assert mul(y=None) == 5 and mul(w=odd) == 6 and mul(ws=odd) == 6 and mul(M=-1) == 1 and mul(N=0) == 1 and mul(K=40) == 1 and mul(K=131072) == 1
    assert mul(ws=None) == 7 and mul(nb=100) == 7 and mul(M=0) == 0 and mul(M=1 << 24, N=1 << 24) == 1
    assert L.pie_int8_workspace_bytes(16, 1000) > 16 * 1000 * 4 and L.pie_int8_workspace_bytes(200, 1000) == 0 and L.pie_int8_workspace_bytes(0, 1000) == 0
    assert L.pie_launch_count() == n0
