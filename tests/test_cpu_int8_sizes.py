"""Products in 8-bit integers of more rows or channels than the kernels count are refused; nothing is launched."""
import ctypes as C

import pytest
import torch

from proxy_inference_engine_b200 import _lib, ops

BF, I8, MOST = torch.bfloat16, torch.int8, 2 ** 31 - 257


def rows(n, dtype, *shape):
    """n rows that lie on one."""
    return torch.zeros((1, *shape), dtype=dtype).expand(n, *shape)


def test_c_calls():
    L, fake = _lib.load(), C.c_void_p(0x1000)
    n0 = L.pie_launch_count()
    mul = lambda M, N: L.pie_int8_matmul(fake, fake, fake, fake, fake, None, M, N, 16, None, 0, None)
    assert mul(MOST + 1, 1) == 1 and mul(2 ** 31 - 1, 1) == 1 and mul(17, MOST + 1) == 1 and mul(1, 2 ** 31 - 1) == 1
    assert mul(1, MOST) == 7   # (a workspace is asked for)
    assert L.pie_launch_count() == n0


@pytest.mark.parametrize("n", [MOST + 1, 2 ** 31, 2 ** 32 + 5])
def test_rows(n):
    one = torch.zeros((1, 16), dtype=I8)
    with pytest.raises(ValueError, match=f"{n} rows are not built"):
        ops.int8_matmul(rows(n, I8, 16), rows(n, torch.float32), one, torch.zeros(1))
    for call in (ops.int8_rows, lambda x: ops.int8_linear(x, one, torch.zeros(1))):
        with pytest.raises(ValueError, match=f"{n} rows of 16 features are not built"):
            call(rows(n, BF, 16))
    with pytest.raises(ValueError, match="CUDA device"):
        ops.int8_matmul(rows(MOST, I8, 16), rows(MOST, torch.float32), one, torch.zeros(1))
