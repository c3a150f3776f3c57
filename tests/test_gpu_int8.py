"""Products in 8-bit integers with a scale for each token and channel against plain arithmetic in 64 bits.

Tolerances.  Codes and scales are defined in 32 bits: equal.  A product: the sum is exact; its conversion to fp32 and two multiplications are off by 2^-24 each, the
rounding to bfloat16 by 2^-8 of the value (half a step); a residual adds another rounding of the sum."""
import pytest
import torch

from proxy_inference_engine_b200 import ops

pytestmark = pytest.mark.gpu
BF, F32, F64, I8 = torch.bfloat16, torch.float32, torch.float64, torch.int8
HALF = 2.0 ** -8


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, std=1.0):
    return (std * torch.randn(shape, generator=g, device="cuda")).to(BF)


def integers(g, *shape, lo=-127):
    return torch.randint(lo, 128, shape, generator=g, device="cuda").to(I8)


def plain_rows(x):
    """The definition, in 32 bits, on the CPU (whose division is exact to the last place)."""
    x = x.float().cpu()
    scales = x.abs().amax(-1) * torch.tensor(1 / 127, dtype=F32)
    ok = torch.isfinite(x).all(-1)
    codes = torch.where((scales > 0)[..., None] & ok[..., None], (x / scales[..., None]).round().clamp(-127, 127), 0.0)
    return torch.nan_to_num(codes).to(I8), torch.where(ok, scales, float("nan"))


def check_rows(x, **kw):
    codes, scales = ops.int8_rows(x, **kw)
    want, of = plain_rows(x)
    assert codes.shape == x.shape and scales.shape == x.shape[:-1]
    assert torch.equal(codes.cpu(), want)
    assert torch.equal(scales.cpu().nan_to_num(-1.0), of.nan_to_num(-1.0))


def check_product(y, codes, scales, weight, ws, residual=None):
    exact = (codes.double() @ weight.double().T) * scales.double()[:, None] * ws.double()
    bound = HALF * exact.abs() * (1 + 2.0 ** -20) + 2.0 ** -130
    if residual is not None:
        exact = exact + residual.double()
        bound = bound + HALF * (exact.abs() + bound)
    off = (y.double() - exact).abs()
    assert y.dtype == BF and bool((off <= bound).all()), float((off - bound).max())


@pytest.mark.parametrize("rows,features", [(1, 16), (3, 48), (8, 4096), (5, 2064), (2, 8208), (2, 16384), (3, 16400), (2, 131072), (700, 320)])
def test_rows(rows, features):
    check_rows(normal(gen(rows), rows, features, std=3.0))


def test_rows_at_the_borders_between_codes():
    """Maxima of 254 2^n: steps are powers of two, and halves of steps are numbers of the type.  And maxima of all other mantissas."""
    x = torch.zeros((128, 512), dtype=BF)
    for r in range(128):
        x[r] = (torch.arange(512) - 256).to(BF) * (0.5 if r == 126 else 0.37) * 2.0 ** (r % 30 - 15)
        x[r, 0] = (128 + r) * 2.0 ** (r % 30 - 8)
    check_rows(x.cuda())


def test_rows_without_a_scale():
    g = gen(1)
    x = normal(g, 12, 256)
    x[1] = 0
    x[2, 17] = float("inf")
    x[3, 200] = float("-inf")
    x[4, 0] = float("nan")
    x[5] = 2.0 ** -133          # the type's lowest number
    x[6] = 0
    x[6, 255] = -3 * 2.0 ** -133
    x[7] = normal(g, 256) * 2.0 ** -120
    x[8] = 3.38e38
    x[9] *= 1e-36
    x[10, 3] = torch.finfo(BF).min
    check_rows(x)
    codes, scales = ops.int8_rows(x)
    y = ops.int8_matmul(codes, scales, integers(g, 40, 256), torch.ones(40, device="cuda"))
    assert bool(y[2:5].isnan().all()) and bool((y[1] == 0).all()) and not bool(y[5:].isnan().any())


def test_rows_that_lie_anywhere():
    g = gen(2)
    side = normal(g, 9, 3 * 256 + 8)
    for x in (side[:, 256:512], side[:, 8:264], side[:, 3:259], side[::2, :256], normal(g, 256, 5).t(), side[:1, 256:512], normal(g, 2, 3, 4, 64), normal(g, 64)):
        check_rows(x)
    assert ops.int8_rows(side[:0, :256])[0].shape == (0, 256)


@pytest.mark.parametrize("rows,features", [(1, 256), (7, 4096), (3, 14336), (2, 20000)])
def test_rows_behind_a_norm(rows, features):
    """The rows of rms_norm, whose sum of squares may be added up in another order: a value in a few hundred may be rounded to the other side."""
    g = gen(3)
    x, w = normal(g, rows, features, std=2.0), 1 + normal(g, features, std=0.1)
    codes, scales = ops.int8_rows(x, norm_weight=w, eps=1e-5)
    want, of = plain_rows(ops.rms_norm(x, w, 1e-5))
    assert float((scales.cpu() / of - 1).abs().max()) <= 2 * HALF
    differ = (codes.cpu().int() - want.int()).abs()
    assert int(differ.max()) <= 1 and float((differ > 0).double().mean()) <= 0.02
    x = x.double()
    h = x / torch.sqrt(x.square().mean(1, keepdim=True) + 1e-5) * w.double()
    off = (codes.double() * scales.double()[:, None] - h).abs()
    # a norm's two roundings, half a step of the codes
    assert bool((off <= 2 * HALF * h.abs() * 1.01 + scales.double()[:, None] * 0.51).all())


SIZES = [(1, 1, 16), (1, 128, 128), (1, 129, 144), (2, 1000, 4096), (5, 7, 112), (16, 300, 272), (17, 300, 272), (32, 640, 1040), (33, 4096, 512), (64, 257, 2048), (64, 5000, 640),
         (65, 257, 2048), (77, 1, 16), (77, 1000, 4096), (128, 7, 112), (129, 384, 4096), (300, 1000, 272), (513, 5003, 144), (1000, 640, 4112), (2050, 2056, 1024)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("with_residual", [False, True])
def test_product(M, N, K, with_residual):
    g = gen(M + N)
    codes, weight = integers(g, M, K), integers(g, N, K, lo=-128)
    scales, ws = torch.rand(M, generator=g, device="cuda") + 0.1, torch.rand(N, generator=g, device="cuda") * 1e-3
    residual = normal(g, M, N, std=100.0) if with_residual else None
    for _ in range(2):   # (the second call finds the workspace as the first one left it)
        check_product(ops.int8_matmul(codes, scales, weight, ws, residual=residual), codes, scales, weight, ws, residual)


@pytest.mark.parametrize("M", [1, 50, 200])
def test_largest_sums(M):
    """All products of one sign and the largest size: the sum is below 2^31."""
    K = 131056
    codes, weight = torch.full((M, K), -128, dtype=I8, device="cuda"), torch.full((130, K), -128, dtype=I8, device="cuda")
    weight[1] = 127
    one = torch.ones(130, device="cuda")
    check_product(ops.int8_matmul(codes, one[:1].expand(M), weight, one), codes, one[:1].expand(M), weight, one)


def test_a_row_does_not_depend_on_the_rows_beside_it():
    g = gen(5)
    codes, weight = integers(g, 700, 1536), integers(g, 1001, 1536)
    scales, ws = torch.rand(700, generator=g, device="cuda"), torch.rand(1001, generator=g, device="cuda")
    whole = ops.int8_matmul(codes, scales, weight, ws)
    for lo, hi in ((0, 1), (3, 19), (100, 130), (640, 700), (0, 65), (200, 500)):
        assert torch.equal(ops.int8_matmul(codes[lo:hi], scales[lo:hi], weight, ws), whole[lo:hi])


@pytest.mark.parametrize("rows", [1, 40, 333])
def test_linear(rows):
    """The layer, with all that goes with it, in its shapes: [batch, rows, features], a norm, a residual."""
    g = gen(6)
    x, w, norm = normal(g, 2, rows, 1024, std=2.0), normal(g, 1300, 1024, std=0.03), 1 + normal(g, 1024, std=0.1)
    weight, ws = ops.int8_rows(w)
    y = ops.int8_linear(x, weight, ws, norm_weight=norm, eps=1e-6)
    codes, scales = ops.int8_rows(x, norm_weight=norm, eps=1e-6)
    assert y.shape == (2, rows, 1300)
    check_product(y.flatten(0, 1), codes.flatten(0, 1), scales.flatten(), weight, ws)
    z = ops.int8_linear(x, weight, ws, residual=y)
    codes, scales = ops.int8_rows(x)
    check_product(z.flatten(0, 1), codes.flatten(0, 1), scales.flatten(), weight, ws, y.flatten(0, 1))
    # what the integers stand for: rounding of a row by at most half a step of its codes, of a channel too
    full = x.double().flatten(0, 1) @ w.double().T
    err = 0.5 * scales.flatten().double()[:, None] * w.double().abs().sum(1) + x.double().flatten(0, 1).abs().sum(1)[:, None] * 0.5 * ws.double()
    assert bool(((z.double() - y.double()).flatten(0, 1) - full).abs().le(1.05 * err + 4 * HALF * (full.abs() + y.double().flatten(0, 1).abs())).all())


def test_graphs_and_streams():
    """Captured and replayed on other inputs, beside eager calls and another graph of the same sizes, on another stream."""
    g = gen(7)
    weight, ws = ops.int8_rows(normal(g, 3000, 2048))
    xs = [normal(g, 5, 2048) for _ in range(4)]
    want = [ops.int8_linear(x, weight, ws) for x in xs]
    graphs = []
    for _ in range(2):
        x, graph = xs[0].clone(), torch.cuda.CUDAGraph()
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            with torch.cuda.graph(graph, stream=stream):
                y = ops.int8_linear(x, weight, ws)
                y = ops.int8_linear(x, weight, ws, residual=y * 0)
        graphs.append((graph, x, y))
    for i in range(12):
        graph, x, y = graphs[i % 2]
        x.copy_(xs[i % 4])
        graph.replay()
        other = ops.int8_linear(xs[(i + 1) % 4], weight, ws)
        assert torch.equal(y, want[i % 4]) and torch.equal(other, want[(i + 1) % 4])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = []
    for i in range(20):
        with torch.cuda.stream(side):
            got.append(ops.int8_linear(xs[i % 4], weight, ws))
        got.append(ops.int8_linear(xs[(i + 1) % 4], weight, ws))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[(i // 2 + i % 2) % 4]) for i, y in enumerate(got))
    ops.check_pipeline()
