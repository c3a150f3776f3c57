"""A model whose linears are of 8-bit integers, beside what a plain call of its parts makes."""
import pytest
import torch

import step_oracle as O

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")


def small(head_dim=64, **kw):
    from parity_util import tiny_args
    from proxy_inference_engine_b200.checkpoint import build_model, random_weights
    args = tiny_args(bits=8, head_dim=head_dim, **kw)
    return args, build_model(args, random_weights(args, seed=5, device="cuda", gen_device="cpu"))


def step(args, model, ids, n_pages=4):
    """A planned step of one prompt, over fresh pools."""
    from proxy_inference_engine_b200.ragged import StepPlan, fp8_pools, ragged_step
    need = O.need(len(ids), 0)
    plan = StepPlan.build(ints(ids), ints([len(ids)]), ints([0]), ints(list(range(need))), num_pages=n_pages, max_blocks=need, num_heads=args.num_attention_heads,
                          num_kv_heads=args.num_key_value_heads)
    plan.check()
    return ragged_step(model, plan, fp8_pools(model, n_pages), all_logits=True)


def test_a_planned_step_calls_a_feed_forward_of_another_class():
    """One that gives nothing: the same bits as a feed-forward whose last matrix is zeros, not those of silu(gate) * up."""
    from proxy_inference_engine_b200.llama import MLP

    class Nothing(MLP):
        def __call__(self, x):
            return torch.zeros_like(x)

    args, model = small()
    model.to_int8()
    ids = [(37 * i + 5) % args.vocab_size for i in range(70)]
    usual = step(args, model, ids)
    for ly in model.layers:
        ly.mlp.__class__ = Nothing
    got = step(args, model, ids)
    for ly in model.layers:
        ly.mlp.__class__ = MLP
        ly.mlp.down_proj.scales.zero_()
    assert torch.equal(got, step(args, model, ids)) and not torch.equal(got, usual)


def test_a_layer_calls_a_norm_of_another_class():
    """One made from RMSNorm whose weights are offsets from one: what the norm gives, through the layer."""
    from proxy_inference_engine_b200 import nn, ops

    class Offset(nn.RMSNorm):
        def __call__(self, x):
            return ops.rms_norm(x, 1 + self.weight, self.eps)

    g = torch.Generator(device="cuda").manual_seed(1)
    x, w = (torch.randn(s, generator=g, device="cuda").to(BF) for s in ((3, 256), (40, 256)))
    lin, norm, offset = nn.Int8Linear.from_linear(w), nn.RMSNorm(256, eps=1e-6), Offset(256, eps=1e-6)
    norm.weight = (1 + 0.1 * torch.randn(256, generator=g, device="cuda")).to(BF)
    offset.weight = norm.weight - 1
    assert torch.equal(lin(x, norm=offset), lin(ops.rms_norm(x, 1 + offset.weight, 1e-6)))
    assert torch.equal(lin(x, norm=norm), ops.int8_linear(x, lin.weight, lin.scales, norm_weight=norm.weight, eps=1e-6))


@pytest.mark.parametrize("features", [2048, 4096, 4112, 8192, 14336, 16400, 40000])
def test_a_row_behind_a_norm_does_not_depend_on_the_rows_beside_it(features):
    """Fewer rows than a GPU has SMs, and more."""
    from proxy_inference_engine_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(features)
    x, w = torch.randn((600, features), generator=g, device="cuda").to(BF), (1 + 0.1 * torch.randn(features, generator=g, device="cuda")).to(BF)
    codes, scales = ops.int8_rows(x, norm_weight=w)
    for lo in range(0, 600, 100):
        part, of = ops.int8_rows(x[lo:lo + 100], norm_weight=w)
        assert torch.equal(part, codes[lo:lo + 100]) and torch.equal(of, scales[lo:lo + 100])


@pytest.mark.parametrize("use_graph", [True, False])
def test_a_decode_engine_keeps_the_weights_it_was_made_with(use_graph):
    """Layers of integers take the place of quantised ones whose addresses an engine's tables hold."""
    import gc
    import weakref
    from proxy_inference_engine_b200.checkpoint import build_model, random_weights
    from proxy_inference_engine_b200.decode import DecodeEngine
    from parity_util import tiny_args
    args = tiny_args(bits=4)
    model = build_model(args, random_weights(args, seed=3, device="cuda", gen_device="cpu"))
    prompt = torch.tensor([[(11 * i + 2) % args.vocab_size for i in range(20)]], dtype=torch.int32, device="cuda")
    engine = DecodeEngine(model, 1, 64, use_graph=use_graph)
    engine.prefill(prompt)
    engine.step(10)
    want = engine.generated()
    engine.prefill(prompt)
    arrays = lambda lin: (lin.weight, lin.scales, lin.biases)
    held = [weakref.ref(t) for ly in model.layers for part, names in ((ly.self_attn, "qkvo"), (ly.mlp, ("gate", "up", "down"))) for n in names for t in arrays(getattr(part, n + "_proj"))]
    model.to_int8()
    gc.collect()
    assert all(t() is not None for t in held)
    spoil = [torch.full((1 << 20,), -1, dtype=torch.int32, device="cuda") for _ in range(8)]   # (what was given back would be these)
    engine.step(10)
    assert torch.equal(engine.generated(), want) and spoil
    with pytest.raises(ValueError, match="8-bit integers"):
        DecodeEngine(model, 1, 64)
