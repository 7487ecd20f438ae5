"""The transformer blocks of the forward models on the library's attention: against the fixtures the stock path is held to, against the
stock path, and a training step with the learned position bias through all of its operators."""
import numpy as np
import pytest
import torch

import golden_util as G
from test_forward_models import build
from wavernn_amd import forward_models as FM

gpu = pytest.mark.gpu
FASTPITCH = [n for n in G.names("fwdmodel_") if "fastpitch" in n]


@gpu
@pytest.mark.parametrize("path", ["fused", "auto"])
@pytest.mark.parametrize("name", FASTPITCH)
def test_forward_and_generate_vs_reference_golden(name, path):
    rec, gold = G.load(name)
    model, batch = build(rec)
    model = model.cuda().set_attention_path(path)
    multi = rec["kind"] != "fast_pitch"
    with torch.no_grad():
        out = model({k: v.cuda() for k, v in batch.items()})
    for k in out:
        assert G.rel_err(out[k].cpu().numpy(), gold["fwd_" + k]) < 1e-4, k
    args = (batch["x"][:1].cuda(),) + ((batch["speaker_emb"][:1].cuda(),) if multi else ())
    gen = model.generate(*args, alpha=0.9, pitch_function=lambda p: p * 1.5)
    for k in gen:
        assert tuple(gen[k].shape) == gold["gen_" + k].shape, k
        if gen[k].dtype == torch.long:
            assert np.array_equal(gen[k].cpu().numpy(), gold["gen_" + k]), k
        else:
            assert G.rel_err(gen[k].cpu().numpy(), gold["gen_" + k]) < 1e-4, k


def test_paths_and_their_refusals():
    t = FM.ForwardTransformer(d_model=16, d_fft=32, layers=2, heads=2, conv1_kernel=3, conv2_kernel=1)
    assert all(b.attention_path == 'stock' for b in t.layers) and t.position_bias is None
    assert not any("position_bias" in k for k in t.state_dict())
    with pytest.raises(ValueError, match="attention path"):
        t.set_attention_path('fast')
    x = torch.randn(2, 5, 16)
    want = t.eval()(x)
    assert torch.equal(t.set_attention_path('auto')(x), want)        # on the CPU: stock
    with pytest.raises(RuntimeError, match="does not apply"):
        t.set_attention_path('fused')(x)
    assert torch.equal(t.set_attention_path('stock')(x), want)


@gpu
def test_dropout_in_training_stays_on_the_stock_path():
    t = FM.ForwardTransformer(d_model=32, d_fft=32, layers=1, heads=2, conv1_kernel=3, conv2_kernel=1, dropout=0.1).cuda().train()
    x = torch.randn(2, 9, 32, device="cuda")
    with pytest.raises(RuntimeError, match="dropout"):
        t.set_attention_path('fused')(x)
    torch.manual_seed(0)
    a = t.set_attention_path('auto')(x)
    torch.manual_seed(0)
    assert torch.equal(a, t.set_attention_path('stock')(x))


def transformer(rel_buckets, dtype=torch.float32, **kw):
    torch.manual_seed(1)
    t = FM.ForwardTransformer(**dict(dict(d_model=96, d_fft=64, layers=2, heads=3, conv1_kernel=3, conv2_kernel=1, dropout=0.0,
                                          rel_buckets=rel_buckets, rel_max_distance=40), **kw))
    if rel_buckets:
        torch.nn.init.normal_(t.position_bias.weight)
    return t.cuda().to(dtype).train()


@gpu
@pytest.mark.parametrize("rel_buckets", [0, 16])
@pytest.mark.parametrize("masked", [False, True])
def test_training_step_vs_stock_path(rel_buckets, masked):
    """A training step on either path: outputs and every parameter's gradient.  Two float32 computations of the same network: they differ by
    roundings of 2^-24 through two blocks of some hundred-term sums, well under 1e-4 of each tensor's largest value."""
    t = transformer(rel_buckets)
    x = torch.randn(4, 57, 96, device="cuda", requires_grad=True)
    mask = torch.arange(57, device="cuda")[None] >= torch.tensor([[57], [40], [13], [1]], device="cuda") if masked else None
    g = torch.randn(4, 57, 96, device="cuda")
    got = {}
    for path in ("stock", "fused"):
        t.set_attention_path(path)
        y = t(x, src_pad_mask=mask)
        names = [n for n, _ in t.named_parameters()]
        # (the scale of the position table takes part too; every parameter has to get a gradient)
        got[path] = dict(zip(["y", "x"] + names, [y.detach(), *torch.autograd.grad(y, [x, *t.parameters()], g)]))
    assert ("position_bias.weight" in got["stock"]) == bool(rel_buckets)
    for n, a in got["stock"].items():
        # (the key part of in_proj_bias shifts all of a row's scores alike: its gradient is rounding, on the scale of the value part's)
        assert float((a - got["fused"][n]).abs().max()) < 1e-4 * float(a.abs().max()), n


@gpu
def test_training_in_bfloat16():
    """bfloat16 on the fused path with the bias table's gradient, on a side stream and on the current one: the same bits."""
    t = transformer(16, torch.bfloat16).set_attention_path('fused')
    params = list(t.parameters())
    x = torch.randn(4, 130, 96, device="cuda").bfloat16()
    g = torch.randn(4, 130, 96, device="cuda").bfloat16()

    def step():
        y = t(x)
        return [y.detach(), *torch.autograd.grad(y, params, g)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    eager = step()
    assert torch.equal(eager[0], other[0])
    assert all(bool(torch.isfinite(v).all()) for v in eager)
    f32 = transformer(16).set_attention_path('stock')
    f32.load_state_dict({k: v.float() for k, v in t.state_dict().items()})
    with torch.no_grad():
        y = f32(x.float())
    # bfloat16 all through: 2^-8 a rounding, some tens of them in a row in two blocks
    assert float((y - eager[0].float()).abs().max()) < 0.15 * float(y.abs().max())


@gpu
def test_masked_out_row_attends_to_nothing():
    t = transformer(0).eval().set_attention_path('fused')
    x = torch.randn(3, 20, 96, device="cuda")
    mask = torch.zeros(3, 20, dtype=torch.bool, device="cuda")
    mask[1] = True
    with torch.no_grad():
        y = t(x, src_pad_mask=mask)
        z = t(x[[0, 2]], src_pad_mask=mask[[0, 2]])
    assert bool(torch.isfinite(y).all())
    assert float((y[[0, 2]] - z).abs().max()) < 1e-5 * float(z.abs().max())


@gpu
def test_models_take_the_position_bias():
    rec, _ = G.load(FASTPITCH[0])
    model = FM.FastPitch(**dict(rec["cfg"], rel_buckets=16, rel_max_distance=40))
    keys = [k for k in model.state_dict() if k.endswith("position_bias.weight")]
    assert len(keys) == 5 and all(tuple(model.state_dict()[k].shape) == (16, 2) for k in keys)     # predictors, prenet, postnet
    model = model.cuda().eval()
    x = torch.randint(1, 20, (1, 15), device="cuda")
    gen = {p: model.set_attention_path(p).generate(x) for p in ("stock", "fused")}
    for k in gen["stock"]:
        assert gen["stock"][k].shape == gen["fused"][k].shape
        assert G.rel_err(gen["fused"][k].cpu().numpy(), gen["stock"][k].cpu().numpy()) < 1e-4, k


@gpu
def test_auto_path_leaves_what_does_not_fit_to_the_stock_path():
    """Types that the operators do not take, in the weights or by autocast, and masks that are added rather than leaving keys out."""
    torch.manual_seed(0)
    block = FM.FFTBlock(32, 2, 3, 1, 64, dropout=0.).cuda()
    x, mask = torch.randn(20, 3, 32, device="cuda"), torch.zeros(3, 20, device="cuda")
    mask[1, 11:] = -np.inf

    def both(*args):
        out = []
        for path in ("stock", "auto"):
            FM.set_attention_path(block, path)
            out.append(block(*args))
        return out

    with torch.autocast("cuda", torch.float16):
        a, b = both(x)
        assert torch.equal(a, b)
        with pytest.raises(RuntimeError, match="float32 or bfloat16"):
            FM.set_attention_path(block, "fused")(x)
    a, b = both(x, mask)
    assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="bool"):
        FM.set_attention_path(block, "fused")(x, mask)
    block.half()
    a, b = both(x.half())
    assert torch.equal(a, b)
    block.double()
    a, b = both(x.double())
    assert torch.equal(a, b)
