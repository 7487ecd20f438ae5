"""FFTBlock's attention paths beside what the block could do before: masks, subclasses, pickles, hooks, modes of the module itself."""
import copy
import pickle
import types

import pytest
import torch
from torch.autograd import forward_ad

import golden_util as G
from wavernn_amd import forward_models as FM


def block(**kw):
    torch.manual_seed(0)
    return FM.FFTBlock(**dict(dict(d_model=32, nhead=2, conv1_kernel=3, conv2_kernel=1, d_fft=48, dropout=0.0), **kw))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_additive_masks_beside_a_position_bias(dtype):
    """On the stock path a mask that is added does what the bool mask does, also where the scores get a bias."""
    b = block()
    x = torch.randn(9, 3, 32)
    leave = torch.arange(9)[None] >= torch.tensor([[9], [5], [1]])
    added = torch.zeros(3, 9, dtype=dtype).masked_fill(leave, -torch.inf)
    bias = torch.randn(2, 9, 9)
    for kw in ({}, dict(position_bias=lambda q_len, k_len: bias)):
        assert torch.equal(b(x, added.float() if not kw else added, **kw), b(x, leave, **kw))


class FormerBlock(FM.FFTBlock):

    def forward(self, src, src_pad_mask=None):
        return super().forward(src, src_pad_mask=src_pad_mask)


def transformer(**kw):
    torch.manual_seed(0)
    return FM.ForwardTransformer(**dict(dict(d_model=32, d_fft=48, layers=2, heads=2, conv1_kernel=3, conv2_kernel=1, dropout=0.0), **kw)).eval()


def test_layers_without_a_position_bias_are_called_as_before():
    """A layer, or a subclass of the block, that takes a source and its mask alone."""
    t, x = transformer(), torch.randn(2, 7, 32)
    want = t(x)
    for layer in t.layers:
        layer.__class__ = FormerBlock
    assert torch.equal(t(x), want)


def test_modules_pickled_before_the_paths_and_the_bias():
    t, x = transformer(), torch.randn(2, 7, 32)
    want = t(x)
    del t.__dict__["position_bias"]
    for layer in t.layers:
        layer.__dict__.pop("attention_path", None)
    old = pickle.loads(pickle.dumps(t))
    assert torch.equal(old(x), want)
    assert all(b.attention_path == 'stock' for b in old.layers) and old.position_bias is None
    new = transformer(rel_buckets=8).set_attention_path('auto')
    for t in (pickle.loads(pickle.dumps(new)), copy.deepcopy(new)):
        assert all(b.attention_path == 'auto' for b in t.layers) and torch.equal(t.position_bias.weight, new.position_bias.weight)


def on_the_gpu(dtype=torch.float32):
    """Stands for a source tensor in the question whether the fused path applies."""
    return types.SimpleNamespace(device=torch.device("cuda"), dtype=dtype)


def test_dropout_of_the_attention_itself_decides():
    """The probabilities' dropout is nn.MultiheadAttention's, which may be in another mode than the block around it."""
    b = block(dropout=0.1).train()
    assert "dropout" in b._why_not_fused(on_the_gpu(), None)
    b.self_attn.eval()
    assert b._why_not_fused(on_the_gpu(), None) is None
    b.eval()
    b.self_attn.train()
    assert "dropout" in b._why_not_fused(on_the_gpu(), None)


@pytest.mark.parametrize("register", ["register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook", "register_full_backward_pre_hook"])
def test_hooks_on_the_attention_keep_the_stock_path(register):
    """'fused' does not call nn.MultiheadAttention: it says so where somebody listens to that call, and 'auto' makes it."""
    b = block().eval()
    handle = getattr(b.self_attn, register)(lambda *a: None)
    assert "hooks" in b._why_not_fused(on_the_gpu(), None)
    handle.remove()
    assert b._why_not_fused(on_the_gpu(), None) is None


@pytest.mark.gpu
def test_other_kinds_of_differentiation_keep_the_stock_path():
    """Forward-mode derivatives and the transforms of torch.func, which the operators refuse."""
    b = block().eval().cuda()
    x, tangent = torch.randn(5, 2, 32, device="cuda"), torch.randn(5, 2, 32, device="cuda")
    w = b.self_attn.in_proj_weight.detach()
    got = {}
    for path in ("stock", "auto"):
        FM.set_attention_path(b, path)
        with forward_ad.dual_level():
            by_source = forward_ad.unpack_dual(b(forward_ad.make_dual(x, tangent))).tangent
            dual = {"self_attn.in_proj_weight": forward_ad.make_dual(w, torch.ones_like(w))}
            by_weight = forward_ad.unpack_dual(torch.func.functional_call(b, dual, (x,))).tangent
        got[path] = [by_source, by_weight, *torch.func.jvp(b, (x,), (tangent,)), torch.func.grad(lambda y: b(y).square().sum())(x)]
    for a, c in zip(*got.values()):
        assert torch.equal(a, c) and bool(a.any())
    FM.set_attention_path(b, "fused")
    with forward_ad.dual_level():
        assert torch.isfinite(b(x)).all()
        with pytest.raises(RuntimeError, match="forward-mode"):
            b(forward_ad.make_dual(x, tangent))
    with pytest.raises(RuntimeError, match="torch.func"):
        torch.func.grad(lambda y: b(y).sum())(x)


@pytest.mark.parametrize("name", [n for n in G.names("fwdmodel_") if "fastpitch" in n])
def test_every_transformer_of_the_models_takes_the_position_bias(name):
    rec, _ = G.load(name)
    multi = rec["kind"] != "fast_pitch"
    model = (FM.MultiFastPitch if multi else FM.FastPitch)(**dict(rec["cfg"], rel_buckets=16, rel_max_distance=40))
    transformers = [m for m in model.modules() if isinstance(m, FM.ForwardTransformer)]
    assert len(transformers) == (6 if multi else 5)
    for t in transformers:
        heads = t.layers[0].self_attn.num_heads
        assert tuple(t.position_bias.weight.shape) == (16, heads) and t.position_bias.max_distance == 40
    plain = (FM.MultiFastPitch if multi else FM.FastPitch)(**rec["cfg"])
    assert not any("position_bias" in k for k in plain.state_dict())


@pytest.mark.gpu
def test_multi_speaker_model_with_the_position_bias_on_either_path():
    rec, _ = G.load([n for n in G.names("fwdmodel_") if "multifastpitch" in n][0])
    torch.manual_seed(0)
    model = FM.MultiFastPitch(**dict(rec["cfg"], rel_buckets=16, rel_max_distance=40))
    for t in (m for m in model.modules() if isinstance(m, FM.ForwardTransformer)):
        torch.nn.init.normal_(t.position_bias.weight)
    model = model.cuda().eval()
    args = torch.randint(1, 20, (1, 15), device="cuda"), torch.randn(1, rec["cfg"]["speaker_emb_dims"], device="cuda")
    gen = {p: model.set_attention_path(p).generate(*args) for p in ("stock", "fused")}
    for k in gen["stock"]:
        assert gen["stock"][k].shape == gen["fused"][k].shape
        assert G.rel_err(gen["fused"][k].cpu().numpy(), gen["stock"][k].cpu().numpy()) < 1e-4, k


def test_autocast_leaves_float64_alone():
    """It casts no float64, so the projections' results are not of autocast's type."""
    b = block()
    torch.set_autocast_enabled("cuda", True)
    torch.set_autocast_dtype("cuda", torch.bfloat16)
    try:
        assert b._why_not_fused(on_the_gpu(), None) is None
        assert "float64" in b._why_not_fused(on_the_gpu(torch.float64), None)
    finally:
        torch.set_autocast_enabled("cuda", False)


def test_a_position_bias_of_ones_own_survives_copies():
    """One that is no module: copies and pickles keep it."""
    t, x = transformer(), torch.randn(2, 7, 32)
    t.position_bias = Slope()
    want = t(x)
    for c in (copy.deepcopy(t), pickle.loads(pickle.dumps(t))):
        assert torch.equal(c(x), want)
    assert not torch.equal(transformer()(x), want)


class Slope:

    def __call__(self, q_len, k_len):
        return -0.3 * (torch.arange(k_len) - torch.arange(q_len)[:, None]).abs().expand(2, q_len, k_len)


def test_the_fused_path_takes_the_library_s_position_bias_alone():
    b = block()
    assert b._why_not_fused(on_the_gpu(), None, FM.RelativePositionBias(2)) is None
    assert "RelativePositionBias" in b._why_not_fused(on_the_gpu(), None, Slope())
