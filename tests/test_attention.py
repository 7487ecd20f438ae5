"""Self-attention and the relative position bias against their definition in 64 bits (tests/attention_ref.py), at the sizes, layouts
and masks where they can go wrong; refusals."""
import ctypes as C
import math

import pytest
import torch

from attention_ref import buckets, check, reference
from wavernn_amd import _lib
from wavernn_amd import attention as A

gpu = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def normal(seed, *shape, dtype=F32, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * spread).to(dtype).cuda()


def run_case(dtype, B, H, G, Tq, Tk, D, *, mask=None, lens=None, start=None, causal=False, scale=None, table=None, max_distance=128,
             bidirectional=True, layout="bhtd", train=True, spread=1.5, seed=0):
    """One case through attention and, with train, its backward pass; everything against the reference."""
    def make(s, n, heads, T, sp=1.0):
        if layout == "bhtd":
            return normal(s, n, heads, T, D, dtype=dtype, spread=sp)
        if layout == "tbhd":        # what a projection of [time, batch, width] gives
            return normal(s, T, n, heads, D, dtype=dtype, spread=sp).permute(1, 2, 0, 3)
        if layout == "odd":         # rows that start off 16 bytes, with a gap behind them
            return normal(s, n, T, heads, D + 3, dtype=dtype, spread=sp)[..., 1:D + 1].permute(0, 2, 1, 3)
        raise ValueError(layout)

    q, k, v = make(seed, B, H, Tq, spread), make(seed + 1, B, G, Tk), make(seed + 2, B, G, Tk)
    dout = make(seed + 3, B, H, Tq) if train else None
    rule = dict(key_mask=mask, key_lens=lens, q_start=start, causal=causal, scale=scale, max_distance=max_distance, bidirectional=bidirectional)
    if train:
        q, k, v = (x.detach().requires_grad_() for x in (q, k, v))
        if table is not None:
            table = table.detach().requires_grad_()
    out, lse = A.attention(q, k, v, bias_table=table, return_lse=True, **rule)
    want = reference(q, k, v, dout, table=table, **rule)
    check("out", out, want["out"])
    check("lse", lse, want["lse"])
    if train:
        leaves = [q, k, v] + ([table] if table is not None else [])
        got = torch.autograd.grad(out, leaves, dout)
        for name, g in zip(("dq", "dk", "dv", "dtable"), got):
            check(name, g, want[name])
    return out


# ------------------------------------------------------------------ CPU: the rule and the refusals


@pytest.mark.parametrize("count,most,two", [(32, 128, True), (32, 128, False), (16, 64, True), (8, 20, False), (4, 2, True), (2, 2, False),
                                            (64, 1000, True), (256, 1024, False), (5, 9, False)])
def test_bucket_edges_are_the_logarithmic_rule(count, most, two):
    edges = A.bucket_edges(count, most, two)
    side = count // 2 if two else count
    e = side // 2
    assert len(edges) == side - e - 1 and edges == sorted(edges)
    far = torch.arange(0, most + 5)
    mine = torch.where(far < e, far, e + torch.bucketize(far, torch.tensor(edges, dtype=torch.int64), right=True))
    assert torch.equal(mine, buckets(-far, count, most, two))
    # and against the logarithms, away from the borders
    for d in range(e + 1, most):
        x = math.log(d / e) / math.log(most / e) * (side - e)
        if abs(x - round(x)) > 1e-9:
            assert int(mine[d]) == min(side - 1, e + int(x))


@pytest.mark.parametrize("rule", [(1, 128, True), (2, 128, True), (7, 128, True), (258, 1024, False), (32, 8, True), (32, 1025, True)])
def test_bucket_rules_outside_the_range_are_refused(rule):
    with pytest.raises(ValueError):
        A.bucket_edges(*rule)
    with pytest.raises(ValueError):
        A.RelativePositionBias(2, *rule)


def test_no_cpu_fallback():
    x = torch.zeros(1, 1, 2, 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        A.attention(x, x, x)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        A.RelativePositionBias(2)(3, 3)


def test_packed_structures_are_the_headers():
    assert A._DESC.size == C.sizeof(_lib.AttentionDesc) and A._GRADS.size == C.sizeof(_lib.AttentionGrads)
    i3 = _lib.I64x3
    e = (C.c_int32 * 3)(1, 2, 3)
    whole = _lib.AttentionDesc(1, 2, 3, 4, 5, 6, 7, 1, 8, 9, 1, 0.5, 11, 12, 13, i3(14, 15, 16), i3(17, 18, 19), i3(20, 21, 22), 23, 24, 25, 26, 27, e)
    assert bytes(whole) == A._DESC.pack(1, 2, 3, 4, 5, 6, 7, 1, 8, 9, 1, 0.5, *range(11, 28), C.addressof(e))
    grads = _lib.AttentionGrads(1, 2, 3, 4, 5, 6, 7, i3(8, 9, 10), i3(11, 12, 13), i3(14, 15, 16), i3(17, 18, 19), i3(20, 21, 22))
    assert bytes(grads) == A._GRADS.pack(*range(1, 23))


def desc(**kw):
    i3 = _lib.I64x3(0, 0, 0)
    d = _lib.AttentionDesc(dtype=0, batch=1, heads=2, kv_heads=2, q_len=4, k_len=4, head_dim=8, scale=1.0, q=16, k=16, v=16, q_stride=i3,
                           k_stride=i3, v_stride=i3)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("change,message", [
    (dict(dtype=2), b"neither float32 nor bfloat16"), (dict(batch=-1), b"negative size"), (dict(q_len=-1), b"negative size"),
    (dict(head_dim=0), b"head dimension"), (dict(head_dim=257), b"head dimension"), (dict(heads=3), b"evenly"),
    (dict(kv_heads=0), b"evenly"), (dict(q=None), b"null pointer"), (dict(v=None), b"null pointer"),
    (dict(q_len=1 << 29), b"2^28"), (dict(batch=1 << 21, q_len=64), b"too large"),
    (dict(bias_table=16, num_buckets=1, max_distance=4), b"buckets"), (dict(bias_table=16, num_buckets=2, max_distance=4, bidirectional=1), b"buckets"),
    (dict(bias_table=16, num_buckets=8, max_distance=4), b"max_distance"), (dict(bias_table=16, num_buckets=8, max_distance=2000), b"max_distance"),
    (dict(bias_table=16, num_buckets=8, max_distance=64), b"bucket edges"),
    (dict(bias_table=16, num_buckets=8, max_distance=64, bucket_edges=(C.c_int32 * 3)(9, 8, 7)), b"ascend"),
    (dict(bias_table=16, num_buckets=8, max_distance=64, bucket_edges=(C.c_int32 * 3)(8, 9, 65)), b"ascend"),
])
def test_c_entry_refuses_before_any_device_work(change, message):
    lib = _lib.load()
    d = desc(**change)
    i3 = _lib.I64x3(0, 0, 0)
    assert lib.wrnn_attention_forward(C.byref(d), 16, i3, None, None, 0, None) != 0
    assert message in lib.wrnn_last_error()
    assert lib.wrnn_attention_backward(C.byref(d), C.byref(_lib.AttentionGrads()), None, 0, None) != 0
    assert message in lib.wrnn_last_error()


def test_c_entry_refuses_missing_outputs_and_workspaces():
    lib = _lib.load()
    d, i3 = desc(), _lib.I64x3(0, 0, 0)
    assert lib.wrnn_attention_forward(None, 16, i3, None, None, 0, None) != 0
    assert lib.wrnn_attention_forward(C.byref(d), None, i3, None, None, 0, None) != 0
    assert lib.wrnn_attention_backward(C.byref(d), None, None, 0, None) != 0
    g = _lib.AttentionGrads(out=16, lse=16, dout=16, dq=16, dk=16, dv=16)
    assert lib.wrnn_attention_backward(C.byref(d), C.byref(g), None, 0, None) != 0 and b"workspace" in lib.wrnn_last_error()
    g.dtable = 16
    assert lib.wrnn_attention_backward(C.byref(d), C.byref(g), 16, 1 << 20, None) != 0 and b"without a table" in lib.wrnn_last_error()
    g.dtable, g.dk = None, None
    assert lib.wrnn_attention_backward(C.byref(d), C.byref(g), 16, 1 << 20, None) != 0 and b"null pointer" in lib.wrnn_last_error()
    one = desc(batch=1, q_len=1, k_len=100000)
    assert lib.wrnn_attention_workspace_bytes(C.byref(one)) > 0
    assert lib.wrnn_attention_forward(C.byref(one), 16, i3, None, None, 0, None) != 0 and b"workspace" in lib.wrnn_last_error()
    assert lib.wrnn_attention_forward(C.byref(desc(batch=0)), None, i3, None, None, 0, None) == 0      # nothing to do
    e = (C.c_int32 * 3)(8, 16, 32)
    assert lib.wrnn_relative_bias_forward(None, 0, 1, 2, 2, 0, 8, 64, 0, e, None, None) != 0 and b"null pointer" in lib.wrnn_last_error()
    assert lib.wrnn_relative_bias_forward(16, 7, 1, 2, 2, 0, 8, 64, 0, e, 16, None) != 0
    assert lib.wrnn_relative_bias_forward(16, 0, 1, -2, 2, 0, 8, 64, 0, e, 16, None) != 0
    assert lib.wrnn_relative_bias_backward(16, 0, 1, 2, 2, 0, 8, 64, 0, e, 16, None, 0, None) != 0 and b"workspace" in lib.wrnn_last_error()


@gpu
def test_refusals():
    x = torch.zeros(2, 4, 3, 8, device="cuda")
    y = torch.zeros(2, 2, 5, 8, device="cuda")
    bad = [lambda: A.attention(x[0], y, y), lambda: A.attention(x, y, y[:, :, :4]), lambda: A.attention(x, y[:1], y[:1]),
           lambda: A.attention(x, y.repeat(1, 2, 1, 1)[:, :3], y.repeat(1, 2, 1, 1)[:, :3]),
           lambda: A.attention(torch.zeros(2, 4, 3, 300, device="cuda"), *[torch.zeros(2, 4, 3, 300, device="cuda")] * 2),
           lambda: A.attention(x, y, y, key_mask=torch.zeros(2, 4, dtype=torch.bool, device="cuda")),
           lambda: A.attention(x, y, y, key_mask=torch.zeros(2, 5, device="cuda")),
           lambda: A.attention(x, y, y, key_mask=torch.zeros(2, 5, dtype=torch.bool)),
           lambda: A.attention(x, y, y, key_lens=torch.zeros(3, dtype=torch.int32, device="cuda")),
           lambda: A.attention(x, y, y, q_start=torch.zeros(2, device="cuda")),
           lambda: A.attention(x, y, y, bias_table=torch.zeros(32, 3, device="cuda")),
           lambda: A.attention(x, y, y, bias_table=torch.zeros(32, 4, device="cuda"), max_distance=5000),
           lambda: A.relative_position_bias(torch.zeros(32, 4, device="cuda"), -1, 3)]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    for f in (lambda: A.attention(x.half(), y.half(), y.half()), lambda: A.attention(x, y.bfloat16(), y), lambda: A.attention(x.double(), y.double(), y.double()),
              lambda: A.relative_position_bias(torch.zeros(32, 4, device="cuda").half(), 3, 3)):
        with pytest.raises(TypeError):
            f()
    with pytest.raises(RuntimeError):
        A.attention(x, y.cpu(), y)


# ------------------------------------------------------------------ GPU: values and gradients


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [1, 3, 8, 12, 36, 64, 65, 80, 128, 196, 256])
def test_head_dims(dtype, D):
    run_case(dtype, 2, 2, 2, 37, 45, D, seed=D)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Tq,Tk", [(1, 1), (1, 33), (2, 300), (31, 32), (32, 31), (33, 64), (129, 65), (128, 128), (200, 1), (257, 511)])
@pytest.mark.parametrize("causal", [False, True])
def test_lengths(dtype, Tq, Tk, causal):
    run_case(dtype, 2, 2, 1, Tq, Tk, 64, causal=causal, seed=Tq + Tk)     # causal with Tq > Tk leaves rows empty


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layout", ["tbhd", "odd"])
@pytest.mark.parametrize("D", [24, 64, 128])
def test_layouts(dtype, layout, D):
    out = run_case(dtype, 3, 4, 4, 70, 70, D, layout=layout, mask=torch.arange(70, device="cuda")[None] >= torch.tensor([[70], [31], [5]], device="cuda"))
    if layout == "tbhd":
        assert out.permute(2, 0, 1, 3).is_contiguous()      # the order of the projections around attention


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("big", [False, True])     # small calls and those with enough workgroups take different kernels
def test_masks_that_leave_rows_empty(dtype, big):
    B, H, T = (40, 4, 160) if big else (4, 2, 50)
    g = torch.Generator().manual_seed(3)
    mask = (torch.rand(B, T, generator=g) < 0.4).cuda()
    mask[0] = True                      # no key at all
    mask[1] = False
    mask[1, :-1] = True                 # the last key alone
    lens = torch.randint(0, T + 1, (B,), generator=g, dtype=torch.int32).cuda()
    lens[2] = 0
    lens[3] = T + 100                   # clamped
    lens[1] = T
    out = run_case(dtype, B, H, H, T, T, 32, mask=mask)
    assert not out[0].any()
    run_case(dtype, B, H, H, T, T, 32, lens=lens.long())
    run_case(dtype, B, H, H, T, T, 32, mask=mask, lens=lens, causal=True)
    lens[2] = -5
    assert not A.attention(*[normal(5, B, H, T, 32, dtype=dtype)] * 3, key_lens=lens)[2].any()


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("big", [False, True])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_what_lies_at_masked_keys_is_never_used(dtype, big, bad):
    B, H, T, D = (40, 4, 160, 64) if big else (2, 2, 50, 64)
    q, k, v, dout = (normal(i, B, H, T, D, dtype=dtype) for i in range(4))
    lens = torch.full((B,), T - 13, dtype=torch.int32, device="cuda")
    mask = torch.zeros(B, T, dtype=torch.bool, device="cuda")
    mask[:, 7] = True
    start = torch.zeros(B, dtype=torch.int32, device="cuda")
    for rule in (dict(key_lens=lens), dict(key_mask=mask), dict(causal=True, q_start=start - T // 2)):
        clean = [x.clone().requires_grad_() for x in (q, k, v)]
        dirty = [x.clone() for x in (q, k, v)]
        for x in dirty[1:]:
            if "key_lens" in rule:
                x[:, :, T - 13:] = bad
            elif "key_mask" in rule:
                x[:, :, 7] = bad
            else:
                x[:, :, T - T // 2:] = bad      # past every query's reach
        dirty = [x.requires_grad_() for x in dirty]
        a, b = A.attention(*clean, **rule), A.attention(*dirty, **rule)
        assert torch.equal(a, b)
        for x, y in zip(torch.autograd.grad(a, clean, dout), torch.autograd.grad(b, dirty, dout)):
            assert torch.equal(x, y)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,G", [(4, 1), (6, 2), (32, 1), (33, 1)])
@pytest.mark.parametrize("Tq", [1, 3, 40])
def test_shared_key_heads_and_caches(dtype, H, G, Tq):
    lens = torch.tensor([200, 7, 133], dtype=torch.int32, device="cuda")
    start = (lens - Tq).clamp(min=0)
    run_case(dtype, 3, H, G, Tq, 200, 64, lens=lens, start=start, causal=True, train=Tq != 1, seed=H + Tq)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Tk", [4096, 5001])
def test_one_token_over_a_long_cache(dtype, Tk):
    lens = torch.tensor([Tk, 1, 0, 2222], dtype=torch.int32, device="cuda")
    table = normal(9, 32, 8)
    run_case(dtype, 4, 8, 2, 1, Tk, 128, lens=lens, train=False)
    run_case(dtype, 4, 8, 2, 1, Tk, 128, lens=lens, start=lens - 1, table=table, bidirectional=False, train=False)
    run_case(dtype, 1, 8, 8, 1, Tk, 40, train=True)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Tq,Tk,D", [(40, 40, 16), (130, 210, 64), (300, 300, 128), (65, 33, 200)])
@pytest.mark.parametrize("count,most,two", [(32, 128, True), (32, 128, False), (8, 20, True), (2, 2, False), (64, 1000, True)])
def test_bias(dtype, Tq, Tk, D, count, most, two):
    g = torch.Generator().manual_seed(1)
    mask = (torch.rand(2, Tk, generator=g) < 0.2).cuda()
    run_case(dtype, 2, 2, 2, Tq, Tk, D, table=normal(7, count, 2), max_distance=most, bidirectional=two, mask=mask, causal=not two)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_bias_with_many_workgroups_and_starts(dtype):
    start = torch.tensor([0, 50, -30, 1000, 7] * 8, dtype=torch.int32, device="cuda")
    run_case(dtype, 40, 4, 2, 140, 150, 64, table=normal(7, 32, 4), start=start)
    run_case(dtype, 40, 4, 2, 140, 150, 64, table=normal(7, 32, 4), start=start, causal=True, bidirectional=False)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("low", [-math.inf, torch.finfo(torch.float32).min])
def test_bias_of_the_lowest_value(dtype, low):
    table = torch.zeros(8, 2)
    table[3:, 0] = low                  # head 0 is left its three nearest distances
    table[:, 1] = low                   # head 1 nothing: empty with -inf, uniform with the lowest finite value
    q, k, v = (normal(i, 1, 2, 40, 16, dtype=dtype) for i in range(3))
    out = A.attention(q, k, v, bias_table=table.cuda(), max_distance=20, bidirectional=False, causal=True)
    ref = reference(q, k, v, table=torch.where(table < -1e30, -1e30, table) if low > -math.inf else table, max_distance=20, bidirectional=False, causal=True)["out"][0]
    if low > -math.inf:
        ref[:, 1] = v[:, 1].double().cpu().cumsum(1) / torch.arange(1, 41)[:, None]      # scores vanish beside the bias
    assert float((out.double().cpu() - ref).abs().max()) < (1e-5 if dtype == F32 else 2 * 2 ** -8 * 4)


@gpu
def test_large_scores():
    for spread in (30.0, 300.0):        # rows whose softmax is nearly one key, far from zero
        run_case(F32, 2, 2, 2, 64, 200, 64, spread=spread)
        run_case(BF16, 2, 2, 2, 64, 200, 64, spread=spread)


@gpu
def test_gradients_against_differences():
    """Central differences of the 64-bit definition along random directions: the gradient's formula itself."""
    q, k, v, dout = normal(0, 1, 4, 9, 8), normal(1, 1, 2, 11, 8), normal(2, 1, 2, 11, 8), normal(3, 1, 4, 9, 8)
    table = normal(4, 8, 4)
    rule = dict(causal=True, max_distance=20, bidirectional=False)
    leaves = [x.requires_grad_() for x in (q, k, v, table)]
    got = torch.autograd.grad(A.attention(*leaves[:3], bias_table=table, **rule), leaves, dout)

    def f(xs):
        out = reference(*xs[:3], table=xs[3], **rule)["out"][0]
        return float((out * dout.double().cpu()).sum())

    for i, g in enumerate(got):
        d = normal(10 + i, *g.shape).double()
        h = 1e-5
        plus = [x.detach().double() + (h * d if j == i else 0) for j, x in enumerate(leaves)]
        minus = [x.detach().double() - (h * d if j == i else 0) for j, x in enumerate(leaves)]
        slope = (f(plus) - f(minus)) / (2 * h)
        # the difference quotient: 1e-10 (h^2) and 1e-11 / h of rounding; the gradient: 32-bit sums, well under 1e-4 of its norm
        assert abs(slope - float((g.double() * d).sum())) < 1e-4 * float(g.double().norm() * d.norm()), i


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_same_bits_every_time_and_no_keys(dtype):
    q, k, v, dout = (normal(i, 2, 4, 300, 64, dtype=dtype).requires_grad_(i < 3) for i in range(4))
    table = normal(5, 32, 4).requires_grad_()
    runs = []
    for _ in range(3):
        out = A.attention(q, k, v, bias_table=table)
        runs.append([out] + list(torch.autograd.grad(out, (q, k, v, table), dout)))
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], r))
    k0 = normal(1, 2, 4, 0, 64, dtype=dtype).requires_grad_()
    out, lse = A.attention(q, k0, k0, return_lse=True)
    assert not out.any() and bool((lse == -math.inf).all())
    assert not torch.autograd.grad(out, q, dout)[0].any()
    for shape in ((0, 4, 5, 8), (2, 4, 0, 8)):
        e = torch.zeros(shape, device="cuda", dtype=dtype, requires_grad=True)
        kk = torch.ones(shape[0], 4, 6, 8, device="cuda", dtype=dtype, requires_grad=True)
        o = A.attention(e, kk, kk)
        assert o.shape == e.shape
        assert not torch.autograd.grad(o.sum(), kk)[0].any()


@gpu
def test_broadcast_inputs_and_partial_gradients():
    q = normal(0, 3, 2, 20, 16).requires_grad_()
    k0, v0 = normal(1, 1, 1, 30, 16).requires_grad_(), normal(2, 1, 1, 30, 16).requires_grad_()
    dout = normal(3, 3, 2, 20, 16)
    k, v = k0.expand(3, 2, 30, 16), v0.expand(3, 2, 30, 16)
    got = torch.autograd.grad(A.attention(q, k, v), (q, k0, v0), dout)
    want = reference(q, k, v, dout)
    check("dq", got[0], want["dq"])
    check("dk", got[1], tuple(x.sum((0, 1), keepdim=True) for x in want["dk"]))
    check("dv", got[2], tuple(x.sum((0, 1), keepdim=True) for x in want["dv"]))
    check("dq alone", torch.autograd.grad(A.attention(q, k.detach(), v.detach()), q, dout)[0], want["dq"])
    # a gradient that is itself a broadcast
    a = torch.autograd.grad(A.attention(q, k, v).sum(), k0)[0]
    b = torch.autograd.grad(A.attention(q, k, v), k0, torch.ones_like(dout))[0]
    assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,Tq,Tk", [(1, 1, 1), (2, 128, 128), (3, 33, 70), (2, 5, 1000), (1, 700, 3), (2, 300, 301)])
@pytest.mark.parametrize("count,most,two,start", [(32, 128, True, None), (32, 128, False, None), (8, 20, True, -40), (2, 2, False, 5)])
def test_dense_bias(dtype, H, Tq, Tk, count, most, two, start):
    table = normal(0, count, H, dtype=dtype).requires_grad_()
    d = normal(1, H, Tq, Tk, dtype=dtype)
    rel = torch.arange(Tk)[None] - torch.arange(Tq)[:, None] - (Tk - Tq if start is None else start)
    which = buckets(rel, count, most, two)
    out = A.relative_position_bias(table, Tq, Tk, q_start=start, max_distance=most, bidirectional=two)
    assert torch.equal(out.cpu(), table.detach().cpu()[which].permute(2, 0, 1))          # copies: exact
    got = torch.autograd.grad(out, table, d)[0]
    hot = torch.nn.functional.one_hot(which, count).double().flatten(0, 1)
    x = d.double().cpu().flatten(1)
    # a lane adds at most rows-of-a-workgroup (64) x Tk / 64 values in 32 bits, then sums of sums; bfloat16 rounds the result
    bound = (64 + Tk + 32) * 2.0 ** -24 * (x.abs() @ hot).t() + torch.finfo(dtype).eps / 2 * (x @ hot).t().abs()
    check("dtable", got, ((x @ hot).t(), bound + 1e-30))


@gpu
def test_dense_bias_empty_and_module():
    m = A.RelativePositionBias(3, num_buckets=16, max_distance=50).cuda()
    assert m(0, 5).shape == (3, 0, 5) and m(5, 0).shape == (3, 5, 0)
    assert not torch.autograd.grad(m(0, 5).sum(), m.weight)[0].any()
    assert "num_buckets=16" in repr(m)
    q, k, v = (normal(i, 2, 3, 60, 16) for i in range(3))
    a = A.attention(q, k, v, bias_table=m.weight, max_distance=50)
    s = torch.softmax((q.double() @ k.double().transpose(-1, -2)) / 4 + m(60, 60).double(), -1) @ v.double()
    assert float((a - s).abs().max()) < 1e-5


@gpu
def test_other_stream_and_graph():
    """On a side stream, and captured: replays with new inputs, the caller's eager work between them."""
    q, k, v, dout = (normal(i, 4, 8, 1, 64) if i in (0, 3) else normal(i, 4, 2, 3000, 64) for i in range(4))
    qs, ks, vs, ds = normal(4, 2, 4, 130, 64), normal(5, 2, 4, 130, 64), normal(6, 2, 4, 130, 64), normal(7, 2, 4, 130, 64)
    table = normal(8, 32, 4)
    inputs = [qs, ks, vs, table]

    def work():
        one = A.attention(q, k, v)
        leaves = [x.detach().requires_grad_() for x in inputs]
        out = A.attention(*leaves[:3], bias_table=leaves[3])
        return [one, out.detach(), *torch.autograd.grad(out, leaves, ds)]

    eager = work()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = work()
        other = work()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    del other
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        static = work()
    for n in range(3):
        with torch.no_grad():
            for i, x in enumerate([q, k, v, ds, *inputs]):
                x.copy_(normal(20 + 10 * n + i, *x.shape))
        g.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in static]
        want = work()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), n


def test_c_entry_refuses_unaligned_workspaces():
    lib = _lib.load()
    one, i3 = desc(batch=1, q_len=1, k_len=100000), _lib.I64x3(0, 0, 0)
    assert lib.wrnn_attention_forward(C.byref(one), 16, i3, None, 8, 1 << 30, None) != 0 and b"on 16 bytes" in lib.wrnn_last_error()
    g = _lib.AttentionGrads(out=16, lse=16, dout=16, dq=16, dk=16, dv=16)
    assert lib.wrnn_attention_backward(C.byref(one), C.byref(g), 8, 1 << 30, None) != 0 and b"on 16 bytes" in lib.wrnn_last_error()


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("move", ["clone", "host", "contiguous"])
def test_saved_tensors_that_come_back_elsewhere(dtype, move):
    """Offloading and checkpointing keep copies of what a node saves: the backward pass works on those, in whatever place and strides."""
    pack, unpack = {"clone": (lambda t: t.clone(), lambda t: t), "host": (lambda t: t.cpu(), lambda t: t.cuda()),
                    "contiguous": (lambda t: t.contiguous().clone(), lambda t: t)}[move]
    def inputs():
        q, k, v = normal(0, 70, 2, 3, 4, 24, dtype=dtype).permute(2, 1, 3, 0, 4).unbind(0)
        return [q, k, v, normal(1, 16, 4)]
    mask = (torch.arange(70) >= torch.tensor([[70], [41]])).t().contiguous().t().cuda()
    lens, start = torch.tensor([66, 50]).cuda(), torch.tensor([3, -2]).cuda()
    dout = normal(2, 2, 4, 70, 24, dtype=dtype)
    def run(leaves, **kw):
        leaves = [x.detach().requires_grad_() for x in leaves]
        out = A.attention(*(x.clone() for x in leaves[:3]), bias_table=leaves[3].clone(), max_distance=40, key_mask=mask, key_lens=lens, q_start=start)
        return out, leaves
    out, leaves = run(inputs())
    want = torch.autograd.grad(out, leaves, dout)
    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        out, leaves = run(inputs())
    torch.cuda.synchronize()
    fill = [torch.full((1 << 20,), math.nan, device="cuda") for _ in range(4)]    # takes what was freed
    got = torch.autograd.grad(out, leaves, dout)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del fill


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Tq,Tk,D", [(300, 70, 64), (70, 300, 128), (150, 150, 200)])
def test_bias_gradient_of_shared_key_heads(dtype, Tq, Tk, D):
    """The table's gradient where a workgroup's share begins or ends inside a head's queries."""
    table = normal(9, 32, 6)
    run_case(dtype, 1, 6, 2, Tq, Tk, D, table=table, lens=torch.tensor([Tk - 3]).cuda())
    run_case(dtype, 2, 6, 1, Tq, Tk, D, table=table, causal=True, bidirectional=False, max_distance=1024)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [64, 128, 200])
def test_table_gradient_alone(dtype, D):
    q, k, v, dout = (normal(i, 2, 4, 200, D, dtype=dtype) for i in range(4))
    leaves = [x.detach().requires_grad_() for x in (q, k, v, normal(4, 32, 4))]
    want = torch.autograd.grad(A.attention(*leaves[:3], bias_table=leaves[3]), leaves, dout)[3]
    got = torch.autograd.grad(A.attention(q, k, v, bias_table=leaves[3]), leaves[3], dout)[0]
    assert torch.equal(got, want)


@gpu
@pytest.mark.parametrize("D", [8, 12, 36, 60, 64, 100, 132, 196, 252])
@pytest.mark.parametrize("Tq,Tk", [(1, 300), (70, 41), (200, 600)])
def test_rows_that_start_on_eight_bytes(D, Tq, Tk):
    """bfloat16 rows between 16-byte borders, with NaN before and behind each and at masked keys; whole fours of elements, so nothing is copied."""
    def rows(seed, heads, T):
        t = torch.full((2, T, heads, D + 8), math.nan, dtype=BF16, device="cuda")
        t[..., 4:4 + D] = normal(seed, 2, T, heads, D, dtype=BF16)
        return t[..., 4:4 + D].permute(0, 2, 1, 3)
    q, k, v, dout = rows(0, 6, Tq), rows(1, 3, Tk), rows(2, 3, Tk), rows(3, 6, Tq)
    assert A._rows(q) is q and A._rows(k) is k
    mask = torch.zeros(2, Tk, dtype=torch.bool, device="cuda")
    mask[0, 5:7] = mask[1, -3:] = True
    k, v = (x.masked_fill(mask[:, None, :, None], math.nan) for x in (k, v))
    clean = [x.detach().masked_fill(mask[:, None, :, None], 0.) for x in (k, v)]
    q, k, v = (x.detach().requires_grad_() for x in (q, k, v))
    out = A.attention(q, k, v, key_mask=mask)
    want = reference(q, clean[0].requires_grad_(), clean[1].requires_grad_(), dout, key_mask=mask)
    check("out", out, want["out"])
    for name, g in zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), dout)):
        check(name, g, want[name])


@pytest.mark.parametrize("change", [dict(head_dim=6), dict(dtype=1, head_dim=4), dict(dtype=1, head_dim=12, q=20), dict(head_dim=12, k=24),
                                    dict(dtype=1, head_dim=12, v_stride=(0, 0, 14))])
def test_c_entry_refuses_rows_it_cannot_read(change):
    lib = _lib.load()
    if "v_stride" in change:
        change = dict(change, v_stride=_lib.I64x3(*change["v_stride"]))
    assert lib.wrnn_attention_forward(C.byref(desc(**change)), 16, _lib.I64x3(0, 0, 0), None, None, 0, None) != 0
    assert b"fours" in lib.wrnn_last_error()
