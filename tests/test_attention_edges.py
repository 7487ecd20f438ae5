"""Self-attention where rows are extreme: scores whose common level hides the sum of their exponentials, queries without keys that hold NaN,
tables with low values of different size, roundings that add up."""
import math

import pytest
import torch

from attention_ref import check, reference
from test_attention import BF16, F32, normal, run_case
from wavernn_amd import _lib
from wavernn_amd import attention as A

gpu = pytest.mark.gpu
LOWEST = torch.finfo(F32).min


def gradients(leaves, dout, **rule):
    leaves = [x.detach().requires_grad_() for x in leaves]
    out = A.attention(*leaves[:3], bias_table=leaves[3] if len(leaves) > 3 else None, **rule)
    return [out.detach(), *torch.autograd.grad(out, leaves, dout)]


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,G,Tq,Tk,D", [(2, 2, 40, 40, 16), (4, 2, 20, 700, 64), (2, 1, 150, 130, 128), (2, 2, 70, 300, 200)])
@pytest.mark.parametrize("low", [-1e5, -1e6, -1e8, -1e9, -1e30, LOWEST, 1e9])
def test_gradients_where_all_biases_of_a_query_lie_far_from_zero(dtype, H, G, Tq, Tk, D, low):
    """A common shift of a row's scores changes neither its softmax nor a gradient, however large it is beside the logarithm of the row's sum.
    Queries are zero, so that the scores are the biases themselves and no bit of them is lost beside the shift: the values and bounds are those
    of the same table without the shift (head 0), or, where a few near distances keep zero (the other heads), with -60 in place of the
    low values: exp(-60) is 1e-26."""
    k, v, dout = normal(1, 2, G, Tk, D, dtype=dtype), normal(2, 2, G, Tk, D, dtype=dtype), normal(3, 2, H, Tq, D, dtype=dtype)
    q = torch.zeros(2, H, Tq, D, device="cuda", dtype=dtype)
    mask = (torch.rand(2, Tk, generator=torch.Generator().manual_seed(4)) < 0.3).cuda()
    mask[1, Tk // 2:] = True                      # queries that are left distant keys alone
    table = torch.full((8, H), low)
    same = torch.zeros(8, H)
    if low < 0:
        table[:2, 1:], same[2:, 1:] = 0.0, -60.0
    rule = dict(key_mask=mask, max_distance=20)
    got = gradients([q, k, v, table.cuda()], dout, **rule)
    want = reference(q, k, v, dout, table=same, **rule)
    # what -60 adds in the reference and the low values do not: less than exp(-60) = 8.8e-27 a pair of P, times |dP| + |delta| < 1e4 (sums of 200
    # products of normal values), over at most 2 x 150 x 700 pairs
    for name, x in zip(("out", "dq", "dk", "dv", "dtable"), got):
        check(name, x, (want[name][0], want[name][1] + 8.8e-27 * 1e4 * 2.1e5))


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [16, 128, 200])
def test_gradients_where_all_scores_of_a_query_lie_far_from_zero(dtype, D):
    """The same by the scores: all keys of a head are one vector, whose products with a query are a common shift of some 1e7; the softmax is even
    and dk = dS^T q is all that the queries enter.  Queries and keys are small whole numbers (times 16), so that every product and sum is
    exact in 32 bits in whatever order a pass takes them, and a score the same number in each."""
    g = torch.Generator().manual_seed(0)
    q = (torch.randint(-255, 256, (2, 2, 90, D), generator=g) * 16).to(dtype).cuda()
    k = torch.randint(-7, 8, (2, 2, 1, D), generator=g).to(dtype).cuda().expand(2, 2, 150, D)
    v, dout = normal(2, 2, 2, 150, D, dtype=dtype), normal(3, 2, 2, 90, D, dtype=dtype)
    out, dq, dk, dv = gradients([q, k, v], dout, scale=64.0)
    even = reference(torch.zeros_like(q), k, v, dout, scale=64.0)
    check("out", out, even["out"])
    check("dv", dv, even["dv"])
    # dq: a sum of dS over the keys, zero but for roundings, times the key; dk from the even softmax's dS
    check("dq", dq, even["dq"])
    go, vd = dout.double().cpu(), v.double().cpu()
    ds = ((go @ vd.transpose(-1, -2)) - (go * vd.mean(2, keepdim=True)).sum(-1, keepdim=True)) / 150
    qd, ub, u = q.double().cpu(), torch.finfo(dtype).eps / 2, 2.0 ** -24
    # dS: rounded where it enters the product (bfloat16), made of 32-bit sums of dP and of delta, delta of the rounded output
    size = (go.abs() @ vd.abs().transpose(-1, -2) + (go.abs() * vd.abs().mean(2, keepdim=True)).sum(-1, keepdim=True)) / 150
    off = 2 * ub * ds.abs() + (2 * D + 400) * u * size + (2 * ub * (go.abs() * vd.abs().mean(2, keepdim=True)).sum(-1, keepdim=True) / 150)
    dkx = ds.transpose(-1, -2) @ qd * 64
    check("dk", dk, (dkx, off.transpose(-1, -2) @ qd.abs() * 64 * (1 + 1e-3) + ub * dkx.abs()))


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Tq,Tk", [(3, 900), (150, 90), (40, 1500)])
def test_backward_entry_that_makes_the_statistics_anew(dtype, Tq, Tk):
    """The C entry without statistics against the one that is handed them: the same bits."""
    q, k, v, dout = (normal(i, 2, 4 if i in (0, 3) else 2, Tq if i in (0, 3) else Tk, 64, dtype=dtype) for i in range(4))
    lens = torch.tensor([Tk, 5], dtype=torch.int32, device="cuda")
    want = gradients([q, k, v], dout, key_lens=lens)
    lib = _lib.load()
    desc = A._desc(q, k, v, None, None, lens, None, False, 0.125, 128, True)
    got = [want[0], *(torch.full_like(x, math.nan) for x in (q, k, v))]
    strides = [x.stride()[:3] for x in (want[0], dout, *got[1:])]
    grads = A._GRADS.pack(want[0].data_ptr(), 0, dout.data_ptr(), *(x.data_ptr() for x in got[1:]), 0, *(s for x in strides for s in x))
    size = lib.wrnn_attention_backward_workspace_bytes(desc)
    space = torch.empty(size, dtype=torch.uint8, device="cuda")
    assert lib.wrnn_attention_backward(desc, grads, space.data_ptr(), size, torch.cuda.current_stream().cuda_stream) == 0
    for x, y in zip(got, want):
        assert torch.equal(x, y)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 1e-6])
@pytest.mark.parametrize("D,Tq,Tk", [(64, 70, 90), (200, 70, 90), (36, 3, 200), (128, 50, 700)])
def test_scales_of_any_sign(dtype, scale, D, Tq, Tk):
    mask = (torch.rand(2, Tk, generator=torch.Generator().manual_seed(2)) < 0.3).cuda()
    run_case(dtype, 2, 4, 2, Tq, Tk, D, scale=scale, mask=mask, causal=True)
    run_case(dtype, 2, 4, 2, Tq, Tk, D, scale=scale, mask=mask, table=normal(3, 16, 4))


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("B,H,G,Tq,Tk,D", [(2, 2, 2, 50, 40, 64), (2, 4, 2, 300, 130, 128), (2, 2, 1, 90, 70, 200), (40, 4, 4, 160, 160, 32),
                                           (2, 2, 2, 7, 300, 64)])
@pytest.mark.parametrize("with_table", [False, True])
def test_what_lies_at_queries_without_keys_is_never_used(dtype, bad, B, H, G, Tq, Tk, D, with_table):
    """Queries that causality or a row's mask leaves no key, with NaN or infinities in q and in the output's gradient: no bit of the other rows'
    results changes, and their own are zero."""
    q, k, v, dout = (normal(i, B, H if i in (0, 3) else G, Tq if i in (0, 3) else Tk, D, dtype=dtype) for i in range(4))
    table = [normal(5, 16, H)] if with_table else []
    start = torch.full((B,), -(Tq // 3), dtype=torch.int32, device="cuda")
    mask = torch.zeros(B, Tk, dtype=torch.bool, device="cuda")
    mask[1], mask[0, 2] = True, True
    lens = torch.full((B,), Tk - 2, dtype=torch.int32, device="cuda")
    lens[1] = 0
    for rule, first in ((dict(causal=True, q_start=start), True), (dict(key_mask=mask), False), (dict(key_lens=lens), False),
                        (dict(key_mask=mask, causal=True, q_start=start), True)):
        empty = torch.zeros(B, Tq, dtype=torch.bool, device="cuda")
        if first:
            empty[:, :Tq // 3] = True
        if "key_mask" in rule or "key_lens" in rule:
            empty[1] = True
        empty = empty[:, None, :, None]
        want = gradients([q, k, v] + table, dout, **rule)
        got = gradients([q.masked_fill(empty, bad), k, v] + table, dout.masked_fill(empty, bad), **rule)
        for name, x, y in zip(("out", "dq", "dk", "dv", "dtable"), got, want):
            assert torch.equal(x, y), (name, rule.keys())
        assert not got[0].masked_select(empty).any() and not got[1].masked_select(empty).any()


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [64, 128, 200])
def test_left_out_keys_get_no_gradient(dtype, D):
    """Keys that a mask leaves out have zero gradients whatever a query in use holds, and table entries of distances that only left-out pairs
    have take no part, NaN included."""
    q, k, v, dout = (normal(i, 2, 2, 80, D, dtype=dtype) for i in range(4))
    mask = torch.zeros(2, 80, dtype=torch.bool, device="cuda")
    mask[:, 60:] = True
    spoiled = q.clone()
    spoiled[:, :, 33] = math.nan
    got = gradients([spoiled, k, v], dout, key_mask=mask)
    assert not got[2][:, :, 60:].any() and not got[3][:, :, 60:].any()
    table = normal(5, 16, 2)
    rule = dict(causal=True, max_distance=20)           # distances ahead (the second half of the table) are never allowed
    want = gradients([q, k, v, table], dout, **rule)
    table[9:] = math.nan
    got = gradients([q, k, v, table], dout, **rule)
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    start = torch.zeros(2, dtype=torch.int32, device="cuda")      # queries 0 .. 3 against keys 0 .. 9 of 80: no distance above 9 is allowed
    mask = torch.arange(80, device="cuda").expand(2, 80) >= 10
    table = normal(5, 64, 2)
    rule = dict(q_start=start, key_mask=mask, max_distance=128)
    want = gradients([q[:, :, :4], k, v, table], dout[:, :, :4], **rule)
    table[32 + 14:] = math.nan
    got = gradients([q[:, :, :4], k, v, table], dout[:, :, :4], **rule)
    for x, y in zip(got, want):
        assert torch.equal(x, y)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Tq,D", [(60, 16), (60, 200), (3, 64)])
@pytest.mark.parametrize("low,lower", [(-1e30, LOWEST), (-1e31, -1e35), (-2e38, LOWEST), (-3e38, LOWEST)])
def test_low_values_of_a_table_keep_their_order(dtype, Tq, D, low, lower):
    """A key whose bias is `lower` gets no weight beside one of `low`, as finite as both are."""
    q, k, v, dout = (normal(i, 1, 2, Tq if i in (0, 3) else 60, D, dtype=dtype) for i in range(4))
    table, same = torch.full((8, 2), lower), torch.full((8, 2), -math.inf)
    table[1::2] = low
    same[1::2] = 0.0
    q = torch.zeros_like(q)               # any score vanishes beside such a bias
    rule = dict(max_distance=20)
    got = gradients([q, k, v, table.cuda()], dout, **rule)
    want = reference(q, k, v, dout, table=same, **rule)
    for name, x in zip(("out", "dq", "dk", "dv", "dtable"), got):
        check(name, x, want[name])
    lse = A.attention(q, k, v, bias_table=table.cuda(), return_lse=True, **rule)[1]
    assert bool(((lse / low - 1).abs() < 1e-5).all())


@gpu
@pytest.mark.parametrize("D", [64, 128, 200])
@pytest.mark.parametrize("Tk", [60, 300, 700, 1000, 1500])
@pytest.mark.parametrize("H", [2, 256])
def test_rounded_outputs_do_not_reach_the_keys_gradients(D, Tk, H):
    """bfloat16, values far from zero: delta = rowsum(dout * out) carries the rounding of out, here some 4 % of the spread of dS, and dk must not,
    in however many shares the keys are worked on.  What may be left: dS is rounded where it enters its product (independent roundings, a
    half step over sqrt 3 each) and dk where it is stored (half a step); all queries are one vector, so neither is magnified."""
    Tq = 100 if H == 2 else 40
    q, k, dout = normal(0, 1, H, 1, D, dtype=BF16).expand(1, H, Tq, D), normal(1, 1, H, Tk, D, dtype=BF16), normal(3, 1, H, Tq, D, dtype=BF16)
    v = (normal(2, 1, H, Tk, D) + 30).to(BF16)
    dk = gradients([q, k, v], dout)[2].double()
    qd, kd, vd, go = (x.double() for x in (q.contiguous(), k, v, dout))
    p = torch.softmax(qd @ kd.transpose(-1, -2).contiguous() / D ** 0.5, -1)
    dp = go @ vd.transpose(-1, -2).contiguous()
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    want = ds.transpose(-1, -2).contiguous() @ qd / D ** 0.5
    half_step = torch.finfo(BF16).eps / 2
    assert float((dk - want).norm() / want.norm()) < (1 + 1 / 3 ** 0.5) * half_step
