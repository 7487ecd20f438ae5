"""Self-attention at the sizes that take a kernel or a branch of their own: long rows in bfloat16 past 64 columns, few queries and divided keys in
float32 past 128, masks whose tail spans several scans, the second plane of dS."""
import pytest
import torch

from attention_ref import buckets, check, reference
from test_attention import BF16, F32, normal, run_case
from wavernn_amd import attention as A

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("D", [100, 128, 200])
@pytest.mark.parametrize("Tq,Tk", [(150, 1100), (70, 1500), (1300, 1300)])
@pytest.mark.parametrize("causal", [False, True])
def test_long_rows_in_bfloat16(D, Tq, Tk, causal):
    """More than 1024 keys: blocks of queries that reach fewer (causality) and more."""
    run_case(BF16, 1, 2, 1, Tq, Tk, D, causal=causal, seed=D)
    run_case(BF16, 1, 2, 2, Tq, Tk, D, causal=causal, table=normal(5, 32, 2), bidirectional=not causal, lens=torch.tensor([Tk - 5]).cuda(), seed=D)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [132, 200, 256])
@pytest.mark.parametrize("Tq", [1, 20, 70, 140])
@pytest.mark.parametrize("Tk", [40, 700, 1100])
def test_many_columns(dtype, D, Tq, Tk):
    """Few queries, and keys divided over workgroups, with the joining launches behind both passes."""
    mask = (torch.rand(2, Tk, generator=torch.Generator().manual_seed(D)) < 0.2).cuda()
    run_case(dtype, 2, 2, 1, Tq, Tk, D, mask=mask, seed=Tq)
    run_case(dtype, 1, 1, 1, Tq, Tk, D, causal=True, table=normal(5, 16, 1), seed=Tq)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Tq,D", [(1, 64), (20, 128), (60, 64), (60, 200)])
@pytest.mark.parametrize("left", [0, 1, 3999, 4000])
def test_masks_with_a_long_tail(dtype, Tq, D, left):
    """The end of a row's keys is found in blocks from behind: here it lies two and three blocks before the last key, or nowhere."""
    Tk = 9000
    mask = torch.ones(2, Tk, dtype=torch.bool, device="cuda")
    mask[:, :left] = False
    mask[1, 5:left] = True
    run_case(dtype, 2, 2, 1, Tq, Tk, D, mask=mask, seed=left)


@gpu
@pytest.mark.parametrize("D,Tk", [(16, 300), (64, 60), (64, 300), (64, 1500), (100, 60), (128, 300), (128, 1000), (200, 1000)])
def test_score_gradients_in_two_planes(D, Tk):
    """bfloat16: dq is off by no more than its own rounding, half a step over sqrt 3 of its norm at most (the mantissas at their smallest).  With dS
    rounded to one plane it is 2.4e-3 to 3.3e-3; one plane is what more than 1024 keys get past 64 columns."""
    q, k, v, dout = (normal(i, 2, 4, 200 if i in (0, 3) else Tk, D, dtype=BF16).requires_grad_(i < 3) for i in range(4))
    got = torch.autograd.grad(A.attention(q, k, v), q, dout)[0].double().cpu()
    x = [t.detach().double().cpu() for t in (q, k, v, dout)]
    p = torch.softmax(x[0] @ x[1].transpose(-1, -2) / D ** 0.5, -1)
    dp = x[3] @ x[2].transpose(-1, -2)
    want = (p * (dp - (p * dp).sum(-1, keepdim=True))) @ x[1] / D ** 0.5
    assert float((got - want).norm() / want.norm()) < torch.finfo(BF16).eps / 2 / 3 ** 0.5


@gpu
@pytest.mark.parametrize("Tq", [1, 40])
def test_offsets_past_32_bits(Tq):
    """A cache of 2.5e9 elements of which the last keys alone are left: the same as those keys by themselves (which another number of workgroups
    sums in another order: the bounds are run_case's on both sides), gradients in their places, everything before them untouched by NaN."""
    H, Tk, D, last = 32, 600_001, 128, 100
    cache = torch.empty(1, Tk, H, D, dtype=BF16, device="cuda")
    assert cache.numel() > 2 ** 31
    cache[:, ::1000] = float("nan")
    cache[:, -last:] = normal(1, 1, last, H, D, dtype=BF16)
    k = cache.permute(0, 2, 1, 3)
    q, dout = normal(0, 1, H, Tq, D, dtype=BF16), normal(2, 1, H, Tq, D, dtype=BF16)
    mask = torch.arange(Tk, device="cuda")[None] < Tk - last
    few = k[:, :, -last:].contiguous()
    want = reference(q, few, few, dout)
    leaves = [q.requires_grad_(), k.requires_grad_()]
    out = A.attention(q, k, k, key_mask=mask)
    check("out", out, want["out"])
    dq, dk = torch.autograd.grad(out, leaves, dout)
    check("dq", dq, want["dq"])
    # dk + dv, added up in bfloat16 by autograd
    value = want["dk"][0] + want["dv"][0]
    check("dk + dv", dk[:, :, -last:], (value, want["dk"][1] + want["dv"][1] + torch.finfo(BF16).eps / 2 * (want["dk"][0].abs() + want["dv"][0].abs())))
    assert not dk[:, :, :-last].any()


@gpu
def test_dense_bias_past_32_bits():
    """3.2e9 values: the last rows, and the gradient of their sum, which counts the pairs of each bucket (whole numbers below 2^24 a workgroup,
    then 64 bits; half a step of bfloat16 where it is stored)."""
    H, T = 3, 32768
    table = normal(0, 32, H, dtype=BF16).requires_grad_()
    out = A.relative_position_bias(table, T, T)
    rel = torch.arange(T) - (T - 1)
    which = buckets(rel, 32, 128, True)
    assert torch.equal(out[-1, -1].cpu(), table.detach()[:, -1].cpu()[which])
    ahead = buckets(-rel, 32, 128, True)                      # of distances 0 .. T - 1 ahead, T - distance pairs each
    pairs = (T + rel).double()
    count = torch.zeros(32, dtype=torch.float64).index_add_(0, which, pairs)
    count.index_add_(0, ahead[:-1], pairs[:-1])
    got = torch.autograd.grad(out, table, torch.ones((), dtype=BF16, device="cuda").expand_as(out))[0].double().cpu()
    assert bool(((got - count[:, None]).abs() <= torch.finfo(BF16).eps / 2 * count[:, None]).all())
