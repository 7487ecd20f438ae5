"""Self-attention at the sizes that take a kernel or a branch of their own: long rows in bfloat16 past 64 columns, few queries and divided keys in
float32 past 128, masks whose tail spans several scans, the second plane of dS."""
import pytest
import torch

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
