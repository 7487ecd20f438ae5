"""Self-attention as it may be called: strides of every kind, other kinds of differentiation, gradients that are not there, lengths and positions
past what the kernels count in, rules made at the same time."""
import ctypes as C
import gc
import threading
import weakref

import pytest
import torch
from torch.autograd import forward_ad

from attention_ref import check, reference
from test_attention import BF16, F32, desc, normal
from wavernn_amd import _lib
from wavernn_amd import attention as A

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_over_dimensions_of_one(dtype):
    """What a stride over a single row or position says does not matter, in gradients as in inputs."""
    q, k, v = (normal(i, 1, 2, 5, 16, dtype=dtype).requires_grad_() for i in range(3))
    dout = normal(3, 1, 2, 5, 16, dtype=dtype)
    odd = dout.as_strided(dout.shape, (161, *dout.stride()[1:]))
    want, got = (torch.autograd.grad(A.attention(q, k, v), (q, k, v), d) for d in (dout, odd))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    q1 = normal(0, 2, 2, 1, 16, dtype=dtype).requires_grad_()
    k, v = (normal(i, 2, 2, 5, 16, dtype=dtype).requires_grad_() for i in (1, 2))
    dout = normal(3, 2, 2, 1, 16, dtype=dtype)
    far = dout.as_strided(dout.shape, (*dout.stride()[:2], 1 << 23, 1))
    want, got = (torch.autograd.grad(A.attention(q1, k, v), (q1, k, v), d) for d in (dout, far))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_broadcast_batch_with_far_positions(dtype):
    """Inputs of one row for a large batch: their gradients' positions lie further apart than the kernels read rows, and are only written."""
    B, H, D = 4096, 4, 256
    q, k, v = (normal(i, 2, H, D, dtype=dtype).requires_grad_() for i in range(3))
    many = [x[None].expand(B, 2, H, D).permute(0, 2, 1, 3) for x in (q, k, v)]
    dout = normal(3, 1, H, 2, D, dtype=dtype)
    got = torch.autograd.grad(A.attention(*many), (q, k, v), dout.expand(B, H, 2, D))
    want = reference(*(x[:1] for x in many), dout)
    for name, g in zip(("dq", "dk", "dv"), got):
        value, bound = want[name]
        # autograd adds the rows' gradients up: B equal values, each addition half a step of the inputs' type or of 32 bits
        check(name, g.double().permute(1, 0, 2)[None] / B, (value, bound + (torch.finfo(dtype).eps + B * 2.0 ** -24) * value.abs()))


class NoGradient(torch.autograd.Function):
    """Passes no gradient on."""

    @staticmethod
    def forward(ctx, x):
        return x.clone()

    @staticmethod
    def backward(ctx, d):
        return None


@gpu
def test_no_gradient_of_the_output():
    q, k, v = (normal(i, 1, 2, 5, 16).requires_grad_() for i in range(3))
    out = NoGradient.apply(A.attention(q, k, v))
    (out.sum() + 2 * q.sum()).backward()
    assert bool((q.grad == 2).all()) and k.grad is None and v.grad is None
    q, k, v = (normal(i, 1, 2, 5, 16).requires_grad_() for i in range(3))
    table = normal(3, 16, 2).requires_grad_()
    (NoGradient.apply(A.relative_position_bias(table, 5, 5)).sum() + 2 * table.sum()).backward()
    assert bool((table.grad == 2).all())


def test_a_description_keeps_its_bucket_edges():
    """The edges whose address a description holds live as long as it, whatever other rules are made meanwhile (the cache holds some dozens)."""
    q = torch.zeros(1, 2, 4, 8)
    table = torch.zeros(14, 2)
    A._edges.cache_clear()
    desc = A._desc(q, q, q, table, None, None, None, False, 1.0, 77, True)
    edges = weakref.ref(A._edges(14, 77, True)[1])
    A._edges.cache_clear()
    gc.collect()
    assert edges() is not None and bytes(desc).endswith(C.addressof(edges()).to_bytes(8, "little"))
    del desc
    gc.collect()
    assert edges() is None


@pytest.mark.parametrize("q_len,k_len,start", [(4, 4, 1 << 32), (4, 4, -(1 << 32)), (4, 4, (1 << 29) + 1), (1 << 32, 0, 0), (0, (1 << 32) + 1, 0),
                                               ((1 << 28) + 1, 1, 0), (4, (1 << 28) + 1, None)])
def test_lengths_and_positions_past_the_kernels_count_are_refused(q_len, k_len, start):
    with pytest.raises(ValueError, match="2\\^"):
        A.relative_position_bias(torch.zeros(32, 2), q_len, k_len, q_start=start)



def test_c_entry_of_the_dense_bias_refuses_more_workgroups_than_a_launch_takes():
    lib = _lib.load()
    e = (C.c_int32 * 3)(8, 16, 32)
    for heads, q_len in ((1 << 22, 300), (1 << 25, 32)):
        assert lib.wrnn_relative_bias_forward(16, 0, heads, q_len, 1, 0, 8, 64, 0, e, 16, None) != 0 and b"too large" in lib.wrnn_last_error()
        size = lib.wrnn_relative_bias_workspace_bytes(heads, q_len, 1, 8, 64)
        assert lib.wrnn_relative_bias_backward(16, 0, heads, q_len, 1, 0, 8, 64, 0, e, 16, 16, size, None) != 0 and b"too large" in lib.wrnn_last_error()
    many = desc(heads=1 << 20, kv_heads=1 << 20, q_len=1, k_len=1, bias_table=16, num_buckets=256, max_distance=1024,
                bucket_edges=(C.c_int32 * 127)(*A.bucket_edges(256, 1024, False)))
    assert lib.wrnn_attention_forward(C.byref(many), 16, _lib.I64x3(0, 0, 0), None, None, 0, None) != 0 and b"too large" in lib.wrnn_last_error()


@gpu
def test_forward_mode_derivatives_and_transforms_are_refused():
    """An error, not a result without them."""
    q, k, v = (normal(i, 1, 2, 5, 16) for i in range(3))
    table = normal(3, 16, 2)
    with forward_ad.dual_level():
        for i in range(4):
            args = [q, k, v, table]
            args[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                    A.attention(*args[:3], bias_table=args[3])
        assert torch.isfinite(A.attention(q, k, v, bias_table=table)).all()     # no dual tensor among them
        with pytest.raises(RuntimeError):
            A.relative_position_bias(forward_ad.make_dual(table, torch.ones_like(table)), 5, 5)
    for transformed in (lambda: torch.func.jvp(lambda x: A.attention(x, k, v), (q,), (torch.ones_like(q),)),
                        lambda: torch.func.vmap(lambda x: A.attention(x, k, v))(q[None]), lambda: torch.func.grad(lambda x: A.attention(x, k, v).sum())(q)):
        with pytest.raises(RuntimeError):
            transformed()


def test_dual_tensors_are_seen():
    x = torch.ones(3)
    A._no_tangents(x, None)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, x)
        A._no_tangents(x, None)
        with pytest.raises(RuntimeError, match="forward-mode"):
            A._no_tangents(x, d)


@gpu
@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("D", [12, 13, 16])
def test_traces_compute_on_their_inputs(grad, D):
    k, v = normal(1, 1, 2, 5, D), normal(2, 1, 2, 5, D)
    table = normal(3, 16, 2)
    with torch.set_grad_enabled(grad):
        traced = torch.jit.trace(lambda x: A.attention(x, k, v, bias_table=table) * 2, (normal(0, 1, 2, 5, D).requires_grad_(grad),), check_trace=False)
        x = normal(4, 1, 2, 5, D)
        assert torch.equal(traced(x), A.attention(x, k, v, bias_table=table) * 2)


def test_copies_of_rows_are_in_the_kernels_form():
    """Whatever a tensor's strides and however few elements it has: what is not taken as it is comes back contiguous."""
    wide = torch.zeros(2, 5, 3, 19)
    for t in (wide[..., 1:17].permute(0, 2, 1, 3)[:, :, :0], wide[:, :1, :, 1:17].permute(0, 2, 1, 3), wide[:0, ..., 1:17], wide.flatten()[1:97].view(1, 2, 3, 16)):
        rows = A._rows(t)
        assert rows.shape == t.shape and torch.equal(rows, t)
        assert all(s % 4 == 0 for s, n in zip(rows.stride()[:3], rows.shape) if n != 1) and rows.stride(3) == 1 and rows.data_ptr() % 16 == 0


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_no_keys_in_a_slice_of_odd_rows(dtype):
    q = normal(0, 3, 16, 4, 99, dtype=dtype)[..., 1:97].permute(0, 2, 1, 3).requires_grad_()
    k = normal(1, 3, 16, 2, 99, dtype=dtype)[:, :0, :, 1:97].permute(0, 2, 1, 3)
    out = A.attention(q, k, k)
    assert not out.any() and not torch.autograd.grad(out, q, torch.ones_like(out))[0].any()


@pytest.mark.parametrize("D", [5, 6, 13, 16])
def test_padded_copies_of_rows_with_the_heads_innermost(D):
    """torch pads a tensor in the order in memory that it finds."""
    t = torch.randn(2, 3, 4, D).to(memory_format=torch.channels_last)
    rows = A._rows(t)
    assert rows.is_contiguous() and torch.equal(rows[..., :D], t) and not rows[..., D:].any()


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [5, 13, 16])
def test_heads_innermost(dtype, D):
    q, k, v, dout = (normal(i, 2, 3, 9, D, dtype=dtype) for i in range(4))
    inner = [x.to(memory_format=torch.channels_last).requires_grad_() for x in (q, k, v)]
    got = A.attention(*inner)
    want = A.attention(*(x.requires_grad_() for x in (q, k, v)))
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got, inner, dout.to(memory_format=torch.channels_last)), torch.autograd.grad(want, (q, k, v), dout)):
        assert torch.equal(a, b)


@gpu
def test_calls_from_several_threads_and_streams_at_once():
    """Each with a rule, sizes and a stream of its own: the bits of the calls one after the other."""
    def case(n):
        D, Tq, Tk = (16, 64, 100, 200)[n], (3, 70, 200, 40)[n], (900, 70, 300, 500)[n]
        leaves = [normal(10 * n + i, 2, 4, Tq if i == 0 else Tk, D, dtype=(F32, BF16)[n % 2]).requires_grad_() for i in range(3)]
        leaves.append(normal(10 * n + 3, 16, 4).requires_grad_())
        return leaves, normal(10 * n + 4, 2, 4, Tq, D, dtype=(F32, BF16)[n % 2])

    def step(leaves, dout, n, k):
        out = A.attention(*leaves[:3], bias_table=leaves[3], max_distance=40 + n + 4 * k)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]

    cases = [case(n) for n in range(4)]
    want = [[step(*c, n, k) for k in range(20)] for n, c in enumerate(cases)]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(n):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[n] = [step(*cases[n], n, k) for k in range(20)]
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(n,)) for n in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(got, want):
        for x, y in zip(a, b):
            assert all(torch.equal(u, v) for u, v in zip(x, y))
