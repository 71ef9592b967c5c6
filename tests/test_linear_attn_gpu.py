"""Linear attention with a decay per head on the GPU against the step recurrence in 64 bits.

Tolerances, element by element, from the roundings made.  A(.) is the same sum over absolute values.
fp32: every sum has at most L + dk + dv terms of relative error 2^-24 each, and a decay power adds a few:
(L + dk + dv + 32) 2^-24 A.  bf16: the output is rounded once (2^-8 |o|) and each of its two products has
one operand rounded to bf16 (the weighted scores, the carried state: 2^-8 A); the state's key or value rows
are split into two bf16 parts (2^-16 A).  Besides, the norm of the error of a bf16 output is held to 2^-8 of
the output's norm: two independent roundings of at most 2^-8 each, with a root mean square of 0.43 2^-8.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")
    from hybrid_model_mamba_xlstm_b200 import kernels
    return kernels


def recur(q, k, v, ld, scale, lengths=None, s0=None):
    """(o, last state) of the step recurrence in float64."""
    q, k, v = q.double(), k.double(), v.double()
    B, L, H, dk = q.shape
    S = torch.zeros(B, H, dk, v.shape[-1], device=q.device, dtype=torch.float64) if s0 is None else s0.double()
    g = ld.double().exp().view(1, H, 1, 1)
    n = torch.full((B,), L, device=q.device) if lengths is None else lengths
    o = []
    for t in range(L):
        on = (t < n).view(B, 1, 1, 1)
        kt, vt, qt = (torch.where(on[..., 0], x[:, t], torch.zeros_like(x[:, t])) for x in (k, v, q))
        S = torch.where(on, g * S + kt[..., None] * vt[..., None, :], S)
        o.append(scale * torch.matmul(qt[..., None, :], S)[..., 0, :])
    return (torch.stack(o, 1) if o else torch.zeros_like(v)), S


def inputs(B, L, H, dk, dv, dtype, seed=0, s0=False, ld=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    q, k, v = r(B, L, H, dk).to(dtype), r(B, L, H, dk).to(dtype), r(B, L, H, dv).to(dtype)
    if ld is None:
        ld = torch.log1p(-torch.exp2(-torch.linspace(1.0, 9.0, H, device="cuda")))
    return q, k, v, ld, (r(B, H, dk, dv) if s0 else None)


def close(got, ref, A, dtype, terms):
    err = (got.double() - ref).abs()
    unit = (terms + 32) * 2.0 ** -24
    tol = unit * A if dtype == F32 else 2.0 ** -8 * (ref.abs() + A) + unit * A
    assert bool((err <= tol + 1e-30).all()), float((err - tol).max())
    if dtype == BF and float(ref.norm()) > 0:
        assert float(err.norm() / ref.norm()) <= 2.0 ** -8


def check_forward(ops, q, k, v, ld, s0, scale, lengths=None):
    B, L, H, dk = q.shape
    dv = v.shape[-1]
    o, sT = ops.linear_attention(q, k, v, ld, scale=scale, lengths=lengths, initial_state=s0, return_final_state=True)
    assert o.dtype == q.dtype and o.shape == v.shape and sT.dtype == F32 and sT.shape == (B, H, dk, dv)
    ref, rS = recur(q, k, v, ld, scale, lengths, s0)
    Ao, AS = recur(q.abs(), k.abs(), v.abs(), ld, abs(scale), lengths, None if s0 is None else s0.abs())
    close(o, ref, Ao, q.dtype, L + dk + dv)
    tol = ((L + dk + dv + 32) * 2.0 ** -24 + (2.0 ** -16 if q.dtype == BF else 0)) * AS
    assert bool(((sT.double() - rS).abs() <= tol + 1e-30).all()), float(((sT.double() - rS).abs() - tol).max())
    return o, sT


# tensor-core shapes (bf16, multiples of 8, dk up to 256) at chunk and tile edges, and the others
SHAPES = [(2, 1, 2, 64, 64), (1, 2, 1, 8, 8), (2, 127, 2, 64, 32), (1, 128, 3, 128, 128), (2, 129, 2, 128, 64),
          (1, 255, 2, 96, 160), (1, 257, 2, 136, 72), (2, 300, 2, 256, 200), (1, 640, 1, 248, 64), (3, 65, 2, 40, 264),
          (1, 33, 2, 7, 5), (1, 70, 2, 33, 129), (1, 40, 1, 300, 20), (1, 40, 1, 512, 36)]


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(ops, shape, dtype):
    B, L, H, dk, dv = shape
    q, k, v, ld, s0 = inputs(B, L, H, dk, dv, dtype, seed=L, s0=L % 2 == 1)
    check_forward(ops, q, k, v, ld, s0, dk ** -0.5)


@pytest.mark.parametrize("dims", [(1, 2048, 40, 128, 128), (5, 1100, 32, 128, 128), (3, 900, 30, 64, 64), (2, 700, 40, 192, 128)])
def test_many_heads_and_chunks(ops, dims):
    """bf16 grids of more CTAs than the GPU has SMs, and many chunks per CTA, with a state on both sides."""
    B, L, H, dk, dv = dims
    q, k, v, ld, s0 = inputs(B, L, H, dk, dv, BF, seed=H, s0=True)
    check_forward(ops, q, k, v, ld, s0, dk ** -0.5)


@pytest.mark.parametrize("dtype,dk", [(F32, 64), (BF, 64), (BF, 192), (BF, 20)])
def test_lengths_and_what_lies_behind_them(ops, dtype, dk):
    """Rows of length 0, 1, a chunk's edge and all; NaN and infinity behind each row's end change nothing, and
    the output there is zero.  Lengths outside [0, L] count as its ends."""
    B, L, H, dv = 7, 300, 2, 72
    q, k, v, ld, s0 = inputs(B, L, H, dk, dv, dtype, seed=5, s0=True)
    lengths = torch.tensor([0, 1, 128, 129, 300, 400, -3], device="cuda", dtype=torch.int32)
    n = lengths.clamp(0, L)
    o, sT = check_forward(ops, q, k, v, ld, s0, 0.3, n)
    behind = torch.arange(L, device="cuda")[None, :] >= n[:, None]
    bad = [x.clone() for x in (q, k, v)]
    for x, value in zip(bad, (float("nan"), float("inf"), float("nan"))):
        x[behind] = value
    o2, sT2 = ops.linear_attention(*bad, ld, scale=0.3, lengths=lengths, initial_state=s0, return_final_state=True)
    assert torch.equal(o, o2) and torch.equal(sT, sT2)
    assert float(o2[behind].abs().max()) == 0
    assert torch.equal(sT2[0], s0[0])
    o3 = ops.linear_attention(*bad, ld, scale=0.3, lengths=lengths.long(), initial_state=s0)
    assert torch.equal(o, o3)


@pytest.mark.parametrize("dtype,dims", [(BF, (64, 64)), (F32, (32, 32)), (BF, (160, 48))])
def test_time_segments(ops, dtype, dims):
    """One head and a long sequence: the call is cut along time; lengths that end in an early segment."""
    B, L, H = 2, 2500, 1
    q, k, v, ld, s0 = inputs(B, L, H, *dims, dtype, seed=7, s0=True, ld=torch.tensor([-0.002], device="cuda"))
    check_forward(ops, q, k, v, ld, s0, 0.2)
    check_forward(ops, q, k, v, ld, s0, 0.2, torch.tensor([700, 2400], device="cuda"))


@pytest.mark.parametrize("dtype", [F32, BF])
def test_decays(ops, dtype):
    """No memory at all (-inf), a decay that underflows inside a chunk, no decay (0), and one near it."""
    ld = torch.tensor([-math.inf, -30.0, -1.0, -1e-5, 0.0], device="cuda")
    q, k, v, ld, s0 = inputs(2, 200, 5, 64, 64, dtype, seed=3, s0=True, ld=ld)
    check_forward(ops, q, k, v, ld, s0, 0.125)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_strides(ops, dtype):
    """Column blocks of one projection, head-major memory, rows that are not 16-byte aligned, a last dim that is
    not dense, heads shared by a zero stride, and a strided, non-fp32 initial state."""
    B, L, H, d = 2, 150, 2, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)
    ld = torch.tensor([-0.1, -0.01], device="cuda")
    qkv = r(B, L, 3 * H * d)
    q, k, v = (x.unflatten(-1, (H, d)) for x in qkv.chunk(3, -1))
    s0 = r(B, H, d, d).transpose(2, 3)
    check_forward(ops, q, k, v, ld, s0, 0.125)
    check_forward(ops, r(B, H, L, d).transpose(1, 2), r(L, B, H, d).transpose(0, 1), r(B, L, H, d + 8)[..., :d], ld, s0, 0.125)
    odd = r(B * L * H * d + 1)[1:].view(B, L, H, d)
    check_forward(ops, odd, r(B, L, H, 2 * d)[..., ::2], r(B, L, 1, d).expand(B, L, H, d), ld, s0, 0.125)
    check_forward(ops, q, r(1, L, 1, d).expand(B, L, H, d), r(B, 1, H, d).expand(B, L, H, d), ld, s0, 0.125)


def test_empty(ops):
    """No rows, no steps, no heads: the state passes through, gradients come out empty or zero."""
    for dtype in (F32, BF):
        q, k, v, ld, s0 = inputs(2, 0, 3, 16, 16, dtype, s0=True)
        o, sT = ops.linear_attention(q, k, v, ld, initial_state=s0, return_final_state=True)
        assert o.shape == (2, 0, 3, 16) and torch.equal(sT, s0)
        o, sT = ops.linear_attention(q, k, v, ld, return_final_state=True)
        assert float(sT.abs().max()) == 0
        dq, dk, dv, ds = ops.linear_attention_bwd(q, k, v, ld, v, initial_state=s0, d_final_state=s0, scale=0.5)
        assert dq.numel() == 0 and torch.allclose(ds, s0, rtol=2.0 ** -22, atol=0)
        q, k, v, ld, s0 = inputs(0, 5, 3, 16, 16, dtype, s0=True)
        o, sT = ops.linear_attention(q, k, v, ld, initial_state=s0, return_final_state=True)
        assert o.shape == (0, 5, 3, 16) and sT.shape == (0, 3, 16, 16)


def grads_ref(q, k, v, ld, scale, lengths, s0, do, dS):
    """The formula's gradients in float64: autograd through the step recurrence."""
    leaves = [x.detach().double().requires_grad_() for x in (q, k, v)] + ([s0.detach().double().requires_grad_()] if s0 is not None else [])
    o, S = recur(*leaves[:3], ld, scale, lengths, leaves[3] if s0 is not None else None)
    loss = (o * do.double()).sum() + ((S * dS.double()).sum() if dS is not None else 0)
    return torch.autograd.grad(loss, leaves)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("shape", [(2, 1, 2, 64, 64), (1, 200, 2, 128, 64), (2, 130, 2, 96, 160), (1, 257, 1, 64, 256),
                                   (1, 50, 2, 20, 12), (1, 36, 1, 7, 9), (2, 1300, 1, 64, 64)])
def test_gradients(ops, shape, dtype):
    """All gradients, with a state on both sides and padded rows; and without any of them."""
    B, L, H, dk, dv = shape
    q, k, v, ld, s0 = inputs(B, L, H, dk, dv, dtype, seed=L + dk, s0=True,
                             ld=torch.log1p(-torch.exp2(-torch.linspace(3.0, 8.0, H, device="cuda"))))
    g = torch.Generator(device="cuda").manual_seed(9)
    do = torch.randn(B, L, H, dv, generator=g, device="cuda").to(dtype)
    dS = torch.randn(B, H, dk, dv, generator=g, device="cuda")
    lengths = torch.tensor([max(1, L - 7)] + [L] * (B - 1), device="cuda")
    scale = 0.2
    for n, s, e in ((lengths, s0, dS), (None, None, None)):
        leaves = [x.clone().requires_grad_() for x in (q, k, v)] + ([s.clone().requires_grad_()] if s is not None else [])
        o, sT = ops.linear_attention(*leaves[:3], ld, scale=scale, lengths=n, initial_state=leaves[3] if s is not None else None,
                                     return_final_state=True)
        loss_outs, loss_grads = ([o, sT], [do, e]) if e is not None else ([o], [do])
        got = torch.autograd.grad(loss_outs, leaves, loss_grads)
        ref = grads_ref(q, k, v, ld, scale, n, s, do, e)
        A = grads_ref(q.abs(), k.abs(), v.abs(), ld, scale, n, None if s is None else s.abs(), do.abs(), None if e is None else e.abs())
        for i, (a, b, c) in enumerate(zip(got, ref, A)):
            if i < 3:
                close(a, b, c, dtype, L + dk + dv)
            else:
                tol = ((L + dk + dv + 32) * 2.0 ** -24 + (2.0 ** -16 if dtype == BF else 0)) * c
                assert bool(((a.double() - b).abs() <= tol).all())


def test_gradients_against_differences(ops):
    """fp32: <gradient, direction> against the central difference of the 64-bit recurrence.  The function is
    cubic along a line, so with h = 1e-3 the difference is off by h^2 times a third derivative of the
    function's own size: 1e-5 relative to the sum of absolute values, which dwarfs the kernel's roundings."""
    q, k, v, ld, s0 = inputs(2, 70, 2, 24, 16, F32, seed=2, s0=True)
    g = torch.Generator(device="cuda").manual_seed(4)
    do = torch.randn(2, 70, 2, 16, generator=g, device="cuda")
    dS = torch.randn(2, 2, 24, 16, generator=g, device="cuda")
    leaves = [x.clone().requires_grad_() for x in (q, k, v, s0)]
    o, sT = ops.linear_attention(*leaves[:3], ld, initial_state=leaves[3], return_final_state=True, scale=0.2)
    got = torch.autograd.grad([o, sT], leaves, [do, dS])
    base = [x.double() for x in (q, k, v, s0)]

    def f(xs):
        o, S = recur(*xs[:3], ld, 0.2, None, xs[3])
        return float((o * do.double()).sum() + (S * dS.double()).sum())

    for i in range(4):
        d = torch.randn(base[i].shape, generator=g, device="cuda").double()
        h = 1e-3
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + h * d, base[i] - h * d
        diff = (f(up) - f(down)) / (2 * h)
        mine = float((got[i].double() * d).sum())
        assert abs(mine - diff) <= 1e-5 * float((got[i].double() * d).abs().sum())


@pytest.mark.parametrize("dtype", [F32, BF])
def test_shared_heads_get_the_sum(ops, dtype):
    """k, v expanded over the heads and v over the batch: the gradient of the shared tensor is the sum over its
    users, each rounded to the dtype once before torch sums them (in fp32 or above)."""
    B, L, H, d = 2, 100, 4, 32
    q, _, _, ld, _ = inputs(B, L, H, d, d, dtype, seed=8)
    g = torch.Generator(device="cuda").manual_seed(3)
    k1 = torch.randn(B, L, 1, d, generator=g, device="cuda").to(dtype).requires_grad_()
    v1 = torch.randn(1, L, 1, d, generator=g, device="cuda").to(dtype).requires_grad_()
    do = torch.randn(B, L, H, d, generator=g, device="cuda").to(dtype)
    o = ops.linear_attention(q, k1.expand(B, L, H, d), v1.expand(B, L, H, d), ld)
    gk, gv = torch.autograd.grad(o, (k1, v1), do)
    full = [x.detach().expand(B, L, H, d).contiguous() for x in (k1, v1)]
    _, rk, rv = grads_ref(q, *full, ld, d ** -0.5, None, None, do, None)
    tol = 3 * 2.0 ** -8 if dtype == BF else 1e-5
    assert gk.shape == k1.shape and gv.shape == v1.shape
    assert float((gk.double() - rk.sum(2, keepdim=True)).norm() / rk.sum(2).norm()) <= tol
    assert float((gv.double() - rv.sum((0, 2), keepdim=True)).norm() / rv.sum((0, 2)).norm()) <= tol


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (7, 5), (33, 130), (512, 36), (1, 1), (48, 200)])
def test_step(ops, dtype, dk, dv):
    """Steps one after another against the recurrence: the state has one fused multiply-add per step (2^-23 of the
    sum of absolute values each, and 2^-24 for the decay), the output a sum over dk and one rounding."""
    B, H, L = 3, 2, 5
    q, k, v, ld, s0 = inputs(B, L, H, dk, dv, dtype, seed=dk, s0=True)
    state = s0.clone()
    ref, rS = recur(q, k, v, ld, 0.4, None, s0)
    A, AS = recur(q.abs(), k.abs(), v.abs(), ld, 0.4, None, s0.abs())
    for t in range(L):
        o = ops.linear_attention_step(q[:, t], k[:, t], v[:, t], ld, state, scale=0.4)
        tol = (dk + 32) * 2.0 ** -24 * A[:, t] + (2.0 ** -8 * ref[:, t].abs() if dtype == BF else 0)
        assert bool(((o.double() - ref[:, t]).abs() <= tol).all())
    assert bool(((state.double() - rS).abs() <= 4 * L * 2.0 ** -24 * AS).all())


def test_step_in_a_pool(ops):
    """A strided state (a slice of a larger pool), `out` given, no memory (-inf): rows outside stay as they were."""
    pool = torch.randn(5, 3, 2, 16, 24, device="cuda")
    before = pool.clone()
    state = pool[1:4, 2]
    q, k, v, _, _ = inputs(3, 1, 2, 16, 20, F32, seed=1)
    ld = torch.tensor([-math.inf, -0.5], device="cuda")
    out = torch.full((3, 2, 40), 7.0, device="cuda")
    view = state[..., 4:]
    want, wS = recur(q, k, v, ld, 0.25, None, view.clone())
    got = ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, view, out=out[..., :20], scale=0.25)
    assert got.data_ptr() == out.data_ptr()
    assert float((got.double() - want[:, 0]).abs().max()) < 1e-5 and float((view.double() - wS).abs().max()) < 1e-5
    assert bool((out[..., 20:] == 7).all())
    before[1:4, 2, :, :, 4:] = pool[1:4, 2, :, :, 4:]
    assert torch.equal(before, pool)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_prompt_in_pieces_then_steps(ops, dtype):
    """A sequence in two calls and single steps equals the recurrence over the whole of it."""
    B, L, H, d = 2, 201, 2, 64
    q, k, v, ld, s0 = inputs(B, L, H, d, d, dtype, seed=6, s0=True)
    ref, rS = recur(q, k, v, ld, 0.125, None, s0)
    A, _ = recur(q.abs(), k.abs(), v.abs(), ld, 0.125, None, s0.abs())
    o1, S = ops.linear_attention(q[:, :130], k[:, :130], v[:, :130], ld, initial_state=s0, return_final_state=True)
    o2, S = ops.linear_attention(q[:, 130:196], k[:, 130:196], v[:, 130:196], ld, initial_state=S, return_final_state=True)
    steps = [ops.linear_attention_step(q[:, t], k[:, t], v[:, t], ld, S) for t in range(196, L)]
    close(torch.cat([o1, o2, torch.stack(steps, 1)], 1), ref, A, dtype, L + 2 * d)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_streams_graphs_and_repeats(ops, dtype):
    """The same bits on a side stream, from two graphs replayed one after the other and at once, and on repeats."""
    args = [inputs(2, 1500, 1, 64, 64, dtype, seed=s, s0=True) for s in (1, 2)]
    call = lambda a: ops.linear_attention(a[0], a[1], a[2], a[3], initial_state=a[4], return_final_state=True)
    want = [call(a) for a in args]
    for a, w in zip(args, want):
        assert all(torch.equal(x, y) for x, y in zip(call(a), w))
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s, a in zip(side, args):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(call(a))
    torch.cuda.synchronize()
    for x, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(x, w))
    graphs, outs = [], []
    for a in args:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(a))
        graphs.append(g)
    for o in outs:
        for t in o:
            t.zero_()
    for s, g in zip(side, graphs):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            g.replay()
            g.replay()
    torch.cuda.synchronize()
    for x, w in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(x, w))


@pytest.mark.parametrize("dtype", [F32, BF])
def test_captured_training_step(ops, dtype):
    """Forward and gradients captured into a graph while an eager graph of the same data lives: through autograd with
    leaves of their own (torch ties a leaf's gradient node to the stream of the graph it was first part of, and
    refuses to capture it from another one), and through linear_attention_bwd with the very same tensors."""
    q, k, v, ld, s0 = inputs(2, 200, 2, 64, 64, dtype, seed=4, s0=True)
    eager = [x.requires_grad_() for x in (q, k, v, s0)]
    fresh = [x.detach().requires_grad_() for x in eager]

    def step(leaves):
        o, sT = ops.linear_attention(*leaves[:3], ld, initial_state=leaves[3], return_final_state=True)
        return o, torch.autograd.grad([o, sT], leaves, [torch.ones_like(o), torch.ones_like(sT)])

    want = step(eager)[1]
    o, sT = ops.linear_attention(*eager[:3], ld, initial_state=eager[3], return_final_state=True)  # lives through both captures
    ones = torch.ones_like(o), torch.ones_like(sT)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        got1 = step(fresh)[1]
    with torch.cuda.graph(g2):
        got2 = ops.linear_attention_bwd(*eager[:3], ld, ones[0], initial_state=eager[3], d_final_state=ones[1])
    for t in got1 + got2:
        t.zero_()
    g1.replay()
    g2.replay()
    torch.cuda.synchronize()
    late = torch.autograd.grad([o, sT], eager, ones)
    for a, b, c, d in zip(want, got1, got2, late):
        assert torch.equal(a, b) and torch.equal(a, c) and torch.equal(a, d)


@pytest.mark.parametrize("dtype,dims", [(F32, (64, 64)), (BF, (64, 72)), (BF, (128, 128)), (BF, (192, 40)), (BF, (20, 12)), (F32, (300, 33))])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_that_are_not_finite_stay_where_they_belong(ops, dtype, dims, bad):
    """One element of q (row 0), of k (row 1), of v (row 2) or of dout (row 3) that is not finite, in the middle of a chunk:
    the recurrence in 64 bits says which outputs, states and gradients are not finite then, and all others keep the
    bits that they have without it (its tile-mates before it, the other columns, heads and rows among them).  Decays that
    keep and that forget within a chunk; one long head, cut along time, too."""
    for L, H, ld in ((300, 3, [-0.01, -0.6, -math.inf]), (1100, 1, [-0.02])):
        q, k, v, ld, s0 = inputs(5, L, H, *dims, dtype, seed=dims[0], s0=True, ld=torch.tensor(ld, device="cuda"))
        g = torch.Generator(device="cuda").manual_seed(2)
        do, dS = torch.randn(v.shape, generator=g, device="cuda").to(dtype), torch.randn(s0.shape, generator=g, device="cuda")
        run = lambda q, k, v, do: (*ops.linear_attention(q, k, v, ld, initial_state=s0, scale=0.2, return_final_state=True),
                                   *ops.linear_attention_bwd(q, k, v, ld, do, initial_state=s0, d_final_state=dS, scale=0.2))
        clean = run(q, k, v, do)
        x = [t.clone() for t in (q, k, v, do)]
        for i in range(4):
            x[i][i, 200, 0, 3] = bad
        got = run(*x)
        ref = (*recur(*x[:3], ld, 0.2, None, s0), *grads_ref(*x[:3], ld, 0.2, None, s0, x[3], dS))
        for i, (a, c, r) in enumerate(zip(got, clean, ref)):
            fine = torch.isfinite(r)
            assert torch.equal(torch.where(fine, a, 0), torch.where(fine, c, 0)), i
            assert not bool((torch.isfinite(a) & ~fine).any()), i


@pytest.mark.parametrize("dtype,dims", [(F32, (64, 64)), (BF, (64, 72)), (BF, (192, 40)), (BF, (20, 12))])
def test_an_infinite_value_leaves_infinite_states(ops, dtype, dims):
    """The state that an infinite v reaches holds infinities of k's signs, as in the recurrence, not NaN."""
    q, k, v, ld, s0 = inputs(1, 300, 2, *dims, dtype, seed=4, s0=True, ld=torch.tensor([-0.01, -0.6], device="cuda"))
    v[0, 200, :, 3] = torch.tensor([float("inf"), -float("inf")], device="cuda")
    _, sT = ops.linear_attention(q, k, v, ld, initial_state=s0, return_final_state=True)
    _, ref = recur(q, k, v, ld, 1.0, None, s0)
    assert torch.equal(sT[..., 3].double(), ref[..., 3]) and bool(torch.isinf(ref[..., 3]).all())
    keep = [c for c in range(dims[1]) if c != 3]
    assert bool(torch.isfinite(sT[..., keep]).all())


def test_rows_behind_the_lengths_of_a_very_long_batch(ops):
    """2^25 rows behind the length, of 75 heads (no cut along time), one value column each: 64 columns a block times the
    rows pass 32 bits.  All of them are zero, and the counted rows are those of a short call."""
    L, H, n = 2 ** 25 + 70, 75, 5
    for dtype in (BF, F32):
        q, k, v, ld, _ = inputs(1, n, H, 1, 1, dtype, seed=1)
        long = [x[:, :1].expand(1, L, H, 1) for x in (q, k, v)]  # a zero stride: no memory of that length
        o = ops.linear_attention(*long, ld, lengths=torch.tensor([n], device="cuda"), scale=1.0)
        want = ops.linear_attention(*(x[:, :1].expand(1, n, H, 1).contiguous() for x in (q, k, v)), ld, scale=1.0)
        assert torch.equal(o[:, :n], want)
        assert int(torch.count_nonzero(o[:, n:])) == 0
        del o


@pytest.mark.parametrize("dims", [(1, 257, 2, 128, 64), (2, 300, 2, 64, 72), (1, 300, 1, 256, 64), (1, 2600, 1, 128, 64)])
def test_bf16_states_to_32_bits(ops, dims):
    """The last state and the first state's gradient of bf16 runs.  k is bf16 as it is, and a weighted v goes into the
    products in three bf16 parts, whose half steps leave at most 2^-8, 2^-16 and 2^-24 of it behind the first, the
    second and the third: two parts would leave some 2^-19 of the state's norm.  With three a term carries the roundings
    of its weight and of its product with v, the parts' rest, and the roundings of the factors of the chunks behind it
    that still count (two): 5 2^-24.  A chunk's sum is 8 steps of 16 terms for each of 3 parts, 24 additions in fp32
    whose errors are independent: sqrt(24) 2^-24 of the norm."""
    B, L, H, dk, dv = dims
    ld = torch.tensor([-0.03, -0.002], device="cuda")[-H:]  # (powers of 1/2 would leave v in one part)
    q, k, v, ld, s0 = inputs(B, L, H, dk, dv, BF, seed=L, s0=True, ld=ld)
    g = torch.Generator(device="cuda").manual_seed(7)
    do, dS = torch.randn(v.shape, generator=g, device="cuda").to(BF), torch.randn(s0.shape, generator=g, device="cuda")
    _, sT = ops.linear_attention(q, k, v, ld, initial_state=s0, scale=0.3, return_final_state=True)
    _, rS = recur(q, k, v, ld, 0.3, None, s0)
    ds = ops.linear_attention_bwd(q, k, v, ld, do, initial_state=s0, d_final_state=dS, scale=0.3)[3]
    rd = grads_ref(q, k, v, ld, 0.3, None, s0, do, dS)[3]
    for a, b in ((sT, rS), (ds, rd)):
        assert float((a.double() - b).norm() / b.norm()) <= (5 + 24 ** 0.5) * 2.0 ** -24


def test_repeats_with_values_behind_the_lengths(ops):
    """NaN and infinities behind the ends of rows of one, two and three chunks, many times over while other work keeps the
    clocks apart: the same bits as with zeros there."""
    lengths = torch.tensor([1, 127, 129, 130, 200, 257, 299], device="cuda")
    behind = torch.arange(300, device="cuda")[None, :] >= lengths[:, None]
    other = torch.randn(2048, 2048, device="cuda")
    for dk in (64, 192):
        q, k, v, ld, s0 = inputs(7, 300, 2, dk, 72, BF, seed=6, s0=True)
        zeros, bad = [x.clone() for x in (q, k, v)], [x.clone() for x in (q, k, v)]
        for x, y, value in zip(zeros, bad, (float("nan"), float("inf"), float("nan"))):
            x[behind], y[behind] = 0, value
        call = lambda x: (*ops.linear_attention(*x, ld, lengths=lengths, initial_state=s0, return_final_state=True),
                          *ops.linear_attention_bwd(*x, ld, x[2], lengths=lengths, initial_state=s0))
        want = call(zeros)
        for i in range(100):
            if i % 2:
                other @ other
            assert all(torch.equal(a, b) for a, b in zip(call(bad), want)), i
