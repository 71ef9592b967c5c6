"""Per-head norms of q and k with the position rotation on the GPU against the formula in 64 bits.

Tolerances: y has one rounding to its dtype (half a step: fp32 2^-24, bf16 2^-8, fp16 2^-11 relative) after fp32
arithmetic: the mean of d squares and its root (the squares' sum d 2^-24, halved by the root, and a few more),
three products, and cosines and sines off by 2^-22 (their 32-bit argument in turns is off by 2^-25 of a turn,
times 2 pi): (d / 2 + 40) 2^-24 of the pair's length.  Gradients have the same products twice.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32, F16 = torch.bfloat16, torch.float32, torch.float16


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")
    from hybrid_model_mamba_xlstm_b200 import kernels
    return kernels


def ref_one(x, w, pos, base, rot, inter, eps):
    x = x.double()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * (1.0 if w is None else w.double())
    if rot == 0:
        return y
    half = rot // 2
    f = base ** (-2.0 * torch.arange(half, device=x.device, dtype=torch.float64) / rot)
    ang = (pos.double()[..., None] * f)[..., None, :]
    if ang.dim() == 3:
        ang = ang[None]
    c, s = ang.cos(), ang.sin()
    a = y[..., :rot]
    x0, x1 = (a[..., 0::2], a[..., 1::2]) if inter else (a[..., :half], a[..., half:])
    r0, r1 = x0 * c - x1 * s, x0 * s + x1 * c
    r = torch.stack([r0, r1], -1).flatten(-2) if inter else torch.cat([r0, r1], -1)
    return torch.cat([r, y[..., rot:]], -1)


def bound(x, w, dtype):
    """Per element: half a step of the value is added by the caller; this is the fp32 part."""
    d = x.shape[-1]
    x = x.double()
    n = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-12)
    big = (n * (1.0 if w is None else w.double())).abs().amax(-1, keepdim=True) * 2
    return (d / 2 + 40) * 2.0 ** -24 * big


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make(B, L, hq, hk, d, dtype, seed=0, weights=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    w = (1 + 0.2 * r(d), 1 + 0.2 * r(d)) if weights else (None, None)
    return (2 * r(B, L, hq, d)).to(dtype), (2 * r(B, L, hk, d)).to(dtype), *w


CASES = [(2, 5, 4, 2, 128, 128, False), (2, 5, 4, 2, 128, 128, True), (1, 1, 1, 1, 64, 64, False), (3, 7, 3, 1, 64, 32, True),
         (1, 9, 2, 2, 96, 96, False), (1, 9, 2, 2, 80, 48, False), (2, 3, 5, 1, 256, 256, False), (2, 3, 2, 2, 512, 512, False),
         (1, 4, 2, 2, 512, 100, True), (1, 4, 2, 3, 1024, 1024, False), (1, 6, 2, 2, 37, 36, False), (1, 6, 2, 2, 37, 36, True),
         (1, 6, 2, 2, 1, 0, False), (2, 6, 1, 1, 40, 12, False), (1, 33, 1, 0, 32, 32, False), (40, 60, 2, 1, 64, 64, False)]


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("case", CASES)
def test_forward(ops, case, dtype):
    B, L, hq, hk, d, rot, inter = case
    q, k, wq, wk = make(B, L, hq, hk, d, dtype, seed=d)
    pos = torch.randint(0, 4000, (B, L), device="cuda")
    got = ops.qk_norm_rope(q, k, wq, wk, pos, rotary_dim=rot, interleaved=inter)
    for x, w, y in ((q, wq, got[0]), (k, wk, got[1])):
        assert y.dtype == dtype and y.shape == x.shape
        ref = ref_one(x, w, pos, 10000.0, rot, inter, 1e-6)
        tol = half_step(dtype) * ref.abs() + bound(x, w, dtype) + (2.0 ** -25 if dtype == F16 else 0)
        assert bool(((y.double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [F32, BF])
def test_far_positions(ops, dtype):
    """Angles stay right up to position 2^31, where a 32-bit product would be off by whole turns (the 64-bit
    turns are off by 2^31 2^-53, below the bound)."""
    q, k, wq, wk = make(1, 6, 2, 1, 64, dtype)
    pos = torch.tensor([0, 1, 10 ** 6, 2 ** 24 + 1, 2 ** 31 - 1, 2 ** 31], device="cuda")
    got = ops.qk_norm_rope(q, k, wq, wk, pos, rope_base=5e5)
    ref = ref_one(q, wq, pos, 5e5, 64, False, 1e-6)
    assert bool(((got[0].double() - ref).abs() <= half_step(dtype) * ref.abs() + 2 * bound(q, wq, dtype)).all())


def test_positions_forms_and_no_rotation(ops):
    """(L,), (B, L), int32 and broadcast positions agree; no positions: the plain norm; no weights: ones."""
    q, k, wq, wk = make(3, 5, 2, 2, 64, F32)
    p = torch.arange(5, device="cuda") + 17
    want = ops.qk_norm_rope(q, k, wq, wk, p)
    for pos in (p.int(), p.expand(3, 5), p.expand(3, 5).contiguous(), torch.stack([p, p], 1)[:, 0]):
        assert all(torch.equal(a, b) for a, b in zip(want, ops.qk_norm_rope(q, k, wq, wk, pos)))
    a, b = ops.qk_norm_rope(q, k, None, wk)
    for y, x, w in ((a, q, None), (b, k, wk)):
        assert bool(((y.double() - ref_one(x, w, None, 1, 0, False, 1e-6)).abs() <= bound(x, w, F32)).all())


@pytest.mark.parametrize("dtype", [F32, BF])
def test_strides_and_empty(ops, dtype):
    """Column blocks of a projection, head-major memory, rows off 16-byte alignment, a dilated last dim, a
    repeated head; and no tokens or heads."""
    g = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)
    B, L, d = 2, 6, 64
    pos = torch.arange(L, device="cuda")
    w = torch.ones(d, device="cuda")
    block = r(B, L, 5 * d)
    pairs = [(block[..., :3 * d].unflatten(-1, (3, d)), block[..., 3 * d:].unflatten(-1, (2, d))),
             (r(B, 3, L, d).transpose(1, 2), r(L, B, 2, d).transpose(0, 1)),
             (r(B * L * 3 * d + 1)[1:].view(B, L, 3, d), r(B, L, 2, 2 * d)[..., ::2]),
             (r(B, L, 1, d).expand(B, L, 3, d), r(1, L, 2, d).expand(B, L, 2, d))]
    for q, k in pairs:
        for x, y in zip((q, k), ops.qk_norm_rope(q, k, w, w, pos)):
            ref = ref_one(x, w, pos, 10000.0, d, False, 1e-6)
            assert bool(((y.double() - ref).abs() <= half_step(dtype) * ref.abs() + bound(x, w, dtype)).all())
    for shape in ((0, 4), (4, 0)):
        a, b = ops.qk_norm_rope(r(*shape, 2, d), r(*shape, 1, d), w, w, torch.zeros(*shape, device="cuda", dtype=torch.long))
        assert a.shape == (*shape, 2, d) and b.shape == (*shape, 1, d)


def test_zero_rows(ops):
    """A row of zeros gives zeros and, through eps, finite gradients."""
    q, k, wq, wk = make(1, 4, 2, 1, 64, F32)
    q[:, 1] = 0
    q.requires_grad_()
    a, b = ops.qk_norm_rope(q, k, wq, wk, torch.arange(4, device="cuda"))
    assert float(a[:, 1].abs().max()) == 0
    (g,) = torch.autograd.grad(a, q, torch.ones_like(a))
    assert bool(torch.isfinite(g).all())


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("case", CASES)
def test_gradients(ops, case, dtype):
    B, L, hq, hk, d, rot, inter = case
    q, k, wq, wk = make(B, L, hq, hk, d, dtype, seed=d + 1)
    g = torch.Generator(device="cuda").manual_seed(3)
    gq = torch.randn(q.shape, generator=g, device="cuda").to(dtype)
    gk = torch.randn(k.shape, generator=g, device="cuda").to(dtype)
    pos = torch.randint(0, 4000, (B, L), device="cuda")
    leaves = [x.clone().requires_grad_() for x in (q, k, wq, wk)]
    y = ops.qk_norm_rope(*leaves, pos, rotary_dim=rot, interleaved=inter)
    got = torch.autograd.grad(y, leaves, (gq, gk))
    rows = B * L * max(hq, hk, 1)
    for x, w, gy, gx, gw in ((q, wq, gq, got[0], got[2]), (k, wk, gk, got[1], got[3])):
        lx, lw = x.double().requires_grad_(), w.double().requires_grad_()
        out = ref_one(lx, lw, pos, 10000.0, rot, inter, 1e-6)
        rx, rw = torch.autograd.grad(out, (lx, lw), gy.double())
        assert gx.dtype == dtype and gw.dtype == w.dtype
        inv = 1 / torch.sqrt((x.double() ** 2).mean(-1, keepdim=True) + 1e-6)
        n = x.double() * inv
        size = 2 * inv * (gy.double().abs().amax(-1, keepdim=True) * 1.5 * w.abs().max() * (2 + n.abs() * n.abs().mean(-1, keepdim=True)))
        tol = half_step(dtype) * rx.abs() + (d + 80) * 2.0 ** -24 * size + (2.0 ** -25 if dtype == F16 else 0)
        assert bool(((gx.double() - rx).abs() <= tol).all())
        # the sum over rows: each term off by the row's (d / 2 + 40) 2^-24, and at most `rows` additions
        sizes = (gy.double().abs().amax(-1, keepdim=True) * 1.5 * n.abs()).flatten(0, 2).sum(0)
        assert bool(((gw.double() - rw).abs() <= (d / 2 + 40 + rows) * 2.0 ** -24 * sizes + 1e-30).all())


def test_gradients_against_differences(ops):
    """fp32 gradients against central differences of the 64-bit formula (step 1e-4: off by about 1e-8)."""
    q, k, wq, wk = make(2, 3, 2, 1, 64, F32, seed=5)
    pos = torch.randint(0, 100, (2, 3), device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    gq, gk = torch.randn(q.shape, generator=g, device="cuda"), torch.randn(k.shape, generator=g, device="cuda")
    leaves = [x.clone().requires_grad_() for x in (q, k, wq, wk)]
    got = torch.autograd.grad(ops.qk_norm_rope(*leaves, pos), leaves, (gq, gk))
    base = [x.double() for x in (q, k, wq, wk)]

    def f(xs):
        return float((ref_one(xs[0], xs[2], pos, 10000.0, 64, False, 1e-6) * gq).sum() +
                     (ref_one(xs[1], xs[3], pos, 10000.0, 64, False, 1e-6) * gk).sum())

    for i in range(4):
        d = torch.randn(base[i].shape, generator=g, device="cuda").double()
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + 1e-4 * d, base[i] - 1e-4 * d
        diff, mine = (f(up) - f(down)) / 2e-4, float((got[i].double() * d).sum())
        assert abs(mine - diff) <= 1e-5 * float((got[i].double() * d).abs().sum())


def test_repeats_streams_graph(ops):
    """Same bits on repeats (weight gradients too), on a side stream, and from a captured forward and backward (with
    leaves of their own, as torch wants it) while an eager graph of the same data lives."""
    q, k, wq, wk = make(4, 100, 4, 2, 128, BF)
    pos = torch.arange(100, device="cuda")
    leaves = [x.requires_grad_() for x in (q, k, wq, wk)]
    fresh = [x.detach().requires_grad_() for x in leaves]

    def step(leaves):
        y = ops.qk_norm_rope(*leaves, pos)
        return y, torch.autograd.grad(y, leaves, [torch.ones_like(t) for t in y])

    want = step(leaves)[1]
    again = step(leaves)[1]
    alive = ops.qk_norm_rope(*leaves, pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        third = step(fresh)[1]
    torch.cuda.synchronize()
    for other in (again, third):
        assert all(torch.equal(a, b) for a, b in zip(want, other))
    fresh = [x.detach().requires_grad_() for x in leaves]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        _, got = step(fresh)
    for t in got:
        t.zero_()
    g.replay()
    torch.cuda.synchronize()
    late = torch.autograd.grad(alive, leaves, [torch.ones_like(t) for t in alive])
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, got, late))


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("case", [(1, 5, 4, 3, 128, 128, False), (2, 37, 3, 1, 64, 32, True), (1, 1191, 3, 1, 64, 64, False),
                                  (1, 3, 1, 2, 1024, 0, False), (1, 6, 2, 1, 37, 36, False)])
def test_gradients_without_eps(ops, case, dtype):
    """eps = 0: the formula is finite for rows that are not zero, and so are its gradients, with fewer heads than groups
    of lanes and a last block that its tokens do not fill.  Tolerances as in test_gradients."""
    B, L, hq, hk, d, rot, inter = case
    q, k, wq, wk = make(B, L, hq, hk, d, dtype, seed=d + 2)
    g = torch.Generator(device="cuda").manual_seed(6)
    gq = torch.randn(q.shape, generator=g, device="cuda").to(dtype)
    gk = torch.randn(k.shape, generator=g, device="cuda").to(dtype)
    pos = torch.randint(0, 4000, (B, L), device="cuda")
    got = ops.qk_norm_rope_bwd(q, k, wq, wk, gq, gk, pos, rotary_dim=rot, interleaved=inter, eps=0.0)
    rows = B * L * max(hq, hk)
    for x, w, gy, gx, gw in ((q, wq, gq, got[0], got[2]), (k, wk, gk, got[1], got[3])):
        lx, lw = x.double().requires_grad_(), w.double().requires_grad_()
        rx, rw = torch.autograd.grad(ref_one(lx, lw, pos, 10000.0, rot, inter, 0.0), (lx, lw), gy.double())
        inv = 1 / torch.sqrt((x.double() ** 2).mean(-1, keepdim=True))
        n = x.double() * inv
        size = 2 * inv * (gy.double().abs().amax(-1, keepdim=True) * 1.5 * w.abs().max() * (2 + n.abs() * n.abs().mean(-1, keepdim=True)))
        tol = half_step(dtype) * rx.abs() + (d + 80) * 2.0 ** -24 * size + (2.0 ** -25 if dtype == F16 else 0)
        assert bool(((gx.double() - rx).abs() <= tol).all())
        sizes = (gy.double().abs().amax(-1, keepdim=True) * 1.5 * n.abs()).flatten(0, 2).sum(0)
        assert bool(((gw.double() - rw).abs() <= (d / 2 + 40 + rows) * 2.0 ** -24 * sizes + 1e-30).all())


@pytest.mark.parametrize("wdtype", [BF, F16])
def test_weights_of_16_bits_are_read_at_each_call(ops, wdtype):
    """The result is that of the weights' values at the call (widened exactly): after a write that autograd's version
    count does not see, for tensors without such a count, from another stream, and at each replay of a graph that was
    captured after a first call."""
    q, k, wq, wk = make(2, 9, 2, 1, 64, BF, seed=3)
    pos = torch.arange(9, device="cuda")
    wq, wk = wq.to(wdtype), wk.to(wdtype)
    f = lambda: torch.cat([t.flatten() for t in ops.qk_norm_rope(q, k, wq, wk, pos)])
    want = lambda: torch.cat([t.flatten() for t in ops.qk_norm_rope(q, k, wq.float(), wk.float(), pos)])
    assert torch.equal(f(), want())
    wq.data.mul_(2)
    wk.data.add_(1)
    assert torch.equal(f(), want())
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        wq.data.mul_(0.5)
        got = f()
    torch.cuda.synchronize()
    assert torch.equal(got, want())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = f()
    for _ in range(2):
        wq.mul_(-2)
        wk.data.mul_(0.5)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want())
    with torch.inference_mode():
        wq, wk = wq.clone(), wk.clone()
        assert torch.equal(f(), want())
