"""The query / key norms with rotation, linear attention and sampling in one run, as a decoder uses them; linear
attention's bounded waits; what the wrappers refuse of CUDA tensors; generate on sample_tokens.

Tolerance of the fp32 runs: an element of q or k comes from a sum of d squares and some ten operations, a sum of the
attention from at most L + dk + dv terms, each with a relative error of 2^-24: (L + dk + dv + 2 d + 64) 2^-24 times
the same sum over absolute values (two norms, hence 2 d).
"""
import threading

import pytest
import torch

from tests.test_linear_attn_gpu import inputs, recur
from tests.test_sample_gpu import ref_row

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")
    torch.cuda.set_device(0)
    from hybrid_model_mamba_xlstm_b200 import kernels
    return kernels


def norm_rope(x, w, pos, base=1e4, eps=1e-6):
    """Plain form in 64 bits, halves as pairs."""
    x, d = x.double(), x.shape[-1]
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    a = pos.double()[..., None, None] * base ** (-torch.arange(0, d, 2, device=x.device, dtype=torch.float64) / d)
    lo, hi = y[..., :d // 2], y[..., d // 2:]
    return torch.cat([lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin()], -1)


def test_a_decoders_prompt_and_steps(ops):
    """Token -> q, k, v (a table) -> norms and rotation -> attention over a padded batch of prompts -> logits ->
    tokens, then steps on the carried states, all positions a row's own.  Each attention output is held to the
    64-bit recurrence over the row's whole history, each token to the sampling rule on the logits."""
    B, L, H, d, V, steps = 3, 70, 2, 64, 50, 6
    g = torch.Generator(device="cuda").manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    table, out_w = r(V, 3 * H * d), r(H * d, V) / (H * d) ** 0.5
    qw, kw, ld = 1 + 0.1 * r(d), 1 + 0.1 * r(d), torch.tensor([-0.02, -0.3], device="cuda")
    lengths = torch.tensor([70, 1, 33], device="cuda")
    ids = torch.randint(0, V, (B, L), generator=g, device="cuda")
    u = torch.rand(B, steps, generator=g, device="cuda")

    def heads(t):
        return (x.unflatten(-1, (H, d)) for x in table[t].chunk(3, -1))

    q, k, v = heads(ids)
    q, k = ops.qk_norm_rope(q, k, qw, kw, torch.arange(L, device="cuda"))
    o, state = ops.linear_attention(q, k, v, ld, lengths=lengths, return_final_state=True)
    last = o[torch.arange(B, device="cuda"), lengths - 1]
    history = [ids[b, :int(lengths[b])] for b in range(B)]
    for i in range(steps):
        for b in range(B):
            q, k, v = (x.double()[None] for x in heads(history[b]))
            at = torch.arange(len(history[b]), device="cuda")[None]
            q, k = norm_rope(q, qw, at), norm_rope(k, kw, at)
            ref = recur(q, k, v, ld, d ** -0.5)[0][0, -1]
            A = recur(q.abs(), k.abs(), v.abs(), ld, d ** -0.5)[0][0, -1]
            # a rotated element is a sum of two: its error is relative to their absolute values
            A = A.amax() * 2
            assert bool(((last[b].double() - ref).abs() <= (len(history[b]) + 4 * d + 64) * 2.0 ** -24 * A).all())
        logits = (last.flatten(1).double() @ out_w.double()).float()
        tokens = ops.sample_tokens(logits, u[:, i], temperature=0.7, top_k=20, top_p=0.9, min_p=0.01)
        for b in range(B):
            t, _, near = ref_row(logits[b].double().cpu().numpy(), float(u[b, i]), float(torch.tensor(0.7)), 20,
                                 float(torch.tensor(0.9)), float(torch.tensor(0.01)))
            assert near < V * 2.0 ** -45 or int(tokens[b]) == t
            history[b] = torch.cat([history[b], tokens[b:b + 1]])
        q, k, v = heads(tokens)
        q, k = ops.qk_norm_rope(q[:, None], k[:, None], qw, kw, (lengths + i)[:, None])
        last = ops.linear_attention_step(q[:, 0], k[:, 0], v, ld, state)


def test_gradients_through_both(ops):
    """Gradients of projections, norm weights and the first state through rotation and attention, against 64-bit
    autograd of the plain forms.  Norm of the error: each of the T = L + dk + dv + 2 d + 64 roundings on the way of
    an element is at most 2^-24 of a sum over absolute values, whose norm is below T times the result's."""
    B, L, H, d = 2, 45, 2, 32
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    leaves = [r(B, L, 3 * H * d), 1 + 0.1 * r(d), 1 + 0.1 * r(d), r(B, H, d, d)]
    ld, w, pos = torch.tensor([-0.02, -0.3], device="cuda"), r(B, L, H, d), torch.arange(L, device="cuda")

    def run(leaves, plain):
        x, qw, kw, s0 = leaves
        q, k, v = (t.unflatten(-1, (H, d)) for t in x.chunk(3, -1))
        if plain:
            q, k = norm_rope(q, qw, pos), norm_rope(k, kw, pos)
            return recur(q, k, v, ld, d ** -0.5, s0=s0)[0]
        q, k = ops.qk_norm_rope(q, k, qw, kw, pos)
        return ops.linear_attention(q, k, v, ld, initial_state=s0)

    a = [t.clone().requires_grad_() for t in leaves]
    b = [t.double().requires_grad_() for t in leaves]
    got = torch.autograd.grad((run(a, False) * w).sum(), a)
    ref = torch.autograd.grad((run(b, True) * w).sum(), b)
    T = L + 4 * d + 64
    for x, y in zip(got, ref):
        assert float((x.double() - y).norm() / y.norm()) <= T * 2.0 ** -24


@pytest.mark.parametrize("L,H,d", [(300, 2, 128), (300, 2, 192), (4000, 1, 64)])
def test_attention_waits_run_out(ops, L, H, d):
    """A negative limit makes every wait give up at once: the kernel drains its own loads, frees its tensor memory,
    sets the word and returns, and the next call is as before (4000 steps of one head: cut along time)."""
    q, k, v, ld, s0 = inputs(1, L, H, d, d, BF, seed=d, s0=True)
    flag = torch.zeros(1, device="cuda", dtype=torch.int32)

    def both(limit):
        o, sT = ops.linear_attention(q, k, v, ld, initial_state=s0, return_final_state=True, error_flag=flag, wait_limit_cycles=limit)
        return (o, sT) + ops.linear_attention_bwd(q, k, v, ld, v, initial_state=s0, error_flag=flag, wait_limit_cycles=limit)

    first = both(0)
    assert int(flag) == 0
    both(-1)
    torch.cuda.synchronize()
    assert int(flag) == 1
    flag.zero_()
    again = both(0)
    assert int(flag) == 0
    for x, y in zip(first, again):
        assert torch.equal(x, y)


def test_first_call_of_a_thread(ops):
    """A thread whose first use of CUDA is one of the calls (its memory comes from the allocator's cache): the
    results are the main thread's."""
    q, k, v, ld, s0 = inputs(1, 200, 2, 64, 64, BF, s0=True)
    x = torch.randn(2, 100, device="cuda")
    calls = [lambda: ops.linear_attention_bwd(q, k, v, ld, v, initial_state=s0), lambda: ops.linear_attention(q, k, v, ld, return_final_state=True),
             lambda: ops.qk_norm_rope(q, k), lambda: (ops.sample_tokens(x, x[:, 0].abs() % 1),),
             lambda: ops.qk_norm_rope_bwd(q, k, ld.new_ones(64), ld.new_ones(64), v, v)]
    for go in calls:
        main = [t.clone() for t in go()]
        got = []
        thread = threading.Thread(target=lambda: got.extend(go()))
        thread.start()
        thread.join()
        torch.cuda.synchronize()
        assert len(got) == len(main) and all(torch.equal(a, b) for a, b in zip(main, got))


@pytest.mark.parametrize("dtype,d", [(BF, 128), (F32, 128)])
def test_attention_offsets_beyond_32_bits(ops, dtype, d):
    """Over 2^31 elements: with no memory between steps (log_decay -inf) o = scale (q k) v for every step, which the last
    rows show; the gradients there are those of the same rows alone."""
    L, H, tail = 2 ** 31 // (16 * d) + 200, 16, 300
    ld = torch.full((H,), -float("inf"), device="cuda")
    big = [torch.zeros(1, L, H, d, device="cuda", dtype=dtype) for _ in range(3)]
    small = inputs(1, tail, H, d, d, dtype, seed=1)[:3]
    for x, y in zip(big, small):
        x[:, -tail:] = y
    q, k, v = (x.double() for x in small)
    ref, size = 0.1 * (q * k).sum(-1, keepdim=True) * v, 0.1 * (q * k).abs().sum(-1, keepdim=True) * v.abs()
    o = ops.linear_attention(*big, ld, scale=0.1)
    unit = (d + 64) * 2.0 ** -24 * size + (2.0 ** -8 * (ref.abs() + size) if dtype == BF else 0)
    assert bool(((o[:, -tail:].double() - ref).abs() <= unit).all()) and float(o[:, :-tail].abs().max()) == 0
    del o
    # chunks begin elsewhere in the long call: the same sums in another order, each product rounded apart
    got = ops.linear_attention_bwd(*big, ld, big[2], scale=0.1)
    want = ops.linear_attention_bwd(*small, ld, small[2], scale=0.1)
    for x, y in zip(got[:3], want[:3]):
        assert float((x[:, -tail:].double() - y.double()).norm() / y.double().norm()) <= (2.0 ** -7 if dtype == BF else (d + 64) * 2.0 ** -24)
        assert float(x[:, :-tail].abs().max()) == 0


def test_other_offsets_beyond_32_bits(ops):
    """The last rows of over 2^31 elements of state, of heads and of logits are those of the same rows alone."""
    g = torch.Generator(device="cuda").manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    B, H, d = 2 ** 31 // (16 * 128 * 128) + 3, 16, 128
    state, ld = torch.zeros(B, H, d, d, device="cuda"), torch.full((H,), -0.1, device="cuda")
    state[-2:] = r(2, H, d, d)
    q, k, v, last = r(B, H, d), r(B, H, d), r(B, H, d), state[-2:].clone()
    o, o2 = ops.linear_attention_step(q, k, v, ld, state), ops.linear_attention_step(q[-2:], k[-2:], v[-2:], ld, last)
    assert torch.equal(o[-2:], o2) and torch.equal(state[-2:], last)
    del state, o
    L = 2 ** 31 // (16 * 128) + 5
    x, w = torch.zeros(1, L, 16, 128, device="cuda", dtype=BF), 1 + 0.1 * r(128)
    x[:, -9:] = r(1, 9, 16, 128).to(BF)
    pos = torch.arange(L, device="cuda")
    y, z = ops.qk_norm_rope(x, x[:, :, :1], w, w, pos)
    y2, z2 = ops.qk_norm_rope(x[:, -9:], x[:, -9:, :1], w, w, pos[-9:])
    assert torch.equal(y[:, -9:], y2) and torch.equal(z[:, -9:], z2)
    dx, _, _, _ = ops.qk_norm_rope_bwd(x, x[:, :, :1], w, w, y, z, pos)
    dx2, _, _, _ = ops.qk_norm_rope_bwd(x[:, -9:], x[:, -9:, :1], w, w, y2, z2, pos[-9:])
    assert torch.equal(dx[:, -9:], dx2)
    del x, y, z, dx
    V = 50304
    B = 2 ** 31 // V + 5
    logits = torch.zeros(B, V, device="cuda", dtype=BF)
    logits[-4:] = r(4, V).to(BF)
    u = torch.rand(B, generator=g, device="cuda")
    for kw in (dict(), dict(top_k=50), dict(top_p=0.9)):
        assert torch.equal(ops.sample_tokens(logits, u, **kw)[-4:], ops.sample_tokens(logits[-4:], u[-4:], **kw))


def test_attention_refusals(ops):
    q, k, v, ld, s0 = inputs(2, 9, 2, 16, 24, F32, s0=True)
    f, step = ops.linear_attention, ops.linear_attention_step
    bad = [lambda: f(q[0], k, v, ld), lambda: f(q, k[:, :-1], v, ld), lambda: f(q, k, v[..., 0], ld), lambda: f(q, k, v, ld[:1]),
           lambda: f(q, k, v, ld, scale=0.0), lambda: f(q, k, v, ld, scale=float("nan")), lambda: f(q, k, v, ld, scale=1e-60),
           lambda: f(q, k, v, ld, lengths=torch.ones(3, device="cuda", dtype=torch.int32)),
           lambda: f(q, k, v, ld, lengths=torch.ones(2, device="cuda")), lambda: f(q, k, v, ld, initial_state=s0[..., :-1]),
           lambda: f(q, k, v, ld.clone().requires_grad_()),
           lambda: f(q.clone().requires_grad_(), k, torch.zeros(2, 9, 2, 520, device="cuda"), ld),
           lambda: ops.linear_attention_bwd(q, k, v, ld, v[:, :-1]), lambda: ops.linear_attention_bwd(q, k, v, ld, v, d_final_state=s0[:1]),
           lambda: step(q[:, 0], k[:, 0], v[:, 0], ld, s0[:1]), lambda: step(q[:, 0], k[:, 0], v[:, 0], ld, s0.to(BF)),
           lambda: step(q[:, 0], k[:, 0], v[:, 0], ld, s0.transpose(2, 3).contiguous().transpose(2, 3)),
           lambda: step(q[:, 0], k[:, 0], v[:, 0], ld, s0[:1].expand(2, -1, -1, -1)),
           lambda: step(q[:, 0], k[:, 0], v[:, 0], ld, s0.clone().requires_grad_()),
           lambda: step(q[:, 0], k[:, 0], v[:, 0], ld, s0, out=torch.empty(2, 2, 16, device="cuda")),
           lambda: step(q[:, 0], k[:, 0], v[:, 0], ld, s0, out=torch.empty(1, 2, 24, device="cuda").expand(2, -1, -1))]
    before = s0.clone()
    for go in bad:
        with pytest.raises(ValueError):
            go()
    for go in (lambda: f(q.half(), k.half(), v.half(), ld), lambda: f(q, k.to(BF), v, ld), lambda: step(q[:, 0], k[:, 0].to(BF), v[:, 0], ld, s0)):
        with pytest.raises(TypeError):
            go()
    with pytest.raises(RuntimeError, match="CUDA device"):
        f(q, k, v, ld.cpu())
    x = torch.zeros(1, 2, 1, 600, device="cuda")
    with pytest.raises(Exception, match="at most 512"):
        f(x, x, x, ld[:1])
    leaf = q.clone().requires_grad_()
    (gr,) = torch.autograd.grad(f(leaf, k, v, ld).sum(), leaf, create_graph=False)
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(f(leaf, k, v, ld).sum(), leaf, create_graph=True)
    assert torch.equal(s0, before)


def test_norm_refusals(ops):
    q, k = torch.randn(2, 5, 4, 32, device="cuda"), torch.randn(2, 5, 1, 32, device="cuda")
    w, pos = torch.ones(32, device="cuda"), torch.arange(5, device="cuda")
    f = ops.qk_norm_rope
    bad = [lambda: f(q[0], k), lambda: f(q, k[:, :-1]), lambda: f(q, k[..., :-1]), lambda: f(q, k, w[:-1]), lambda: f(q, k, w, w[:-1]),
           lambda: f(q, k, w, w, pos, rotary_dim=3), lambda: f(q, k, w, w, pos, rotary_dim=34), lambda: f(q, k, w, w, pos, rotary_dim=-2),
           lambda: f(q, k, rotary_dim=8), lambda: f(q, k, w, w, pos.float()), lambda: f(q, k, w, w, pos[:-1]),
           lambda: f(q, k, w, w, pos, rope_base=0.0), lambda: f(q, k, w, w, pos, rope_base=float("inf")),
           lambda: ops.qk_norm_rope_bwd(q, k, w, w, q[:, :-1], k, pos)]
    for go in bad:
        with pytest.raises(ValueError):
            go()
    for go in (lambda: f(q.double(), k.double()), lambda: f(q, k.to(BF))):
        with pytest.raises(TypeError):
            go()
    with pytest.raises(RuntimeError, match="CUDA device"):
        f(q, k, w.cpu())
    leaf = q.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(f(leaf, k)[0].square().sum(), leaf, create_graph=True)


def test_sampling_refusals(ops):
    x, u = torch.randn(3, 40, device="cuda"), torch.rand(3, device="cuda")
    f = ops.sample_tokens
    bad = [lambda: f(x[0], u), lambda: f(x, u[:2]), lambda: f(x[:, :0], u), lambda: f(x, u, temperature=-1.0),
           lambda: f(x, u, temperature=float("nan")), lambda: f(x, u, top_k=-1), lambda: f(x, u, top_k=1.5), lambda: f(x, u, top_p=1.1),
           lambda: f(x, u, top_p=-0.1), lambda: f(x, u, min_p=2.0), lambda: f(x, u, min_p=float("nan")),
           lambda: f(x, u, temperature=torch.ones(2, device="cuda")), lambda: f(x, u, top_p=torch.ones(3, 1, device="cuda"))]
    for go in bad:
        with pytest.raises(ValueError):
            go()
    for go in (lambda: f(x.double(), u), lambda: f(x, u, top_k=torch.ones(3, device="cuda"))):
        with pytest.raises(TypeError):
            go()
    with pytest.raises(RuntimeError, match="CUDA device"):
        f(x, u.cpu())


@pytest.mark.parametrize("graph", [True, False])
def test_generate_from_uniforms(ops, graph):
    """The tokens of generate are sample_tokens' on the model's own logits, repeat exactly for the same numbers, and
    are the largest logits' at temperature 0; without min_p and uniforms the sampling is as before."""
    import hybrid_model_mamba_xlstm_b200.layers as layers
    torch.manual_seed(0)
    cfg = layers.HybridConfig(vocab_size=97, dim=64, num_layers=4, layer_pattern=["mamba", "mamba", "mlstm", "slstm"], state_size=16,
                              conv_size=4, expand_factor=2, head_dim=32, num_heads=2, slstm_num_heads=4, dropout=0.0, slstm_recurrent=False)
    model = layers.HybridLanguageModel(cfg).cuda().eval()
    g = torch.Generator(device="cuda").manual_seed(1)
    prompt, u = torch.randint(0, 97, (2, 9), device="cuda", generator=g), torch.rand(2, 6, device="cuda", generator=g)
    args = dict(max_new_tokens=6, temperature=0.8, top_k=30, top_p=0.95, cuda_graph=graph)
    out = model.generate(prompt, min_p=0.02, uniforms=u, **args)
    assert out.shape == (2, 15) and torch.equal(out[:, :9], prompt)
    assert torch.equal(out, model.generate(prompt, min_p=0.02, uniforms=u, **args))
    with torch.no_grad():  # the same pieces: prompt, then one token at a time
        caches = model.init_caches()
        logits = model(prompt, caches=caches)[:, -1, :]
        for i in range(6):
            t = ops.sample_tokens(logits, u[:, i], temperature=0.8, top_k=30, top_p=0.95, min_p=0.02)
            assert torch.equal(t, out[:, 9 + i])
            logits = model(t[:, None], caches=caches)[:, -1, :]
    greedy = model.generate(prompt, max_new_tokens=6, temperature=0, uniforms=u, cuda_graph=graph)
    assert torch.equal(greedy, model.generate(prompt, max_new_tokens=6, top_k=1, cuda_graph=graph))
    drawn = model.generate(prompt, min_p=0.1, **args)
    assert drawn.shape == (2, 15) and 0 <= int(drawn.min()) and int(drawn.max()) < 97
    with pytest.raises(ValueError, match="uniforms"):
        model.generate(prompt, max_new_tokens=6, uniforms=u[:, :5])


def test_norms_refuse_an_eps_that_is_none(ops):
    q, w = torch.randn(2, 5, 4, 32, device="cuda"), torch.ones(32, device="cuda")
    for eps in (-1e-6, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            ops.qk_norm_rope(q, q, w, w, eps=eps)
        with pytest.raises(ValueError, match="eps"):
            ops.qk_norm_rope_bwd(q, q, w, w, q, q, eps=eps)


def test_threads_with_calls_of_other_sizes(ops):
    """Threads whose calls of one kernel need different amounts of shared memory: each result is the one of a call alone
    (no call is refused because another thread's needs less)."""
    def attn(dk, L):
        q, k, v, ld, s0 = inputs(1, L, 2, dk, 20, F32, seed=dk)
        return lambda: ops.linear_attention(q, k, v, ld)

    def norms(d):
        x = torch.randn(1, 3, 2, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(d))
        w = torch.ones(d, device="cuda")
        return lambda: torch.cat([t.flatten() for t in ops.qk_norm_rope_bwd(x, x, w, w, x, x)])

    def tokens(V):
        x = torch.randn(2, V, device="cuda", generator=torch.Generator(device="cuda").manual_seed(V))
        u = torch.tensor([0.3, 0.8], device="cuda")
        return lambda: ops.sample_tokens(x, u, top_k=20)

    kinds = [[attn(20, 40), attn(130, 40), attn(250, 40)], [norms(33), norms(501), norms(1001)], [tokens(300), tokens(50000), tokens(260000)]]
    for calls in kinds:
        want = [c().clone() for c in calls]
        torch.cuda.synchronize()
        wrong, errors = [], []

        def work(i):
            try:
                with torch.cuda.stream(torch.cuda.Stream()):
                    for _ in range(300):
                        got = calls[i % 3]()
                    torch.cuda.current_stream().synchronize()
                    if not torch.equal(got, want[i % 3]):
                        wrong.append(i)
            except Exception as e:
                errors.append(e)

        threads = [threading.Thread(target=work, args=(i,)) for i in range(9)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not errors and not wrong, (errors[:1], wrong)


@pytest.mark.parametrize("kind", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64])
def test_integers_of_every_type(ops, kind):
    """lengths, per-row top_k and positions in a type that does not reach the sequence's or the vocabulary's size."""
    n = torch.tensor([0, 1, 100], device="cuda")
    q, k, v, ld, _ = inputs(3, 777, 2, 16, 16, F32, seed=1)
    assert torch.equal(ops.linear_attention(q, k, v, ld, lengths=n.to(kind)), ops.linear_attention(q, k, v, ld, lengths=n.int()))
    x, u = torch.randn(3, 50304, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)), torch.tensor([0.1, 0.5, 0.9], device="cuda")
    assert torch.equal(ops.sample_tokens(x, u, top_k=n.to(kind)), ops.sample_tokens(x, u, top_k=n.int()))
    a, b = ops.qk_norm_rope(q[:, :3], k[:, :3], None, None, n.to(kind)), ops.qk_norm_rope(q[:, :3], k[:, :3], None, None, n)
    assert all(torch.equal(s, t) for s, t in zip(a, b))
    if kind not in (torch.uint8,):
        m = torch.tensor([-3, 5, 127], device="cuda")
        assert torch.equal(ops.linear_attention(q, k, v, ld, lengths=m.to(kind)), ops.linear_attention(q, k, v, ld, lengths=m.clamp(min=0)))
        assert torch.equal(ops.sample_tokens(x, u, top_k=m.to(kind)), ops.sample_tokens(x, u, top_k=m.clamp(min=0)))


def test_a_state_that_autograd_keeps_is_not_changed_behind_its_back(ops):
    """A step updates its state in place: gradients that need the old state say so, as for any torch operator that
    writes in place, and so do those that need what `out` held."""
    q, k, v, ld, s0 = inputs(2, 9, 2, 16, 24, F32, seed=2, s0=True)
    leaf = q.clone().requires_grad_()
    for change in (lambda: ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s0),
                   lambda: ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s0.clone(), out=v[:, 3])):
        o = ops.linear_attention(leaf, k, v, ld, initial_state=s0)
        change()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(o.sum(), leaf)
    with torch.inference_mode():
        s = s0.clone()
        ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s)


def test_error_flags_that_are_no_flags(ops):
    """error_flag is one 32-bit word that a kernel may write: any other tensor is refused."""
    q, k, v, ld, _ = inputs(1, 9, 2, 16, 24, F32)
    for flag in (torch.zeros(1, device="cuda", dtype=torch.uint8), torch.zeros(0, device="cuda", dtype=torch.int32),
                 torch.zeros(1, device="cuda"), torch.zeros(1, device="cuda", dtype=torch.int64)):
        with pytest.raises(ValueError, match="error_flag"):
            ops.linear_attention(q, k, v, ld, error_flag=flag)
        with pytest.raises(ValueError, match="error_flag"):
            ops.linear_attention_bwd(q, k, v, ld, v, error_flag=flag)
    flag = torch.zeros(2, device="cuda", dtype=torch.int32)
    ops.linear_attention(q, k, v, ld, error_flag=flag)
    assert int(flag.abs().sum()) == 0


def test_a_step_does_not_write_into_a_graph(ops):
    """An `out` that autograd has a history or a gradient for is refused, as by torch's own out= functions."""
    q, k, v, ld, s0 = inputs(2, 1, 2, 16, 24, F32, seed=2, s0=True)
    before = s0.clone()
    leaf = torch.zeros(2, 2, 24, device="cuda", requires_grad=True)
    for out in (leaf, leaf * 2):
        with pytest.raises(ValueError, match="no gradient"):
            ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s0, out=out)
    assert torch.equal(s0, before)
    with torch.no_grad():
        ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s0, out=leaf)
