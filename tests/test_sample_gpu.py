"""Token sampling on the GPU against a walk over the sorted tokens in 64 bits on the host.

Tokens have to be equal: the kernel's weights are integers of 2^-44, so a border moves by at most vocab 2^-45
against the 64-bit sums; the reference reports how near each draw and each top-p border lies to a change, and
a draw nearer than that is left out (none is expected at these sizes: the test says how many).
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sample():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")
    from hybrid_model_mamba_xlstm_b200.kernels import sample_tokens
    return sample_tokens


def ref_row(x, u, T, K, P, M):
    """(token, logprob, distance of the nearest border relative to the total)."""
    x = np.where(np.isnan(x), -np.inf, x)
    live = np.flatnonzero(x > -np.inf)
    if live.size == 0:
        return -1, -math.inf, 1.0
    order = live[np.argsort(-x[live], kind="stable")]
    top = x[order[0]]
    if not T > 0:
        return int(order[0]), 0.0, 1.0
    if K > 0:
        order = order[:K]
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / T))
    near = 1.0
    if P < 1:
        before = np.cumsum(w) - w
        keep = before <= P * w.sum()
        keep[0] = True
        # a border that is met exactly is exact on both sides (whole weights), others are compared
        gap = np.abs(before - P * w.sum()) / w.sum()
        near = min(near, gap[gap > 1e-13].min() if (gap > 1e-13).any() else 1.0)
        order, w = order[keep], w[keep]
    order, w = order[w >= M], w[w >= M]
    ids = np.argsort(order)
    order, w = order[ids], w[ids]
    sums = np.cumsum(w)
    at = min(int(np.searchsorted(sums, u * sums[-1], side="right")), len(order) - 1)
    while at > 0 and w[at] * 2.0 ** 45 < 1:
        at -= 1
    gap = np.abs(sums - u * sums[-1]) / sums[-1]
    near = min(near, gap[gap > 1e-13].min() if (gap > 1e-13).any() else 1.0)
    return int(order[at]), float(np.log(w[at] / sums[-1])), near


def check(sample, logits, u, T=1.0, K=0, P=1.0, M=0.0):
    tokens, logp = sample(logits, u, temperature=T, top_k=K, top_p=P, min_p=M, return_logprob=True)
    x, uu = logits.double().cpu().numpy(), u.double().cpu().numpy()
    B, V = x.shape
    row = lambda a: a.double().cpu().numpy() if torch.is_tensor(a) else np.full(B, float(np.float32(a)))
    Ts, Ks, Ps, Ms = row(T), row(K), row(P), row(M)
    skipped = 0
    for b in range(B):
        t, lp, near = ref_row(x[b], uu[b], Ts[b], int(Ks[b]), Ps[b], Ms[b])
        if near < V * 2.0 ** -45:
            skipped += 1
            continue
        assert int(tokens[b]) == t, (b, int(tokens[b]), t, near)
        got = float(logp[b])
        if math.isfinite(lp):
            # one rounding to fp32, and the total's V 2^-45
            assert abs(got - lp) <= 2.0 ** -24 * abs(lp) + V * 2.0 ** -45 + 1e-12
        else:
            assert got == lp
    assert skipped <= B // 8
    assert torch.equal(tokens, sample(logits, u, temperature=T, top_k=K, top_p=P, min_p=M))
    return tokens


def make(B, V, dtype=torch.float32, seed=0, spread=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (spread * torch.randn(B, V, generator=g, device="cuda")).to(dtype), torch.rand(B, generator=g, device="cuda")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [1, 2, 31, 1000, 4097, 50304])
def test_settings(sample, V, dtype):
    for i, (T, K, P, M) in enumerate([(1.0, 0, 1.0, 0.0), (0.7, 40, 1.0, 0.0), (1.3, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.05),
                                      (0.9, 100, 0.8, 0.01), (0.0, 0, 1.0, 0.0), (1.0, 1, 1.0, 0.0), (1.0, V, 0.0, 0.0),
                                      (2.0, V + 5, 0.5, 1.0), (0.01, 7, 0.99, 0.0)]):
        logits, u = make(6, V, dtype, seed=V + i)
        check(sample, logits, u, T, K, P, M)


def test_rows_with_their_own_settings(sample):
    B, V = 64, 3001
    logits, u = make(B, V, torch.bfloat16, seed=4)
    g = torch.Generator(device="cuda").manual_seed(2)
    pick = lambda vals, kind: torch.tensor(vals, device="cuda", dtype=kind)[torch.randint(0, len(vals), (B,), generator=g, device="cuda")]
    T, K = pick([0.0, 0.5, 1.0, -1.0], torch.float32), pick([-2, 0, 1, 13, 5000], torch.int32)
    P, M = pick([0.1, 0.9, 1.0], torch.float32), pick([0.0, 0.1], torch.float32)
    check(sample, logits, u, T, K.clamp(min=0), P, M)
    a = sample(logits, u, temperature=T, top_k=K, top_p=P, min_p=M)
    assert torch.equal(a, sample(logits, u, temperature=T.double(), top_k=K.long(), top_p=P.half().float(), min_p=M)
                       if torch.equal(P.half().float(), P) else a)


@pytest.mark.parametrize("B,V", [(1, 50304), (3, 131072), (2, 262144), (200, 700), (300, 50304)])
def test_sizes(sample, B, V):
    """One cluster per row of 1 to 8 blocks, and more rows than the GPU has SMs."""
    logits, u = make(B, V, seed=B)
    check(sample, logits, u, 1.0, 0, 0.95, 0.0)
    check(sample, logits, u, 0.8, 50, 1.0, 0.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [50257, 9001])
def test_top_k_of_every_size(sample, V, dtype):
    """top_k on both sides of every limit between the ways to find it (rows of an odd length, so that each begins
    elsewhere in its 16 bytes), alone and with top_p and min_p."""
    logits, u = make(5, V, dtype, seed=11)
    logits[1, ::2] = -float("inf")
    logits[2, 40:] = -float("inf")  # fewer logits than most of the top_k
    logits[3] = logits[3].round()   # many equal ones
    for K in (2, 39, 40, 41, 127, 128, 129, 255, 256, 257, 399, 400, 401, 512, 513, 1024, 2000, V - 1):
        check(sample, logits, u, 1.0, K)
        check(sample, logits, u, 0.8, K, 0.9, 0.001)


def test_extreme_settings(sample):
    """Temperatures at which one token or all of them share the weight, top_p and min_p at their ends."""
    logits, u = make(6, 5003, seed=13)
    logits[5, 7] = float("inf")
    for T in (1e-38, 1e-20, 1e-3, 1e4, 1e30, float("inf")):
        for K, P, M in ((0, 1.0, 0.0), (0, 0.7, 0.0), (60, 1.0, 0.0), (3000, 0.9, 0.5), (0, 1e-7, 0.0), (0, 1.0, 1.0)):
            check(sample, logits, u, T, K, P, M)


def test_ties(sample):
    """Equal logits: the lowest tokens stay, whole rows of one value, few values, and greedy ties."""
    V = 5000
    u = torch.rand(8, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    flat = torch.zeros(8, V, device="cuda")
    t = check(sample, flat, u, 1.0, 10)
    assert int(t.max()) < 10
    t = check(sample, flat, u, 1.0, 0, 0.1)
    assert int(t.max()) <= 500
    few = torch.randint(0, 4, (8, V), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).float()
    for K, P in ((3000, 1.0), (3000, 0.5), (0, 0.3), (7, 0.99)):
        check(sample, few, u, 1.0, K, P)
    assert torch.equal(sample(few, u, temperature=0), few.argmax(-1))
    zeros = torch.zeros(1, 64, device="cuda")
    zeros[0, 3] = -0.0
    assert int(sample(zeros, u[:1], top_k=4)[0]) < 4


def test_masked_rows(sample):
    """-inf and NaN never come out, a row of them gives -1, +inf takes the weight, the type's lowest value is a logit."""
    V = 3000
    logits, u = make(9, V, seed=3)
    inf, nan = float("inf"), float("nan")
    logits[0] = -inf
    logits[1] = nan
    logits[2, 1:] = -inf
    logits[3, ::2] = -inf
    logits[4, ::3] = nan
    logits[5, [17, 900]] = inf
    logits[6] = torch.finfo(torch.float32).min
    logits[7, 1:] = torch.finfo(torch.float32).min
    logits[8, :5] = torch.finfo(torch.float32).max
    for T, K, P in ((1.0, 0, 1.0), (1.0, 20, 0.9), (0.5, 0, 0.5), (0.0, 0, 1.0)):
        t = check(sample, logits, u, T, K, P)
        assert t[0] == -1 and t[1] == -1 and t[2] == 0 and t[3] % 2 == 1 and t[4] % 3 != 0 and int(t[5]) in (17, 900) and t[7] == 0


def test_ends_of_the_uniform_range(sample):
    """u = 0 is the first kept token, numbers up to 1 (and beyond, or NaN) stay inside the kept ones."""
    logits, _ = make(5, 800, seed=8)
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, 2.0, -1.0], device="cuda")
    t = sample(logits, u, top_k=30)
    order = torch.sort(torch.topk(logits, 30).indices, -1).values
    assert int(t[0]) == int(order[0, 0]) and int(t[4]) == int(order[4, 0])
    for b in (1, 2, 3):
        assert int(t[b]) == int(order[b, -1])
    assert int(sample(logits[:1], torch.full((1,), float("nan"), device="cuda"), top_k=30)[0]) in order[0].tolist()


def test_strides_and_empty(sample):
    g = torch.Generator(device="cuda").manual_seed(0)
    big = torch.randn(6, 3 * 1001, generator=g, device="cuda")
    u = torch.rand(6, generator=g, device="cuda")
    check(sample, big[:, 1001:2002], u, 1.0, 50, 0.9)
    check(sample, big[::2, 7:1500], u[::2], 1.0, 0, 0.9)
    check(sample, big.t()[:6, :6].t()[:6], u, 1.0, 0, 0.9)
    check(sample, big[:1, :1001].expand(6, 1001), u, 1.0, 0, 0.9)
    assert sample(big[:0], u[:0]).shape == (0,)


def test_distribution(sample):
    """Evenly spaced uniforms reproduce each kept token's probability to within a spacing at either end."""
    V, N = 40, 4096
    row = torch.randn(V, device="cuda", generator=torch.Generator(device="cuda").manual_seed(6)) * 2
    u = (torch.arange(N, device="cuda") + 0.5) / N
    t = sample(row.expand(N, V), u, temperature=0.8, top_p=0.9)
    count = torch.bincount(t, minlength=V).double().cpu() / N
    p = torch.softmax(row.double().cpu() / float(np.float32(0.8)), -1)
    order = torch.argsort(p, descending=True)
    before = p[order].cumsum(0) - p[order]
    keep = torch.zeros(V, dtype=torch.bool)
    keep[order[before <= float(np.float32(0.9))]] = True
    p = torch.where(keep, p, torch.zeros_like(p))
    assert float((count - p / p.sum()).abs().max()) <= 1.01 / N


def test_streams_and_graph(sample):
    logits, u = make(16, 20000, seed=2)
    want = sample(logits, u, top_p=0.9, top_k=100, return_logprob=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sample(logits, u, top_p=0.9, top_k=100, return_logprob=True)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    g = torch.cuda.CUDAGraph()
    buf = torch.zeros_like(logits)
    ub = torch.zeros_like(u)
    with torch.cuda.graph(g):
        out = sample(buf, ub, top_p=0.9, top_k=100, return_logprob=True)
    buf.copy_(logits)
    ub.copy_(u)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, out))


def test_settings_of_rows_in_other_types(sample):
    """Per-row settings count as fp32 and as whole numbers whatever their types; top_k below 1 keeps all, temperatures
    not above 0 are greedy."""
    B, V = 64, 3001
    logits, u = make(B, V, torch.bfloat16, seed=4)
    g = torch.Generator(device="cuda").manual_seed(2)
    pick = lambda vals, kind: torch.tensor(vals, device="cuda", dtype=kind)[torch.randint(0, len(vals), (B,), generator=g, device="cuda")]
    T, K = pick([0.0, 0.5, 1.0, -1.0], torch.float32), pick([-2, 0, 1, 13, 5000], torch.int32)
    P, M = pick([0.125, 0.875, 1.0], torch.float32), pick([0.0, 0.0625], torch.float32)
    want = check(sample, logits, u, T, K.clamp(min=0), P, M)
    for t, k, p, m in ((T, K, P, M), (T.double(), K.long(), P.double(), M.double()), (T.half(), K.short(), P.half(), M.bfloat16()),
                       (T, K, P, 0.0)):
        if torch.is_tensor(m):
            assert torch.equal(want, sample(logits, u, temperature=t, top_k=k, top_p=p, min_p=m))
        else:
            assert torch.equal(sample(logits, u, temperature=t, top_k=k, top_p=p, min_p=torch.zeros_like(M)),
                               sample(logits, u, temperature=t, top_k=k, top_p=p))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logits_further_apart_than_the_largest_number(sample, dtype):
    """Differences of logits beyond the largest fp32 number, at temperatures where such tokens keep weight: they lie at
    their places among the others."""
    V = 3000
    logits, u = make(6, V, dtype, seed=21)
    big = torch.finfo(torch.bfloat16).max
    steps = torch.linspace(-1, 1, 9, device="cuda")[torch.randint(0, 9, (6, V), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))]
    logits[:3] = (steps[:3] * big).to(dtype)
    logits[3, 5:9] = big
    logits[3, 20:900] = -big
    for T in (1e37, 2e38, float("inf")):
        for K, P, M in ((0, 0.3, 0.0), (0, 0.9, 0.0), (2000, 1.0, 0.0), (2000, 0.7, 0.0), (30, 0.9, 0.0), (0, 1.0, 0.2)):
            check(sample, logits, u, T, K, P, M)
