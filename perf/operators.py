"""Cases that measure three sets of operators against their plain forms.

linear attention   S_t = e^(d_h) S_(t-1) + k_t v_t^T,  o_t = scale S_t^T q_t  with one decay d_h <= 0
                   for each head: the whole sequence (prompts, with lengths and a carried state),
                   its gradients, and the single token that continues a state.
query / key norms  RMS norm of every head of q and k with the position rotation, and its gradients.
sampling           one token for each row of logits from a given uniform number, with temperature,
                   top-k, top-p and min-p.

``own`` chooses between the plain forms below (elementary torch operations in 32 bits, 64 where a
far position's angle or a value next to a border needs them) and the package's kernels.
"""
import math

import torch

own = False

# ---------------------------------------------------------------------------------------------
# cases


def listed():
    return [
        # a training-size prompt batch: enough (sequence, head) pairs to fill the GPU, final state kept for decoding
        dict(name="attn prompt 8x2048 h16 d128", op="attn", dtype="bf16", batch=8, seqlen=2048, heads=16, dk=128, dv=128,
             lengths=False, state=True),
        # one long prompt: few heads, so the work has to be split along the sequence
        dict(name="attn prompt 1x32768 h8 d128", op="attn", dtype="bf16", batch=1, seqlen=32768, heads=8, dk=128, dv=128,
             lengths=False, state=True),
        # a right-padded batch of prompts with odd sizes, an empty one and a one-token one among them
        dict(name="attn padded 5x777 h12 d96/160", op="attn", dtype="bf16", batch=5, seqlen=777, heads=12, dk=96, dv=160,
             lengths=True, state=True),
        # one training step of an attention layer, all gradients
        dict(name="attn train 4x2048 h16 d128", op="attn_train", dtype="bf16", batch=4, seqlen=2048, heads=16, dk=128,
             dv=128, lengths=False, state=False),
        # fp32 training with a carried state and padded rows, as gradient checks and small models run it
        dict(name="attn train f32 2x513 h4 d64", op="attn_train", dtype="fp32", batch=2, seqlen=513, heads=4, dk=64,
             dv=64, lengths=True, state=True),
        # decoding: one token of every sequence of a large serving batch; bound by the state's traffic
        dict(name="attn step 128 h16 d128", op="attn_step", dtype="bf16", batch=128, heads=16, dk=128, dv=128),
        # q and k of a prompt batch, fewer key heads than query heads
        dict(name="norm-rotate 8x2048 h16/4 d128", op="qk", dtype="bf16", batch=8, seqlen=2048, hq=16, hk=4, dim=128,
             rotary=128, interleaved=False),
        # its training step
        dict(name="norm-rotate train 4x2048 h16/16", op="qk_train", dtype="bf16", batch=4, seqlen=2048, hq=16, hk=16,
             dim=128, rotary=128, interleaved=False),
        # one token at far positions of a serving batch: launch latency counts
        dict(name="norm-rotate 32x1 h16/4 d128", op="qk", dtype="bf16", batch=32, seqlen=1, hq=16, hk=4, dim=128,
             rotary=64, interleaved=True),
        # one sequence's next token: latency counts
        dict(name="sample 1x50304", op="sample", dtype="fp32", batch=1, vocab=50304, temperature=0.8, top_k=50,
             top_p=0.95, min_p=0.0),
        # a serving batch whose rows each have their own settings (0 in the place of a setting: off, greedy for the temperature)
        dict(name="sample 256x50304 mixed", op="sample", dtype="bf16", batch=256, vocab=50304, temperature=-1.0, top_k=-1,
             top_p=-1.0, min_p=-1.0),
        # plain nucleus sampling over a wide vocabulary
        dict(name="sample 32x131072 top-p", op="sample", dtype="fp32", batch=32, vocab=131072, temperature=1.0, top_k=0,
             top_p=0.9, min_p=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn_train", "attn_step", "qk", "qk_train", "sample", "sample"])
    if op in ("attn", "attn_train"):
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
        dk, dv = 8 * rng.randint(4, 32), 8 * rng.randint(4, 32)
        heads = rng.randint(1, 16)
        small = dtype == "fp32" or op == "attn_train"
        tokens = _log(rng, 64, 2048 if small else 16384)
        batch = min(tokens, _log(rng, 1, 8))
        return dict(op=op, dtype=dtype, batch=batch, seqlen=max(1, tokens // batch), heads=heads, dk=dk, dv=dv,
                    lengths=rng.random() < 0.5, state=rng.random() < 0.5)
    if op == "attn_step":
        return dict(op=op, dtype=rng.choice(["bf16", "fp32"]), batch=_log(rng, 1, 128), heads=rng.randint(1, 16),
                    dk=8 * rng.randint(2, 16), dv=8 * rng.randint(2, 16))
    if op in ("qk", "qk_train"):
        dim = 8 * rng.randint(4, 32)
        hk = rng.randint(1, 8)
        tokens = _log(rng, 1, 8192)
        batch = min(tokens, _log(rng, 1, 32))
        return dict(op=op, dtype=rng.choice(["bf16", "fp32"]), batch=batch, seqlen=max(1, tokens // batch),
                    hq=hk * rng.randint(1, 2), hk=hk, dim=dim, rotary=rng.choice([0, 2 * rng.randint(1, dim // 2), dim]),
                    interleaved=rng.random() < 0.5)
    return dict(op=op, dtype=rng.choice(["bf16", "fp32"]), batch=_log(rng, 1, 128), vocab=_log(rng, 1000, 90000),
                temperature=rng.choice([0.7, 1.0, -1.0]), top_k=rng.choice([0, 1, 40, 500, -1]),
                top_p=rng.choice([0.0, 0.5, 0.95, -1.0]), min_p=rng.choice([0.0, 0.05, -1.0]))


# ---------------------------------------------------------------------------------------------
# inputs


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _dtype(case)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")
    unif = lambda *s: torch.rand(*s, generator=g, device="cuda")
    s = {"op": case["op"]}
    if case["op"] in ("attn", "attn_train", "attn_step"):
        B, H, dk, dv = case["batch"], case["heads"], case["dk"], case["dv"]
        # decays 1 - 2^-x from 1 - 2^-3 to 1 - 2^-10, spread over the heads
        x = 3 + 7 * (torch.arange(H, device="cuda") + unif(H)) / H
        s["log_decay"] = torch.log1p(-torch.exp2(-x)).float()
        s["scale"] = dk ** -0.5
        if case["op"] == "attn_step":
            s["q"], s["k"], s["v"] = rand(B, H, dk).to(dt), rand(B, H, dk).to(dt), rand(B, H, dv).to(dt)
            s["state"] = 4 * rand(B, H, dk, dv)
            return s
        L = case["seqlen"]
        s["q"], s["k"], s["v"] = rand(B, L, H, dk).to(dt), rand(B, L, H, dk).to(dt), rand(B, L, H, dv).to(dt)
        s["state"] = 2 * rand(B, H, dk, dv) if case["state"] else None
        s["lengths"] = None
        if case["lengths"]:
            n = (unif(B) * (L + 1)).floor().clamp(max=L).int()
            n[0] = L
            if B > 3:
                n[1], n[2] = 0, 1
            s["lengths"] = n
        if case["op"] == "attn_train":
            s["dout"] = rand(B, L, H, dv).to(dt)
            s["dstate"] = rand(B, H, dk, dv) if case["state"] else None
            for name in ("q", "k", "v") + (("state",) if case["state"] else ()):
                s[name].requires_grad_()
        return s
    if case["op"] in ("qk", "qk_train"):
        B, L, D = case["batch"], case["seqlen"], case["dim"]
        # q and k are column blocks of one projection's output
        width = (case["hq"] + case["hk"]) * D
        qk = (2 * rand(B, L, width)).to(dt)
        s["q"] = qk[..., :case["hq"] * D].unflatten(-1, (case["hq"], D))
        s["k"] = qk[..., case["hq"] * D:].unflatten(-1, (case["hk"], D))
        s["wq"], s["wk"] = 1 + 0.1 * rand(D), 1 + 0.1 * rand(D)
        s["positions"] = (unif(B, 1) * 100000).long() + torch.arange(L, device="cuda")
        s["rotary"], s["interleaved"] = case["rotary"], case["interleaved"]
        if case["op"] == "qk_train":
            s["dq"], s["dk"] = rand(B, L, case["hq"], D).to(dt), rand(B, L, case["hk"], D).to(dt)
            for name in ("q", "k", "wq", "wk"):
                s[name] = s[name].detach().requires_grad_()
        return s
    B, V = case["batch"], case["vocab"]
    logits = 2.5 * rand(B, V)
    # a model's rows: some spread out, some with a few tokens far above the others
    logits += torch.where(unif(B, V) < 20.0 / V, 6 + 3 * rand(B, V), torch.zeros((), device="cuda")) * (unif(B, 1) < 0.7)
    s["logits"] = logits.to(dt)
    s["uniforms"] = unif(B)
    pick = lambda values, kind: torch.tensor(values, device="cuda", dtype=kind)[(unif(B) * len(values)).long()]
    # a setting of -1: every row has its own
    s["temperature"] = (pick([0.0, 0.6, 0.8, 1.0, 1.3], torch.float32) if case["temperature"] < 0 else case["temperature"])
    s["top_k"] = pick([0, 1, 20, 50, 200], torch.int32) if case["top_k"] < 0 else case["top_k"]
    s["top_p"] = pick([1.0, 0.8, 0.9, 0.95, 0.99], torch.float32) if case["top_p"] < 0 else case["top_p"] or 1.0
    s["min_p"] = pick([0.0, 0.02, 0.1], torch.float32) if case["min_p"] < 0 else case["min_p"]
    return s


# ---------------------------------------------------------------------------------------------
# plain forms


def _powers(log_decay, steps):
    """e^(d_h n) for n of `steps` (int64), (H, ...), formed in 64 bits; n < 0 gives 0 and n = 0 gives 1."""
    e = torch.exp(log_decay.double().view(-1, *[1] * steps.dim()) * steps.clamp(min=1))
    return torch.where(steps > 0, e, (steps == 0).double()).float()


def _plain_attn(q, k, v, log_decay, scale, lengths, state):
    """Chunks of C steps: inside a chunk the masked product (q k^T * decay) v, and q times the state that enters the
    chunk, which is the decayed sum of the earlier chunks' k^T v."""
    B, L, H, dk = q.shape
    C = 64
    N = -(-L // C)
    t = torch.arange(N * C, device=q.device)
    n = torch.full((B,), L, device=q.device) if lengths is None else lengths.long()
    live = t < n.view(B, 1)                                                      # (B, N*C)

    def chunks(x):
        x = torch.nn.functional.pad(x.float(), (0, 0, 0, 0, 0, N * C - L))
        return torch.where(live[..., None, None], x, torch.zeros((), device=x.device)).permute(0, 2, 1, 3).unflatten(2, (N, C))

    qc, kc, vc = chunks(q), chunks(k), chunks(v)                                 # (B, H, N, C, d)
    i = torch.arange(C, device=q.device)
    c = torch.arange(N, device=q.device)
    inside = _powers(log_decay, i[:, None] - i[None, :])                         # (H, C, C)
    o = torch.matmul(torch.matmul(qc, kc.transpose(-1, -2)) * inside[:, None], vc)
    sums = torch.matmul((kc * _powers(log_decay, C - 1 - i)[:, None, :, None]).transpose(-1, -2), vc)  # (B, H, N, dk, dv)
    across = _powers(log_decay, (c[:, None] - 1 - c[None, :]) * C)               # (H, N, N): 0 at and above the diagonal
    enter = torch.matmul(across, sums.flatten(3)).view(sums.shape)
    if state is not None:
        enter = enter + _powers(log_decay, c * C)[:, :, None, None] * state.float()[:, :, None]
    o = o + torch.matmul(qc * _powers(log_decay, i + 1)[:, None, :, None], enter)
    o = (scale * o).flatten(2, 3)[:, :, :L].permute(0, 2, 1, 3)
    left = n.view(1, B, 1) - 1 - t                                               # steps from t to the row's last one
    w = torch.where(left[0] >= 0, _powers(log_decay, left[0]), torch.zeros((), device=q.device)).permute(1, 0, 2)  # (B, H, N*C)
    last = torch.matmul((kc.flatten(2, 3) * w[..., None]).transpose(-1, -2), vc.flatten(2, 3))
    if state is not None:
        last = last + _powers(log_decay, n).t()[:, :, None, None] * state.float()
    return o, last


def _plain_qk(q, k, wq, wk, positions, rotary, interleaved, eps=1e-6, base=10000.0):
    half = rotary // 2
    angle = positions.double()[..., None] * torch.pow(torch.tensor(base, dtype=torch.float64, device=q.device),
                                                     -torch.arange(half, device=q.device).double() / max(half, 1))
    cos, sin = torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]

    def one(x, w):
        x = x.float()
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w
        a, rest = y[..., :rotary], y[..., rotary:]
        x0, x1 = (a[..., 0::2], a[..., 1::2]) if interleaved else (a[..., :half], a[..., half:])
        r0, r1 = x0 * cos - x1 * sin, x1 * cos + x0 * sin
        r = torch.stack([r0, r1], -1).flatten(-2) if interleaved else torch.cat([r0, r1], -1)
        return torch.cat([r, rest], -1)

    return one(q, wq), one(k, wk)


def _plain_sample(logits, uniforms, temperature, top_k, top_p, min_p):
    """In 64 bits: a cumulative sum of weights is compared with borders."""
    B, V = logits.shape
    full = lambda x: (x if torch.is_tensor(x) else torch.full((B,), x, device=logits.device, dtype=torch.float32)).double()
    temperature, top_k, top_p, min_p = full(temperature), full(top_k), full(top_p), full(min_p)
    greedy = temperature <= 0
    x = logits.double() / torch.where(greedy, torch.ones_like(temperature), temperature)[:, None]
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)               # ties: the lowest token first
    w = torch.exp(x - x[:, :1])
    rank = torch.arange(V, device=logits.device)
    k = torch.where(greedy, torch.ones_like(top_k), torch.where(top_k > 0, top_k, torch.full_like(top_k, V)))
    w = torch.where(rank < k[:, None], w, torch.zeros_like(w))
    before = w.cumsum(-1) - w
    w = torch.where(before <= top_p[:, None] * w.sum(-1, keepdim=True), w, torch.zeros_like(w))
    w = torch.where(w >= min_p[:, None], w, torch.zeros_like(w))
    total = w.sum(-1)
    p = torch.zeros_like(w).scatter(1, order, w)                                 # in the order of the tokens
    over = p.cumsum(-1) > (uniforms.double() * total)[:, None]
    token = over.int().argmax(-1)
    return token, (p.gather(1, token[:, None])[:, 0] / total).log().float()


def run(state):
    s = state
    if s["op"] == "attn":
        if own:
            from hybrid_model_mamba_xlstm_b200.kernels import linear_attention
            return linear_attention(s["q"], s["k"], s["v"], s["log_decay"], scale=s["scale"], lengths=s["lengths"],
                                    initial_state=s["state"], return_final_state=True)
        o, last = _plain_attn(s["q"], s["k"], s["v"], s["log_decay"], s["scale"], s["lengths"], s["state"])
        return o.to(s["q"].dtype), last
    if s["op"] == "attn_train":
        leaves = [s["q"], s["k"], s["v"]] + ([s["state"]] if s["state"] is not None else [])
        if own:
            from hybrid_model_mamba_xlstm_b200.kernels import linear_attention
            out = linear_attention(s["q"], s["k"], s["v"], s["log_decay"], scale=s["scale"], lengths=s["lengths"],
                                   initial_state=s["state"], return_final_state=s["state"] is not None)
            o, last = out if s["state"] is not None else (out, None)
            outs, douts = ([o, last], [s["dout"], s["dstate"]]) if last is not None else ([o], [s["dout"]])
            return (o.detach(),) + torch.autograd.grad(outs, leaves, douts)
        wide = [x.detach().float().requires_grad_() for x in leaves]
        o, last = _plain_attn(*wide[:3], s["log_decay"], s["scale"], s["lengths"], wide[3] if len(wide) > 3 else None)
        outs, douts = ([o, last], [s["dout"].float(), s["dstate"]]) if len(wide) > 3 else ([o], [s["dout"].float()])
        grads = torch.autograd.grad(outs, wide, douts)
        return (o.detach().to(s["q"].dtype),) + tuple(d.to(x.dtype) for d, x in zip(grads, leaves))
    if s["op"] == "attn_step":
        if own:
            from hybrid_model_mamba_xlstm_b200.kernels import linear_attention_step
            return linear_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], scale=s["scale"]), s["state"]
        q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
        s["state"].copy_(torch.exp(s["log_decay"])[:, None, None] * s["state"] + k[..., None] * v[..., None, :])
        return (s["scale"] * torch.matmul(q[..., None, :], s["state"])[..., 0, :]).to(s["q"].dtype), s["state"]
    if s["op"] in ("qk", "qk_train"):
        if own:
            from hybrid_model_mamba_xlstm_b200.kernels import qk_norm_rope
            q, k = qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["positions"], rotary_dim=s["rotary"],
                                interleaved=s["interleaved"])
            if s["op"] == "qk":
                return q, k
            return (q.detach(), k.detach()) + torch.autograd.grad([q, k], [s["q"], s["k"], s["wq"], s["wk"]],
                                                                  [s["dq"], s["dk"]])
        if s["op"] == "qk":
            q, k = _plain_qk(s["q"], s["k"], s["wq"], s["wk"], s["positions"], s["rotary"], s["interleaved"])
            return q.to(s["q"].dtype), k.to(s["k"].dtype)
        wide = [s[n].detach().float().requires_grad_() for n in ("q", "k", "wq", "wk")]
        q, k = _plain_qk(*wide, s["positions"], s["rotary"], s["interleaved"])
        grads = torch.autograd.grad([q, k], wide, [s["dq"].float(), s["dk"].float()])
        dt = s["q"].dtype
        return (q.detach().to(dt), k.detach().to(dt), grads[0].to(dt), grads[1].to(dt), grads[2], grads[3])
    if own:
        from hybrid_model_mamba_xlstm_b200.kernels import sample_tokens
        return sample_tokens(s["logits"], s["uniforms"], temperature=s["temperature"], top_k=s["top_k"],
                             top_p=s["top_p"], min_p=s["min_p"], return_logprob=True)
    return _plain_sample(s["logits"], s["uniforms"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])


# ---------------------------------------------------------------------------------------------
# work and exact values


def work(case):
    """Every input read once and every output written once; the products of the step-by-step definition."""
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] in ("attn", "attn_train"):
        B, L, H, dk, dv = case["batch"], case["seqlen"], case["heads"], case["dk"], case["dv"]
        rows, states = B * L * H, B * H * dk * dv * 4
        # per step and head: k v^T into the state, and the state times q
        if case["op"] == "attn":
            return {"bytes": rows * (2 * dk + 2 * dv) * e + states * (2 if case["state"] else 1), "flops": 4 * rows * dk * dv}
        # gradients: the state again, its adjoint, and a product with one of them for each of dq, dk, dv
        return {"bytes": rows * (4 * dk + 4 * dv) * e + (3 * states if case["state"] else 0), "flops": 14 * rows * dk * dv}
    if case["op"] == "attn_step":
        B, H, dk, dv = case["batch"], case["heads"], case["dk"], case["dv"]
        return {"bytes": B * H * (8 * dk * dv + (2 * dk + 2 * dv) * e), "flops": 5 * B * H * dk * dv}
    if case["op"] in ("qk", "qk_train"):
        n = case["batch"] * case["seqlen"] * (case["hq"] + case["hk"]) * case["dim"]
        if case["op"] == "qk":
            return {"bytes": 2 * n * e + case["batch"] * case["seqlen"] * 8, "flops": 8 * n}
        return {"bytes": 4 * n * e + case["batch"] * case["seqlen"] * 8, "flops": 24 * n}
    n = case["batch"] * case["vocab"]
    return {"bytes": n * e + 16 * case["batch"], "flops": 4 * n}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"attn": _exact_attn, "attn_train": _exact_train, "attn_step": _exact_step, "qk": _exact_qk,
                "qk_train": _exact_qk, "sample": _exact_sample}[case["op"]](s)


def _exact_attn(s):
    """The recurrence, one step after another."""
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    B, L, H, dk = q.shape
    S = torch.zeros(B, H, dk, v.shape[-1], device=q.device, dtype=torch.float64)
    if s["state"] is not None:
        S += s["state"]
    f = s["log_decay"].double().exp().view(1, H, 1, 1)
    out = torch.zeros(B, L, H, v.shape[-1], device=q.device, dtype=torch.float64)
    rows = torch.arange(B, device=q.device)
    n = [L] * B if s["lengths"] is None else s["lengths"].tolist()
    cut = sorted(set([0] + n))
    for lo, hi in zip(cut, cut[1:]):  # the rows that are longer than `lo`
        r = torch.tensor([b for b in range(B) if n[b] > lo], device=q.device)
        T = S[r]
        for t in range(lo, hi):
            T.mul_(f).addcmul_(k[r, t][..., None], v[r, t][..., None, :])
            out[r, t] = torch.einsum("bhk,bhkv->bhv", q[r, t], T) * s["scale"]
        S[rows[r]] = T
    return out, S


def _exact_train(s):
    """All pairs of steps of one sequence at a time: W = e^(d (i - j)) for j <= i, A = scale W * (q k^T) and so on."""
    q, k, v, do = (s[n].detach().double().permute(0, 2, 1, 3) for n in ("q", "k", "v", "dout"))
    B, H, L, dk = q.shape
    if B * H * L * L > 2 ** 31:
        return None
    d, scale = s["log_decay"].double(), s["scale"]
    S0 = s["state"].detach().double() if s["state"] is not None else None
    dST = s["dstate"].double() if S0 is not None else None
    n = [L] * B if s["lengths"] is None else s["lengths"].tolist()
    o, dq, dkk, dv = (torch.zeros_like(x) for x in (v, q, k, v))
    dS0 = torch.zeros_like(S0) if S0 is not None else None
    for b in range(B):
        m = n[b]
        t = torch.arange(m, device=q.device, dtype=torch.float64)
        gap = t[:, None] - t[None, :]
        W = torch.where(gap >= 0, torch.exp(gap * d[:, None, None]), torch.zeros((), device=q.device, dtype=torch.float64))
        Q, K, V, G = q[b, :, :m], k[b, :, :m], v[b, :, :m], do[b, :, :m]
        A = scale * W * (Q @ K.transpose(-1, -2))
        E = scale * W * (G @ V.transpose(-1, -2))
        o[b, :, :m], dq[b, :, :m] = A @ V, E @ K
        dkk[b, :, :m], dv[b, :, :m] = E.transpose(-1, -2) @ Q, A.transpose(-1, -2) @ G
        if S0 is not None:
            since = torch.exp(d[:, None, None] * (t + 1)[:, None])               # (H, m, 1): decay from the first state to step t
            till = torch.exp(d[:, None, None] * (m - 1 - t)[:, None])            # from step t to the last state
            o[b, :, :m] += scale * since * (Q @ S0[b])
            dq[b, :, :m] += scale * since * (G @ S0[b].transpose(-1, -2))
            dkk[b, :, :m] += till * (V @ dST[b].transpose(-1, -2))
            dv[b, :, :m] += till * (K @ dST[b])
            dS0[b] = torch.exp(d * m)[:, None, None] * dST[b] + scale * (since * Q).transpose(-1, -2) @ G
    back = [x.permute(0, 2, 1, 3) for x in (o, dq, dkk, dv)]
    return tuple(back + ([dS0] if dS0 is not None else []))


def _exact_step(s):
    S = s["state"].double() * s["log_decay"].double().exp()[:, None, None]
    S = S + torch.einsum("bhk,bhv->bhkv", s["k"].double(), s["v"].double())
    return torch.einsum("bhk,bhkv->bhv", s["q"].double(), S) * s["scale"], S


def _exact_qk(s, eps=1e-6, base=10000.0):
    r = s["rotary"]
    pair = torch.arange(r // 2, device="cuda", dtype=torch.float64)
    angle = s["positions"].double()[:, :, None, None] * torch.exp(-math.log(base) * 2 * pair / max(r, 1))
    turn = torch.polar(torch.ones_like(angle), angle)                            # e^(i angle)

    def pairs(y):
        return y.unflatten(-1, (r // 2, 2)) if s["interleaved"] else y.unflatten(-1, (2, r // 2)).transpose(-1, -2)

    def flat(z):
        y = torch.view_as_real(z)
        return y.flatten(-2) if s["interleaved"] else y.transpose(-1, -2).flatten(-2)

    def rotated(y, by):
        if r == 0:
            return y
        z = torch.view_as_complex(pairs(y[..., :r]).contiguous()) * by
        return torch.cat([flat(z), y[..., r:]], -1)

    outs, grads, weights = [], [], []
    for x, w, g in ((s["q"], s["wq"], s.get("dq")), (s["k"], s["wk"], s.get("dk"))):
        x, w = x.detach().double(), w.detach().double()
        inv = 1 / torch.sqrt((x ** 2).mean(-1, keepdim=True) + eps)
        n = x * inv
        outs.append(rotated(n * w, turn))
        if g is not None:
            g = rotated(g.double(), turn.conj())                                 # the rotation's transpose
            weights.append((g * n).flatten(0, 2).sum(0))
            g = g * w
            grads.append(inv * (g - n * (g * n).mean(-1, keepdim=True)))
    return tuple(outs + grads + weights)


def _exact_sample(s):
    """Row by row on the host: tokens sorted by (logit down, token up), cut, then walked in the order of the tokens."""
    import numpy as np
    logits, u = s["logits"].double().cpu().numpy(), s["uniforms"].double().cpu().numpy()
    B, V = logits.shape
    per_row = lambda x: x.double().cpu().numpy() if torch.is_tensor(x) else np.full(B, np.float64(np.float32(x)))
    T, K, P, M = (per_row(s[n]) for n in ("temperature", "top_k", "top_p", "min_p"))
    tokens, logps = np.zeros(B, np.int64), np.zeros(B)
    for b in range(B):
        if T[b] <= 0:
            tokens[b] = int(np.argmax(logits[b]))
            continue
        order = np.argsort(-logits[b], kind="stable")
        if K[b] > 0:
            order = order[:int(K[b])]
        w = np.exp((logits[b][order] - logits[b][order[0]]) / T[b])
        sums = np.cumsum(w)
        keep = ((sums - w) <= P[b] * sums[-1]) & (w >= M[b])
        ids = np.sort(order[keep])
        w = np.exp((logits[b][ids] - logits[b].max()) / T[b])
        sums = np.cumsum(w)
        at = min(int(np.searchsorted(sums, u[b] * sums[-1], side="right")), len(ids) - 1)
        tokens[b], logps[b] = ids[at], np.log(w[at] / sums[-1])
    return torch.from_numpy(tokens), torch.from_numpy(logps)
