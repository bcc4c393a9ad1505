"""Reading a text: the linear attention over its tokens, and its score.

  prompt   gated linear attention over packed sequences of many tokens
  step     one token for each of a batch of sequences, their states in place
  loss     the log-likelihood of each token under the tied-embedding head
  grad     the same, and its gradients to the hidden states and the table

Linear attention, for a value head with key q_t, k_t, value v_t, decay a_t:

    S' = a_t S;  u = b_t (v_t - S'^T k_t)  (without b: u = v_t)
    S  = S' + k_t u^T;  o_t = scale S^T q_t

States are float32, a head's dim_k x dim_v matrix in the decode runtime's
blocks of 4 x 4 (qwen_kernels.h).  Sizes are the model's (16 heads of 128,
hidden 1024, vocabulary 65536, bf16 table) or generic.
"""
import math
import os
import sys

import torch

own = False


def _lib():
    """The library's Python side; only the calls of `own` use it."""
    p = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen35-ax7020-edge-llm_amd")
    if p not in sys.path:
        sys.path.insert(0, p)
    import qwen_kernels_gpu

    return qwen_kernels_gpu


def listed():
    model = {"heads_k": 16, "heads_v": 16, "dim_k": 128, "dim_v": 128}
    return [
        # decoding one sequence: the smallest call, all latency
        {"name": "step_1", "kind": "step", "batch": 1, "slots": 1, "delta": True, "type": "f32", **model},
        # serving many sequences: bound by the states' bytes
        {"name": "step_256", "kind": "step", "batch": 256, "slots": 256, "delta": True, "type": "bf16", **model},
        # a part of a pool of states, heads that share keys, no delta rule
        {"name": "step_pool", "kind": "step", "batch": 37, "slots": 64, "delta": False, "type": "f32",
         "heads_k": 4, "heads_v": 12, "dim_k": 64, "dim_v": 96},
        # a chat turn: one sequence of odd length
        {"name": "prompt_517", "kind": "prompt", "sequences": 1, "tokens": 517, "delta": True, "type": "bf16", **model},
        # a long document: one sequence, little to run side by side
        {"name": "prompt_16k", "kind": "prompt", "sequences": 1, "tokens": 16384, "delta": True, "type": "bf16", **model},
        # a prefill batch of ragged prompts in the runtime's own type, value heads sharing keys
        {"name": "prompt_ragged", "kind": "prompt", "sequences": 24, "tokens": 9001, "delta": True, "type": "f32",
         "heads_k": 8, "heads_v": 16, "dim_k": 128, "dim_v": 128},
        # decay alone (no delta rule), ragged
        {"name": "prompt_decay", "kind": "prompt", "sequences": 9, "tokens": 12345, "delta": False, "type": "bf16", **model},
        # scoring one more token: bound by the table's bytes
        {"name": "loss_1", "kind": "loss", "rows": 1, "vocab": 65536, "hidden": 1024, "ignored": 0.0, "type": "f32"},
        # perplexity of a text
        {"name": "loss_4096", "kind": "loss", "rows": 4096, "vocab": 65536, "hidden": 1024, "ignored": 0.0, "type": "bf16"},
        # an odd vocabulary, an odd width, a prompt whose own tokens do not count
        {"name": "loss_odd", "kind": "loss", "rows": 333, "vocab": 50001, "hidden": 1001, "ignored": 0.3, "type": "f32"},
        # fitting prompt vectors or a head on a few tokens: bound by the table and its gradient
        {"name": "grad_48", "kind": "grad", "rows": 48, "vocab": 65536, "hidden": 1024, "ignored": 0.1, "type": "f32"},
        # a training step's head
        {"name": "grad_4096", "kind": "grad", "rows": 4096, "vocab": 65536, "hidden": 1024, "ignored": 0.2, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("step", "prompt", "prompt", "loss", "grad"))
    c = {"kind": kind, "type": rng.choice(("f32", "bf16"))}
    if kind in ("step", "prompt"):
        heads = rng.choice(((16, 16), (16, 16), (8, 16), (4, 12), (2, 6), (1, 8), (5, 5)))
        dims = rng.choice(((128, 128), (128, 128), (64, 128), (64, 64), (4 * rng.randint(4, 32), 4 * rng.randint(4, 32)),
                           (256, 4 * rng.randint(8, 32))))
        c.update(delta=rng.random() < 0.6, heads_k=heads[0], heads_v=heads[1], dim_k=dims[0], dim_v=dims[1])
    if kind == "step":
        c["batch"] = _log(rng, 1, 256)
        c["slots"] = c["batch"] + rng.choice((0, rng.randint(1, 40)))
    elif kind == "prompt":
        c.update(sequences=_log(rng, 1, 32), tokens=_log(rng, 20, 12000))
    else:
        c.update(rows=_log(rng, 1, 4096), vocab=rng.choice((65536, _log(rng, 1000, 65536))),
                 hidden=rng.choice((1024, 1024, 8 * rng.randint(32, 128), rng.randint(256, 1024))),
                 ignored=rng.choice((0.0, round(rng.uniform(0.05, 0.9), 2))))
    return c


# ---- inputs, from the seed alone -------------------------------------------------------
_TYPE = {"f32": torch.float32, "bf16": torch.bfloat16}


def _lengths(case, seed):
    """Ragged lengths that add up to the case's tokens; some sequences may be empty."""
    n, total = case["sequences"], case["tokens"]
    g = torch.Generator().manual_seed(seed * 7 + 3)
    cuts = (torch.rand(n - 1, generator=g) * (total + 1)).long().clamp(0, total).sort().values.tolist()
    ends = cuts + [total]
    return [b - a for a, b in zip([0] + ends[:-1], ends)]


def _blocked(S):
    """[.., dim_k, dim_v] to the runtime's 4 x 4 blocks, flat: block (j / 4, i / 4), in it j % 4, then i % 4."""
    n, h, dk, dv = S.shape
    return S.reshape(n, h, dk // 4, 4, dv // 4, 4).permute(0, 1, 4, 2, 5, 3).reshape(n, h, dk * dv).contiguous()


def _unblocked(flat, dk, dv):
    n, h = flat.shape[:2]
    return flat.reshape(n, h, dv // 4, dk // 4, 4, 4).permute(0, 1, 3, 5, 2, 4).reshape(n, h, dk, dv)


def _attention_inputs(case, g, rows, states):
    """What the layers hand to the attention: q and k of a short convolution's
    silu, normalised; decays from nearly none to strong, by head; beta a sigmoid."""
    hk, hv, dk, dv, t = case["heads_k"], case["heads_v"], case["dim_k"], case["dim_v"], _TYPE[case["type"]]
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    silu = lambda x: x / (1 + (-x).exp())  # noqa: E731
    # one row of a projection holds q, k and v side by side
    qkv = torch.empty(rows, 2 * hk * dk + hv * dv, dtype=t, device="cuda")
    q = qkv[:, : hk * dk].view(rows, hk, dk)
    k = qkv[:, hk * dk : 2 * hk * dk].view(rows, hk, dk)
    v = qkv[:, 2 * hk * dk :].view(rows, hv, dv)
    for x in (q, k):
        y = silu(normal(rows, hk, dk))
        x.copy_(y / (y.square().sum(-1, keepdim=True) + 1e-6).sqrt())
    v.copy_(silu(normal(rows, hv, dv)))
    rate = torch.exp(torch.linspace(-6.0, 0.5, hv, device="cuda"))
    alpha = torch.exp(-rate * torch.log1p(torch.exp(normal(rows, hv))))
    beta = 1 / (1 + torch.exp(-normal(rows, hv))) if case["delta"] else None
    state = _blocked(0.1 * normal(states, hv, dk, dv))
    return {"q": q, "k": k, "v": v, "alpha": alpha, "beta": beta, "scale": dk ** -0.5, "state": state}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 17)
    s = {"case": case}
    if case["kind"] == "step":
        s.update(_attention_inputs(case, g, case["batch"], case["slots"]))
        s["slots"] = None
        if case["slots"] > case["batch"]:
            s["slots"] = torch.randperm(case["slots"], generator=g, device="cuda")[: case["batch"]].to(torch.int32)
    elif case["kind"] == "prompt":
        s.update(_attention_inputs(case, g, case["tokens"], case["sequences"]))
        ends = torch.tensor([0] + _lengths(case, seed)).cumsum(0)
        s["starts"] = ends.to(torch.int32).cuda()
        s["longest"] = int((ends[1:] - ends[:-1]).max())
    else:
        n, v, h = case["rows"], case["vocab"], case["hidden"]
        s["table"] = (0.03 * torch.randn(v, h, generator=g, device="cuda")).to(torch.bfloat16)
        s["h"] = (1.5 * torch.randn(n, h, generator=g, device="cuda")).to(_TYPE[case["type"]])
        s["targets"] = torch.randint(0, v, (n,), generator=g, device="cuda", dtype=torch.int32)
        drop = torch.randperm(n, generator=g, device="cuda")[: int(n * case["ignored"])]
        s["targets"][drop] = -100
        counted = max(1, n - int(n * case["ignored"]))
        s["grad_loss"] = torch.rand(n, generator=g, device="cuda") * 2 / counted
    return s


# ---- one pass ----------------------------------------------------------------------------
def _padded(s, t=torch.float32):
    """Each sequence's rows at [sequence, 0 ..], the gaps zero: q, k, v, decay, beta, and where each row went."""
    case, starts = s["case"], s["starts"].long()
    rows = torch.arange(case["tokens"], device="cuda")
    seq = torch.searchsorted(starts, rows, right=True) - 1
    at = (seq, rows - starts[seq])
    longest = -(-max(s["longest"], 1) // 64) * 64
    reach = case["heads_v"] // case["heads_k"]

    def pad(x, fill=0.0):
        y = torch.full((case["sequences"], longest, *x.shape[1:]), fill, dtype=t, device="cuda")
        y[at] = x.to(t)
        return y.movedim(1, 2)  # [sequence, head, token, ..]

    q, k = (pad(s[n].repeat_interleave(reach, 1)) for n in ("q", "k"))
    beta = None if s["beta"] is None else pad(s["beta"])
    return q, k, pad(s["v"]), pad(s["alpha"], 1.0), beta, at


def _plain_prompt(s):
    """Chunks of 64 tokens: within one, a triangular system; from one to the next, the state."""
    case, dk, dv, C = s["case"], s["case"]["dim_k"], s["case"]["dim_v"], 64
    q, k, v, alpha, beta, at = _padded(s)
    n, h, longest = q.shape[:3]
    cut = lambda x: x.reshape(n, h, longest // C, C, *x.shape[3:])  # noqa: E731
    q, k, v = cut(q), cut(k), cut(v)
    g = cut(alpha).double().log().cumsum(3)
    lower = torch.ones(C, C, device="cuda").tril().bool()
    decay = torch.where(lower, (g[..., :, None] - g[..., None, :]).clamp(max=0), float("-inf")).exp().float()
    up, down, last = g.exp().float(), (g[..., -1:] - g).exp().float(), g[..., -1].exp().float()
    P = (q @ k.transpose(-1, -2)) * decay
    if beta is not None:
        L = (k @ k.transpose(-1, -2)) * decay * cut(beta)[..., None] * ~torch.eye(C, device="cuda").bool()
        T = torch.zeros_like(L)
        for i in range(C):  # forward substitution, a row of every chunk at a time: (I + L) T = diag(beta)
            T[..., i, :] = -(L[..., i : i + 1, :i] @ T[..., :i, :])[..., 0, :]
            T[..., i, i] += cut(beta)[..., i]
    S = _unblocked(s["state"], dk, dv)
    O = torch.empty_like(v)
    for c in range(longest // C):  # the state goes from chunk to chunk
        kc, U = k[:, :, c], v[:, :, c]
        if beta is not None:
            U = T[:, :, c] @ (U - up[:, :, c, :, None] * (kc @ S))
        O[:, :, c] = up[:, :, c, :, None] * (q[:, :, c] @ S) + P[:, :, c] @ U
        S = last[:, :, c, None, None] * S + kc.transpose(-1, -2) @ (down[:, :, c, :, None] * U)
    O = O.reshape(n, h, longest, dv).movedim(2, 1)[at]
    return (s["scale"] * O).to(s["v"].dtype), _blocked(S)


def _plain_step(s, t=torch.float32):
    case, dk, dv = s["case"], s["case"]["dim_k"], s["case"]["dim_v"]
    slots = torch.arange(case["batch"], device="cuda") if s["slots"] is None else s["slots"].long()
    reach = case["heads_v"] // case["heads_k"]
    q, k = (s[n].to(t).repeat_interleave(reach, 1) for n in ("q", "k"))
    S = s["alpha"].to(t)[..., None, None] * _unblocked(s["state"][slots].to(t), dk, dv)
    u = s["v"].to(t)
    if s["beta"] is not None:
        u = s["beta"].to(t)[..., None] * (u - (S * k[..., None]).sum(-2))
    S = S + k[..., None] * u[..., None, :]
    out = s["scale"] * (S * q[..., None]).sum(-2)
    return out, slots, _blocked(S)


def _plain_loss(s):
    z = s["h"].float() @ s["table"].float().t()
    counted = s["targets"] >= 0
    top = z.amax(1, keepdim=True)
    lse = (z - top).exp().sum(1).log() + top[:, 0]
    at = z.gather(1, s["targets"].clamp(min=0).long()[:, None])[:, 0]
    return z, counted, torch.where(counted, lse - at, 0.0), torch.where(counted, lse, 0.0)


def run(s):
    kind = s["case"]["kind"]
    if own:
        qk = _lib()
        if kind == "prompt":
            return qk.linear_attention_prompt(s["q"], s["k"], s["v"], s["alpha"], s["beta"], s["starts"],
                                              scale=s["scale"], state_in=s["state"])
        if kind == "step":
            out = qk.linear_attention_step(s["q"], s["k"], s["v"], s["alpha"], s["beta"], s["state"],
                                           scale=s["scale"], slots=s["slots"])
            return out, s["state"]
        loss, lse = qk.lm_head_loss(s["h"], s["table"], s["targets"])
        if kind == "loss":
            return loss, lse
        return loss, *qk.lm_head_loss_grad(s["h"], s["table"], s["targets"], lse, s["grad_loss"])
    if kind == "prompt":
        return _plain_prompt(s)
    if kind == "step":
        out, slots, S = _plain_step(s)
        s["state"][slots] = S
        return out.to(s["v"].dtype), s["state"]
    z, counted, loss, lse = _plain_loss(s)
    if kind == "loss":
        return loss, lse
    D = (z - lse[:, None]).exp()
    D[torch.arange(len(D), device="cuda"), s["targets"].clamp(min=0).long()] -= 1
    D = torch.where(counted[:, None], D * s["grad_loss"][:, None], 0.0)
    return loss, (D @ s["table"].float()).to(s["h"].dtype), (D.t() @ s["h"].float()).to(torch.bfloat16)


# ---- 64 bits ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "step":
        out, slots, S = _exact_tokens(s, [torch.arange(case["batch"], device="cuda")],
                                      s["state"] if s["slots"] is None else s["state"][s["slots"].long()])
        state = s["state"].double()
        state[slice(None) if s["slots"] is None else s["slots"].long()] = S
        return out, state
    if case["kind"] == "prompt":
        starts = s["starts"].tolist()
        steps = [[a + i if a + i < b else -1 for a, b in zip(starts[:-1], starts[1:])] for i in range(s["longest"])]
        steps = list(torch.tensor(steps, device="cuda").reshape(s["longest"], -1))
        out, _, S = _exact_tokens(s, steps, s["state"])
        return out, S
    h, W, y = s["h"].double(), s["table"].double(), s["targets"].long()
    z = torch.mm(h, W.t())
    lse = torch.logsumexp(z, 1)
    p = torch.exp(z - lse[:, None])
    keep = (y >= 0).double()
    hot = torch.zeros_like(z).scatter_(1, y.clamp(min=0)[:, None], 1.0)
    loss = keep * (lse - (z * hot).sum(1))
    if case["kind"] == "loss":
        return loss, keep * lse
    D = (keep * s["grad_loss"].double())[:, None] * (p - hot)
    return loss, torch.mm(D, W), torch.mm(D.t(), h)


def _exact_tokens(s, steps, state):
    """The recurrence itself, token by token; steps[i][b] is sequence b's i-th row, or -1 past its end."""
    case, dk, dv = s["case"], s["case"]["dim_k"], s["case"]["dim_v"]
    of = torch.arange(case["heads_v"], device="cuda") // (case["heads_v"] // case["heads_k"])
    q, k, v, a = (s[n].double() for n in ("q", "k", "v", "alpha"))
    b = None if s["beta"] is None else s["beta"].double()
    out = torch.zeros(len(v) + 1, case["heads_v"], dv, dtype=torch.float64, device="cuda")
    S = state.double().view(-1, case["heads_v"], dv // 4, dk // 4, 4, 4).permute(0, 1, 2, 4, 3, 5)
    S = S.reshape(-1, case["heads_v"], dv, dk).clone()  # transposed: a row for each value
    for rows in steps:
        r = rows.clamp(min=0)
        kk, qq = k[r][:, of], q[r][:, of]
        N = S * a[r][..., None, None]
        u = v[r]
        if b is not None:
            u = (u - torch.matmul(N, kk[..., None])[..., 0]) * b[r][..., None]
        N = N + u[..., None] * kk[..., None, :]
        out[rows] = s["scale"] * torch.matmul(N, qq[..., None])[..., 0]  # row -1 is spare
        S = torch.where((rows >= 0)[:, None, None, None], N, S)
    n, h = S.shape[:2]
    S = S.reshape(n, h, dv // 4, 4, dk // 4, 4).permute(0, 1, 2, 4, 3, 5).reshape(n, h, dk * dv)
    return out[:-1], None, S


def work(case):
    es = 4 if case["type"] == "f32" else 2
    if case["kind"] in ("step", "prompt"):
        rows = case["batch" if case["kind"] == "step" else "tokens"]
        states = case["batch" if case["kind"] == "step" else "sequences"]
        hk, hv, dk, dv = case["heads_k"], case["heads_v"], case["dim_k"], case["dim_v"]
        row = es * (2 * hk * dk + 2 * hv * dv) + 4 * hv * (2 if case["delta"] else 1)
        return {"bytes": rows * row + 8 * states * hv * dk * dv, "flops": rows * hv * dk * dv * (6 if case["delta"] else 4)}
    n, v, h = case["rows"], case["vocab"], case["hidden"]
    counted = n - int(n * case["ignored"])
    if case["kind"] == "loss":
        return {"bytes": 2 * v * h + es * counted * h + 12 * n, "flops": 2 * counted * v * h}
    return {"bytes": 4 * v * h + es * (counted + n) * h + 12 * n, "flops": 6 * counted * v * h}
