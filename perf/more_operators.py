"""A full-attention layer's operators: rotary positions, a paged cache of keys and values, and the
attention over it.

  rotary, rotary_grad   positions rotated into queries and keys, and the gradient
  append                a call's keys and values to the cache, keys and queries rotated on the way
  step, prompt          the attention: one token for each sequence, or many (causal)
  tree                  drafted tokens that share a sequence's cache, each seeing its own ancestors

For pair i of a head's first rot elements at position p, angle t = p f_i:

    a' = A (a cos t - b sin t);  b' = A (a sin t + b cos t)

Attention of a row's head h, on key head h / (heads_q / heads_k), over the keys j that it sees:

    o = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale q . k_j)

The cache is pages x page x heads_k x dim, a sequence's pages in its row of a table.  Sizes are the
model's (8 query heads on 2 key heads of 256, pages of 16 tokens, 64 elements rotated) or generic.
"""
import math
import os
import random
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
    model = {"heads_q": 8, "heads_k": 2, "dim": 256, "page": 16}
    turn = {"rot": 64, "interleaved": False}
    return [
        # decoding: the query and key heads of one token, all latency
        {"name": "rotary_1", "kind": "rotary", "rows": 1, "heads": 10, "dim": 256, **turn, "far": 4096, "amplitude": 1.0,
         "type": "f32"},
        # a long document's queries and keys, far positions, frequencies stretched for long contexts
        {"name": "rotary_16k", "kind": "rotary", "rows": 16384, "heads": 10, "dim": 256, **turn, "far": 262144,
         "amplitude": 1.1386, "type": "bf16"},
        # training: the gradient, neighbours as pairs, whole heads
        {"name": "rotary_grad", "kind": "rotary_grad", "rows": 5003, "heads": 12, "dim": 96, "rot": 96,
         "interleaved": True, "far": 5003, "amplitude": 1.0, "type": "f32"},
        # decoding one sequence in the runtime's own type
        {"name": "append_1", "kind": "append", "sequences": 1, "tokens": 1, "cached": 700, **model, **turn, "type": "f32"},
        # a prefill batch of ragged prompts, some of them continued
        {"name": "append_9001", "kind": "append", "sequences": 24, "tokens": 9001, "cached": 6000, **model, **turn,
         "type": "bf16"},
        # decoding one sequence: little to run side by side
        {"name": "step_1", "kind": "step", "sequences": 1, "tokens": 1, "cached": 4096, **model, "type": "bf16"},
        # serving many sequences of ragged lengths: bound by the cache's bytes
        {"name": "step_64", "kind": "step", "sequences": 64, "tokens": 64, "cached": 262144, **model, "type": "bf16"},
        # the runtime's own type, other heads, pages that tiles of keys do not end with
        {"name": "step_f32", "kind": "step", "sequences": 7, "tokens": 7, "cached": 10007, "heads_q": 12, "heads_k": 4,
         "dim": 64, "page": 24, "type": "f32"},
        # checking one sequence's drafted tree
        {"name": "tree_1", "kind": "tree", "sequences": 1, "tokens": 26, "cached": 6001, **model, "type": "bf16"},
        # checking the drafts of a batch, ragged trees
        {"name": "tree_48", "kind": "tree", "sequences": 48, "tokens": 1500, "cached": 100000, "heads_q": 16, "heads_k": 4,
         "dim": 128, "page": 16, "type": "bf16"},
        # a long document: bound by the matrix cores
        {"name": "prompt_16k", "kind": "prompt", "sequences": 1, "tokens": 16384, "cached": 0, **model, "type": "bf16"},
        # a batch of prompts that go on from cached turns, in the runtime's own type, an odd width
        {"name": "prompt_ragged", "kind": "prompt", "sequences": 9, "tokens": 3001, "cached": 5000, "heads_q": 6,
         "heads_k": 2, "dim": 80, "page": 16, "type": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("rotary", "rotary_grad", "append", "step", "step", "tree", "prompt", "prompt"))
    c = {"kind": kind, "type": rng.choice(("f32", "bf16", "bf16"))}
    dim = rng.choice((64, 128, 128, 256, 256, 8 * rng.randint(4, 32)))
    turn = {"rot": rng.choice((dim, dim // 4 // 2 * 2, 2 * rng.randint(2, dim // 2))), "interleaved": rng.random() < 0.4}
    if kind in ("rotary", "rotary_grad"):
        c.update(rows=_log(rng, 1, 16384), heads=_log(rng, 1, 16), dim=dim, **turn, far=_log(rng, 16, 1 << 20),
                 amplitude=rng.choice((1.0, round(rng.uniform(0.7, 1.5), 4))))
        return c
    heads = rng.choice(((8, 2), (8, 2), (8, 8), (16, 4), (6, 2), (12, 4), (5, 1), (16, 1), (3, 3)))
    c.update(heads_q=heads[0], heads_k=heads[1], dim=dim, page=rng.choice((16, 16, 16, 32, 64, 128, rng.randint(1, 100))))
    if kind == "append":
        n = _log(rng, 1, 32)
        c.update(sequences=n, tokens=_log(rng, n, 12000), cached=rng.choice((0, _log(rng, 1, 12000))), **turn)
    elif kind == "step":
        n = _log(rng, 1, 64)
        c.update(sequences=n, tokens=n, cached=n * _log(rng, 1, 4000))
    elif kind == "tree":
        n = _log(rng, 1, 48)
        c.update(sequences=n, tokens=n * _log(rng, 2, 48), cached=n * _log(rng, 1, 2500))
    else:
        c.update(sequences=_log(rng, 1, 24), tokens=_log(rng, 2, 8000), cached=rng.choice((0, _log(rng, 1, 8000))))
    return c


# ---- inputs, from the seed alone (lengths and trees from the case) -----------------------
_TYPE = {"f32": torch.float32, "bf16": torch.bfloat16}


def _ragged(rng, n, total, least):
    """n lengths of at least `least` that add up to total (as near as that allows)."""
    spare = max(0, total - n * least)
    cuts = sorted(rng.randint(0, spare) for _ in range(n - 1))
    return [least + b - a for a, b in zip([0] + cuts, cuts + [spare])]


def _shape(case):
    """-> each sequence's new tokens, cached tokens, and the parents of a tree's."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    n = case["sequences"]
    if case["kind"] == "step":
        new = [1] * n
    else:
        new = _ragged(rng, n, case["tokens"], 1 if case["kind"] == "tree" else 0)
    cached = _ragged(rng, n, case["cached"], 0)
    rng.shuffle(cached)
    parents = []
    for k in new if case["kind"] == "tree" else ():
        # a draft's best continuations are drafted further: parents are mostly late nodes, some start afresh
        parents += [max(-1, i - 1 - int(rng.expovariate(1 / (1 + i / 3)))) for i in range(k)]
    return new, cached, parents


def _freqs(rot, stretched):
    """Radians a position, each pair's; stretched: the slow half at a quarter, as for a context four times as long."""
    f = torch.tensor(1e7, dtype=torch.float64) ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if stretched:
        f[len(f) // 2 :] /= 4
    return f.cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 29)
    t = _TYPE[case["type"]]
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    s = {"case": case}
    if case["kind"] in ("rotary", "rotary_grad"):
        s["x"] = normal(case["rows"], case["heads"], case["dim"]).to(t)
        first = torch.randint(0, case["far"], (case["rows"],), generator=g, device="cuda")
        s["positions"] = first.to(torch.int32)
        s["freqs"] = _freqs(case["rot"], case["amplitude"] != 1.0)
        return s
    hq, hk, dim, page, n = (case[k] for k in ("heads_q", "heads_k", "dim", "page", "sequences"))
    new, cached, parents = _shape(case)
    rows, total = sum(new), [a + b for a, b in zip(new, cached)]
    need = [-(-x // page) for x in total]
    pages = sum(need) + 3  # some of the pool is other sequences'
    wide = max(max(need), 1)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    tables, at = torch.full((n, wide), -1, dtype=torch.int32), 0
    order = order.cpu()
    for i, k in enumerate(need):
        tables[i, :k] = order[at : at + k]
        at += k
    s["tables"] = tables.cuda()
    s["cached"] = torch.tensor(cached, dtype=torch.int32).cuda()
    ends = torch.tensor([0] + new).cumsum(0)
    s["starts"] = ends.to(torch.int32).cuda()
    s["longest"], s["rows"] = max(new), rows
    s["key_cache"] = normal(pages, page, hk, dim).to(t)
    s["value_cache"] = normal(pages, page, hk, dim).to(t)
    # queries that look hard at some keys: scores of a standard deviation of 1.5
    if case["kind"] == "append":
        qkv = normal(rows, (hq + 2 * hk) * dim).to(t)  # one projection's rows
        s["q"] = qkv[:, : hq * dim].view(rows, hq, dim)
        s["k"] = qkv[:, hq * dim : (hq + hk) * dim].view(rows, hk, dim)
        s["v"] = qkv[:, (hq + hk) * dim :].view(rows, hk, dim)
        s["freqs"] = _freqs(case["rot"], False)
        return s
    s["q"] = (1.5 * normal(rows, hq, dim)).to(t)
    s["scale"] = dim ** -0.5
    if parents:
        s["parents"] = torch.tensor(parents, dtype=torch.int32).cuda()
    if own:  # a serving program keeps its workspace
        qk = _lib()
        need = qk.paged_attention_work_bytes(rows, n, hq, hk, dim, t)
        s["work"] = torch.empty(need, dtype=torch.uint8, device="cuda")
    return s


# ---- one pass ----------------------------------------------------------------------------
def _plain_rotary(x, positions, freqs, interleaved, amplitude, back=False):
    rot = 2 * len(freqs)
    angle = (positions.double()[:, None] * freqs)[:, None, :]
    c, n = (amplitude * angle.cos()).float(), (amplitude * angle.sin()).float()
    if back:
        n = -n
    y = x.float().clone()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    u, w = x[..., a].float(), x[..., b].float()
    y[..., a], y[..., b] = u * c - w * n, u * n + w * c
    return y.to(x.dtype)


def _owner(s):
    """Each row's sequence and its place in it."""
    starts, rows = s["starts"].long(), torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(starts, rows, right=True) - 1
    return seq, rows - starts[seq]


def _plain_append(s):
    case = s["case"]
    seq, i = _owner(s)
    place = s["cached"].long()[seq] + i
    page, slot = s["tables"].long()[seq, place // case["page"]], place % case["page"]
    turn = (s["freqs"], case["interleaved"], 1.0)
    s["key_cache"][page, slot] = _plain_rotary(s["k"], place, *turn)
    s["value_cache"][page, slot] = s["v"]
    return _plain_rotary(s["q"], place, *turn), s["key_cache"], s["value_cache"]


def _plain_tree(s):
    """Each row's ancestors as bits, and its position."""
    words = -(-s["longest"] // 32)
    seq, i = _owner(s)
    first = s["starts"].long()[seq]
    bits = torch.zeros(s["rows"], words * 32, dtype=torch.bool, device="cuda")
    bits[torch.arange(s["rows"], device="cuda"), i] = True
    depth, up = torch.zeros_like(i), s["parents"].long()
    for _ in range(s["longest"] - 1):  # a generation at a time
        live = up >= 0
        bits |= live[:, None] & (torch.arange(words * 32, device="cuda") == up[:, None])
        depth += live
        up = torch.where(live, s["parents"].long()[(first + up).clamp(min=0)], up)
    value = (bits.view(-1, words, 32).long() << torch.arange(32, device="cuda")).sum(2)
    mask = torch.where(value >= 1 << 31, value - (1 << 32), value).to(torch.int32)
    return bits, mask, (s["cached"].long()[seq] + depth).to(torch.int32)


def _plain_sequences(s, many, bits=None):
    """Sequences `many` side by side, padded to the longest."""
    case = s["case"]
    hq, hk, dim, page = (case[k] for k in ("heads_q", "heads_k", "dim", "page"))
    new, cached, _ = _shape(case)
    n, most = max(new[m] for m in many), max(new[m] + cached[m] for m in many)
    first = [sum(new[:m]) for m in many]
    at = torch.arange(most, device="cuda")
    which = torch.tensor(many, device="cuda")
    pages = s["tables"].long()[which][:, at // page].clamp(min=0)
    K, V = (s[c][pages, at % page].float().transpose(1, 2) for c in ("key_cache", "value_cache"))  # [sequence, head, key, dim]
    held = torch.tensor([cached[m] for m in many], device="cuda")[:, None]
    count = torch.tensor([new[m] for m in many], device="cuda")[:, None]
    i = torch.arange(n, device="cuda")
    rows = (torch.tensor(first, device="cuda")[:, None] + i).clamp(max=s["rows"] - 1)
    q = s["q"][rows].float().view(len(many), n, hk, hq // hk, dim).permute(0, 2, 3, 1, 4).reshape(len(many), hk, -1, dim)
    if bits is None:
        sees = at <= (held + i)[..., None]
    else:
        drafted = at[None] - held  # [sequence, key]
        sees = (drafted < 0)[:, None] | (drafted >= 0)[:, None] & torch.gather(
            bits[rows], 2, drafted.clamp(0, bits.shape[1] - 1)[:, None].expand(-1, n, -1))
        sees = sees & (drafted < count)[:, None]
    z = (q @ K.transpose(2, 3).contiguous()).view(len(many), hk, hq // hk, n, most)
    z = (z * s["scale"]).masked_fill_(~sees[:, None, None], float("-inf"))
    w = z.sub_(z.amax(-1, keepdim=True)).exp_()
    total = w.sum(-1, keepdim=True)
    o = (w.view(len(many), hk, -1, most) @ V.contiguous()).view(len(many), hk, hq // hk, n, dim) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(len(many), n, hq, dim)
    return o[i < count].to(s["q"].dtype)


def _plain_attention(s, bits=None):
    new, _, _ = _shape(s["case"])
    if s["case"]["kind"] == "prompt":  # long ones one by one
        return torch.cat([_plain_sequences(s, [m]) for m, n in enumerate(new) if n])
    return _plain_sequences(s, list(range(len(new))), bits)


def run(s):
    case, kind = s["case"], s["case"]["kind"]
    if own:
        qk = _lib()
        if kind in ("rotary", "rotary_grad"):
            f = qk.rotary if kind == "rotary" else qk.rotary_grad
            return f(s["x"], s["positions"], s["freqs"], interleaved=case["interleaved"], amplitude=case["amplitude"])
        cache = (s["key_cache"], s["value_cache"], s["tables"], s["cached"])
        if kind == "append":
            q = qk.kv_cache_append(s["k"], s["v"], *cache, s["starts"], freqs=s["freqs"],
                                   interleaved=case["interleaved"], q=s["q"])
            return q, s["key_cache"], s["value_cache"]
        if kind == "step":
            return qk.paged_attention(s["q"], *cache, scale=s["scale"], work=s["work"])
        if kind == "prompt":
            return qk.paged_attention(s["q"], *cache, s["starts"], scale=s["scale"], work=s["work"])
        mask, positions = qk.draft_tree(s["parents"], s["cached"], s["starts"], longest=s["longest"])
        return qk.paged_attention(s["q"], *cache, s["starts"], scale=s["scale"], mask=mask, work=s["work"]), mask, positions
    if kind in ("rotary", "rotary_grad"):
        return _plain_rotary(s["x"], s["positions"], s["freqs"], case["interleaved"], case["amplitude"], kind == "rotary_grad")
    if kind == "append":
        return _plain_append(s)
    if kind == "tree":
        bits, mask, positions = _plain_tree(s)
        return _plain_attention(s, bits), mask, positions
    return _plain_attention(s)


# ---- 64 bits ---------------------------------------------------------------------------
def _exact_rotation(x, positions, freqs, interleaved, amplitude):
    """As a product with each row's rotation of the complex plane."""
    x, half = x.double().clone(), len(freqs)
    turn = torch.polar(torch.full((len(x), half), amplitude, dtype=torch.float64, device="cuda"),
                       positions.double()[:, None] * freqs[None])
    part = x[..., : 2 * half]
    pairs = part.unflatten(-1, (half, 2)) if interleaved else part.unflatten(-1, (2, half)).movedim(-2, -1)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn[:, None])
    x[..., : 2 * half] = z.flatten(-2) if interleaved else z.movedim(-1, -2).flatten(-2)
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("rotary", "rotary_grad"):
        sign = 1.0 if case["kind"] == "rotary" else -1.0
        return _exact_rotation(s["x"], s["positions"], sign * s["freqs"], case["interleaved"], case["amplitude"])
    new, cached, parents = _shape(case)
    hq, hk, page = case["heads_q"], case["heads_k"], case["page"]
    tables = s["tables"].tolist()
    first = [sum(new[:m]) for m in range(len(new))]
    places = [[(tables[m][j // page], j % page) for j in range(cached[m] + new[m])] for m in range(len(new))]
    if case["kind"] == "append":
        positions = torch.tensor([c + i for n, c in zip(new, cached) for i in range(n)], device="cuda")
        at = torch.tensor([p for m, c in enumerate(cached) for p in places[m][c:]], device="cuda").reshape(-1, 2)
        K, V = s["key_cache"].double(), s["value_cache"].double()
        K[at[:, 0], at[:, 1]] = _exact_rotation(s["k"], positions, s["freqs"], case["interleaved"], 1.0)
        V[at[:, 0], at[:, 1]] = s["v"].double()
        return _exact_rotation(s["q"], positions, s["freqs"], case["interleaved"], 1.0), K, V
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for m, (n, c) in enumerate(zip(new, cached)):
        if not n:
            continue
        at = torch.tensor(places[m], device="cuda")
        K, V = (s[x][at[:, 0], at[:, 1]].double() for x in ("key_cache", "value_cache"))
        hidden = torch.ones(n, c + n, dtype=torch.bool).tril(c).logical_not()
        if parents:
            hidden[:, c:] = True
            for i in range(n):
                j = i
                while j >= 0:
                    hidden[i, c + j] = False
                    j = parents[first[m] + j]
        hidden = hidden.cuda()
        for h in range(hq):
            z = torch.mm(s["q"][first[m] : first[m] + n, h].double(), K[:, h // (hq // hk)].t()) * s["scale"]
            z[hidden] = -math.inf
            out[first[m] : first[m] + n, h] = torch.mm(torch.softmax(z, 1), V[:, h // (hq // hk)])
    return (out, None, None) if parents else out


def _pairs(case):
    """Pairs of a query and a key that it sees."""
    new, cached, parents = _shape(case)
    if case["kind"] != "tree":
        return sum(n * c + n * (n + 1) // 2 for n, c in zip(new, cached))
    seen, at = 0, 0
    for n, c in zip(new, cached):
        deep = []
        for p in parents[at : at + n]:
            deep.append(1 + (deep[p] if p >= 0 else 0))
        seen += n * c + sum(deep)
        at += n
    return seen


def work(case):
    es = 4 if case["type"] == "f32" else 2
    if case["kind"] in ("rotary", "rotary_grad"):
        n = case["rows"] * case["heads"]
        return {"bytes": n * case["dim"] * 2 * es + 4 * case["rows"] + 4 * case["rot"], "flops": 3 * n * case["rot"]}
    hq, hk, dim = case["heads_q"], case["heads_k"], case["dim"]
    new, cached, _ = _shape(case)
    rows = sum(new)
    if case["kind"] == "append":
        return {"bytes": rows * 2 * es * dim * (hq + 2 * hk) + 4 * rows, "flops": 3 * rows * case["rot"] * (hq + hk)}
    keys = sum(c + n for n, c in zip(new, cached) if n)
    return {"bytes": 2 * es * dim * (hk * keys + hq * rows) + 4 * (keys // case["page"] + len(new)),
            "flops": 4 * dim * hq * _pairs(case)}
