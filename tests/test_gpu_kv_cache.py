"""Rotary positions, the paged cache's append and drafted tokens' masks on the GPU, against 64 bits; and a
layer's steps together.

Tolerances of a rotated pair (x, y).  The angle as half turns of at most 1 is rounded to float32, 2^-25 half turns of
pi: 1.6 x 2^-24; sine and cosine are taken to be off by 2 steps (4 x 2^-24), the amplitude, the two products
and the sum round by 2^-24 each: 10 x 2^-24 of amplitude (|x| + |y|).  The angle itself, a double, is off by
3 x 2^-53 of itself: 2^31 positions of one radian, 2^-20.4.  bf16 results add half a step, 2^-8 of the value."""
import pytest
import torch

from test_gpu_paged_attention import near as attention_near
from test_gpu_paged_attention import oracle as attention

pytestmark = pytest.mark.gpu
F, BF16 = torch.float32, torch.bfloat16


def freqs_of(rot, base=10000.0):
    return torch.tensor(base, dtype=torch.float64) ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)


def rotated(x, positions, freqs, interleaved, amplitude=1.0, back=False):
    """-> (result, |x| + |y| of each element's pair), 64 bits on the CPU."""
    x = x.double().cpu()
    t = positions.double().cpu()[:, None, None] * freqs.double().cpu()
    c, s = amplitude * torch.cos(t), amplitude * torch.sin(t) * (-1 if back else 1)
    rot = 2 * len(freqs)
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    out, size = x.clone(), torch.zeros_like(x)
    out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    size[..., a] = size[..., b] = abs(amplitude) * (x[..., a].abs() + x[..., b].abs())
    return out, size


def near(got, want, size, far=0.0):
    dtype = got.dtype
    got = got.double().cpu()
    bound = size * (10 * 2.0 ** -24 + far * 3 * 2.0 ** -53)
    if dtype == BF16:
        bound = bound + want.abs() * 2.0 ** -8
    off = (got - want).abs()
    assert bool((off <= bound).all()), float((off - bound).max())


SHAPES = [(10, 256, 64), (3, 96, 96), (1, 64, 16), (5, 80, 22), (2, 7, 4), (4, 130, 2), (1, 1024, 1024), (16, 128, 120)]


@pytest.mark.parametrize("dtype", [F, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,dim,rot", SHAPES)
def test_rotary(gpu, heads, dim, rot, interleaved, dtype):
    f = freqs_of(rot)
    for rows in (1, 37, 2051):
        g = torch.Generator().manual_seed(rows)
        wide = torch.randn(rows, heads, dim + (3 if rows == 37 else 0), generator=g).to(dtype).cuda()
        x = wide[..., :dim]  # (37 rows: three elements apart)
        keep = x.clone()
        positions = torch.randint(-10, 5000, (rows,), generator=g).to(torch.int32).cuda()
        out = gpu.rotary(x, positions, f.cuda(), interleaved=interleaved, amplitude=1.25)
        near(out, *rotated(keep, positions, f, interleaved, 1.25), far=5000)
        assert torch.equal(out[..., rot:], keep[..., rot:]) and torch.equal(x, keep)
        grad = gpu.rotary_grad(x, positions, f.cuda(), interleaved=interleaved, amplitude=1.25)
        near(grad, *rotated(keep, positions, f, interleaved, 1.25, back=True), far=5000)
        assert gpu.rotary(x, positions, f.cuda(), interleaved=interleaved, amplitude=1.25, out=x) is x
        assert torch.equal(x, out)
        if rows == 37:
            assert torch.equal(wide[..., dim:], torch.randn(rows, heads, dim + 3, generator=torch.Generator().manual_seed(37))
                               .to(dtype).cuda()[..., dim:])


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_gradient_against_differences(gpu, interleaved):
    """sum(w . rotary(x)) changes by grad . dx; the operator is linear, so that any step does."""
    g = torch.Generator().manual_seed(5)
    x, dx, w = (torch.randn(9, 2, 24, generator=g).cuda() for _ in range(3))
    positions = torch.randint(0, 1 << 20, (9,), generator=g).to(torch.int32).cuda()
    f = freqs_of(16).cuda()
    call = lambda y: gpu.rotary(y, positions, f, interleaved=interleaved, amplitude=0.75).double()  # noqa: E731
    grad = gpu.rotary_grad(w, positions, f, interleaved=interleaved, amplitude=0.75).double()
    change = (w.double() * (call(x + dx) - call(x))).sum((1, 2))
    want = (grad * ((x + dx).double() - x.double())).sum((1, 2))
    # 48 products of magnitudes up to about 4 x 8, each off by 10 x 2^-24 of them, on both sides
    assert bool(((change - want).abs() <= 2 * 48 * 32 * 10 * 2.0 ** -24).all())


def test_rotary_far_positions(gpu):
    """Angles of up to 2^31 radians, of either sign; a float32 angle would be off by whole turns."""
    x = torch.randn(6, 3, 8, generator=torch.Generator().manual_seed(1)).cuda()
    positions = torch.tensor([2 ** 31 - 1, -(2 ** 31), 2 ** 24 + 1, 1 << 20, -(1 << 20), 0], dtype=torch.int32).cuda()
    f = freqs_of(8)
    near(gpu.rotary(x, positions, f.cuda()), *rotated(x, positions, f, False), far=2.0 ** 31)
    # NaN and infinity stay within their pair
    x[3, 1, 2] = float("nan")
    x[4, 2, 1] = float("inf")
    out = gpu.rotary(x, positions, f.cuda())
    odd = ~torch.isfinite(out)
    assert odd.sum() == 4 and bool(odd[3, 1, [2, 6]].all()) and bool(odd[4, 2, [1, 5]].all())


def test_rotary_strides_and_empty(gpu):
    f = freqs_of(32).cuda()
    x = torch.randn(4, 50, 64, generator=torch.Generator().manual_seed(2)).cuda().transpose(0, 1)  # heads before rows
    positions = torch.arange(50, dtype=torch.int32).cuda()
    near(gpu.rotary(x, positions, f), *rotated(x, positions, f, False), far=50)
    one = x[:1, :1].expand(50, 4, 64)  # one head read by all
    near(gpu.rotary(one, positions, f), *rotated(one, positions, f, False), far=50)
    assert gpu.rotary(x[:0], positions[:0], f).shape == (0, 4, 64)
    for bad in (lambda: gpu.rotary(x, positions, f, out=torch.empty(50, 4, 64, device="cuda")[:1].expand(50, 4, 64)),
                lambda: gpu.rotary(x, positions, freqs_of(66).cuda()), lambda: gpu.rotary(x, positions, f[:0]),
                lambda: gpu.rotary(x, positions, f, amplitude=float("nan"))):
        with pytest.raises(RuntimeError):
            bad()
    for bad in (lambda: gpu.rotary(x, positions[:-1], f), lambda: gpu.rotary(x, positions.long(), f),
                lambda: gpu.rotary(x, positions, f.float()), lambda: gpu.rotary(x.half(), positions, f),
                lambda: gpu.rotary(x, positions, f.cpu()), lambda: gpu.rotary(x, positions, f, out=x.bfloat16()),
                lambda: gpu.rotary(x.clone().requires_grad_(), positions, f)):
        with pytest.raises(ValueError):
            bad()


def test_frequencies(gpu):
    import math

    f, a = gpu.rotary_frequencies(64, 1e7)
    assert torch.equal(f.cpu(), freqs_of(64, 1e7)) and a == 1.0 and f.dtype == torch.float64
    lin, a = gpu.rotary_frequencies(64, 1e7, scaling="linear", factor=4.0)
    assert torch.allclose(lin * 4, f, rtol=1e-15, atol=0) and a == 1.0
    ntk, a = gpu.rotary_frequencies(64, 1e4, scaling="ntk", factor=4.0)
    base, _ = gpu.rotary_frequencies(64, 1e4)
    assert abs(float(base[-1] / ntk[-1]) - 4) < 1e-12 and float(ntk[0]) == 1.0
    y, a = gpu.rotary_frequencies(128, 1e4, scaling="yarn", factor=4.0, original=4096)
    ratio = (freqs_of(128) / y.cpu())
    turns = freqs_of(128) * 4096 / (2 * math.pi)
    assert abs(a - (0.1 * math.log(4) + 1)) < 1e-15
    assert bool((ratio[turns > 36] == 1).all()) and bool(((ratio[turns < 0.9] - 4).abs() < 1e-12).all())
    assert bool((ratio[1:] >= ratio[:-1] - 1e-12).all()) and 1.5 < float(ratio[(turns > 5) & (turns < 7)].mean()) < 3
    for bad in (dict(rot=3), dict(rot=0), dict(rot=8, base=-1.0), dict(rot=8, scaling="other"),
                dict(rot=8, scaling="yarn", factor=2.0), dict(rot=8, factor=0.0)):
        with pytest.raises(ValueError):
            gpu.rotary_frequencies(**bad)


# ---- the cache ------------------------------------------------------------------------------
def cache_case(new, cached, hq, hk, dim, page, dtype, gap=0, heads_first=False, seed=1):
    """One projection's rows (q, k, v), a pool full of 7, tables, cached, starts."""
    g = torch.Generator().manual_seed(seed)
    rows = sum(new)
    qkv = torch.randn(rows, (hq + 2 * hk) * dim + gap, generator=g).to(dtype).cuda()
    q = qkv[:, : hq * dim].view(rows, hq, dim)
    k = qkv[:, hq * dim : (hq + hk) * dim].view(rows, hk, dim)
    v = qkv[:, (hq + hk) * dim : (hq + 2 * hk) * dim].view(rows, hk, dim)
    need = [-(-(max(c, 0) + n) // page) for n, c in zip(new, cached)]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=g).to(torch.int32)
    tables, at = torch.full((len(new), max(max(need, default=1), 1)), -1, dtype=torch.int32), 0
    for s, n in enumerate(need):
        tables[s, :n] = order[at : at + n]
        at += n
    shape = (pages, hk, page, dim) if heads_first else (pages, page, hk, dim)
    K, V = (torch.full(shape, 7.0, dtype=dtype, device="cuda") for _ in range(2))
    if heads_first:
        K, V = K.transpose(1, 2), V.transpose(1, 2)
    starts = torch.tensor([0] + list(new)).cumsum(0).to(torch.int32).cuda()
    return q, k, v, K, V, tables.cuda(), torch.tensor(cached, dtype=torch.int32).cuda(), starts


def places_of(tables, cached, starts, page, pages):
    """Of every row: (sequence, place, page, slot), page -1 where there is none, sequence -1 where skipped."""
    tables, cached, starts = tables.tolist(), cached.tolist(), starts.tolist()
    out = []
    for s, held in enumerate(cached):
        for i in range(starts[s + 1] - starts[s]):
            j = held + i
            there = held >= 0 and j // page < len(tables[s]) and 0 <= tables[s][j // page] < pages
            out.append((s if held >= 0 else -1, j, tables[s][j // page] if there else -1, j % page))
    return out


@pytest.mark.parametrize("dtype", [F, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hq,hk,dim,rot,page", [(8, 2, 256, 64, 16), (4, 4, 80, 80, 7), (6, 1, 64, 10, 1),
                                                (3, 3, 8, 0, 3), (16, 4, 128, 128, 100)])
def test_append(gpu, hq, hk, dim, rot, page, interleaved, dtype):
    f = freqs_of(rot) if rot else None
    for new, cached, gap, first in (([1], [0], 0, False), ([1, 1, 1], [5, 0, 31], 3, True),
                                    ([40, 0, 3, 70], [0, 9, 100, 16], 0, True), ([2100, 7], [3, 0], 0, False),
                                    ([9, 4, 5], [10, -1, 30], 8, False)):
        q, k, v, K, V, tables, held, starts = cache_case(new, cached, hq, hk, dim, page, dtype, gap, first)
        if len(new) == 3 and new[0] == 9:
            tables[0, 0] = K.shape[0]
            tables[2, 30 // page] = -1
        where = places_of(tables, held, starts, page, K.shape[0])
        positions = torch.tensor([w[1] for w in where])
        out = torch.full((len(where), hq, dim), 9.0, dtype=dtype, device="cuda")
        got = gpu.kv_cache_append(k, v, K, V, tables, held, starts, freqs=None if f is None else f.cuda(),
                                  interleaved=interleaved, amplitude=0.9, q=q if rot else None, q_out=out if rot else None)
        assert got is (out if rot else None)
        want_k, size_k = rotated(k, positions, f if rot else freqs_of(0), interleaved, 0.9)
        rows = [r for r, w in enumerate(where) if w[2] >= 0]
        at = torch.tensor([where[r][2:] for r in rows], dtype=torch.long).reshape(-1, 2)
        near(K[at[:, 0], at[:, 1]], want_k[rows], size_k[rows], far=2200)
        assert torch.equal(V[at[:, 0], at[:, 1]], v[rows])
        untouched = torch.ones(K.shape[:2], dtype=torch.bool)
        untouched[at[:, 0], at[:, 1]] = False
        assert bool((K[untouched] == 7).all()) and bool((V[untouched] == 7).all())
        if rot:
            want_q, size_q = rotated(q, positions, f, interleaved, 0.9)
            live = torch.tensor([w[0] >= 0 for w in where])
            near(out[live], want_q[live], size_q[live], far=2200)
            assert bool((out[~live] == 9).all())


@pytest.mark.parametrize("dtype", [F, BF16])
def test_append_one_each_and_in_place(gpu, dtype):
    """Without starts; positions given; q in place; a table that is too short; values at odd elements."""
    f = freqs_of(32)
    q, k, v, K, V, tables, held, starts = cache_case([1] * 5, [0, 3, 15, 16, 40], 4, 2, 64, 16, dtype, gap=1)
    positions = torch.tensor([9, 100, -4, 1 << 20, 0], dtype=torch.int32).cuda()
    want_q, size_q = rotated(q, positions, f, False)
    want_k, size_k = rotated(k, positions, f, False)
    assert gpu.kv_cache_append(k, v, K, V, tables[:, :2], held, positions=positions, freqs=f.cuda(), q=q, q_out=q) is q
    near(q, want_q, size_q, far=1 << 20)
    for s, j in enumerate(held.tolist()):
        if j < 32:
            p = int(tables[s, j // 16])
            near(K[p, j % 16], want_k[s], size_k[s], far=1 << 20)
            assert torch.equal(V[p, j % 16], v[s])
    assert bool((K[int(tables[4, 2])] == 7).all())
    # no sequences, no rows, no pages
    assert gpu.kv_cache_append(k[:0], v[:0], K, V, tables, held) is None
    gpu.kv_cache_append(k, v, K[:0], V[:0], tables, held)
    gpu.kv_cache_append(k, v, K, V, tables[:, :0], held)


def test_append_refusals(gpu):
    q, k, v, K, V, tables, held, starts = cache_case([3, 2], [0, 3], 4, 2, 64, 16, BF16)
    f = freqs_of(32).cuda()
    call = gpu.kv_cache_append
    for bad in (lambda: call(k, v.float(), K, V, tables, held, starts), lambda: call(k, v[:-1], K, V, tables, held, starts),
                lambda: call(k, v, K.float(), V.float(), tables, held, starts),
                lambda: call(k[:, :1], v[:, :1], K, V, tables, held, starts),
                lambda: call(k, v, K, V, tables, held, starts, q=q),
                lambda: call(k, v, K, V, tables, held, starts, freqs=f, q_out=q),
                lambda: call(k, v, K, V, tables, held, starts, freqs=f, q=q[..., :32]),
                lambda: call(k, v, K, V, tables, held, starts, freqs=f, positions=starts),
                lambda: call(k.clone().requires_grad_(), v, K, V, tables, held, starts)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: call(k, v, K[:1].expand(K.shape), V[:1].expand(V.shape), tables, held, starts),
                lambda: call(k, v, K, V, tables, held), lambda: call(k, v, K, V, tables[:1].expand(2, -1), held, starts),
                lambda: call(k, v, K, V, tables, held, starts, freqs=freqs_of(66).cuda()),
                lambda: call(k, v, K, V, tables, held, starts, freqs=f, q=q[:, :3])):
        with pytest.raises(RuntimeError):
            bad()


# ---- trees -----------------------------------------------------------------------------------
def tree_oracle(parents, cached, starts, words):
    mask, positions = torch.zeros(len(parents), words, dtype=torch.int64), []
    for s, held in enumerate(cached):
        for i in range(starts[s + 1] - starts[s]):
            j, depth = i, 0
            if held < 0:
                positions.append(0)
                continue
            while True:
                if j < 32 * words:
                    mask[starts[s] + i, j // 32] |= 1 << (j % 32)
                up = parents[starts[s] + j]
                if up < 0 or up >= j:
                    break
                j, depth = up, depth + 1
            positions.append(held + depth)
    return torch.where(mask >= 1 << 31, mask - (1 << 32), mask).to(torch.int32), torch.tensor(positions, dtype=torch.int32)


def test_trees(gpu):
    g = torch.Generator().manual_seed(1)
    for new in ([1], [32, 33, 0, 7, 64], [5000, 3], [100] * 4):
        parents = []
        for n in new:
            parents += [int(torch.randint(-1, i, (1,), generator=g)) if i else -1 for i in range(n)]
        if new[0] == 32:  # values that are no earlier token
            parents[5], parents[6], parents[40], parents[10] = 5, 31, 1 << 30, -(1 << 31)
        if new[0] == 5000:
            parents[:5000] = range(-1, 4999)  # a chain
        cached = [10 * i - (1 if i == 1 else 0) * 20 for i in range(len(new))]
        starts = torch.tensor([0] + new).cumsum(0)
        words = -(-max(new) // 32)
        want = tree_oracle(parents, cached, starts.tolist(), words)
        p = torch.tensor(parents, dtype=torch.int32).cuda()
        c = torch.tensor(cached, dtype=torch.int32).cuda()
        mask, positions = gpu.draft_tree(p, c, starts.to(torch.int32).cuda(), longest=max(new))
        assert torch.equal(mask.cpu(), want[0]) and torch.equal(positions.cpu(), want[1])
        mask, _ = gpu.draft_tree(p, c, starts.to(torch.int32).cuda(), longest=1)
        assert torch.equal(mask.cpu(), want[0][:, :1])
        if len(set(new)) == 1:
            mask, positions = gpu.draft_tree(p, c)
            assert torch.equal(mask.cpu(), want[0]) and torch.equal(positions.cpu(), want[1])
    for bad in (lambda: gpu.draft_tree(p.long(), c), lambda: gpu.draft_tree(p, c, mask=mask.float()),
                lambda: gpu.draft_tree(p, c, positions=positions[:-1])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        gpu.draft_tree(p[:-1], c)


@pytest.mark.parametrize("n", [256, 257, 20000])
def test_long_trees(gpu, n):
    """Chains, and two that take turns (a token follows the one before the last), as long as a text: the bits by their
    formula.  And several sequences of them, some skipped."""
    device = dict(dtype=torch.int32, device="cuda")
    words = -(-n // 32)
    word, row = torch.arange(words, device="cuda")[None], torch.arange(n, device="cuda")[:, None]
    upto = (row - 32 * word).clamp(-1, 31)  # the last bit that a row has in a word
    ones = (torch.ones_like(upto) << (upto + 1)) - 1
    for stride, bits in ((1, ones), (2, ones & torch.where(row % 2 == 0, 0x55555555, 0xAAAAAAAA))):
        parents = torch.arange(n, **device) - stride
        want = bits.to(torch.int32), (7 + row[:, 0] // stride).to(torch.int32)
        got = gpu.draft_tree(parents, torch.tensor([7], **device))
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        if n < 1000:
            several = gpu.draft_tree(parents.repeat(3), torch.tensor([7, -1, 2 ** 31 - 3], **device))
            for x, y in zip(several, want):
                assert torch.equal(x[:n], y) and bool((x[n : 2 * n] == 0).all())
            assert torch.equal(several[0][2 * n :], want[0])
            far = (want[1].long() - 7 + 2 ** 31 - 3).clamp(max=2 ** 31 - 1)
            assert torch.equal(several[1][2 * n :].long(), far)


# ---- together --------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F, BF16])
def test_a_layer_reads_drafts_and_goes_on(gpu, dtype):
    """A prompt in two parts, a drafted tree, and the accepted branch read again in place of the tree, then single tokens:
    the attention of each call against the whole text's, with keys rotated in 64 bits."""
    hq, hk, dim, rot, page, n_seq = 8, 2, 64, 32, 16, 2
    g = torch.Generator().manual_seed(11)
    f = freqs_of(rot)
    K, V = (torch.full((20, page, hk, dim), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    tables = torch.randperm(20, generator=g)[:16].to(torch.int32).view(2, 8).cuda()
    texts = [dict(k=[], v=[]) for _ in range(n_seq)]  # the tokens that stay: their keys as projected, and values
    held = torch.zeros(n_seq, dtype=torch.int32, device="cuda")

    def call(new, parents=None, keep=None):
        """new tokens of each sequence; keep: which of them stay (None: all)."""
        nonlocal held
        rows = sum(new)
        q, k, v = (torch.randn(rows, h, dim, generator=g).to(dtype).cuda() for h in (hq, hk, hk))
        starts = torch.tensor([0] + new).cumsum(0).to(torch.int32).cuda()
        mask = positions = None
        if parents is not None:
            mask, positions = gpu.draft_tree(torch.tensor(parents, dtype=torch.int32).cuda(), held, starts, longest=max(new))
        turned = gpu.kv_cache_append(k, v, K, V, tables, held, starts, positions=positions, freqs=f.cuda(), q=q)
        out = gpu.paged_attention(turned, K, V, tables, held, starts, mask=mask)
        at = 0
        for s, n in enumerate(new):
            before = len(texts[s]["k"])
            for i in range(n):
                path = list(range(i + 1))
                if parents is not None:
                    path, j = [], i
                    while j >= 0:
                        path.insert(0, j)
                        j = parents[at + j]
                ks = torch.stack(texts[s]["k"] + [k[at + j] for j in path]).cpu()
                vs = torch.stack(texts[s]["v"] + [v[at + j] for j in path]).cpu()
                size = len(ks)
                assert size == before + len(path)
                kr = rotated(ks, torch.arange(size), f, False)[0].to(dtype)
                qr = rotated(q[at + i : at + i + 1], torch.tensor([size - 1]), f, False)[0].to(dtype)
                args = (qr, kr[None], vs[None], torch.zeros(1, 1, dtype=torch.int32), torch.tensor([size - 1]))
                want, spread, top = attention(*args, torch.tensor([0, 1]), dim ** -0.5)
                # the oracle's rotated operands may round to the other neighbour: a step of bf16 on scores of up to
                # 20 is 2^-8 x 20 on a weight's exponent at the worst, and far less in the mean of 64 products
                near_rounding = spread * (2.0 ** -4 if dtype == BF16 else 0)
                attention_near(out[at + i : at + i + 1], want, spread + near_rounding * 2 ** 8 / 8, top, dtype)
            for i in range(n) if keep is None else keep[s]:
                texts[s]["k"].append(k[at + i])
                texts[s]["v"].append(v[at + i])
            at += n
        if keep is None:
            held = held + torch.tensor(new, dtype=torch.int32, device="cuda")
            return
        # the accepted branch's keys and values move to the places that follow the text
        at = 0
        for s, n in enumerate(new):
            base = int(held[s])
            for to, i in enumerate(keep[s]):
                for cache in (K, V):
                    a, b = base + i, base + to
                    cache[int(tables[s, b // page]), b % page] = cache[int(tables[s, a // page]), a % page]
            held[s] += len(keep[s])
            at += n

    call([20, 7])
    call([5, 13])
    call([6, 4], [-1, 0, 0, 1, 2, -1, -1, -1, 1, 2], [[0, 2, 4], [1, 2, 3]])
    call([1, 1])
    call([1, 1])


def test_a_layer_captured(gpu):
    """Tree, append and attention in one graph, replayed with other drafts, against eager calls."""
    hq, hk, dim, page, n = 8, 2, 256, 16, 3
    g = torch.Generator().manual_seed(2)
    K, V = (torch.randn(30, page, hk, dim, generator=g).bfloat16().cuda() for _ in range(2))
    tables = torch.randperm(30, generator=g).to(torch.int32).view(3, 10).cuda()
    held = torch.tensor([100, 3, 50], dtype=torch.int32).cuda()
    parents = torch.tensor([-1, 0, 0, 1, -1, 0, 1, 2, -1, -1, -1, 2], dtype=torch.int32).cuda()
    q, k, v = (torch.randn(12, h, dim, generator=g).bfloat16().cuda() for h in (hq, hk, hk))
    f = freqs_of(64).cuda()
    mask, positions = torch.zeros(12, 1, dtype=torch.int32, device="cuda"), torch.zeros(12, dtype=torch.int32, device="cuda")
    turned, out = torch.zeros_like(q), torch.zeros_like(q)
    work = torch.empty(gpu.paged_attention_work_bytes(12, n, hq, hk, dim, torch.bfloat16), dtype=torch.uint8, device="cuda")

    def step(K, V, mask, positions, turned, out, work):
        gpu.draft_tree(parents, held, mask=mask, positions=positions)
        gpu.kv_cache_append(k, v, K, V, tables, held, positions=positions, freqs=f, q=q, q_out=turned)
        gpu.paged_attention(turned, K, V, tables, held, mask=mask, out=out, work=work)

    step(K, V, mask, positions, turned, out, work)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(K, V, mask, positions, turned, out, work)
    for i in range(4):
        q.copy_(torch.randn(12, hq, dim, generator=g).bfloat16())
        parents[1::4] = -1 if i % 2 else 0
        held += torch.tensor([i, 10, 20], dtype=torch.int32, device="cuda")
        mine = [K.clone(), V.clone(), mask.clone(), positions.clone(), turned.clone(), out.clone(), None]
        torch.cuda.synchronize()
        graph.replay()
        step(*mine)
        torch.cuda.synchronize()
        for a, b in zip((K, V, mask, positions, turned, out), mine):
            assert torch.equal(a, b)
