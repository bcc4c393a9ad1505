"""Attention over the paged cache on the GPU, against 64 bits.

Tolerances.  Float32: a score is a sum of up to 256 products, rounded on the way at random; with q . k of up to
about 100 before the scale, sqrt(256) 2^-24 x 100 = 1e-4, times the scale of 1 / 16 or (fewer elements)
less of each: 6e-6 on a weight's exponent, and 2^-24 of the exponent itself, 1e-6 at 20.  An output is a
mean of values with weights so far off: 2 x 7e-6 of the largest value, F32 = 2e-5 of it.
bf16: the result's own rounding, 2^-8 of it, and that of the weights, 2^-8 of each.  The sum that divides takes the
rounded weights, so that with w (1 + e) the result is off by sum w e (v - o) / sum w (1 + e): at most
2^-8 / (1 - 2^-8) of the mean of |v - o|, which the oracle computes."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F, BF16 = torch.float32, torch.bfloat16
F32 = 2e-5
NAN, INF = float("nan"), float("inf")


def case(new, cached, hq, hk, dim, page, dtype, seed=1, spread=1.5, heads_first=False, gap=0, free=NAN, columns=0):
    """q (rows `gap` elements apart), caches whose free places hold `free`, tables, cached, starts."""
    g = torch.Generator().manual_seed(seed)
    n, rows = len(new), sum(new)
    total = [max(c, 0) + m for m, c in zip(new, cached)]
    need = [-(-t // page) for t in total]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=g).tolist()
    wide = max(max(need, default=0), columns, 1)
    tables = torch.full((n, wide), -1, dtype=torch.int32)
    K = torch.full((pages, page, hk, dim), free)
    V = K.clone()
    at = 0
    for s, t in enumerate(total):
        mine = order[at : at + need[s]]
        at += need[s]
        tables[s, : len(mine)] = torch.tensor(mine, dtype=torch.int32)
        for i, p in enumerate(mine):
            k = min(page, t - i * page)
            K[p, :k] = torch.randn(k, hk, dim, generator=g)
            V[p, :k] = torch.randn(k, hk, dim, generator=g)
    q = spread * torch.randn(rows, hq, dim + gap, generator=g)
    if heads_first:  # pages x heads x page x dim in memory
        K, V = (x.transpose(1, 2).contiguous().to(dtype).cuda().transpose(1, 2) for x in (K, V))
    else:
        K, V = K.to(dtype).cuda(), V.to(dtype).cuda()
    starts = torch.tensor([0] + new).cumsum(0).to(torch.int32).cuda()
    return (q.to(dtype).cuda()[..., :dim], K, V, tables.cuda(), torch.tensor(cached, dtype=torch.int32).cuda()), starts


def oracle(q, K, V, tables, cached, starts, scale, mask=None):
    """-> (out, mean |v - out|, the largest |v| seen), 64 bits on the CPU; rows of no (or a skipped) sequence NaN."""
    dev = "cpu"
    q, K, V = (x.to(dev).double() for x in (q, K, V))
    tables, cached, starts = tables.tolist(), cached.tolist(), starts.tolist()
    pages, page, hk, dim = K.shape
    rows, hq, _ = q.shape
    group = hq // hk
    out = torch.full(q.shape, NAN, dtype=torch.float64)
    dev_sum = torch.zeros_like(out)
    bits = None if mask is None else mask.cpu().long()
    top = 0.0
    for s, held in enumerate(cached):
        a, b = starts[s], starts[s + 1]
        if held < 0 or a == b:
            continue
        n = b - a
        places = [j for j in range(min(held + n, len(tables[s]) * page)) if 0 <= tables[s][j // page] < pages]
        pid = torch.tensor([tables[s][j // page] for j in places], dtype=torch.long)
        slot = torch.tensor([j % page for j in places], dtype=torch.long)
        where = torch.tensor(places, dtype=torch.long)
        Ks, Vs = K[pid, slot], V[pid, slot]
        i = torch.arange(n)[:, None]
        if bits is None:
            sees = where[None] <= held + i
        else:
            j = (where - held).clamp(min=0)
            word = (j // 32).clamp(max=bits.shape[1] - 1)
            hit = (bits[a:b][:, word] >> (j % 32)) & 1
            hit = hit.bool() & (j // 32 < bits.shape[1])
            sees = (where[None] < held) | hit
        fin = Vs[torch.isfinite(Vs)]
        if fin.numel():
            top = max(top, float(fin.abs().max()))
        for h in range(hq):
            k, v = Ks[:, h // group], Vs[:, h // group]
            z = (q[a:b, h] @ k.t()) * scale
            z = torch.where(sees, z, torch.tensor(-INF, dtype=torch.float64))
            if z.shape[1] == 0:
                out[a:b, h] = 0
                continue
            m = z.amax(1, keepdim=True)
            w = torch.where(sees, torch.exp(z - m), torch.tensor(0.0, dtype=torch.float64))
            w = torch.where(torch.isneginf(m), torch.tensor(0.0, dtype=torch.float64), w)
            l = w.sum(1, keepdim=True)
            if torch.isfinite(v).all():
                o = w @ v
            else:  # what a row does not see is not multiplied by 0
                o = torch.stack([(w[r][sees[r]][:, None] * v[sees[r]]).sum(0) for r in range(n)])
            o = torch.where(l == 0, torch.tensor(0.0, dtype=torch.float64), o / l)
            out[a:b, h] = o
            for lo in range(0, n, 64):
                part = (v[None] - o[lo : lo + 64, None]).abs() * w[lo : lo + 64, :, None]
                part = torch.nan_to_num(part, nan=0, posinf=0)
                dev_sum[a + lo : a + min(n, lo + 64), h] = part.sum(1) / l[lo : lo + 64].clamp(min=1e-300)
    return out, dev_sum, top


def near(got, want, spread, top, dtype):
    got = got.double().cpu()
    held = ~torch.isnan(want)
    assert torch.equal(torch.isnan(got), ~held)
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    fine = held & ~inf
    got, want, spread = got[fine], want[fine], spread[fine]
    bound = torch.full_like(want, F32 * max(top, 1e-3))
    if dtype == BF16:
        bound += want.abs() * 2.0 ** -8 + spread * (2.0 ** -8 / (1 - 2.0 ** -8))
    off = (got - want).abs()
    assert bool((off <= bound).all()), (float((off / bound).max()), float(off.max()))


def check(gpu, args, starts, dtype, mask=None, scale=None, pass_starts=True, **kw):
    dim = args[0].shape[2]
    got = gpu.paged_attention(*args, starts if pass_starts else None, scale=scale, mask=mask, **kw)
    want, spread, top = oracle(*args, starts, dim ** -0.5 if scale is None else scale, mask)
    skipped = torch.isnan(want) if not kw else None
    if skipped is not None:  # (a new out is 0 there)
        a = args[4].cpu()
        for s in range(len(a)):
            if a[s] < 0:
                want[starts[s] : starts[s + 1]] = 0
    near(got, want, spread, top, dtype)
    return got


SHAPES = [(8, 2, 256, 16), (16, 4, 128, 16), (6, 2, 80, 7), (5, 5, 64, 1), (16, 1, 64, 64), (3, 1, 8, 3), (12, 4, 200, 100),
          (40, 2, 96, 33)]


@pytest.mark.parametrize("dtype", [F, BF16])
@pytest.mark.parametrize("hq,hk,dim,page", SHAPES)
def test_single_tokens(gpu, hq, hk, dim, page, dtype):
    """One token of each sequence, from an empty cache on."""
    for cached in ([0], [1], [31], [32, 0, 33, 100, 7], [513] * 3, [2000]):
        n = len(cached)
        args, starts = case([1] * n, cached, hq, hk, dim, page, dtype)
        check(gpu, args, starts, dtype, pass_starts=False)
        check(gpu, args, starts, dtype)


@pytest.mark.parametrize("dtype", [F, BF16])
@pytest.mark.parametrize("hq,hk,dim,page", SHAPES)
def test_prompts(gpu, hq, hk, dim, page, dtype):
    """Ragged prompts, new and continued ones, sequences without tokens; every number of wavefronts."""
    for new, cached in (([2, 3], [5, 0]), ([17, 0, 1, 40], [0, 9, 64, 100]), ([130, 70], [3, 200]), ([333], [0]),
                        ([1, 1, 200, 1], [400, 0, 31, 1])):
        args, starts = case(new, cached, hq, hk, dim, page, dtype)
        check(gpu, args, starts, dtype)


@pytest.mark.parametrize("dtype", [F, BF16])
@pytest.mark.parametrize("rows", [1, 2, 4, 5, 8, 9, 16, 17, 32, 33, 63, 65, 127, 129, 257])
def test_rows_of_a_tile(gpu, rows, dtype):
    """Every size of a tile of rows, the same number of rows for each sequence."""
    args, starts = case([rows] * 3, [40, 0, 95], 4, 1, 128, 16, dtype)
    check(gpu, args, starts, dtype, pass_starts=False)


@pytest.mark.parametrize("dtype", [F, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_long_sequences_shared_by_workgroups(gpu, dim, dtype):
    args, starts = case([1, 1], [70001, 300], 4, 2, dim, 16, dtype)
    check(gpu, args, starts, dtype, pass_starts=False)
    args, starts = case([70], [20000], 4, 1, dim, 16, dtype)
    check(gpu, args, starts, dtype)


@pytest.mark.parametrize("dtype", [F, BF16])
def test_many_sequences(gpu, dtype):
    """More places than a workgroup remembers the tiles of."""
    cached = [(7 * i) % 40 for i in range(1500)]
    args, starts = case([1] * 1500, cached, 2, 1, 64, 16, dtype)
    check(gpu, args, starts, dtype, pass_starts=False)
    new = [(5 * i) % 3 for i in range(1500)]
    args, starts = case(new, cached, 2, 1, 64, 16, dtype)
    check(gpu, args, starts, dtype)


@pytest.mark.parametrize("dtype", [F, BF16])
def test_strides(gpu, dtype):
    """Heads of q apart (a gate between them) or at odd elements, caches with heads before tokens, tables that are
    part of a larger one, an out with rows of its own."""
    for gap in (0, 128, 3):
        args, starts = case([9, 1, 30], [100, 0, 31], 8, 2, 128, 16, dtype, heads_first=True, gap=gap)
        check(gpu, args, starts, dtype)
        q, K, V, tables, cached = args
        wide = torch.full((3, tables.shape[1] + 5), 9999, dtype=torch.int32, device="cuda")
        wide[:, : tables.shape[1]] = tables
        args = (q, K, V, wide[:, : tables.shape[1]], cached)
        out = torch.full((40, 8, 128 + gap + 1), 7.0, dtype=dtype, device="cuda")
        view = out[..., :128]
        check(gpu, args, starts, dtype, out=view)
        assert bool((out[..., 128:] == 7).all())
    # heads before rows
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    check(gpu, (qt, *args[1:]), starts, dtype)
    # both caches in one tensor
    both = torch.stack((K, V), 1)
    check(gpu, (q, both[:, 0], both[:, 1], *args[3:]), starts, dtype)


@pytest.mark.parametrize("dtype", [F, BF16])
def test_absent_places(gpu, dtype):
    """Table entries that are no page, places past the table, skipped sequences, rows that no sequence holds."""
    args, starts = case([20, 4, 50, 3, 6], [100, -1, 40, 30, -5], 4, 2, 64, 16, dtype)
    q, K, V, tables, cached = args
    tables[0, 1] = -1
    tables[0, 3] = K.shape[0]
    tables[2, :] = 2 ** 31 - 1  # nothing of this sequence is there
    tables[3] = -(2 ** 31)
    got = check(gpu, args, starts, dtype)
    assert bool((got[24:77] == 0).all()) and bool((got[20:24] == 0).all())
    short = tables[:, :2].contiguous()  # 32 places of 120
    check(gpu, (q, K, V, short, cached), starts, dtype)
    none = tables[:, :0]
    assert bool((gpu.paged_attention(q, K, V, none, cached, starts) == 0).all())
    assert bool((gpu.paged_attention(q, K[:0], V[:0], short, cached, starts) == 0).all())
    # few rows on a key head
    few, fstarts = case([4, 1, 2, 3], [100, -1, 40, 700], 4, 2, 64, 16, dtype)
    few[3][0, 1] = -1
    few[3][0, 4] = 2 ** 31 - 1
    few[3][2] = -7
    few[3][3, 5:40:7] = few[1].shape[0]
    check(gpu, few, fstarts, dtype)
    assert bool((gpu.paged_attention(few[0], K[:0], V[:0], *few[3:], fstarts) == 0).all())
    # rows in front of and behind the sequences, and of skipped ones, stay as they were
    q2 = torch.cat((q, q, q))
    out = torch.full_like(q2, 5.0)
    inner = starts + len(q)
    gpu.paged_attention(q2, K, V, tables, cached, inner, out=out)
    n = len(q)
    assert bool((out[:n] == 5).all()) and bool((out[2 * n :] == 5).all())
    assert bool((out[n + 20 : n + 24] == 5).all()) and bool((out[n + 77 : n + 83] == 5).all())
    assert torch.equal(out[n : n + 20], got[:20])


def random_mask(rows, words, seed=3, share=0.3):
    g = torch.Generator().manual_seed(seed)
    bits = torch.rand(rows, words, 32, generator=g) < share
    value = (bits.long() << torch.arange(32)).sum(2)
    return torch.where(value >= 1 << 31, value - (1 << 32), value).to(torch.int32).cuda()


@pytest.mark.parametrize("dtype", [F, BF16])
@pytest.mark.parametrize("hq,hk,dim,page", SHAPES)
def test_masks(gpu, hq, hk, dim, page, dtype):
    """Any bits: rows that see nothing are 0; words that are too few; lengths that no tile ends with."""
    for new, cached, words in (([5, 1, 30], [0, 0, 3], 1), ([70, 33, 64], [45, 0, 31], 3), ([40], [5], 1),
                               ([8, 8], [1000, 33], 1), ([200], [0], 7)):
        args, starts = case(new, cached, hq, hk, dim, page, dtype)
        mask = random_mask(sum(new), words)
        mask[0] = 0
        check(gpu, args, starts, dtype, mask=mask)


@pytest.mark.parametrize("dtype", [F, BF16])
@pytest.mark.parametrize("dim", [64, 80, 128, 256])
def test_values_that_are_not_finite(gpu, dim, dtype):
    """A NaN or infinity in a value shows in the rows that see it, in its element, and in no other; in a
    key in all elements of them; what no row sees nowhere.  Causal and with a mask; first in a tile and inside."""
    for new, cached, masked in (([40, 3], [0, 70], False), ([100], [29], False), ([40, 20], [3, 40], True), ([300], [0], False)):
        args, starts = case(new, cached, 4, 2, dim, 16, dtype, free=INF)
        q, K, V, tables, held = args
        mask = random_mask(sum(new), 2) if masked else None

        def put(cache, s, j, d, x):
            cache[int(tables[s, j // 16]), j % 16, 1, d] = x

        put(V, 0, cached[0], 0, NAN)
        put(V, 0, cached[0] + 5, 1, INF)
        put(V, 0, cached[0] + 7, 1, -INF)
        put(V, 0, cached[0] + 9, dim - 1, -INF)
        put(V, 0, cached[0] + 33, 2, INF)
        got = check(gpu, args, starts, dtype, mask=mask)
        assert bool(torch.isnan(got).any()) and bool(torch.isinf(got).any()) and bool(torch.isfinite(got[:, :2]).all())
        put(K, 0, cached[0] + 20, 3, NAN)
        got = check(gpu, args, starts, dtype, mask=mask)
        if not masked:
            assert bool(torch.isnan(got[20:new[0], 2:]).all()) and bool(torch.isfinite(got[new[0] :]).all())


@pytest.mark.parametrize("dtype", [F, BF16])
@pytest.mark.parametrize("dim", [64, 80, 128, 256])
def test_values_that_are_not_finite_few_rows(gpu, dim, dtype):
    """The same with up to 16 rows on a key head, at a place that a wavefront has last and one that it has first."""
    for cached, masked in ((0, False), (59, False), (64, False), (200, True), (14, True)):
        args, starts = case([7, 1], [cached, 33], 4, 2, dim, 16, dtype, free=NAN)
        q, K, V, tables, held = args
        mask = random_mask(8, 1) if masked else None
        for j, d, x in ((0, 0, NAN), (1, 1, INF), (3, 1, -INF), (4, dim - 1, -INF), (5, 2, INF), (2, 3, INF)):
            V[int(tables[0, (cached + j) // 16]), (cached + j) % 16, 1, d] = x
        got = check(gpu, args, starts, dtype, mask=mask)
        assert bool(torch.isfinite(got[:, :2]).all()) and bool(torch.isfinite(got[7]).all())
        if not masked:
            assert bool(torch.isnan(got[:7, 2:, 0]).all()) and bool(torch.isinf(got[1:3, 2:, 1]).all())
        K[int(tables[0, (cached + 5) // 16]), (cached + 5) % 16, 1, 3] = NAN
        got = check(gpu, args, starts, dtype, mask=mask)
        if not masked:
            assert bool(torch.isnan(got[5:7, 2:]).all())


@pytest.mark.parametrize("dtype", [F, BF16])
def test_mostly_empty_batches(gpu, dtype):
    """Long runs of skipped and of empty sequences between those that are at work, more than a workgroup remembers."""
    live = {3: 700, 70: 5, 300: 64, 1290: 1500}
    for new, rest in ((1, -1), (2, -1), (40, -1), (1, 0), (40, 0)):  # rest 0: the others have no rows, with tokens held
        lens = [new if s in live or rest < 0 and new < 40 else 0 for s in range(1300)]
        held = [live.get(s, rest) for s in range(1300)]
        args, starts = case(lens, held, 4, 2, 64, 16, dtype)
        check(gpu, args, starts, dtype, pass_starts=len(set(lens)) > 1)


def test_two_streams_at_once(gpu):
    """Two calls that overlap, each with its own work."""
    a, sa = case([1] * 3, [3000, 200, 9000], 8, 2, 256, 16, BF16)
    b, sb = case([40], [7000], 8, 2, 128, 16, BF16)
    want = gpu.paged_attention(*a), gpu.paged_attention(*b, sb)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        for s, args, starts in ((streams[0], a, None), (streams[1], b, sb)):
            with torch.cuda.stream(s):
                outs.append(gpu.paged_attention(*args, starts))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert torch.equal(o, want[i % 2])


@pytest.mark.parametrize("dtype", [F, BF16])
def test_equal_weights(gpu, dtype):
    """Equal keys: the mean of the values, with no error from the weights' rounding."""
    args, starts = case([3, 60], [777, 100], 8, 2, 128, 16, dtype)
    q, K, V, tables, cached = args
    K[:] = K[int(tables[0, 0]), 0].clone()
    V[torch.isnan(V)] = 0
    out = gpu.paged_attention(*args, starts)
    want, _, top = oracle(*args, starts, 128 ** -0.5)
    near(out, want, torch.zeros_like(want), top, dtype)


@pytest.mark.parametrize("dtype", [F, BF16])
def test_large_scores_and_scales(gpu, dtype):
    """Scores that grow along the keys by much more than exp takes, one key that has all the weight, tiny scales."""
    args, starts = case([2, 40], [300, 90], 4, 2, 64, 16, dtype)
    for scale in (1e-6, 3.0):
        got = gpu.paged_attention(*args, starts, scale=scale)
        want, spread, top = oracle(*args, starts, scale)
        # (a score of up to 3 x 100 is off by 2^-24 of itself and by its sum's rounding: 1e-4)
        near(got, want, spread + (spread * 1e-4 * 2 ** 8 if scale > 1 else 0), top * (20 if scale > 1 else 1), dtype)
    q, K, V, tables, cached = args
    for j in range(300):
        K[int(tables[0, j // 16]), j % 16] *= 1 + j  # (bf16 values: the oracle has the same)
    got = gpu.paged_attention(*args, starts, scale=0.01)
    want, spread, top = oracle(*args, starts, 0.01)
    near(got, want, spread * (2 if dtype == BF16 else 1), top * 20, dtype)
    q[0] = 3e38 if dtype == F else 1e38  # scores that are not finite: NaN for that row alone
    got = gpu.paged_attention(*args, starts, scale=1.0)
    assert bool(torch.isnan(got[0]).all()) and bool(torch.isfinite(got[1:]).all())


def test_offsets_past_32_bits(gpu):
    """Pages 2^31 elements apart, and a pool of 5 GB."""
    args, starts = case([2, 1], [30, 20], 4, 2, 64, 16, BF16)
    q, K, V, tables, cached = args
    want = gpu.paged_attention(*args, starts)
    pages = K.shape[0]
    n = 16 * 2 * 64
    far = torch.empty((1 << 31) + (pages + 2) * 2 * n, dtype=BF16, device="cuda")
    strides = ((1 << 31) // (pages - 1) // 8 * 8, 128, 64, 1)
    K2 = torch.as_strided(far, K.shape, strides)
    V2 = torch.as_strided(far, K.shape, strides, n)
    K2.copy_(K)
    V2.copy_(V)
    assert torch.equal(gpu.paged_attention(q, K2, V2, tables, cached, starts), want)


def test_work_streams_and_repeats(gpu):
    """The same bits again, with a work buffer full of NaN, on another stream, and out given."""
    args, starts = case([50, 1, 3], [500, 3000, 0], 8, 2, 256, 16, BF16)
    want = check(gpu, args, starts, BF16)
    need = gpu.paged_attention_work_bytes(54, 3, 8, 2, 256, BF16)
    work = torch.full((need // 4,), NAN, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        out = torch.full_like(args[0], NAN)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            assert gpu.paged_attention(*args, starts, out=out, work=work) is out
        torch.cuda.current_stream().wait_stream(stream)
        assert torch.equal(out, want)
    a = torch.empty(need + 1, dtype=torch.uint8, device="cuda")
    for bad in (a[1:], a[: need - 256]):
        with pytest.raises(RuntimeError, match="work"):
            gpu.paged_attention(*args, starts, work=bad)


def test_captured_call_follows_its_lengths(gpu):
    """A call in a graph, replayed as the sequences grow, against eager calls."""
    args, starts = case([1] * 4, [0, 10, 100, 700], 8, 2, 256, 16, BF16, columns=60)
    q, K, V, tables, cached = args
    V[torch.isnan(V)] = 0.5
    K[torch.isnan(K)] = 0.25
    tables[tables < 0] = 0
    out = torch.zeros_like(q)
    work = torch.empty(gpu.paged_attention_work_bytes(4, 4, 8, 2, 256, BF16), dtype=torch.uint8, device="cuda")
    gpu.paged_attention(*args, out=out, work=work)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu.paged_attention(*args, out=out, work=work)
    for i in range(5):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, gpu.paged_attention(*args))
        cached += torch.tensor([1, 0, 37, -90], dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [F, BF16])
def test_shared_pages(gpu, dtype):
    """Sequences with the same first pages."""
    args, starts = case([3, 3], [64, 64], 4, 2, 64, 16, dtype)
    q, K, V, tables, cached = args
    tables[1, :3] = tables[0, :3]
    check(gpu, args, starts, dtype)


def test_refusals(gpu):
    args, starts = case([3, 2], [10, 20], 4, 2, 64, 16, BF16)
    q, K, V, tables, cached = args
    call = gpu.paged_attention
    for bad in (lambda: call(q.float(), K, V, tables, cached, starts), lambda: call(q, K.float(), V, tables, cached, starts),
                lambda: call(q[..., :32], K, V, tables, cached, starts), lambda: call(q, K, V[:-1], tables, cached, starts),
                lambda: call(q, K, V, tables.long(), cached, starts), lambda: call(q, K, V, tables[:1], cached, starts),
                lambda: call(q, K, V, tables, cached.long(), starts), lambda: call(q, K, V, tables, cached, starts[:2]),
                lambda: call(q, K, V.transpose(1, 2).contiguous().transpose(1, 2), tables, cached, starts),
                lambda: call(q, K, V, tables, cached, starts, mask=torch.zeros(5, 1, device="cuda")),
                lambda: call(q, K, V, tables, cached, starts, mask=torch.zeros(5, 0, dtype=torch.int32, device="cuda")),
                lambda: call(q.cpu(), K, V, tables, cached, starts), lambda: call(q, K, V, tables.cpu(), cached, starts),
                lambda: call(q, K, V, tables, cached, starts, out=q.float()),
                lambda: call(q[0], K, V, tables, cached, starts)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: call(q[:, :3], K, V, tables, cached, starts), lambda: call(q, K, V, tables, cached),
                lambda: call(q, K, V, tables, cached, starts, scale=0.0),
                lambda: call(q, K, V, tables, cached, starts, scale=-1.0),
                lambda: call(q, K, V, tables, cached, starts, scale=NAN),
                lambda: call(q, K, V, tables, cached, starts, out=q[:1].expand(5, 4, 64).clone()[:1].expand(5, 4, 64))):
        with pytest.raises(RuntimeError):
            bad()
    assert call(q[:0], K, V, tables[:0], cached[:0], starts[:1]).shape == (0, 4, 64)
    with pytest.raises(ValueError, match="requires a gradient"):
        call(q.clone().requires_grad_(), K, V, tables, cached, starts)
