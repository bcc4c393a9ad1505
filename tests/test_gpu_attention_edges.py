"""Edges of the attention over the paged cache and of the append: scores that are all NaN or infinite, a pool without pages, drafts
in a stretched context, caches that span more than 32 bits.
A row is NaN or it is not: what is finite has the tolerances of test_gpu_paged_attention.py."""
import pytest
import torch

from test_gpu_paged_attention import BF16, F, INF, NAN, case, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F, BF16])
@pytest.mark.parametrize("dim", [64, 80, 128, 256])
@pytest.mark.parametrize("cached", [[0], [15, 200, 3], [20000], [1, 5000]])
def test_a_query_that_is_nan(gpu, cached, dim, dtype):
    """Its row is NaN, in a batch of any size, split over workgroups or not; the others have the bits that they had."""
    n = len(cached)
    for new in (1, 2, 40):
        args, starts = case([new] * n, cached, 4, 2, dim, 16, dtype)
        want = check(gpu, args, starts, dtype, pass_starts=False)
        args[0][0, 1, dim - 1] = NAN
        args[0][n * new - 1, 2] = NAN
        got = check(gpu, args, starts, dtype, pass_starts=False)
        nan = torch.zeros(n * new, 4, dtype=torch.bool, device="cuda")
        nan[0, 1] = nan[n * new - 1, 2] = True
        assert bool(torch.isnan(got[nan]).all()) and torch.equal(got[~nan], want[~nan])


@pytest.mark.parametrize("dtype", [F, BF16])
@pytest.mark.parametrize("dim", [64, 80, 128, 256])
def test_keys_that_are_all_nan(gpu, dim, dtype):
    """A first token's own key, the only key that a wavefront has, a page of them, the only one that a mask leaves."""
    for new, cached, places in ((1, 0, [0]), (2, 0, [0, 1]), (1, 16, [16]), (1, 64, [64]), (1, 3000, range(1600, 1664)),
                                (1, 100, range(101)), (40, 0, [0]), (40, 3000, range(1600, 1664))):
        args, starts = case([1, new, 1], [7, cached, 90], 4, 2, dim, 16, dtype)
        q, K, V, tables, held = args
        for j in places:
            K[int(tables[1, j // 16]), j % 16, 1, 5] = NAN
        got = check(gpu, args, starts, dtype)
        assert bool(torch.isnan(got[1 + places[-1] - cached if places[-1] > cached else 1 : -1, 2:]).all())
        assert bool(torch.isfinite(got[:, :2]).all()) and bool(torch.isfinite(got[0]).all() and torch.isfinite(got[-1]).all())
    for new in (3, 30):
        args, starts = case([new], [0], 4, 2, dim, 16, dtype)
        q, K, V, tables, held = args
        K[int(tables[0, 0]), 2, 0, 0] = NAN
        mask = torch.zeros(new, 1, dtype=torch.int32, device="cuda")
        mask[1] = 4  # the NaN key alone
        mask[2] = 2
        got = check(gpu, args, starts, dtype, mask=mask)
        assert bool(torch.isnan(got[1, :2]).all()) and bool((got[0] == 0).all()) and bool(torch.isfinite(got[2]).all())


@pytest.mark.parametrize("dtype,code", [(F, 0), (BF16, 1)])
def test_a_pool_without_pages(gpu, dtype, code):
    """No caches and no tables (NULL), as the entry points allow it where there are no pages: the queries are rotated
    as ever, attention gives 0."""
    rows, n, hq, hk, dim = 6, 3, 4, 2, 64
    q, k = torch.randn(rows, hq, dim, device="cuda").to(dtype), torch.randn(rows, hk, dim, device="cuda").to(dtype)
    cached = torch.tensor([0, 5, -1], dtype=torch.int32, device="cuda")
    freqs, _ = gpu.rotary_frequencies(32)
    out = torch.full_like(q, 7)
    sizes = dict(cached=cached.data_ptr(), rows=rows, n_seq=n, pages=0, page=16, table_pages=4, table_row=4, heads_q=hq, heads_k=hk,
                 dim=dim, dtype=code, q=q.data_ptr(), q_row=hq * dim, q_head=dim)
    a = gpu.kv_dev_append_args(k=k.data_ptr(), v=k.data_ptr(), q_out=out.data_ptr(), freqs=freqs.data_ptr(), k_row=hk * dim, k_head=dim,
                               v_row=hk * dim, v_head=dim, q_out_row=hq * dim, q_out_head=dim, rot=32, amplitude=1.0, **sizes)
    gpu.check(gpu.load().kv_dev_append(a, None), "append")
    positions = torch.tensor([0, 1, 5, 6, 0, 0], dtype=torch.int32, device="cuda")
    assert torch.equal(out[:4], gpu.rotary(q, positions, freqs)[:4]) and bool((out[4:] == 7).all())
    work = torch.empty(gpu.paged_attention_work_bytes(rows, n, hq, hk, dim, dtype), dtype=torch.uint8, device="cuda")
    a = gpu.attn_dev_args(out=out.data_ptr(), out_row=hq * dim, out_head=dim, work=work.data_ptr(), work_bytes=work.numel(), scale=0.125,
                          **sizes)
    gpu.check(gpu.load().attn_dev_paged(a, None), "attention")
    assert bool((out[:4] == 0).all()) and bool((out[4:] == 7).all())


@pytest.mark.parametrize("dtype", [F, BF16])
def test_drafts_in_a_stretched_context(gpu, dtype):
    """Frequencies and amplitude of a context four times as long: drafted tokens that follow one another get the keys
    and queries, to the bit, that the same tokens get as text, and attention sees the same."""
    freqs, amplitude = gpu.rotary_frequencies(64, 1e6, scaling="yarn", factor=4.0, original=512)
    assert amplitude > 1.1
    args, starts = case([7, 0, 21], [40, 9, 1000], 8, 2, 128, 16, dtype)
    q, K, V, tables, cached = args
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn(28, 2, 128, generator=g).to(dtype).cuda() for _ in range(2))
    parents = torch.tensor([*range(-1, 6), *range(-1, 20)], dtype=torch.int32, device="cuda")
    mask, positions = gpu.draft_tree(parents, cached, starts, longest=21)
    results = []
    for drafted in (False, True):
        k_cache, v_cache = K.clone(), V.clone()
        turned = gpu.kv_cache_append(k, v, k_cache, v_cache, tables, cached, starts, q=q, positions=positions if drafted else None,
                                     freqs=freqs, amplitude=amplitude)
        check(gpu, (turned, k_cache, v_cache, tables, cached), starts, dtype, mask=mask if drafted else None)
        results.append((turned, k_cache.nan_to_num(9.0), v_cache.nan_to_num(9.0)))
    assert all(torch.equal(x, y) for x, y in zip(*results))
    want = gpu.rotary(q, positions, freqs, amplitude=amplitude)
    assert torch.equal(results[1][0], want)


@pytest.mark.parametrize("dtype", [F, BF16])
@pytest.mark.parametrize("stride", [1 << 31, (1 << 31) + (1 << 20) + 64])  # (elements between pages)
def test_caches_past_32_bits(gpu, stride, dtype):
    """Pages 2^31 elements apart: every entry point's offsets, in elements and in bytes, past 32 bits for each page but
    the first.  The same bits as from a cache in one piece, from single tokens, from prompts and by the append."""
    for new, held in (([2, 1], [30, 20]), ([40, 3], [20, 5]), ([300], [10])):  # (one to eight wavefronts)
        args, starts = case(new, held, 4, 2, 64, 16, dtype)
        q, K, V, tables, cached = args
        pages, n = K.shape[0], 16 * 2 * 64
        order = torch.randperm(pages - 1, generator=torch.Generator().manual_seed(3)).to(torch.int32) + 1
        repeated = pages > 7  # (not more than six pages far apart: their tokens again and again)
        if repeated:
            tables.copy_((tables % 5 + 1).where(tables >= 0, tables))
            K, V = K[:7].nan_to_num(1.0), V[:7].nan_to_num(1.0)
            pages = 7
        else:
            K, V = K.clone(), V.clone()
            back = torch.full((pages,), -1, dtype=torch.int32)
            used = tables[tables >= 0].long().cpu()
            back[used] = order[: len(used)]
            for old, to in zip(used.tolist(), back[used].tolist()):
                K[to], V[to] = args[1][old], args[2][old]
            tables[tables >= 0] = back.cuda()[tables[tables >= 0].long()]
        assert bool((tables[tables >= 0] >= 1).all())  # (no page that 32 bits would reach)
        far = torch.empty((pages - 1) * stride + 2 * n, dtype=dtype, device="cuda")
        K2, V2 = (torch.as_strided(far, K.shape, (stride, 128, 64, 1), i * n) for i in range(2))
        K2.copy_(K)
        V2.copy_(V)
        near = gpu.paged_attention(q, K, V, tables, cached, starts)
        assert bool(torch.isfinite(near).all())
        assert torch.equal(gpu.paged_attention(q, K2, V2, tables, cached, starts), near)
        if repeated:
            continue  # (two rows must not meet in one place)
        freqs, _ = gpu.rotary_frequencies(32)
        k, v = (torch.randn(sum(new), 2, 64, device="cuda").to(dtype) for _ in range(2))
        for caches in ((K, V), (K2, V2)):
            gpu.kv_cache_append(k, v, *caches, tables, cached, starts, freqs=freqs)
        at = tables[tables >= 0].long()
        for x, y in ((K, K2), (V, V2)):
            assert torch.equal(x[at].nan_to_num(9.0), y[at].nan_to_num(9.0))
        del far, K2, V2


@pytest.mark.parametrize("dtype", [F, BF16])
@pytest.mark.parametrize("dim", [64, 80, 256])
def test_keys_with_an_infinity(gpu, dim, dtype):
    """A score of -infinity is a weight of 0, one of infinity makes its row NaN, and a row whose every score is -infinity
    is 0: in single tokens, drafts and prompts, split over workgroups or not."""
    for new, cached, places in ((1, 0, [0]), (1, 500, [0, 300, 499]), (5, 20000, [17, 9000]), (40, 60, [3, 61, 99]),
                                (40, 0, [0, 1, 2])):
        args, starts = case([new, 2], [cached, 33], 4, 2, dim, 16, dtype)
        q, K, V, tables, held = args
        for j in places:
            K[int(tables[0, j // 16]), j % 16, 0, 7] = INF
            K[int(tables[0, j // 16]), j % 16, 1, 7] = -INF
        q[0, :, 7] = torch.tensor([-1.0, 1.0, 1.0, -1.0])
        got = check(gpu, args, starts, dtype)
        assert bool(torch.isfinite(got[0, [0, 2]]).all()) and bool(torch.isnan(got[0, [1, 3]]).all())
        if cached == 0:
            assert bool((got[0, [0, 2]] == 0).all())
