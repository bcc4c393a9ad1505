"""Edges of the attention over the paged cache and of the append: scores that are all NaN, and what a batch
does with them.  A row is NaN or it is not: what is finite has the tolerances of test_gpu_paged_attention.py."""
import pytest
import torch

from test_gpu_paged_attention import BF16, F, NAN, case, check

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
