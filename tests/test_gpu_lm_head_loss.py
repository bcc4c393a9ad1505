"""The tied-embedding head's loss and its gradient on the GPU, against 64 bits.

Tolerances.  Products of bf16 values are exact in float32; a float32 hidden state
keeps its 24 bits; sums are float32.  A logit is a sum of at most 2048 products:
rounded on the way at most sqrt(2048) x 2^-24 of the norms' product |w| |h| (about
10 here for logits of a few), 3e-5 absolute at the worst, and lse and the loss
are means of such errors: 4e-5 absolute.  D is off by that and by 2^-20 of itself.
A gradient sums D times inputs: relative to the gradient row's largest value
2e-4 leaves a factor of ten for float32 (grad_h); a bf16 gradient (grad_table, and
grad_h with bf16 states) adds half a step, 2^-8 of the value, and, with bf16
states, D's own half steps: 2^-9 of sqrt(sum of squares of its terms) at random,
at most 2^-8 of the sum of their magnitudes, which is what is taken."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
F, BF16 = torch.float32, torch.bfloat16


def inputs(rows, vocab, hidden, dtype, seed=1, pad=0, ignored=0.25):
    g = torch.Generator().manual_seed(seed)
    table = torch.zeros(vocab, hidden + pad, dtype=BF16)
    table[:, :hidden] = (torch.randn(vocab, hidden, generator=g) * 2.0 / hidden ** 0.5).to(BF16)
    h = torch.randn(rows, hidden + pad, generator=g).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g, dtype=torch.int32)
    t[torch.rand(rows, generator=g) < ignored] = -100
    gl = torch.rand(rows, generator=g) + 0.1
    return h.cuda()[:, :hidden], table.cuda()[:, :hidden], t.cuda(), gl.cuda()


def oracle(h, table, t, gl):
    h, w, t, gl = h.double().cpu(), table.double().cpu(), t.long().cpu(), gl.double().cpu()
    keep = (t >= 0) & (t < len(w))
    z = h[keep] @ w.t()
    lse = torch.logsumexp(z, 1)
    at = t[keep]
    loss, all_lse = torch.zeros(len(h), dtype=torch.float64), torch.zeros(len(h), dtype=torch.float64)
    loss[keep], all_lse[keep] = lse - z.gather(1, at[:, None])[:, 0], lse
    bad = t >= len(w)
    loss[bad] = all_lse[bad] = float("nan")
    D = torch.exp(z - lse[:, None])
    D[torch.arange(len(at)), at] -= 1
    D *= gl[keep][:, None]
    gh = torch.zeros_like(h)
    gh[keep] = D @ w
    gh[bad] = float("nan")
    gw = D.t() @ h[keep]
    mags = torch.zeros_like(h)
    mags[keep] = D.abs() @ w.abs()
    return loss, all_lse, gh, gw, mags, D.abs().t() @ h[keep].abs()


def near(got, want, bound):
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    off = torch.where(torch.isnan(want), 0.0, (got - want).abs())
    over = off - torch.nan_to_num(bound) if torch.is_tensor(bound) else off - bound
    assert bool((over <= 0).all()), (float(over.max()), float(off.max()))


def row_top(x):
    return torch.nan_to_num(x).abs().amax(1, keepdim=True).clamp(min=1e-9)


def check_all(gpu, h, table, t, gl):
    loss, lse, gh, gw, mags_h, mags_w = oracle(h, table, t, gl)
    got_loss, got_lse = gpu.lm_head_loss(h, table, t)
    near(got_loss, loss, 4e-5)
    near(got_lse, lse, 4e-5)
    got_h, got_w = gpu.lm_head_loss_grad(h, table, t, got_lse, gl)
    if h.dtype == F:
        near(got_h, gh, 2e-4 * row_top(gh))
        near(got_w, gw, gw.abs() * 2 ** -8 + 2e-4 * row_top(gw))
    else:
        near(got_h, gh, gh.abs() * 2 ** -8 + 2e-4 * row_top(gh) + mags_h * 2 ** -8)
        near(got_w, gw, gw.abs() * 2 ** -8 + 2e-4 * row_top(gw) + mags_w * 2 ** -8)


@pytest.mark.parametrize("dtype", [F, BF16])
@pytest.mark.parametrize("rows,vocab,hidden", [
    (1, 1, 8), (1, 129, 64), (2, 1000, 8), (31, 300, 128), (33, 257, 72), (64, 128, 1024), (65, 640, 136), (130, 1111, 200),
    (300, 2500, 320), (7, 50, 1), (40, 333, 33), (100, 700, 1001), (129, 131, 63), (1100, 900, 320), (1025, 2305, 72)])
def test_loss_and_gradients(gpu, rows, vocab, hidden, dtype):
    check_all(gpu, *inputs(rows, vocab, hidden, dtype))
