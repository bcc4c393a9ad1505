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


@pytest.mark.parametrize("dtype", [F, BF16])
def test_strided_and_unaligned(gpu, dtype):
    for pad in (1, 8):
        check_all(gpu, *inputs(70, 400, 64, dtype, pad=pad))
    h, table, t, gl = inputs(70, 401, 64, dtype)
    check_all(gpu, h, table[1:], t.clamp(max=399), gl)
    flat = torch.empty(400 * 64 + 1, dtype=BF16, device="cuda")
    odd = flat[1:].view(400, 64)  # rows at odd 16-bit addresses
    odd.copy_(table[:400])
    check_all(gpu, h, odd, t.clamp(max=399), gl)


@pytest.mark.parametrize("dtype,rows,vocab", [(BF16, 8192, 18001), (F, 4096, 11000)])
def test_several_pieces_of_the_vocabulary(gpu, dtype, rows, vocab):
    check_all(gpu, *inputs(rows, vocab, 64, dtype, ignored=0.9))


@pytest.mark.parametrize("dtype", [F, BF16])
@pytest.mark.parametrize("rows,vocab,hidden", [(130, 20001, 520), (130, 20001, 513), (200, 17000, 257), (65, 33000, 264)])
def test_more_tiles_than_compute_units(gpu, rows, vocab, hidden, dtype):
    """Float32 states' wide tiles, with the last ones cut in each direction; table rows at odd elements."""
    check_all(gpu, *inputs(rows, vocab, hidden, dtype))


@pytest.mark.parametrize("dtype", [F, BF16])
@pytest.mark.parametrize("rows", [8193, 16400])
def test_many_rows(gpu, rows, dtype):
    """More rows than the workgroups that gather them have at a time, whose last run is not full."""
    check_all(gpu, *inputs(rows, 40, 72, dtype))


@pytest.mark.parametrize("dtype", [F, BF16])
def test_ignored_rows_hold_anything(gpu, dtype):
    h, table, t, gl = inputs(90, 300, 96, dtype)
    t[3], t[50], t[89] = 300, 2 ** 31 - 1, -1
    h[t < 0] = float("nan")
    h[50] = float("inf")
    check_all(gpu, h, table, t, torch.where(t < 0, float("nan"), gl))
    for target in (-5, 300):
        t[:] = target
        loss, lse = gpu.lm_head_loss(h, table, t)
        gh, gw = gpu.lm_head_loss_grad(h, table, t, lse, gl)
        assert bool((gw == 0).all())
        assert bool((gh == 0).all() if target < 0 else torch.isnan(gh).all())
        assert bool((loss == 0).all() if target < 0 else torch.isnan(loss).all())


@pytest.mark.parametrize("dtype", [F, BF16])
def test_extreme_logits(gpu, dtype):
    """Logits far apart, near the type's lowest value, and infinite."""
    h = torch.zeros(5, 8, device="cuda")
    h[:, 0] = torch.tensor([1.0, 1.0, -1.0, 1e-3, 0.0], device="cuda")
    table = torch.zeros(300, 8, device="cuda", dtype=BF16)
    table[:, 0] = torch.linspace(-3e4, 3e4, 300)
    table[7, 0] = torch.finfo(BF16).min / 4
    h = h.to(dtype)
    t = torch.tensor([299, 0, 299, 3, 8], dtype=torch.int32, device="cuda")
    loss, lse = gpu.lm_head_loss(h, table, t)
    z = h.double().cpu() @ table.double().cpu().t()
    want = torch.logsumexp(z, 1)
    at = z.gather(1, t.long().cpu()[:, None])[:, 0]
    for r in range(5):
        assert abs(float(lse[r]) - float(want[r])) <= 2 ** -22 * abs(float(want[r])) + 1e-6, r
        assert abs(float(loss[r]) - float(want[r] - at[r])) <= 2 ** -21 * float(want[r].abs() + at[r].abs()) + 1e-6, r
    # infinities of the table: as a bf16 row's -infinity they count as nothing, else the row's loss is NaN
    table[:] = 0.0
    table[9, 1], table[11, 2] = float("-inf"), float("inf")
    h = torch.zeros(2, 3, device="cuda")
    h[0, 1], h[1, 2] = 1.0, 1.0
    for r, col in ((0, [1]), (1, [2])):
        loss, _ = gpu.lm_head_loss(h[r:r + 1, col].to(dtype), table[:, col], t[3:4])
        if r == 0 and dtype == BF16:
            assert abs(float(loss) - np.log(299)) < 1e-5
        else:
            assert bool(torch.isnan(loss).all())


def test_gradient_is_the_differences(gpu):
    """Central differences of the float32 loss; step 2^-5: the third derivative's part is below 2^-10 x the
    largest third derivative / 6, and the losses' rounding 2 x 4e-5 / 2^-4 = 1.3e-3."""
    h, table, t, gl = inputs(6, 200, 16, F, ignored=0.0)
    loss, lse = gpu.lm_head_loss(h, table, t)
    gh, gw = gpu.lm_head_loss_grad(h, table, t, lse, gl)
    eps = 2.0 ** -5
    for r, c in ((0, 0), (3, 7), (5, 15)):
        up, down = h.clone(), h.clone()
        up[r, c] += eps
        down[r, c] -= eps
        d = ((gpu.lm_head_loss(up, table, t)[0] - gpu.lm_head_loss(down, table, t)[0]).double() * gl.double()).sum() / (2 * eps)
        assert abs(float(d) - float(gh[r, c])) < 3e-3
    for v, c in ((int(t[0]), 2), (11, 5)):
        up, down = table.clone(), table.clone()
        up[v, c] += eps
        down[v, c] -= eps
        width = float(up[v, c].double() - down[v, c].double())
        d = ((gpu.lm_head_loss(h, up, t)[0] - gpu.lm_head_loss(h, down, t)[0]).double() * gl.double()).sum() / width
        assert abs(float(d) - float(gw[v, c])) < 3e-3 + 2 ** -8 * abs(float(d))


@pytest.mark.parametrize("rows", [20, 200])
def test_one_gradient_alone(gpu, rows):
    h, table, t, gl = inputs(rows, 500, 64, F)
    _, lse = gpu.lm_head_loss(h, table, t)
    gh, gw = gpu.lm_head_loss_grad(h, table, t, lse, gl)
    a, b = gpu.lm_head_loss_grad(h, table, t, lse, gl, need_table=False)
    assert b is None and torch.equal(a, gh)
    into = torch.full((500, 80), 3.0, dtype=BF16, device="cuda")
    a, b = gpu.lm_head_loss_grad(h, table, t, lse, gl, need_h=False, grad_table=into[:, 5:69])
    assert a is None and torch.equal(b, gw) and bool((into[:, :5] == 3).all()) and bool((into[:, 69:] == 3).all())
    into = torch.full((rows, 71), 3.0, device="cuda")
    a, _ = gpu.lm_head_loss_grad(h, table, t, lse, gl, need_table=False, grad_h=into[:, :64])
    assert torch.equal(a, gh) and bool((into[:, 64:] == 3).all())


def test_no_rows(gpu):
    h, table, t, gl = inputs(0, 100, 64, F)
    loss, lse = gpu.lm_head_loss(h, table, t)
    assert loss.numel() == 0
    gh, gw = gpu.lm_head_loss_grad(h, table, t, lse, gl)
    assert gh.shape == (0, 64) and bool((gw == 0).all())


@pytest.mark.parametrize("rows,dtype", [(5, F), (300, BF16), (1100, BF16)])
def test_graph_stream_and_repeats(gpu, rows, dtype):
    h, table, t, gl = inputs(rows, 3000, 128, dtype)
    loss0, lse0 = gpu.lm_head_loss(h, table, t)
    g0 = gpu.lm_head_loss_grad(h, table, t, lse0, gl)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        loss1, lse1 = gpu.lm_head_loss(h, table, t)
        g1 = gpu.lm_head_loss_grad(h, table, t, lse1, gl)
    for i in range(3):
        for x in (loss1, lse1, *g1):
            x.zero_()
        graph.replay()
        loss2, lse2 = gpu.lm_head_loss(h, table, t)
        g2 = gpu.lm_head_loss_grad(h, table, t, lse2, gl)
        torch.cuda.synchronize()
        for got, want in zip((loss1, lse1, *g1, loss2, lse2, *g2), (loss0, lse0, *g0) * 2):
            assert torch.equal(got, want), i


def test_table_past_32_bits(gpu):
    """2.2 million rows of 1000: offsets past 2^31 elements."""
    V, H = 2_200_000, 1000
    g = torch.Generator(device="cuda").manual_seed(3)
    table = torch.empty(V, H, dtype=BF16, device="cuda")
    for i in range(0, V, 200_000):
        table[i:i + 200_000] = torch.randn(min(200_000, V - i), H, generator=g, device="cuda").to(BF16) * 0.05
    h = torch.randn(3, H, generator=g, device="cuda")
    t = torch.tensor([V - 1, 5, V - 4321], dtype=torch.int32, device="cuda")
    loss, lse = gpu.lm_head_loss(h, table, t)
    z = torch.cat([h.double() @ table[i:i + 100_000].double().t() for i in range(0, V, 100_000)], 1)
    want = torch.logsumexp(z, 1)
    near(lse, want.cpu(), 4e-5)
    near(loss, (want - z.gather(1, t.long()[:, None])[:, 0]).cpu(), 4e-5)
    gl = torch.ones(3, device="cuda")
    gh, gw = gpu.lm_head_loss_grad(h, table, t, lse, gl)
    D = torch.exp(z - want[:, None])
    D[torch.arange(3), t.long()] -= 1
    gh_want = sum(D[:, i:i + 100_000] @ table[i:i + 100_000].double() for i in range(0, V, 100_000))
    near(gh, gh_want.cpu(), 2e-4 * row_top(gh_want.cpu()))
    for v in (0, 5, V - 4321, V - 1):
        w = (D[:, v] @ h.double()).cpu()
        near(gw[v], w, w.abs() * 2 ** -8 + 2e-4 * float(w.abs().max()))


def test_reading_a_text(gpu):
    """A prompt through a linear-attention layer, its score and the score's gradient, then the answer's first token
    from the state that the prompt left."""
    T, H, D, V = 210, 2, 64, 500
    g = torch.Generator().manual_seed(8)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k, v = (torch.nn.functional.normalize(rnd(T + 1, H, D), dim=-1).cuda() for _ in range(3))
    al, be = torch.sigmoid(rnd(T + 1, H) + 2).cuda(), torch.sigmoid(rnd(T + 1, H)).cuda()
    table = rnd(V, H * D).to(BF16).cuda()
    t = torch.randint(0, V, (T,), generator=g, dtype=torch.int32).cuda()
    t[:50] = -100
    ones = torch.full((T,), 1.0 / 160, device="cuda")
    out, state = gpu.linear_attention_prompt(q[:T], k[:T], v[:T], al[:T], be[:T], scale=D ** -0.5)
    h = out.view(T, H * D)
    loss, lse = gpu.lm_head_loss(h, table, t)
    gh, gw = gpu.lm_head_loss_grad(h, table, t, lse, ones)
    nxt = gpu.linear_attention_step(q[T:], k[T:], v[T:], al[T:], be[T:], state, scale=D ** -0.5)
    # the same in 64 bits
    Q, K, W, A, B = (x.double().cpu() for x in (q, k, v, al, be))
    S, outs = torch.zeros(H, D, D, dtype=torch.float64), []
    for i in range(T + 1):
        S = S * A[i][:, None, None]
        u = B[i][:, None] * (W[i] - (S * K[i][:, :, None]).sum(1))
        S = S + K[i][:, :, None] * u[:, None, :]
        outs.append(D ** -0.5 * (S * Q[i][:, :, None]).sum(1))
    O = torch.stack(outs)
    near(nxt, O[T:], 2e-5 * float(O.abs().max()))
    l0, _, g0, w0, _, _ = oracle(O[:T].reshape(T, -1), table, t, ones)
    near(loss, l0, 1e-4)
    near(gh, g0, 4e-4 * row_top(g0))
    near(gw, w0, w0.abs() * 2 ** -8 + 4e-4 * row_top(w0))


def test_python_refusals(gpu):
    h, table, t, gl = inputs(4, 50, 16, F)
    loss, lse = gpu.lm_head_loss(h, table, t)
    for bad in (lambda: gpu.lm_head_loss(h.cpu(), table, t), lambda: gpu.lm_head_loss(h, table.float(), t),
                lambda: gpu.lm_head_loss(h, table, t.long()), lambda: gpu.lm_head_loss(h, table[:, :8], t),
                lambda: gpu.lm_head_loss(h.half(), table, t), lambda: gpu.lm_head_loss(h, table.t(), t),
                lambda: gpu.lm_head_loss_grad(h, table, t, lse[:3], gl),
                lambda: gpu.lm_head_loss_grad(h, table, t, lse, gl, grad_h=torch.empty(4, 16, dtype=BF16, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        gpu.lm_head_loss(h, table, t, work=torch.empty(256, dtype=torch.uint8, device="cuda"))


@pytest.mark.parametrize("weights", ["equal", "two", "negative"])
@pytest.mark.parametrize("rows", [150, 1300])
def test_weights_do_not_bias_bf16_gradients(gpu, rows, weights):
    """bf16 states under a mean loss: every row's target has D = -g (1 - p) with the same g, whose rounding no sum
    takes out.  1.0035 is rounded by 0.0035 of itself as a bf16.

    What is allowed, in the norm of a gradient: a rounding to bf16 is off by at most 2^-8 of the value, and as a
    uniform error by 2^-8 / sqrt 3 of the values' norm; that is taken for the result and for the terms p of D.
    A target's entry -1 + p is off by at most min(p, 2^-9); where its row has another weight than the call's largest it
    is rounded like any number, by up to 2^-8 of itself, in all rows of that weight the same way.  Along the gradient
    itself independent roundings have a standard deviation of 2^-8 / sqrt 3 over sqrt(elements) for either of the two: 6 of
    those, the targets' part, and 2^-13 for sums in float32."""
    V, H = 4000, 128
    h, table, _, _ = inputs(rows, V, H, BF16, ignored=0.0)
    table = (table.float() * 0.5).to(BF16)
    g = torch.Generator().manual_seed(5)
    t = torch.randperm(V, generator=g)[:rows].to(torch.int32).cuda()  # (each its own row of the table)
    gl = torch.full((rows,), 1.0035 / 1024)
    if weights == "two":
        gl[::3] *= 0.3
    elif weights == "negative":
        gl = -gl
    gl = gl.cuda()
    _, _, gh, gw, _, _ = oracle(h, table, t, gl)
    _, lse = gpu.lm_head_loss(h, table, t)
    got_h, got_w = gpu.lm_head_loss_grad(h, table, t, lse, gl)
    H64, W, G, T = h.double().cpu(), table.double().cpu(), gl.double().cpu(), t.long().cpu()
    p = torch.softmax(H64 @ W.t(), 1)
    off = p[torch.arange(rows), T].clamp(max=2.0 ** -9)
    off[G.abs() < G.abs().max()] = 2.0 ** -8
    p[torch.arange(rows), T] = 0.0
    D2 = (p * G[:, None]) ** 2
    step = 2.0 ** -8 / 3 ** 0.5
    for got, want, of_rows, terms, share in ((got_h, gh, gh, D2 @ W ** 2, G.abs() * W[T].norm(dim=1)),
                                             (got_w, gw, gw[T], D2.t() @ H64 ** 2, G.abs() * H64.norm(dim=1))):
        got, top = got.double().cpu(), float(want.norm())
        err = float((got - want).norm())
        assert err <= step * (top + float(terms.sum()) ** 0.5) + float((off * share).norm()), err / top
        along = float((got * want).sum()) / top ** 2 - 1
        targets = float((off * share * of_rows.norm(dim=1)).sum()) / top ** 2
        assert abs(along) <= 12 * step / want.numel() ** 0.5 + targets + 2.0 ** -13, along


def test_weights_at_their_ends(gpu):
    """bf16 states: weights of 0 alone, far apart, and next to one that is not finite, whose row and table rows alone
    show it."""
    h, table, t, gl = inputs(70, 300, 64, BF16, ignored=0.0)
    _, lse = gpu.lm_head_loss(h, table, t)
    gh, gw = gpu.lm_head_loss_grad(h, table, t, lse, torch.zeros_like(gl))
    assert bool((gh == 0).all()) and bool((gw == 0).all())
    far = gl.clone()
    far[::2] *= 1e-30
    far[0] = 0.0
    check_all(gpu, h, table, t, far)
    check_all(gpu, h, table, t, gl * 1e-40)  # (subnormal)
    far[7] = float("inf")
    gh, gw = gpu.lm_head_loss_grad(h, table, t, lse, far)
    keep = torch.arange(70, device="cuda") != 7
    want = gpu.lm_head_loss_grad(h, table, t, lse, torch.where(keep, far, 0.0))[0]
    assert torch.equal(gh[keep], want[keep]) and not bool(torch.isfinite(gh[7]).any())
    assert not bool(torch.isfinite(gw).any())  # every p is above 0


@pytest.mark.parametrize("rows,vocab,hidden,pad,base", [
    (1025, 2305, 73, 0, 0), (1100, 900, 321, 0, 0), (1030, 1400, 72, 5, 0), (1024, 641, 64, 0, 1), (1111, 2200, 128, 8, 0)])
def test_many_bf16_rows_and_any_table(gpu, rows, vocab, hidden, pad, base):
    """bf16 rows enough for wide tiles of grad_table, over table rows at any elements, whose logits' tiles are narrower:
    columns of D that no tile of logits writes hold what the work buffer held, here NaN.

    Besides the bounds of every element, the gradients' norms: the result's rounding and D's, 2^-8 / sqrt 3 of the
    norms of values and of terms, and for the targets' entries, which need not be independent, 2^-8 of their sums."""
    h, table, t, gl = inputs(rows, vocab, hidden, BF16, pad=pad)
    if base:
        flat = torch.empty(vocab * hidden + base, dtype=BF16, device="cuda")
        odd = flat[base:].view(vocab, hidden)
        odd.copy_(table)
        table = odd
    loss, lse, gh, gw, mags_h, mags_w = oracle(h, table, t, gl)
    nan = lambda **kw: torch.full((gpu.lm_head_loss_work_bytes(rows, vocab, hidden, BF16, **kw),), 255,  # noqa: E731
                                  dtype=torch.uint8, device="cuda")
    got_loss, got_lse = gpu.lm_head_loss(h, table, t, work=nan())
    near(got_loss, loss, 4e-5)
    got_h, got_w = gpu.lm_head_loss_grad(h, table, t, got_lse, gl, work=nan(grad=True))
    near(got_h, gh, gh.abs() * 2 ** -8 + 2e-4 * row_top(gh) + mags_h * 2 ** -8)
    near(got_w, gw, gw.abs() * 2 ** -8 + 2e-4 * row_top(gw) + mags_w * 2 ** -8)
    keep = (t >= 0).cpu()
    H, W, T = h.double().cpu()[keep], table.double().cpu(), t.long().cpu()[keep]
    D = torch.softmax(H @ W.t(), 1) * gl.double().cpu()[keep, None]
    hit = D[torch.arange(len(T)), T] - gl.double().cpu()[keep]
    D[torch.arange(len(T)), T] = 0.0
    step = 2.0 ** -8 / 3 ** 0.5
    sums = torch.zeros(vocab, hidden, dtype=torch.float64).index_add_(0, T, hit.abs()[:, None] * H.abs())
    for got, want, terms, targets in ((got_h, gh, D ** 2 @ W ** 2, hit * W[T].norm(dim=1)),
                                      (got_w, gw, (D ** 2).t() @ H ** 2, sums)):
        off = float((got.double().cpu() - want).norm())
        assert off <= step * (float(want.norm()) + float(terms.sum()) ** 0.5) + 2.0 ** -8 * float(targets.norm()), off


@pytest.mark.parametrize("rows,vocab,hidden", [(40, 900, 73), (150, 4000, 128), (1300, 4000, 128), (1024, 2305, 321)])
def test_states_gradients_have_their_targets_whole(gpu, rows, vocab, hidden):
    """bf16 states with a weight for each sequence: a row's gradient is mostly its target's, whose part is kept in float32.
    What is left of D's rounding are the other entries', 2^-8 / sqrt 3 of their terms' norm, besides the result's own; along
    the gradient, which no weight may stretch, 6 standard deviations of either and 2^-13 for sums in float32."""
    h, table, _, _ = inputs(rows, vocab, hidden, BF16, ignored=0.0)
    table = (table.float() * 0.5).to(BF16)
    t = torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(6), dtype=torch.int32).cuda()
    lengths = torch.tensor([1.0, 173, 41, 331]).repeat_interleave((rows + 3) // 4)[:rows]
    gl = (1.0 / lengths).cuda()
    _, _, want, _, _, _ = oracle(h, table, t, gl)
    _, lse = gpu.lm_head_loss(h, table, t)
    got, _ = gpu.lm_head_loss_grad(h, table, t, lse, gl)
    p = torch.softmax(h.double().cpu() @ table.double().cpu().t(), 1)
    p[torch.arange(rows), t.long().cpu()] = 0.0
    step = 2.0 ** -8 / 3 ** 0.5
    terms = (p ** 2 @ table.double().cpu() ** 2).sum(1).sqrt() * gl.double().cpu()
    got = got.double().cpu()
    for first in range(0, rows, (rows + 3) // 4):  # each weight by itself
        r = slice(first, first + (rows + 3) // 4)
        top = float(want[r].norm())
        assert float((got[r] - want[r]).norm()) <= step * (top + float(terms[r].norm()))
        along = float((got[r] * want[r]).sum()) / top ** 2 - 1
        assert abs(along) <= 12 * step / want[r].numel() ** 0.5 + 2.0 ** -13, along
