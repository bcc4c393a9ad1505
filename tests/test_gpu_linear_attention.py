"""Gated linear attention on the GPU against the recurrence in 64 bits.

Tolerances.  A bf16 output is a float32 value rounded once: half a step, 2^-8 of
the value.  The float32 values themselves: every product is exact to 2^-22 or
better of the magnitudes it adds (bf16 outputs: 2^-15, from operands of two
terms), sums are in float32.  Magnitudes can exceed the value they cancel to, so
errors are held against the largest of the tensor: 64 tokens x 256 long sums
accumulate at most about sqrt(320) 2^-23 = 2.1e-6 of it per chunk; decays below 1
and the delta rule forget earlier chunks' errors.  F32 = 2e-5 leaves a factor of
ten for sums that grow; OUT16 = 2^-8 of the value and 2^-14 of the largest."""
import ctypes

import numpy as np
import pytest
import torch

import oracle_lib as ol

pytestmark = pytest.mark.gpu
F32 = 2e-5
BF16, F = torch.bfloat16, torch.float32


def blocked(S):
    n, h, dk, dv = S.shape
    return S.reshape(n, h, dk // 4, 4, dv // 4, 4).permute(0, 1, 4, 2, 5, 3).reshape(n, h, dk * dv).contiguous()


def unblocked(flat, dk, dv):
    n, h = flat.shape[:2]
    return flat.reshape(n, h, dv // 4, dk // 4, 4, 4).permute(0, 1, 3, 5, 2, 4).reshape(n, h, dk, dv)


def inputs(rows, hk, hv, dk, dv, dtype, delta, n_state, seed=1, packed=True):
    g = torch.Generator().manual_seed(seed)
    width = 2 * hk * dk + hv * dv
    qkv = torch.randn(rows, width + (0 if packed else 3), generator=g)[:, : width]
    q = qkv[:, : hk * dk].reshape(rows, hk, dk)
    k = qkv[:, hk * dk : 2 * hk * dk].reshape(rows, hk, dk)
    q, k = (x / x.norm(dim=-1, keepdim=True).clamp(min=1e-6) for x in (q, k))
    k = 0.7 * k + 0.3 * k[:1] if rows else k  # keys that have much in common
    buf = torch.empty(rows, width + (0 if packed else 3)).to(dtype).cuda()
    buf[:, : hk * dk] = q.reshape(rows, hk * dk).to(dtype).cuda()
    buf[:, hk * dk : 2 * hk * dk] = k.reshape(rows, hk * dk).to(dtype).cuda()
    buf[:, 2 * hk * dk : width] = qkv[:, 2 * hk * dk :].to(dtype).cuda()
    alpha = torch.sigmoid(2 * torch.randn(rows, hv, generator=g) + 2).cuda()
    beta = torch.sigmoid(torch.randn(rows, hv, generator=g)).cuda() if delta else None
    state = blocked(0.2 * torch.randn(n_state, hv, dk, dv, generator=g)).cuda()
    return (buf[:, : hk * dk].view(rows, hk, dk), buf[:, hk * dk : 2 * hk * dk].view(rows, hk, dk),
            buf[:, 2 * hk * dk : width].view(rows, hv, dv), alpha, beta, state)


def oracle(q, k, v, alpha, beta, scale, state, spans, slots=None):
    """The recurrence in 64 bits on the CPU -> (out, state); rows of no sequence are NaN."""
    q, k, v, a = (x.double().cpu() for x in (q, k, v, alpha))
    b = None if beta is None else beta.double().cpu()
    reach = v.shape[1] // q.shape[1]
    q, k = q.repeat_interleave(reach, 1), k.repeat_interleave(reach, 1)
    dk, dv = q.shape[2], v.shape[2]
    S = unblocked(state.double().cpu(), dk, dv).clone()
    out = torch.full(v.shape, float("nan"), dtype=torch.float64)
    for s, (lo, hi) in enumerate(spans):
        at = s if slots is None else slots[s]
        if at < 0 or at >= len(S):
            continue
        M = S[at]
        for t in range(lo, hi):
            M = M * a[t][:, None, None]
            u = v[t]
            if b is not None:
                u = b[t][:, None] * (u - (M * k[t][:, :, None]).sum(1))
            M = M + k[t][:, :, None] * u[:, None, :]
            out[t] = scale * (M * q[t][:, :, None]).sum(1)
        S[at] = M
    return out, blocked(S)


def near(got, want, dtype=F, halves=1):
    """halves: the roundings between got and want.  Where want is the kernels' own
    bf16 output, x being what both approximate, |got - want| <= |got - x| + |x - want|:
    two, of half a step (2^-8 of the value) each, and twice the float32 part."""
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = ~torch.isnan(want)
    got, want = got[fine], want[fine]
    if not got.numel():
        return
    top = want.abs().max()
    bound = F32 * top if dtype == F else halves * (want.abs() * 2.0 ** -8 + top * 2.0 ** -14)
    off = (got - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max() if dtype != F else off.max() / top)


def spans_of(lengths, gap_after=0):
    ends = np.cumsum([0] + list(lengths))
    return list(zip(ends[:-1].tolist(), ends[1:].tolist())), torch.tensor(ends, dtype=torch.int32).cuda()


SHAPES = [(16, 16, 128, 128), (2, 6, 64, 96), (1, 2, 256, 64), (3, 3, 32, 16), (2, 2, 20, 36), (1, 1, 4, 4),
          (1, 2, 100, 256)]


@pytest.mark.parametrize("dtype", [F, BF16])
@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("hk,hv,dk,dv", SHAPES)
def test_step(gpu, hk, hv, dk, dv, delta, dtype):
    for B in (1, 5):
        q, k, v, al, be, st = inputs(B, hk, hv, dk, dv, dtype, delta, B)
        want, wst = oracle(q, k, v, al, be, 0.5, st, [(i, i + 1) for i in range(B)])
        out = gpu.linear_attention_step(q, k, v, al, be, st, scale=0.5)
        near(out, want, dtype)
        near(st, wst)


# many sequences (32 value columns a workgroup where there are heads enough), few, and one
LENGTHS = {"many": [1, 0, 64, 63, 130, 65, 0, 200, 2], "few": [257, 70], "one": [449]}


@pytest.mark.parametrize("dtype", [F, BF16])
@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("hk,hv,dk,dv", SHAPES)
@pytest.mark.parametrize("which,packed", [("many", False), ("many", True), ("few", True), ("one", False)])
def test_prompt(gpu, which, packed, hk, hv, dk, dv, delta, dtype):
    """packed: rows of a projection as they are (16-byte aligned for most shapes); else three elements apart."""
    lengths = LENGTHS[which]
    spans, starts = spans_of(lengths)
    q, k, v, al, be, st = inputs(sum(lengths), hk, hv, dk, dv, dtype, delta, len(lengths), packed=packed)
    want, wst = oracle(q, k, v, al, be, 0.25, st, spans)
    out, got = gpu.linear_attention_prompt(q, k, v, al, be, starts, scale=0.25, state_in=st)
    near(out, want, dtype)
    near(got, wst)


@pytest.mark.parametrize("dtype", [F, BF16])
@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("hk,hv,dk,dv", SHAPES)
def test_prompt_of_short_sequences(gpu, hk, hv, dk, dv, delta, dtype):
    """Sequences that go token by token: a few short ones alone, and many with longer ones between them."""
    many = 256 // (8 * hv * -(-dv // 32)) + 1
    for lengths in ([3, 0, 9, 1], [16], [1], [1, 0, 16, 17, 5, 70, 3, 2] * many):
        spans, starts = spans_of(lengths)
        q, k, v, al, be, st = inputs(sum(lengths), hk, hv, dk, dv, dtype, delta, len(lengths), packed=len(lengths) > 4)
        want, wst = oracle(q, k, v, al, be, 0.5, st, spans)
        out, got = gpu.linear_attention_prompt(q, k, v, al, be, starts, scale=0.5, state_in=st)
        near(out, want, dtype)
        near(got, wst)
        _, other = gpu.linear_attention_prompt(q, k, v, al, be, starts, state_in=st, state_out=st, out=out)
        assert other is st and torch.equal(st, got)


@pytest.mark.parametrize("hk,hv,dk,dv", [(2, 64, 16, 32), (16, 16, 128, 128)])
def test_slots_of_short_sequences(gpu, hk, hv, dk, dv):
    slots = [5, -1, 0, 9, 5, 2, 1000000, 3]
    spans, starts = spans_of([12, 10, 0, 16, 3, 1, 2, 30])
    q, k, v, al, be, st = inputs(spans[-1][1] + 37, hk, hv, dk, dv, F, True, 9)
    q[spans[1][0]:spans[1][1]] = float("nan")
    v[spans[-1][1]:] = float("nan")
    st[7] = float("nan")
    taken = [s if s < 9 and i != 4 else -1 for i, s in enumerate(slots)]
    want, wst = oracle(q, k, v, al, be, 1.0, st, spans, taken)
    out = torch.full(v.shape, float("nan"), device="cuda")
    before = torch.full_like(st, 7.0)
    _, state = gpu.linear_attention_prompt(q, k, v, al, be, starts, state_in=st, state_out=before, out=out,
                                           slots=torch.tensor(slots, dtype=torch.int32).cuda())
    for i in (1, 4, 6, 7, 8):
        assert bool((state[i] == 7.0).all())
        wst[i] = 7.0
    near(out, want)
    near(state, wst)


def test_short_sequences_in_a_graph(gpu):
    """Short and long ones in one captured call, replayed; states past 128 MiB; NaN stays with its tokens."""
    lengths = [4, 16, 1, 0, 30] * 30
    spans, starts = spans_of(lengths)
    q, k, v, al, be, st = inputs(sum(lengths), 4, 16, 128, 128, BF16, True, len(lengths))
    v[spans[1][0] + 7, 3, 5] = float("nan")
    want, wst = oracle(q, k, v, al, be, 1.0, st, spans)
    out, got = gpu.linear_attention_prompt(q, k, v, al, be, starts, state_in=st)
    near(out, want, BF16)
    near(got, wst)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again, state = gpu.linear_attention_prompt(q, k, v, al, be, starts, state_in=st)
    for _ in range(3):
        again.zero_()
        state.zero_()
        graph.replay()
        other = gpu.linear_attention_step(q[:2], k[:2], v[:2], al[:2], be[:2], st[:2].clone())
        torch.cuda.synchronize()
        assert bool(torch.isfinite(other).all())
        assert torch.equal(torch.nan_to_num(again), torch.nan_to_num(out))
        assert torch.equal(torch.nan_to_num(state), torch.nan_to_num(got))


def test_prompt_of_one_sequence_from_zeros(gpu):
    q, k, v, al, be, st = inputs(300, 4, 4, 64, 64, F, True, 1)
    want, wst = oracle(q, k, v, al, be, 1.0, torch.zeros_like(st), [(0, 300)])
    out, got = gpu.linear_attention_prompt(q, k, v, al, be)
    near(out, want)
    near(got, wst)


@pytest.mark.parametrize("dtype", [F, BF16])
def test_prompt_then_steps_is_the_longer_prompt(gpu, dtype):
    """A prompt, then its answer token by token: the states and outputs of one long prompt."""
    q, k, v, al, be, st = inputs(150, 2, 4, 128, 128, dtype, True, 1)
    whole, last = gpu.linear_attention_prompt(q, k, v, al, be, state_in=st)
    out, state = gpu.linear_attention_prompt(q[:139], k[:139], v[:139], al[:139], be[:139], state_in=st)
    parts = [out] + [gpu.linear_attention_step(q[t:t + 1], k[t:t + 1], v[t:t + 1], al[t:t + 1], be[t:t + 1], state)
                     for t in range(139, 150)]
    near(torch.cat(parts), whole.double().cpu(), dtype, halves=2)
    near(state, last.double().cpu())


def test_state_is_the_decode_runtimes(gpu):
    """A prompt's state goes on in gdn_recurrent_step (host pointers, one token)."""
    lib = gpu.load()
    H, D = 16, 128
    q, k, v, al, be, st = inputs(71, H, H, D, D, F, True, 1)
    _, state = gpu.linear_attention_prompt(q[:70], k[:70], v[:70], al[:70], be[:70], state_in=st)
    host = state[0].cpu().numpy().copy()
    out = np.zeros(H * D, np.float32)
    row = [x[70].cpu().numpy().copy() for x in (q, k, v, al, be)]
    lib.gdn_recurrent_step(out.ctypes.data, host.ctypes.data, *[r.ctypes.data for r in row], H, D)
    want, wst = oracle(q, k, v, al, be, 1.0, st, [(0, 71)])
    near(torch.from_numpy(out).view(H, D), want[70])
    near(torch.from_numpy(host)[None], wst)
    assert np.allclose(ol.gdn_state_from_blocked(host, H, D), unblocked(wst, D, D)[0].numpy(), atol=1e-4)


@pytest.mark.parametrize("dtype", [F, BF16])
def test_long_sequence(gpu, dtype):
    """Errors do not pile up over 60 chunks."""
    q, k, v, al, be, st = inputs(3841, 1, 1, 128, 128, dtype, True, 1)
    want, wst = oracle(q, k, v, al, be, 1.0, st, [(0, 3841)])
    out, got = gpu.linear_attention_prompt(q, k, v, al, be, state_in=st)
    near(out, want, dtype)
    near(got, wst)


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("dtype", [F, BF16])
def test_decays_at_their_ends(gpu, delta, dtype):
    """A decay of 0 forgets everything before it; 1 keeps it; tiny ones underflow; a beta of 0 writes nothing."""
    q, k, v, al, be, st = inputs(200, 2, 2, 64, 64, dtype, delta, 1)
    al[:] = 1.0
    al[70, :] = 0.0
    al[100:110, 0] = 1e-38
    al[110:112, 1] = 1e-45  # subnormal
    al[199, 1] = 0.0
    if delta:
        be[::3] = 0.0
        be[1::3] = 1.0
    want, wst = oracle(q, k, v, al, be, 1.0, st, [(0, 200)])
    out, got = gpu.linear_attention_prompt(q, k, v, al, be, state_in=st)
    near(out, want, dtype)
    near(got, wst)
    for t in range(0, 200):
        o = gpu.linear_attention_step(q[t:t + 1], k[t:t + 1], v[t:t + 1], al[t:t + 1], None if be is None else be[t:t + 1],
                                      st)
        near(o, want[t:t + 1], dtype)
    near(st, wst)


@pytest.mark.parametrize("form", ["prompt", "step"])
def test_slots(gpu, form):
    """Slots in any order; empty places, slots outside the pool and a slot named before are skipped, their rows and
    states left as they were, as are rows behind the last sequence."""
    slots = [5, -1, 0, 9, 5, 2, 1000000, 3]
    lengths = [1] * 8 if form == "step" else [70, 10, 0, 64, 3, 1, 20, 129]
    spans, starts = spans_of(lengths)
    rows = spans[-1][1] + (0 if form == "step" else 37)
    q, k, v, al, be, st = inputs(rows, 2, 4, 64, 32, F, True, 9)
    st[7] = float("nan")  # a state of no sequence
    q[spans[1][0]:spans[1][1]] = float("nan")  # and rows that are skipped
    if form == "prompt":
        v[spans[-1][1]:] = float("nan")
    taken = [s if s < 9 and i != 4 else -1 for i, s in enumerate(slots)]
    want, wst = oracle(q, k, v, al, be, 1.0, st, spans, taken)
    sl = torch.tensor(slots, dtype=torch.int32).cuda()
    out = torch.full((rows, 4, 32), float("nan"), device="cuda")
    if form == "step":
        gpu.linear_attention_step(q, k, v, al, be, st, slots=sl, out=out)
        state = st
    else:
        before = torch.full_like(st, 7.0)
        _, state = gpu.linear_attention_prompt(q, k, v, al, be, starts, state_in=st, state_out=before, slots=sl, out=out)
        for i in (1, 4, 6, 7, 8):
            assert bool((state[i] == 7.0).all())
            wst[i] = 7.0
    near(out, want)
    near(state, wst)


def test_in_place_states_and_strided_gates(gpu):
    q, k, v, al, be, st = inputs(140, 2, 2, 32, 32, F, True, 2)
    spans, starts = spans_of([75, 65])
    want, wst = oracle(q, k, v, al, be, 1.0, st, spans)
    gates = torch.full((140, 7), float("nan"), device="cuda")
    gates[:, :2], gates[:, 4:6] = al, be
    wide = torch.full((140, 3, 32), 5.0, device="cuda")
    _, got = gpu.linear_attention_prompt(q, k, v, gates[:, :2], gates[:, 4:6], starts, state_in=st, state_out=st,
                                         out=wide[:, :2])
    assert got is st
    near(wide[:, :2], want)
    near(st, wst)
    assert bool((wide[:, 2] == 5.0).all())


def test_step_of_parts_of_rows(gpu):
    """Whole tensors and parts of a projection's rows give the same; one row's gates may lie anywhere."""
    for rows in (1, 3):
        q, k, v, al, be, st = inputs(rows, 2, 4, 64, 32, F, True, rows, packed=False)
        want = gpu.linear_attention_step(q.contiguous(), k.contiguous(), v.contiguous(), al, be, st.clone())
        gates = torch.cat([al, be, al], 1)
        assert torch.equal(gpu.linear_attention_step(q, k, v, gates[:, :4], gates[:, 4:8], st.clone()), want)
        if rows == 1:
            assert torch.equal(gpu.linear_attention_step(q, k, v, al, gates[:, 4:8], st.clone()), want)
        else:
            with pytest.raises(ValueError, match="stride"):
                gpu.linear_attention_step(q, k, v, al, gates[:, 4:8], st.clone())


@pytest.mark.parametrize("dtype", [F, BF16])
def test_nan_stays_in_its_sequence_head_and_time(gpu, dtype):
    q, k, v, al, be, st = inputs(400, 2, 2, 64, 64, dtype, True, 2)
    spans, starts = spans_of([200, 200])
    v[130, 1, 3] = float("nan")
    want, wst = oracle(q, k, v, al, be, 1.0, st, spans)
    out, got = gpu.linear_attention_prompt(q, k, v, al, be, starts, state_in=st)
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[128:200, 1] = True  # from its chunk on
    keep = ~bad
    near(out[keep], want[keep.cpu()], dtype)
    assert bool(torch.isnan(out[130:200, 1, 3]).all())
    assert bool(torch.isfinite(got[1]).all()) and bool(torch.isfinite(got[0, 0]).all())
    near(got[1], wst[1])


def test_offsets_past_32_bits(gpu):
    """A pool of states and rows far apart, both past 2^31 elements."""
    n = 8200  # 8200 x 16 x 128 x 128 floats
    pool = torch.empty(n, 16, 128 * 128, device="cuda")
    q, k, v, al, be, st = inputs(3, 16, 16, 128, 128, F, True, 3)
    at = [n - 1, 0, n - 7]
    for i, s in enumerate(at):
        pool[s] = st[i]
    want, wst = oracle(q, k, v, al, be, 1.0, st, [(0, 1), (1, 2), (2, 3)])
    out = gpu.linear_attention_step(q, k, v, al, be, pool, slots=torch.tensor(at, dtype=torch.int32).cuda())
    near(out, want)
    near(torch.stack([pool[s] for s in at]), wst)
    del pool
    q, k, v, al, be, st = inputs(150, 1, 1, 128, 128, BF16, True, 1)
    want, wst = oracle(q, k, v, al, be, 1.0, st, [(0, 150)])
    for far in ((1 << 24) - 8, 1 << 24):  # within and past what lanes hold as an offset
        big = torch.empty(149 * far + 128, dtype=BF16, device="cuda")
        vv = big.as_strided((150, 1, 128), (far, 128, 1))
        vv.copy_(v)
        out, got = gpu.linear_attention_prompt(q, k, vv, al, be, state_in=st)
        near(out, want, BF16)
        near(got, wst)
        del big, vv


def test_graph_stream_and_repeats(gpu):
    """Captured on a stream of its own, replayed with other work between, and bit for bit the eager result."""
    spans, starts = spans_of([100, 29, 300])
    q, k, v, al, be, st = inputs(429, 4, 8, 64, 64, BF16, True, 3)
    out0, state0 = gpu.linear_attention_prompt(q, k, v, al, be, starts, state_in=st)
    step0 = gpu.linear_attention_step(q[:3], k[:3], v[:3], al[:3], be[:3], state0.clone())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out1, state1 = gpu.linear_attention_prompt(q, k, v, al, be, starts, state_in=st)
        again = state1.clone()
        step1 = gpu.linear_attention_step(q[:3], k[:3], v[:3], al[:3], be[:3], again)
    for i in range(3):
        out1.zero_()
        graph.replay()
        other = gpu.linear_attention_prompt(q, k, v, al, be, starts, state_in=st)
        torch.cuda.synchronize()
        for got, want in ((out1, out0), (state1, state0), (step1, step0), (other[0], out0), (other[1], state0)):
            assert torch.equal(got, want), i
    with torch.cuda.stream(side):
        got = gpu.linear_attention_prompt(q, k, v, al, be, starts, state_in=st)
    side.synchronize()
    assert torch.equal(got[0], out0) and torch.equal(got[1], state0)


@pytest.mark.parametrize("rows,n", [(200, 3), (600, 40), (2000, 40), (700, 70)])
def test_replays_with_other_lengths(gpu, rows, n):
    """A captured call reads the lengths when it runs: short for long, long for short, most of them none."""
    q, k, v, al, be, st = inputs(rows, 4, 8, 64, 64, BF16, True, n)
    ends = torch.zeros(n + 1, dtype=torch.int32)
    ends[1:] = torch.arange(1, n + 1) * (rows // n)
    starts = ends.cuda()
    gpu.linear_attention_prompt(q, k, v, al, be, starts, state_in=st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, got = gpu.linear_attention_prompt(q, k, v, al, be, starts, state_in=st)
    g = torch.Generator().manual_seed(3)
    for kind in range(4):
        if kind == 1:
            ends[1:] = torch.randint(0, rows + 1, (n,), generator=g).sort().values
        elif kind == 2:
            ends[1:] = rows
        elif kind == 3:
            ends[1:] = torch.arange(1, n + 1)
        starts.copy_(ends)
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        at = ends.tolist()
        want, wst = oracle(q, k, v, al, be, 1.0, st, list(zip(at[:-1], at[1:])))
        near(out, want, BF16)
        near(got, wst)


def test_step_over_a_large_batch(gpu):
    """States of more than 128 MiB, which pass the caches by."""
    B = 140
    q, k, v, al, be, st = inputs(B, 4, 16, 128, 128, BF16, True, B)
    want, wst = oracle(q, k, v, al, be, 0.5, st, [(i, i + 1) for i in range(B)])
    near(gpu.linear_attention_step(q, k, v, al, be, st, scale=0.5), want, BF16)
    near(st, wst)


def test_no_sequences_and_no_tokens(gpu):
    q, k, v, al, be, st = inputs(0, 2, 2, 32, 32, F, True, 3)
    out, got = gpu.linear_attention_prompt(q, k, v, al, be, torch.zeros(4, dtype=torch.int32).cuda(), state_in=st)
    assert out.shape[0] == 0 and torch.equal(got, st)
    _, got = gpu.linear_attention_prompt(q, k, v, al, be, torch.zeros(4, dtype=torch.int32).cuda())
    assert bool((got == 0).all())
    out, got = gpu.linear_attention_prompt(q, k, v, al, be, torch.zeros(1, dtype=torch.int32).cuda(), state_out=st[:0])
    assert got.shape[0] == 0
    assert gpu.linear_attention_step(q, k, v, al, be, st[:0]).shape[0] == 0


def test_starts_outside_the_rows_are_held_inside(gpu):
    """starts that leave the rows or fall do not reach memory outside: sequences are cut, or empty."""
    q, k, v, al, be, st = inputs(100, 1, 1, 32, 32, F, True, 3)
    starts = torch.tensor([-50, 40, 30, 100000], dtype=torch.int32).cuda()
    want, wst = oracle(q, k, v, al, be, 1.0, st, [(0, 40), (40, 40), (30, 100)])
    out, got = gpu.linear_attention_prompt(q, k, v, al, be, starts, state_in=st)
    near(got[:2], wst[:2])  # (the last one's rows meet the first one's)
    assert bool(torch.isfinite(out).all())


def test_python_refusals(gpu):
    q, k, v, al, be, st = inputs(4, 2, 4, 32, 32, F, True, 4)
    step = gpu.linear_attention_step
    for bad in (lambda: step(q.cpu(), k, v, al, be, st), lambda: step(q, k.cpu(), v, al, be, st),
                lambda: step(q, k.to(BF16), v, al, be, st), lambda: step(q, k, v, al.double(), be, st),
                lambda: step(q[:, :, ::2], k[:, :, ::2], v, al, be, st), lambda: step(q, k, v, al, be, st[:3]),
                lambda: step(q, k, v, al, be, st, slots=torch.zeros(4, dtype=torch.int64, device="cuda")),
                lambda: step(q, k, v, al, be, st, out=torch.empty(4, 4, 16, device="cuda")),
                lambda: gpu.linear_attention_prompt(q, k, v, al, be, torch.zeros(7, dtype=torch.int32).cuda(), state_in=st),
                lambda: gpu.linear_attention_prompt(q, k, v, al, be, slots=torch.zeros(1, dtype=torch.int32).cuda()),
                lambda: step(q, k, v, al, be, st.transpose(0, 1).contiguous().transpose(0, 1))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        gpu.linear_attention_prompt(q, k, v, al, be, work=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(RuntimeError):  # 3 key heads do not divide 4 value heads
        step(torch.zeros(4, 3, 32, device="cuda"), torch.zeros(4, 3, 32, device="cuda"), v, al, be, st)


def test_products_of_a_state_keep_their_bits(gpu):
    """One token's k u^T through the chunked form: each element a single product of two float32.  Six pairs of three
    terms leave out 2^-23 of it, and the sums of the pairs in float32 are allowed a last place, 2^-23."""
    q, k, v, al, _, _ = inputs(64, 16, 16, 128, 128, F, False, 1)
    k, v = (3 * torch.randn(x.shape, generator=torch.Generator().manual_seed(i)).cuda() for i, x in enumerate((k, v)))
    v[:5], v[6:] = 0.0, 0.0
    _, got = gpu.linear_attention_prompt(q, k, v, torch.ones_like(al))
    want = k[5].double()[:, :, None] * v[5].double()[:, None, :]
    off = (unblocked(got, 128, 128)[0].double() - want).abs() / want.abs()
    assert float(off.max()) <= 2.0 ** -22, float(off.max()) * 2 ** 22


def _new_memory_is_nan(like):
    """What the allocator hands out next held NaN."""
    x = [torch.full_like(like, float("nan")) for _ in range(3)]
    torch.cuda.synchronize()
    del x


@pytest.mark.parametrize("dtype", [F, BF16])
@pytest.mark.parametrize("heads,dv", [(2, 32), (16, 100)])
@pytest.mark.parametrize("lengths", [[1] * 8, [12, 10, 0, 16, 3, 1, 2, 30], [70, 10, 0, 64, 3, 1, 20, 129], [3, 10, 90, 2, 1, 4, 5, 6],
                                     [0, 100, 0, 0, 0, 0, 0, 0]])
def test_rows_of_no_sequence_are_zero_in_a_new_output(gpu, lengths, heads, dv, dtype):
    """Rows in front of the first sequence, behind the last and of skipped ones, whichever way each goes."""
    slots = torch.tensor([-1, 4, 0, 9, 4, 2, 1000000, -5], dtype=torch.int32).cuda()
    ends = np.cumsum([9] + lengths)
    rows = int(ends[-1]) + 21
    q, k, v, al, be, st = inputs(rows, heads, heads, 64, dv, dtype, True, 9)
    starts = torch.tensor(ends, dtype=torch.int32).cuda()
    taken = [-1, 4, 0, -1, -1, 2, -1, -1]
    want, _ = oracle(q, k, v, al, be, 1.0, st, list(zip(ends[:-1].tolist(), ends[1:].tolist())), taken)
    _new_memory_is_nan(v.contiguous())
    out, _ = gpu.linear_attention_prompt(q, k, v, al, be, starts, state_in=st, state_out=st.clone(), slots=slots)
    near(out, want.nan_to_num(0.0), dtype)
    if lengths[0] == 1:
        q, k, v, al, be = (x[:8].contiguous() for x in (q, k, v, al, be))
        want, _ = oracle(q, k, v, al, be, 1.0, st, [(i, i + 1) for i in range(8)], taken)
        _new_memory_is_nan(v)
        near(gpu.linear_attention_step(q, k, v, al, be, st, slots=slots), want.nan_to_num(0.0), dtype)
        none = torch.zeros(1, dtype=torch.int32).cuda()
        _new_memory_is_nan(v)
        assert bool((gpu.linear_attention_prompt(q, k, v, al, be, none)[0] == 0).all())


@pytest.mark.parametrize("dtype", [F, BF16])
@pytest.mark.parametrize("lengths", [[17] * 60 + [0] * 80, [1] * 300 + [400] + [2] * 60, [65, 0, 0, 0, 0, 0, 0, 0, 16, 0, 0, 0, 130] * 12,
                                     [0] * 130 + [449], [200, 17, 3], [16] * 9])
def test_work_is_as_large_as_it_says(gpu, lengths, dtype):
    """Long sequences next to each other, behind and in front of many short ones: each chunk has a place of its own,
    within the bytes asked for, whatever they held."""
    spans, starts = spans_of(lengths)
    rows = spans[-1][1]
    q, k, v, al, be, st = inputs(rows, 2, 4, 64, 64, dtype, True, len(lengths))
    need = gpu.linear_attention_prompt_work_bytes(rows, len(lengths), 2, 4, 64, 64, dtype)
    work = torch.full((need + 65536,), 255, dtype=torch.uint8, device="cuda")
    want, wst = oracle(q, k, v, al, be, 0.5, st, spans)
    out, got = gpu.linear_attention_prompt(q, k, v, al, be, starts, scale=0.5, state_in=st, work=work[:need])
    near(out, want, dtype)
    near(got, wst)
    assert bool((work[need:] == 255).all())


@pytest.mark.parametrize("dtype", [F, BF16])
@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("hk,hv,dk,dv,packed", [(2, 2, 64, 64, True), (16, 16, 128, 128, True), (2, 4, 128, 32, False), (1, 2, 20, 36, True),
                                                (1, 1, 256, 32, True)])
def test_nan_and_infinity_do_not_go_back(gpu, hk, hv, dk, dv, packed, delta, dtype):
    """Whatever is not finite in a token shows from that token on, in its head (q: that token, v: its column; a state:
    its column), as the recurrence has it: within a chunk, at its ends, in a last chunk that is not whole."""
    spans, starts = spans_of([90, 200, 143])
    h = hv - 1
    for i, (kind, token) in enumerate([("q", 90 + 130), ("k", 90 + 64), ("v", 90 + 127), ("alpha", 90 + 100), ("beta", 90 + 31),
                                       ("state", 0), ("k", 289), ("v", 90), ("v2", 90 + 40)]):
        q, k, v, al, be, st = inputs(433, hk, hv, dk, dv, dtype, delta, 3, packed=packed)
        value = float("nan") if i % 2 else float("inf")
        if kind in ("q", "k"):
            (q if kind == "q" else k)[token, hk - 1, dk // 2] = value
        elif kind == "v":
            v[token, h, dv // 2 + 1] = value
        elif kind == "v2":  # two columns, two tokens of a chunk
            v[token, h, 1], v[token + 9, h, dv - 1], v[token + 12, h, 1] = -value, value, value
        elif kind == "alpha":
            al[token, h] = float("nan")
        elif kind == "beta":
            if not delta:
                continue
            be[token, h] = value
        else:
            view = st.view(3, hv, dv // 4, dk // 4, 4, 4)
            view[1, h, dv // 8, dk // 8, 2, 1] = value  # S[.., 4 (dv / 8) + 2] of sequence 1
        want, wst = oracle(q, k, v, al, be, 0.5, st, spans)
        out, got = gpu.linear_attention_prompt(q, k, v, al, be, starts, scale=0.5, state_in=st)
        assert torch.equal(torch.isfinite(out).cpu(), torch.isfinite(want)), kind
        nan = float("nan")
        near(torch.where(torch.isfinite(out), out, nan), torch.where(torch.isfinite(want), want, nan), dtype)
        if kind in ("k", "alpha", "beta"):  # (of such a state all is lost, whichever rows the recurrence keeps)
            heads = range(h + 1 - hv // hk, hv) if kind == "k" else [h]
            for x in heads:
                assert not bool(torch.isfinite(got[1, x]).any()), kind
                got[1, x], wst[1, x] = 0.0, 0.0
        assert torch.equal(torch.isfinite(got).cpu(), torch.isfinite(wst)), kind
        near(torch.where(torch.isfinite(got), got, nan), torch.where(torch.isfinite(wst), wst, nan))


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("kind", ["k", "v"])
def test_values_past_bf16s_largest_do_not_go_back(gpu, kind, delta):
    """A float32's largest value counts as infinite: what it is in shows it from its token on, and not before."""
    q, k, v, al, be, st = inputs(150, 2, 2, 64, 64, F, delta, 1)
    (k if kind == "k" else v)[100, 1, 7] = torch.finfo(F).max
    want, _ = oracle(q, k, v, al, be, 1.0, st, [(0, 150)])
    out, got = gpu.linear_attention_prompt(q, k, v, al, be, state_in=st)
    near(out[:100], want[:100])
    near(out[:, 0], want[:, 0])
    columns = slice(None) if kind == "k" else 7
    assert not bool(torch.isfinite(out[100:, 1, columns]).any())
    if kind == "v":
        keep = torch.arange(64) != 7
        near(out[:, 1, keep.cuda()], want[:, 1, keep])
