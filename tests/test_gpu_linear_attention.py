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
    buf[:, : hk * dk] = q.reshape(rows, -1).to(dtype).cuda()
    buf[:, hk * dk : 2 * hk * dk] = k.reshape(rows, -1).to(dtype).cuda()
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


@pytest.mark.parametrize("dtype", [F, BF16])
@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("hk,hv,dk,dv", SHAPES)
def test_prompt(gpu, hk, hv, dk, dv, delta, dtype):
    lengths = [1, 0, 64, 63, 130, 65, 0, 200, 2]
    spans, starts = spans_of(lengths)
    q, k, v, al, be, st = inputs(sum(lengths), hk, hv, dk, dv, dtype, delta, len(lengths), packed=False)
    want, wst = oracle(q, k, v, al, be, 0.25, st, spans)
    out, got = gpu.linear_attention_prompt(q, k, v, al, be, starts, scale=0.25, state_in=st)
    near(out, want, dtype)
    near(got, wst)


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
