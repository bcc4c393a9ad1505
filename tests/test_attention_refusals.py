"""What the operators of a full-attention layer refuse, on the host: invalid sizes, pointers, strides and work
buffers give BFP8_EINVAL and a message before anything touches a GPU."""
import ctypes

import pytest
import torch

import qwen_kernels_gpu as qk

P = 1 << 20  # a pointer that is never followed
NAN, INF = float("nan"), float("inf")


def made(args, over, **base):
    for k, v in {**base, **over}.items():
        setattr(args, k, v)
    return args


def rope(**over):
    return made(qk.rope_dev_args(), over, out=P, x=2 * P, positions=P, freqs=P, out_row=256, out_head=64, x_row=256, x_head=64,
                rows=5, heads=4, dim=64, rot=32, dtype=qk.QWEN_BF16, amplitude=1.0)


CACHE = dict(key_cache=P, value_cache=P, tables=P, cached=P, starts=P, cache_page=16 * 2 * 64, cache_token=2 * 64, cache_head=64,
             table_row=8, rows=6, n_seq=3, pages=10, page=16, table_pages=8, heads_q=4, heads_k=2, dim=64, dtype=qk.QWEN_BF16)


def append(**over):
    return made(qk.kv_dev_append_args(), over, **CACHE, k=P, v=P, q=P, q_out=2 * P, positions=P, freqs=P, k_row=128, k_head=64,
                v_row=128, v_head=64, q_row=256, q_head=64, q_out_row=256, q_out_head=64, rot=32, amplitude=1.0)


def paged(**over):
    return made(qk.attn_dev_args(), over, **CACHE, out=2 * P, q=P, mask=P, work=P, work_bytes=1 << 40, q_row=256, q_head=64,
                out_row=256, out_head=64, mask_words=1, scale=0.125)


def tree(**over):
    return made(qk.attn_dev_tree_args(), over, mask=P, positions=P, parents=P, cached=P, starts=P, rows=6, n_seq=3, words=1)


def refused(f, a):
    assert f(a, None) == qk.BFP8_EINVAL
    assert len(qk.load().bfp8_last_error()) > 20


@pytest.mark.parametrize("over", [
    dict(dtype=2), dict(dim=1), dict(dim=1025), dict(rot=0), dict(rot=66), dict(rot=31), dict(rows=-1), dict(heads=0),
    dict(heads=65537), dict(rows=1 << 27), dict(amplitude=NAN), dict(amplitude=INF), dict(out=None), dict(x=None),
    dict(positions=None), dict(freqs=None), dict(out=P + 1), dict(x=P + 1), dict(x=P + 2, dtype=0), dict(positions=P + 2),
    dict(freqs=P + 4), dict(x_row=-1), dict(x_head=-64), dict(out_row=-256), dict(out_head=(1 << 34) + 1), dict(out_row=64),
    dict(out_head=32), dict(out_row=0), dict(out=2 * P, out_row=512), dict(out=2 * P, out_row=64, out_head=512)])
def test_rotary_refuses(over):
    refused(qk.load().rope_dev_apply, rope(**over))
    refused(qk.load().rope_dev_grad, rope(**over))


def test_rotary_of_nothing():
    lib = qk.load()
    for f in (lib.rope_dev_apply, lib.rope_dev_grad):
        assert f(None, None) == qk.BFP8_EINVAL
        assert f(rope(rows=0, x=None, out=None), None) == qk.BFP8_OK


SHARED = [dict(dtype=2), dict(dim=0), dict(dim=4), dict(dim=60), dict(dim=264), dict(n_seq=-1), dict(n_seq=(1 << 20) + 1),
          dict(rows=-1), dict(heads_k=0), dict(heads_k=65537), dict(rows=1 << 28), dict(page=0), dict(page=65537),
          dict(pages=-1), dict(table_pages=-1), dict(table_pages=1 << 27), dict(starts=None, rows=7), dict(cached=None),
          dict(cached=P + 2), dict(starts=P + 2), dict(tables=P + 1), dict(tables=None), dict(table_row=7), dict(table_row=-8),
          dict(key_cache=None), dict(value_cache=None), dict(key_cache=P + 8), dict(value_cache=P + 2), dict(cache_page=2052),
          dict(cache_token=132), dict(cache_head=68), dict(cache_page=-2048), dict(cache_page=1024), dict(cache_token=64),
          dict(cache_head=0), dict(cache_page=0), dict(cache_page=(1 << 40) + 8), dict(heads_q=3), dict(heads_q=1),
          dict(rows=1 << 26, heads_q=8)]


@pytest.mark.parametrize("over", SHARED + [
    dict(rot=-2), dict(rot=3), dict(rot=66), dict(rot=0), dict(amplitude=NAN), dict(k=None), dict(v=None), dict(q_out=None),
    dict(freqs=None), dict(k=P + 1), dict(v=P + 1), dict(q=P + 1), dict(q_out=P + 1), dict(positions=P + 1), dict(freqs=P + 4),
    dict(k_row=-1), dict(v_head=-1), dict(q_row=-1), dict(q_out_row=64), dict(q_out_head=0), dict(q=2 * P, q_row=512)])
def test_append_refuses(over):
    refused(qk.load().kv_dev_append, append(**over))


@pytest.mark.parametrize("over", SHARED + [
    dict(scale=0.0), dict(scale=-1.0), dict(scale=NAN), dict(scale=INF), dict(scale=1e-39), dict(scale=2e38), dict(mask_words=-1), dict(mask_words=65537),
    dict(mask=P + 1), dict(out=None), dict(q=None), dict(out=P + 1), dict(q=P + 1), dict(q_row=-1), dict(out_head=-1),
    dict(cache_page=1 << 39, pages=1 << 20), dict(out=P),
    dict(out_row=64), dict(out_head=8), dict(work=None), dict(work=P + 16), dict(work_bytes=1000)])
def test_attention_refuses(over):
    refused(qk.load().attn_dev_paged, paged(**over))


@pytest.mark.parametrize("over", [dict(n_seq=-1), dict(n_seq=(1 << 20) + 1), dict(rows=-1), dict(words=-1), dict(words=0),
                                  dict(rows=1 << 20, words=1 << 10), dict(starts=None, rows=7), dict(mask=None),
                                  dict(parents=None), dict(cached=None), dict(mask=P + 1), dict(positions=P + 2),
                                  dict(parents=P + 2), dict(cached=P + 1), dict(starts=P + 3)])
def test_trees_refuse(over):
    refused(qk.load().attn_dev_tree, tree(**over))


def test_nothing_to_do():
    lib = qk.load()
    for f, make in ((lib.kv_dev_append, append), (lib.attn_dev_paged, paged), (lib.attn_dev_tree, tree)):
        assert f(None, None) == qk.BFP8_EINVAL
        assert f(make(rows=0), None) == qk.BFP8_OK and f(make(n_seq=0), None) == qk.BFP8_OK
        assert f(make(rows=0, starts=None), None) == qk.BFP8_OK


def test_attention_work():
    lib = qk.load()
    f = lib.attn_dev_paged_work_bytes
    assert f(None) == 0 and f(paged(dim=60)) == 0 and f(paged(heads_q=3)) == 0
    need = f(paged())
    assert need > 0 and lib.attn_dev_paged(paged(work_bytes=need - 1), None) == qk.BFP8_EINVAL
    assert f(paged(pages=0, page=0, table_pages=-1, scale=0.0, work=None)) == need  # the sizes alone
    g = qk.paged_attention_work_bytes
    assert g(6, 3, 4, 2, 64, torch.bfloat16) == need
    for rows, n in ((1, 1), (1 << 20, 1), (4096, 4096), (1 << 20, 1 << 20), (0, 0), (0, 5)):
        for dtype in (torch.float32, torch.bfloat16):
            assert 0 < g(rows, n, 16, 4, 256, dtype) < 1 << 28
    for bad in (lambda: g(-1, 1, 4, 2, 64, torch.float32), lambda: g((1 << 32) + 1, 1, 4, 2, 64, torch.float32),
                lambda: g(1, 1, 4, 2, 64, torch.float16)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        g(1, 1, 4, 3, 64, torch.float32)


def test_structs_have_the_headers_layout():
    assert ctypes.sizeof(qk.rope_dev_args) == 4 * 8 + 4 * 8 + 6 * 4 + 4 + 4 == qk._ROPE_PACK.size
    assert ctypes.sizeof(qk.kv_dev_append_args) == 11 * 8 + 12 * 8 + 11 * 4 + 4 == qk._APPEND_PACK.size
    assert ctypes.sizeof(qk.attn_dev_args) == 10 * 8 + 8 * 8 + 10 * 4 + 2 * 4 == qk._ATTN_PACK.size
    assert ctypes.sizeof(qk.attn_dev_tree_args) == 5 * 8 + 3 * 4 + 4 == qk._TREE_PACK.size


@pytest.mark.parametrize("struct,pack", [("rope_dev_args", "_ROPE_PACK"), ("kv_dev_append_args", "_APPEND_PACK"),
                                         ("attn_dev_args", "_ATTN_PACK"), ("attn_dev_tree_args", "_TREE_PACK")])
def test_packings_are_in_the_fields_order(struct, pack):
    """Each field of its own value, through the packing and back."""
    struct, pack = getattr(qk, struct), getattr(qk, pack)
    values = [float(i + 1) if t is ctypes.c_float else i + 1 for i, (_, t) in enumerate(struct._fields_)]
    a = struct.from_buffer_copy(pack.pack(*values))
    assert [getattr(a, name) for name, _ in struct._fields_] == values


def test_inputs_that_require_a_gradient():
    """Refused before the tensors are looked at (on the CPU here), unless gradients are off."""
    x, p, f = torch.zeros(2, 1, 8), torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.float64)
    c, t = torch.zeros(1, 4, 1, 8), torch.zeros(1, 1, dtype=torch.int32)
    h = torch.zeros(1, dtype=torch.int32)
    calls = [lambda y: qk.rotary(y, p, f), lambda y: qk.kv_cache_append(y, x, c, c, t, h),
             lambda y: qk.kv_cache_append(x, y, c, c, t, h), lambda y: qk.kv_cache_append(x, x, c, c, t, h, freqs=f, q=y),
             lambda y: qk.paged_attention(y, c, c, t, h)]
    caches = [lambda y: qk.paged_attention(x, y, c, t, h), lambda y: qk.paged_attention(x, c, y, t, h),
              lambda y: qk.kv_cache_append(x, x, y, c, t, h), lambda y: qk.kv_cache_append(x, x, c, y, t, h)]
    for call, y in [(f_, x) for f_ in calls] + [(f_, c) for f_ in caches]:
        y = y.clone().requires_grad_()
        with pytest.raises(ValueError, match="requires a gradient"):
            call(y)
        with torch.no_grad(), pytest.raises(ValueError, match="on a GPU"):
            call(y)
    with pytest.raises(ValueError, match="on a GPU"):  # (a gradient is an ordinary input)
        qk.rotary_grad(x.clone().requires_grad_(), p, f)
