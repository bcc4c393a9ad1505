"""What the operators over a text's tokens refuse, on the host: invalid sizes, pointers
and work buffers give BFP8_EINVAL and a message before anything touches a GPU."""
import ctypes

import pytest
import torch

import qwen_kernels_gpu as qk

P = 1 << 20  # a pointer that is never followed


def gdn(**over):
    a = qk.gdn_dev_args()
    a.out = a.q = a.k = a.v = a.alpha = a.beta = a.state_in = a.state_out = a.work = P
    a.q_row = a.k_row = a.v_row = a.out_row = 256
    a.gate_row = 4
    a.rows = a.n_seq = a.n_slots = 3
    a.heads_k, a.heads_v, a.dim_k, a.dim_v, a.dtype, a.scale = 2, 4, 64, 64, qk.QWEN_F32, 1.0
    a.starts = P
    a.work_bytes = 1 << 40
    for k, v in over.items():
        setattr(a, k, v)
    return a


def loss(**over):
    a = qk.lm_head_loss_args()
    a.loss = a.lse = a.grad_h = a.grad_table = a.h = a.table = a.targets = a.grad_loss = a.work = P
    a.work_bytes = 1 << 40
    a.h_row = a.table_row = a.grad_h_row = a.grad_table_row = 64
    a.rows, a.vocab, a.hidden, a.dtype = 5, 100, 64, qk.QWEN_F32
    for k, v in over.items():
        setattr(a, k, v)
    return a


SIZES = [dict(dtype=2), dict(dtype=-1), dict(heads_k=0), dict(heads_v=3), dict(heads_v=1), dict(dim_k=0), dict(dim_k=66),
         dict(dim_k=260), dict(dim_v=2), dict(dim_v=512), dict(rows=-1), dict(n_seq=-1), dict(n_slots=-1),
         dict(heads_k=1, heads_v=65540), dict(n_seq=1 << 30, rows=1 << 30),
         dict(n_seq=(1 << 18) + 1, rows=(1 << 18) + 1), dict(heads_k=16, heads_v=16, n_seq=4, rows=1 << 25)]
POINTERS = [dict(state_out=None), dict(state_out=P + 4), dict(state_in=P + 8), dict(out=None), dict(q=None), dict(k=None),
            dict(v=None), dict(alpha=None), dict(q=P + 2), dict(out=P + 1, dtype=1), dict(alpha=P + 2), dict(beta=P + 1),
            dict(slots=P + 2), dict(q_row=64), dict(v_row=100), dict(out_row=0), dict(gate_row=2), dict(k_row=-256)]


@pytest.mark.parametrize("over", SIZES + POINTERS)
def test_linear_attention_refuses(over):
    lib = qk.load()
    for f in (lib.gdn_dev_prompt, lib.gdn_dev_step):
        assert f(gdn(**over), None) == qk.BFP8_EINVAL
        assert len(lib.bfp8_last_error()) > 20


@pytest.mark.parametrize("over", SIZES)
def test_linear_attention_work_of_invalid_sizes(over):
    assert qk.load().gdn_dev_prompt_work_bytes(gdn(**over)) == 0


def test_linear_attention_refuses_its_forms_own():
    lib = qk.load()
    a = gdn()
    need = lib.gdn_dev_prompt_work_bytes(a)
    assert need > 0
    for over in (dict(work=None), dict(work=P + 8), dict(work_bytes=need - 1), dict(starts=None), dict(starts=P + 2)):
        assert lib.gdn_dev_prompt(gdn(**over), None) == qk.BFP8_EINVAL
    assert lib.gdn_dev_step(gdn(rows=4), None) == qk.BFP8_EINVAL
    assert lib.gdn_dev_prompt(None, None) == qk.BFP8_EINVAL and lib.gdn_dev_step(None, None) == qk.BFP8_EINVAL
    assert lib.gdn_dev_prompt_work_bytes(None) == 0
    assert lib.gdn_dev_prompt(gdn(n_seq=0, rows=0), None) == qk.BFP8_OK  # nothing to do


@pytest.mark.parametrize("over", [
    dict(dtype=3), dict(rows=-1), dict(rows=(1 << 20) + 1), dict(vocab=0), dict(vocab=(1 << 28) + 1), dict(hidden=0),
    dict(hidden=65537), dict(rows=1 << 20, vocab=1 << 28), dict(rows=2048, vocab=1 << 27), dict(table=None),
    dict(table=P + 1), dict(table_row=63), dict(table_row=(1 << 22) + 1), dict(h=None), dict(targets=None), dict(h=P + 2), dict(targets=P + 2), dict(loss=P + 1),
    dict(lse=P + 2), dict(h_row=10), dict(work=None), dict(work=P + 16), dict(work_bytes=100)])
def test_loss_refuses(over):
    lib = qk.load()
    for f in (lib.bf16_dev_lm_head_loss, lib.bf16_dev_lm_head_loss_grad):
        assert f(loss(**over), None) == qk.BFP8_EINVAL
        assert len(lib.bfp8_last_error()) > 20


@pytest.mark.parametrize("over", [dict(lse=None), dict(grad_loss=None), dict(grad_h=P + 2), dict(grad_table=P + 1),
                                  dict(grad_h_row=3), dict(grad_table_row=3), dict(grad_loss=P + 2)])
def test_gradient_refuses(over):
    assert qk.load().bf16_dev_lm_head_loss_grad(loss(**over), None) == qk.BFP8_EINVAL


def test_loss_work():
    lib = qk.load()
    assert lib.bf16_dev_lm_head_loss_work_bytes(None) == 0 and lib.bf16_dev_lm_head_loss(None, None) == qk.BFP8_EINVAL
    assert lib.bf16_dev_lm_head_loss_grad(None, None) == qk.BFP8_EINVAL
    for f, g in ((lib.bf16_dev_lm_head_loss_work_bytes, lib.bf16_dev_lm_head_loss),
                 (lib.bf16_dev_lm_head_loss_grad_work_bytes, lib.bf16_dev_lm_head_loss_grad)):
        need = f(loss())
        assert need > 0 and g(loss(work_bytes=need - 1), None) == qk.BFP8_EINVAL
    # a gradient's work does not grow with the vocabulary once a piece is full
    big = [lib.bf16_dev_lm_head_loss_grad_work_bytes(loss(rows=4096, vocab=v, grad_h=None)) for v in (1 << 17, 1 << 24)]
    assert big[0] == big[1] < 256 << 20
    assert lib.bf16_dev_lm_head_loss(loss(rows=0), None) == qk.BFP8_OK
    assert lib.bf16_dev_lm_head_loss_grad(loss(grad_h=None, grad_table=None), None) == qk.BFP8_OK


def test_work_has_to_be_contiguous():
    """A view's elements times their size are not its bytes: one byte expanded would pass for any size."""
    x = torch.zeros(64, dtype=torch.uint8)
    assert qk._work_of(None) == (0, 0) and qk._work_of(x) == (x.data_ptr(), 64)
    assert qk._work_of(torch.zeros(8)[2:])[1] == 24
    for bad in (torch.zeros(1, dtype=torch.uint8).expand(1 << 30), x[::2], torch.zeros(4, 4).t()):
        with pytest.raises(ValueError, match="contiguous"):
            qk._work_of(bad)
    q = torch.zeros(1, 1, 4)
    gate, state = torch.zeros(1, 1), torch.zeros(1, 1, 16)
    with pytest.raises(ValueError, match="contiguous"):
        qk._gdn_args(q, q, q, gate, gate, 1.0, None, state, None, None, 1, x[::2], torch.zeros(1, 1, 4), False)
    with pytest.raises(ValueError, match="contiguous"):
        qk._loss_call("bf16_dev_lm_head_loss", loss(), x[::2], q)


def test_work_bytes_of_sizes_past_32_bits():
    """A size whose lower half is valid is refused, not taken for that half; so is another type."""
    f, g = qk.lm_head_loss_work_bytes, qk.linear_attention_prompt_work_bytes
    assert f(5, 100, 64, torch.float32) > 0 and g(5, 1, 1, 1, 64, 64, torch.bfloat16) > 0
    for far in ((1 << 32) + 5, 1 << 31, -(1 << 32) + 5, -1):
        for bad in (lambda: f(far, 100, 64, torch.float32), lambda: f(5, far, 64, torch.float32),
                    lambda: f(5, 100, far, torch.float32), lambda: g(far, 1, 1, 1, 64, 64, torch.float32),
                    lambda: g(5, far, 1, 1, 64, 64, torch.float32)):
            with pytest.raises(ValueError):
                bad()
    for bad in (lambda: f(5, 100, 64, torch.float16), lambda: g(5, 1, 1, 1, 64, 64, torch.float16)):
        with pytest.raises(ValueError):
            bad()


def test_inputs_that_require_a_gradient():
    """Results without a graph would end the gradient without a word: refused, before the tensors are looked at (on
    the CPU here), unless gradients are off."""
    z = lambda *s: torch.zeros(*s)  # noqa: E731
    q, gate, state = z(2, 1, 4), z(2, 1), z(2, 1, 16)
    h, table, t = z(2, 4), z(5, 4), torch.zeros(2, dtype=torch.int32)
    for i in range(6):
        a = [q, q, q, gate, gate, state]
        a[i] = a[i].clone().requires_grad_()
        for f in (lambda: qk.linear_attention_step(*a), lambda: qk.linear_attention_prompt(*a[:5], state_in=a[5])):
            with pytest.raises(ValueError, match="requires a gradient"):
                f()
            with torch.no_grad(), pytest.raises(ValueError, match="on a GPU"):
                f()
    for a in ((h.clone().requires_grad_(), table), (h, table.clone().requires_grad_())):
        with pytest.raises(ValueError, match="requires a gradient.*lm_head_loss_grad"):
            qk.lm_head_loss(*a, t)
        with torch.no_grad(), pytest.raises(ValueError, match="on a GPU"):
            qk.lm_head_loss(*a, t)
        with pytest.raises(ValueError, match="on a GPU"):  # (gradients of inputs that autograd knows are ordinary)
            qk.lm_head_loss_grad(*a, t, z(2), z(2))


def test_work_of_many_short_sequences():
    """Sequences that go token by token have no place in the work buffer, whose size never falls with the rows or the
    sequences (a buffer for the largest call does for the smaller ones)."""
    f = qk.linear_attention_prompt_work_bytes
    assert f(1024, 1024, 16, 16, 128, 128, torch.bfloat16) < 96 << 20
    assert f(8192, 8192, 16, 16, 128, 128, torch.float32) < 3 << 29
    sizes = sorted({0, 1, 15, 16, 17, 63, 64, 65, 255, 256, 257, 1000, 4095, 4096, 4097, 30000})
    for heads, dim_v in ((1, 4), (3, 96), (16, 128)):
        table = [[f(r, n, heads, heads, 64, dim_v, torch.bfloat16) for n in sizes[1:]] for r in sizes]
        for row in table:
            assert row == sorted(row)
        for column in zip(*table):
            assert list(column) == sorted(column)


def test_structs_have_the_headers_layout():
    assert ctypes.sizeof(qk.gdn_dev_args) == 12 * 8 + 5 * 8 + 9 * 4 + 4
    assert ctypes.sizeof(qk.lm_head_loss_args) == 10 * 8 + 4 * 8 + 4 * 4
