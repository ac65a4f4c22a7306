"""Rotary frequencies, refusals of the C entry points before any launch, and
the shapes that the ops give to tensors without storage.  No GPU."""
import ctypes
import math

import pytest
import torch

from pyramidkv import _abi as A, _ops, rope

FAKE = 0x1000  # an address that is never read: every call here is refused first


def _attn(**kw):
    a = A.BlockAttnArgs(q=FAKE, k=FAKE, v=FAKE, o=FAKE, lists=FAKE, cu_seqlens_q=FAKE, cu_seqlens_k=FAKE, total_q=8,
                        total_k=64, q_tok_stride=128, q_head_stride=128, kv_tok_stride=128, kv_head_stride=0,
                        o_tok_stride=128, o_head_stride=128, num_batches=1, num_heads_q=1, num_heads_kv=1, head_dim=128,
                        kv_per_head=1, max_seqlen_q=8, block_q=8, block_k=64, topk=1, causal=0, softmax_scale=0.1,
                        dtype=0)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def _select(**kw):
    a = A.BlockSelectArgs(q=FAKE, means=FAKE, lists=FAKE, cu_seqlens_q=FAKE, cu_seqlens_k=FAKE, total_q=8, total_k=64,
                          q_tok_stride=128, q_head_stride=128, num_batches=1, num_heads_q=1, num_heads_kv=1,
                          head_dim=128, kv_per_head=1, max_seqlen_q=8, max_seqlen_k=64, block_q=8, block_k=64, topk=4,
                          dtype=0)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def _means(**kw):
    a = A.BlockMeansArgs(k=FAKE, means=FAKE, cu_seqlens_k=FAKE, total_k=64, kv_tok_stride=128, num_seqs=1, num_heads=1,
                         head_dim=128, block_k=64, dtype=0)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def _rotary(**kw):
    a = A.RotaryArgs(q=FAKE, q_out=FAKE, pos=FAKE, freqs=FAKE, rows=4, q_tok_stride=128, q_head_stride=128,
                     num_heads_q=1, head_dim=128, num_axes=1, axis_pairs=(64, 0, 0, 0), dtype=0, scale=1.0)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


TILE_FAULTS = [dict(head_dim=96), dict(block_k=32), dict(block_k=96), dict(block_k=2048), dict(block_k=0),
               dict(block_q=0), dict(block_q=257), dict(block_q=-1), dict(topk=0), dict(topk=1025), dict(dtype=2),
               dict(num_heads_q=3, num_heads_kv=2), dict(num_heads_kv=0), dict(num_batches=-1), dict(total_q=-1),
               dict(total_k=-1), dict(max_seqlen_q=-1), dict(causal=1), dict(q=None), dict(lists=None),
               dict(cu_seqlens_q=None), dict(cu_seqlens_k=None), dict(q_tok_stride=129), dict(q_head_stride=4),
               dict(total_q=1 << 31), dict(num_heads_q=64, num_heads_kv=1, block_q=5)]


def _refused(rc):
    assert rc in (A.PKV_ERR_INVALID, A.PKV_ERR_UNSUPPORTED, A.PKV_ERR_CAPACITY), rc
    assert A.lib().pkv_last_error()


@pytest.mark.parametrize("fault", TILE_FAULTS + [
    dict(k=None), dict(v=None), dict(o=None), dict(kv_tok_stride=129), dict(kv_head_stride=4), dict(o_tok_stride=2),
    dict(kv_tok_stride=-128), dict(kv_tok_stride=0), dict(kv_tok_stride=120), dict(kv_tok_stride=1 << 24), dict(softmax_scale=0.0), dict(softmax_scale=-1.0),
    dict(softmax_scale=float("nan")), dict(softmax_scale=float("inf")), dict(max_seqlen_q=1 << 30, block_q=1), dict(max_seqlen_q=1 << 23, block_q=1),
], ids=str)
def test_attention_refusals(fault):
    a = _attn(**fault)
    _refused(A.lib().pkv_block_attn(ctypes.byref(a), FAKE, 1 << 40, None))


@pytest.mark.parametrize("fault", TILE_FAULTS + [
    dict(means=None), dict(sink_blocks=-1), dict(recent_blocks=-1), dict(sink_blocks=3, recent_blocks=2),
    dict(sink_blocks=0x7fffffff, recent_blocks=0x7fffffff), dict(max_seqlen_k=-1), dict(max_seqlen_k=32769 * 64),
    dict(num_batches=65536), dict(num_heads_q=65536, num_heads_kv=65536),
], ids=str)
def test_selection_refusals(fault):
    a = _select(**fault)
    _refused(A.lib().pkv_block_select(ctypes.byref(a), FAKE, 1 << 40, None))


def test_selection_needs_its_workspace():
    a = _select(max_seqlen_k=64 * 20000)  # (few blocks need none: scores and choice in one launch)
    need = A.lib().pkv_block_select_workspace_size(ctypes.byref(a))
    assert need >= 20000 * 4 and A.lib().pkv_block_select_workspace_size(ctypes.byref(_select())) == 0
    _refused(A.lib().pkv_block_select(ctypes.byref(a), FAKE, need - 1, None))
    _refused(A.lib().pkv_block_select(ctypes.byref(a), None, need, None))
    assert A.lib().pkv_block_select_workspace_size(ctypes.byref(_select(head_dim=96))) == 0


@pytest.mark.parametrize("fault", [dict(total_q=(1 << 31) - 4095), dict(total_k=(1 << 31) - 4095), dict(total_k=1 << 31),
                                   dict(max_seqlen_q=(1 << 31) - 4095)], ids=str)
def test_sizes_that_rounding_up_would_wrap(fault):
    """Lengths are rounded up to whole tiles and blocks in 32 bits."""
    _refused(A.lib().pkv_block_attn(ctypes.byref(_attn(**dict(dict(block_q=128, num_heads_q=1), **fault))), FAKE, 1 << 40, None))
    _refused(A.lib().pkv_block_select(ctypes.byref(_select(**fault)), FAKE, 1 << 40, None))
    if "total_k" in fault:
        _refused(A.lib().pkv_block_means(ctypes.byref(_means(**fault)), None))


def test_attention_needs_its_workspace():
    a = _attn(block_q=1, max_seqlen_q=1, topk=64)  # one token over 4,096 keys: split over workgroups
    need = A.lib().pkv_block_attn_workspace_size(ctypes.byref(a))
    assert need > 0
    _refused(A.lib().pkv_block_attn(ctypes.byref(a), FAKE, need - 1, None))
    assert A.lib().pkv_block_attn_workspace_size(ctypes.byref(_attn(block_q=64))) == 0


@pytest.mark.parametrize("fault", [dict(head_dim=32), dict(block_k=100), dict(dtype=2), dict(num_heads=0),
                                   dict(num_seqs=-1), dict(total_k=-1), dict(last=-1), dict(max_seqlen_k=-1),
                                   dict(k=None), dict(means=None), dict(cu_seqlens_k=None), dict(kv_tok_stride=4),
                                   dict(kv_head_stride=1), dict(num_seqs=1 << 24)], ids=str)
def test_means_refusals(fault):
    a = _means(**fault)
    _refused(A.lib().pkv_block_means(ctypes.byref(a), None))


@pytest.mark.parametrize("fault", [dict(head_dim=127), dict(head_dim=0), dict(rows=-1), dict(q=None), dict(q_out=None),
                                   dict(num_heads_k=1), dict(pos=None), dict(freqs=None), dict(num_axes=0),
                                   dict(num_axes=5), dict(axis_pairs=(0, 0, 0, 0)), dict(axis_pairs=(65, 0, 0, 0)),
                                   dict(axis_pairs=(-1, 0, 0, 0)), dict(axis_pairs=(257, 0, 0, 0), head_dim=1024),
                                   dict(num_axes=2, axis_pairs=(60, 5, 0, 0)), dict(dtype=3)], ids=str)
def test_rotary_refusals(fault):
    if "axis_pairs" in fault:
        fault = dict(fault, axis_pairs=(ctypes.c_int32 * 4)(*fault["axis_pairs"]))
    _refused(A.lib().pkv_rotary(ctypes.byref(_rotary(**fault)), None))


def test_null_arguments():
    for f in (A.lib().pkv_rotary, A.lib().pkv_block_means):
        _refused(f(None, None))
    _refused(A.lib().pkv_block_select(None, None, 0, None))
    _refused(A.lib().pkv_block_attn(None, None, 0, None))


def test_nothing_to_do():
    lib = A.lib()
    assert lib.pkv_rotary(ctypes.byref(_rotary(rows=0)), None) == A.PKV_OK
    assert lib.pkv_block_means(ctypes.byref(_means(num_seqs=0)), None) == A.PKV_OK
    assert lib.pkv_block_select(ctypes.byref(_select(num_batches=0)), None, 0, None) == A.PKV_OK
    assert lib.pkv_block_attn(ctypes.byref(_attn(num_batches=0)), None, 0, None) == A.PKV_OK


# ---- frequencies -------------------------------------------------------------
def test_frequencies():
    f, s = rope.rotary_frequencies(8, 10000.0)
    assert s == 1.0 and f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15)
    # the definition that the cache's own tables have
    assert torch.allclose(torch.polar(torch.ones(22, dtype=torch.float64), 5 * rope.rotary_frequencies(44)[0]),
                          rope.rope_params(6, 44)[5], rtol=1e-14)
    lin, _ = rope.rotary_frequencies(8, scaling="linear", factor=4.0)
    assert torch.equal(lin, f / 4)
    base, _ = rope.rotary_frequencies(8, scaling="base", factor=4.0)
    assert base[0] == 1.0 and math.isclose(base[-1], f[-1] / 4, rel_tol=1e-13)
    parts, s = rope.rotary_frequencies(128, scaling="parts", factor=16.0, trained_length=4096)
    f, _ = rope.rotary_frequencies(128)
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(parts[turns >= 32], f[turns >= 32]) and torch.equal(parts[turns <= 1], f[turns <= 1] / 16)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and ((parts[mid] < f[mid]) & (parts[mid] > f[mid] / 16)).all()
    assert math.isclose(s, 0.1 * math.log(16) + 1)


@pytest.mark.parametrize("call", [lambda: rope.rotary_frequencies(7), lambda: rope.rotary_frequencies(0),
                                  lambda: rope.rotary_frequencies(8, scaling="other"),
                                  lambda: rope.rotary_frequencies(8, scaling="linear", factor=0.5),
                                  lambda: rope.rotary_frequencies(8, scaling="parts", factor=2.0),
                                  lambda: rope.rotary_frequencies(8, scaling="parts", factor=2.0, trained_length=10,
                                                                  fast_turns=1, slow_turns=1)])
def test_frequency_refusals(call):
    with pytest.raises(ValueError):
        call()


# ---- shapes ---------------------------------------------------------------------
def test_meta_shapes():
    m = dict(device="meta")
    ops = _ops.ops()
    q, k = torch.empty(10, 8, 128, dtype=torch.bfloat16, **m), torch.empty(100, 2, 128, dtype=torch.bfloat16, **m)
    cu_q, cu_k = torch.empty(3, dtype=torch.int32, **m), torch.empty(3, dtype=torch.int32, **m)
    means = ops.block_means(k, cu_k, 64)
    assert means.shape == (100 // 64 + 2, 2, 128) and means.dtype == torch.float32
    lists = ops.block_select(q, means, cu_q, cu_k, 5, 50, 3, 4, 64)
    assert lists.shape == (10 // 4 + 2, 2, 3) and lists.dtype == torch.int32
    out = ops.block_sparse_attention(q, k, k, cu_q, cu_k, 5, lists, 0.1, 4, 64, False, True)
    assert out[0].shape == q.shape and out[0].dtype == q.dtype
    assert out[1].shape == (8, 10) and out[1].dtype == torch.float32
    assert len(ops.block_sparse_attention(q, k, k, cu_q, cu_k, 5, lists, 0.1, 4, 64)) == 1
    flat = torch.empty(100, 128, dtype=torch.float16, **m)
    cu_flat = torch.empty(5, dtype=torch.int32, **m)
    assert ops.block_means(flat, cu_flat, 128).shape == (100 // 128 + 4, 128)
    assert ops.block_select(q.half(), ops.block_means(flat, cu_flat, 64), cu_q, cu_flat, 5, 50, 3, 4, 64).shape == (4, 2, 3)
    pos, f = torch.empty(10, dtype=torch.int64, **m), torch.empty(16, dtype=torch.float64, **m)
    r = ops.rotary(q, q[:, :2], pos, f, [16], True, 1.0, False)
    assert [t.shape for t in r] == [q.shape, (10, 2, 128)]
    assert len(ops.rotary(q, None, pos, f, [16], True, 1.0, False)) == 1


@pytest.mark.parametrize("causal", [-1, 3])
def test_selection_refuses_other_causal_forms(causal):
    _refused(A.lib().pkv_block_select(ctypes.byref(_select(causal=causal, block_q=1)), FAKE, 1 << 40, None))


# ---- derivatives ------------------------------------------------------------------
def test_rotary_keeps_forward_derivatives():
    """On tensors without storage: a tangent comes out where one goes in."""
    from torch.autograd import forward_ad as fw
    m = dict(device="meta")
    q, k = torch.empty(10, 8, 64, **m), torch.empty(10, 2, 64, **m)
    pos, f = torch.empty(10, dtype=torch.int64, **m), torch.empty(32, dtype=torch.float64, **m)
    with fw.dual_level():
        dual = lambda x: fw.make_dual(x, torch.empty_like(x))
        assert fw.unpack_dual(rope.rotary(dual(q), pos, f)).tangent.shape == q.shape
        a, b = (fw.unpack_dual(x) for x in rope.rotary(dual(q), pos, f, k=dual(k)))
        assert a.tangent.shape == q.shape and b.tangent.shape == k.shape
        assert fw.unpack_dual(rope.rotary(q, pos, f, k=dual(k))[1]).tangent.shape == k.shape
    y, t = torch.func.jvp(lambda x: rope.rotary(x, pos, f), (q,), (torch.empty_like(q),))
    assert y.shape == t.shape == q.shape
    assert torch.func.grad(lambda x: rope.rotary(x, pos, f).sum())(q).shape == q.shape
    assert torch.func.vmap(lambda x: rope.rotary(x, pos, f))(torch.empty(3, 10, 8, 64, **m)).shape == (3, 10, 8, 64)
    with pytest.raises(RuntimeError):
        rope.rotary(q, pos, f.requires_grad_())


@pytest.mark.parametrize("block", [0, -64])
def test_meta_refusals(block):
    """Shapes of no block size raise (a division by zero would end the process)."""
    m = dict(device="meta")
    ops = _ops.ops()
    q, k = torch.empty(10, 8, 128, dtype=torch.bfloat16, **m), torch.empty(100, 2, 128, dtype=torch.bfloat16, **m)
    cu, means = torch.empty(3, dtype=torch.int32, **m), torch.empty(3, 2, 128, **m)
    none = torch.empty(0, dtype=torch.int32, **m)
    for call in (lambda: ops.block_means(k, cu, block), lambda: ops.block_means(k[0, 0], cu, 64),
                 lambda: ops.block_means(k, none, 64), lambda: ops.block_select(q, means, cu, cu, 5, 50, 3, block, 64),
                 lambda: ops.block_select(q, means, cu, cu, 5, 50, block, 4, 64),
                 lambda: ops.block_select(q[0], means, cu, cu, 5, 50, 3, 4, 64),
                 lambda: ops.block_select(q, means, none, none, 5, 50, 3, 4, 64)):
        with pytest.raises(RuntimeError):
            call()


def test_refusals_of_unaligned_pointers():
    """Read and written in 16-byte pieces (o in 8-byte ones)."""
    lib = A.lib()
    for name in ("k", "means"):
        _refused(lib.pkv_block_means(ctypes.byref(_means(**{name: FAKE + 8})), None))
    for name in ("q", "means"):
        _refused(lib.pkv_block_select(ctypes.byref(_select(**{name: FAKE + 8})), FAKE, 1 << 40, None))
    _refused(lib.pkv_block_select(ctypes.byref(_select(max_seqlen_k=64 * 20000)), FAKE + 8, 1 << 40, None))
    for name, off in (("q", 8), ("k", 8), ("v", 2), ("o", 4)):
        _refused(lib.pkv_block_attn(ctypes.byref(_attn(**{name: FAKE + off})), FAKE, 1 << 40, None))
    _refused(lib.pkv_block_attn(ctypes.byref(_attn(block_q=1, max_seqlen_q=1, topk=64)), FAKE + 8, 1 << 40, None))


def test_derivatives_that_are_not_there_raise():
    """Not a warning and no gradient."""
    from torch.autograd import forward_ad as fw
    m = dict(device="meta")
    ops = _ops.ops()
    q, k = torch.empty(10, 8, 128, dtype=torch.bfloat16, **m), torch.empty(100, 2, 128, dtype=torch.bfloat16, **m)
    cu, lists = torch.empty(3, dtype=torch.int32, **m), torch.empty(4, 2, 3, dtype=torch.int32, **m)
    pos, f = torch.empty(10, dtype=torch.int64, **m), torch.empty(32, dtype=torch.float64, **m)
    calls = dict(means=(lambda x, y: ops.block_means(y, cu, 64), k),
                 attend=(lambda x, y: ops.block_sparse_attention(x, y, y, cu, cu, 5, lists, 0.1, 4, 64)[0], q),
                 rotary=(lambda x, y: ops.rotary(x, None, pos, f, [32], True, 1.0, False)[0], q))
    for name, (call, x) in calls.items():
        pair = lambda z: (z, k) if x is q else (q, z)
        out = call(*pair(x.clone().requires_grad_()))
        with pytest.raises(RuntimeError, match="not implemented"):
            out.sum().backward()
        with fw.dual_level(), pytest.raises(NotImplementedError):
            call(*pair(fw.make_dual(x, torch.empty_like(x))))
    # what chooses blocks is no function to derive, and its result no floating number
    assert not ops.block_select(q.clone().requires_grad_(), torch.empty(3, 2, 128, **m), cu, cu, 5, 50, 3, 4, 64).requires_grad


def test_selection_in_one_launch_where_few_means_are_read_again():
    """One launch needs no workspace.  Rows that share their sequence's means: up
    to 48 MiB of them in all; single tokens, which share none: any number."""
    need = lambda **kw: A.lib().pkv_block_select_workspace_size(ctypes.byref(_select(**dict(
        dict(block_q=1, num_heads_q=8, num_heads_kv=2, total_q=1 << 20, total_k=1 << 22), **kw))))
    assert need(max_seqlen_q=700, max_seqlen_k=4000) == 0       # 1,400 rows of 63 blocks of 512 bytes: 43 MiB
    assert need(max_seqlen_q=2047, max_seqlen_k=4000) > 0       # 123 MiB
    assert need(max_seqlen_q=1200, max_seqlen_k=2047) == 0      # 37 MiB
    assert need(max_seqlen_q=2047, max_seqlen_k=2047) > 0       # 62 MiB
    assert need(max_seqlen_q=2047, max_seqlen_k=2047, causal=1) == 0  # half of that on average
    assert need(max_seqlen_q=4000, max_seqlen_k=4000, causal=1) > 0
    assert need(max_seqlen_q=4000, max_seqlen_k=1000, causal=1) == 0  # most rows see nothing
    assert need(max_seqlen_q=1, max_seqlen_k=8000, num_batches=4096) == 0
    assert need(max_seqlen_q=13, max_seqlen_k=8000) > 0         # 125 blocks of 128 columns: too long for a wave


def test_choices_and_means_in_place_carry_no_derivative():
    """A cache's means keep no history of the keys that they were brought up to
    date from, and blocks are chosen for queries with a tangent too."""
    from torch.autograd import forward_ad as fw
    m = dict(device="meta")
    ops = _ops.ops()
    q, k = torch.empty(10, 8, 128, dtype=torch.bfloat16, **m), torch.empty(100, 2, 128, dtype=torch.bfloat16, **m)
    cu, means = torch.empty(3, dtype=torch.int32, **m), torch.empty(3, 2, 128, **m)
    for _ in range(2):
        ops.block_means_(means, k.clone().requires_grad_(), cu, 64, 1)
        assert not means.requires_grad and means.grad_fn is None
    with fw.dual_level():
        lists = ops.block_select(fw.make_dual(q, torch.empty_like(q)), means, cu, cu, 5, 50, 3, 4, 64)
    assert lists.dtype == torch.int32 and not lists.requires_grad
