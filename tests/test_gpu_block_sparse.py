"""Block means, block selection and attention over listed blocks against plain
restatements in 64 bits."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from pyramidkv import _abi as A, block_sparse as bs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF = torch.bfloat16, torch.float16
INF = float("inf")


def cu(lens):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32), device=DEV)


def rnd(*shape, dtype=BF):
    return torch.randn(*shape, device=DEV).to(dtype)


def mean_rows(lens, block):
    """First row of every sequence, and the number of rows."""
    c = np.concatenate([[0], np.cumsum(lens)])
    return [int(c[s]) // block + s for s in range(len(lens))], int(c[-1]) // block + len(lens)


# ---------------------------------------------------------------------------
# means
# ---------------------------------------------------------------------------
def _check_means(got, k, lens, block, used=None):
    """n fp32 additions and a division: (n + 1) 2^-24 of the mean magnitude."""
    first, rows = mean_rows(lens, block)
    assert got.shape == (rows,) + k.shape[1:] and got.dtype == torch.float32
    want, bound = torch.zeros(got.shape, dtype=torch.float64), torch.zeros(got.shape, dtype=torch.float64)
    x, c = k.cpu().double(), 0
    for s, n in enumerate(lens):
        m = n if used is None else min(n, used[s])
        for j in range(-(-m // block)):
            y = x[c + j * block:c + min(m, (j + 1) * block)]
            want[first[s] + j] = y.mean(dim=0)
            bound[first[s] + j] = y.abs().mean(dim=0) * (y.shape[0] + 1) * 2.0 ** -24
        c += n
    assert ((got.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [BF, HF], ids=str)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,block,heads", [
    ([1], 64, None), ([0, 0], 64, 2), ([64, 0, 63, 1, 65], 64, None), ([130, 1, 700], 128, 3), ([1000, 333], 1024, 1),
    ([513] * 7, 192, None), ([3] * 70000, 64, None)])
def test_means(lens, block, heads, D, dtype):
    k = rnd(sum(lens), D, dtype=dtype) if heads is None else rnd(sum(lens), heads, D, dtype=dtype)
    for longest in (0, max(lens), 1):  # (1: a bound too small only makes the launch loop)
        _check_means(bs.block_means(k, cu(lens), block, max_seqlen_k=longest), k, lens, block)


def test_means_of_slices_and_rows_in_use():
    """Keys out of a fused projection, in a buffer longer than its sequences,
    of which each has some rows in use; what lies behind them may be anything."""
    lens, used = [200, 130, 64], [70, 0, 64]
    buf = rnd(500, 3, 4, 128)
    k = buf[:, 1, ::2]
    k[70:200], k[200:330], k[394:] = float("nan"), INF, float("nan")
    got = bs.block_means(k, cu(lens), 64, seqlens_k=torch.tensor(used, dtype=torch.int32, device=DEV))
    _check_means(got[:mean_rows(lens, 64)[1]], k[:394], lens, 64, used)
    assert got.shape[0] == 500 // 64 + 3 and not got[mean_rows(lens, 64)[1]:].any()


def test_means_brought_up_to_date():
    """A cache that grows in place by one key and by many at a time."""
    lens = [300, 257, 64]
    c, k = cu(lens), rnd(sum(lens), 2, 64)
    used = torch.tensor([1, 200, 0], dtype=torch.int32, device=DEV)
    means = bs.block_means(k, c, 64, seqlens_k=used)
    for more in (1, 1, 62, 1, 33):
        used = torch.minimum(used + more, torch.tensor(lens, dtype=torch.int32, device=DEV))
        assert bs.block_means(k, c, 64, seqlens_k=used, out=means, last=more, max_seqlen_k=300) is means
        assert torch.equal(means, bs.block_means(k, c, 64, seqlens_k=used))
    with pytest.raises(ValueError):
        bs.block_means(k, c, 64, last=1)
    with pytest.raises(RuntimeError):
        bs.block_means(k, c, 64, out=means, last=0)
    with pytest.raises(RuntimeError):
        bs.block_means(k, c, 64, out=means[1:], last=1)
    # rows outside the blocks asked for are left as they were
    marked = torch.full_like(means, 7.0)
    bs.block_means(k, c, 64, seqlens_k=used, out=marked, last=1)
    assert ((marked == 7.0).all(dim=-1).all(dim=-1).sum() == marked.shape[0] - int((used > 0).sum()))


def test_means_past_32_bit_offsets():
    """Rows 64 Ki elements apart: the last key begins past 2^32 elements."""
    rows = 66000
    k = torch.empty(rows, 1 << 16, dtype=BF, device=DEV)[:, :128]
    k[-130:] = rnd(130, 128)
    got = bs.block_means(k, torch.tensor([0, rows - 130, rows], dtype=torch.int32, device=DEV), 64)
    first = (rows - 130) // 64 + 1
    _check_means(got[first:first + 3], k[-130:].clone(), [130], 64)


# ---------------------------------------------------------------------------
# selection
# ---------------------------------------------------------------------------
def _layout(q_lens, k_lens, hkv, per_head):
    """Start and length of the key sequence of (batch, KV head)."""
    c = np.concatenate([[0], np.cumsum(k_lens)])
    return lambda b, h: ((s := b * hkv + h if per_head else b), int(c[s]), int(k_lens[s]))


def _select_ref(q, means, q_lens, k_lens, hkv, per_head, topk, bq, bk, sink, recent, causal, used=None):
    first_k, _ = mean_rows(k_lens, bk)
    first_q, rows = mean_rows(q_lens, bq)
    key_of = _layout(q_lens, k_lens, hkv, per_head)
    G = q.shape[1] // hkv
    out = np.full((q.shape[0] // bq + len(q_lens), hkv, topk), -1, dtype=np.int32)
    q, means, c = q.cpu().double(), means.cpu().double(), 0
    for b, lq in enumerate(q_lens):
        for i in range(-(-lq // bq)):
            for h in range(hkv):
                s, _, n = key_of(b, h)
                n = n if used is None else min(n, used[s])
                limit = max(0, n - lq + i + 1) if causal else n
                nb = -(-limit // bk)
                rows = q[c + i * bq:c + min(lq, (i + 1) * bq), h * G:(h + 1) * G].sum(dim=(0, 1))
                m = means[first_k[s]:first_k[s] + nb] if per_head else means[first_k[s]:first_k[s] + nb, h]
                sc = (m * rows).sum(dim=-1).float().numpy()
                sc = np.where(np.isnan(sc), -np.inf, sc)
                j = np.arange(nb)
                forced = (j < sink) | (j >= nb - recent)
                order = np.lexsort((j, -sc, ~forced))[:topk]
                out[first_q[b] + i, h, :len(order)] = np.sort(order)
        c += lq
    return out


def _run_select(q, means, q_lens, k_lens, hkv, per_head, topk, bq, bk, sink=0, recent=0, causal=False, used=None,
                max_q=None, max_k=None):
    u = None if used is None else torch.tensor(used, dtype=torch.int32, device=DEV)
    return bs.block_select(q, means, cu(q_lens), cu(k_lens), max(q_lens) if max_q is None else max_q,
                           max(k_lens) if max_k is None else max_k, topk, block_q=bq, block_k=bk, sink_blocks=sink,
                           recent_blocks=recent, causal=causal, seqlens_k=u)


SELECT = [  # q lens, k lens per batch, hkv, G, per_head, topk, bq, bk, sink, recent, causal
    ([1], [1], 1, 1, False, 1, 1, 64, 0, 0, False),
    ([1, 1, 1], [640, 0, 65], 2, 4, False, 3, 1, 64, 1, 1, False),
    ([300, 7, 0, 128], [5000, 64, 100, 0], 3, 1, True, 10, 120, 64, 2, 3, False),
    ([129], [9000], 2, 2, False, 17, 64, 128, 0, 1, False),
    ([77], [77], 2, 8, False, 4, 1, 64, 1, 1, True),
    ([33, 20], [500, 10], 1, 16, False, 5, 1, 64, 0, 2, True),    # more tokens than keys: the first see none
    ([64], [20000], 1, 1, True, 200, 16, 64, 5, 5, False),
    ([2], [180000], 1, 1, False, 1024, 1, 64, 1, 1, False),        # thousands of blocks
    ([16], [600000], 1, 2, True, 700, 16, 64, 0, 0, False),        # more than one wave of them holds
    ([260], [700], 1, 1, False, 11, 256, 64, 0, 0, False),         # all there are
]


@pytest.mark.parametrize("dtype,D", [(BF, 128), (HF, 64)])
@pytest.mark.parametrize("case", SELECT, ids=lambda c: f"q{c[0]}k{c[1]}")
def test_select(case, dtype, D):
    q_lens, k_lens, hkv, G, per_head, topk, bq, bk, sink, recent, causal = case
    if per_head:
        k_lens = [max(0, n - 37 * h) for n in k_lens for h in range(hkv)]
    q = rnd(sum(q_lens), hkv * G, D, dtype=dtype)
    rows = mean_rows(k_lens, bk)[1]
    means = torch.randn(rows, D, device=DEV) if per_head else torch.randn(rows, hkv, D, device=DEV)
    got = _run_select(q, means, q_lens, k_lens, hkv, per_head, topk, bq, bk, sink, recent, causal)
    want = _select_ref(q, means, q_lens, k_lens, hkv, per_head, topk, bq, bk, sink, recent, causal)
    assert np.array_equal(got.cpu().numpy(), want)


def test_select_ties_and_values_without_order():
    """Equal scores go to the lower block, NaN counts as -inf, -0 as 0."""
    D, bk, n = 128, 64, 64 * 40
    q = torch.ones(1, 1, D, device=DEV, dtype=BF)
    means = torch.zeros(n // bk + 1, D, device=DEV)
    means[5] = means[17] = means[30] = 1.0
    means[3], means[9], means[20] = float("nan"), INF, -INF
    means[7, 0], means[8, 0] = -0.0, 0.0
    means[11, 0], means[11, 1] = INF, -INF  # NaN
    for topk in (1, 2, 3, 4, 6, 37, 38, 39, 40, 64):
        got = _run_select(q, means, [1], [n], 1, True, topk, 1, bk)
        want = _select_ref(q, means, [1], [n], 1, True, topk, 1, bk, 0, 0, False)
        assert np.array_equal(got.cpu().numpy(), want), topk
    same = torch.ones_like(means)
    assert _run_select(q, same, [1], [n], 1, True, 6, 1, bk, 1, 2)[0, 0].tolist() == [0, 1, 2, 3, 38, 39]
    # forced blocks precede any score
    means[0] = means[39] = -INF
    assert {0, 39} <= set(_run_select(q, means, [1], [n], 1, True, 3, 1, bk, 1, 1)[0, 0].tolist())


def test_select_near_ties_by_the_exact_product():
    """Scores that fp32 sums would misorder: large terms that cancel."""
    D = 128
    q = torch.ones(1, 1, D, device=DEV, dtype=BF)
    means = torch.zeros(9, D, device=DEV)
    means[:, 0], means[:, 127] = 2.0 ** 30, -2.0 ** 30
    means[:8, 64] = torch.tensor([1.0, 5.0, 3.0, 8.0, 2.0, 7.0, 4.0, 6.0], device=DEV) * 2.0 ** -6
    assert _run_select(q, means, [1], [512], 1, True, 3, 1, 64)[0, 0].tolist() == [3, 5, 7]


def test_select_rows_in_use_bounds_and_padding_rows():
    q_lens, k_lens, used = [100, 0, 31], [1000, 640, 2000], [64, 640, 0]
    q, means = rnd(150, 4, 64), torch.randn(mean_rows(k_lens, 64)[1], 2, 64, device=DEV)
    got = _run_select(q, means, q_lens, k_lens, 2, False, 4, 32, 64, used=used)
    want = _select_ref(q, means, q_lens, k_lens, 2, False, 4, 32, 64, 0, 0, False, used)
    assert np.array_equal(got.cpu().numpy(), want)
    # bounds below the lengths: fewer blocks are considered, later tiles have none
    got = _run_select(q, means, q_lens, k_lens, 2, False, 4, 32, 64, max_q=40, max_k=500)
    want = _select_ref(q, means, q_lens, [min(n, 512) for n in k_lens], 2, False, 4, 32, 64, 0, 0, False)
    ref = np.full_like(got.cpu().numpy(), -1)
    # (the blocks' rows in the means go by the sequences' own lengths)
    full = _select_ref(q, means, q_lens, k_lens, 2, False, 4, 32, 64, 0, 0, False, [512, 512, 512])
    first, _ = mean_rows(q_lens, 32)
    for b, lq in enumerate(q_lens):
        n = min(-(-lq // 32), 2)
        ref[first[b]:first[b] + n] = full[first[b]:first[b] + n]
    assert want.shape == ref.shape and np.array_equal(got.cpu().numpy(), ref)
    assert (_run_select(q, means, q_lens, k_lens, 2, False, 4, 32, 64, max_q=0).cpu() == -1).all()
    assert (_run_select(q, means, q_lens, k_lens, 2, False, 4, 32, 64, max_k=0).cpu() == -1).all()


def test_select_in_several_launches():
    """More tiles than the workspace holds scores for at once."""
    n, k_len = 40000, 64 * 1024
    q, means = rnd(n, 1, 64), torch.randn(k_len // 64 + 1, 64, device=DEV)
    a = A.BlockSelectArgs(total_q=n, total_k=k_len, num_batches=1, num_heads_q=1, num_heads_kv=1, head_dim=64,
                          kv_per_head=1, max_seqlen_q=n, max_seqlen_k=k_len, block_q=1, block_k=64, topk=9)
    assert A.lib().pkv_block_select_workspace_size(ctypes.byref(a)) < n * 1024 * 4
    got = _run_select(q, means, [n], [k_len], 1, True, 9, 1, 64)
    sc = (q[:, 0].double() @ means[:1024].double().t()).float()
    want = sc.sort(dim=-1, descending=True, stable=True).indices[:, :9].sort(dim=-1).values
    assert torch.equal(got[:n, 0].long(), want) and (got[n:] == -1).all()


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def _attend_check(out, lse, q, k, v, lists, q_lens, k_lens, hkv, per_head, bq, bk, causal=False, used=None, scale=None):
    """out and lse against softmax in 64 bits.  Bound of a value, u = half a step of the type:
    its own rounding, u |o|; each probability's rounding to that type and its
    error in fp32, (u + d) sum p |v|, where d holds the score's sum of D products
    (each side of the softmax: 2 (D + 2) 2^-24 scale sum |q k|), the exponential
    and the running rescales (2^-20), and the sums over n keys (2 n 2^-24); in fp16
    also the smallest step of a probability, 2^-25 of the largest |v| a key."""
    D = q.shape[2]
    scale = D ** -0.5 if scale is None else scale
    G = q.shape[1] // hkv
    u = torch.finfo(q.dtype).eps / 2
    key_of = _layout(q_lens, k_lens, hkv, per_head)
    first_q, _ = mean_rows(q_lens, bq)
    q, k, v, lists, c = q.double(), k.double(), v.double(), lists.cpu().numpy(), 0
    for b, lq in enumerate(q_lens):
        for i in range(-(-lq // bq)):
            for h in range(hkv):
                s, at, n = key_of(b, h)
                n = n if used is None else min(n, used[s])
                limit = max(0, n - lq + i + 1) if causal else n
                blocks = sorted({int(x) for x in lists[first_q[b] + i, h] if 0 <= x < -(-limit // bk)})
                idx = [at + j for x in blocks for j in range(x * bk, min(limit, (x + 1) * bk))]
                r0, r1 = c + i * bq, c + min(lq, (i + 1) * bq)
                heads = slice(h * G, (h + 1) * G)
                got = out[r0:r1, heads].double()
                if not idx:
                    assert not got.any()
                    if lse is not None:
                        assert (lse[heads, r0:r1] == -INF).all()
                    continue
                kk, vv = (k[idx], v[idx]) if per_head else (k[idx, h], v[idx, h])
                qq = q[r0:r1, heads].reshape(-1, D)
                x = qq @ kk.t() * scale
                p = torch.softmax(x, dim=-1)
                o = (p @ vv).view(got.shape)
                d = 2 * (D + 2) * 2.0 ** -24 * scale * (qq.abs() @ kk.abs().t()).amax(dim=-1) + 2.0 ** -20 + \
                    2 * len(idx) * 2.0 ** -24
                spread = ((u + d)[:, None] * (p @ vv.abs())).view(got.shape)
                tiny = len(idx) * 2.0 ** -25 * vv.abs().amax() + 2.0 ** -25 if out.dtype == HF else 0.0
                over = (got - o).abs() - (u * (o.abs() + spread) + spread + tiny)
                assert (over <= 0).all(), (b, i, h, over.max().item())
                if lse is not None:
                    ref = torch.logsumexp(x, dim=-1).view(r1 - r0, G).t()
                    err = (lse[heads, r0:r1].double() - ref).abs()
                    assert (err <= (d.view(r1 - r0, G).t() + 2.0 ** -22 * (1 + ref.abs()))).all(), err.max().item()
        c += lq


def _lists(q_lens, k_lens, hkv, per_head, bq, bk, topk, rng, messy=False):
    key_of = _layout(q_lens, k_lens, hkv, per_head)
    first, rows = mean_rows(q_lens, bq)
    out = np.full((rows, hkv, topk), -1, dtype=np.int32)
    for b, lq in enumerate(q_lens):
        for i in range(-(-lq // bq)):
            for h in range(hkv):
                nb = -(-key_of(b, h)[2] // bk)
                if messy:  # any order, repeated, outside
                    out[first[b] + i, h] = rng.integers(-2, nb + 2, topk)
                else:
                    x = np.sort(rng.permutation(nb)[:topk])
                    out[first[b] + i, h, :len(x)] = x
    return torch.from_numpy(out).to(DEV)


ATTEND = [  # q lens, k lens, hkv, G, per_head, topk, bq, bk, causal
    ([1], [1], 1, 1, False, 1, 1, 64, False),
    ([1, 1, 1], [640, 0, 65], 2, 4, False, 3, 1, 64, False),
    ([1], [5000], 1, 1, True, 64, 1, 64, False),                    # one row, split over workgroups
    ([1, 1], [4000, 130], 2, 16, False, 20, 1, 128, False),
    ([1], [9000], 1, 7, False, 9, 1, 1024, False),
    ([77], [77], 2, 8, False, 4, 1, 64, True),
    ([33, 20], [500, 10], 1, 16, False, 5, 1, 64, True),
    ([50, 3], [700, 200], 2, 2, False, 4, 16, 64, False),           # 32 rows
    ([50, 3], [700, 200], 2, 2, False, 4, 17, 64, False),           # 34
    ([64, 0, 65], [900, 70, 64], 1, 1, True, 6, 64, 64, False),
    ([300, 7, 0, 128], [5000, 64, 100, 0], 3, 1, True, 10, 120, 64, False),
    ([128], [513], 2, 2, False, 5, 64, 192, False),
    ([257, 255], [1000, 3000], 1, 1, True, 7, 256, 64, False),
    ([100], [2000], 1, 3, False, 12, 85, 128, False),
    ([100], [2000], 1, 48, False, 3, 5, 64, False),
    # many small tiles: several of them to a workgroup
    ([700], [700], 2, 8, False, 6, 1, 64, True), ([310, 250], [900, 100], 2, 16, False, 5, 1, 64, True),
    ([2047], [1500], 1, 16, False, 3, 1, 128, True), ([1000], [640], 3, 1, True, 4, 4, 64, False),
    ([1030], [70000], 1, 8, False, 8, 2, 64, False), ([5, 900], [0, 300], 1, 7, False, 2, 3, 64, False),
    # few tiles of many rows: split over workgroups
    ([120], [5000], 2, 1, True, 40, 120, 64, False), ([1], [9000], 1, 48, False, 80, 1, 64, False),
    ([40, 3], [3000, 0], 1, 6, False, 24, 40, 64, False), ([70], [20000], 1, 2, False, 9, 32, 1024, False),
    ([1, 1], [2500, 130], 1, 128, False, 33, 1, 64, True), ([9], [70000], 1, 16, False, 1024, 9, 64, False),
    # many tiles of 33 to 64 rows: steps of 32 keys, split or not
    ([590], [900, ], 1, 40, False, 5, 1, 64, True), ([260], [3000], 1, 33, False, 17, 1, 128, False),
]


@pytest.mark.parametrize("dtype", [BF, HF], ids=str)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("case", ATTEND, ids=lambda c: f"q{c[0]}k{c[1]}b{c[6]}")
def test_attend(case, D, dtype):
    q_lens, k_lens, hkv, G, per_head, topk, bq, bk, causal = case
    if per_head:
        k_lens = [max(0, n - 37 * h) for n in k_lens for h in range(hkv)]
    rng = np.random.default_rng(D)
    q = rnd(sum(q_lens), hkv * G, D, dtype=dtype) * 2
    shape = (sum(k_lens), D) if per_head else (sum(k_lens), hkv, D)
    k, v = rnd(*shape, dtype=dtype), rnd(*shape, dtype=dtype)
    for messy in (False, True):
        lists = _lists(q_lens, k_lens, hkv, per_head, bq, bk, topk, rng, messy)
        out, lse = bs.block_sparse_attention(q, k, v, cu(q_lens), cu(k_lens), max(q_lens), lists, block_q=bq, block_k=bk,
                                             causal=causal, return_lse=True)
        _attend_check(out, lse, q, k, v, lists, q_lens, k_lens, hkv, per_head, bq, bk, causal)
        again = bs.block_sparse_attention(q, k, v, cu(q_lens), cu(k_lens), max(q_lens), lists, block_q=bq, block_k=bk,
                                          causal=causal)
        assert torch.equal(out, again)


def test_attend_in_the_largest_groups():
    """32 tiles of 2 rows to a workgroup, more than one window of blocks long."""
    q_len, k_len, hkv = 1400, 66000, 6
    q, k, v = rnd(q_len, 2 * hkv, 64), rnd(k_len, hkv, 64), rnd(k_len, hkv, 64)
    lists = _lists([q_len], [k_len], hkv, False, 1, 64, 3, np.random.default_rng(8))
    out, lse = bs.block_sparse_attention(q, k, v, cu([q_len]), cu([k_len]), q_len, lists, block_q=1, return_lse=True)
    assert torch.isfinite(out).all()
    some = torch.arange(0, q_len, 7, device=DEV)  # (every seventh token, as a sequence of its own lists)
    _attend_check(out[some], lse[:, some], q[some], k, v, lists[:q_len][some], [len(some)], [k_len], hkv, False, 1, 64)


@pytest.mark.parametrize("poison", [float("nan"), INF])
def test_attend_neighbours_blocks(poison):
    """Tiles that a workgroup takes together: a value that is no number reaches
    the rows whose tile lists its block, and leaves every other as it was."""
    n, G = 600, 8
    q, k, v = rnd(n, 2 * G, 128), rnd(n, 2, 128), rnd(n, 2, 128)
    lists = _lists([n], [n], 2, False, 1, 64, 5, np.random.default_rng(5))
    run = lambda vv: bs.block_sparse_attention(q, k, vv, cu([n]), cu([n]), n, lists, block_q=1, causal=True,
                                               return_lse=True)
    want, lse = run(v)
    bad = v.clone()
    bad[130, 0, 7] = bad[599, 1] = poison
    out, lse2 = run(bad)
    assert torch.equal(lse, lse2)
    hit = torch.zeros(n, 2 * G, 128, dtype=torch.bool, device=DEV)
    seen = lambda h, j: (lists[:n, h] == j // 64).any(dim=-1) & (torch.arange(n, device=DEV) >= j)
    hit[seen(0, 130), :G, 7] = True
    hit[seen(1, 599), G:] = True
    assert hit.any() and torch.equal(~torch.isfinite(out), hit)
    assert torch.equal(out[~hit], want[~hit])
    bad = k.clone()  # (a key that is no number takes its rows' sums with it)
    bad[130, 0] = poison
    out, lse2 = bs.block_sparse_attention(q, bad, v, cu([n]), cu([n]), n, lists, block_q=1, causal=True, return_lse=True)
    hit[:, :G] = seen(0, 130)[:, None, None]
    hit[:, G:] = False
    assert torch.equal(out[~hit], want[~hit]) and torch.equal(lse2[:, ~seen(0, 130)], lse[:, ~seen(0, 130)])
    assert torch.isnan(out[hit]).all()


@pytest.mark.parametrize("bq", [1, 64, 200])
def test_attend_scores_of_all_sizes(bq):
    """Rising and falling scores: references that move by much, probabilities that vanish."""
    n = 64 * 12
    q = rnd(bq, 1, 128)
    k, v = rnd(n, 128), rnd(n, 128)
    for step in (3.0, -3.0, 20.0, -20.0):
        kk = (k.float() + q[:1, 0].float() * step * torch.arange(n, device=DEV)[:, None] / n).to(BF)
        lists = _lists([bq], [n], 1, True, bq, 64, 12, np.random.default_rng(0))
        out, lse = bs.block_sparse_attention(q, kk, v, cu([bq]), cu([n]), bq, lists, block_q=bq, return_lse=True)
        _attend_check(out, lse, q, kk, v, lists, [bq], [n], 1, True, bq, 64)


@pytest.mark.parametrize("bq", [1, 40])
def test_attend_infinities(bq):
    """What no list names, and what lies behind a sequence's end, is not read
    into a result; a row whose keys all score -inf is NaN, and one -inf key
    weighs nothing, wherever it stands."""
    n = 300
    q = torch.ones(bq, 1, 128, device=DEV, dtype=BF)
    k, v = rnd(400, 128), rnd(400, 128)
    k[n:], v[n:] = float("nan"), INF
    k[64:128], v[64:128] = INF, float("nan")           # block 1 is not listed
    lists = torch.full((400 // bq + 1, 1, 4), -1, dtype=torch.int32, device=DEV)[:bq // bq + 1]
    lists[0, 0] = torch.tensor([0, 2, 4, -1])
    args = lambda kk: (q, kk, v, cu([bq]), torch.tensor([0, n], dtype=torch.int32, device=DEV), bq, lists)
    out, lse = bs.block_sparse_attention(*args(k), block_q=bq, return_lse=True)
    clean_k, clean_v = k[:n].clone(), v[:n].clone()
    clean_k[64:128], clean_v[64:128] = 0, 0
    _attend_check(out, lse, q, clean_k, clean_v, lists, [bq], [n], 1, True, bq, 64)
    for lo, hi in ((0, 64), (0, 40), (128, 192), (256, 300), (270, 300)):
        kk = k.clone()
        kk[lo:hi] = 0
        kk[lo:hi, 0] = -INF
        out, lse = bs.block_sparse_attention(*args(kk), block_q=bq, return_lse=True)
        x = (q[:, 0].double() @ kk[:n].double().t()) * 128 ** -0.5
        x[:, 64:128] = x[:, 192:256] = -INF
        p = torch.softmax(x, dim=-1)
        want = p[:, [*range(64), *range(128, 192), *range(256, n)]] @ v[[*range(64), *range(128, 192), *range(256, n)]].double()
        assert torch.isfinite(out).all()
        assert ((out[:, 0].double() - want).abs() <= 2.0 ** -7 * (p @ torch.nan_to_num(v[:n].double(), 0.0).abs())).all()
        assert ((lse[0].double() - torch.logsumexp(x, dim=-1)).abs() <= 1e-5).all()
    kk = torch.zeros_like(k)
    kk[:, 0] = -INF
    out, lse = bs.block_sparse_attention(*args(kk), block_q=bq, return_lse=True)
    assert torch.isnan(out).all() and (lse == -INF).all()


@pytest.mark.parametrize("dtype", [BF, HF], ids=str)
@pytest.mark.parametrize("tokens,bq,topk", [(1, 1, 5), (1, 1, 18), (300, 1, 5), (600, 1, 5), (40, 40, 5), (40, 40, 40)])
def test_attend_infinite_values(tokens, bq, topk, dtype):
    """An infinity among the listed values is one of its column, two of opposite
    signs NaN, and the other columns are as without it."""
    n = 64 * topk - 20
    q, k, v = rnd(tokens, 2, 64, dtype=dtype), rnd(n, 64, dtype=dtype), rnd(n, 64, dtype=dtype)
    v[:, :3] = 0
    lists = torch.arange(topk, dtype=torch.int32, device=DEV).expand(tokens // bq + 1, 1, topk).contiguous()
    vv = v.clone()
    vv[7, 0], vv[70, 1], vv[n - 1, 2], vv[n - 3, 2] = INF, -INF, INF, -INF
    out, lse = bs.block_sparse_attention(q, k, vv, cu([tokens]), cu([n]), tokens, lists, block_q=bq, return_lse=True)
    assert (out[..., 0] == INF).all() and (out[..., 1] == -INF).all() and torch.isnan(out[..., 2]).all()
    out[..., :3] = 0
    _attend_check(out, lse, q, k, v, lists, [tokens], [n], 1, True, bq, 64)


def test_attend_strides_rows_in_use_and_other_rows():
    """q, k and v as slices of wider buffers, keys in use, an output whose other rows stay."""
    q_lens, k_lens, used = [30, 5], [300, 260], [129, 260]
    qb, kvb = rnd(50, 3, 8, 128), rnd(600, 2, 5, 128)
    q, k, v = qb[:, 1, ::2], kvb[:, 0, 1:3], kvb[:, 1, 1:3]
    k[129:300], v[129:300], k[560:] = float("nan"), INF, float("nan")
    u = torch.tensor(used, dtype=torch.int32, device=DEV)
    for bq in (4, 30):
        rows = 50 // bq + 2
        lists = torch.full((rows, 2, 5), -1, dtype=torch.int32, device=DEV)
        real = _lists(q_lens, k_lens, 2, False, bq, 64, 5, np.random.default_rng(3))
        lists[:real.shape[0]] = real
        o = torch.full((50, 4, 128), 3.0, dtype=BF, device=DEV)
        lse = torch.full((4, 50), 3.0, device=DEV)
        cq, ck = cu(q_lens), cu(k_lens)
        a = A.BlockAttnArgs(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), o=o.data_ptr(), lse=lse.data_ptr(),
                            lists=lists.data_ptr(), cu_seqlens_q=cq.data_ptr(), cu_seqlens_k=ck.data_ptr(),
                            seqlens_k=u.data_ptr(), total_q=50, total_k=600, q_tok_stride=q.stride(0),
                            q_head_stride=q.stride(1), kv_tok_stride=k.stride(0), kv_head_stride=k.stride(1),
                            o_tok_stride=512, o_head_stride=128, num_batches=2, num_heads_q=4, num_heads_kv=2,
                            head_dim=128, max_seqlen_q=30, block_q=bq, block_k=64, topk=5, softmax_scale=128 ** -0.5)
        need = A.lib().pkv_block_attn_workspace_size(ctypes.byref(a))
        ws = torch.empty(max(need, 1), dtype=torch.uint8, device=DEV)
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        A.check(A.lib().pkv_block_attn(ctypes.byref(a), ctypes.c_void_p(ws.data_ptr()), need, stream), "block_attn")
        assert (o[35:] == 3.0).all() and (lse[:, 35:] == 3.0).all()
        got, l2 = bs.block_sparse_attention(q, k, v, cq, ck, 30, lists, block_q=bq, return_lse=True, seqlens_k=u)
        assert torch.equal(got[:35], o[:35]) and torch.equal(l2[:, :35], lse[:, :35])
        kc, vc = torch.nan_to_num(k[:560].float(), 0.0), torch.nan_to_num(v[:560].float(), 0.0, 0.0, 0.0)
        _attend_check(o[:35], lse[:, :35], q[:35], kc, vc, lists, q_lens, k_lens, 2, False, bq, 64, used=used)


@pytest.mark.parametrize("q_len,most,bq", [(30, 17, 4), (300, 257, 1), (90, 50, 30), (5, 5, 1), (5, 9, 8)])
def test_attend_leaves_tokens_past_the_longest(q_len, most, bq):
    """Tokens past max_seqlen_q stay as they were, where they share a tile or a
    workgroup with earlier ones too."""
    q, k, v = rnd(q_len, 4, 64), rnd(300, 2, 64), rnd(300, 2, 64)
    lists = _lists([q_len], [300], 2, False, bq, 64, 5, np.random.default_rng(5))
    o, lse = torch.full((q_len, 4, 64), 3.0, dtype=BF, device=DEV), torch.full((4, q_len), 3.0, device=DEV)
    cq, ck = cu([q_len]), cu([300])
    a = A.BlockAttnArgs(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), o=o.data_ptr(), lse=lse.data_ptr(),
                        lists=lists.data_ptr(), cu_seqlens_q=cq.data_ptr(), cu_seqlens_k=ck.data_ptr(), total_q=q_len,
                        total_k=300, q_tok_stride=256, q_head_stride=64, kv_tok_stride=128, kv_head_stride=64,
                        o_tok_stride=256, o_head_stride=64, num_batches=1, num_heads_q=4, num_heads_kv=2, head_dim=64,
                        max_seqlen_q=most, block_q=bq, block_k=64, topk=5, softmax_scale=0.125)
    need = A.lib().pkv_block_attn_workspace_size(ctypes.byref(a))
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device=DEV)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    A.check(A.lib().pkv_block_attn(ctypes.byref(a), ctypes.c_void_p(ws.data_ptr()), need, stream), "block_attn")
    assert (o[most:] == 3.0).all() and (lse[:, most:] == 3.0).all()
    n = min(most, q_len)
    _attend_check(o[:n], lse[:, :n], q[:n], k, v, lists, [n], [300], 2, False, bq, 64)


def test_attend_past_32_bit_offsets():
    rows = 66000
    buf = torch.empty(rows, 1 << 16, dtype=BF, device=DEV)
    k, v = buf[:, :128], buf[:, 128:256]
    k[-130:], v[-130:] = rnd(130, 128), rnd(130, 128)
    for bq in (1, 64):
        q = rnd(bq, 1, 128)
        lists = torch.tensor([[[0, 1, 2]], [[-1, -1, -1]]], dtype=torch.int32, device=DEV)[:bq // bq + 1]
        ck = torch.tensor([rows - 130, rows], dtype=torch.int32, device=DEV)
        out = bs.block_sparse_attention(q, k, v, cu([bq]), ck, bq, lists, block_q=bq)
        _attend_check(out, None, q, k[-130:].clone(), v[-130:].clone(), lists, [bq], [130], 1, True, bq, 64)


def test_attend_empty_inputs():
    q, k = rnd(0, 2, 64), rnd(10, 2, 64)
    z = torch.zeros(2, dtype=torch.int32, device=DEV)
    lists = torch.zeros(1, 2, 3, dtype=torch.int32, device=DEV)
    assert bs.block_sparse_attention(q, k, k, z, cu([10]), 0, lists, block_q=4).shape == q.shape
    none = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert bs.block_sparse_attention(q, k, k, none, none, 0, lists[:0], block_q=4).shape == q.shape
    # no keys at all
    q, k = rnd(5, 2, 64), rnd(0, 2, 64)
    lists = torch.zeros(5 // 4 + 1, 2, 3, dtype=torch.int32, device=DEV)
    out, lse = bs.block_sparse_attention(q, k, k, cu([5]), cu([0]), 5, lists, block_q=4, return_lse=True)
    assert not out.any() and (lse == -INF).all()
    assert not bs.block_means(k, cu([0]), 64).any()


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
def _pipeline(q, k, v, cq, ck, mq, mk, sparse, **kw):
    return bs.sparse_ragged_attention(q, k, v, cq, ck, mq, mk, sparse, **kw)


def test_pipeline_finds_what_stands_out():
    """Queries that match the keys of certain blocks attend to those blocks."""
    B, hkv, G, D, n = 2, 2, 4, 128, 64 * 30
    cq, ck = cu([1] * B), cu([n] * B)
    q = rnd(B, hkv, 1, D).expand(B, hkv, G, D).reshape(B, hkv * G, D).contiguous()
    k, v = rnd(B * n, hkv, D) * 0.05, rnd(B * n, hkv, D)
    want = torch.full((B, hkv, 5), -1, dtype=torch.int32)
    for b in range(B):
        for h in range(hkv):
            x = sorted({0, 29, *(3 + 7 * b + h, 11 + h, 20 - b)})
            want[b, h] = torch.tensor(x)
            for j in x[1:-1]:
                k[b * n + 64 * j:b * n + 64 * (j + 1), h] += q[b, h * G]
    sparse = bs.BlockSparse(topk=5, block_q=1, sink_blocks=1, recent_blocks=1)
    means = bs.block_means(k, ck, 64)
    lists = bs.block_select(q, means, cq, ck, 1, n, 5, block_q=1, sink_blocks=1, recent_blocks=1)
    assert torch.equal(lists[[0, 2]].cpu() if lists.shape[0] == 4 else lists[:B].cpu(), want)
    out = _pipeline(q, k, v, cq, ck, 1, n, sparse)
    _attend_check(out, None, q, k, v, lists, [1] * B, [n] * B, hkv, False, 1, 64)
    assert torch.equal(out, _pipeline(q, k, v, cq, ck, 1, n, sparse, means=means))


def _state():
    q_lens, k_lens = [130, 40], [2000, 700, 1500, 90]
    return dict(q=rnd(170, 2, 128), k=rnd(sum(k_lens), 128), v=rnd(sum(k_lens), 128), cq=cu(q_lens), ck=cu(k_lens), mq=130,
                mk=2000, sparse=bs.BlockSparse(topk=6, block_q=60, sink_blocks=1, recent_blocks=2))


def test_pipeline_replayed():
    """Captured once, replayed on new inputs between eager calls; two graphs of the same tensors."""
    s = _state()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _pipeline(**s)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_pipeline(**s))
        graphs.append(g)
    for i in range(4):
        for n in ("q", "k", "v"):
            s[n].copy_(torch.randn(s[n].shape, device=DEV))
        s["ck"].copy_(cu([2000, 700 - 60 * i, 1500, 90 + 60 * i]))
        graphs[i % 2].replay()
        want = _pipeline(**s)
        torch.cuda.synchronize()
        assert torch.equal(outs[i % 2], want)


def test_pipeline_on_two_streams():
    """Calls that overlap have workspaces of their own."""
    a, b = _state(), _state()
    want = [_pipeline(**a), _pipeline(**b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i, (st, s) in enumerate(zip(streams, (a, b))):
            with torch.cuda.stream(st):
                got[i].append(_pipeline(**s))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_cache_attends_to_its_blocks():
    """MegaCache.attend(sparse=...): with every block it is the dense attention;
    with some it is the attention over the lists that the packed keys give."""
    from pyramidkv import factory
    from pyramidkv._mega_cache import build_mega_caches
    from pyramidkv.rope import wan_freqs
    H, D, FS, W, F = 3, 128, 160, 16, 3
    cache = build_mega_caches(1, H, D, FS, 3, 24, 4, factory.shipped_compositions(1, H, labels=[[-1, 1, 2]]),
                              max_attend_chunks=F, device=DEV, freqs=wan_freqs(D), spatial_width=W,
                              spatial_height=FS // W, **factory.PYRAMID_FORCING_REMAP)[0]
    for blk in range(4):
        for mode in ("noisy", "clean"):
            cache.update(rnd(1, F * FS, H, D), rnd(1, F * FS, H, D), blk * F * FS, cache_update_mode=mode)
    start = 3 * F * FS
    q = rnd(1, F * FS, H, D)
    dense = cache.attend(q, start)
    all_blocks = cache.attend(q, start, sparse=bs.BlockSparse(topk=64, block_q=100))
    mgr = cache.ctx.mgr
    ck = cache.attend_kv(start, F).clone()
    lens = (ck[1:] - ck[:-1]).tolist()
    assert max(lens) <= 64 * 64
    k, v = mgr.k_flat_out().view(-1, D)[:sum(lens)].clone(), mgr.v_flat_out().view(-1, D)[:sum(lens)].clone()
    full = _lists([FS] * F, lens, H, True, 100, 64, 64, np.random.default_rng(0))
    _attend_check(all_blocks[0], None, q[0], k, v, full, [FS] * F, lens, H, True, 100, 64)
    _attend_check(dense[0], None, q[0], k, v, full, [FS] * F, lens, H, True, 100, 64)
    sparse = bs.BlockSparse(topk=6, block_q=100, sink_blocks=1, recent_blocks=2)
    got = cache.attend(q, start, sparse=sparse)
    means = bs.block_means(k, ck, 64)
    lists = _select_ref(q[0], means, [FS] * F, lens, H, True, 6, 100, 64, 1, 2, False)
    _attend_check(got[0], None, q[0], k, v, torch.from_numpy(lists), [FS] * F, lens, H, True, 100, 64)
    with pytest.raises(RuntimeError):
        cache.attend(q, start, sparse=sparse, causal=True)


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
def _args():
    return dict(q=rnd(10, 4, 64), k=rnd(200, 2, 64), v=rnd(200, 2, 64), cq=cu([10]), ck=cu([200]), mq=10, mk=200,
                lists=torch.zeros(10 // 4 + 1, 2, 3, dtype=torch.int32, device=DEV), block_q=4, block_k=64,
                causal=False, used=None, means=torch.zeros(200 // 64 + 1, 2, 64, device=DEV), topk=3, scale=0.1)


BREAKS = {
    "q on the host": lambda a: a.update(q=a["q"].cpu()),
    "q of fp32": lambda a: a.update(q=a["q"].float()),
    "q of two dimensions": lambda a: a.update(q=a["q"][:, 0]),
    "q's columns apart": lambda a: a.update(q=rnd(10, 4, 128)[..., ::2]),
    "q off 16 bytes": lambda a: a.update(q=rnd(10, 4, 72)[..., 1:65]),
    "head_dim 32": lambda a: a.update(q=rnd(10, 4, 32), k=rnd(200, 2, 32), v=rnd(200, 2, 32),
                                      means=torch.zeros(4, 2, 32, device=DEV)),
    "heads that do not divide": lambda a: a.update(q=rnd(10, 5, 64)),
    "cu_seqlens_q of int64": lambda a: a.update(cq=a["cq"].long()),
    "cu_seqlens_k on the host": lambda a: a.update(ck=a["ck"].cpu()),
    "cu_seqlens_k of other batches": lambda a: a.update(ck=cu([100, 100])),
    "seqlens_k too short": lambda a: a.update(used=torch.zeros(0, dtype=torch.int32, device=DEV)),
    "seqlens_k of int64": lambda a: a.update(used=torch.zeros(1, dtype=torch.int64, device=DEV)),
    "block_q 0": lambda a: a.update(block_q=0),
    "tiles of 258 rows": lambda a: a.update(block_q=129, lists=a["lists"][:1]),
    "causal tiles": lambda a: a.update(causal=True),
    "block_k 96": lambda a: a.update(block_k=96),
    "a negative bound": lambda a: a.update(mq=-1),
}
ATTEND_BREAKS = {
    "k of another type": lambda a: a.update(k=a["k"].half()),
    "one key for all tokens": lambda a: a.update(k=rnd(1, 2, 64).expand(200, 2, 64), v=rnd(1, 2, 64).expand(200, 2, 64)),
    "v of other strides": lambda a: a.update(v=rnd(200, 4, 64)[:, ::2]),
    "k off 16 bytes": lambda a: a.update(k=rnd(200, 2, 72)[..., 1:65], v=rnd(200, 2, 72)[..., 1:65]),
    "flat keys of other batches": lambda a: a.update(k=rnd(200, 64), v=rnd(200, 64), cq=cu([5, 5]),
                                                     ck=cu([50, 50, 100])),
    "lists of int64": lambda a: a.update(lists=a["lists"].long()),
    "lists of other tiles": lambda a: a.update(lists=a["lists"][1:]),
    "lists of other heads": lambda a: a.update(lists=a["lists"][:, :1].contiguous()),
    "lists of no entries": lambda a: a.update(lists=a["lists"][..., :0].contiguous()),
    "lists of 1,025": lambda a: a.update(lists=torch.zeros(3, 2, 1025, dtype=torch.int32, device=DEV)),
    "a scale of 0": lambda a: a.update(scale=0.0),
}
SELECT_BREAKS = {
    "means of bf16": lambda a: a.update(means=a["means"].to(BF)),
    "means of another head_dim": lambda a: a.update(means=torch.zeros(4, 2, 128, device=DEV)),
    "means of no rows": lambda a: a.update(means=a["means"][:0]),
    "topk 0": lambda a: a.update(topk=0),
    "topk 1,025": lambda a: a.update(topk=1025),
    "a negative key bound": lambda a: a.update(mk=-1),
}


@pytest.mark.parametrize("name", [*BREAKS, *ATTEND_BREAKS])
def test_attend_refuses(name):
    a = _args()
    {**BREAKS, **ATTEND_BREAKS}[name](a)
    with pytest.raises((RuntimeError, NotImplementedError)):
        bs.block_sparse_attention(a["q"], a["k"], a["v"], a["cq"], a["ck"], a["mq"], a["lists"], block_q=a["block_q"],
                                  block_k=a["block_k"], softmax_scale=a["scale"], causal=a["causal"], seqlens_k=a["used"])


@pytest.mark.parametrize("name", [*BREAKS, *SELECT_BREAKS])
def test_select_refuses(name):
    a = _args()
    {**BREAKS, **SELECT_BREAKS}[name](a)
    with pytest.raises((RuntimeError, NotImplementedError)):
        bs.block_select(a["q"], a["means"], a["cq"], a["ck"], a["mq"], a["mk"], a["topk"], block_q=a["block_q"],
                        block_k=a["block_k"], causal=a["causal"], seqlens_k=a["used"])


@pytest.mark.parametrize("break_", [dict(k=lambda: rnd(9, 2, 64).float()), dict(k=lambda: rnd(9, 2, 64).cpu()),
                                    dict(k=lambda: rnd(9, 2, 32)), dict(k=lambda: rnd(9)), dict(block=63), dict(block=0)],
                         ids=str)
def test_means_refuse(break_):
    with pytest.raises((RuntimeError, NotImplementedError)):
        bs.block_means(break_["k"]() if "k" in break_ else rnd(9, 2, 64), cu([9]), break_.get("block", 64))


def test_arguments_are_sound():
    """What the refusals above start from is taken."""
    a = _args()
    bs.block_sparse_attention(a["q"], a["k"], a["v"], a["cq"], a["ck"], a["mq"], a["lists"], block_q=4)
    bs.block_select(a["q"], a["means"], a["cq"], a["ck"], a["mq"], a["mk"], 3, block_q=4)


# ---------------------------------------------------------------------------
# causal choices
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("n,hkv,G,topk,sink,bk", [(640, 1, 2, 3, 0, 64), (1000, 2, 4, 4, 1, 128), (300, 2, 8, 1, 0, 64),
                                                  (9000, 1, 1, 5, 0, 64), (500, 1, 1, 2, 2, 64)])
def test_causal_choice_sees_no_later_keys(n, hkv, G, topk, sink, bk):
    """Keys after token i, and what they do to its own block's mean, leave the
    lists and results of the tokens up to i as they were, with no recent block
    asked for too; and a token decoded by itself chooses as it does in the prompt."""
    tokens = min(n, 700)  # (a prompt, or the last part of one over a longer context)
    q, k, v = rnd(tokens, hkv * G, 64), rnd(n, hkv, 64), rnd(n, hkv, 64)
    sparse = bs.BlockSparse(topk=topk, block_q=1, block_k=bk, sink_blocks=sink)

    def both(kk):
        means = bs.block_means(kk, cu([n]), bk)
        return (bs.block_select(q, means, cu([tokens]), cu([n]), tokens, n, topk, block_q=1, block_k=bk, sink_blocks=sink,
                                causal=True),
                bs.sparse_ragged_attention(q, kk, v, cu([tokens]), cu([n]), tokens, n, sparse, causal=True))

    lists, out = both(k)
    for last in (n - 1, n - 60, n - bk - 7, n - tokens + 130):  # the last key that stays
        i = last - (n - tokens)
        if not 0 <= i < tokens:
            continue
        for size in (30.0, -30.0):
            kk = k.clone()
            kk[last + 1:] = (rnd(n - last - 1, hkv, 64) + q[i].view(hkv, G, 64).sum(dim=1)) * size
            l2, o2 = both(kk)
            assert torch.equal(l2[:i + 1], lists[:i + 1]) and torch.equal(o2[:i + 1], out[:i + 1])
        used = torch.tensor([last + 1], dtype=torch.int32, device=DEV)
        one = bs.block_select(q[i:i + 1], bs.block_means(k, cu([n]), bk, seqlens_k=used), cu([1]), cu([n]), 1, n, topk,
                              block_q=1, block_k=bk, sink_blocks=sink, causal=True, seqlens_k=used)
        assert torch.equal(one[0], lists[i])
    # the list of a token: its own block, and the best of those before
    j = lists[tokens - 1].cpu()
    assert ((j == (n - 1) // bk).any(dim=-1) | (sink >= topk)).all()


def test_own_blocks_ranked():
    """rank_own: the formula as it stands, later keys and all."""
    for n, hkv, G, topk, sink in ((640, 1, 2, 3, 0), (300, 2, 8, 1, 0), (500, 1, 1, 1, 1)):
        q, means = rnd(n, hkv * G, 64), torch.randn(n // 64 + 1, hkv, 64, device=DEV)
        got = bs.block_select(q, means, cu([n]), cu([n]), n, n, topk, block_q=1, sink_blocks=sink, causal=True, rank_own=True)
        want = _select_ref(q, means, [n], [n], hkv, False, topk, 1, 64, sink, 0, True)
        assert np.array_equal(got.cpu().numpy(), want)
        # the own block taken: the formula with one recent block
        if topk > sink:
            got = bs.block_select(q, means, cu([n]), cu([n]), n, n, topk, block_q=1, sink_blocks=sink, causal=True)
            want = _select_ref(q, means, [n], [n], hkv, False, topk, 1, 64, sink, 1, True)
            assert np.array_equal(got.cpu().numpy(), want)


def _poison(*shape, dtype):
    """Memory that the next tensor of this size is likely to get holds no zeros."""
    torch.cuda.synchronize()
    x = torch.full(shape, 7, dtype=dtype, device=DEV)
    torch.cuda.synchronize()
    del x


def test_rows_before_the_first_sequence():
    """Sequences that begin behind a buffer's first rows: what lies there is no
    block's and no tile's."""
    k, cq, ck = rnd(700, 2, 64), torch.tensor([40, 70], dtype=torch.int32, device=DEV), \
        torch.tensor([330, 700], dtype=torch.int32, device=DEV)
    _poison(700 // 64 + 1, 2, 64, dtype=torch.float32)
    means = bs.block_means(k, ck, 64)
    assert not means[:330 // 64].any()
    _check_means(means[330 // 64:330 // 64 + 6], k[330:].clone(), [370], 64)
    q = rnd(80, 2, 64)
    for bq in (1, 8):
        _poison(80 // bq + 1, 2, 3, dtype=torch.int32)
        lists = bs.block_select(q, means, cq, ck, 30, 370, 3, block_q=bq)
        tiles = -(-30 // bq)
        first = 40 // bq
        assert (lists[:first] == -1).all() and (lists[first:first + tiles] >= 0).all()
        assert (lists[first + tiles:] == -1).all()
    # many blocks: scores through the workspace
    k, ck = rnd(20000, 64), torch.tensor([330, 20000], dtype=torch.int32, device=DEV)
    _poison(20000 // 64 + 1, 64, dtype=torch.float32)
    means = bs.block_means(k, ck, 64)
    assert not means[:330 // 64].any()
    _poison(80 // 8 + 1, 1, 3, dtype=torch.int32)
    lists = bs.block_select(q, means, cq, ck, 30, 19670, 3, block_q=8)
    assert (lists[:5] == -1).all() and (lists[5:9] >= 0).all() and (lists[9:] == -1).all()


def test_no_sequences():
    none = torch.zeros(1, dtype=torch.int32, device=DEV)
    q, k = rnd(40, 2, 64), rnd(300, 2, 64)
    _poison(300 // 64, 2, 64, dtype=torch.float32)
    means = bs.block_means(k, none, 64)
    assert means.shape == (4, 2, 64) and not means.any()
    _poison(40 // 8, 2, 3, dtype=torch.int32)
    lists = bs.block_select(q, means, none, none, 0, 0, 3, block_q=8)
    assert lists.shape == (5, 2, 3) and (lists == -1).all()


def test_cache_attends_to_its_blocks_whatever_the_start():
    """MegaCache.attend(sparse=...) bounds a head's keys by its policy, which
    holds for queries of earlier frames than the cache has seen too."""
    from pyramidkv import _mega_cache, factory
    from pyramidkv._mega_cache import build_mega_caches
    from pyramidkv.rope import wan_freqs
    H, D, FS, W, F = 3, 128, 160, 16, 3
    cache = build_mega_caches(1, H, D, FS, 3, 24, 4, factory.shipped_compositions(1, H, labels=[[-1, 1, 2]]),
                              max_attend_chunks=F, device=DEV, freqs=wan_freqs(D), spatial_width=W,
                              spatial_height=FS // W, **factory.PYRAMID_FORCING_REMAP)[0]
    mgr, seen = cache.ctx.mgr, []
    plain = _mega_cache.sparse_ragged_attention

    def spy(q, k, v, cu_q, cu_k, max_q, max_k, *args, **kw):
        seen.append((max_k, k.shape[0], int((cu_k[1:] - cu_k[:-1]).max()), int(cu_k[-1])))
        return plain(q, k, v, cu_q, cu_k, max_q, max_k, *args, **kw)

    _mega_cache.sparse_ragged_attention = spy
    try:
        for blk in range(12):
            for mode in ("noisy", "clean"):
                cache.update(rnd(1, F * FS, H, D), rnd(1, F * FS, H, D), blk * F * FS, cache_update_mode=mode)
            q = rnd(1, F * FS, H, D)
            for start in {0, blk * F * FS}:
                dense = cache.attend(q, start)
                ck = cache.attend_kv(start, F).clone()
                lens = (ck[1:] - ck[:-1]).tolist()
                k, v = (x.view(-1, D)[:sum(lens)].clone() for x in (mgr.k_flat_out(), mgr.v_flat_out()))
                got = cache.attend(q, start, sparse=bs.BlockSparse(topk=128, block_q=80))
                full = _lists([FS] * F, lens, H, True, 80, 64, 128, np.random.default_rng(0))
                _attend_check(got[0], None, q[0], k, v, full, [FS] * F, lens, H, True, 80, 64)
                _attend_check(dense[0], None, q[0], k, v, full, [FS] * F, lens, H, True, 80, 64)
    finally:
        _mega_cache.sparse_ragged_attention = plain
    capacity = int(mgr.max_pack_tokens()) // (F * H)
    kept = cache.ctx.layer_max_keys[0]
    assert 0 < kept < capacity
    for max_k, rows, longest, total in seen:
        assert longest <= max_k == kept and total <= rows == F * H * kept
    # a context without a policy's bound: the capacity
    cache.ctx.layer_max_keys, seen[:] = [], []
    _mega_cache.sparse_ragged_attention = spy
    try:
        cache.attend(q, 0, sparse=bs.BlockSparse(topk=8, block_q=80))
    finally:
        _mega_cache.sparse_ragged_attention = plain
    assert seen[0][0] == capacity


def test_means_off_16_bytes_are_refused():
    k, c = rnd(200, 64), cu([200])
    buf = torch.zeros(200 // 64 + 1 + 1, 64, device=DEV).view(-1)
    with pytest.raises(RuntimeError):
        bs.block_means(k, c, 64, out=buf[1:1 + 4 * 64].view(4, 64), last=1)
    bs.block_means(k, c, 64, out=buf[4:4 + 4 * 64].view(4, 64), last=1)


@pytest.mark.parametrize("n,blocks,hkv,causal", [(2100, 64, 2, False), (4096, 64, 2, True), (600, 100, 1, False), (1300, 20, 2, True)])
def test_select_of_many_rows(n, blocks, hkv, causal):
    """Prompts of few blocks, in one launch or in several."""
    q, means = rnd(n, 2 * hkv, 128), torch.randn(blocks + 1, hkv, 128, device=DEV)
    keys = blocks * 64 - 17
    got = _run_select(q, means, [n], [keys], hkv, False, 7, 1, 64, 1, 2, causal)
    tile = q.view(n, hkv, 2, 128).double().sum(dim=2).cpu()
    score = torch.matmul(tile.transpose(0, 1), means[:blocks].cpu().double().permute(1, 2, 0).contiguous()).float()
    limit = (keys - n + 1 + torch.arange(n)).clamp(min=0) if causal else torch.full((n,), keys)
    here = -(-limit // 64)                                              # blocks of a token
    j = torch.arange(blocks)
    score = torch.where((j < 1) | (j >= here[:, None] - 2), INF, score)
    score = torch.where(j < here[:, None], score, -INF)
    want = score.sort(dim=-1, descending=True, stable=True).indices[..., :7]
    want = torch.where(want < here[:, None], want, 1 << 20).sort(dim=-1).values
    want = torch.where(want < 1 << 20, want, -1).transpose(0, 1)
    assert torch.equal(got[:n].cpu().long(), want) and (got[n:] == -1).all()
