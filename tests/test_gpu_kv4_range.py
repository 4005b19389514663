"""Attention over the 4-bit cache at the ends of its contract's range: queries, scales and keys far from 1 whose scores are
ordinary numbers. Tolerances as in test_gpu_kv4.py."""

import pytest
import torch

import kv4_ref as R
from test_gpu_kv4 import DEV, K, close, rand, tables  # noqa: F401

pytestmark = pytest.mark.gpu

# one row each and a few rows (blocks of 16 rows), a piece of a prompt (blocks of 128)
SIZES = [(6, 2, 64, [1, 1]), (28, 4, 128, [5, 2]), (12, 1, 64, [50, 60]), (14, 1, 128, [70, 20])]


def moved(pages, keys):
    """The pool with keys times 2^keys."""
    _, _, sk, _ = (x.to(DEV) for x in R.places(pages.shape[3] // 17))
    pages[:, :, :, sk] = (pages[:, :, :, sk].int() + keys).to(torch.uint8)


def case(K, nh, n_kv, hd, sizes, seed):
    pages, table = tables(K, 2, n_kv, hd, 32, 200, seed)
    lengths = torch.tensor([130, 90], device=DEV)
    starts = torch.tensor([0, sizes[0], sum(sizes)], device=DEV)
    return pages, table, lengths, starts, rand(seed + 1, sum(sizes), nh, hd)


@pytest.mark.parametrize("nh,n_kv,hd,sizes", SIZES)
@pytest.mark.parametrize("query,scale,key", [(-121, None, 122), (-112, None, 112), (-30, 2.0 ** -93, 122), (60, 2.0 ** 36, -97), (60, 2.0 ** 38, -99)])
def test_small_and_large_queries(K, nh, n_kv, hd, sizes, query, scale, key):  # noqa: F811
    pages, table, lengths, starts, q = case(K, nh, n_kv, hd, sizes, 3)
    moved(pages, key)
    q = q * 2.0 ** query
    q[0, 1] = 0
    q[-1, -1] *= 2.0 ** -9      # (beside rows that are far larger; below fp32's normal numbers where the others are just above)
    close(K.kv4_attn(q, pages, table, lengths, starts=starts, scale=scale), pages, table, lengths, q, starts=starts, scale=scale)


@pytest.mark.parametrize("nh,n_kv,hd,sizes", SIZES)
@pytest.mark.parametrize("query,scale", [(2.0 ** 30, 2.0 ** 100), (2.0 ** 126, 4.0), (1.5 * 2.0 ** 127, 2.0 ** -9), (2.0 ** -20, 2.0 ** 126)])
def test_products_beyond_the_range(K, nh, n_kv, hd, sizes, query, scale):  # noqa: F811
    """A query times the scale beyond fp32: zero keys leave scores of 0, one key of 2^-98 takes all of its sequence's rows."""
    pages, table, lengths, starts, _ = case(K, nh, n_kv, hd, sizes, 5)
    pk, _, sk, _ = (x.to(DEV) for x in R.places(hd))
    pages[:, :, :, pk] = 0
    q = torch.full((sum(sizes), nh, hd), query, device=DEV)
    close(K.kv4_attn(q, pages, table, lengths, starts=starts, scale=scale), pages, table, lengths, q, starts=starts, scale=scale)
    slot = 77
    for b in range(2):
        tile = pages[int(table[b, slot // 32]), :, slot % 32 // 16]
        tile[:, pk[slot % 16]] = 0x22                                # 1 times 2^-98
        tile[:, sk[slot % 16]] = 127 - 98
    got = K.kv4_attn(q, pages, table, lengths, starts=starts, scale=scale)
    seq = torch.repeat_interleave(torch.arange(2, device=DEV), starts.diff())
    v = torch.stack([R.rows_of(pages, table[b])[1][:, slot] for b in range(2)]).float()
    assert torch.equal(got, v.repeat_interleave(nh // n_kv, 1)[seq])     # scores of 2^13 and more beside zeros: its probability is 1, the others' 0


@pytest.mark.parametrize("nh,n_kv,hd,sizes", SIZES)
def test_half_queries_and_large_keys(K, nh, n_kv, hd, sizes):  # noqa: F811
    """Products of fp16 queries and keys beyond fp32 before a small scale."""
    pages, table, lengths, starts, q = case(K, nh, n_kv, hd, sizes, 7)
    moved(pages, 122)
    q = (q * 2000).half()
    for scale in (2.0 ** -134, -2.0 ** -133):
        close(K.kv4_attn(q, pages, table, lengths, starts=starts, scale=scale), pages, table, lengths, q, starts=starts, scale=scale)


@pytest.mark.parametrize("nh,n_kv,hd,sizes", SIZES)
def test_half_queries_and_scales(K, nh, n_kv, hd, sizes):  # noqa: F811
    """Scales of every kind for fp16 queries, the smallest among them."""
    pages, table, lengths, starts, q = case(K, nh, n_kv, hd, sizes, 9)
    q = q.half()
    q[0, 1], q[-1, 0] = 0, q[-1, 0] * 2.0 ** -22
    q[1 % len(q), 2] = q[1 % len(q), 2] * 400
    for scale in (-0.2, 0.0, 1.0, 0.999, 2.0 ** -140):
        close(K.kv4_attn(q, pages, table, lengths, starts=starts, scale=scale), pages, table, lengths, q, starts=starts, scale=scale)
    moved(pages, -97)
    close(K.kv4_attn(q, pages, table, lengths, starts=starts, scale=2.0 ** 94), pages, table, lengths, q, starts=starts, scale=2.0 ** 94)
    q[0, 3, 9], q[0, 4, 2] = float("inf"), float("nan")
    got = K.kv4_attn(q, pages, table, lengths, starts=starts, scale=2.0 ** 94)
    assert bool(got[0, 3:5].isnan().all()) and bool(got[0, 5].isfinite().all()) and bool(got[1:].isfinite().all())
