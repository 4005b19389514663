"""The paged 4-bit cache on the GPU: append and read against the rounding in 64 bits, equal to the last bit; attention
against softmax in 64 bits over the values that the pages stand for.

Tolerance of the attention, relative to sum p |v| / sum p: a score's three (two) bf16 parts leave 2^-27 (nothing) of the
query, its four steps of 32 products and parts each at most 2^-22 of the magnitudes so far, a rounded
scale and the subtraction of the maximum the rest of 2^-19 of the score's magnitude A; the exponential 2^-22; a
probability's parts 2^-25 (fp32), 2^-17 (fp16); both numerator and denominator. Sums over n keys: a lane's n / 4
additions, three parts of every 32 keys, 64 joins, each 2^-24. A probability, or a part of one, that is below 2^-126 of its
row's largest has no normal fp32 number and may be lost: 2^-126 |v| of a key, in numerator and denominator. Stored in fp16 half a step more, 2^-11 (2^-25 at least)."""

import math

import pytest
import torch

import kv4_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def K():
    from pico_hip import kernels
    return kernels


def rand(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)


def tables(K, B, n_kv, hd, page, slots, seed, spare=2, fill=True):
    per = -(-slots // page)
    pages = K.kv4_pages(B * per + spare, n_kv, hd, page, DEV)
    if fill:
        R.fill(pages, seed, key=0.7)
    perm = torch.randperm(B * per + spare, generator=torch.Generator().manual_seed(seed))[:B * per]
    return pages, perm.view(B, per).int().to(DEV)


def close(got, pages, table, lengths, q, starts=None, first=1, scale=None, rows=None):
    hd = q.shape[2]
    ref, mags, tops, sums = R.attention(q, pages, table, lengths, starts, first, hd ** -0.5 if scale is None else scale)
    n = table.shape[1] * pages.shape[2] * 16
    half = got.dtype is torch.float16
    tol = mags * (2 * (tops * 2.0 ** -19 + 2.0 ** -22 + (2.0 ** -17 if half else 2.0 ** -25)) + (n / 4 + 3 * n / 32 + 64) * 2.0 ** -24)
    tol = tol + sums * 2.0 ** -125
    if half:
        tol = tol + (ref.abs() * 2.0 ** -11).clamp_min(2.0 ** -25)
    err = (got.double() - ref).abs()
    keep = torch.ones(q.shape[0], dtype=torch.bool, device=DEV) if rows is None else rows
    ok = (err <= tol) | (got.isnan() & ref.isnan())
    bad = ~ok[keep]
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, at most {float(err[keep].nan_to_num(9e9).max())}"


# ---- append and read ------------------------------------------------------------------------

def appended(pages, table, lengths, starts, k, v, freqs, amp, il, w, eps):
    """A copy of the pages with the rows stored, on the CPU."""
    want = pages.clone().cpu()
    T = k.shape[0]
    edges = list(range(T + 1)) if starts is None else starts.tolist()
    tab, cap = table.cpu(), table.shape[1] * pages.shape[2] * 16
    for b, n in enumerate(lengths.tolist()):
        for t in range(edges[b], edges[b + 1]):
            slot = n + t - edges[b]
            kk = k[t:t + 1].double()
            if w is not None:
                kk = R.normed(kk, w, eps)
            if freqs is not None:
                kk = R.turned(kk, torch.tensor([slot], device=DEV), freqs, amp, il)[0]
            page_tokens = pages.shape[2] * 16
            if n < 0 or slot >= cap or not 0 <= int(tab[b, slot // page_tokens]) < pages.shape[0]:
                continue
            R.store(want, tab, b, slot, kk[0].cpu(), v[t].double().cpu())
    return want


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("il", [False, True])
@pytest.mark.parametrize("B,nh,n_kv,hd,page,rot,sizes", [(1, 14, 2, 64, 32, 64, [1]), (3, 28, 4, 128, 64, 128, [1, 1, 1]),
                                                         (5, 25, 5, 64, 16, 20, [7, 0, 33, 1, 18]), (2, 12, 1, 64, 48, 32, [1, 30]),
                                                         (4, 16, 16, 128, 112, 126, [3, 2, 0, 40]), (70, 2, 2, 64, 16, 64, [1] * 70)])
def test_append(K, B, nh, n_kv, hd, page, rot, sizes, dtype, il):
    T = sum(sizes)
    pages, table = tables(K, B, n_kv, hd, page, 150, 3, fill=False)
    pages.random_(generator=torch.Generator(device=DEV).manual_seed(1))      # bytes of any kind, that must stay
    lengths = torch.randint(0, 100, (B,), generator=torch.Generator(device=DEV).manual_seed(2), device=DEV)
    starts = None if sizes == [1] * B else torch.tensor([sum(sizes[:b]) for b in range(B + 1)], device=DEV)
    fused = (rand(4, T, (nh + 2 * n_kv) * hd) * 1.5).to(dtype).view(T, nh + 2 * n_kv, hd)
    q, k, v = fused[:, :nh], fused[:, nh:nh + n_kv], fused[:, nh + n_kv:]
    freqs, amp = K.rope_freqs(rot, 1e6)
    wq, wk = 1 + rand(5, hd) * 0.2, 1 + rand(6, hd) * 0.2
    seq = torch.repeat_interleave(torch.arange(B, device=DEV), torch.tensor(sizes, device=DEV))
    edges = torch.tensor([sum(sizes[:b]) for b in range(B)], device=DEV)
    pos = lengths[seq] + torch.arange(T, device=DEV) - edges[seq]
    for w1, w2, fr, a in ((wq, wk, freqs, 1.25), (None, None, freqs, 1.0), (wq, wk, None, 1.0), (None, None, None, 1.0)):
        mine = pages.clone()
        got = K.kv4_append(k, v, mine, table, lengths, starts=starts, q=q, freqs=fr, amp=a, interleaved=il, q_norm=w1, k_norm=w2, eps=1e-5)
        assert torch.equal(mine.cpu(), appended(pages, table, lengths, starts, k, v, fr, a, il, w2, 1e-5))
        ref = q.double() if w1 is None else R.normed(q, w1, 1e-5)
        ref, mags = R.turned(ref, pos, fr, a, il) if fr is not None else (ref, ref.abs())
        tol = mags * (2.0 ** -20 + 2.0 ** -21)           # as qk_norm_rope
        if dtype is torch.float16:
            tol = tol + (ref.abs() * 2.0 ** -11).clamp_min(2.0 ** -25)
        assert bool(((got.double() - ref).abs() <= tol).all())
        # without q, int32 lengths and starts, rows apart in memory: the same pages
        other = pages.clone()
        st32 = None if starts is None else starts.int()
        assert K.kv4_append(k.transpose(0, 1).contiguous().transpose(0, 1), v.contiguous(), other, table, lengths.int(), starts=st32,
                            freqs=fr, amp=a, interleaved=il, k_norm=w2, eps=1e-5) is None
        assert torch.equal(other, mine)


def test_append_unaligned(K):
    """Rows that 16 bytes do not divide, in and out."""
    pages, table = tables(K, 3, 2, 128, 32, 40, 1, fill=False)
    lengths = torch.tensor([3, 0, 31], device=DEV)
    freqs, _ = K.rope_freqs(50, 1e4)
    x = rand(1, 3, 5 * 131 + 7)
    q, k, v = (x[:, a:a + n * 131].view(3, n, 131)[:, :, 1:129] for a, n in ((1, 2), (263, 2), (394, 2)))
    wide = torch.full((3, 2, 135), 5.0, device=DEV)
    got = K.kv4_append(k, v, pages, table, lengths, q=q, freqs=freqs, out=wide[:, :, 3:131])
    other = K.kv4_pages(pages.shape[0], 2, 128, 32, DEV)
    want = K.kv4_append(k.contiguous(), v.contiguous(), other, table, lengths, q=q.contiguous(), freqs=freqs)
    assert torch.equal(pages, other) and torch.equal(got, want) and bool((wide[:, :, :3] == 5).all() and (wide[:, :, 131:] == 5).all())
    assert K.kv4_append(k, v, pages, table, lengths, q=q, freqs=freqs, out=q) is q and torch.equal(q, want)


def test_append_left_out(K):
    """Rows of no sequence, sequences that take no part, slots behind the table, pages that there are not."""
    B, n_kv, hd, page = 5, 2, 64, 16
    pages, table = tables(K, B, n_kv, hd, page, 32, 1, fill=False)
    pages.random_(generator=torch.Generator(device=DEV).manual_seed(1))
    table[2, 1], table[3, 0] = -1, pages.shape[0]
    lengths = torch.tensor([-1, 30, 15, 14, 1 << 45], device=DEV)
    starts = torch.tensor([2, 4, 8, 10, 14, 15], device=DEV)
    T = 17
    q, k, v = rand(1, T, 4, hd), rand(2, T, n_kv, hd), rand(3, T, n_kv, hd)
    freqs, _ = K.rope_freqs(hd)
    before, out = pages.clone(), torch.full((T, 4, hd), 7.0, device=DEV)
    K.kv4_append(k, v, pages, table, lengths, starts=starts, q=q, freqs=freqs, out=out)
    lengths[4] = 1 << 29      # as far behind the table, and what the oracle can count
    assert torch.equal(pages.cpu(), appended(before, table, lengths, starts, k, v, freqs, 1.0, False, None, 0))
    assert bool((out[:2] == 7).all()) and bool((out[15:] == 7).all()) and not bool((out[2:15] == 7).any())


def test_append_values(K):
    """Zero rows, the smallest and largest blocks, infinities and NaN: the block's bytes, and only that block's."""
    pages, table = tables(K, 1, 1, 64, 16, 16, 1, fill=False)
    table[0, 0] = 0
    v = rand(1, 8, 1, 64)
    v[0], v[1, 0, :32], v[2, 0, :32], v[3, 0, 5], v[4, 0, 40] = 0, v[1, 0, :32] * 2.0 ** -99, v[2, 0, :32] * 2.0 ** 125, float("inf"), float("nan")
    v[5, 0, 3], v[6, 0, :32], v[7, 0, 32:] = -3.4e38, v[6, 0, :32] * 2.0 ** -130, 7.0
    starts, lengths = torch.tensor([0, 8], device=DEV), torch.tensor([4], device=DEV)
    before = pages.clone()
    K.kv4_append(v, v, pages, table, lengths, starts=starts)
    assert torch.equal(pages.cpu(), appended(before, table, lengths, starts, v, v, None, 1.0, False, None, 0))
    k2, v2 = K.kv4_read(pages, table, lengths + 8, 14)
    assert torch.equal(k2.nan_to_num(9.0), v2.nan_to_num(9.0)) and k2.isnan().sum() == 64 and bool(k2[0, 0, 7, :32].isnan().all() and k2[0, 0, 8, 32:].isnan().all())
    assert bool((k2[0, 0, :5] == 0).all()) and bool((k2[0, 0, 12:] == 0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("B,n_kv,hd,page,rows", [(1, 2, 64, 32, 500), (3, 4, 128, 16, 33), (2, 1, 64, 48, 1), (4, 5, 128, 80, 200)])
def test_read(K, B, n_kv, hd, page, rows, dtype):
    pages, table = tables(K, B, n_kv, hd, page, rows - rows // 3, 5)
    table[B - 1, 0] = pages.shape[0] if B > 2 else table[B - 1, 0]
    cap = table.shape[1] * page
    lengths = torch.tensor([rows + 9, 0, 17, -4][:B], device=DEV)
    for ln in (lengths, lengths.int()):
        k, v = K.kv4_read(pages, table, ln, rows, dtype=dtype)
        assert k.shape == v.shape == (B, n_kv, rows, hd)
        for b in range(B):
            n = max(0, min(int(lengths[b]), rows, cap))
            for got, ref in zip((k[b], v[b]), R.rows_of(pages, table[b])):
                want = torch.zeros(n_kv, rows, hd, dtype=torch.float64, device=DEV)
                want[:, :n] = ref[:, :n].nan_to_num(0.0)       # no page: zeros
                assert torch.equal(got.double(), want.to(dtype).double())
    assert K.kv4_read(pages, table, lengths, 0)[0].shape == (B, n_kv, 0, hd)


def test_every_code_and_scale(K):
    """All 16 codes under all 256 scale bytes, read back."""
    pages = K.kv4_pages(1, 256, 64, 16, DEV)
    pages.random_(generator=torch.Generator(device=DEV).manual_seed(1))
    pages[0, :, 0, 1024:] = torch.arange(256, device=DEV, dtype=torch.uint8)[:, None]
    table, lengths = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.tensor([16], device=DEV)
    k, v = K.kv4_read(pages, table, lengths, 16)
    for got, ref in zip((k[0], v[0]), R.rows_of(pages, table[0])):
        # bytes below 2 and above 252 (scales that append never makes, but 255) reach beyond fp32's normal numbers
        assert torch.equal(got[2:253].double(), ref[2:253]) and bool(got[255].isnan().all())


# ---- attention ------------------------------------------------------------------------------

HEADS = [(14, 2, 64), (28, 4, 128), (16, 16, 64), (12, 1, 64), (25, 5, 64), (32, 8, 128), (40, 1, 128)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("nh,n_kv,hd", HEADS)
@pytest.mark.parametrize("page,lengths", [(32, [0]), (16, [0, 1, 14, 15, 16, 17]), (48, [62, 63, 64, 65, 127, 128]),
                                          (64, [255, 3, 256, 257]), (112, [1030])])
def test_attn_one_row_each(K, nh, n_kv, hd, page, lengths, dtype):
    B = len(lengths)
    pages, table = tables(K, B, n_kv, hd, page, max(lengths) + 1, 7)
    q = (rand(8, B, nh, hd) * 0.5).to(dtype)
    ln = torch.tensor(lengths, device=DEV)
    got = K.kv4_attn(q, pages, table, ln)
    close(got, pages, table, ln, q)
    assert torch.equal(K.kv4_attn(q, pages, table, ln.int()), got)
    none = K.kv4_attn(q, pages, table, ln, first=-max(lengths), scale=0.3)     # the longest sees none
    close(none, pages, table, ln, q, first=-max(lengths), scale=0.3)
    assert bool((none[lengths.index(max(lengths))] == 0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("nh,n_kv,hd,page,sizes,lengths", [
    (14, 2, 64, 32, [2, 1], [100, 40]), (28, 4, 128, 64, [4, 0, 5], [300, 10, 0]), (12, 1, 64, 16, [3, 2, 2], [0, 5, 333]),
    (14, 2, 64, 48, [19, 40, 1], [50, 0, 700]), (28, 4, 128, 16, [70], [11]), (16, 16, 64, 80, [130, 3], [5, 900]),
    (32, 8, 128, 128, [65, 64, 0, 63], [200, 1, 5, 64]), (25, 5, 64, 16, [1] * 90, list(range(90)))])
def test_attn_ragged(K, nh, n_kv, hd, page, sizes, lengths, dtype):
    B, T = len(sizes), sum(sizes) + 3
    pages, table = tables(K, B, n_kv, hd, page, max(a + b for a, b in zip(sizes, lengths)), 9)
    edges = [1 + sum(sizes[:b]) for b in range(B + 1)]          # a row before the first, two behind the last
    starts, ln = torch.tensor(edges, device=DEV), torch.tensor(lengths, device=DEV)
    q = (rand(8, T, nh, hd) * 0.5).to(dtype)
    out = torch.full((T, nh, hd), 7.0, device=DEV, dtype=dtype)
    got = K.kv4_attn(q, pages, table, ln, starts=starts, out=out)
    assert got is out and bool((out[0] == 7).all() and (out[-2:] == 7).all())
    rows = torch.ones(T, dtype=torch.bool, device=DEV)
    rows[0] = rows[-2:] = False
    close(got, pages, table, ln, q, starts=starts, rows=rows)
    again = K.kv4_attn(q, pages, table, ln, starts=starts.int())
    assert torch.equal(again[rows], got[rows])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("nh,n_kv,hd,lengths", [(14, 2, 64, [5000]), (12, 1, 128, [9000, 3, 700]), (28, 4, 128, [2500] * 3 + [1] * 70)])
def test_attn_cut(K, nh, n_kv, hd, lengths, dtype):
    """Long sequences beside short ones: keys cut over workgroups and joined."""
    B = len(lengths)
    pages, table = tables(K, B, n_kv, hd, 256, max(lengths) + 9, 7, spare=0)
    q = (rand(8, B, nh, hd) * 0.5).to(dtype)
    ln = torch.tensor(lengths, device=DEV)
    assert K.kv4_attn_workspace(B, B, nh, n_kv, hd, table.shape[1] * 256, DEV).numel() > 0
    got = K.kv4_attn(q, pages, table, ln)
    close(got, pages, table, ln, q)
    assert torch.equal(K.kv4_attn(q, pages, table, ln), got)
    sizes = [5] + [1] * (B - 1)
    starts = torch.tensor([sum(sizes[:b]) for b in range(B + 1)], device=DEV)
    q = (rand(8, sum(sizes), nh, hd) * 0.5).to(dtype)
    close(K.kv4_attn(q, pages, table, ln, starts=starts), pages, table, ln, q, starts=starts)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("sizes", [[1, 1, 1, 1], [6, 1, 40, 9]])
def test_attn_left_out(K, sizes, dtype):
    """Sequences that take no part, pages that there are not, a length behind the table; bytes of any kind where no row
    looks, not-a-numbers among them."""
    nh, n_kv, hd, page, B = 14, 2, 64, 16, 4
    pages, table = tables(K, B, n_kv, hd, page, 640, 7)
    junk = torch.randint(0, 256, pages.shape, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV, dtype=torch.uint8)
    junk[..., 1024:][junk[..., 1024:] > 128] = 255
    lengths = torch.tensor([70, -1, 300, 1 << 35], device=DEV)
    table[2, 3], table[2, 9] = -7, 1 << 30
    first, T = 1, sum(sizes)
    starts = None if T == B else torch.tensor([sum(sizes[:b]) for b in range(B + 1)], device=DEV)
    # behind a sequence's last seen slot: junk
    pk, pv, sk, sv = (x.to(DEV) for x in R.places(hd))
    for b in (0, 2):
        last = int(lengths[b]) + first + sizes[b] - 1
        for slot in range(last, 640):
            p, off = int(table[b, slot // page]), slot % page
            if not 0 <= p < pages.shape[0]:
                continue
            for f in (pk, pv, sk, sv):
                pages[p][:, 0, f[off]] = junk[p][:, 0, f[off]]
    for p in set(range(pages.shape[0])) - set(table.flatten().tolist()):
        pages[p] = junk[p]
    for p in table[1].tolist():
        pages[p] = 255
    q = (rand(8, T, nh, hd) * 0.5).to(dtype)
    got = K.kv4_attn(q, pages, table, lengths, starts=starts, first=first)
    lengths[3] = 640
    close(got, pages, table, lengths, q, starts=starts, first=first)
    lo = 1 if starts is None else int(starts[1])
    assert bool((got[lo:lo + sizes[1]] == 0).all()) and bool(got.isfinite().all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("hd,new", [(64, 1), (64, 12), (128, 40), (128, 3)])
def test_attn_no_numbers(K, hd, new, dtype):
    """A key or value block that is no number reaches the rows that see it (a value's only its 32 channels) and no other."""
    nh, n_kv, page = 4, 2, 16
    pages, table = tables(K, 1, n_kv, hd, page, 200, 7)
    lengths, starts = torch.tensor([130], device=DEV), torch.tensor([0, new], device=DEV)
    pk, pv, sk, sv = (x.to(DEV) for x in R.places(hd))
    for slot, f, h, block in ((130 + new // 2, sv, 0, 1), (130 + new - 1, sk, 1, 0), (5, sv, 1, 0)):
        pages[int(table[0, slot // page]), h, 0, f[slot % page, block]] = 255
    q = (rand(8, new, nh, hd) * 0.5).to(dtype)
    got = K.kv4_attn(q, pages, table, lengths, starts=starts)
    close(got, pages, table, lengths, q, starts=starts)
    ok = got.isnan()
    assert bool(ok[:, 2:, :32].all()) and bool(ok[new // 2:, :2, 32:64].all()) and bool(ok[-1, 2:].all())
    assert not bool(ok[:new // 2, :2].any()) and not bool(ok[:, :2, :32].any()) and not bool(ok[:-1, 2:, 32:].any())


def test_attn_values(K):
    """Large and small scales, huge queries, a negative scale, equal scores."""
    pages, table = tables(K, 2, 2, 64, 32, 100, 7)
    lengths = torch.tensor([99, 50], device=DEV)
    q = rand(8, 2, 6, 64)
    q[0, 0], q[0, 1], q[1, 2] = q[0, 0] * 200, 0, q[1, 2] * 2.0 ** -100
    for scale in (-0.2, 0.0, 1.0):
        close(K.kv4_attn(q, pages, table, lengths, scale=scale), pages, table, lengths, q, scale=scale)
    pk, pv, sk, sv = (x.to(DEV) for x in R.places(64))
    pages[:, 0][:, :, sk] = (pages[:, 0][:, :, sk].int() - 95).to(torch.uint8)         # keys of 2^-95, values of 2^100
    pages[:, 0][:, :, sv] = (pages[:, 0][:, :, sv].int() + 100).to(torch.uint8)
    q[:, :3] *= 2.0 ** 95
    q[1, 2] *= 2.0 ** 100
    close(K.kv4_attn(q, pages, table, lengths), pages, table, lengths, q)
    q[0, 4, 9] = float("inf")
    got = K.kv4_attn(q, pages, table, lengths)
    assert bool(got[0, 4].isnan().all()) and bool(got[0, 5].isfinite().all()) and bool(got[1].isfinite().all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_attn_strides(K, dtype):
    """Queries and outputs inside wider rows, heads first, unaligned; pages of one layer among several; shared pages."""
    nh, n_kv, hd, B = 6, 2, 64, 3
    big = torch.zeros(12, 3, n_kv, 2, 17 * hd, device=DEV, dtype=torch.uint8)
    pages = big[:, 1]
    R.fill(pages, 3)
    big[:, 0], big[:, 2] = 255, 255
    wide = torch.tensor([[3, 4, 5, 0], [3, 4, 1, 0], [7, 2, 11, 0]], dtype=torch.int32, device=DEV)
    table = wide[:, :3]
    lengths = torch.tensor([90, 80, 95], device=DEV)
    want = K.kv4_attn((rand(8, B, nh, hd) * 0.5).to(dtype), pages.contiguous(), table.contiguous(), lengths)
    src = (rand(8, B, nh, hd) * 0.5).to(dtype)
    views = [src.transpose(0, 1).contiguous().transpose(0, 1), torch.zeros(B, nh, hd + 3, device=DEV, dtype=dtype)[:, :, 3:],
             torch.zeros(B, 2 * nh, hd, device=DEV, dtype=dtype)[:, ::2], src.transpose(1, 2).contiguous().transpose(1, 2)]
    for q in views:
        q.copy_(src)
        out = torch.full((B, nh + 1, hd + 1), 7.0, device=DEV, dtype=dtype)
        got = K.kv4_attn(q, pages, table, lengths, out=out[:, :nh, 1:])
        assert torch.equal(got, want) and bool((out[:, nh] == 7).all() and (out[:, :, 0] == 7).all())
    assert torch.equal(K.kv4_attn(src[:1].expand(B, nh, hd), pages, table[:1].expand(B, 3), lengths[:1].expand(B).contiguous()),
                       want[:1].expand(B, nh, hd))


def test_pages_of_one_head(K):
    """Pools whose one kv head, or one tile, has a stride of any kind."""
    q, lengths = rand(1, 2, 4, 64), torch.tensor([40, 20], device=DEV)
    for heads, tiles in ((1, 2), (1, 1), (2, 1)):
        pages, table = tables(K, 2, heads, 64, 16 * tiles, 64, 3, spare=0)
        want = K.kv4_attn(q, pages, table, lengths)
        odd = torch.empty_strided(pages.shape, (heads * tiles * 1088, 7 if heads == 1 else 1088, 5 if tiles == 1 else 1088, 1),
                                  dtype=torch.uint8, device=DEV)
        odd.copy_(pages)
        assert torch.equal(K.kv4_attn(q, odd, table, lengths), want)
    pages, table = tables(K, 2, 2, 64, 32, 64, 3, spare=0)
    for bad in (pages.transpose(1, 2), pages.flatten(1)):
        with pytest.raises(ValueError):
            K.kv4_attn(q, bad, table, lengths)


def test_attn_far_pages(K):
    """A pool of more than 4 GB, the pages at its end."""
    page, n_kv, hd = 256, 8, 128
    each = n_kv * 16 * 17 * hd
    n = (1 << 32) // each + 5
    pages = torch.empty(n, n_kv, 16, 17 * hd, device=DEV, dtype=torch.uint8)
    R.fill(pages[-4:], 1)
    R.fill(pages[:1], 2)
    table = torch.tensor([[n - 1, n - 3], [0, n - 4]], dtype=torch.int32, device=DEV)
    lengths = torch.tensor([500, 300], device=DEV)
    q = rand(3, 2, 16, hd) * 0.5
    small = torch.cat([pages[:1], pages[-4:]])
    t2 = torch.tensor([[4, 2], [0, 1]], dtype=torch.int32, device=DEV)
    got = K.kv4_attn(q, pages, table, lengths)
    close(got, small, t2, lengths, q)
    k, v = rand(4, 2, n_kv, hd), rand(5, 2, n_kv, hd)
    K.kv4_append(k, v, pages, table, lengths)
    K.kv4_append(k, v, small, t2, lengths)
    assert torch.equal(pages[-4:], small[1:]) and torch.equal(pages[:1], small[:1])
    for a, b in zip(K.kv4_read(pages, table, lengths + 1, 512), K.kv4_read(small, t2, lengths + 1, 512)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("B", [1, 62, 63, 64, 65, 129])
def test_ragged_around_a_wave(K, B):
    """As many sequences as a wave finds at once, one fewer and more: rows before the first and behind the last stay as they
    were, sequences without rows, two chunks and more to join."""
    nh, n_kv, hd, page = 8, 1, 64, 16
    sizes = [(b * 7 + 3) % 4 if b else 2 for b in range(B)]
    pages, table = tables(K, B, n_kv, hd, page, 1600, 7, spare=0)
    lengths = torch.randint(0, 1590, (B,), generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)
    starts = torch.tensor([2 + sum(sizes[:b]) for b in range(B + 1)], device=DEV)
    T = int(starts[-1]) + 3
    q, k, v = rand(2, T, nh, hd) * 0.5, rand(3, T, n_kv, hd), rand(4, T, n_kv, hd)
    out = torch.full_like(q, 7.0)
    K.kv4_attn(q, pages, table, lengths, starts=starts, out=out)
    before = pages.clone()
    turned = torch.full_like(q, 7.0)
    K.kv4_append(k, v, pages, table, lengths, starts=starts, q=q, out=turned)
    for y in (out, turned):
        assert bool((y[:2] == 7).all() and (y[-3:] == 7).all())
    assert torch.equal(turned[2:-3], q[2:-3])
    some = sorted({b for b in (0, 1, B // 2, B - 3, B - 2, B - 1) if 0 <= b < B})
    for b in some:
        lo, hi = starts[b:b + 2].tolist()
        if hi > lo:
            close(out[lo:hi], before, table[b:b + 1], lengths[b:b + 1], q[lo:hi], starts=torch.tensor([0, hi - lo], device=DEV))
    assert torch.equal(pages.cpu(), appended(before, table, lengths, starts, k, v, None, 1.0, False, None, 0))


def test_starts_out_of_order(K):
    """They name rows twice or before their sequence begins: only pages of the table and rows of the output are written."""
    nh, n_kv, hd, page, T = 4, 1, 64, 16, 64
    for edges in ([0, 64, 0, 64, 0], [40, 0, 8, 64, 64], [64, 32, 0, 16, 8], [-(1 << 40), 1 << 40, -5, 70, 3]):
        B = len(edges) - 1
        pages, table = tables(K, B, n_kv, hd, page, 4096, 7, spare=64)
        starts, lengths = torch.tensor(edges, device=DEV), torch.tensor([4000, 0, 3990, 30], device=DEV)
        spare = torch.tensor(sorted(set(range(len(pages))) - set(table.flatten().tolist())), device=DEV)
        before = pages[spare].clone()
        k, q = rand(1, T, n_kv, hd), rand(2, T, nh, hd)
        wide = torch.full((T + 2, nh, hd), 7.0, device=DEV)
        K.kv4_append(k, k, pages, table, lengths, starts=starts, q=q, out=wide[1:-1])
        assert torch.equal(pages[spare], before) and bool((wide[0] == 7).all() and (wide[-1] == 7).all())
        R.fill(pages, 3)
        for heads in (4, 48):  # in blocks of 16 rows and of 128
            q = rand(2, T, heads, hd)
            need = K.kv4_attn_workspace(T, B, heads, n_kv, hd, 4096, DEV, ragged=True).numel()
            room = torch.full((need + 4096,), 77, device=DEV, dtype=torch.uint8)
            wide = torch.full((T + 2, heads, hd), 7.0, device=DEV)
            K.kv4_attn(q, pages, table, lengths, starts=starts, workspace=room[:need], out=wide[1:-1])
            assert need and bool((room[need:] == 77).all() and (wide[0] == 7).all() and (wide[-1] == 7).all())


def test_empty(K):
    pages, table = tables(K, 2, 2, 64, 16, 16, 1)
    none = torch.empty(0, device=DEV, dtype=torch.int64)
    assert K.kv4_attn(rand(1, 0, 4, 64), pages, table[:0], none).shape == (0, 4, 64)
    assert K.kv4_append(rand(1, 0, 2, 64), rand(1, 0, 2, 64), pages, table[:0], none) is None
    # tables without pages: nobody sees a key
    ln = torch.tensor([5, 0], device=DEV)
    assert bool((K.kv4_attn(rand(1, 2, 4, 64), pages, table[:, :0], ln) == 0).all())
    assert bool((K.kv4_read(pages, table[:, :0], ln, 3)[0] == 0).all())


def test_refused(K):
    pages, table = tables(K, 3, 2, 64, 32, 5000, 1, fill=False)
    ln, q, k = torch.tensor([1, 2, 3], device=DEV), rand(1, 3, 4, 64), rand(2, 3, 2, 64)
    st = torch.tensor([0, 1, 2, 3], device=DEV)
    freqs, _ = K.rope_freqs(64)
    w = torch.ones(64, device=DEV)
    attn = lambda q=q, pages=pages, table=table, ln=ln, **kw: K.kv4_attn(q, pages, table, ln, **kw)
    app = lambda k=k, v=k, pages=pages, table=table, ln=ln, **kw: K.kv4_append(k, v, pages, table, ln, **kw)
    bad = [lambda: attn(q=q.double()), lambda: attn(q=q[:2]), lambda: attn(q=q[:, :3]), lambda: attn(q=rand(1, 3, 4, 128)),
           lambda: attn(pages=pages.int()), lambda: attn(pages=pages[:0]), lambda: attn(pages=pages[..., :-1]), lambda: attn(pages=pages[:, :, ::2]),
           lambda: attn(table=table.long()), lambda: attn(table=table[:2]), lambda: attn(table=table.t()), lambda: attn(ln=ln.float()),
           lambda: attn(ln=ln[None]), lambda: attn(ln=ln.cpu()), lambda: attn(starts=st[:3]), lambda: attn(starts=st.float()),
           lambda: attn(scale=float("nan")), lambda: attn(workspace=torch.empty(16, device=DEV, dtype=torch.uint8)),
           lambda: attn(out=torch.empty(3, 4, 64, device=DEV, dtype=torch.float16)), lambda: attn(out=torch.empty(3, 4, 63, device=DEV)),
           lambda: app(k=k.half()), lambda: app(v=k[:2]), lambda: app(k=rand(1, 3, 3, 64), v=rand(1, 3, 3, 64)), lambda: app(starts=st[:2]),
           lambda: app(k=k[:2], v=k[:2]), lambda: app(freqs=freqs.float()), lambda: app(freqs=K.rope_freqs(128)[0]), lambda: app(q_norm=w),
           lambda: app(k_norm=w[:32]), lambda: app(q=q, q_norm=w.half()), lambda: app(q=q.half()), lambda: app(out=q), lambda: app(q=q[:, :0]),
           lambda: K.kv4_read(pages, table, ln, -1), lambda: K.kv4_read(pages, table, ln, 4, dtype=torch.bfloat16),
           lambda: K.kv4_pages(4, 2, 64, 24, DEV), lambda: K.kv4_pages(4, 2, 96, 32, DEV)]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError)):
            f()
            pytest.fail(f"call {i} was not refused")


@pytest.mark.parametrize("new", [1, 3, 50])
def test_steps_in_a_graph(K, new):
    """Steps as they are used: append, attention, longer lengths, captured once and replayed beside eager steps."""
    B, nh, n_kv, hd, page = 3, 14, 2, 64, 16
    pages, table = tables(K, B, n_kv, hd, page, 900, 7, fill=False)
    mine = pages.clone()
    lengths = torch.tensor([0, 300, -1], device=DEV)
    starts = None if new == 1 else torch.arange(B + 1, device=DEV) * new
    freqs, _ = K.rope_freqs(hd)
    w = 1 + rand(5, hd) * 0.1
    x = rand(1, B * new, (nh + 2 * n_kv) * hd)
    ws = K.kv4_attn_workspace(B * new, B, nh, n_kv, hd, table.shape[1] * page, DEV, ragged=new > 1)

    def step(pool, workspace):
        h = x.view(B * new, nh + 2 * n_kv, hd)
        q = K.kv4_append(h[:, nh:nh + n_kv], h[:, nh + n_kv:], pool, table, lengths, starts=starts, q=h[:, :nh], freqs=freqs, q_norm=w, k_norm=w)
        return K.kv4_attn(q, pool, table, lengths, starts=starts, workspace=workspace), q

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out, _ = step(pages, ws)
        with torch.cuda.graph(g2, stream=s):         # a second graph with the same workspace
            out2, _ = step(pages, ws)
    torch.cuda.current_stream().wait_stream(s)
    for i in range(4):
        x.copy_(rand(10 + i, *x.shape))
        want, q = step(mine, None)
        (g2 if i == 2 else g).replay()
        torch.cuda.synchronize()
        got = out2 if i == 2 else out
        assert torch.equal(got, want) and torch.equal(pages, mine), i
        close(want, mine, table, lengths, q, starts=starts)
        lengths.copy_(torch.where(lengths < 0, lengths, lengths + new))


def test_two_streams(K):
    """Calls that overlap on two streams, each with its own workspace."""
    B, nh, n_kv, hd = 4, 28, 4, 128
    pages, table = tables(K, B, n_kv, hd, 64, 3000, 7, spare=0)
    lengths = torch.tensor([2999, 2000, 5, 1000], device=DEV)
    q = [rand(i, B, nh, hd) for i in range(2)]
    want = [K.kv4_attn(x, pages, table, lengths) for x in q]
    streams = [torch.cuda.Stream() for _ in q]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for x, s in zip(q, streams):
            with torch.cuda.stream(s):
                got.append(K.kv4_attn(x, pages, table, lengths))
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert torch.equal(x, want[i % 2]), i


def test_moved_pages_in_a_graph(K):
    """A captured call reads the table anew: pages handed out again between replays, eager work of the same kind beside it."""
    B, nh, n_kv, hd, page = 3, 28, 4, 128, 32
    pages, table = tables(K, B, n_kv, hd, page, 2000, 7, spare=40)
    lengths = torch.tensor([1999, 700, 31], device=DEV)
    q = rand(1, B, nh, hd) * 0.5
    g = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        K.kv4_attn(q, pages, table, lengths)
        with torch.cuda.graph(g, stream=s):
            out = K.kv4_attn(q, pages, table, lengths)
            k, v = K.kv4_read(pages, table, lengths, 100)
    torch.cuda.current_stream().wait_stream(s)
    for i in range(4):
        perm = torch.randperm(pages.shape[0], generator=torch.Generator().manual_seed(i))[:table.numel()]
        table.copy_(perm.view(table.shape).int())
        lengths.copy_(torch.tensor([[5, 1999, 300], [1999, 1, 0], [800, -1, 1200], [64, 63, 65]][i]))
        want, rows = K.kv4_attn(q, pages, table, lengths), K.kv4_read(pages, table, lengths, 100)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(k, rows[0]) and torch.equal(v, rows[1]), i
        close(want, pages, table, lengths, q)


@pytest.mark.parametrize("sizes", [None, [1, 0, 3] * 100, [90] * 70])
def test_many_sequences(K, sizes):
    """More sequences than a wave looks at together, one row each, ragged, and in the kernel of many rows."""
    B, nh, n_kv, hd, page = 300 if sizes is None else len(sizes), 8, 1, 64, 16
    pages, table = tables(K, B, n_kv, hd, page, 600, 7, spare=0)
    lengths = torch.randint(0, 500, (B,), generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)
    starts = None if sizes is None else torch.tensor([sum(sizes[:b]) for b in range(B + 1)], device=DEV)
    q = (rand(2, B if sizes is None else sum(sizes), nh, hd) * 0.5).half()
    got = K.kv4_attn(q, pages, table, lengths, starts=starts)
    some = list(range(0, B, 37)) + [B - 1]                    # (the oracle goes row by row)
    for b in some:
        lo, hi = (b, b + 1) if starts is None else starts[b:b + 2].tolist()
        if hi > lo:
            close(got[lo:hi], pages, table[b:b + 1], lengths[b:b + 1], q[lo:hi], starts=torch.tensor([0, hi - lo], device=DEV))
    k, v = rand(3, q.shape[0], n_kv, hd), rand(4, q.shape[0], n_kv, hd)
    before = pages.clone()
    K.kv4_append(k, v, pages, table, lengths, starts=starts)
    for b in some:
        lo, hi = (b, b + 1) if starts is None else starts[b:b + 2].tolist()
        want = appended(before, table[b:b + 1], lengths[b:b + 1], torch.tensor([0, hi - lo], device=DEV), k[lo:hi], v[lo:hi], None, 1.0, False, None, 0)
        for p in table[b].tolist():
            assert torch.equal(pages[p].cpu(), want[p])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_one_kv_head_for_many(K, dtype):
    """More query heads on a kv head than the kernel of few rows takes."""
    pages, table = tables(K, 2, 1, 64, 32, 700, 7)
    lengths = torch.tensor([650, 3], device=DEV)
    q = (rand(2, 2, 530, 64) * 0.5).to(dtype)
    close(K.kv4_attn(q, pages, table, lengths), pages, table, lengths, q)


@pytest.mark.parametrize("nh,n_kv,hd", [(14, 2, 64), (28, 4, 128)])
def test_as_the_plain_caches(K, nh, n_kv, hd):
    """The operators one after the other against those of plain caches on the values that are read back: norms, rotation
    and attention of a piece of a prompt, then of a token behind it. Both attentions keep 2^-17 of a score's magnitude
    (up to 2^6 here) and of the probabilities: 2^-10 of sum p |v|, which is under 4."""
    page, L, old = 32, 60, 200
    pages = K.kv4_pages(12, n_kv, hd, page, DEV)
    table = torch.randperm(12, generator=torch.Generator().manual_seed(1)).view(1, 12).int().to(DEV)
    freqs, _ = K.rope_freqs(hd)
    w = 1 + rand(5, hd) * 0.1
    lengths, at = torch.tensor([0], device=DEV), 0
    for rows in (old, L, 1):
        x = rand(rows, rows, (nh + 2 * n_kv), hd)
        starts = torch.tensor([0, rows], device=DEV)
        q = K.kv4_append(x[:, nh:nh + n_kv], x[:, nh + n_kv:], pages, table, lengths, starts=starts, q=x[:, :nh], freqs=freqs, q_norm=w, k_norm=w)
        got = K.kv4_attn(q, pages, table, lengths, starts=starts)
        q2, k2 = K.qk_norm_rope(x[:, :nh], x[:, nh:nh + n_kv], w, w, torch.arange(at, at + rows, device=DEV), freqs)
        assert torch.allclose(q, q2, rtol=2.0 ** -18, atol=2.0 ** -18)
        k, v = K.kv4_read(pages, table, lengths + rows, at + rows)
        want = K.prefill_attn(q, k[0].contiguous(), v[0].contiguous(), pos0=at)
        assert float((got.view(rows, -1) - want).abs().max()) < 4 * 2.0 ** -10
        # a code is off by one scale at most, at 5 (kept as 4) of a block whose largest is 5 at least; by a half at most below
        # 4, of a block whose largest is beyond 3.5; by one beyond 6, at 7: a fifth of the largest, 2^-18 for k2's own rounding
        top = k2.unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True).expand(-1, -1, -1, 32).flatten(-2)
        assert bool(((k[0, :, at:].transpose(0, 1) - k2).abs() <= top * (0.2 + 2.0 ** -18)).all())
        lengths += rows
        at += rows
