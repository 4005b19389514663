"""Attention over the 4-bit cache for pieces of prompts and for keys cut into chunks, against softmax in 64 bits. The calls
are made with a workspace, whose plan says of every sequence how its work was cut: tests hold that the kernel meant (blocks
of 16 or of 128 rows) and the join of chunks were reached. Tolerances as in test_gpu_kv4.py."""

import pytest
import torch

import kv4_ref as R
from test_gpu_kv4 import DEV, K, close, rand, tables  # noqa: F401

pytestmark = pytest.mark.gpu


def attn(K, q, pages, table, lengths, starts, **kw):  # noqa: F811
    """kv4_attn's output, and (chunks, row blocks) of every sequence that has rows."""
    B, T = len(lengths), q.shape[0]
    ws = K.kv4_attn_workspace(T, B, q.shape[1], pages.shape[1], q.shape[2], table.shape[1] * pages.shape[2] * 16, DEV, ragged=starts is not None)
    assert ws.numel(), "no call of this test is a single launch"
    ws.fill_(0)
    out = K.kv4_attn(q, pages, table, lengths, starts=starts, workspace=ws, **kw)
    return out, ws[:16 * B].view(torch.int32).view(B, 4)[:, 1:3].tolist()


def ragged(sizes, before=1):
    return torch.tensor([before + sum(sizes[:b]) for b in range(len(sizes) + 1)], device=DEV)


def hold(plan, sizes, group, rows, cut=None):
    """Row blocks of ``rows`` everywhere; the sequences ``cut`` in two chunks at least."""
    for b, n in enumerate(sizes):
        if n:
            assert plan[b][1] == -(-n * group // rows), (b, plan[b])
            assert cut is None or b not in cut or plan[b][0] > 1, (b, plan[b])


# heads, tokens of a page, new rows of every sequence, rows of a block; slots held before, over 2000 where keys are cut
PIECES = [(28, 4, 128, 64, [130, 3, 0, 180], [200, 0, 9, 1700], 128), (12, 1, 64, 16, [70, 40, 45], [2500, 0, 31], 128),
          (14, 2, 64, 48, [200, 1, 61], [0, 640, 3000], 128), (2, 2, 128, 256, [600, 530], [1, 2800], 128),
          (40, 1, 128, 16, [26, 5, 17], [17, 4000, 300], 128), (48, 1, 64, 32, [12] * 70, [13 * b for b in range(70)], 128),
          (14, 2, 64, 32, [60, 2, 0, 7], [100, 2600, 5, 0], 16), (28, 4, 128, 16, [50, 1, 20], [2400, 70, 0], 16)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("nh,n_kv,hd,page,sizes,lengths,rows", PIECES)
def test_pieces(K, nh, n_kv, hd, page, sizes, lengths, rows, dtype):  # noqa: F811
    """Ragged pieces behind caches of all lengths: last blocks that are not full, waves without rows, sequences without rows, rows
    before the first sequence and behind the last."""
    T, B = sum(sizes) + 3, len(sizes)
    pages, table = tables(K, B, n_kv, hd, page, max(a + b for a, b in zip(sizes, lengths)), 9)
    starts, ln = ragged(sizes), torch.tensor(lengths, device=DEV)
    q = (rand(8, T, nh, hd) * 0.5).to(dtype)
    out = torch.full((T, nh, hd), 7.0, device=DEV, dtype=dtype)
    got, plan = attn(K, q, pages, table, ln, starts, out=out)
    hold(plan, sizes, nh // n_kv, rows, [b for b in range(B) if lengths[b] > 2000])
    assert got is out and bool((out[0] == 7).all() and (out[-2:] == 7).all())
    keep = torch.zeros(T, dtype=torch.bool, device=DEV)
    keep[1:-2] = True
    close(got, pages, table, ln, q, starts=starts, rows=keep)
    again = K.kv4_attn(q, pages, table, ln.int(), starts=starts.int())
    assert torch.equal(again[keep], got[keep])


LONG = [(14, 2, 64, [40, 3, 5, 8], 16), (28, 4, 128, [4, 1, 7, 2], 16), (14, 2, 64, [150, 60, 40, 70], 128), (28, 4, 128, [140, 60, 70, 90], 128)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("nh,n_kv,hd,sizes,rows", LONG)
def test_left_out(K, nh, n_kv, hd, sizes, rows, dtype):  # noqa: F811
    """A sequence that takes no part, single pages that there are not, a whole chunk of them, a length behind the table; bytes of
    any kind, not-a-numbers among them, where no row looks."""
    page, slots, B, T = 64, 3008, 4, sum(sizes)
    pages, table = tables(K, B, n_kv, hd, page, slots, 7)
    junk = torch.randint(0, 256, pages.shape, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV, dtype=torch.uint8)
    junk[..., 16 * hd:][junk[..., 16 * hd:] > 128] = 255
    lengths = torch.tensor([2810, -1, 2700, 1 << 35], device=DEV)
    table[0, :40] = -1                          # whole chunks, the first among them
    table[2, 3], table[2, 9], table[2, 42] = -7, 1 << 30, pages.shape[0]
    starts = ragged(sizes, 0)
    at = R.places(hd)
    for b in (0, 2):
        for slot in range(int(lengths[b]) + sizes[b], slots):
            p, off = int(table[b, slot // page]), slot % page
            if 0 <= p < pages.shape[0]:
                for f in at:
                    pages[p][:, off // 16, f[off % 16].to(DEV)] = junk[p][:, off // 16, f[off % 16].to(DEV)]
    used = set(table.flatten().tolist())
    for p in range(pages.shape[0]):
        if p not in used:
            pages[p] = junk[p]
    for p in table[1].tolist():
        pages[p] = 255
    q = (rand(8, T, nh, hd) * 0.5).to(dtype)
    got, plan = attn(K, q, pages, table, lengths, starts)
    hold(plan, sizes, nh // n_kv, rows, (0, 2, 3))
    assert 64 * 40 > 2 * -(-2860 // plan[0][0])  # (a chunk is all among the pages that there are not)
    lengths[3] = slots
    close(got, pages, table, lengths, q, starts=starts)
    lo = int(starts[1])
    assert bool((got[lo:lo + sizes[1]] == 0).all()) and bool(got.isfinite().all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("nh,n_kv,hd,sizes,rows", [(4, 2, 64, [12], 16), (4, 2, 128, [3], 16), (4, 2, 64, [290], 128), (4, 2, 128, [300], 128)])
def test_no_numbers(K, nh, n_kv, hd, sizes, rows, dtype):  # noqa: F811
    """A key or value block that is no number, in one chunk of many, reaches the rows that see it (a value's only its 32 channels)
    and no other."""
    page, old, new = 32, 2500, sizes[0]
    pages, table = tables(K, 1, n_kv, hd, page, old + new + 20, 7)
    lengths, starts = torch.tensor([old], device=DEV), torch.tensor([0, new], device=DEV)
    at = [x.to(DEV) for x in R.places(hd)]

    def spoil(slot, field, head, block):
        pages[int(table[0, slot // page]), head, slot % page // 16, at[field][slot % 16, block]] = 255

    q = (rand(8, new, nh, hd) * 0.5).to(dtype)
    spoil(old + new // 2, 3, 0, 1)                # a value among the new rows: half of them see it
    spoil(old + new, 2, 0, 0)                     # a key and a value that nobody sees
    spoil(old + new, 3, 1, 0)
    got, plan = attn(K, q, pages, table, lengths, starts)
    hold(plan, sizes, nh // n_kv, rows, (0,))
    close(got, pages, table, lengths, q, starts=starts)
    gone = got.isnan()
    assert bool(gone[new // 2:, :2, 32:64].all()) and int(gone.sum()) == (new - new // 2) * 2 * 32
    spoil(old + new - 1, 2, 1, 0)                 # the last row's own key
    spoil(5, 3, 1, 0)                             # a value that all see, in the first chunk
    spoil(1300, 2, 0, 1)                          # a key that all see, in a chunk between
    got, _ = attn(K, q, pages, table, lengths, starts)
    close(got, pages, table, lengths, q, starts=starts)
    gone = got.isnan()
    assert bool(gone[:, :2].all()) and bool(gone[-1, 2:].all()) and bool(gone[:, 2:, :32].all()) and not bool(gone[:-1, 2:, 32:].any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("nh,n_kv,hd,rows", [(14, 2, 64, 128), (28, 4, 128, 128), (28, 4, 128, 16)])
def test_pieces_in_a_graph(K, nh, n_kv, hd, rows, dtype):  # noqa: F811
    """Pieces appended and looked at, captured in two graphs that share a workspace and replayed with eager work between."""
    page, sizes = 32, [100, 0, 75, 140] if rows == 128 else [30, 0, 5, 20]
    B, T = len(sizes), sum(sizes)
    pages, table = tables(K, B, n_kv, hd, page, 3000, 7)
    mine = pages.clone()
    lengths = torch.tensor([0, 40, 2200, -1], device=DEV)
    starts = ragged(sizes, 0)
    freqs, _ = K.rope_freqs(hd)
    x = rand(1, T, nh + 2 * n_kv, hd).to(dtype)
    ws = K.kv4_attn_workspace(T, B, nh, n_kv, hd, table.shape[1] * page, DEV, ragged=True)

    def step(pool, **kw):
        q = K.kv4_append(x[:, nh:nh + n_kv], x[:, nh + n_kv:], pool, table, lengths, starts=starts, q=x[:, :nh], freqs=freqs)
        return K.kv4_attn(q, pool, table, lengths, starts=starts, **kw), q

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
        for g in graphs:
            with torch.cuda.graph(g, stream=s):
                outs.append(step(pages, workspace=ws)[0])
    torch.cuda.current_stream().wait_stream(s)
    for i in range(4):
        x.copy_(rand(10 + i, *x.shape))
        lengths.copy_(torch.tensor([[0, 40, 2200, -1], [100, 40, 2275, 5], [200, -1, 2350, 145], [2500, 3, -1, 0]][i]))
        want, q = step(mine)
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[i % 2], want) and torch.equal(pages, mine), i
        if i % 2 == 0:
            close(want, mine, table, lengths, q, starts=starts)
            _, plan = attn(K, q, mine, table, lengths, starts)
            hold(plan, sizes, nh // n_kv, rows, (2,))


def test_chunks_that_fit(K):  # noqa: F811
    """As many chunks as the launch has room for are taken: 5005 keys in 20 of 256, for three blocks of rows."""
    pages, table = tables(K, 1, 2, 64, 64, 5120, 7)
    lengths, starts, q = torch.tensor([5000], device=DEV), torch.tensor([0, 5], device=DEV), rand(8, 5, 14, 64) * 0.5
    got, plan = attn(K, q, pages, table, lengths, starts)
    assert plan == [[20, 3]]
    close(got, pages, table, lengths, q, starts=starts)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("hd", [64, 128])
def test_cut_among_many_rows(K, hd, dtype):  # noqa: F811
    """Cut sequences around one of many rows that is not: the workspace has fewer records than the launch has workgroups, and
    theirs follow one another."""
    heads, sizes, lengths = 16, [600, 19000, 590], [400, -1, 430]
    pages, table = tables(K, 3, heads, hd, 64, 1024, 7)
    starts, ln, T = ragged(sizes, 0), torch.tensor(lengths, device=DEV), sum(sizes)
    q = (rand(8, T, heads, hd) * 0.5).to(dtype)
    need = K.kv4_attn_workspace(T, 3, heads, heads, hd, 1024, DEV, ragged=True).numel()
    assert need < heads * (-(-T // 128) + 100) * 128 * (hd + 2) * 4
    room = torch.full((need + 4096,), 77, device=DEV, dtype=torch.uint8)
    got = K.kv4_attn(q, pages, table, ln, starts=starts, workspace=room[:need])
    plan = room[:48].view(torch.int32).view(3, 4).tolist()
    assert plan[0][1] > 1 and plan[1][1] == 1 and plan[2][1] > 1
    assert plan[0][0] == 0 and plan[2][0] == plan[0][1] * plan[0][2] and bool((room[need:] == 77).all())
    assert bool((got[600:-590] == 0).all())
    for b, rows in ((0, slice(0, 600)), (2, slice(T - 590, T))):
        some = slice(rows.start, rows.stop, 37)                  # (the oracle goes row by row)
        for t in range(some.start, some.stop, some.step):
            seen = ln[b:b + 1] + (t - rows.start)
            close(got[t:t + 1], pages, table[b:b + 1], seen, q[t:t + 1])
