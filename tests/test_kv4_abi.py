"""The C entries of the paged 4-bit cache and of the head norms refuse bad calls with their status before any launch
(no GPU needed); the description of a page against itself."""

import ctypes

import pytest
import torch

from kv4_ref import MAGS, places, quantize, value

F, ODD = 0x1000, 0x1002


@pytest.fixture(scope="module")
def lib():
    from pico_hip import _lib
    return _lib.lib


def call_of(fn, cls, d):
    def call(**kw):
        v = {**d, **kw}
        return fn(ctypes.byref(cls(*[v.get(n) if v.get(n) is not None or t is ctypes.c_void_p else t() for n, t in cls._fields_])), None)
    return call


def pool(**kw):
    from pico_hip._lib import Kv4Pool
    d = dict(pages=F, n_pages=9, page_stride=2 * 2 * 17 * 64, page_tokens=32, table=F, table_stride=5, table_cols=5)
    return Kv4Pool(*{**d, **kw}.values())


BAD_POOLS = (dict(n_pages=0), dict(n_pages=1 << 31), dict(page_tokens=0), dict(page_tokens=24), dict(page_tokens=1 << 21),
             dict(page_stride=2 * 2 * 17 * 64 - 16), dict(table_cols=-1), dict(table_cols=1 << 26), dict(table_stride=-1))


def test_qk_norm_rope(lib):
    from pico_hip._lib import QkNormArgs
    d = dict(type=0, q=F, q_token=384, q_head=64, q_out=F, q_out_token=384, q_out_head=64, q_weight=F, q_weight_head=0, k=F,
             k_token=128, k_head=64, k_out=F, k_out_token=128, k_out_head=64, k_weight=F, k_weight_head=64, positions=F,
             pos_dtype=2, freqs=F, rot_dim=64, amp=1.0, interleaved=0, eps=1e-6, tokens=4, n_head=6, n_kv=2, head_dim=64)
    call = call_of(lib.pe_qk_norm_rope, QkNormArgs, d)
    assert lib.pe_qk_norm_rope(None, None) == 1
    assert call(tokens=0, q=None) == 0
    for kw in (dict(type=8), dict(pos_dtype=0), dict(pos_dtype=3)):
        assert call(**kw) == 2, kw
    for kw in (dict(tokens=-1), dict(n_head=0, n_kv=0), dict(n_head=4097), dict(n_kv=4097), dict(n_head=-1), dict(head_dim=0),
               dict(head_dim=513), dict(rot_dim=0), dict(rot_dim=63), dict(rot_dim=66), dict(q_token=-1), dict(q_out_head=63),
               dict(k_out_token=63), dict(k_out_token=100), dict(k_weight_head=32), dict(q_head=32), dict(k_token=256)):
        assert call(**kw) == 3, kw
    for name in ("q", "k", "q_out", "k_out", "positions", "freqs"):
        assert call(**{name: None}) == 1, name
    for name in ("q", "k", "q_out", "k_out", "positions", "freqs", "q_weight", "k_weight"):
        assert call(**{name: ODD}) == 4, name
    # one side alone, unweighted: the other's pointers are not looked at (as far as the misaligned positions)
    assert call(n_kv=0, k=None, k_out=None, k_weight=ODD, positions=ODD) == 4
    assert call(n_head=0, q=None, q_out=None, k_weight=None, positions=ODD) == 4


def test_append(lib):
    from pico_hip._lib import Kv4AppendArgs
    d = dict(type=0, q=F, q_token=256, q_head=64, q_out=F, q_out_token=256, q_out_head=64, k=F, k_token=128, k_head=64, v=F,
             v_token=128, v_head=64, pool=pool(), lengths=F, lengths_dtype=2, starts=F, starts_dtype=2, freqs=F, rot_dim=64,
             amp=1.0, interleaved=0, q_weight=F, k_weight=F, eps=1e-6, tokens=7, batch=3, n_head=4, n_kv=2, head_dim=64)
    call = call_of(lib.pe_kv4_append, Kv4AppendArgs, d)
    assert lib.pe_kv4_append(None, None) == 1
    assert call(tokens=0, k=None) == 0 and call(batch=0, k=None) == 0
    for kw in (dict(type=2), dict(lengths_dtype=0), dict(starts_dtype=0)):
        assert call(**kw) == 2, kw
    for kw in (dict(tokens=-1), dict(tokens=1 << 23), dict(batch=-1), dict(batch=(1 << 20) + 1), dict(starts=None), dict(n_head=0),
               dict(n_head=4097), dict(n_kv=0), dict(head_dim=96), dict(rot_dim=0), dict(rot_dim=65), dict(rot_dim=66),
               dict(k_token=-1), dict(q_out_head=63), dict(q_out_token=128), dict(q_token=512), dict(n_kv=3),
               *[dict(pool=pool(**kw)) for kw in BAD_POOLS]):
        assert call(**kw) == 3, kw
    for name in ("k", "v", "q_out", "lengths"):
        assert call(**{name: None}) == 1, name
    assert call(pool=pool(pages=None)) == 1 and call(pool=pool(table=None)) == 1
    for name in ("q", "q_out", "k", "v", "lengths", "starts", "freqs", "q_weight", "k_weight"):
        assert call(**{name: ODD}) == 4, name
    for kw in (dict(pages=F + 8), dict(table=ODD), dict(page_stride=2 * 2 * 17 * 64 + 8)):
        assert call(pool=pool(**kw)) == 4, kw


def test_read(lib):
    d = dict(type=0, pool=ctypes.byref(pool()), lengths=F, dtype=2, batch=3, n_kv=2, hd=64, rows=70, k=F, v=F)
    call = lambda **kw: lib.pe_kv4_read(*{**d, **kw}.values(), None)
    assert call(pool=None) == 1 and call(batch=0) == 0 and call(rows=0, k=None) == 0
    assert call(type=8) == 2 and call(dtype=0) == 2
    for kw in (dict(batch=-1), dict(rows=-1), dict(rows=(1 << 30) + 1), dict(hd=80), dict(n_kv=0), dict(n_kv=3), dict(rows=1 << 28),
               *[dict(pool=ctypes.byref(pool(**kw))) for kw in BAD_POOLS]):
        assert call(**kw) == 3, kw
    for name in ("lengths", "k", "v"):
        assert call(**{name: None}) == 1, name
        assert call(**{name: ODD}) == 4, name


def test_attn(lib):
    from pico_hip._lib import Kv4AttnArgs
    d = dict(type=1, q=F, q_token=256, q_head=64, out=F, out_token=256, out_head=64, pool=pool(table_cols=300), lengths=F, lengths_dtype=2,
             first=1, starts=F, starts_dtype=1, tokens=7, batch=3, n_head=4, n_kv=2, head_dim=64, scale=0.125, workspace=F,
             workspace_bytes=1 << 30)
    call = call_of(lib.pe_kv4_attn, Kv4AttnArgs, d)
    assert lib.pe_kv4_attn(None, None) == 1
    assert call(tokens=0, q=None) == 0 and call(batch=0, q=None) == 0
    for kw in (dict(type=0x99), dict(lengths_dtype=3), dict(starts_dtype=0)):
        assert call(**kw) == 2, kw
    for kw in (dict(tokens=-1), dict(tokens=(1 << 22) + 1), dict(batch=-1), dict(starts=None), dict(n_head=5), dict(n_head=0),
               dict(n_kv=0), dict(head_dim=96), dict(scale=float("nan")), dict(scale=float("inf")), dict(first=1 << 41),
               dict(out_head=63), dict(out_token=128), dict(q_head=-1), *[dict(pool=pool(**kw)) for kw in BAD_POOLS]):
        assert call(**kw) == 3, kw
    for name in ("q", "out", "lengths", "workspace"):
        assert call(**{name: None}) == 1, name
    for kw in (dict(q=0x1001), dict(out=0x1001), dict(lengths=ODD), dict(starts=ODD), dict(workspace=ODD), dict(pool=pool(pages=F + 8, table_cols=300)),
               dict(pool=pool(table=ODD))):
        assert call(**kw) == 4, kw
    size = lib.pe_kv4_attn_workspace_bytes
    need = size(7, 3, 1, 4, 2, 64, 300 * 32)
    assert need > 0 and call(workspace_bytes=need - 1) == 6
    assert size(3, 3, 0, 4, 2, 64, 64) == 0      # few keys: one launch
    for args in ((7, 3, 0, 4, 2, 64, 64), (7, 0, 1, 4, 2, 64, 64), (7, 3, 1, 5, 2, 64, 64), (7, 3, 1, 4, 2, 80, 64), (7, 3, 1, 4, 2, 64, -1)):
        assert size(*args) == -3, args


def test_attn_most_rows(lib):
    """2^26 - 1 rows of heads: the join's grid of four rows a workgroup would be 2^32 threads."""
    from pico_hip._lib import Kv4AttnArgs
    d = dict(type=1, q=F, q_token=2731 * 64, q_head=64, out=F, out_token=2731 * 64, out_head=64, lengths=F, lengths_dtype=2, first=1,
             starts=F, starts_dtype=1, tokens=24573, batch=3, n_head=2731, n_kv=1, head_dim=64, scale=0.125, workspace=F,
             workspace_bytes=1 << 50, pool=pool(table_cols=300))
    assert 24573 * 2731 == (1 << 26) - 1
    assert call_of(lib.pe_kv4_attn, Kv4AttnArgs, d)() == 3


def test_public_names():
    from pico_hip import kernels
    names = {"qk_norm_rope", "kv4_pages", "kv4_append", "kv4_read", "kv4_attn", "kv4_attn_workspace"}
    assert names <= set(kernels.__all__) and all(hasattr(kernels, n) for n in kernels.__all__)


@pytest.mark.parametrize("hd", [64, 128])
def test_places_fill_a_tile(hd):
    """Every byte of a tile belongs to one field, two elements share each code byte."""
    pk, pv, sk, sv = places(hd)
    assert sorted(pk[:, 0::2].flatten().tolist()) == list(range(8 * hd)) and torch.equal(pk[:, 0::2], pk[:, 1::2])
    assert sorted(pv[:, 0::2].flatten().tolist()) == list(range(8 * hd, 16 * hd)) and torch.equal(pv[:, 0::2], pv[:, 1::2])
    assert sorted(torch.cat([sk, sv]).flatten().tolist()) == list(range(16 * hd, 17 * hd))


def test_quantize():
    x = torch.zeros(4, 32)
    x[0, :10] = torch.tensor([7.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -5.1, -0.26])
    x[1, 0], x[2, 0], x[2, 5], x[3, 3] = 7.0001, float("inf"), 1.0, 2.0 ** -120
    code, scale = quantize(x)
    assert value(code, scale)[0, :10].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, -6, -0.5] and scale[:, 0].tolist() == [127, 128, 255, 27]
    assert value(code, scale)[1, 0] == 8 and bool(value(code, scale)[2].isnan().all()) and bool((value(code, scale)[3] == 0).all())
    assert len(MAGS) == 8


@pytest.mark.parametrize("tokens,batch,n_head,n_kv,hd,capacity", [
    (65536, 1, 32, 8, 128, 65536), (1 << 20, 16, 32, 8, 128, 65536), (200000, 3, 14, 2, 64, 100000), (64, 64, 32, 8, 128, 16384),
    (5, 1, 14, 2, 64, 5120), (1 << 20, 1 << 20, 8, 1, 64, 4096)])
def test_attn_workspace_bound(lib, tokens, batch, n_head, n_kv, hd, capacity):
    """Room for the chunks of keys that are cut alone, 2^14 a launch and two a sequence, however many rows there are."""
    ragged = tokens != batch
    got = lib.pe_kv4_attn_workspace_bytes(tokens, batch, int(ragged), n_head, n_kv, hd, capacity)
    rows = 128 if -(-tokens // batch) * (n_head // n_kv) > 512 else 16
    assert 0 < got <= batch * 16 + (2 ** 14 + n_kv * 2 * (1 + batch)) * rows * (hd + 2) * 4 + 16


def test_qk_norm_most_rows(lib):
    """2^26 rows of single elements, four a workgroup: a grid of 2^32 threads."""
    from pico_hip._lib import QkNormArgs
    d = dict(type=0, q=F, q_token=2, q_head=2, q_out=F, q_out_token=2, q_out_head=2, positions=F, pos_dtype=2, freqs=F, rot_dim=2,
             amp=1.0, eps=1e-6, tokens=1 << 26, n_head=1, n_kv=0, head_dim=2)
    assert call_of(lib.pe_qk_norm_rope, QkNormArgs, d)() == 3
