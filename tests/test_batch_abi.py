"""The C entries of a batch of continuations (rotary positions, shared-prefix attention, logit rules)
refuse bad calls with their status before any launch (no GPU needed)."""

import ctypes

import pytest

F, ODD = 0x1000, 0x1002


@pytest.fixture(scope="module")
def lib():
    from pico_hip import _lib
    return _lib.lib


def test_rope_positions(lib):
    d = dict(type=0, x=F, x_token=128, x_head=64, positions=F, pos_dtype=2, freqs=F, rot=64, amp=1.0, il=0, y=F,
             y_token=128, y_head=64, tokens=4, n_head=2, hd=64)
    call = lambda **kw: lib.pe_rope_positions(*{**d, **kw}.values(), None)
    assert call(tokens=0, x=None) == 0
    for kw in (dict(type=8), dict(pos_dtype=0), dict(pos_dtype=3)):
        assert call(**kw) == 2, kw
    for kw in (dict(tokens=-1), dict(n_head=0), dict(n_head=4097), dict(hd=0), dict(rot=0), dict(rot=63), dict(rot=66),
               dict(y_token=63), dict(y_head=63), dict(y_token=64, y_head=64), dict(y_token=100), dict(x_token=-1),
               dict(y_token=0), dict(y_head=0), dict(x_token=192), dict(x_head=0), dict(y_token=64, y_head=256)):
        assert call(**kw) == 3, kw
    for name in ("x", "positions", "freqs", "y"):
        assert call(**{name: None}) == 1, name
        assert call(**{name: ODD}) == 4, name


def test_rope_append(lib):
    d = dict(qkv=F, stride=512, positions=F, pos_dtype=2, freqs=F, cos=None, sin=None, rows=0, rot=64, amp=1.0, il=0,
             n_head=4, n_kv=2, hd=64, batch=3, q=F, cache=0, k=F, v=F, capacity=5, offset=0)
    call = lambda **kw: lib.pe_rope_append(*{**d, **kw}.values(), None)
    assert call(batch=0, qkv=None) == 0
    for kw in (dict(cache=6), dict(pos_dtype=0)):
        assert call(**kw) == 2, kw
    for kw in (dict(stride=511), dict(batch=-1), dict(batch=1 << 31), dict(n_head=0), dict(n_kv=0), dict(hd=0), dict(rot=0),
               dict(rot=65), dict(rot=66), dict(capacity=0), dict(freqs=None, cos=F, sin=F), dict(batch=1 << 28)):
        assert call(**kw) == 3, kw
    for kw in (dict(qkv=None), dict(positions=None), dict(q=None), dict(k=None), dict(v=None),
               dict(freqs=None, cos=F, rows=9), dict(freqs=None, sin=F, rows=9)):
        assert call(**kw) == 1, kw
    for name in ("qkv", "positions", "freqs", "q", "k", "v"):
        assert call(**{name: ODD}) == 4, name


def test_shared_prefix_attn(lib):
    from pico_hip._lib import SharedPrefixArgs
    d = dict(q=F, cache_type=0, k_prefix=F, v_prefix=F, prefix_capacity=3000, prefix_len=None, prefix_len_dtype=0,
             prefix_len_add=3000, k_own=F, v_own=F, own_capacity=40, own_len=F, own_len_dtype=2, own_len_add=0, batch=3,
             n_head=14, n_kv=2, head_dim=64, scale=0.125, round_fp16=0, out=F, workspace=F, workspace_bytes=1 << 30)
    def call(**kw):
        v = {**d, **kw}
        return lib.pe_shared_prefix_attn(ctypes.byref(SharedPrefixArgs(*[v[n] for n, _ in SharedPrefixArgs._fields_])), None)
    assert lib.pe_shared_prefix_attn(None, None) == 1
    assert call(batch=0, q=None) == 0
    for kw in (dict(cache_type=8), dict(prefix_len_dtype=3), dict(own_len_dtype=-1)):
        assert call(**kw) == 2, kw
    for kw in (dict(batch=-1), dict(n_head=15), dict(n_kv=0), dict(head_dim=96), dict(prefix_capacity=-1),
               dict(own_capacity=-1), dict(prefix_capacity=(1 << 30) + 1, prefix_len_add=1 << 40), dict(batch=1 << 21)):
        assert call(**kw) == 3, kw
    for kw in (dict(q=None), dict(out=None), dict(k_prefix=None), dict(v_prefix=None), dict(k_own=None), dict(v_own=None),
               dict(own_len=None), dict(prefix_len_dtype=1), dict(workspace=None)):
        assert call(**kw) == 1, kw
    for name in ("q", "out", "k_prefix", "v_prefix", "k_own", "v_own", "workspace", "own_len"):
        assert call(**{name: ODD}) == 4, name
    size = lib.pe_shared_prefix_attn_workspace_bytes
    need = size(0, 3, 14, 2, 64, 3000, 40)
    assert need > 0 and call(workspace_bytes=need - 1) == 6
    # a shorter prefix needs less; one whose length is on the device, the capacity's
    less = size(0, 3, 14, 2, 64, 1000, 40)
    assert less < need and call(prefix_len=F, prefix_len_dtype=2, workspace_bytes=less) == 6
    assert size(0, 3, 14, 2, 64, 300, 40) == 0      # few keys: one launch
    for args in ((0, 14, 2, 64, 300, 40), (3, 14, 3, 64, 300, 40), (3, 14, 2, 80, 300, 40), (3, 14, 2, 64, -1, 40)):
        assert size(0, *args) == -3, args
    assert size(8, 3, 14, 2, 64, 300, 40) == -2


def test_adjust_logits(lib):
    from pico_hip._lib import LogitArgs
    d = {n: None for n, _ in LogitArgs._fields_}
    d.update(type=0, x=F, x_stride=100, y=F, y_stride=100, batch=2, vocab=100, history=F, history_dtype=2, history_stride=9,
             history_len=9, lengths=F, lengths_dtype=2, prompt=F, prompt_dtype=2, prompt_stride=0, prompt_len=4,
             repetition_rows=F, frequency_rows=F, presence_rows=F, repetition=1.0, frequency=0.0, presence=0.0, bias=F,
             bias_stride=0, mask=F, mask_stride=4)
    def call(**kw):
        v = {**d, **kw}
        return lib.pe_adjust_logits(ctypes.byref(LogitArgs(*[v[n] for n, _ in LogitArgs._fields_])), None)
    assert lib.pe_adjust_logits(None, None) == 1
    assert call(batch=0, x=None) == 0
    for kw in (dict(type=2), dict(history_dtype=0), dict(lengths_dtype=3), dict(prompt_dtype=0)):
        assert call(**kw) == 2, kw
    for kw in (dict(batch=-1), dict(vocab=0), dict(vocab=1 << 31), dict(y_stride=99), dict(x_stride=-1), dict(history_len=-1),
               dict(prompt_len=1 << 31), dict(history_stride=-1), dict(bias_stride=-1), dict(mask_stride=-1),
               dict(x_stride=101), dict(x_stride=0)):
        assert call(**kw) == 3, kw
    for name in ("x", "y"):
        assert call(**{name: None}) == 1, name
    for name in ("x", "y", "history", "lengths", "prompt", "repetition_rows", "frequency_rows", "presence_rows", "bias", "mask"):
        assert call(**{name: ODD}) == 4, name


def test_shared_prefix_attn_scale(lib):
    """A scale that is no number, or infinite, is refused."""
    from pico_hip._lib import SharedPrefixArgs
    d = dict(q=F, cache_type=1, k_prefix=F, v_prefix=F, prefix_capacity=3000, prefix_len_add=3000, k_own=F, v_own=F,
             own_capacity=40, own_len=F, own_len_dtype=2, batch=3, n_head=14, n_kv=2, head_dim=64, out=ODD, workspace=F,
             workspace_bytes=1 << 30)
    call = lambda x: lib.pe_shared_prefix_attn(ctypes.byref(SharedPrefixArgs(scale=x, **d)), None)
    assert [call(x) for x in (0.125, -2.0, 0.0, 3e38)] == [4] * 4      # as far as the misaligned output
    assert [call(x) for x in (float("nan"), float("inf"), float("-inf"))] == [3] * 3


def test_public_names():
    """The batch operators are among the names that the module offers."""
    from pico_hip import kernels
    names = {"rope_freqs", "rope_positions", "rope_append", "shared_prefix_attn", "shared_prefix_attn_workspace", "adjust_logits"}
    assert names <= set(kernels.__all__) and all(hasattr(kernels, n) for n in kernels.__all__)
