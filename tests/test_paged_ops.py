"""CPU tests of the paged-cache operators' refusals: every bad call is turned
away by the C entry before any device work (the pointers here are never
touched), and by the Python wrapper for tensors that are not on a GPU."""
import ctypes as C

import pytest

from strataflow_b200 import build as B
from strataflow_b200 import lib as L

X = 1 << 20  # a 16-byte aligned address that nothing reads


@pytest.fixture(scope="module")
def sfk():
    B.build()
    return L.load()


APPEND = dict(io=L.TYPE_F32, q=X, qs=8 * 64, k=X, ks=2 * 64, v=X, vs=2 * 64, n=3, hq=8, hkv=2, hd=64, qw=None, kw=None,
              eps=1e-6, neox=0, n_rot=64, freqs=X, rope_pos=None, n_axes=0, axis=None, kvt=L.KV_F16, kp=X, vp=X,
              n_pages=4, table=X, n_seq=3, max_pages=2, seq=None, pos=X, out=X, outs=8 * 64, status=None, stream=None)
DECODE = dict(io=L.TYPE_F32, q=X, qs=8 * 64, kvt=L.KV_F16, kp=X, vp=X, n_pages=4, table=X, max_pages=2, pos=X, n=3, hq=8,
              hkv=2, hd=64, scale=0.0, window=0, sink=0, out=X, ws=None, ws_bytes=0, status=None, stream=None)
PREFILL = dict(io=L.TYPE_F32, q=X, qs=8 * 64, n_tok=5, kvt=L.KV_F16, kp=X, vp=X, n_pages=4, table=X, max_pages=2, start=X,
               lens=X, n=3, hq=8, hkv=2, hd=64, scale=0.0, window=0, sink=0, out=X, status=None, stream=None)


def call(sfk, fn, base, **kw):
    assert set(kw) <= set(base)
    return getattr(sfk, fn)(*{**base, **kw}.values())


@pytest.mark.parametrize("kw,why", [
    (dict(io=L.TYPE_Q8_0), b"element type"), (dict(kvt=7), b"element type"), (dict(hd=60), b"head_dim"),
    (dict(hd=264), b"head_dim"), (dict(hd=0), b"head_dim"), (dict(hq=0), b"heads"), (dict(hkv=0), b"heads"),
    (dict(n_rot=66), b"n_rot"), (dict(n_rot=12), b"n_rot"), (dict(n_rot=24, neox=1), b"n_rot"), (dict(n_rot=-8), b"n_rot"),
    (dict(n=-1), b"sizes"), (dict(n_pages=0), b"sizes"), (dict(max_pages=0), b"sizes"), (dict(n_seq=-1), b"sizes"),
    (dict(max_pages=(1 << 27) + 1), b"sizes"), (dict(qw=X, eps=-1.0), b"eps"), (dict(kw=X, eps=float("nan")), b"eps"),
    (dict(n_axes=3), b"axes"), (dict(rope_pos=X, n_axes=0), b"axes"), (dict(rope_pos=X, n_axes=9), b"axes"),
    (dict(axis=bytes(32)), b"axes"), (dict(rope_pos=X, n_axes=2, axis=bytes([0] * 31 + [2])), b"axis 2"),
    (dict(q=None), b"null"), (dict(k=None), b"null"), (dict(v=None), b"null"), (dict(kp=None), b"null"),
    (dict(vp=None), b"null"), (dict(table=None), b"null"), (dict(pos=None), b"null"), (dict(out=None), b"null"),
    (dict(freqs=None), b"null"), (dict(n_seq=2), b"without a sequence list"), (dict(kp=X + 8), b"16-byte"),
    (dict(vp=X + 2), b"16-byte"), (dict(qs=511), b"strides"), (dict(ks=127), b"strides"), (dict(vs=0), b"strides"),
    (dict(outs=1), b"strides"),
])
def test_append_refusals(sfk, kw, why):
    assert call(sfk, "sfk_qk_norm_rope_append", APPEND, **kw) == L.SFK_ERR_INVALID_ARGUMENT
    assert why in sfk.sfk_last_error()


ATTN = [
    (dict(io=3), b"element type"), (dict(kvt=-1), b"element type"), (dict(io=L.TYPE_BF16), b"own type"),
    (dict(io=L.TYPE_F16, kvt=L.KV_F32), b"own type"), (dict(hd=96), b"head_dim"), (dict(hd=0), b"head_dim"),
    (dict(hq=0), b"heads"), (dict(hkv=3), b"heads"), (dict(hkv=-2), b"heads"), (dict(n_pages=0), b"pages"),
    (dict(max_pages=0), b"pages"), (dict(max_pages=(1 << 27) + 1), b"pages"), (dict(window=-1), b"window"),
    (dict(sink=-1), b"window"), (dict(scale=float("inf")), b"scale"), (dict(scale=float("nan")), b"scale"),
    (dict(scale=-1.0), b"scale"), (dict(q=None), b"null"), (dict(kp=None), b"null"), (dict(vp=None), b"null"),
    (dict(table=None), b"null"), (dict(out=None), b"null"), (dict(kp=X + 4), b"16-byte"), (dict(vp=X + 8), b"16-byte"),
    (dict(qs=100), b"q_stride"),
]


@pytest.mark.parametrize("kw,why", ATTN + [(dict(pos=None), b"null"), (dict(n=-1), b"sequences"),
                                           (dict(n=65536), b"sequences"), (dict(ws=X + 8, ws_bytes=64), b"workspace")])
def test_decode_refusals(sfk, kw, why):
    assert call(sfk, "sfk_attn_decode_window", DECODE, **kw) == L.SFK_ERR_INVALID_ARGUMENT
    assert why in sfk.sfk_last_error()


@pytest.mark.parametrize("kw,why", ATTN + [(dict(start=None), b"null"), (dict(lens=None), b"null"), (dict(n=-1), b"sizes"),
                                           (dict(n_tok=-1), b"sizes"), (dict(n=65536), b"sizes"), (dict(n_tok=1 << 29), b"in one call")])
def test_prefill_refusals(sfk, kw, why):
    assert call(sfk, "sfk_attn_prefill_window", PREFILL, **kw) == L.SFK_ERR_INVALID_ARGUMENT
    assert why in sfk.sfk_last_error()


def test_scale_that_overflows_and_out_over_q(sfk):
    for fn, base in (("sfk_attn_decode_window", DECODE), ("sfk_attn_prefill_window", PREFILL)):
        assert call(sfk, fn, base, scale=3e38) == L.SFK_ERR_INVALID_ARGUMENT
        assert b"scale" in sfk.sfk_last_error()
    assert call(sfk, "sfk_attn_prefill_window", PREFILL, out=PREFILL["q"]) == L.SFK_ERR_INVALID_ARGUMENT
    assert b"out is q" in sfk.sfk_last_error()


def test_empty_calls_do_nothing(sfk):
    """No token, no sequence: fine without any pointer, and no launch."""
    assert call(sfk, "sfk_qk_norm_rope_append", APPEND, n=0, q=None, k=None, v=None, pos=None, out=None) == L.SFK_OK
    assert call(sfk, "sfk_attn_decode_window", DECODE, n=0, q=None, out=None, pos=None) == L.SFK_OK
    assert call(sfk, "sfk_attn_prefill_window", PREFILL, n=0, q=None) == L.SFK_OK
    assert call(sfk, "sfk_attn_prefill_window", PREFILL, n_tok=0, q=None) == L.SFK_OK


def test_decode_workspace(sfk):
    """Asked for where a small batch reads a long context, refused sizes need none."""
    f = sfk.sfk_attn_decode_window_workspace
    assert f(1, 32, 8, 128, 2048, 0, 0) > 0
    assert f(1, 32, 8, 128, 2048, 256, 4) == 0 and f(1, 32, 8, 128, 16, 0, 0) == 0  # a short context
    assert f(64, 32, 8, 128, 2048, 0, 0) == 0                                       # a batch that fills the GPU
    assert f(0, 32, 8, 128, 2048, 0, 0) == 0 and f(1, 31, 8, 128, 2048, 0, 0) == 0 and f(1, 32, 8, 128, 0, 0, 0) == 0


def test_device_status_needs_a_word(sfk):
    assert sfk.sfk_device_status(None, None) == L.SFK_ERR_INVALID_ARGUMENT


def test_wrapper_refuses_cpu_tensors():
    import torch

    from strataflow_b200 import ops
    q, pool = torch.zeros(1, 2, 32), torch.zeros(2, 1, 16, 32)
    t, pos = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(L.SfkError) as e:
        ops.attn_decode_window(q, pool, pool, t, pos)
    assert e.value.status == L.SFK_ERR_INVALID_ARGUMENT
    with pytest.raises(L.SfkError):
        ops.attn_prefill_window(q, pool, pool, t, pos, pos)
    with pytest.raises(L.SfkError):
        ops.qk_norm_rope_append(q, q[:, :1], q[:, :1], pool, pool, t, pos)
    with pytest.raises(L.SfkError):
        ops.check_status(pos)


def test_rope_axes():
    from strataflow_b200 import ops
    assert ops.rope_axes([2, 3, 1]) == bytes([0, 0, 1, 1, 1, 2])
    assert ops.rope_axes([3, 1, 2], interleaved=True) == bytes([0, 1, 2, 0, 2, 0])
    f = ops.rope_freqs(8, 10000.0, 0.5, device="cpu").tolist()
    assert f == pytest.approx([0.5, 0.05, 0.005, 0.0005], rel=1e-7)


def test_abi_struct_free(sfk):
    """The entries take plain values only: the table's argument counts are the calls' above."""
    for fn, base in (("sfk_qk_norm_rope_append", APPEND), ("sfk_attn_decode_window", DECODE),
                     ("sfk_attn_prefill_window", PREFILL)):
        assert len(L._SIGS[fn][1]) == len(base) and L._SIGS[fn][0] is C.c_int32
