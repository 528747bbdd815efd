"""Operator-level entry points over torch CUDA tensors (device memory only).

Each call forwards device pointers to libsfk.so (include/sfk.h) on the tensor's
current CUDA stream.  Mirrors the ggml ops the reference's decode path issues
(src/model/engine/engine.cpp): ggml_get_rows dequant (:2712), ggml_mul_mat
(:1882-1889,1905,2994), ggml_mul_mat_id (:1967-1970), the fused expert segment
(:1956-1989) and the decode attention (:1751-1761).
"""
from __future__ import annotations

import ctypes as C
import functools

import torch

from . import lib as L


def _ptr(t: torch.Tensor):
    assert t.is_cuda and t.is_contiguous()
    return C.c_void_p(t.data_ptr())


def _stream(t: torch.Tensor):
    return C.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def dev_row_bytes(qtype: int, K: int) -> int:
    return int(L.load().sfk_dev_row_bytes(qtype, K))


def repack(qtype: int, gguf: torch.Tensor, nrows: int, K: int) -> torch.Tensor:
    """GGUF rows (uint8 CUDA tensor) -> device-layout weight tensor."""
    out = torch.empty(nrows * dev_row_bytes(qtype, K), dtype=torch.uint8, device=gguf.device)
    L.check(L.load().sfk_repack(qtype, _ptr(gguf), _ptr(out), nrows, K, _stream(gguf)))
    return out


def unpack(qtype: int, dev: torch.Tensor, nrows: int, K: int, gguf_bytes: int) -> torch.Tensor:
    out = torch.empty(gguf_bytes, dtype=torch.uint8, device=dev.device)
    L.check(L.load().sfk_unpack(qtype, _ptr(dev), _ptr(out), nrows, K, _stream(dev)))
    return out


def dequantize(qtype: int, gguf: torch.Tensor, n: int) -> torch.Tensor:
    out = torch.empty(n, dtype=torch.float32, device=gguf.device)
    L.check(L.load().sfk_dequantize(qtype, _ptr(gguf), _ptr(out), n, _stream(gguf)))
    return out


def quantize_act(act_type: int, x: torch.Tensor) -> torch.Tensor:
    """[b][K] f32 -> GGUF Q8_K (292 B / 256) or Q8_0 (34 B / 32) blocks."""
    b, K = x.shape
    nbytes = (K // 256) * 292 if act_type == L.TYPE_Q8_K else (K // 32) * 34
    out = torch.empty(b * nbytes, dtype=torch.uint8, device=x.device)
    L.check(L.load().sfk_quantize_act(act_type, _ptr(x), b, K, _ptr(out), _stream(x)))
    return out


def mul_mat(qtype: int, w_dev: torch.Tensor, rows: int, K: int, x: torch.Tensor) -> torch.Tensor:
    b = x.shape[0]
    y = torch.empty((b, rows), dtype=torch.float32, device=x.device)
    L.check(L.load().sfk_mul_mat(qtype, _ptr(w_dev), rows, K, _ptr(x), b, _ptr(y), _stream(x)))
    return y


def mul_mat_tc(qtype: int, w_dev: torch.Tensor, rows: int, K: int, x: torch.Tensor) -> torch.Tensor:
    """The same product for any number of activation rows on the tensor cores
    (sfk_mul_mat_tc): y [n][rows]."""
    n = x.shape[0]
    y = torch.empty((n, rows), dtype=torch.float32, device=x.device)
    L.check(L.load().sfk_mul_mat_tc(qtype, _ptr(w_dev), rows, K, _ptr(x), n, _ptr(y), _stream(x)))
    return y


def mul_mat_id(qtype: int, w_dev: torch.Tensor, n_expert: int, rows: int, K: int, x: torch.Tensor,
               ids: torch.Tensor) -> torch.Tensor:
    """x: [b][K] (broadcast over each token's experts) or [b][k][K]."""
    b, k = ids.shape
    per_pair = 1 if x.dim() == 3 else 0
    y = torch.empty((b, k, rows), dtype=torch.float32, device=x.device)
    L.check(L.load().sfk_mul_mat_id(qtype, _ptr(w_dev), n_expert, rows, K, _ptr(x), per_pair, _ptr(ids), b, k,
                                    _ptr(y), _stream(x)))
    return y


def mul_mat_id_tc(qtype: int, w_dev: torch.Tensor, n_expert: int, rows: int, K: int, x: torch.Tensor,
                  ids: torch.Tensor) -> torch.Tensor:
    """mul_mat_id on the tensor cores (sfk_mul_mat_id_tc), for batches of
    many routed pairs; the same arguments and result layout as mul_mat_id."""
    b, k = ids.shape
    per_pair = 1 if x.dim() == 3 else 0
    y = torch.empty((b, k, rows), dtype=torch.float32, device=x.device)
    L.check(L.load().sfk_mul_mat_id_tc(qtype, _ptr(w_dev), n_expert, rows, K, _ptr(x), per_pair, _ptr(ids), b, k,
                                       _ptr(y), _stream(x)))
    return y


def moe_ffn(type_gu: int, type_down: int, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor, n_expert: int,
            d: int, F: int, x: torch.Tensor, res: torch.Tensor | None, ids: torch.Tensor,
            w: torch.Tensor) -> torch.Tensor:
    b, k = ids.shape
    out = torch.empty((b, d), dtype=torch.float32, device=x.device)
    L.check(L.load().sfk_moe_ffn(type_gu, type_down, _ptr(gate), _ptr(up), _ptr(down), n_expert, d, F, _ptr(x),
                                 _ptr(res) if res is not None else None, _ptr(ids), _ptr(w), b, k, _ptr(out),
                                 _stream(x)))
    return out


def attn_decode_paged(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                      positions: torch.Tensor, n_head: int, n_head_kv: int, head_dim: int) -> torch.Tensor:
    b = q.shape[0]
    kv_type = L.KV_F16 if k_pages.dtype == torch.float16 else L.KV_F32
    out = torch.empty((b, n_head * head_dim), dtype=torch.float32, device=q.device)
    L.check(L.load().sfk_attn_decode_paged(_ptr(q), _ptr(k_pages), _ptr(v_pages), kv_type, k_pages.shape[0],
                                           _ptr(page_table),
                                           page_table.shape[1], _ptr(positions), b, n_head, n_head_kv, head_dim,
                                           _ptr(out), _stream(q)))
    return out


def sample_logits(logits: torch.Tensor, temperature: float, top_k: int = 0, top_p: float = 1.0, seed: int = 0,
                  step: int = 0) -> int:
    """The generate loop's device sampler on f32 logits [V] (sfk_sample_logits)."""
    sp = L.Sampling(float(temperature), float(top_p), int(top_k), int(seed), 0, -1)
    tok = C.c_int32()
    L.check(L.load().sfk_sample_logits(_ptr(logits), int(logits.numel()), C.byref(sp), int(step), C.byref(tok),
                                       _stream(logits)))
    return tok.value


# ---- paged-cache operators (sfk_qk_norm_rope_append, sfk_attn_*_window) ---------
# They run on the current stream of the tensors' device and return without
# waiting; nothing is allocated but the output and, for single tokens over a long
# context, a workspace (by torch, on that stream), so they can be captured into a
# CUDA graph.  Refusals raise SfkError (invalid argument).  `status`, an int32
# CUDA tensor of one zero, collects what only the device can see (a page id or a
# position outside its range, a wait inside a kernel that ran out: the outputs
# concerned are NaN then); check_status reads it.
_ROW_TYPES = {torch.float32: L.TYPE_F32, torch.float16: L.TYPE_F16, torch.bfloat16: L.TYPE_BF16}
_KV_TYPES = {torch.float32: L.KV_F32, torch.float16: L.KV_F16, torch.bfloat16: L.KV_BF16}


def _refuse(msg: str):
    raise L.SfkError(L.SFK_ERR_INVALID_ARGUMENT, msg)


def _rows(t: torch.Tensor, what: str, heads: int, hd: int, dtype, dev: int) -> tuple[int, int]:
    """Pointer and token stride of [tokens][heads][hd] rows whose heads are contiguous."""
    shape, s = t.shape, t.stride()
    if len(shape) != 3 or shape[1] != heads or shape[2] != hd or t.dtype is not dtype or t.get_device() != dev:
        _refuse(f"{what}: {dtype} [tokens][{heads}][{hd}] on cuda:{dev} is wanted, got {t.dtype} {tuple(shape)} on "
                f"{t.device}")
    if s[2] != 1 or (s[1] != hd and heads > 1):
        _refuse(f"{what}: a token's heads have to be contiguous, got strides {s}")
    return t.data_ptr(), (s[0] if shape[0] > 1 else max(s[0], heads * hd))


def _plain(t: torch.Tensor, what: str, dtype, shape, dev: int) -> int:
    """Pointer of a contiguous tensor of that type and shape."""
    if t.dtype is not dtype or t.shape != shape or t.get_device() != dev or not t.is_contiguous():
        _refuse(f"{what}: contiguous {dtype} {list(shape)} on cuda:{dev} is wanted, got {t.dtype} {list(t.shape)} on "
                f"{t.device}")
    return t.data_ptr()


def _int32(t: torch.Tensor, what: str, shape, dev: int) -> int:
    return _plain(t, what, torch.int32, shape, dev)


def _f32(t: torch.Tensor | None, what: str, n: int, dev: int) -> int | None:
    return None if t is None else _plain(t, what, torch.float32, (n,), dev)


def _pools(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, dev: int) -> tuple[int, int, int]:
    """(kv type, kv heads, head_dim) of a checked cache."""
    shape, kvt = k_pages.shape, _KV_TYPES.get(k_pages.dtype)
    if len(shape) != 4 or shape[2] != 16 or v_pages.shape != shape or v_pages.dtype is not k_pages.dtype or kvt is None:
        _refuse(f"page pools: two [n_pages][n_head_kv][16][head_dim] of one type (f32, f16, bf16) are wanted, got "
                f"{k_pages.dtype} {tuple(k_pages.shape)} and {v_pages.dtype} {tuple(v_pages.shape)}")
    if (not (k_pages.is_contiguous() and v_pages.is_contiguous()) or k_pages.get_device() != dev or
            v_pages.get_device() != dev):
        _refuse(f"page pools: contiguous and on cuda:{dev}")
    if page_table.dim() != 2:
        _refuse("page_table: [n_seq][max_pages] is wanted")
    return kvt, shape[1], shape[3]


def _cuda_device(t: torch.Tensor, what: str) -> int:
    dev = t.get_device()
    if dev < 0:
        _refuse(f"{what}: a CUDA tensor is wanted, got one on {t.device}")
    return dev


def _elsewhere(dev: int) -> bool:
    """Whether `dev` is not the current device, on which the library launches."""
    return dev != torch.cuda.current_device()


def _stream_of(dev: int) -> int:
    return torch._C._cuda_getCurrentRawStream(dev)


def _status(status: torch.Tensor | None, dev: int) -> int | None:
    return None if status is None else _int32(status, "status", (1,), dev)


def check_status(status: torch.Tensor) -> None:
    """Wait for the current stream; raise SfkError if the status word of earlier
    paged-cache calls records an error, and clear it."""
    dev = _cuda_device(status, "status")
    with torch.cuda.device(dev):
        L.check(L.load().sfk_device_status(_status(status, dev), _stream_of(dev)))


def rope_freqs(n_rot: int, base: float = 10000.0, scale: float = 1.0, device="cuda") -> torch.Tensor:
    """Rotation frequencies base^(-2i / n_rot) * scale, f32 [n_rot / 2]."""
    i = torch.arange(n_rot // 2, dtype=torch.float64)
    return (base ** (-2 * i / n_rot) * scale).to(torch.float32).to(device)


def rope_axes(sections, interleaved: bool = False) -> bytes:
    """The axis of each pair: `sections[a]` pairs on axis a, in runs, or dealt
    out in turn (each axis as long as it has pairs left) when interleaved."""
    if not interleaved:
        return bytes(a for a, n in enumerate(sections) for _ in range(n))
    left, out = list(sections), []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                out.append(a)
    return bytes(out)


def qk_norm_rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor,
                        v_pages: torch.Tensor, page_table: torch.Tensor, pos: torch.Tensor, *,
                        seq: torch.Tensor | None = None, freqs: torch.Tensor | None = None, neox: bool = False,
                        q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, eps: float = 1e-6,
                        rope_pos: torch.Tensor | None = None, axes: bytes | None = None,
                        out: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """sfk_qk_norm_rope_append: norm (q_norm / k_norm [hd]) and rotate
    (freqs [n_rot / 2], None: no rotation) the heads of q [tokens][Hq][hd] and
    k [tokens][Hkv][hd], append k and v to the cache at position pos[t] of
    sequence seq[t] (None: t), and return the rotated q (`out`, which may be
    q).  rope_pos [n_axes][tokens] with axes (rope_axes) replaces the cache
    positions in the rotation.  Rows with pos < 0 are padding."""
    dev = _cuda_device(q, "q")
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return qk_norm_rope_append(q, k, v, k_pages, v_pages, page_table, pos, seq=seq, freqs=freqs, neox=neox,
                                       q_norm=q_norm, k_norm=k_norm, eps=eps, rope_pos=rope_pos, axes=axes, out=out,
                                       status=status)
    kvt, kvh, hd = _pools(k_pages, v_pages, page_table, dev)
    dtype, shape = q.dtype, q.shape
    n, heads = shape[0], shape[1] if len(shape) == 3 else 0
    io = _ROW_TYPES.get(dtype)
    if io is None:
        _refuse(f"q: f32, f16 or bf16 is wanted, got {dtype}")
    qp, qs = _rows(q, "q", heads, hd, dtype, dev)
    kp, ks = _rows(k, "k", kvh, hd, dtype, dev)
    vp, vs = _rows(v, "v", kvh, hd, dtype, dev)
    if k.shape[0] != n or v.shape[0] != n:
        _refuse(f"q, k and v: {n}, {k.shape[0]} and {v.shape[0]} tokens")
    if out is None:
        out = q.new_empty(shape)
        op, os_ = out.data_ptr(), heads * hd
    else:
        op, os_ = _rows(out, "out", heads, hd, dtype, dev)
        if out.shape[0] != n:
            _refuse(f"out: {n} tokens are wanted, got {out.shape[0]}")
    n_seq, max_pages = page_table.shape
    fp, n_rot = None, 0
    if freqs is not None:
        n_rot = 2 * freqs.numel()
        fp = _plain(freqs, "freqs", torch.float32, (n_rot // 2,), dev)
    rp, n_axes = None, 0
    if rope_pos is not None:
        n_axes = rope_pos.shape[0] if rope_pos.dim() == 2 else 0
        rp = _int32(rope_pos, "rope_pos", (n_axes, n), dev)
    if axes is not None and len(axes) != n_rot // 2:
        _refuse(f"axes: {n_rot // 2} pairs are rotated, got {len(axes)}")
    st = L.load().sfk_qk_norm_rope_append(
        io, qp, qs, kp, ks, vp, vs, n, heads, kvh, hd, None if q_norm is None else _f32(q_norm, "q_norm", hd, dev),
        None if k_norm is None else _f32(k_norm, "k_norm", hd, dev), eps, neox, n_rot, fp, rp, n_axes, axes, kvt,
        k_pages.data_ptr(), v_pages.data_ptr(), k_pages.shape[0],
        _int32(page_table, "page_table", (n_seq, max_pages), dev), n_seq, max_pages,
        None if seq is None else _int32(seq, "seq", (n,), dev), _int32(pos, "pos", (n,), dev), op, os_,
        None if status is None else _status(status, dev), _stream_of(dev))
    if st:
        L.check(st)
    return out


def _attn_rows(q: torch.Tensor, k_pages: torch.Tensor, kvh: int, hd: int, window: int, n_sink: int,
               out: torch.Tensor | None, dev):
    if not (0 <= window < 1 << 31 and 0 <= n_sink < 1 << 31):
        _refuse(f"window {window}, n_sink {n_sink}")
    heads = q.shape[1] if q.dim() == 3 else 0
    if q.dtype not in _ROW_TYPES:
        _refuse(f"q: f32, f16 or bf16 is wanted, got {q.dtype}")
    if q.dtype != torch.float32 and q.dtype != k_pages.dtype:
        _refuse(f"q: {q.dtype} rows need a cache of their own type, got {k_pages.dtype}")
    qp, qs = _rows(q, "q", heads, hd, q.dtype, dev)
    shape = (q.shape[0], heads * hd)
    if out is None:
        out = q.new_empty(shape)
        return heads, qp, qs, out, out.data_ptr()
    return heads, qp, qs, out, _plain(out, "out", q.dtype, shape, dev)


@functools.lru_cache(maxsize=4096)
def _decode_workspace(dev: int, *sizes: int) -> int:
    with torch.cuda.device(dev):
        return int(L.load().sfk_attn_decode_window_workspace(*sizes))


def attn_decode_window(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                       positions: torch.Tensor, *, window: int = 0, n_sink: int = 0, scale: float = 0.0,
                       out: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """sfk_attn_decode_window: q [n_seq][Hq][hd], one token of each sequence at
    positions[t] (negative: padding, zeros) over the keys it sees: j <= p and,
    with window > 0, j > p - window or j < n_sink.  Returns [n_seq][Hq * hd]
    (`out`, which may be q's own memory where q is contiguous)."""
    dev = _cuda_device(q, "q")
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return attn_decode_window(q, k_pages, v_pages, page_table, positions, window=window, n_sink=n_sink,
                                      scale=scale, out=out, status=status)
    kvt, kvh, hd = _pools(k_pages, v_pages, page_table, dev)
    heads, qp, qs, out, op = _attn_rows(q, k_pages, kvh, hd, window, n_sink, out, dev)
    n, max_pages = q.shape[0], page_table.shape[1]
    ws_bytes = _decode_workspace(dev, n, heads, kvh, hd, max_pages, window, n_sink)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device) if ws_bytes else None
    st = L.load().sfk_attn_decode_window(
        _ROW_TYPES[q.dtype], qp, qs, kvt, k_pages.data_ptr(), v_pages.data_ptr(), k_pages.shape[0],
        _int32(page_table, "page_table", (n, max_pages), dev), max_pages, _int32(positions, "positions", (n,), dev), n,
        heads, kvh, hd, scale, window, n_sink, op, None if ws is None else ws.data_ptr(), ws_bytes,
        None if status is None else _status(status, dev), _stream_of(dev))
    if st:
        L.check(st)
    return out


def attn_prefill_window(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                        q_start: torch.Tensor, kv_len: torch.Tensor, *, window: int = 0, n_sink: int = 0,
                        scale: float = 0.0, out: torch.Tensor | None = None,
                        status: torch.Tensor | None = None) -> torch.Tensor:
    """sfk_attn_prefill_window: rows q_start[s] .. q_start[s+1]-1 of q
    [tokens][Hq][hd] are the newest of the kv_len[s] tokens of sequence s in
    the cache; each attends over the keys it sees (attn_decode_window).
    Returns [tokens][Hq * hd] (`out`, apart from q); rows of no sequence are
    not written."""
    dev = _cuda_device(q, "q")
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return attn_prefill_window(q, k_pages, v_pages, page_table, q_start, kv_len, window=window, n_sink=n_sink,
                                       scale=scale, out=out, status=status)
    kvt, kvh, hd = _pools(k_pages, v_pages, page_table, dev)
    heads, qp, qs, out, op = _attn_rows(q, k_pages, kvh, hd, window, n_sink, out, dev)
    n, max_pages = page_table.shape
    st = L.load().sfk_attn_prefill_window(
        _ROW_TYPES[q.dtype], qp, qs, q.shape[0], kvt, k_pages.data_ptr(), v_pages.data_ptr(), k_pages.shape[0],
        _int32(page_table, "page_table", (n, max_pages), dev), max_pages, _int32(q_start, "q_start", (n + 1,), dev),
        _int32(kv_len, "kv_len", (n,), dev), n, heads, kvh, hd, scale, window, n_sink, op,
        None if status is None else _status(status, dev), _stream_of(dev))
    if st:
        L.check(st)
    return out
