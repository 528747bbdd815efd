"""GPU tests of the paged-cache operators against the formulas in 64 bits.

Tolerances, derived from the arithmetic:
  append     an f32 computation of a few operations rounded once: half a step of
             the output type, plus 2^-20 of the pair's magnitude (angle within
             pi 2^-24 of the exact one, sine and cosine to 2 ulp, the norm's sum
             of at most 16 terms a lane and 5 shuffles, a square root and a
             division).
  attention  per row, with A the largest sum_i |q_i k_i| * scale and W the
             weighted mean of |v|: a score is off by at most (hd + 6) 2^-24 A (hd
             f32 additions; rows split in two 16-bit terms add 2^-22), times
             ln 2 and the exponential's 2 ulp; numerator and denominator both
             carry it, and n f32 additions each: 4 (hd + 6) 2^-24 A + (n + 16)
             2^-23, times the row's largest |v|.  A 16-bit output adds half a
             step of itself; prompts with a 16-bit cache also round the weights
             to that type, half a step of W, and take some of the exponentials
             from a polynomial within 7.5e-5 (bf16) or 2.7e-6 (f16), which the
             numerator and the denominator both carry: twice that of W.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
PG = 16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def half_step(t):
    return torch.finfo(t).eps / 2


class Cache:
    """A pool whose pages are handed out in a permuted order; whatever no sequence holds is NaN, the
    table entries of pages that are not held are far outside the pool."""

    def __init__(self, lens, kvh, hd, dtype, seed, extra_pages=2, poison=True):
        g = gen(seed)
        self.lens, self.kvh, self.hd = lens, kvh, hd
        used = [(n + PG - 1) // PG for n in lens]
        n_pages = sum(used) + extra_pages
        ids = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
        fill = math.nan if poison else 0.0
        self.k = torch.full((n_pages, kvh, PG, hd), fill, device="cuda", dtype=dtype)
        self.v = torch.full((n_pages, kvh, PG, hd), fill, device="cuda", dtype=dtype)
        self.table = torch.full((len(lens), max(used + [1])), 1 << 30, dtype=torch.int32, device="cuda")
        self.table[:, 1::2] = -5
        self.keys, self.values = [], []
        at = 0
        for s, n in enumerate(lens):
            self.table[s, :used[s]] = ids[at:at + used[s]]
            at += used[s]
            k = torch.randn((n, kvh, hd), generator=g, device="cuda").to(dtype)
            v = torch.randn((n, kvh, hd), generator=g, device="cuda").to(dtype)
            j = torch.arange(n, device="cuda")
            self.k[self.table[s, j // PG].long(), :, j % PG] = k
            self.v[self.table[s, j // PG].long(), :, j % PG] = v
            self.keys.append(k)
            self.values.append(v)

    def hide(self, s, window, n_sink, p_first):
        """The pages that positions >= p_first of sequence s do not see leave the table (freed pages)."""
        for page in range((p_first - window + 1) // PG if window else 0):
            if page * PG >= n_sink:
                self.table[s, page] = -7


def reference(q, k, v, pos, window, n_sink, scale=None):
    """(out, tolerance without the output's own rounding, weighted mean of |v|) in 64 bits; q [n][Hq][hd]."""
    n, hq, hd = q.shape
    group = hq // k.shape[1]
    q64 = q.double()
    k64 = k.double().repeat_interleave(group, 1)
    v64 = v.double().repeat_interleave(group, 1)
    scale = hd ** -0.5 if scale is None else scale
    s = torch.einsum("nhd,jhd->nhj", q64, k64) * scale
    p = torch.as_tensor(pos, device=q.device)[:, None]
    j = torch.arange(k.shape[0], device=q.device)[None]
    seen = j <= p
    if window:
        seen &= (j > p - window) | (j < n_sink)
    s = s.masked_fill(~seen[:, None], -math.inf)
    w = torch.softmax(s, -1).nan_to_num(0.0) * seen[:, None]
    out = torch.einsum("nhj,jhd->nhd", w, v64)
    absv = torch.einsum("nhj,jhd->nhd", w, v64.abs())
    a = (torch.einsum("nhd,jhd->nhj", q64.abs(), k64.abs()) * scale).masked_fill(~seen[:, None], 0).amax(-1, keepdim=True)
    vmax = torch.where(seen[:, None, :, None], v64.abs().permute(1, 0, 2)[None], 0.0).amax((2, 3))[..., None]
    tol = (4 * (hd + 6) * 2.0 ** -24 * a + (k.shape[0] + 16) * 2.0 ** -23) * vmax
    return out, tol, absv


def weight_tol(kv, absv):
    """What a prompt's weights in a 16-bit type cost (see above)."""
    return (half_step(kv) + 2 * (7.5e-5 if kv == BF16 else 2.7e-6)) * absv


def check(got, want, tol):
    assert torch.isfinite(got).all()
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((got.double() - want).abs() / tol).max()))


# ---- append ---------------------------------------------------------------------------------------
def append_reference(x, weight, eps, where, freqs, neox):
    """x [n][h][hd], where [n][pairs]: (normed and rotated, magnitude of each element's pair)."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    r = 0 if freqs is None else 2 * freqs.numel()
    mag, y = x.abs(), x.clone()
    if r:
        ang = (where.double() * freqs.double())[:, None]
        if neox:
            ia, ib = torch.arange(r // 2), torch.arange(r // 2) + r // 2
        else:
            ia, ib = torch.arange(0, r, 2), torch.arange(1, r, 2)
        a, b = x[..., ia], x[..., ib]
        y[..., ia], y[..., ib] = a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()
        mag = mag.clone()
        mag[..., ia] = mag[..., ib] = a.abs() + b.abs()
    return y, mag


def append_tol(want, mag, dtype):
    return half_step(dtype) * want.abs() + 2.0 ** -20 * mag + (2.0 ** -25 if dtype == F16 else 0)


@pytest.mark.parametrize("io,kv", [(F32, F16), (F32, F32), (F32, BF16), (F16, F16), (BF16, BF16), (BF16, F32), (F16, BF16)])
@pytest.mark.parametrize("hd,hq,hkv,neox,n_rot,norm,axes", [
    (128, 32, 8, False, 128, False, 1), (128, 5, 1, True, 128, True, 3), (64, 8, 8, True, 32, True, 1),
    (32, 8, 4, False, 8, False, 2), (96, 3, 3, True, 96, False, 1), (256, 4, 2, True, 256, True, 1),
    (8, 2, 1, False, 8, True, 1), (80, 6, 2, True, 32, True, 1), (64, 1, 1, False, 0, False, 1),
])
@pytest.mark.parametrize("layout", ["packed", "odd"])
def test_append(cuda, io, kv, hd, hq, hkv, neox, n_rot, norm, axes, layout):
    from strataflow_b200 import ops
    for n_seq, n_tok in ((1, 1), (3, 50), (2, 333)):
        g = gen(n_tok + hd)
        lens = [n_tok // n_seq + (1 if i < n_tok % n_seq else 0) for i in range(n_seq)]
        past = [0 if i == 1 else 100000 + 7 * i for i in range(n_seq)]
        max_pages = max(p + n for p, n in zip(past, lens)) // PG + 1
        seq = torch.tensor([s for s, n in enumerate(lens) for _ in range(n)], dtype=torch.int32, device="cuda")
        pos = torch.tensor([past[s] + i for s, n in enumerate(lens) for i in range(n)], dtype=torch.int32, device="cuda")
        need = sorted({(int(s), int(p) // PG) for s, p in zip(seq.tolist(), pos.tolist())})
        table = torch.full((n_seq, max_pages), -1, dtype=torch.int32, device="cuda")
        ids = torch.randperm(len(need) + 2, generator=g, device="cuda").to(torch.int32)
        table[[s for s, _ in need], [p for _, p in need]] = ids[:len(need)]
        shape = (len(need) + 2, hkv, PG, hd)
        kp, vp = (torch.randn(shape, generator=g, device="cuda").to(kv) for _ in range(2))
        k0, v0 = kp.clone(), vp.clone()
        width = (hq + 2 * hkv) * hd
        if layout == "packed":
            x = torch.randn((n_tok, width), generator=g, device="cuda").to(io)
        else:  # rows that start off any 16-byte boundary
            x = torch.randn((n_tok, width + 3), generator=g, device="cuda").to(io)[:, 1:1 + width]
        x = x.unflatten(1, (hq + 2 * hkv, hd))
        q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
        qw = 1 + 0.2 * torch.randn(hd, generator=g, device="cuda") if norm else None
        kw = 1 + 0.2 * torch.randn(hd, generator=g, device="cuda") if norm else None
        freqs = ops.rope_freqs(n_rot) if n_rot else None
        kwargs = {}
        where = pos[:, None].expand(-1, n_rot // 2)
        if axes > 1:
            kwargs["rope_pos"] = torch.randint(0, 5000, (axes, n_tok), generator=g, device="cuda", dtype=torch.int32)
            kwargs["axes"] = bytes(i % axes for i in range(n_rot // 2))
            where = kwargs["rope_pos"][torch.arange(n_rot // 2) % axes].t()
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = ops.qk_norm_rope_append(q, k, v, kp, vp, table, pos, seq=seq, freqs=freqs, neox=neox, q_norm=qw, k_norm=kw,
                                      eps=1e-5, status=status, **kwargs)
        ops.check_status(status)
        want, mag = append_reference(q, qw, 1e-5, where, freqs, neox)
        check(out, want, append_tol(want, mag, io))
        page = table[seq.long(), (pos // PG).long()].long()
        slot = (pos % PG).long()
        want, mag = append_reference(k, kw, 1e-5, where, freqs, neox)
        check(kp[page, :, slot], want, append_tol(want, mag, kv))
        assert torch.equal(vp[page, :, slot], v.to(kv))
        k0[page, :, slot], v0[page, :, slot] = kp[page, :, slot], vp[page, :, slot]
        assert torch.equal(kp, k0) and torch.equal(vp, v0)  # nothing else was written


def test_append_in_place_and_padding(cuda):
    """q_out = q; rows of a negative position are left as they were, in q and in the cache."""
    from strataflow_b200 import ops
    g = gen(5)
    x = torch.randn((6, 4, 64), generator=g, device="cuda")
    kv = torch.randn((6, 2, 64), generator=g, device="cuda")
    kp, vp = torch.zeros(4, 2, PG, 64, device="cuda"), torch.zeros(4, 2, PG, 64, device="cuda")
    table = torch.tensor([[0], [1], [2], [3], [0], [1]], dtype=torch.int32, device="cuda")
    pos = torch.tensor([3, -1, 15, 0, -1, -9], dtype=torch.int32, device="cuda")
    f = ops.rope_freqs(64)
    y = x.clone()
    apart = ops.qk_norm_rope_append(x, kv, kv, kp.clone(), vp.clone(), table, pos, freqs=f, neox=True,
                                    out=torch.full_like(x, 7.0))
    got = ops.qk_norm_rope_append(y, kv, kv, kp, vp, table, pos, freqs=f, neox=True, out=y)
    live = pos >= 0
    assert got is y and torch.equal(y[~live], x[~live]) and torch.equal(y[live], apart[live])
    assert (apart[~live] == 7.0).all()
    assert int((vp != 0).any(-1).any(1).sum()) == 3


@pytest.mark.parametrize("what", ["page", "high page", "position", "sequence"])
def test_append_out_of_range_is_reported_and_not_written(cuda, what):
    from strataflow_b200 import lib as L
    from strataflow_b200 import ops
    x = torch.ones(2, 2, 32, device="cuda")
    kp, vp = torch.zeros(3, 2, PG, 32, device="cuda"), torch.zeros(3, 2, PG, 32, device="cuda")
    table = torch.tensor([[1, 2], [0, {"page": -1, "high page": 3}.get(what, 2)]], dtype=torch.int32, device="cuda")
    pos = torch.tensor([0, 32 if what == "position" else 20], dtype=torch.int32, device="cuda")
    seq = torch.tensor([0, 2 if what == "sequence" else 1], dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.qk_norm_rope_append(x, x, x, kp, vp, table, pos, seq=seq, status=status)
    with pytest.raises(L.SfkError) as e:
        ops.check_status(status)
    assert e.value.status == L.SFK_ERR_RUNTIME
    ops.check_status(status)  # cleared
    assert int((vp != 0).sum()) == 2 * 32 and int((kp != 0).sum()) == 2 * 32  # token 0 alone


# ---- decode ------------------------------------------------------------------------------------------
TYPES = [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)]


def run_decode(lens, hq, hkv, hd, io, kv, window, n_sink, seed=0, scale=0.0, qscale=1.0):
    from strataflow_b200 import ops
    c = Cache(lens, hkv, hd, kv, seed)
    for s, n in enumerate(lens):
        if n:
            c.hide(s, window, n_sink, n - 1)
    q = (qscale * torch.randn((len(lens), hq, hd), generator=gen(seed + 1), device="cuda")).to(io)
    pos = torch.tensor(lens, dtype=torch.int32, device="cuda") - 1
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = ops.attn_decode_window(q, c.k, c.v, c.table, pos, window=window, n_sink=n_sink, scale=scale, status=status)
    ops.check_status(status)
    got = got.view(len(lens), hq, hd)
    for s, n in enumerate(lens):
        if n == 0:
            assert (got[s] == 0).all()
            continue
        want, tol, _ = reference(q[s:s + 1], c.keys[s], c.values[s], [n - 1], window, n_sink, scale or None)
        if io != F32:
            tol = tol + half_step(io) * want.abs()
        check(got[s:s + 1], want, tol)
    return q, c, pos, got


@pytest.mark.parametrize("io,kv", TYPES)
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("window,n_sink", [(0, 0), (1, 0), (16, 1), (37, 20), (200, 4)])
def test_decode(cuda, io, kv, hd, window, n_sink):
    run_decode([1, 15, 16, 17, 0, 33, 257, 1000, 64], 8, 2, hd, io, kv, window, n_sink, seed=hd + window)


@pytest.mark.parametrize("io,kv", [(F32, F32), (F32, F16), (BF16, BF16)])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (5, 5), (14, 2), (16, 1), (17, 1), (40, 1), (71, 1), (64, 8)])
def test_decode_head_layouts(cuda, io, kv, hq, hkv):
    run_decode([100, 7, 513], hq, hkv, 128, io, kv, 0, 0, seed=hq)


@pytest.mark.parametrize("io,kv", [(F32, F16), (BF16, BF16), (F32, F32)])
@pytest.mark.parametrize("lens", [[5000], [20000, 1], [0, 0], [1] * 70, [300] * 33])
def test_decode_batches_and_lengths(cuda, io, kv, lens):
    run_decode(lens, 8, 2, 128, io, kv, 0, 0, seed=len(lens))


@pytest.mark.parametrize("io,kv", [(F32, F16), (BF16, BF16), (F32, F32), (F32, BF16)])
@pytest.mark.parametrize("hd", [64, 256])
def test_decode_long_windows(cuda, io, kv, hd):
    """Windows long enough to be split over many CTAs, a start inside a page, more sinks than a page holds."""
    run_decode([20000, 300, 9001], 4, 1, hd, io, kv, 9000, 40, seed=hd)


def test_decode_with_a_wide_table(cuda):
    """A table for far longer contexts than the sequences have; without a workspace the result is the same."""
    from strataflow_b200 import lib as L
    from strataflow_b200 import ops
    c = Cache([700, 40, 0], 2, 128, BF16, 1)
    table = torch.full((3, 5000), -1, dtype=torch.int32, device="cuda")
    table[:, :c.table.shape[1]] = c.table
    q = torch.randn((3, 8, 128), generator=gen(2), device="cuda").to(BF16)
    pos = torch.tensor([699, 39, -1], dtype=torch.int32, device="cuda")
    got = ops.attn_decode_window(q, c.k, c.v, table, pos)
    bare = torch.empty_like(got)
    L.check(L.load().sfk_attn_decode_window(L.TYPE_BF16, q.data_ptr(), 8 * 128, L.KV_BF16, c.k.data_ptr(), c.v.data_ptr(),
                                            c.k.shape[0], table.data_ptr(), 5000, pos.data_ptr(), 3, 8, 2, 128, 0.0, 0, 0,
                                            bare.data_ptr(), None, 0, None, torch.cuda.current_stream().cuda_stream))
    for s, n in enumerate((700, 40)):
        want, tol, _ = reference(q[s:s + 1], c.keys[s], c.values[s], [n - 1], 0, 0)
        tol = tol + half_step(BF16) * want.abs()
        check(got[s:s + 1].view_as(want), want, tol)
        check(bare[s:s + 1].view_as(want), want, tol)
    assert (got[2] == 0).all() and (bare[2] == 0).all()


def test_decode_large_scores(cuda):
    """Scores in the hundreds: the running maximum decides; f16 keys and 32-bit queries far from 1."""
    run_decode([700], 8, 2, 128, F32, F16, 0, 0, scale=1.0, qscale=30.0)
    run_decode([700], 8, 2, 128, F32, F16, 0, 0, scale=1e-9, qscale=1e6)
    run_decode([700], 8, 2, 128, F32, F16, 0, 0, scale=1e6, qscale=1e-7)


def test_decode_strided_queries_streams_and_repeats(cuda):
    """Queries inside a packed row; another stream than the tensors' own; the same bits each time."""
    from strataflow_b200 import ops
    q, c, pos, got = run_decode([1000, 37, 512], 8, 2, 128, BF16, BF16, 300, 4)
    packed = torch.randn((3, 12, 128), generator=gen(9), device="cuda").to(BF16)
    packed[:, :8] = q
    again = ops.attn_decode_window(packed[:, :8], c.k, c.v, c.table, pos, window=300, n_sink=4)
    assert torch.equal(again.view_as(got), got)
    odd = torch.zeros((3, 8 * 128 + 1), device="cuda", dtype=BF16)[:, 1:].unflatten(1, (8, 128))
    odd.copy_(q)
    assert torch.equal(ops.attn_decode_window(odd, c.k, c.v, c.table, pos, window=300, n_sink=4).view_as(got), got)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        other = ops.attn_decode_window(q, c.k, c.v, c.table, pos, window=300, n_sink=4)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(other.view_as(got), got)


@pytest.mark.parametrize("io,kv,hd", [(F32, F32, 64), (F32, F16, 128), (BF16, BF16, 128), (F16, F16, 256),
                                      (F32, F32, 128), (F32, BF16, 256)])
def test_decode_bad_pages_and_positions(cuda, io, kv, hd):
    from strataflow_b200 import lib as L
    from strataflow_b200 import ops
    c = Cache([100, 100, 100], 2, hd, kv, 3)
    q = torch.randn((3, 4, hd), generator=gen(4), device="cuda").to(io)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    good = ops.attn_decode_window(q, c.k, c.v, c.table, torch.tensor([99, 50, 99], dtype=torch.int32, device="cuda"),
                                  status=status)
    ops.check_status(status)
    pos = torch.tensor([99, 50, c.table.shape[1] * PG], dtype=torch.int32, device="cuda")
    got = ops.attn_decode_window(q, c.k, c.v, c.table, pos, status=status)
    with pytest.raises(L.SfkError):
        ops.check_status(status)
    assert torch.equal(got[:2], good[:2]) and (got[2] == 0).all()
    for bad in (-1, c.k.shape[0], 1 << 30):
        table = c.table.clone()
        table[0, 3] = bad
        got = ops.attn_decode_window(q, c.k, c.v, table, pos.clamp(max=99), status=status)
        with pytest.raises(L.SfkError):
            ops.check_status(status)
        assert torch.equal(got[1], good[1])


@pytest.mark.parametrize("io,kv", TYPES)
@pytest.mark.parametrize("hd", [32, 128, 256])
@pytest.mark.parametrize("n", [40, 700, 20000])
def test_decode_infinite_and_nan_keys_and_values(cuda, io, kv, hd, n):
    """Of keys that are seen: what the formula gives, in the heads of the key's kv head alone."""
    from strataflow_b200 import ops
    q, c, pos, _ = run_decode([n], 8, 2, hd, io, kv, 0, 0)
    j, x0 = n - 7, q[0, :4, 0].float()
    at = (c.table[0, j // PG], 0, j % PG)
    k, v = c.k[at].clone(), c.v[at].clone()

    def run():
        return ops.attn_decode_window(q, c.k, c.v, c.table, pos).view(8, hd).float()

    good = run()
    c.v[at][3] = math.inf
    got = run()
    assert (got[:4, 3] == math.inf).all() and torch.equal(got[4:], good[4:])
    others = [d for d in range(hd) if d != 3]
    assert torch.equal(got[:, others], good[:, others])
    c.v[at] = v
    c.k[at] = 0
    for x in (math.inf, -math.inf, math.nan):
        c.k[at][0] = x
        got = run()
        s = x * x0
        assert got[:4][s != -math.inf].isnan().all() and torch.equal(got[4:], good[4:])
        low = s == -math.inf  # the key's weight is 0: as if it were not there
        assert got[:4][low].isfinite().all()
    c.k[at] = k


# ---- prefill -------------------------------------------------------------------------------------------
def run_prefill(n_qs, pasts, hq, hkv, hd, io, kv, window, n_sink, seed=0, scale=0.0, qscale=1.0, gap=3):
    """Ragged prompts with `gap` rows of no sequence before the first and behind the last."""
    from strataflow_b200 import ops
    lens = [n + p for n, p in zip(n_qs, pasts)]
    c = Cache(lens, hkv, hd, kv, seed)
    for s in range(len(lens)):
        c.hide(s, window, n_sink, pasts[s])
    total = sum(n_qs)
    q = (qscale * torch.randn((total + 2 * gap, hq, hd), generator=gen(seed + 1), device="cuda")).to(io)
    start = torch.tensor([gap + sum(n_qs[:i]) for i in range(len(n_qs) + 1)], dtype=torch.int32, device="cuda")
    kv_len = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = torch.full((total + 2 * gap, hq * hd), 77.0, dtype=io, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = ops.attn_prefill_window(q, c.k, c.v, c.table, start, kv_len, window=window, n_sink=n_sink, scale=scale, out=out,
                                  status=status)
    ops.check_status(status)
    assert (out[:gap] == 77.0).all() and (out[gap + total:] == 77.0).all()
    got = got.view(-1, hq, hd)
    at = gap
    for s, n in enumerate(n_qs):
        if n:
            want, tol, absv = reference(q[at:at + n], c.keys[s], c.values[s], range(pasts[s], lens[s]), window, n_sink,
                                        scale or None)
            if io != F32:
                tol = tol + half_step(io) * want.abs() + weight_tol(kv, absv)
            check(got[at:at + n], want, tol)
        at += n
    return q, c, start, kv_len, out


@pytest.mark.parametrize("io,kv", TYPES)
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("window,n_sink", [(0, 0), (1, 0), (16, 1), (37, 20), (150, 4)])
def test_prefill(cuda, io, kv, hd, window, n_sink):
    run_prefill([1, 70, 0, 129, 33, 300], [0, 0, 5, 300, 17, 111], 8, 2, hd, io, kv, window, n_sink, seed=hd + window)


@pytest.mark.parametrize("io,kv", [(F32, F16), (BF16, BF16), (F32, F32)])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (5, 5), (14, 2), (16, 1), (40, 1), (130, 1), (64, 8)])
def test_prefill_head_layouts(cuda, io, kv, hq, hkv):
    run_prefill([50, 131, 1], [20, 0, 400], hq, hkv, 128, io, kv, 0, 0, seed=hq)


@pytest.mark.parametrize("io,kv,hd", [(F16, F16, 64), (BF16, BF16, 128), (F32, F16, 128)])
@pytest.mark.parametrize("n_qs,pasts,window,n_sink", [
    ([1200], [0], 0, 0), ([1200], [0], 256, 4), ([700], [1500], 500, 200), ([5], [3000], 0, 0), ([5], [3000], 100, 16), ([70], [2500], 0, 0), ([33, 1], [1000, 4000], 900, 3),
    ([1] * 40, list(range(40)), 0, 0), ([600, 600], [0, 640], 64, 0), ([256], [0], 0, 0), ([257], [255], 1000, 1)])
def test_prefill_lengths(cuda, io, kv, hd, n_qs, pasts, window, n_sink):
    run_prefill(n_qs, pasts, 8, 2, hd, io, kv, window, n_sink, seed=len(n_qs) + window)


@pytest.mark.parametrize("io,kv,hd", [(BF16, BF16, 128), (F32, F16, 64), (F32, F32, 32)])
def test_prefill_many_sequences(cuda, io, kv, hd):
    """More sequences than one look at the batch takes, most of them with one token or none."""
    n_qs = [(i * 7) % 5 if i % 3 else 1 for i in range(300)]
    run_prefill(n_qs, [(i * 37) % 90 for i in range(300)], 4, 2, hd, io, kv, 20, 1)


@pytest.mark.parametrize("io,kv", [(F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("n_qs,pasts,window,n_sink", [
    ([1200], [0], 0, 0), ([700], [1500], 500, 200), ([5], [3000], 0, 0), ([33, 1, 0, 129], [1000, 4000, 3, 79], 900, 3)])
def test_prefill_wide_heads(cuda, io, kv, n_qs, pasts, window, n_sink):
    """Heads of 256 of 16-bit rows, one row tile to a CTA: several tiles, split keys, ragged ends."""
    run_prefill(n_qs, pasts, 8, 2, 256, io, kv, window, n_sink, seed=len(n_qs) + window)
    run_prefill(n_qs, pasts, 3, 3, 256, io, kv, window, n_sink, seed=7)


def test_prefill_long_context_keeps_32_bits(cuda):
    """32-bit rows at 30000 keys: within the bound, and free of the drift that one accumulator over all keys shows."""
    from strataflow_b200 import ops
    for n_q, past in ((300, 30000), (3, 30000)):
        c = Cache([n_q + past], 1, 128, F16, 5)
        q = torch.randn((n_q, 4, 128), generator=gen(6), device="cuda")
        start = torch.tensor([0, n_q], dtype=torch.int32, device="cuda")
        got = ops.attn_prefill_window(q, c.k, c.v, c.table, start, start[1:] + past).view_as(q)
        want = torch.cat([reference(q[i:i + 30], c.keys[0], c.values[0], range(past + i, past + min(i + 30, n_q)), 0, 0)[0]
                          for i in range(0, n_q, 30)])
        # The accumulator truncates: a loss of 2^-24 of the sum on average each time.  A tile is 12 of them: a gain
        # 12 * 2^-24 = 7.2e-7 below 1 at most, where one accumulator over all keys (3800 of them) would lose 2e-4 at
        # most and lost 7.6e-6 over 440.  Beside it: 8 truncations of a score (rms 1.5: 8 * 2^-24 * 1.5 = 7.2e-7), the
        # exponential and the two terms of P (2^-22 each): 1.1e-6 as a root of squares, below 2^-19.
        assert abs(float((got * want).sum() / (want * want).sum()) - 1) < 2.0 ** -20
        assert float((got - want).norm() / want.norm()) < 2.0 ** -19


def test_prefill_large_scores(cuda):
    for io, kv in ((F32, F16), (F16, F16), (BF16, BF16)):
        run_prefill([300], [100], 8, 2, 128, io, kv, 0, 0, scale=1.0, qscale=8.0)
    run_prefill([200], [0], 8, 2, 128, F32, F16, 0, 0, scale=1e-9, qscale=1e6)
    run_prefill([200], [0], 8, 2, 128, F32, F16, 0, 0, scale=1e6, qscale=1e-7)


@pytest.mark.parametrize("n_q,past", [(200, 60), (130, 700)])
@pytest.mark.parametrize("io,kv,hd", [(F32, F32, 64), (F32, F16, 128), (F16, F16, 64), (BF16, BF16, 128), (F16, F16, 256),
                                      (F32, F32, 128), (F32, BF16, 256)])
def test_prefill_values_of_unseen_keys_do_not_leak(cuda, io, kv, hd, n_q, past):
    """A key whose value is infinite or NaN touches the rows that see it and no other, in the same tile too."""
    from strataflow_b200 import ops
    window, n_sink = n_q * 9 // 20, 2
    q, c, start, kv_len, _ = run_prefill([n_q], [past], 8, 2, hd, io, kv, window, n_sink, gap=0)
    bad = (past + n_q * 9 // 20, past + n_q // 5)
    for j, x in zip(bad, (math.inf, math.nan)):
        c.v[c.table[0, j // PG], :, j % PG] = x
    got = ops.attn_prefill_window(q, c.k, c.v, c.table, start, kv_len, window=window, n_sink=n_sink)
    p = past + torch.arange(n_q, device="cuda")
    touched = torch.zeros_like(p, dtype=torch.bool)
    for j in bad:
        touched |= (p >= j) & (p < j + window)
    assert not torch.isfinite(got[touched]).any()
    want, tol, absv = reference(q, c.keys[0], c.values[0], range(past, past + n_q), window, n_sink)
    if io != F32:
        tol = tol + half_step(io) * want.abs() + weight_tol(kv, absv)
    check(got.view_as(want)[~touched], want[~touched], tol[~touched])


@pytest.mark.parametrize("n_q,past", [(200, 60), (130, 700)])
@pytest.mark.parametrize("io,kv,hd", [(F32, F32, 64), (F32, BF16, 128), (F32, F16, 128), (F16, F16, 64), (BF16, BF16, 32),
                                      (BF16, BF16, 64), (BF16, BF16, 128), (BF16, BF16, 256)])
def test_prefill_largest_values_of_unseen_keys_do_not_leak(cuda, io, kv, hd, n_q, past):
    """The largest finite values of the cache's type at keys that some rows of a tile see and others do not: a weight
    of 2^-126 instead of 0 would already add 4."""
    from strataflow_b200 import ops
    window, n_sink = n_q * 9 // 20, 2
    q, c, start, kv_len, _ = run_prefill([n_q], [past], 8, 2, hd, io, kv, window, n_sink, gap=0)
    first = past + n_q * 9 // 20
    bad = range(first, first + 12)
    for j in bad:
        c.v[c.table[0, j // PG], :, j % PG] = torch.finfo(kv).max
    got = ops.attn_prefill_window(q, c.k, c.v, c.table, start, kv_len, window=window, n_sink=n_sink)
    p = past + torch.arange(n_q, device="cuda")
    touched = (p >= bad[0]) & (p < bad[-1] + window)
    assert touched.any() and not touched.all()
    want, tol, absv = reference(q, c.keys[0], c.values[0], range(past, past + n_q), window, n_sink)
    if io != F32:
        tol = tol + half_step(io) * want.abs() + weight_tol(kv, absv)
    check(got.view_as(want)[~touched], want[~touched], tol[~touched])


@pytest.mark.parametrize("n_q,past", [(200, 60), (130, 700)])
@pytest.mark.parametrize("io,kv,hd", [(F32, F32, 64), (F32, BF16, 128), (F32, F16, 128), (F16, F16, 64), (BF16, BF16, 64),
                                      (BF16, BF16, 128), (BF16, BF16, 256)])
@pytest.mark.parametrize("at", [0, 1, 2, 3, 5, 7, 8, 14])
def test_prefill_a_bad_key_shows_in_the_rows_that_see_it(cuda, io, kv, hd, n_q, past, at):
    """A NaN in a key makes every row NaN that sees it, at any place of a tile, and no other row."""
    from strataflow_b200 import ops
    window = n_q * 9 // 20
    q, c, start, kv_len, _ = run_prefill([n_q], [past], 8, 2, hd, io, kv, window, 0, gap=0)
    j = (past + n_q * 9 // 20) // PG * PG + at
    want, tol, absv = reference(q, c.keys[0], c.values[0], range(past, past + n_q), window, 0)
    if io != F32:
        tol = tol + half_step(io) * want.abs() + weight_tol(kv, absv)
    p = past + torch.arange(n_q, device="cuda")
    sees = (p >= j) & (p < j + window)
    for x in (math.nan, math.inf):
        c.k[c.table[0, j // PG], :, j % PG] = 0
        c.k[c.table[0, j // PG], :, j % PG, 0] = x
        got = ops.attn_prefill_window(q, c.k, c.v, c.table, start, kv_len, window=window).view_as(want)
        # inf times q's first number: +inf (a NaN row), -inf (the key has weight 0) or, for a zero, NaN
        nan = sees[:, None] & (torch.full_like(q[:, :, 0], x) * q[:, :, 0] != -math.inf)
        assert got[nan].isnan().all() and not got[~nan].isnan().any()
        check(got[~sees], want[~sees], tol[~sees])


def test_prefill_tokens_before_the_first_position(cuda):
    """kv_len below the tokens: the first ones have negative positions and give zeros."""
    from strataflow_b200 import ops
    for io, kv, hd in ((F32, F32, 32), (BF16, BF16, 128), (F32, F16, 64)):
        c = Cache([40], 2, hd, kv, 1)
        q = torch.randn((50, 4, hd), generator=gen(2), device="cuda").to(io)
        start = torch.tensor([0, 50], dtype=torch.int32, device="cuda")
        for n in (40, 0):
            got = ops.attn_prefill_window(q, c.k, c.v, c.table, start, torch.tensor([n], dtype=torch.int32, device="cuda"))
            assert (got[:50 - n] == 0).all()
            if n:
                want, tol, absv = reference(q[10:], c.keys[0], c.values[0], range(40), 0, 0)
                check(got[10:].view(40, 4, hd), want,
                      tol + (half_step(io) * want.abs() + weight_tol(kv, absv) if io != F32 else 0))


@pytest.mark.parametrize("io,kv,hd", [(F32, F32, 64), (F32, F16, 128), (BF16, BF16, 128)])
def test_prefill_bad_pages_and_lengths(cuda, io, kv, hd):
    from strataflow_b200 import lib as L
    from strataflow_b200 import ops
    q, c, start, kv_len, good = run_prefill([50, 60, 70], [10, 200, 0], 4, 2, hd, io, kv, 0, 0, gap=0)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for bad in (-1, c.k.shape[0], 1 << 30):
        table = c.table.clone()
        table[1, 2] = bad
        got = ops.attn_prefill_window(q, c.k, c.v, table, start, kv_len, status=status)
        with pytest.raises(L.SfkError):
            ops.check_status(status)
        assert torch.equal(got[:50], good[:50]) and torch.equal(got[110:], good[110:])
    long = kv_len.clone()
    long[1] = c.table.shape[1] * PG + 1
    backwards = start.clone()
    backwards[2] = 1000
    for s, n in ((start, long), (backwards, kv_len)):
        out = torch.full_like(good, 5.0)
        ops.attn_prefill_window(q, c.k, c.v, c.table, s, n, out=out, status=status)
        with pytest.raises(L.SfkError):
            ops.check_status(status)
        assert torch.equal(out[:50], good[:50])


# ---- the cache beyond 32-bit offsets, graphs, the three together -----------------------------------------
def test_offsets_beyond_32_bits(cuda):
    """The last pages of a pool of more than 2^32 bytes and 2^31 elements."""
    from strataflow_b200 import ops
    hkv, hd = 8, 128
    n_pages = (1 << 31) // (hkv * PG * hd) + 9
    kp = torch.empty((n_pages, hkv, PG, hd), dtype=BF16, device="cuda")
    vp = torch.empty_like(kp)
    n = 70
    table = torch.arange(n_pages - 1, n_pages - 6, -1, dtype=torch.int32, device="cuda")[None].contiguous()
    g = gen(1)
    x = torch.randn((n, 16 + 2 * hkv, hd), generator=g, device="cuda").to(BF16)
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    q = ops.qk_norm_rope_append(x[:, :16], x[:, 16:24], x[:, 24:], kp, vp, table, pos, seq=torch.zeros_like(pos),
                                freqs=ops.rope_freqs(hd))
    k = kp[table[0].long()].transpose(1, 2).reshape(-1, hkv, hd)[:n]
    assert torch.equal(vp[table[0].long()].transpose(1, 2).reshape(-1, hkv, hd)[:n], x[:, 24:])
    want, tol, absv = reference(q, k, x[:, 24:], range(n), 0, 0)
    tol = tol + half_step(BF16) * want.abs() + weight_tol(BF16, absv)
    got = ops.attn_prefill_window(q, kp, vp, table, torch.tensor([0, n], dtype=torch.int32, device="cuda"),
                                  torch.tensor([n], dtype=torch.int32, device="cuda"))
    check(got.view_as(want), want, tol)
    got = ops.attn_decode_window(q[-1:], kp, vp, table, pos[-1:])
    check(got.view(1, 16, hd), want[-1:], tol[-1:])


@pytest.mark.parametrize("io,kv,hd,window,n_sink", [(BF16, BF16, 128, 0, 0), (F32, F16, 128, 48, 3), (F16, F16, 64, 100, 16),
                                                     (F32, F32, 32, 20, 1)])
def test_a_run_of_the_three(cuda, io, kv, hd, window, n_sink):
    """Prompts in two chunks, then single tokens in a captured graph, against dense attention in 64 bits over
    what the appends should have stored (rounded to the cache's type)."""
    from strataflow_b200 import ops
    hq, hkv, n_seq, steps = 8, 2, 3, 20
    n1, n2 = [40, 7, 150], [33, 90, 1]
    total = [a + b + steps for a, b in zip(n1, n2)]
    max_pages = max(total) // PG + 1
    g = gen(11)
    ids = torch.randperm(n_seq * max_pages, generator=g, device="cuda").to(torch.int32)
    table = ids.view(n_seq, max_pages)
    kp = torch.full((n_seq * max_pages, hkv, PG, hd), math.nan, device="cuda", dtype=kv)
    vp = torch.full_like(kp, math.nan)
    x = [torch.randn((t, hq + 2 * hkv, hd), generator=g, device="cuda").to(io) for t in total]
    f = ops.rope_freqs(hd)
    qw, kw = 1 + 0.1 * torch.randn((2, hd), generator=g, device="cuda").unbind(0)[0], torch.ones(hd, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def append(rows, seq, pos, out=None):
        return ops.qk_norm_rope_append(rows[:, :hq], rows[:, hq:hq + hkv], rows[:, hq + hkv:], kp, vp, table, pos, seq=seq,
                                       freqs=f, neox=True, q_norm=qw, k_norm=kw, out=out, status=status)

    got = [[] for _ in range(n_seq)]
    queries = [[] for _ in range(n_seq)]
    done = [0] * n_seq
    for chunk in (n1, n2):
        rows = torch.cat([x[s][done[s]:done[s] + n] for s, n in enumerate(chunk)])
        seq = torch.tensor([s for s, n in enumerate(chunk) for _ in range(n)], dtype=torch.int32, device="cuda")
        pos = torch.tensor([done[s] + i for s, n in enumerate(chunk) for i in range(n)], dtype=torch.int32, device="cuda")
        q = append(rows, seq, pos)
        done = [d + n for d, n in zip(done, chunk)]
        start = torch.tensor([sum(chunk[:i]) for i in range(n_seq + 1)], dtype=torch.int32, device="cuda")
        y = ops.attn_prefill_window(q, kp, vp, table, start, torch.tensor(done, dtype=torch.int32, device="cuda"),
                                    window=window, n_sink=n_sink, status=status)
        for s in range(n_seq):
            got[s].append(y[start[s]:start[s + 1]])
            queries[s].append(q[start[s]:start[s + 1]])
    n_prompt = list(done)
    rows = torch.empty((n_seq, hq + 2 * hkv, hd), dtype=io, device="cuda")
    pos = torch.zeros(n_seq, dtype=torch.int32, device="cuda")
    pos.fill_(-1)
    append(rows, None, pos)  # warm: a batch of padding
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = append(rows, None, pos)
        y = ops.attn_decode_window(q, kp, vp, table, pos, window=window, n_sink=n_sink, status=status)
    for i in range(steps):
        rows.copy_(torch.stack([x[s][done[s] + i] for s in range(n_seq)]))
        pos.copy_(torch.tensor([done[s] + i for s in range(n_seq)], dtype=torch.int32))
        graph.replay()
        for s in range(n_seq):
            got[s].append(y[s:s + 1].clone())
            queries[s].append(q[s:s + 1].clone())
    ops.check_status(status)
    for s in range(n_seq):
        where = torch.arange(total[s], device="cuda")[:, None].expand(-1, hd // 2)
        k, mag = append_reference(x[s][:, hq:hq + hkv], kw, 1e-6, where, f, True)
        j = torch.arange(total[s], device="cuda")
        stored = kp[table[s, j // PG].long(), :, j % PG]
        check(stored, k, append_tol(k, mag, kv))
        q = torch.cat(queries[s])
        want_q, mag = append_reference(x[s][:, :hq], qw, 1e-6, where, f, True)
        check(q, want_q, append_tol(want_q, mag, io))
        want, tol, absv = reference(q, stored, x[s][:, hq + hkv:].to(kv), range(total[s]), window, n_sink)
        if io != F32:
            tol = tol + half_step(io) * want.abs()
            tol[:n_prompt[s]] += weight_tol(kv, absv[:n_prompt[s]])
        check(torch.cat(got[s]).view_as(want), want, tol)


def test_two_graphs_at_once(cuda):
    """Two captured calls replayed on two streams at the same time share nothing."""
    from strataflow_b200 import ops
    cases = []
    for seed, n in ((1, 4000), (2, 900)):
        c = Cache([n] * 4, 2, 128, BF16, seed)
        q = torch.randn((4, 8, 128), generator=gen(seed), device="cuda").to(BF16)
        pos = torch.full((4,), n - 1, dtype=torch.int32, device="cuda")
        start = torch.arange(5, dtype=torch.int32, device="cuda")
        args = (q, c, pos, start, pos + 1)
        want = (ops.attn_decode_window(q, c.k, c.v, c.table, pos),
                ops.attn_prefill_window(q, c.k, c.v, c.table, start, pos + 1))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = (ops.attn_decode_window(q, c.k, c.v, c.table, pos),
                   ops.attn_prefill_window(q, c.k, c.v, c.table, start, args[4]))
        cases.append((graph, got, want, torch.cuda.Stream(), args))
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, _, _, st, _ in cases:
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for _, got, want, _, _ in cases:
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---- refusals that need CUDA tensors ------------------------------------------------------------------------
def test_wrapper_refusals(cuda):
    from strataflow_b200 import lib as L
    from strataflow_b200 import ops
    q = torch.zeros(2, 4, 64, device="cuda", dtype=BF16)
    kv = torch.zeros(2, 2, 64, device="cuda", dtype=BF16)
    pool = torch.zeros(3, 2, PG, 64, device="cuda", dtype=BF16)
    table = torch.zeros(2, 2, device="cuda", dtype=torch.int32)
    pos = torch.zeros(2, device="cuda", dtype=torch.int32)
    start = torch.zeros(3, device="cuda", dtype=torch.int32)
    f = ops.rope_freqs(64)
    dec, pre, app = ops.attn_decode_window, ops.attn_prefill_window, ops.qk_norm_rope_append
    bad = [
        lambda: dec(q.double(), pool, pool, table, pos), lambda: dec(q.half(), pool, pool, table, pos),
        lambda: dec(q[:, :3], pool, pool, table, pos), lambda: dec(q.transpose(0, 1), pool, pool, table, pos),
        lambda: dec(q[..., ::2], pool, pool, table, pos), lambda: dec(q, pool, pool[:2], table, pos),
        lambda: dec(q, pool, pool.half(), table, pos), lambda: dec(q, pool.transpose(0, 1), pool, table, pos),
        lambda: dec(q, pool[:, :, :8], pool[:, :, :8], table, pos), lambda: dec(q, pool, pool, table.long(), pos),
        lambda: dec(q, pool, pool, table[:1], pos), lambda: dec(q, pool, pool, table, pos[:1]),
        lambda: dec(q, pool, pool, table, pos.cpu()), lambda: dec(q, pool, pool, table, pos, window=-1),
        lambda: dec(q, pool, pool, table, pos, window=1 << 32), lambda: dec(q, pool, pool, table, pos, n_sink=1 << 31),
        lambda: dec(q, pool, pool, table, pos, out=torch.zeros_like(q)),
        lambda: dec(q, pool, pool, table, pos, status=start), lambda: dec(q, pool, pool, table.t(), pos),
        lambda: pre(q, pool, pool, table, pos, pos), lambda: pre(q, pool, pool, table, start, start),
        lambda: pre(q[0], pool, pool, table, start, pos), lambda: app(q, kv[:1], kv, pool, pool, table, pos),
        lambda: app(q, kv, kv.float(), pool, pool, table, pos), lambda: app(q, kv, kv, pool, pool, table, pos[:1]),
        lambda: app(q, kv, kv, pool, pool, table, pos, freqs=f.double()),
        lambda: app(q, kv, kv, pool, pool, table, pos, freqs=torch.cat([f, f])),
        lambda: app(q, kv, kv, pool, pool, table, pos, freqs=f, axes=bytes(32)),
        lambda: app(q, kv, kv, pool, pool, table, pos, freqs=f, axes=bytes(3), rope_pos=pos[None]),
        lambda: app(q, kv, kv, pool, pool, table, pos, freqs=f, rope_pos=pos),
        lambda: app(q, kv, kv, pool, pool, table, pos, q_norm=f), lambda: app(q, kv, kv, pool, pool, table[:1], pos),
        lambda: app(q, kv, kv, pool, pool, table, pos, out=torch.zeros_like(kv)),
        lambda: app(q, kv, kv, pool, pool, table, pos, seq=pos.long()),
    ]
    for i, fn in enumerate(bad):
        with pytest.raises(L.SfkError) as e:
            fn()
        assert e.value.status == L.SFK_ERR_INVALID_ARGUMENT, i
    torch.cuda.synchronize()


def test_calls_right_behind_what_they_read_and_before_what_they_wrote(cuda):
    """Each operator directly behind copies, fills, kernels and another stream's work that make its inputs, and in front
    of kernels that change them: eager and captured, many steps without a host wait."""
    from strataflow_b200 import ops
    n, steps, hd = 3, 40, 64
    g = gen(11)
    rows = torch.randn((steps, n, 8 + 2 + 2, hd), generator=g, device="cuda")
    freqs = ops.rope_freqs(hd)
    table = torch.arange(1, 1 + n * 4, dtype=torch.int32, device="cuda").view(n, 4)
    wide = torch.randn((1 << 23,), generator=g, device="cuda")

    def fresh():
        return dict(k=torch.zeros(1 + n * 4, 2, PG, hd, device="cuda", dtype=torch.float16),
                    v=torch.zeros(1 + n * 4, 2, PG, hd, device="cuda", dtype=torch.float16),
                    pos=torch.full((n,), -1, dtype=torch.int32, device="cuda"), x=torch.empty_like(rows[0]),
                    q=torch.empty((n, 8, hd), device="cuda"), o=torch.empty((n, 8 * hd), device="cuda"),
                    p=torch.empty((n, 8 * hd), device="cuda"), start=torch.arange(n + 1, dtype=torch.int32, device="cuda"),
                    len=torch.zeros(n, dtype=torch.int32, device="cuda"), at=torch.zeros(1, dtype=torch.long, device="cuda"),
                    sums=torch.zeros(n, 8 * hd, device="cuda"), side=torch.cuda.Stream())

    def step(s, wait):
        s["q"].zero_()
        wide.mul_(1.0)  # a kernel that is still busy when the next launches arrive
        s["x"].copy_(rows[s["at"]][0])
        s["pos"].add_(1)
        if wait:
            torch.cuda.synchronize()
        x = s["x"]
        ops.qk_norm_rope_append(x[:, :8], x[:, 8:10], x[:, 10:], s["k"], s["v"], table, s["pos"], freqs=freqs, out=s["q"])
        if wait:
            torch.cuda.synchronize()
        ops.attn_decode_window(s["q"], s["k"], s["v"], table, s["pos"], out=s["o"])
        s["side"].wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s["side"]):
            torch.add(s["pos"], 1, out=s["len"])
        torch.cuda.current_stream().wait_stream(s["side"])
        if wait:
            torch.cuda.synchronize()
        ops.attn_prefill_window(s["q"], s["k"], s["v"], table, s["start"], s["len"], out=s["p"])
        s["sums"].add_(s["o"]).add_(s["p"])
        s["at"].add_(1)
        s["x"].fill_(math.nan)
        s["o"].fill_(math.nan)

    want = fresh()
    for _ in range(steps):
        step(want, True)
    eager = fresh()
    for _ in range(steps):
        step(eager, False)
    torch.cuda.synchronize()
    captured = fresh()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(captured, False)
    for _ in range(steps):
        graph.replay()
    torch.cuda.synchronize()
    assert want["sums"].isfinite().all() and int(want["at"]) == steps
    for got in (eager, captured):
        for name in ("sums", "k", "v", "pos", "q", "p"):
            assert torch.equal(got[name], want[name]), name
