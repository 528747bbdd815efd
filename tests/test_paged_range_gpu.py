"""GPU tests of the paged-cache attention at the ends of its range, against the formulas in 64 bits: weights far below
the row's largest, the largest finite values at keys that are seen, infinite keys and values of tiny weight, contexts
long enough that a lost page hides below an elementwise bound, tails of one accumulator.  Inputs, the 64-bit form and the
elementwise bounds are those of test_paged_ops_gpu.py."""
import math

import pytest
import torch

from test_paged_ops_gpu import BF16, F16, F32, PG, TYPES, Cache, check, gen, half_step, reference, run_decode

pytestmark = pytest.mark.gpu


def one_number(n, hq, hkv, hd, io, kv, scores, seed, scale=0.125):
    """(q, cache of one sequence) with score_j = scores[j] at every query: q is 1 in dim 0, keys hold nothing else."""
    c = Cache([n], hkv, hd, kv, seed)
    q = torch.randn((1, hq, hd), generator=gen(seed + 1), device="cuda").to(io)
    q[..., 0] = 1
    c.keys[0].zero_()
    c.keys[0][..., 0] = (scores / scale).to(kv)[:, None]
    store(c)
    return q, c


def store(c):
    """The cache's pages from c.keys and c.values."""
    for s, n in enumerate(c.lens):
        j = torch.arange(n, device="cuda")
        c.k[c.table[s, j // PG].long(), :, j % PG] = c.keys[s]
        c.v[c.table[s, j // PG].long(), :, j % PG] = c.values[s]


def prefill(q, c, past, **kw):
    from strataflow_b200 import ops
    n = q.shape[0]
    start = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    return ops.attn_prefill_window(q, c.k, c.v, c.table, start, start[1:] + past, **kw).view_as(q)


def decode(q, c, **kw):
    from strataflow_b200 import ops
    pos = torch.tensor(c.lens, dtype=torch.int32, device="cuda") - 1
    return ops.attn_decode_window(q, c.k, c.v, c.table, pos, **kw).view_as(q)


# ---- a dominant key over a long tail ---------------------------------------------------------------------
@pytest.mark.parametrize("io,kv", TYPES)
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("n_q,hq", [(3, 4), (2400, 8)])
def test_prefill_dominant_key_of_zero_value(cuda, io, kv, hd, n_q, hq):
    """One key 18 nats above 30000 others, its value 0, the others' of one sign: the output is the tail alone, of which
    each weight is 2^-26 of the largest.  With few tokens the keys are split, with 2400 they are not.

    A weight w (1 at the largest) is rounded once: 16-bit rows to half a step of their type, or, in f16, to half of its
    smallest step, where the largest weight stands for 2^11: 2^-36.  The rest is 32-bit arithmetic: the exponential and
    the scores, below 18 here, to 2^-20 of a weight, and sums over n keys."""
    n = 30000 + n_q
    g = gen(hd + n_q)
    scores = 0.3 * torch.randn(n, generator=g, device="cuda")
    scores[0] = 18.0
    q, c = one_number(n, hq, 1, hd, io, kv, scores, 3)
    c.values[0].copy_(0.5 + torch.rand((n, 1, hd), generator=g, device="cuda"))
    c.values[0][0] = 0
    store(c)
    q = q.expand(n_q, -1, -1).contiguous()
    got = prefill(q, c, n - n_q, scale=0.125)[:, 0].double()
    s = c.keys[0][:, 0, 0].double() * 0.125
    w = (s - s[0]).exp()
    v = c.values[0][:, 0].double()
    l = w.cumsum(0)[-n_q:, None]
    want = (w[:, None] * v).cumsum(0)[-n_q:] / l
    # rows and cache of 32 bits, or f32 rows over 16 bits: sums of n positive numbers, 2^-24 each at worst
    tol = (2.0 ** -19 + n * 2.0 ** -24) * want
    if io != F32:
        tol = tol + 2 * half_step(io) * want + 2 * 7.5e-5 * want
    if kv == F16:
        tol = tol + 2.0 ** -36 * v.cumsum(0)[-n_q:] / l
    check(got, want, tol)


# ---- the largest finite values at keys that are seen ------------------------------------------------------
@pytest.mark.parametrize("io,kv", [(F32, F32), (F32, BF16), (BF16, BF16)])
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("n", [40, 700, 20000])
def test_large_finite_values_of_seen_keys(cuda, io, kv, hd, n):
    """A weight of at most 1 times a finite value stays finite."""
    _, c, _, _ = run_decode([n], 8, 2, hd, io, kv, 0, 0)
    q = torch.randn((1, 8, hd), generator=gen(1), device="cuda").to(io)
    good = decode(q, c)
    others = [d for d in range(hd) if d != 3]
    for j, x in ((n - 7, 1e36), (0, -1e36), (n // 2, torch.finfo(kv).max)):
        value = c.values[0][j].clone()
        c.values[0][j, :, 3] = x
        store(c)
        got = decode(q, c)
        assert torch.equal(got[..., others], good[..., others])
        want, tol, absv = reference(q, c.keys[0], c.values[0], [n - 1], 0, 0)
        tol = (tol + half_step(io) * want.abs())[..., 3]
        check(got[..., 3], want[..., 3], tol)
        if io != F32:
            tol = tol + (half_step(kv) + 1.5e-4) * absv[..., 3]
        check(prefill(q, c, n - 1)[..., 3], want[..., 3], tol)
        c.values[0][j] = value
    store(c)


@pytest.mark.parametrize("io,kv", [(F32, F32), (F32, BF16), (BF16, BF16)])
@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("rise", [0.5, 2.0, 2.7, 2.9, 9.0])
def test_decode_largest_value_at_a_score_above_the_running_maximum(cuda, io, kv, hd, rise):
    """The largest value sits at a key that rises over all before it by less than what moves a running maximum, or by
    more: at every place of the pages that one warp takes."""
    n = 700
    for j in range(0, n, 61):
        scores = torch.zeros(n, device="cuda")
        scores[j] = rise
        q, c = one_number(n, 4, 1, hd, io, kv, scores, 5)
        c.values[0].zero_()
        c.values[0][j] = torch.finfo(kv).max
        store(c)
        want, tol, _ = reference(q, c.keys[0], c.values[0], [n - 1], 0, 0, 0.125)
        check(decode(q, c, scale=0.125), want, tol + half_step(io) * want.abs())


# ---- tails of one accumulator --------------------------------------------------------------------------
def decode_as(form, q, c, table, pos):
    """attn_decode_window with its workspace, or without one (a cluster joins the parts, or nobody)."""
    from strataflow_b200 import lib as L
    from strataflow_b200 import ops
    if form == "workspace":
        return ops.attn_decode_window(q, c.k, c.v, table, pos).view_as(q)
    out = torch.empty_like(q)
    n, hq, hd = q.shape
    L.check(L.load().sfk_attn_decode_window(ops._ROW_TYPES[q.dtype], q.data_ptr(), hq * hd, ops._KV_TYPES[c.k.dtype],
                                            c.k.data_ptr(), c.v.data_ptr(), c.k.shape[0], table.data_ptr(),
                                            table.shape[1], pos.data_ptr(), n, hq, c.kvh, hd, 0.0, 0, 0, out.data_ptr(),
                                            None, 0, None, torch.cuda.current_stream().cuda_stream))
    return out


# "many": the same sequence as many times as it takes to give each (sequence, kv head) one CTA
FORMS = [("workspace", 1), ("cluster", 1), ("many", 300)]


@pytest.mark.parametrize("form,copies", FORMS)
@pytest.mark.parametrize("kv", [F32, F16, BF16])
def test_decode_of_32_bit_rows_has_no_drift(cuda, form, copies, kv):
    """Values of one sign at 131072 keys: sums that only grow.  A sum of c numbers, each addition rounded to nearest:
    steps of 2^-23 of the partial sum at most, 0.72 of that on average, rms 0.72 * 2^-23 / 12^(1/2) (c / 3)^(1/2) of the
    result.  A warp of a sequence's only CTA adds a quarter of the keys: 2.6e-6, and four of them meet: 1.3e-6 an
    element, of which 2^-18 is three times.  The gain is a mean over 1024 such elements, with the error of the weights'
    sum (32 sums of an eighth of these: 1.6e-7): below 2^-20.  Additions that truncate would lose
    0.72 * 2^-24 c / 2 with c the products on one accumulator."""
    n, hd = 131072, 128
    c = Cache([n], 1, hd, kv, 14)
    c.values[0].copy_(0.5 + torch.rand((n, 1, hd), generator=gen(15), device="cuda"))
    store(c)
    copies = min(copies, 600) * 2
    q = torch.randn((copies, 4, hd), generator=gen(16), device="cuda") * 0.25
    table, pos = c.table.expand(copies, -1).contiguous(), torch.full((copies,), n - 1, dtype=torch.int32, device="cuda")
    got = decode_as(form, q, c, table, pos)[:2].double()
    want = reference(q[:2], c.keys[0], c.values[0], [n - 1] * 2, 0, 0)[0]
    gain = float((got * want).sum() / (want * want).sum()) - 1
    assert abs(gain) < 2.0 ** -20, gain
    assert float((got - want).norm() / want.norm()) < 2.0 ** -18


@pytest.mark.parametrize("form,copies", FORMS)
@pytest.mark.parametrize("kv", [F16, BF16])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_decode_of_16_bit_rows_has_no_drift(cuda, form, copies, kv, hd):
    """The same of 16-bit rows, each dim in a scale of its own, so that their roundings are independent: the gain is
    off by the mean of hd of them, 0.42 half_step / hd^(1/2) as a root of squares, four of these 0.21 half_step at 64,
    and by what a sum may lose: a quarter of half a step for both."""
    n = 131072
    c = Cache([n], 1, hd, kv, 14)
    scales = 2.0 ** (torch.arange(hd, device="cuda") / hd)
    c.values[0].copy_((0.5 + torch.rand((n, 1, hd), generator=gen(15), device="cuda")) * scales)
    store(c)
    copies = min(copies, 600) * 2
    q = (torch.randn((copies, 4, hd), generator=gen(16), device="cuda") * 0.25).to(kv)
    table, pos = c.table.expand(copies, -1).contiguous(), torch.full((copies,), n - 1, dtype=torch.int32, device="cuda")
    got = decode_as(form, q, c, table, pos)[:2].double()
    want = reference(q[:2], c.keys[0], c.values[0], [n - 1] * 2, 0, 0)[0]
    gain = float((got * want).sum() / (want * want).sum()) - 1
    assert abs(gain) < half_step(kv) / 4, gain
    assert float((got - want).norm() / want.norm()) < half_step(kv)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("pages", [8, 12, 13, 16, 17])
def test_decode_of_32_bit_rows_has_no_drift_at_short_chains(cuda, hd, pages):
    """32 warps of a cluster take `pages` pages each of values of one sign: 2^-20, as at long contexts."""
    n = pages * 32 * PG
    c = Cache([n], 1, hd, F16, 14)
    c.values[0].copy_(0.5 + torch.rand((n, 1, hd), generator=gen(15), device="cuda"))
    store(c)
    q = torch.randn((1, 4, hd), generator=gen(16), device="cuda") * 0.25
    got = decode_as("cluster", q, c, c.table, torch.full((1,), n - 1, dtype=torch.int32, device="cuda")).double()
    want = reference(q, c.keys[0], c.values[0], [n - 1], 0, 0)[0]
    assert abs(float((got * want).sum() / (want * want).sum()) - 1) < 2.0 ** -20


@pytest.mark.parametrize("kv", [F16, BF16])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n_q", [3, 2400])
def test_prefill_of_16_bit_rows_has_no_drift(cuda, kv, hd, n_q):
    """Prompts at 131072 keys of one sign, their keys split over CTAs (few tokens) or not.  The gain: as above 0.21
    half_step for the outputs' roundings; those of the weights are independent and 131072 of them meet; a fifth of
    half a step may be lost in sums."""
    n = 131072
    c = Cache([n], 1, hd, kv, 14)
    scales = 2.0 ** (torch.arange(hd, device="cuda") / hd)
    c.values[0].copy_((0.5 + torch.rand((n, 1, hd), generator=gen(15), device="cuda")) * scales)
    store(c)
    q = (torch.randn((n_q, 8, hd), generator=gen(16), device="cuda") * 0.25).to(kv)
    got = prefill(q, c, n - n_q)
    for i in (0, n_q // 2, n_q - 1):
        want = reference(q[i:i + 1], c.keys[0], c.values[0], [n - n_q + i], 0, 0)[0]
        gain = float((got[i:i + 1].double() * want).sum() / (want * want).sum()) - 1
        assert abs(gain) < 0.41 * half_step(kv), gain
        assert float((got[i:i + 1].double() - want).norm() / want.norm()) < half_step(kv)


@pytest.mark.parametrize("kv", [F16, BF16])
@pytest.mark.parametrize("hd", [32, 128])
@pytest.mark.parametrize("n_q,hq", [(3, 4), (2400, 8)])
def test_prefill_through_a_long_window(cuda, kv, hd, n_q, hq):
    """A window of 25000 of 32000 keys behind 100 sinks, scores that rise along the context so that the maximum moves in
    every run of keys, values of both signs: by the norm, half a step for the output, half a step and the polynomial for
    the weights."""
    n, window, n_sink = 32000, 25000, 100
    scores = torch.arange(n, device="cuda") / n * 12 + 0.5 * torch.randn(n, generator=gen(1), device="cuda")
    q, c = one_number(n, hq, 1, hd, kv, kv, scores, 3)
    q = q.expand(n_q, -1, -1).contiguous()
    got = prefill(q, c, n - n_q, scale=0.125, window=window, n_sink=n_sink).double()
    for i in (0, n_q // 2, n_q - 1):
        want, _, absv = reference(q[i:i + 1], c.keys[0], c.values[0], [n - n_q + i], window, n_sink, 0.125)
        bound = half_step(kv) * want.norm() + (half_step(kv) + 1.5e-4) * absv.norm()
        assert float((got[i:i + 1] - want).norm()) < float(bound)
        assert torch.equal(got[i], got[i][:1].expand_as(got[i]))  # every head has the same scores


@pytest.mark.parametrize("kv", [F16, BF16])
def test_a_million_keys_of_one_sign(cuda, kv):
    """What sums lose does not grow with the context: the bounds of 131072 keys at eight times as many, for single
    tokens of a batch that gives each sequence one CTA and for prompts whose keys are not split."""
    n, hd = 1 << 20, 64
    c = Cache([n], 1, hd, kv, 14, poison=False)
    scales = 2.0 ** (torch.arange(hd, device="cuda") / hd)
    c.values[0].copy_((0.5 + torch.rand((n, 1, hd), generator=gen(15), device="cuda")) * scales)
    store(c)
    q = (torch.randn((2400, 8, hd), generator=gen(16), device="cuda") * 0.25).to(kv)
    table, pos = c.table.expand(600, -1).contiguous(), torch.full((600,), n - 1, dtype=torch.int32, device="cuda")
    one = decode_as("many", q[-600:], c, table, pos)[-1:].double()
    all_ = prefill(q, c, n - 2400)[-1:].double()
    want = reference(q[-1:], c.keys[0], c.values[0], [n - 1], 0, 0)[0]
    for got, bound in ((one, 0.25), (all_, 0.41)):
        gain = float((got * want).sum() / (want * want).sum()) - 1
        assert abs(gain) < bound * half_step(kv), gain
        assert float((got - want).norm() / want.norm()) < half_step(kv)


# ---- no weight at all ------------------------------------------------------------------------------------
@pytest.mark.parametrize("io,kv", TYPES)
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("n", [40, 700, 9000])
def test_rows_of_scores_of_minus_infinity_alone(cuda, io, kv, hd, n):
    """A row all of whose seen keys score -inf has no weights: NaN; later rows are as if those keys were not there."""
    hidden = 21
    c = Cache([n], 2, hd, kv, 9)
    q = torch.randn((n, 4, hd), generator=gen(10), device="cuda").to(io)
    q[..., 0] = q[..., 0].abs() + 1
    c.keys[0][:hidden] = 0
    c.keys[0][:hidden, :, 0] = -math.inf
    store(c)
    got = prefill(q, c, 0)
    assert got[:hidden].isnan().all()
    rows = sorted({hidden, hidden + 1, n - 1})
    want, tol, absv = reference(q[rows], c.keys[0][hidden:], c.values[0][hidden:], [r - hidden for r in rows], 0, 0)
    if io != F32:
        tol = tol + half_step(io) * want.abs() + (half_step(kv) + 1.5e-4) * absv
    check(got[rows], want, tol)
    assert got[hidden:].isfinite().all()
    from strataflow_b200 import ops
    pos = torch.tensor([hidden - 1], dtype=torch.int32, device="cuda")
    assert ops.attn_decode_window(q[hidden - 1:hidden], c.k, c.v, c.table, pos).isnan().all()


# ---- infinite keys and values of tiny weight --------------------------------------------------------------
@pytest.mark.parametrize("io,kv", TYPES)
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("n", [40, 700, 20000])
@pytest.mark.parametrize("below", [10.0, 20.0, 40.0, 80.0])
def test_infinite_value_of_a_tiny_weight(cuda, io, kv, hd, n, below):
    """e^-below of the row's largest weight times an infinite value is infinite, for single tokens and for prompts; the
    other kv head and the other dims are as they were.  (Down to e^-80 = 2^-116: from 2^-126 on a weight is 0.)"""
    from strataflow_b200 import ops
    scores = torch.zeros(n, device="cuda")
    j = n // 2 + 3
    scores[j] = -below
    q, c = one_number(n, 8, 2, hd, io, kv, scores, 7)
    others = [d for d in range(hd) if d != 3]
    start = torch.tensor([0, 1], dtype=torch.int32, device="cuda")

    def prompt():
        return ops.attn_prefill_window(q, c.k, c.v, c.table, start, start[1:] * n, scale=0.125).view_as(q)

    for f in (lambda: decode(q, c, scale=0.125), prompt):
        good = f()
        for x in (math.inf, -math.inf, math.nan):
            value = c.v[c.table[0, j // PG], 0, j % PG, 3].clone()
            c.v[c.table[0, j // PG], 0, j % PG, 3] = x
            got = f()
            c.v[c.table[0, j // PG], 0, j % PG, 3] = value
            want = torch.full((4,), x, device="cuda", dtype=io)
            assert torch.allclose(got[0, :4, 3], want, equal_nan=True)
            assert torch.equal(got[0, 4:], good[0, 4:])
            w, tol, absv = reference(q, c.keys[0], c.values[0], [n - 1], 0, 0, 0.125)
            if io != F32:
                tol = tol + half_step(io) * w.abs() + (half_step(kv) + 1.5e-4) * absv
            check(got[..., others], w[..., others], tol.expand_as(w)[..., others])


@pytest.mark.parametrize("io,kv", [(F32, F32), (F32, F16), (F32, BF16)])
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("n", [40, 700, 20000])
def test_infinite_key_times_a_tiny_query(cuda, io, kv, hd, n):
    """A number of q 2^-30 below the row's largest times an infinite key: -inf takes the key out, +inf makes the row NaN."""
    _, c, _, _ = run_decode([n], 8, 2, hd, io, kv, 0, 0)
    q = torch.randn((1, 8, hd), generator=gen(1), device="cuda")
    q[..., 0] = torch.tensor([1.0, -1.0], device="cuda").repeat(4) * 2.0 ** -30
    j = n // 2 + 3
    kept = [i for i in range(n) if i != j]
    want, tol, _ = reference(q, c.keys[0][kept], c.values[0][kept], [n - 2], 0, 0)
    c.keys[0][j] = 0
    c.keys[0][j, :, 0] = math.inf
    store(c)
    for got in (decode(q, c), prefill(q, c, n - 1)):
        assert got[:, 0::2].isnan().all()
        check(got[:, 1::2], want[:, 1::2], tol[:, 1::2])


# ---- out and q in one buffer --------------------------------------------------------------------------------
@pytest.mark.parametrize("io,kv", TYPES)
@pytest.mark.parametrize("n,n_seq", [(40, 1), (700, 3), (20000, 1), (300, 40)])
def test_decode_in_place_and_between_rows(cuda, io, kv, n, n_seq):
    """out = q, out in the gap between q's rows, out right behind and right before q's rows: the bits of an out of its
    own.  out over a wider q is refused."""
    from strataflow_b200 import lib as L
    hq, hd = 8, 64
    c = Cache([n] * n_seq, 2, hd, kv, 1)
    q = torch.randn((n_seq, hq, hd), generator=gen(2), device="cuda").to(io)
    want = decode(q, c)
    mine = q.clone()
    decode(mine, c, out=mine.view(n_seq, hq * hd))
    assert torch.equal(mine, want)
    buf = torch.zeros((n_seq, (n_seq + 1) * hq * hd), dtype=io, device="cuda")
    wide = buf[:, :hq * hd].unflatten(1, (hq, hd))
    wide.copy_(q)
    decode(wide, c, out=buf[0, hq * hd:].view(n_seq, hq * hd))
    assert torch.equal(buf[0, hq * hd:].view_as(want), want) and torch.equal(wide, q)
    flat = torch.zeros((3 * n_seq, hq * hd), dtype=io, device="cuda")
    own = flat[n_seq:2 * n_seq].unflatten(1, (hq, hd))
    own.copy_(q)
    for out in (flat[:n_seq], flat[2 * n_seq:]):
        decode(own, c, out=out)
        assert torch.equal(out.view_as(want), want) and torch.equal(own, q)
    if n_seq > 1:
        with pytest.raises(L.SfkError, match="overlaps"):
            decode(wide, c, out=buf.view(-1)[:n_seq * hq * hd].view(n_seq, -1))


@pytest.mark.parametrize("io", [F32, F16, BF16])
@pytest.mark.parametrize("n", [1, 5, 3000])
def test_append_in_place_of_a_packed_row(cuda, io, n):
    """q_out = q inside packed rows, its k and v beside it: the bits of an out of its own; k and v as they were.  q_out
    over k, or over q in another stride, is refused."""
    from strataflow_b200 import lib as L
    from strataflow_b200 import ops
    hq, hkv, hd = 8, 2, 64
    x = torch.randn((n, hq + 2 * hkv, hd), generator=gen(3), device="cuda").to(io)
    y = x.clone()
    pages = (n + PG - 1) // PG
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None].contiguous()
    pos = torch.arange(n, dtype=torch.int32, device="cuda")

    def run(rows, out):
        pools = torch.zeros((2, pages, hkv, PG, hd), dtype=io, device="cuda")
        got = ops.qk_norm_rope_append(rows[:, :hq], rows[:, hq:hq + hkv], rows[:, hq + hkv:], pools[0], pools[1], table, pos,
                                      seq=torch.zeros_like(pos), freqs=ops.rope_freqs(hd), neox=True, out=out)
        return got, pools

    want, pools = run(x, None)
    got, mine = run(y, y[:, :hq])
    assert torch.equal(got, want) and torch.equal(mine, pools) and torch.equal(y[:, hq:], x[:, hq:])
    for bad in (x[:, 1:hq + 1], x[:, 2 * hkv:], x.view(-1)[:n * hq * hd].view(n, hq, hd)):
        if n == 1 and bad.data_ptr() == x.data_ptr():
            continue
        with pytest.raises(L.SfkError, match="overlaps"):
            run(x, bad)


# ---- long contexts: what an elementwise bound cannot see ---------------------------------------------------
@pytest.mark.parametrize("form,copies", FORMS)
@pytest.mark.parametrize("io,kv", TYPES)
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("n", [20000, 9001])
def test_decode_counts_every_key_once(cuda, form, copies, io, kv, hd, n):
    """Equal weights (q = 0) and values that are 1 at one dim of each key: each dim is the share of its keys, about
    n / hd of them.  A page lost or taken twice is 16 keys of dims of their own, 16 / (n / hd) or more of these.  Weights,
    sums of whole numbers up to n and of weights are exact; one division and the output's rounding are left."""
    c = Cache([n], 2, hd, kv, 11)
    j = torch.arange(n, device="cuda")
    c.values[0].copy_((j[:, None] // PG % hd == torch.arange(hd, device="cuda"))[:, None])
    store(c)
    q = torch.zeros((copies, 8, hd), dtype=io, device="cuda")
    table, pos = c.table.expand(copies, -1).contiguous(), torch.full((copies,), n - 1, dtype=torch.int32, device="cuda")
    got = decode_as(form, q, c, table, pos).double()
    want = c.values[0][:, 0].double().mean(0).expand_as(got)
    assert want.min() > 0
    check(got, want, (2.0 ** -21 + half_step(io)) * want)


@pytest.mark.parametrize("form,copies", FORMS)
@pytest.mark.parametrize("io,kv", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_decode_long_contexts_by_their_norm(cuda, form, copies, io, kv, hd):
    """Random scores and values at 20000 keys.  Errors of the elements are independent: as a root of squares the scores'
    rounding (hd + 6 steps of 2^-24 of a sum whose rms is 1: 2^-24 (hd + 6)^(1/2) < 2^-19), the exponential's 2^-22 and
    n additions of 2^-24 of a partial sum, which is the output's size at the end and less before, 2^-24 n^(1/2) < 2^-16.
    A 16-bit output adds at most half a step of itself.  A page of 1250 would be 2^-5."""
    n = 20000
    c = Cache([n], 2, hd, kv, 12)
    q = torch.randn((copies, 8, hd), generator=gen(13), device="cuda").to(io)
    table, pos = c.table.expand(copies, -1).contiguous(), torch.full((copies,), n - 1, dtype=torch.int32, device="cuda")
    got = decode_as(form, q, c, table, pos)[:4].double()
    want = reference(q[:4], c.keys[0], c.values[0], [n - 1] * min(4, copies), 0, 0)[0]
    bound = 2.0 ** -16 + (half_step(io) if io != F32 else 0)
    assert float((got - want).norm() / want.norm()) < bound
    assert abs(float((got * want).sum() / (want * want).sum()) - 1) < bound


@pytest.mark.parametrize("io,kv", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("window,n_sink", [(0, 0), (7003, 40)])
@pytest.mark.parametrize("n_q", [3, 700])
def test_windows_and_prompts_count_every_key_once(cuda, io, kv, hd, window, n_sink, n_q):
    """The same for a window with sinks and for prompts, their keys split over CTAs or not.  A prompt's polynomial
    exponential makes weights of a few columns 7.5e-5 (bf16) or 2.7e-6 (f16) smaller before they are rounded."""
    n = 20000
    c = Cache([n], 2, hd, kv, 11)
    j = torch.arange(n, device="cuda")
    c.values[0].copy_((j[:, None] // PG % hd == torch.arange(hd, device="cuda"))[:, None])
    store(c)
    q = torch.zeros((n_q, 8, hd), dtype=io, device="cuda")
    p = torch.arange(n - n_q, n, device="cuda")[:, None]
    seen = j <= p
    if window:
        seen &= (j > p - window) | (j < n_sink)
    want = (seen.double() @ c.values[0][:, 0].double() / seen.sum(-1, keepdim=True))[:, None]
    tol = (2.0 ** -21 + (half_step(io) if io != F32 else 0)) * want
    check(decode(q[-1:], c, window=window, n_sink=n_sink), want[-1:], tol[-1:])
    if io != F32:
        tol = tol + (7.5e-5 if kv == BF16 else 2.7e-6) * want
    check(prefill(q, c, n - n_q, window=window, n_sink=n_sink), want, tol)


# ---- an error of another call -------------------------------------------------------------------------------
@pytest.mark.parametrize("io,kv", [(F32, F32), (BF16, BF16)])
def test_an_earlier_error_is_not_reported_again(cuda, io, kv):
    """An engine larger than the card fails to allocate; the operators' calls after it are fine."""
    from strataflow_b200 import engine as E
    from strataflow_b200 import lib as L
    from strataflow_b200 import ops
    c = Cache([20], 2, 64, kv, 1)
    q = torch.randn((20, 4, 64), generator=gen(2), device="cuda").to(io)
    k = torch.randn((20, 2, 64), generator=gen(3), device="cuda").to(io)
    pos, freqs = torch.arange(20, dtype=torch.int32, device="cuda"), ops.rope_freqs(64)
    calls = (lambda: ops.qk_norm_rope_append(q, k, k, c.k, c.v, c.table, pos, seq=torch.zeros_like(pos), freqs=freqs),
             lambda: prefill(q, c, 0), lambda: decode(q[:1], c))
    for f in calls:
        want = f()
        with pytest.raises(L.SfkError):
            E.Engine(E.tiny_config(n_vocab=800_000_000))
        assert torch.equal(f(), want)


# ---- sequences whose rows overlap ---------------------------------------------------------------------------
@pytest.mark.parametrize("io,kv,hd", [(F32, F32, 64), (F32, F16, 128), (BF16, BF16, 128)])
@pytest.mark.parametrize("first,late", [(0, 2), (3, 6), (125, 127), (126, 128), (127, 129), (60, 140)])
def test_prefill_q_start_that_descends_leaves_the_other_sequences_alone(cuda, io, kv, hd, first, late):
    """q_start goes back once, into the rows of sequence `first`: the sequence that ends there and the one that begins
    there are reported and touch nothing, all others are as they were."""
    from strataflow_b200 import lib as L
    from strataflow_b200 import ops
    n_seq, each = 150, 20
    c = Cache([each] * n_seq, 1, hd, kv, 1)
    q = torch.randn((n_seq * each, 2, hd), generator=gen(2), device="cuda").to(io)
    start = torch.arange(n_seq + 1, dtype=torch.int32, device="cuda") * each
    kv_len = torch.full((n_seq,), each, dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    good = ops.attn_prefill_window(q, c.k, c.v, c.table, start, kv_len, status=status)
    ops.check_status(status)
    start[late] = first * each + 10
    out = torch.full_like(good, 5.0)
    ops.attn_prefill_window(q, c.k, c.v, c.table, start, kv_len, out=out, status=status)
    with pytest.raises(L.SfkError, match="position or length"):
        ops.check_status(status)
    a, b = (late - 1) * each, (late + 1) * each
    assert torch.equal(out[:a], good[:a]) and torch.equal(out[b:], good[b:])
    assert (out[a:b] == 5.0).all()


# ---- queries at the ends of f32 -----------------------------------------------------------------------------
@pytest.mark.parametrize("kv", [F32, F16, BF16])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("n", [40, 700])
def test_tiny_and_huge_queries(cuda, kv, hd, n):
    """q near 2^-126 under a small scale: scores of 0, the mean of the values.  q near 2^127 under a scale above 1, keys
    of at most 2^-2: scores up to 2^127 and the others 2^100 below, the largest key's value alone."""
    c = Cache([n], 2, hd, kv, 1)
    g = gen(2)
    v = c.values[0].double().repeat_interleave(2, 1)
    q = torch.randn((1, 4, hd), generator=g, device="cuda") * 1e-37
    want = v.mean(0, keepdim=True)
    for got in (decode(q, c, scale=1e-9), prefill(q, c, n - 1, scale=1e-9)):
        check(got, want, (n + 16) * 2.0 ** -23 * v.abs().amax().expand_as(want))
    top = n // 3
    scores = torch.arange(n, device="cuda").float() / n * 2.0 ** -4
    scores[top] = 2.0 ** -2
    c.keys[0].zero_()
    c.keys[0][..., 0] = scores.to(kv)[:, None]
    store(c)
    q.zero_()
    q[..., 0] = 2.0 ** 126
    want = v[top][None]
    for got in (decode(q, c, scale=4.0), prefill(q, c, n - 1, scale=4.0)):
        check(got, want, 2.0 ** -20 * want.abs())
