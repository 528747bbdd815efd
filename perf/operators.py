"""Cases of the paged-cache operators: appending rotated keys and values, and attention with a sliding window over the
cache, for single tokens and for prompts.

The cache is the engine's: a pool of 16-token pages [n_pages][n_head_kv][16][head_dim] for keys and one for values, and a
table of page ids for each sequence.
  append   q, k of each head normed (optional) and rotated, q returned, k and v written to their slots
  decode   one new token of each sequence over the keys it sees
  prefill  the newest tokens of each sequence, each over the keys it sees
Key j is seen from position p if j <= p and (window is 0, or j > p - window, or j < n_sink).
"""
import math

import torch

own = False

PAGE = 16
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BASE = 10000.0
EPS = 1e-6


# ---- cases --------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token of one sequence into an f16 cache, q and k in 32 bits: what the engine's own decode step hands over
        dict(name="append 1 f32 to f16", op="append", n_seq=1, n_tok=1, past=700, heads=32, kv_heads=8, dim=128, io="f32",
             kv="f16", norm=False, neox=False, rot=128, axes=1),
        # a prompt of 8192 tokens of a model that norms each head of q and k, bf16 throughout
        dict(name="append 8192 bf16 normed", op="append", n_seq=1, n_tok=8192, past=100000, heads=64, kv_heads=8, dim=128,
             io="bf16", kv="bf16", norm=True, neox=True, rot=128, axes=1),
        # images and text of five requests: three position axes, part of each head rotated, an odd number of tokens
        dict(name="append 5041 f16 three axes", op="append", n_seq=5, n_tok=5041, past=300, heads=28, kv_heads=4, dim=128,
             io="f16", kv="f16", norm=False, neox=True, rot=96, axes=3),
        # the smallest call: one token over a short 32-bit cache (the small test model's heads and context)
        dict(name="decode 1 x 77 f32", op="decode", n_seq=1, ctx=77, ragged=False, heads=8, kv_heads=4, dim=32, io="f32",
             kv="f32", window=0, n_sink=0),
        # one user, a long context, the engine's types
        dict(name="decode 1 x 32768 f32 over f16", op="decode", n_seq=1, ctx=32768, ragged=False, heads=32, kv_heads=8,
             dim=128, io="f32", kv="f16", window=0, n_sink=0),
        # a serving batch of uneven lengths, a window of 1024 keys and four sinks
        dict(name="decode 48 ragged window bf16", op="decode", n_seq=48, ctx=8192, ragged=True, heads=64, kv_heads=8,
             dim=128, io="bf16", kv="bf16", window=1024, n_sink=4),
        # the largest cache: eight sequences of 131072 tokens
        dict(name="decode 8 x 131072 bf16", op="decode", n_seq=8, ctx=131072, ragged=False, heads=64, kv_heads=8, dim=128,
             io="bf16", kv="bf16", window=0, n_sink=0),
        # a short prompt over a 32-bit cache (the small test model)
        dict(name="prefill 37 f32", op="prefill", n_seq=1, n_q=37, past=0, ragged=False, heads=8, kv_heads=4, dim=32,
             io="f32", kv="f32", window=0, n_sink=0),
        # one prompt chunk of the engine's size in the engine's types, behind an earlier chunk
        dict(name="prefill 512 f32 over f16", op="prefill", n_seq=1, n_q=512, past=500, ragged=False, heads=32,
             kv_heads=8, dim=128, io="f32", kv="f16", window=0, n_sink=0),
        # six uneven prompts at once, some behind a cached prefix, heads of 64
        dict(name="prefill 6 ragged f16", op="prefill", n_seq=6, n_q=1999, past=1500, ragged=True, heads=32, kv_heads=8,
             dim=64, io="f16", kv="f16", window=0, n_sink=0),
        # a long prompt through a window of 2048 keys and four sinks
        dict(name="prefill 8192 window bf16", op="prefill", n_seq=1, n_q=8192, past=0, ragged=False, heads=32, kv_heads=8,
             dim=128, io="bf16", kv="bf16", window=2048, n_sink=4),
        # a chunk of 2048 tokens far into a long context
        dict(name="prefill 2048 at 30000 bf16", op="prefill", n_seq=1, n_q=2048, past=28001, ragged=False, heads=32,
             kv_heads=8, dim=128, io="bf16", kv="bf16", window=0, n_sink=0),
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_once(rng):
    op = rng.choice(["append", "decode", "prefill"])
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8])
    io, kv = rng.choice([("f32", "f16"), ("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "bf16")])
    c = dict(op=op, heads=heads, kv_heads=kv_heads, dim=dim, io=io, kv=kv)
    if op == "append":
        n_seq = _spread(rng, 1, 64)
        axes = rng.choice([1, 1, 3])
        c.update(n_seq=n_seq, n_tok=max(n_seq, _spread(rng, 1, 8192)), past=_spread(rng, 1, 100000 // n_seq),
                 norm=rng.random() < 0.5, neox=rng.random() < 0.5, rot=rng.choice([dim, dim, dim // 2]), axes=axes)
        return c
    window = rng.choice([0, 0, _spread(rng, 16, 4096)])
    c.update(window=window, n_sink=rng.choice([0, 1, 4, 17]) if window else 0, ragged=rng.random() < 0.5)
    if op == "decode":
        c.update(n_seq=_spread(rng, 1, 128), ctx=_spread(rng, 1, 131072))
    else:
        c.update(n_seq=_spread(rng, 1, 8), n_q=_spread(rng, 1, 8192), past=rng.choice([0, _spread(rng, 1, 28001)]))
    return c


def _cost(c):
    """What a case asks of memory and time, the plain form's included."""
    w = work(c)
    scores = 0
    if c["op"] == "prefill":
        scores = c["n_seq"] * c["heads"] * c["n_q"] * (c["n_q"] + c["past"])
    return w["bytes"], w["flops"], scores


def draw(rng):
    most = {}
    for c in listed():
        most[c["op"]] = [max(a, b) for a, b in zip(most.get(c["op"], (0, 0, 0)), _cost(c))]
    while True:
        c = _draw_once(rng)
        if all(a <= b for a, b in zip(_cost(c), most[c["op"]])):
            return c


def _mixed(n, i):
    """A fixed spread of 0..n-1 over i: lengths of a ragged batch."""
    return (i * 7919 + 3571) % 10007 * n // 10007


def _lengths(c):
    """[(new tokens, cached tokens before them)] of each sequence."""
    n = c["n_seq"]
    if c["op"] == "append":
        first = c["n_tok"] // n
        return [(first + (1 if i < c["n_tok"] % n else 0), c["past"] if i % 2 == 0 else c["past"] // 3) for i in range(n)]
    if c["op"] == "decode":
        return [(1, c["ctx"] - 1 if not c["ragged"] or i == 0 else _mixed(c["ctx"], i)) for i in range(n)]
    if not c["ragged"]:
        return [(c["n_q"], c["past"])] * n
    return [(c["n_q"] if i == 0 else 1 + _mixed(c["n_q"], i), c["past"] if i % 2 == 0 else _mixed(c["past"] + 1, i)) for i in range(n)]


def _seen(p, window, n_sink):
    """How many keys position p sees."""
    if not window or p + 1 <= window:
        return p + 1
    return window + min(n_sink, p + 1 - window)


def work(case):
    c = case
    row = c["dim"]
    if c["op"] == "append":
        n = c["n_tok"]
        q = n * c["heads"] * row * SIZE[c["io"]]
        kv = 2 * n * c["kv_heads"] * row
        return {"bytes": 2 * q + kv * (SIZE[c["io"]] + SIZE[c["kv"]]), "flops": 6 * n * (c["heads"] + c["kv_heads"]) * row}
    pairs, keys, rows = 0, 0, 0
    for n_q, past in _lengths(c):
        total = past + n_q
        w, s = c["window"], c["n_sink"]
        if not w or total <= w:
            pairs += n_q * past + n_q * (n_q + 1) // 2
        else:
            pairs += sum(_seen(p, w, s) for p in range(past, total))
        first = max(0, past - w + 1) if w else 0
        keys += total - first + min(s, first)
        rows += n_q
    return {"bytes": 2 * keys * c["kv_heads"] * row * SIZE[c["kv"]] + 2 * rows * c["heads"] * row * SIZE[c["io"]],
            "flops": 4 * pairs * c["heads"] * row}


# ---- inputs -------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    c = case
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    io, kv = TYPES[c["io"]], TYPES[c["kv"]]
    lens = _lengths(c)
    n_seq, heads, kvh, dim = c["n_seq"], c["heads"], c["kv_heads"], c["dim"]
    used = [(a + b + PAGE - 1) // PAGE for a, b in lens]
    if c["op"] == "append":  # the pages that hold the new tokens, and the ones before them: pages seen here alone
        first = [b // PAGE for a, b in lens]
    else:
        first = [0] * n_seq
    n_pages = sum(u - f for u, f in zip(used, first)) + 3
    ids = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
    table = torch.zeros(n_seq, max(used), dtype=torch.int32, device=dev)
    at = 0
    for s in range(n_seq):
        table[s, first[s]:used[s]] = ids[at:at + used[s] - first[s]]
        at += used[s] - first[s]
    shape = (n_pages, kvh, PAGE, dim)
    st = {"case": c, "table": table,
          "k_pages": torch.randn(shape, generator=g, device=dev, dtype=kv),
          "v_pages": torch.randn(shape, generator=g, device=dev, dtype=kv)}
    new = torch.tensor([a for a, b in lens], device=dev)
    past = torch.tensor([b for a, b in lens], device=dev)
    start = torch.zeros(n_seq + 1, dtype=torch.int64, device=dev)
    start[1:] = new.cumsum(0)
    n_tok = sum(a for a, b in lens)
    if c["op"] == "append":
        st["qkv"] = torch.randn((n_tok, (heads + 2 * kvh) * dim), generator=g, device=dev, dtype=io)
        seq = torch.repeat_interleave(torch.arange(n_seq, device=dev), new, output_size=n_tok)
        pos = past[seq] + torch.arange(n_tok, device=dev) - start[seq]
        st["seq"], st["pos"] = seq.to(torch.int32), pos.to(torch.int32)
        st["freqs"] = (BASE ** (-torch.arange(c["rot"] // 2, device=dev, dtype=torch.float64) * 2 / c["rot"])).float()
        if c["norm"]:
            st["q_norm"] = 1 + 0.1 * torch.randn(dim, generator=g, device=dev)
            st["k_norm"] = 1 + 0.1 * torch.randn(dim, generator=g, device=dev)
        if c["axes"] > 1:  # time, row and column of image patches: 40 patches to a row
            i = pos - past[seq]
            st["rope_pos"] = torch.stack([past[seq] + i // 1600, i // 40 % 40, i % 40]).to(torch.int32)
            st["axes"] = bytes(min(2, 3 * i // (c["rot"] // 2)) for i in range(c["rot"] // 2))
        return st
    st["q"] = torch.randn((n_tok, heads, dim), generator=g, device=dev).to(io)
    if c["op"] == "decode":
        st["positions"] = past.to(torch.int32)
    else:
        st["q_start"] = start.to(torch.int32)
        st["kv_len"] = (past + new).to(torch.int32)
        st["n_q_max"] = max(a for a, b in lens)
    return st


# ---- one pass -----------------------------------------------------------------------------------------------------
def run(state):
    return {"append": _append, "decode": _decode, "prefill": _prefill}[state["case"]["op"]](state)


def _split(state):
    """q, k and v of each token: views of the packed rows."""
    c = state["case"]
    h, g, d = c["heads"], c["kv_heads"], c["dim"]
    x = state["qkv"].view(-1, h + 2 * g, d)
    return x[:, :h], x[:, h:h + g], x[:, h + g:]


def _append(state):
    c = state["case"]
    q, k, v = _split(state)
    if own:
        from strataflow_b200 import ops
        out = ops.qk_norm_rope_append(q, k, v, state["k_pages"], state["v_pages"], state["table"], state["pos"],
                                      seq=state["seq"], freqs=state["freqs"], neox=c["neox"],
                                      q_norm=state.get("q_norm"), k_norm=state.get("k_norm"), eps=EPS,
                                      rope_pos=state.get("rope_pos"), axes=state.get("axes"))
        return {"q": out, "k_pages": state["k_pages"], "v_pages": state["v_pages"]}
    freqs = state["freqs"].double()
    if c["axes"] > 1:
        axis = torch.frombuffer(bytearray(state["axes"]), dtype=torch.uint8).long().to(freqs.device)
        where = state["rope_pos"][axis].t().double()
    else:
        where = state["pos"].double()[:, None]
    angle = where * freqs
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turned(x, weight):
        x = x.float()
        if weight is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight
        r = c["rot"]
        if c["neox"]:
            a, b = x[..., :r // 2], x[..., r // 2:r]
            return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., r:]], -1)
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
        return torch.cat([y, x[..., r:]], -1)

    page = state["table"][state["seq"].long(), state["pos"].long() // PAGE].long()
    slot = state["pos"].long() % PAGE
    kp, vp = state["k_pages"], state["v_pages"]
    kp[page, :, slot] = turned(k, state.get("k_norm")).to(kp.dtype)
    vp[page, :, slot] = v.to(vp.dtype)
    return {"q": turned(q, state.get("q_norm")).to(q.dtype), "k_pages": kp, "v_pages": vp}


def _gathered(state):
    """Keys and values of each sequence in order, in 32 bits: [n_seq][kv_heads][keys][dim]."""
    t = state["table"].long()
    return [p[t].permute(0, 2, 1, 3, 4).flatten(2, 3).float() for p in (state["k_pages"], state["v_pages"])]


def _weighted(scores, seen, v):
    """softmax over the seen keys, then the sum of the values: scores [n, kv_heads, rows, keys]."""
    scores = scores.masked_fill_(~seen, -math.inf)
    p = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    return torch.matmul(p, v) / p.sum(-1, keepdim=True)


def _decode(state):
    c = state["case"]
    if own:
        from strataflow_b200 import ops
        return ops.attn_decode_window(state["q"], state["k_pages"], state["v_pages"], state["table"],
                                      state["positions"], window=c["window"], n_sink=c["n_sink"])
    q = state["q"]
    k, v = _gathered(state)
    n, h, d = q.shape
    scores = torch.matmul(q.float().view(n, c["kv_heads"], -1, d), k.transpose(-1, -2)) * d ** -0.5
    j = torch.arange(k.shape[2], device=q.device)
    p = state["positions"].long()[:, None]
    seen = j <= p
    if c["window"]:
        seen = seen & ((j > p - c["window"]) | (j < c["n_sink"]))
    return _weighted(scores, seen[:, None, None], v).reshape(n, h * d).to(q.dtype)


def _prefill(state):
    c = state["case"]
    if own:
        from strataflow_b200 import ops
        return ops.attn_prefill_window(state["q"], state["k_pages"], state["v_pages"], state["table"], state["q_start"],
                                       state["kv_len"], window=c["window"], n_sink=c["n_sink"])
    q = state["q"]
    k, v = _gathered(state)
    n_tok, h, d = q.shape
    kvh, group = c["kv_heads"], h // c["kv_heads"]
    start, kv_len = state["q_start"].long(), state["kv_len"].long()
    n_q = start[1:] - start[:-1]
    i = torch.arange(state["n_q_max"], device=q.device)
    row = (start[:-1, None] + i).clamp_(max=n_tok - 1)  # of each sequence's i-th token; the ones past its end are left out below
    x = q[row].float().unflatten(2, (kvh, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    scores = torch.matmul(x, k.transpose(-1, -2)).mul_(d ** -0.5)
    j = torch.arange(k.shape[2], device=q.device)
    p = ((kv_len - n_q)[:, None] + i)[:, :, None]
    seen = j <= p
    if c["window"]:
        seen = seen & ((j > p - c["window"]) | (j < c["n_sink"]))
    y = _weighted(scores.unflatten(2, (group, -1)), seen[:, None, None], v[:, :, None])
    y = y.permute(0, 3, 1, 2, 4).flatten(2)
    return y[i < n_q[:, None]].to(q.dtype)


# ---- the definition in 64 bits ------------------------------------------------------------------------------------
def exact(case, seed):
    c = case
    st = prepare(case, seed)
    lens = _lengths(c)
    if c["op"] == "append":
        return _exact_append(c, st, lens)
    out = []
    at = 0
    group = c["heads"] // c["kv_heads"]
    dev = st["q"].device
    for s, (n_q, past) in enumerate(lens):
        total = past + n_q
        pages = st["table"][s, :(total + PAGE - 1) // PAGE].long()
        p = torch.arange(past, total, device=dev)[:, None]
        j = torch.arange(total, device=dev)[None]
        hidden = (j > p) | ((j <= p - c["window"]) & (j >= c["n_sink"])) if c["window"] else j > p
        rows = []
        for h in range(c["heads"]):
            k = st["k_pages"][pages, h // group].reshape(-1, c["dim"])[:total].double()
            v = st["v_pages"][pages, h // group].reshape(-1, c["dim"])[:total].double()
            x = st["q"][at:at + n_q, h].double()
            a = torch.where(hidden, -math.inf, x @ k.T / math.sqrt(c["dim"]))
            rows.append(torch.softmax(a, -1) @ v)
        out.append(torch.stack(rows, 1).flatten(1))
        at += n_q
    return torch.cat(out)


def _exact_append(c, st, lens):
    h, kvh, d, r = c["heads"], c["kv_heads"], c["dim"], c["rot"]
    dev = st["qkv"].device
    x = st["qkv"].double().reshape(-1, h + 2 * kvh, d)
    f = st["freqs"].double()
    k_pages, v_pages = st["k_pages"].double(), st["v_pages"].double()
    pos = torch.cat([torch.arange(b, a + b, device=dev) for a, b in lens])
    if c["axes"] > 1:
        theta = torch.stack([st["rope_pos"][st["axes"][i]].double() * f[i] for i in range(r // 2)], -1)
    else:
        theta = pos.double()[:, None] * f[None]
    z = torch.polar(torch.ones_like(theta), theta)[:, None]

    def one(y, w):
        if w is not None:
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / d + EPS) * w.double()
        y = y.clone()
        if c["neox"]:
            t = torch.complex(y[..., :r // 2], y[..., r // 2:r]) * z
            y[..., :r // 2], y[..., r // 2:r] = t.real, t.imag
        else:
            t = torch.complex(y[..., 0:r:2].contiguous(), y[..., 1:r:2].contiguous()) * z
            y[..., 0:r:2], y[..., 1:r:2] = t.real, t.imag
        return y

    q = one(x[:, :h], st.get("q_norm"))
    k = one(x[:, h:h + kvh], st.get("k_norm"))
    at = 0
    for s, (n, past) in enumerate(lens):
        p = torch.arange(past, past + n, device=dev)
        page = st["table"][s, p // PAGE].long()
        k_pages[page, :, p % PAGE] = k[at:at + n]
        v_pages[page, :, p % PAGE] = x[at:at + n, h + kvh:]
        at += n
    return {"q": q, "k_pages": k_pages, "v_pages": v_pages}
