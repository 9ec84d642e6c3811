"""The operators of the paged 4-bit KV cache, as cases that can be timed.

Many sessions share one pool of cache pages per layer.  Keys and values are held
as 4-bit codes in groups of 32 channels, each group with one half-precision
scale (the values of GGUF's Q4_0: d * (c - 8)):

  append     one step's queries and keys rotated to their positions, keys and
             values quantized into their pages; the stored rows read back
  read       the stored rows of sessions as numbers (a session saved or moved)
  attention  the step's queries over the pages of their own session
  step       append, then attention, as a layer of a batched step calls them

Head layouts are this repository's own configurations; lengths run from one
token to the longest context it names.  `own` picks the library's calls; without
it the same numbers come from elementary torch operations on the same bytes.

Page layout.  A page holds `page` tokens; for each kv head it is one block of
page * 18 * G bytes, G = 2, 4 or 8 groups of 32 channels (the head size rounded
up): page * 16 * G bytes of codes, then half-precision scales [page][G].
  K codes, per token: dwords [kc 0..3][g], nibble n = channel 32 g + 8 kc + n
  V codes, per four tokens: [c 0..15][token 0..3][g] bytes, low nibble = channel
  32 g + c, high nibble = channel 32 g + 16 + c
"""
from __future__ import annotations

import math

import torch

own = False
DEV = "cuda:0"

# (query heads, kv heads, head size, rotation pairs split in halves) of the configurations
HEADS = {"llama3-8b": (32, 8, 128, False), "qwen2.5-14b": (40, 8, 128, True), "tinyllama": (32, 4, 64, False),
         "gpt-oss": (64, 8, 64, True)}
THETA = {"llama3-8b": 500000.0, "qwen2.5-14b": 1000000.0, "tinyllama": 10000.0, "gpt-oss": 150000.0}
MOST = 131072  # positions of the longest context


# ---- the cases ---------------------------------------------------------------------
def listed():
    return [
        # one user, one new token: what a call costs at least
        dict(name="append-1", kind="append", heads="llama3-8b", dtype="f32", page=32, seqs=1, new=1, ctx=4097),
        # one decode step of many sessions, some of them far into a long context
        dict(name="append-200-far", kind="append", heads="gpt-oss", dtype="bf16", page=16, seqs=200, new=1,
             ctx=MOST),
        # prompts of several sessions in one batch, ragged
        dict(name="append-prompts", kind="append", heads="qwen2.5-14b", dtype="f32", page=64, seqs=9, new=1700,
             ctx=2500),
        # a few short sessions handed to another process
        dict(name="read-33-short", kind="read", heads="gpt-oss", dtype="bf16", page=16, seqs=33, new=300, ctx=300),
        # one long session saved
        dict(name="read-20001", kind="read", heads="llama3-8b", dtype="f32", page=32, seqs=1, new=20001, ctx=20001),
        # the smallest attention: one user early in a conversation
        dict(name="decode-1-ctx130", kind="attention", heads="llama3-8b", dtype="f32", page=32, seqs=1, new=1,
             ctx=130, window=0, sinks=False),
        # one user at the end of the longest context: few rows, a long axis
        dict(name="decode-1-long", kind="attention", heads="llama3-8b", dtype="bf16", page=64, seqs=1, new=1,
             ctx=MOST, window=0, sinks=False),
        # a server's decode step: 48 sessions of ragged lengths
        dict(name="decode-48", kind="attention", heads="llama3-8b", dtype="f32", page=32, seqs=48, new=1, ctx=8192,
             window=0, sinks=False),
        # the sliding-window layers of gpt-oss with sinks, 256 sessions
        dict(name="decode-256-window", kind="attention", heads="gpt-oss", dtype="bf16", page=16, seqs=256, new=1,
             ctx=4096, window=128, sinks=True),
        # a first prompt of 512 tokens
        dict(name="prefill-512", kind="attention", heads="llama3-8b", dtype="f32", page=32, seqs=1, new=512, ctx=512,
             window=0, sinks=False),
        # ragged chunks of long prompts over what is cached of them
        dict(name="prefill-chunks", kind="attention", heads="qwen2.5-14b", dtype="bf16", page=64, seqs=6, new=1024,
             ctx=9001, window=0, sinks=False),
        # a batched step of a full-attention gpt-oss layer: decoding sessions and one prompt's chunk together
        dict(name="step-mixed", kind="step", heads="gpt-oss", dtype="bf16", page=16, seqs=25, new=400, ctx=3500,
             window=0, sinks=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "read", "attention", "attention", "attention", "attention", "step"])
    heads = rng.choice(sorted(HEADS))
    c = dict(kind=kind, heads=heads, dtype=rng.choice(["f32", "bf16"]), page=rng.choice([16, 32, 48, 64, 128]))
    if kind in ("append", "read"):
        c["seqs"] = _log(rng, 1, 200)
        c["new"] = _log(rng, 1, max(1, min(8000, 12000 // c["seqs"])))
        c["ctx"] = max(c["new"], _log(rng, 1, MOST if kind == "append" else 8000))
        return c
    if kind == "attention" and rng.random() < 0.6:
        c["seqs"], c["new"] = _log(rng, 1, 256), 1
        c["ctx"] = _log(rng, 1, min(MOST, 300000 // c["seqs"]))
    else:
        c["seqs"] = rng.randint(1, 8)
        c["new"] = _log(rng, 2, 1000 // c["seqs"] + 24)
        c["ctx"] = max(c["new"], _log(rng, 16, 8000))
    c["window"] = rng.choice([0, 0, 128, _log(rng, 1, 2000)])
    c["sinks"] = heads == "gpt-oss" or rng.random() < 0.2
    return c


# ---- what the layout says ----------------------------------------------------------
def _groups(dim):
    return 2 if dim <= 64 else 4 if dim <= 128 else 8


def _half_t(c):
    return torch.float32 if c["dtype"] == "f32" else torch.bfloat16


def _lengths(c):
    """Tokens in the cache and new tokens of each session (host ints): part of
    the case, the same whatever its inputs' seed."""
    n, ctx, new = c["seqs"], c["ctx"], c["new"]
    gen = torch.Generator().manual_seed(1)
    if n == 1:
        return [ctx], [new]
    at = torch.rand(n, generator=gen)
    q = [max(1, int(new * (0.3 + 0.7 * float(a)))) for a in at]
    if c["kind"] == "step":  # one session's chunk, the others decode
        q = [new] + [1] * (n - 1)
    q[0] = new
    kv = [max(q[i], int(ctx * (0.15 + 0.85 * float(b)))) for i, b in enumerate(torch.rand(n, generator=gen))]
    kv[0] = ctx
    if c["kind"] == "read":
        q = [min(a, b) for a, b in zip(q, kv)]
    return kv, q


def _rope_tables(heads):
    hd = HEADS[heads][2]
    inv = (1.0 / THETA[heads] ** (torch.arange(0, hd, 2, dtype=torch.float64, device=DEV) / hd)).float()
    ang = torch.arange(MOST, dtype=torch.float64, device=DEV)[:, None] * inv.double()
    return ang.cos().float(), ang.sin().float()


def _quantize(x):
    """Codes [.., 32] (0..15) and half scales [..] of groups of 32 f32 values."""
    top, low = x.amax(-1), x.amin(-1)
    d = (torch.where(top >= -low, top, low) * -0.125).clamp(-8188.0, 8188.0).half()
    r = torch.where(d == 0, torch.zeros_like(top), 1.0 / d.float())
    return ((x * r[..., None]).round().clamp(-8.0, 7.0).nan_to_num(0.0) + 8.0).to(torch.uint8), d


def _parts(s, which):
    """Strided views of a pool: codes and scales by page and kv head."""
    c, pool = s["case"], s["k_pages" if which == "k" else "v_pages"]
    _, n_kv, hd, _ = HEADS[c["heads"]]
    g, ps = _groups(hd), c["page"]
    pool = pool.view(-1, n_kv, ps * 18 * g)
    codes, scales = pool[:, :, :ps * 16 * g], pool[:, :, ps * 16 * g:].view(torch.float16).unflatten(-1, (ps, g))
    if which == "k":
        return codes.unflatten(-1, (ps, 4, g, 4)), scales
    return codes.unflatten(-1, (ps // 4, 16, 4, g)), scales


def _store(s, which, x, page, off):
    """Rows [n][kv head][channel] (f32) into the pool at (page, off)."""
    n, n_kv, hd = x.shape
    g = _groups(hd)
    q, d = _quantize(torch.nn.functional.pad(x, (0, 32 * g - hd)).view(n, n_kv, g, 32))
    codes, scales = _parts(s, which)
    if which == "k":
        q = q.view(n, n_kv, g, 4, 4, 2)
        codes[page, :, off] = (q[..., 0] | (q[..., 1] << 4)).transpose(2, 3)
    else:
        codes[page, :, off // 4, :, off % 4] = (q[..., :16] | (q[..., 16:] << 4)).transpose(2, 3)
    scales[page, :, off] = d


def _load(s, which, page, off):
    """Rows [..][kv head][channel] (f32) of the pool at (page, off)."""
    _, n_kv, hd, _ = HEADS[s["case"]["heads"]]
    g = _groups(hd)
    codes, scales = _parts(s, which)
    lead = page.shape
    page, off = page.reshape(-1), off.reshape(-1)
    if which == "k":
        q = codes[page, :, off].transpose(2, 3)
        q = torch.stack((q & 15, q >> 4), -1).reshape(-1, n_kv, g, 32)
    else:
        q = codes[page, :, off // 4, :, off % 4].transpose(2, 3)
        q = torch.cat((q & 15, q >> 4), -1)
    x = (q.float() - 8.0) * scales[page, :, off].float()[..., None]
    return x.reshape(*lead, n_kv, 32 * g)[..., :hd]


# ---- inputs ------------------------------------------------------------------------
def prepare(case, seed):
    c = dict(case)
    n_heads, n_kv, hd, neox = HEADS[c["heads"]]
    t = _half_t(c)
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kv, q = _lengths(c)
    g, ps = _groups(hd), c["page"]
    pages = [-(-n // ps) for n in kv]
    n_pages, stride = sum(pages) + 3, max(pages) + 1
    table = torch.full((len(kv), stride), -1, dtype=torch.int32)
    order = torch.randperm(n_pages, generator=host).int()
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n in q:
        starts.append(starts[-1] + n)
    n_tok = starts[-1]
    randn = lambda *shape: torch.randn(*shape, generator=gen, device=DEV)  # noqa: E731
    s = {"case": c, "table": table.to(DEV), "kv_lens": torch.tensor(kv, dtype=torch.int32, device=DEV),
         "q_starts": torch.tensor(starts, dtype=torch.int32, device=DEV), "n_tok": n_tok, "max_q": max(q),
         "max_kv": max(kv), "q": (1.5 * randn(n_tok, n_heads, hd)).to(t)}
    size = n_pages * n_kv * ps * 18 * g
    s["k_pages"] = torch.zeros(size, dtype=torch.uint8, device=DEV)
    s["v_pages"] = torch.zeros(size, dtype=torch.uint8, device=DEV)
    spread = (0.4 * randn(n_kv, hd)).exp()  # keys' channels differ in size
    if c["kind"] != "append":  # the pool's pages hold earlier tokens
        for lo in range(0, n_pages, 65536 // ps):
            hi = min(n_pages, lo + 65536 // ps)
            page = torch.arange(lo, hi, device=DEV).repeat_interleave(ps)
            off = torch.arange(ps, device=DEV).repeat(hi - lo)
            _store(s, "k", randn(page.numel(), n_kv, hd) * spread, page, off)
            _store(s, "v", 0.5 * randn(page.numel(), n_kv, hd), page, off)
    if c["kind"] in ("append", "step"):
        s["k"] = (randn(n_tok, n_kv, hd) * spread).to(t)
        s["v"] = (0.5 * randn(n_tok, n_kv, hd)).to(t)
        s["q_rot"] = torch.empty_like(s["q"])
        s["cos"], s["sin"] = _rope_tables(c["heads"])
    if c["kind"] in ("append", "read"):
        s["k_out"] = torch.empty(n_tok, n_kv, hd, dtype=t, device=DEV)
        s["v_out"] = torch.empty_like(s["k_out"])
    else:
        s["out"] = torch.empty_like(s["q"])
        s["sinks"] = randn(n_heads) * 2 if c["sinks"] else None
    if own:
        from rustyllm_amd import hip
        s["hip"] = hip
        s["cache"] = hip.PagedKv(s["k_pages"], s["v_pages"], n_pages, ps, n_kv, hd)
        s["batch"] = hip.PagedBatch(s["table"], s["kv_lens"], s["q_starts"], s["max_q"], s["max_kv"])
        if "out" in s:
            s["workspace"] = torch.empty(hip.paged_attention_workspace(s["cache"], s["batch"], n_tok, n_heads),
                                         dtype=torch.uint8, device=DEV)
    return s


# ---- one pass ------------------------------------------------------------------------
def _rows(s):
    """Session, position, page and place in it of every new token."""
    starts, ps = s["q_starts"], s["case"]["page"]
    i = torch.arange(s["n_tok"], device=DEV)
    seq = torch.searchsorted(starts[1:], i.int(), right=True)
    pos = s["kv_lens"][seq] - starts[seq + 1] + i
    return seq, pos, s["table"][seq, pos // ps].long(), pos % ps


def _rotate(x, cos, sin, neox):
    x = x.float()
    if neox:
        a, b = x.chunk(2, -1)
    else:
        a, b = x[..., 0::2], x[..., 1::2]
    u, w = a * cos - b * sin, a * sin + b * cos
    return torch.cat((u, w), -1) if neox else torch.stack((u, w), -1).flatten(-2)


def _append(s):
    neox = HEADS[s["case"]["heads"]][3]
    _, pos, page, off = _rows(s)
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    _store(s, "k", _rotate(s["k"], cos, sin, neox), page, off)
    _store(s, "v", s["v"].float(), page, off)
    return _rotate(s["q"], cos, sin, neox).to(s["q"].dtype)


def _read(s):
    _, _, page, off = _rows(s)
    t = _half_t(s["case"])
    return _load(s, "k", page, off).to(t), _load(s, "v", page, off).to(t)


def _attention(s, q):
    c = s["case"]
    n_heads, n_kv, hd, _ = HEADS[c["heads"]]
    n, most_q, most_kv = c["seqs"], s["max_q"], s["max_kv"]
    starts, kv = s["q_starts"].long(), s["kv_lens"].long()
    q_len = starts[1:] - starts[:-1]
    key = torch.arange(most_kv, device=DEV)
    page = s["table"][:, key // c["page"]].long()
    off = (key % c["page"]).expand(n, -1)
    k = _load(s, "k", page.clamp(min=0), off)
    v = _load(s, "v", page.clamp(min=0), off)
    i = torch.arange(most_q, device=DEV)
    rows = (starts[:-1, None] + i).clamp(max=s["n_tok"] - 1)
    q = q.float()[rows].view(n, most_q, n_kv, n_heads // n_kv, hd).permute(0, 2, 1, 3, 4)
    q = q.reshape(n, n_kv, -1, hd)
    pos = (kv - q_len)[:, None] + i
    ok = (key <= pos[..., None]) & (page >= 0)[:, None] & (i < q_len[:, None])[..., None]
    if c["window"]:
        ok &= key > pos[..., None] - c["window"]
    w = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()).view(n, n_kv, most_q, -1, most_kv) * hd ** -0.5
    w = w.masked_fill(~ok[:, None, :, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    if c["sinks"]:
        sink = s["sinks"].view(1, n_kv, 1, -1, 1)
        top = torch.maximum(top, sink)
    top = top.masked_fill(top == -math.inf, 0.0)
    w = (w - top).exp()
    total = w.sum(-1, keepdim=True)
    if c["sinks"]:
        total = total + (sink - top).exp()
    out = torch.matmul(w.view(n, n_kv, -1, most_kv), v.permute(0, 2, 1, 3).contiguous())
    out = out.view(n, n_kv, most_q, -1, hd) / total.clamp(min=1e-30)
    out = out.permute(0, 2, 1, 3, 4).reshape(n, most_q, n_heads, hd)
    at = torch.arange(s["n_tok"], device=DEV)
    seq = torch.searchsorted(s["q_starts"][1:], at.int(), right=True)
    return out[seq, at - starts[seq]].to(_half_t(c))


def run(s):
    c = s["case"]
    kind = c["kind"]
    if own:
        hip, cache, batch = s["hip"], s["cache"], s["batch"]
        q = s["q"]
        if kind in ("append", "step"):
            assert hip.paged_append_dev(cache, batch, s["k"], s["v"], s["cos"], s["sin"], q=q, q_out=s["q_rot"],
                                        neox=HEADS[c["heads"]][3])
            q = s["q_rot"]
        if kind in ("append", "read"):
            assert hip.paged_read_dev(cache, batch, s["k_out"], s["v_out"])
            return {"k": s["k_out"], "v": s["v_out"]} | ({"q": q} if kind == "append" else {})
        assert hip.paged_attention_dev(cache, batch, q, s["out"], q.shape[-1] ** -0.5, s["workspace"],
                                       sinks=s["sinks"], window=c["window"])
        return {"out": s["out"]}
    if kind == "append":
        q = _append(s)
        k, v = _read(s)
        return {"k": k, "v": v, "q": q}
    if kind == "read":
        k, v = _read(s)
        return {"k": k, "v": v}
    return {"out": _attention(s, _append(s) if kind == "step" else s["q"])}


# ---- what a pass cannot do without ---------------------------------------------------
def work(case):
    c = dict(case)
    n_heads, n_kv, hd, _ = HEADS[c["heads"]]
    item = 4 if c["dtype"] == "f32" else 2
    kv, q = _lengths(c)
    n = sum(q)
    row = n_kv * hd * 9 / 16  # codes and scales of one token's keys, or values
    if c["kind"] == "read":
        return {"bytes": n * (2 * row + 2 * n_kv * hd * item), "flops": 2.0 * n * n_kv * hd}
    moved = n * (2 * row + (2 * n_heads + 2 * n_kv) * hd * item + 4 * hd)  # q in and out, k, v, rows stored, angles
    if c["kind"] == "append":
        return {"bytes": moved + n * (2 * row + 2 * n_kv * hd * item), "flops": n * (6.0 * n_heads + 14 * n_kv) * hd}
    pairs = seen = 0
    for a, b in zip(kv, q):
        w = c["window"] or a
        pairs += sum(min(w, p + 1) for p in range(a - b, a))
        seen += min(a, w + b - 1)
    total = {"bytes": seen * 2 * row + 2 * n * n_heads * hd * item, "flops": 4.0 * pairs * n_heads * hd}
    if c["kind"] == "step":
        total = {"bytes": total["bytes"] + moved, "flops": total["flops"] + n * (6.0 * n_heads + 14 * n_kv) * hd}
    return total


# ---- the definition in 64 bits --------------------------------------------------------
def _exact_rows(s, which, page, off):
    """Stored values by the layout's byte addresses, [..][kv head][channel]."""
    c = s["case"]
    _, n_kv, hd, _ = HEADS[c["heads"]]
    g, ps = _groups(hd), c["page"]
    pool = s["k_pages" if which == "k" else "v_pages"]
    block = (page[..., None] * n_kv + torch.arange(n_kv, device=DEV)) * (ps * 18 * g)
    ch = torch.arange(hd, device=DEV)
    off = off[..., None, None]
    if which == "k":
        place = off * (16 * g) + ((ch % 32) // 8 * g + ch // 32) * 4 + ch % 8 // 2
        shift = ch % 2 * 4
    else:
        place = ((off // 4 * 16 + ch % 16) * 4 + off % 4) * g + ch // 32
        shift = ch % 32 // 16 * 4
    code = (pool[block[..., None] + place].int() >> shift) & 15
    d = pool.view(torch.float16)[(block[..., None] + ps * 16 * g) // 2 + off * g + ch // 32]
    return (code - 8).double() * d.double()


def _exact_codes(x):
    """Values that a row (f64, already of f32) is stored as: the scale rounded to
    half, its inverse and the quotient to f32, the code to the nearest integer."""
    hd = x.shape[-1]
    out = torch.empty_like(x)
    for lo in range(0, hd, 32):
        part = x[..., lo:lo + 32]
        big = part.abs().amax(-1, keepdim=True)
        sign = torch.where((part == big).any(-1, keepdim=True), 1.0, -1.0)
        d = (-big * sign / 8).clamp(-8188, 8188).float().half().double()
        inv = torch.where(d == 0, 0.0, 1.0 / d).float().double()
        code = (part * inv).float().double().round().clamp(-8, 7)
        out[..., lo:lo + 32] = code * d
    return out


def _exact_rotated(x, cos, sin, neox, rounded):
    """`rounded`: each product and each sum to f32, as a key is defined."""
    keep = (lambda y: y.float().double()) if rounded else (lambda y: y)
    x, h = x.double(), x.shape[-1] // 2
    out = torch.empty_like(x)
    for p in range(h):
        i, j = (p, p + h) if neox else (2 * p, 2 * p + 1)
        co, si = cos[:, p, None].double(), sin[:, p, None].double()
        out[..., i] = keep(keep(x[..., i] * co) - keep(x[..., j] * si))
        out[..., j] = keep(keep(x[..., i] * si) + keep(x[..., j] * co))
    return out


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    c = s["case"]
    n_heads, n_kv, hd, neox = HEADS[c["heads"]]
    starts, kv, table, ps = s["q_starts"].tolist(), s["kv_lens"].tolist(), s["table"].long(), c["page"]
    pos = torch.cat([torch.arange(kv[i] - (b - a), kv[i]) for i, (a, b) in enumerate(zip(starts, starts[1:]))]).to(DEV)
    seq = torch.cat([torch.full((b - a,), i) for i, (a, b) in enumerate(zip(starts, starts[1:]))]).to(DEV)
    if c["kind"] == "read":
        page, off = table[seq, pos // ps], pos % ps
        return {"k": _exact_rows(s, "k", page, off), "v": _exact_rows(s, "v", page, off)}
    q, new_k, new_v = s["q"].double(), None, None
    if "cos" in s:
        cos, sin = s["cos"][pos], s["sin"][pos]
        q = _exact_rotated(s["q"], cos, sin, neox, False)
        new_k = _exact_codes(_exact_rotated(s["k"], cos, sin, neox, True))
        new_v = _exact_codes(s["v"].double())
    if c["kind"] == "append":
        return {"k": new_k, "v": new_v, "q": q}
    if new_k is not None:
        q = q.to(_half_t(c)).double()  # attention is given the rotated queries as they are stored
    out = torch.zeros(s["n_tok"], n_heads, hd, dtype=torch.float64, device=DEV)
    for i, (a, b) in enumerate(zip(starts, starts[1:])):
        last = kv[i] - (b - a)
        first = max(0, last - c["window"] + 1) if c["window"] else 0
        at = torch.arange(first, kv[i], device=DEV)
        page, off = table[i, at // ps], at % ps
        k, v = _exact_rows(s, "k", page, off), _exact_rows(s, "v", page, off)
        if new_k is not None:
            k[last - first:], v[last - first:] = new_k[a:b], new_v[a:b]
        p = torch.arange(last, kv[i], device=DEV)[:, None]
        hide = (at > p) | ((at <= p - c["window"]) if c["window"] else torch.zeros_like(at > p))
        for h in range(n_heads):
            j = h * n_kv // n_heads
            w = (q[a:b, h] @ k[:, j].T.contiguous()) / math.sqrt(hd)
            w = w.masked_fill(hide, -math.inf)
            if c["sinks"]:
                w = torch.cat((w, s["sinks"][h].double().expand(b - a, 1)), 1)
            out[a:b, h] = torch.softmax(w, 1)[:, :at.numel()] @ v[:, j].contiguous()
    return {"out": out}
