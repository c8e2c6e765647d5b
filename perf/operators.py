"""Measured cases of the paged KV cache: appending keys and values (head norms and position rotation applied on the
way, cache held in f16 or in 4 bits) and the attention that reads it (sliding window and sink slots, one query row a
sequence or several).

Every case is one pass through one of the two operators:
  "append"  rows of q|k|v -> rotated q, keys and values in the pages; what the pages then stand for is read back.
  "attn"    q rows against the pages -> o and the logarithm of the softmax sum.

The page layout (include/e4b_b200.h, e4b_paged_kv): a page holds `page` slots of every KV head; a head's slots come in
pieces of 16, and inside a piece the elements are ordered for the matrix unit's operands.  _order() gives that order.
"""
import importlib
import math
import random

import torch

own = False

F64, F32, F16 = torch.float64, torch.float32, torch.float16


# ------------------------------------------------------------------ cases
def _case(name, op, qh, kvh, hd, bits, page, nseq, lo, hi, rows=1, window=0, sinks=0, half=0, keqv=0, norm=1, frac=1.0,
          theta=10000.0, out="f16", lens_seed=1):
    """lo..hi: tokens cached before the pass, spread over the logarithm; rows: new tokens a sequence, 1 or 1..rows."""
    c = dict(op=op, qh=qh, kvh=kvh, hd=hd, bits=bits, page=page, nseq=nseq, lo=lo, hi=hi, rows=rows, lens_seed=lens_seed)
    if op == "append":
        c.update(half=half, keqv=keqv, norm=norm, frac=frac, theta=theta)
    else:
        c.update(window=window, sinks=sinks, out=out)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # one new token of one conversation, the smallest model's heads: all latency
        _case("append one token", "append", 4, 1, 128, 4, 16, 1, 100, 100),
        # a decode step of 64 conversations of unequal length, 4-bit cache, the MoE model's heads
        _case("append 64 tokens", "append", 16, 4, 256, 4, 64, 64, 1, 4000),
        # prompts of unequal length entering a 4-bit cache behind a shared prefix: the ordinary prefill of a server
        _case("append prompts 4 bit", "append", 16, 4, 256, 4, 64, 16, 1, 2000, rows=1000),
        # f16 projections of a layer whose values are its keys (a quarter of the pairs rotates) into an f16 cache, far positions
        _case("append prompts f16", "append", 16, 4, 256, 16, 32, 8, 1000, 100000, rows=500, half=1, keqv=1, frac=0.25,
              theta=1000000.0),
        # one conversation on a sliding layer of the dense model: latency
        _case("attn one token", "attn", 8, 2, 256, 16, 16, 1, 551, 551, window=512),
        # the decode step of the MoE benchmark point: 64 conversations after a prompt of 1024
        _case("attn 64 tokens", "attn", 16, 4, 256, 4, 64, 64, 1034, 1034),
        # a sliding layer with sinks, conversations from one token to long ones, f16 cache
        _case("attn sinks f16", "attn", 16, 4, 256, 16, 32, 64, 1, 8000, window=1024, sinks=4),
        # one very long document, two KV heads: few rows, the axis has to be split
        _case("attn long", "attn", 8, 2, 256, 4, 128, 1, 131000, 131000),
        # small heads, ragged lengths, a window with sinks over the 4-bit cache
        _case("attn ragged", "attn", 4, 1, 128, 4, 16, 48, 0, 16000, window=4096, sinks=17, out="f32"),
        # speculated or chunked rows: several queries a sequence behind a 4-bit cache
        _case("attn chunk 4 bit", "attn", 16, 4, 256, 4, 64, 8, 300, 4000, rows=64, window=1024, sinks=16),
        # a prompt chunk with one query head a KV head, f16 cache
        _case("attn chunk f16", "attn", 8, 8, 64, 16, 16, 2, 1, 1500, rows=250),
        # a full server: 32 long conversations, 4-bit cache
        _case("attn 32 long", "attn", 16, 4, 256, 4, 64, 32, 8000, 16000),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    hd = rng.choice([64, 128, 256])
    kvh = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 3, 4, 4, 4, 5, 8])
    bits = rng.choice([4, 4, 16])
    page = rng.choice([16, 32, 48, 64, 128])
    common = dict(qh=kvh * group, kvh=kvh, hd=hd, bits=bits, page=page, lens_seed=rng.randrange(1 << 30))
    if rng.random() < 0.4:
        rows = rng.choice([1, 1, _log_int(rng, 2, 1000)])
        width = (kvh * group + 2 * kvh) * hd * max(1, rows // 2)
        nseq = _log_int(rng, 1, max(1, min(128, 40_000_000 // width)))
        return _case(None, "append", nseq=nseq, lo=rng.choice([0, 1, 50]), hi=_log_int(rng, 100, 30000), rows=rows,
                     half=rng.choice([0, 1]), keqv=rng.choice([0, 0, 1]), norm=rng.choice([0, 1, 1]),
                     frac=rng.choice([1.0, 0.5, 0.25]), theta=rng.choice([10000.0, 1000000.0]), **common)
    rows = rng.choice([1, 1, 1, _log_int(rng, 2, 128)])
    hi = _log_int(rng, 40, 40000 if rows == 1 else 4000)
    most = min(32 * 10000 * 4 * 256 * 4 // (hi * kvh * hd * bits), 8 * 2000 * 32 * 16 // (hi * kvh * group * rows))
    nseq = _log_int(rng, 1, max(1, min(96, most)))
    window = rng.choice([0, 0, _log_int(rng, 1, hi), 1024])
    return _case(None, "attn", nseq=nseq, lo=rng.choice([0, 1, max(1, hi // 4), hi]), hi=hi, rows=rows, window=window,
                 sinks=rng.choice([0, 1, 4, 16, 33]) if window else 0, out=rng.choice(["f16", "f16", "f32"]), **common)


def _lengths(case):
    """Tokens cached before the pass and rows of the pass, for each sequence: the same for every seed."""
    rng = random.Random(case["lens_seed"])
    lo, hi, n = case["lo"], case["hi"], case["nseq"]
    lens = [int((lo + 1) * ((hi + 1) / (lo + 1)) ** rng.random()) - 1 if lo < hi else lo for _ in range(n)]
    rows = [rng.randint(1, case["rows"]) if case["rows"] > 1 else 1 for _ in range(n)]
    return lens, rows


def _piece_bytes(case):
    return 32 * case["hd"] if case["bits"] == 16 else 9 * case["hd"]


# ------------------------------------------------------------------ page layout
def _order(case, value):
    """The order of a 16-slot piece's elements (f16 cache) or of its groups of four 4-bit codes: sizes of the stored
    axes, and the permutation that brings them to (slot..., dim...)."""
    hd = case["hd"]
    if case["bits"] == 16:
        if value:  # [64-dim group][slot/8][slot%2][8-dim group][slot/2%4][8 dims]
            return (hd // 64, 2, 2, 8, 4, 8), (1, 4, 2, 0, 3, 5)
        return (hd // 32, 16, 32), (1, 0, 2)  # [32-dim block][slot][32 dims]
    if value:  # [slot/8][slot%2][4-dim group of a block][slot/2%4][block]
        return (2, 2, 8, 4, hd // 32), (0, 3, 1, 4, 2)
    nb = min(4, hd // 32)  # [run of nb blocks][slot][8-dim group of a block][block of the run][half of it]
    return (hd // 32 // nb, 16, 4, nb, 2), (1, 0, 3, 2, 4)


def _pack(case, codes, value):
    """codes [..., 16, n] (f16 bits, or four 4-bit codes to an int16; n = HD or HD/4) -> the stored order, flat."""
    sizes, perm = _order(case, value)
    lead = codes.shape[:-2]
    x = codes.reshape(*lead, *[sizes[p] for p in perm])
    k = len(lead)
    back = [perm.index(i) for i in range(len(perm))]
    return x.permute(*range(k), *[k + b for b in back]).reshape(*lead, -1)


def _unpack(case, flat, value):
    sizes, perm = _order(case, value)
    lead = flat.shape[:-1]
    k = len(lead)
    return flat.reshape(*lead, *sizes).permute(*range(k), *[k + p for p in perm]).reshape(*lead, 16, -1)


def _values(case, pieces, value):
    """Pieces as stored, int16 [..., piece bytes / 2] -> f32 [..., 16, HD]."""
    hd = case["hd"]
    if case["bits"] == 16:
        return _unpack(case, pieces, value).contiguous().view(F16).float()
    scale = pieces[..., : hd // 2]
    if value:
        scale = scale.unflatten(-1, (4, hd // 32, 2, 2)).movedim(-2, -4).transpose(-1, -2).flatten(-4)
    scale = scale.contiguous().view(F16).float().reshape(*pieces.shape[:-1], 16, hd // 32, 1)
    quads = _unpack(case, pieces[..., hd // 2:], value).int()
    codes = torch.stack([(quads >> (4 * i)) & 15 for i in range(4)], -1).float() - 8.0
    return (codes.reshape(*codes.shape[:-2], hd // 32, 32) * scale).reshape(*codes.shape[:-2], hd)


# ------------------------------------------------------------------ inputs
def _page_table(case, lens, rows, g):
    """Pages of the pool in random order; the entries past a sequence's end name no page."""
    need = [-(-(a + b) // case["page"]) for a, b in zip(lens, rows)]
    width, total = max(need), sum(need)
    order = torch.randperm(total, generator=g, device="cuda").int()
    table = torch.full((case["nseq"], width), -1, dtype=torch.int32, device="cuda")
    at = torch.arange(width, device="cuda")[None] < torch.tensor(need, device="cuda")[:, None]
    table[at] = order
    return table, total


def _full_pool(case, n_pages, value, g):
    """A cache of normally distributed keys or values."""
    n = n_pages * case["kvh"] * case["page"] // 16
    hd = case["hd"]
    if case["bits"] == 16:
        return torch.randn((n, 16 * hd), generator=g, device="cuda").half().view(torch.int16).reshape(-1)
    scale = (0.25 + 0.05 * torch.rand((n, hd // 2), generator=g, device="cuda")).half()
    sign = torch.randint(0, 2, scale.shape, generator=g, device="cuda") * 2 - 1
    quads = torch.zeros((n, 16, hd // 4), dtype=torch.int32, device="cuda")
    for i in range(4):
        quads |= (torch.randn(quads.shape, generator=g, device="cuda") * 3.6 + 8).round().clamp(0, 15).int() << (4 * i)
    quads = _pack(case, quads, value)
    return torch.cat([(scale * sign).view(torch.int16), quads.to(torch.int16)], 1).reshape(-1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    lens, rows = _lengths(case)
    n, (qh, kvh, hd) = sum(rows), (case["qh"], case["kvh"], case["hd"])
    table, n_pages = _page_table(case, lens, rows, g)
    first = [sum(rows[:i]) for i in range(len(rows) + 1)]
    s = dict(case=case, n=n, n_pages=n_pages, table=table, max_len=max(a + b for a, b in zip(lens, rows)), max_rows=max(rows),
             lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
             first=torch.tensor(first, dtype=torch.int32, device="cuda"))
    if case["op"] == "append":
        words = n_pages * kvh * case["page"] // 16 * _piece_bytes(case) // 2
        s["k"], s["v"] = (torch.zeros(words, dtype=torch.int16, device="cuda") for _ in range(2))
        width = (qh + kvh * (1 if case["keqv"] else 2)) * hd
        s["qkv"] = torch.randn((n, width), generator=g, device="cuda").to(F16 if case["half"] else F32)
        s["qw"], s["kw"] = (1 + 0.15 * torch.randn(hd, generator=g, device="cuda") for _ in range(2))
        s["q_out"] = torch.empty((n, qh, hd), dtype=F32, device="cuda")
        s["k_out"], s["v_out"] = (torch.empty((n, kvh, hd), dtype=F16, device="cuda") for _ in range(2))
    else:
        s["k"], s["v"] = _full_pool(case, n_pages, False, g), _full_pool(case, n_pages, True, g)
        s["q"] = torch.randn((n, qh, hd), generator=g, device="cuda") * (2.0 / math.sqrt(hd))
        s["out"] = torch.empty((n, qh, hd), dtype=F16 if case["out"] == "f16" else F32, device="cuda")
        s["lse"] = torch.empty((n, qh), dtype=F32, device="cuda")
        s["scratch"] = torch.zeros(1 << 23, dtype=torch.uint8, device="cuda")
    return s


# ------------------------------------------------------------------ plain forms
def _row_places(s):
    """Sequence and position of every row of the pass."""
    r = torch.arange(s["n"], device="cuda")
    seq = torch.searchsorted(s["first"].long(), r, right=True) - 1
    return seq, s["lens"].long()[seq] + r - s["first"].long()[seq]


def _plain_append(s):
    case = s["case"]
    qh, kvh, hd, half = case["qh"], case["kvh"], case["hd"], case["hd"] // 2
    seq, pos = _row_places(s)
    x = s["qkv"].double().reshape(s["n"], -1, hd)
    q, k = x[:, :qh], x[:, qh:qh + kvh]
    v = k if case["keqv"] else x[:, qh + kvh:]
    if case["norm"]:
        q, k, v = (t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt() for t in (q, k, v))
        q, k = q * s["qw"].double(), k * s["kw"].double()
    turn = int(case["frac"] * half)
    freq = torch.pow(torch.tensor(case["theta"], dtype=F64, device="cuda"), torch.arange(turn, device="cuda").double() * (-2.0 / hd))
    angle = pos[:, None, None] * freq
    cos, sin = angle.cos(), angle.sin()

    def rotated(t):
        a, b = t[..., :turn], t[..., half:half + turn]
        return torch.cat([a * cos - b * sin, t[..., turn:half], a * sin + b * cos, t[..., half + turn:]], -1)

    q, k = rotated(q).float(), rotated(k).half()
    v = v.half()
    piece = ((s["table"].long()[seq, pos // case["page"]] * kvh)[:, None] + torch.arange(kvh, device="cuda")) * (
        case["page"] // 16) + (pos % case["page"] // 16)[:, None]
    return q, _store(s, s["k"], piece, pos % 16, k, False), _store(s, s["v"], piece, pos % 16, v, True)


def _store(s, pool, piece, slot, x, value):
    """Writes rows x [n, KVH, HD] (f16) into the pages and gives what the pages then hold for them."""
    case, hd = s["case"], s["case"]["hd"]
    words = _piece_bytes(case) // 2
    units = torch.arange(16 * (hd if case["bits"] == 16 else hd // 4), device="cuda").reshape(16, -1)
    where = torch.empty_like(units).reshape(-1)
    where[_pack(case, units, value)] = units.reshape(-1)  # the word at which the piece holds (slot, unit)
    at = piece[..., None] * words + where.reshape(16, -1)[slot][:, None]
    if case["bits"] == 16:
        pool[at] = x.view(torch.int16)
        return pool[at].view(F16)
    blocks = x.float().reshape(*x.shape[:-1], hd // 32, 32)
    top = blocks.gather(-1, blocks.abs().argmax(-1, keepdim=True))
    d = top / -8.0
    codes = torch.where(d == 0, 8.0, (blocks / torch.where(d == 0, 1.0, d) + 8.5).trunc().clamp(0, 15)).int()
    quads = codes.reshape(*x.shape[:-1], hd // 4, 4) << torch.tensor([0, 4, 8, 12], device="cuda")
    block = torch.arange(hd // 32, device="cuda")
    at_d = (slot // 2 % 4 * (hd // 8) + slot // 8 * 2 + slot % 2)[:, None, None] + 4 * block if value else (
        slot * (hd // 32))[:, None, None] + block
    at_d = piece[..., None] * words + at_d
    pool[at + hd // 2] = quads.sum(-1).to(torch.int16)
    pool[at_d] = d.half().view(torch.int16).squeeze(-1)
    got = (pool[at + hd // 2].int()[..., None] >> torch.tensor([0, 4, 8, 12], device="cuda")) & 15
    return ((got.reshape(blocks.shape).float() - 8.0) * pool[at_d].view(F16).float()[..., None]).reshape(x.shape).half()


def _plain_attn(s):
    case = s["case"]
    qh, kvh, hd, nseq = case["qh"], case["kvh"], case["hd"], case["nseq"]
    n_piece, words = case["page"] // 16, _piece_bytes(case) // 2
    pages = s["table"].long().clamp(min=0)

    def cached(pool, value):  # [nseq, KVH, slots, HD]
        p = pool.reshape(s["n_pages"], kvh, n_piece, words)[pages]
        return _values(case, p, value).permute(0, 2, 1, 3, 4, 5).reshape(nseq, kvh, -1, hd)

    seq, pos = _row_places(s)
    row = torch.arange(s["n"], device="cuda") - s["first"].long()[seq]
    q = torch.zeros((nseq, s["max_rows"], qh, hd), device="cuda")
    q[seq, row] = s["q"]
    q = q.reshape(nseq, -1, kvh, qh // kvh, hd).permute(0, 2, 3, 1, 4).reshape(nseq, kvh, -1, hd)
    score = q @ cached(s["k"], False).transpose(-1, -2)
    slot = torch.arange(score.shape[-1], device="cuda")
    at = s["lens"].long()[:, None] + torch.arange(s["max_rows"], device="cuda")
    seen = slot <= at[..., None]
    if case["window"]:
        seen &= (slot > at[..., None] - case["window"]) | (slot < case["sinks"])
    score = score.reshape(nseq, kvh, qh // kvh, s["max_rows"], -1).masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    # slots that no query sees hold what was there before
    v = cached(s["v"], True)
    v = torch.where(seen.any(1)[:, None, :, None], v, torch.zeros((), device="cuda"))
    o = (p.reshape(nseq, kvh, -1, p.shape[-1]) @ v).reshape(nseq, kvh, qh // kvh, s["max_rows"], hd) / total
    lse = (top + total.log()).squeeze(-1)
    o = o.permute(0, 3, 1, 2, 4).reshape(nseq, -1, qh, hd)[seq, row]
    return o.to(s["out"].dtype), lse.permute(0, 3, 1, 2).reshape(nseq, -1, qh)[seq, row]


# ------------------------------------------------------------------ the framework's calls
_dev = None


def _own(s):
    """The device context and the cache's handle, as a program holds them."""
    global _dev
    e4b = importlib.import_module("e4b-webgpu_b200")
    if _dev is None:
        _dev = e4b.Device(torch.cuda.current_device())
    c = s["case"]
    s["kv"] = e4b.PagedKV(_dev, BITS=c["bits"], PAGE=c["page"], PAGES=s["n_pages"], MAX_PAGES=s["table"].shape[1], SEQS=c["nseq"],
                          KV_HEADS=c["kvh"], HEAD_DIM=c["hd"], k=s["k"].data_ptr(), v=s["v"].data_ptr(),
                          pages=s["table"].data_ptr(), lens=s["lens"].data_ptr(),
                          rows=s["first"].data_ptr() if c["rows"] > 1 else None)
    s["ops"], s["ptr"] = e4b.ops, {k: t.data_ptr() for k, t in s.items() if isinstance(t, torch.Tensor)}


def run(s):
    c = s["case"]
    if not own:
        if c["op"] == "append":
            q, k, v = _plain_append(s)
            return {"q": q, "k": k, "v": v}
        o, lse = _plain_attn(s)
        return {"o": o, "lse": lse}
    if "kv" not in s:
        _own(s)
    ops, p = s["ops"], s["ptr"]
    if c["op"] == "append":
        ops.headprep_paged(_dev, s["kv"], p["qkv"], p["qw"], p["kw"], p["q_out"], QH=c["qh"],
                           ROPE_ANGLES=int(c["frac"] * (c["hd"] // 2)), THETA=c["theta"], NORM=c["norm"], KEQV=c["keqv"],
                           XF16=c["half"], ROWS=s["n"])
        ops.kvread_paged(_dev, s["kv"], p["k_out"], p["v_out"], ROWS=s["n"])
        return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}
    half = c["out"] == "f16"
    ops.attn_paged(_dev, s["kv"], p["q"], p["out"] if half else None, None if half else p["out"], p["lse"], p["scratch"],
                   Q_HEADS=c["qh"], WINDOW=c["window"], SINKS=c["sinks"], ROWS=s["n"])
    return {"o": s["out"], "lse": s["lse"]}


# ------------------------------------------------------------------ what a pass cannot do without
def _seen(case, lens, rows):
    """Slots that some row of a sequence sees, and pairs of a row and a slot that it sees, over all sequences."""
    slots = pairs = 0
    for a, b in zip(lens, rows):
        w, t = case["window"], case["sinks"]
        if not w:
            slots += a + b
            pairs += b * a + b * (b + 1) // 2
            continue
        slots += a + b - max(0, max(0, a + 1 - w) - t)
        pairs += sum(min(p + 1, w) + min(max(0, p + 1 - w), t) for p in range(a, a + b))
    return slots, pairs


def work(case):
    lens, rows = _lengths(case)
    n, qh, kvh, hd = sum(rows), case["qh"], case["kvh"], case["hd"]
    row = 2 * kvh * _piece_bytes(case) // 16  # a token's keys and values in the cache
    table = 4 * (case["nseq"] * 2 + sum(-(-(a + b) // case["page"]) for a, b in zip(lens, rows)))
    if case["op"] == "append":
        width = (qh + kvh * (1 if case["keqv"] else 2)) * hd
        return {"bytes": n * (width * (2 if case["half"] else 4) + qh * hd * 4 + 2 * row + 2 * kvh * hd * 2) + table,
                "flops": n * (qh + 2 * kvh) * hd * 8}
    slots, pairs = _seen(case, lens, rows)
    return {"bytes": slots * row + n * qh * (hd * (4 + (2 if case["out"] == "f16" else 4)) + 4) + table,
            "flops": pairs * qh * hd * 4}


# ------------------------------------------------------------------ the definition in 64 bits
def _element(case, value):
    """For (slot, dim) of a piece: the int16 word that holds it and the shift of its bits there, by the layout's index
    formulas."""
    hd = case["hd"]
    s = torch.arange(16, device="cuda")[:, None]
    d = torch.arange(hd, device="cuda")[None]
    block, in_block = d // 32, d % 32
    i, t = s // 8 * 2 + s % 2, s // 2 % 4
    if case["bits"] == 16:
        if value:
            return ((((d // 64) * 4 + i) * 8 + d % 64 // 8) * 4 + t) * 8 + d % 8, 0 * (s + d)
        return (block * 16 + s) * 32 + in_block, 0 * (s + d)
    if value:
        return hd // 2 + ((i * 8 + in_block // 4) * 4 + t) * (hd // 32) + block, 4 * (in_block % 4) + 0 * s
    nb = min(4, hd // 32)
    return hd // 2 + ((((block // nb) * 16 + s) * 4 + in_block // 8) * nb + block % nb) * 2 + in_block // 4 % 2, 4 * (in_block % 4) + 0 * s


def _exact_attn(case, s):
    lens, rows = _lengths(case)
    qh, kvh, hd, page = case["qh"], case["kvh"], case["hd"], case["page"]
    words, out, lse, at = _piece_bytes(case) // 2, [], [], 0
    for b, (a, n) in enumerate(zip(lens, rows)):
        pos = torch.arange(a + n, device="cuda")
        piece = (s["table"][b].long()[pos // page][:, None] * kvh + torch.arange(kvh, device="cuda")) * (page // 16) + (pos % page // 16)[:, None]

        def rows_of(pool, value):
            word, shift = _element(case, value)
            got = pool[piece[..., None] * words + word[pos % 16][:, None]]
            if case["bits"] == 16:
                return got.view(F16).double()
            in_piece, block = pos % 16, torch.arange(hd, device="cuda") // 32
            if value:
                at_d = 2 * (in_piece // 8)[:, None] + (in_piece % 2)[:, None] + 4 * (block + (in_piece // 2 % 4)[:, None] * (hd // 32))
            else:
                at_d = in_piece[:, None] * (hd // 32) + block
            d = pool[piece[..., None] * words + at_d[:, None]]
            return d.view(F16).double() * (((got.int() >> shift[pos % 16][:, None].int()) & 15) - 8)

        k, v = rows_of(s["k"], False), rows_of(s["v"], True)
        q = s["q"][at:at + n].double().reshape(n, kvh, qh // kvh, hd)
        here = torch.arange(a, a + n, device="cuda")[:, None]
        hidden = pos[None] > here
        if case["window"]:
            hidden |= (pos[None] <= here - case["window"]) & (pos[None] >= case["sinks"])
        score = torch.einsum("rkgd,skd->rkgs", q, k)
        score[hidden[:, None, None].expand_as(score)] = -math.inf
        lse.append(torch.logsumexp(score, -1).reshape(n, qh))
        out.append(torch.einsum("rkgs,skd->rkgd", torch.softmax(score, -1), v).reshape(n, qh, hd))
        at += n
    return {"o": torch.cat(out), "lse": torch.cat(lse)}


def _exact_append(case, s):
    lens, rows = _lengths(case)
    qh, kvh, hd, half = case["qh"], case["kvh"], case["hd"], case["hd"] // 2
    pos = torch.cat([torch.arange(a, a + n, device="cuda") for a, n in zip(lens, rows)]).double()
    x = s["qkv"].double().reshape(s["n"], -1, hd)
    turn = int(case["frac"] * half)
    phase = torch.polar(torch.ones((), dtype=F64, device="cuda"), pos[:, None] * torch.exp(
        torch.arange(turn, device="cuda").double() * (-2.0 * math.log(case["theta"]) / hd)))

    def head(i, weight, turned):
        t = x[:, i]
        if case["norm"]:
            t = t / torch.sqrt((t * t).sum(-1, keepdim=True) / hd + 1e-6)
            t = t if weight is None else t * weight.double()
        if turned:
            z = torch.complex(t[:, :half].contiguous(), t[:, half:].contiguous())
            z[:, :turn] *= phase
            t = torch.cat([z.real, z.imag], -1)
        return t

    def held(t):
        t = t.half().double()
        if case["bits"] == 16:
            return t
        blocks = t.reshape(s["n"], hd // 32, 32)
        top = torch.where(blocks.amax(-1) > -blocks.amin(-1), blocks.amax(-1), blocks.amin(-1))
        both = blocks.amax(-1) == -blocks.amin(-1)  # the first of the two gives the sign
        lead = blocks.gather(-1, (blocks.abs() == top.abs()[..., None]).int().argmax(-1, keepdim=True)).squeeze(-1)
        d = torch.where(both, lead, top) / -8
        code = torch.floor(blocks / torch.where(d == 0, 1.0, d)[..., None] + 0.5).clamp(-8, 7)
        return (code * d.half().double()[..., None]).reshape(s["n"], hd)

    q = torch.stack([head(i, s["qw"], True) for i in range(qh)], 1)
    k = torch.stack([held(head(qh + i, s["kw"], True)) for i in range(kvh)], 1)
    v = torch.stack([held(head(qh + i if case["keqv"] else qh + kvh + i, None, False)) for i in range(kvh)], 1)
    return {"q": q, "k": k, "v": v}


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_append(case, s) if case["op"] == "append" else _exact_attn(case, s)
