"""The paged 4-bit cache's operators as cases that can be prepared, run and checked: appending rotated keys and
values, reading rows back, and attention over the pages.

A cache is a pool of pages of `page` tokens each, keys and values held as Q4_0 blocks (32 values: an f16 scale d and
32 codes of 4 bits, a code c standing for d (c - 8)). A batch is n_seq sequences with `rows` new tokens each, packed
one after the other: sequence s owns rows starts[s] .. starts[s + 1] - 1, its row j has position past[s] + j, and
position p lies in page pages[s][p / page] at slot p % page.

The pool's bytes: [page][KV head][tile of 32 tokens][36 D bytes]. A tile, for heads of D values, byte i of a token
holding dim i in its low nibble and dim i + D / 2 in its high one:
  keys     16 D bytes  [token][g 4][b D/64][j 8], i = 32 b + 8 g + j
  values   16 D bytes  [t D/64][g 4][c 16][u 2][m 8], token 8 g + m, i = 16 (2 t + u) + c
  key scales, value scales   2 D bytes each, f16 [block D/32][32], token t at 8 (t / 8) + ORDER[t % 8]

`run` computes an operator from elementary torch operations, or, where `own` is set, through the framework.
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

ORDER = (0, 2, 1, 3, 4, 6, 5, 7)  # its own inverse


def listed() -> list[dict]:
    return [
        # One conversation's next token in an 8B-shaped layer: the smallest call, latency alone.
        _append("append_token", H=32, Hkv=8, D=128, page=64, n_seq=1, rows=1, past=(4000, 4000), n_dims=128),
        # A serving step: 64 conversations of very different lengths, one token each.
        _append("append_step", H=32, Hkv=8, D=128, page=64, n_seq=64, rows=1, past=(1, 100000), n_dims=128),
        # Two long prompts entering together (odd lengths) behind a shared-size history.
        _append("append_prompts", H=32, Hkv=8, D=128, page=128, n_seq=2, rows=1999, past=(0, 4096), n_dims=128),
        # Reading back a few draft tokens of a small model's sequences.
        _read("read_drafts", Hkv=2, D=64, page=32, n_seq=5, rows=7, past=(10, 900)),
        # A cached prompt handed over to a contiguous cache: 4096 tokens of one sequence.
        _read("read_prefix", Hkv=8, D=128, page=64, n_seq=1, rows=4096, past=(0, 0)),
        # One conversation's decode step early on: latency.
        _attn("attn_token", H=32, Hkv=8, D=128, page=64, n_seq=1, rows=1, past=(500, 500)),
        # A serving step over 32 conversations, lengths spread from short to 8192.
        _attn("attn_step", H=32, Hkv=8, D=128, page=64, n_seq=32, rows=1, past=(200, 8191)),
        # One very long conversation.
        _attn("attn_long", H=32, Hkv=8, D=128, page=256, n_seq=1, rows=1, past=(131070, 131070)),
        # Draft tokens checked together, sliding window, a small model's heads (7 query heads per KV head of 64).
        _attn("attn_drafts", H=14, Hkv=2, D=64, page=32, n_seq=16, rows=5, past=(300, 6000), window=1024),
        # A 512-token chunk late in a long prompt.
        _attn("attn_chunk", H=32, Hkv=8, D=128, page=64, n_seq=1, rows=512, past=(3584, 3584)),
        # Prompts of odd lengths entering together from empty caches.
        _attn("attn_prompts", H=32, Hkv=8, D=128, page=64, n_seq=4, rows=1047, rows_min=600, past=(0, 0)),
        # A mixed step: one prompt chunk beside fifteen decoding conversations, wide heads.
        _attn("attn_mixed", H=16, Hkv=8, D=256, page=64, n_seq=16, rows=256, chunks=1, past=(100, 4096)),
    ]


def draw(rng) -> dict:
    """One more case of the listed ranges: sizes spread over their logarithm."""
    kind = rng.choice(["append", "append", "read", "step", "step", "few", "chunk", "chunk", "mixed"])
    D = rng.choice([64, 128, 128, 128, 256])
    Hkv = rng.choice([1, 2, 4, 8, 8])
    H = Hkv * rng.choice([1, 2, 3, 4, 4, 7, 8, 12])
    page, mix = rng.choice([32, 64, 64, 128, 256]), rng.randrange(1 << 30)
    if kind in ("append", "read"):
        n_seq = _log_int(rng, 1, 128)
        rows = _log_int(rng, 1, max(1, 4096 // n_seq))
        last = _log_int(rng, 1, min(1 << 17, (1 << 30 if kind == "read" else 1 << 32) // (n_seq * Hkv * D)))
        first = _log_int(rng, 1, last)
        c = {"n_seq": n_seq, "rows": rows, "past": (first - 1, last - 1), "page": page, "mix": mix, "rows_min": _log_int(rng, 1, rows)}
        if kind == "read":
            return _read("", Hkv=Hkv, D=D, **c)
        return _append("", H=H, Hkv=Hkv, D=D, n_dims=rng.choice([D, D, D // 2]), **c)
    # keys of all sequences, and rows x keys, no more than the largest listed case's
    if kind in ("step", "few"):
        n_seq = _log_int(rng, 1, 64)
        rows = 1 if kind == "step" else rng.randint(2, 8)
        rows_min, chunks = rows if rng.random() < 0.5 else 1, 0
        last = _log_int(rng, 32, max(64, min(131070, (131072 * 8 * 128) // (n_seq * Hkv * D))))
    else:
        n_seq = _log_int(rng, 1, 6) if kind == "chunk" else _log_int(rng, 2, 24)
        chunks = 1 if kind == "mixed" else 0
        rows, level = _log_int(rng, 9, 1024), rng.random() < 0.3
        wide = n_seq if kind == "chunk" else 1
        while wide * rows * rows * H * D > 512 * 2048 * 32 * 128:
            rows = rows * 2 // 3
        rows_min = rows if level else max(1, rows // 8)
        limit = 512 * 4096 * 32 * 128 // (wide * rows * H * D) - rows
        # (the plain form pads every sequence to the widest and longest)
        limit = min(limit, (3 << 30) // (4 * n_seq * rows * H) - rows, 16384)
        last = _log_int(rng, 1, limit) if limit >= 1 else 1
    first = last if rng.random() < 0.2 else _log_int(rng, 1, last)
    window = rng.choice([0, 0, 0, _log_int(rng, 1, 4096)])
    return _attn("", H=H, Hkv=Hkv, D=D, page=page, n_seq=n_seq, rows=rows, rows_min=rows_min, chunks=chunks,
                 past=(first - 1, last - 1), window=window, mix=mix)


def _case(kind, name, past, rows, rows_min=0, chunks=0, mix=7, **kw) -> dict:
    c = {"kind": kind, **kw, "rows": rows, "rows_min": rows_min or rows, "chunks": chunks, "past_min": past[0],
         "past_max": past[1], "mix": mix}
    return {"name": name, **c} if name else c


def _append(name, **kw) -> dict:
    return _case("append", name, **kw)


def _read(name, **kw) -> dict:
    return _case("read", name, **kw)


def _attn(name, window=0, **kw) -> dict:
    return _case("attn", name, window=window, **kw)


def _log_int(rng, lo: int, hi: int) -> int:
    lo, hi = max(1, lo), max(1, hi)
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _lengths(case) -> tuple[list[int], list[int]]:
    """New rows and past tokens of each sequence, spread over their logarithm. With `chunks`, that many sequences
    have all the rows and the others one."""
    rng = random.Random(case["mix"])
    n = case["n_seq"]
    rows = [_log_int(rng, case["rows_min"], case["rows"]) for _ in range(n)]
    if case["chunks"]:
        rows = [case["rows"] if s < case["chunks"] else 1 for s in range(n)]
        rng.shuffle(rows)
    past = [_log_int(rng, case["past_min"] + 1, case["past_max"] + 1) - 1 for _ in range(n)]
    return rows, past


def _pairs(case) -> tuple[int, int]:
    """(row, key) pairs that one head sees, and the keys that are read for them."""
    w, lengths = case.get("window") or 1 << 40, list(zip(*_lengths(case)))
    return sum(min(p + j + 1, w) for n, p in lengths for j in range(n)), sum(min(p + n, w + n - 1) for n, p in lengths)


def work(case) -> dict:
    D, Hkv, n = case["D"], case["Hkv"], sum(_lengths(case)[0])
    q4 = D / 32 * 18
    if case["kind"] == "append":  # q, k, v in; q out in f16; the rows written, read back and given out in f32
        H = case["H"]
        return {"bytes": n * (4 * D * (H + 2 * Hkv) + 2 * D * H + 2 * Hkv * (2 * q4 + 4 * D)),
                "flops": n * D * (3 * (H + Hkv) + 2 * Hkv * 4)}
    if case["kind"] == "read":
        return {"bytes": n * 2 * Hkv * (q4 + 4 * D), "flops": n * 2 * Hkv * D * 2}
    pairs, keys = _pairs(case)
    return {"bytes": keys * 2 * Hkv * q4 + n * case["H"] * D * (2 + 4), "flops": 4 * pairs * case["H"] * D}


# ------------------------------------------------------------------------------------------ inputs


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rows, past = _lengths(case)
    D, Hkv, page, n = case["D"], case["Hkv"], case["page"], sum(rows)
    need = [(p + r + page - 1) // page for p, r in zip(past, rows)]
    n_pages = sum(need) + 3  # (some pages belong to nobody)
    order = torch.randperm(n_pages, generator=g, device="cuda")
    table, at = torch.full((len(need), max(need) + 1), -1, dtype=torch.int32, device="cuda"), 0
    for s, m in enumerate(need):
        table[s, :m] = order[at:at + m].to(torch.int32)
        at += m
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    state = {"kind": case["kind"], "D": D, "Hkv": Hkv, "page": page, "n_pages": n_pages, "n": n, "max_rows": max(rows),
             "max_keys": max(p + r for p, r in zip(past, rows)), "pages": table,
             "starts": torch.tensor(starts, dtype=torch.int32, device="cuda"),
             "past": torch.tensor(past, dtype=torch.int32, device="cuda")}
    if case["kind"] == "append":
        # a layer's stacked projections of the rows, as a mat-mul leaves them
        H = case["H"]
        qkv = _normal(g, n, (H + 2 * Hkv) * D)
        heads = qkv.view(n, H + 2 * Hkv, D)
        half = case["n_dims"] // 2
        state |= {"H": H, "n_dims": case["n_dims"], "q": heads[:, :H], "k": heads[:, H:H + Hkv], "v": heads[:, H + Hkv:],
                  "freqs": torch.tensor([500000.0 ** (-i / half) for i in range(half)], dtype=torch.float32, device="cuda"),
                  "data": torch.zeros(n_pages * Hkv * (page // 32) * 36 * D, dtype=torch.uint8, device="cuda")}
        return state
    # a pool that appends have filled
    T = n_pages * Hkv * (page // 32)
    k, v = _normal(g, T, 32, D), _normal(g, T, 32, D)
    state["data"] = _pack(*_encode(k), *_encode(v)).reshape(-1)
    if case["kind"] == "attn":
        state |= {"H": case["H"], "window": case["window"], "scale": D ** -0.5,
                  "q": (_normal(g, n, case["H"], D) * 1.5).half()}
    return state


# -------------------------------------------------------------------------------------- plain form


def _encode(x):
    """f32 [.., D] -> codes int32 [.., D] and scales f16 [.., D / 32], by the Q4_0 encoder's 32-bit arithmetic."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    a = b.abs()
    at = torch.arange(32, device=x.device).expand_as(b)
    first = torch.where(a == a.amax(-1, keepdim=True), at, 32).amin(-1, keepdim=True)
    d = b.gather(-1, first) / -8.0
    inv = torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
    codes = (b * inv + 8.5).to(torch.int32).clamp(0, 15)
    return codes.reshape(x.shape), d.squeeze(-1).half()


def _nibbles(codes):
    half = codes.shape[-1] // 2
    return (codes[..., :half] | codes[..., half:] << 4).to(torch.uint8)


def _pack(kc, kd, vc, vd):
    """Whole tiles: codes [T, 32, D] and scales [T, 32, D / 32] of keys and values -> bytes [T, 36 D]."""
    T, _, D = kc.shape
    k = _nibbles(kc).view(T, 32, D // 64, 4, 8).transpose(2, 3).reshape(T, -1)
    v = _nibbles(vc).view(T, 4, 8, D // 64, 2, 16).permute(0, 3, 1, 5, 4, 2).reshape(T, -1)
    order = torch.tensor(ORDER, device=kc.device)
    scales = [d.view(T, 4, 8, D // 32)[:, :, order].permute(0, 3, 1, 2).contiguous().view(torch.uint8).reshape(T, -1)
              for d in (kd, vd)]
    return torch.cat([k, v, *scales], 1)


def _unpack(t):
    """Bytes [.., 36 D] of whole tiles -> keys and values, f32 [.., 32, D] each."""
    lead, D = t.shape[:-1], t.shape[-1] // 36
    k = t[..., :16 * D].reshape(-1, 32, 4, D // 64, 8).transpose(2, 3).reshape(-1, 32, D // 2)
    v = t[..., 16 * D:32 * D].reshape(-1, D // 64, 4, 16, 2, 8).permute(0, 2, 5, 1, 4, 3).reshape(-1, 32, D // 2)
    scales = t[..., 32 * D:].contiguous().view(torch.float16).reshape(-1, 2, D // 32, 4, 8)
    order = torch.tensor(ORDER, device=t.device)
    scales = scales[..., order].permute(1, 0, 3, 4, 2).reshape(2, -1, 32, D // 32, 1).float()

    def values(c, d):
        c = torch.cat([c & 15, c >> 4], -1).reshape(-1, 32, D // 32, 32)
        return ((c.float() - 8.0) * d).reshape(*lead, 32, D)

    return values(k, scales[0]), values(v, scales[1])


def _row_positions(st):
    """The sequence and the position of each row."""
    r = torch.arange(st["n"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(st["starts"], r, right=True) - 1
    return seq, (st["past"][seq] + r - st["starts"][seq]).long()


def _addresses(st):
    """Byte addresses of the rows' codes, [n, Hkv, D / 2] each, and f16 addresses of their scales, [n, Hkv, D / 32]."""
    D, Hkv, page = st["D"], st["Hkv"], st["page"]
    seq, pos = _row_positions(st)
    tile = (st["pages"][seq, pos // page].long()[:, None] * Hkv + torch.arange(Hkv, device="cuda")) * (page // 32)
    tile = (tile + (pos % page // 32)[:, None])[..., None] * (36 * D)
    slot = (pos % 32)[:, None, None]
    i = torch.arange(D // 2, device="cuda")
    k = tile + slot * (D // 2) + (i // 8 % 4) * (D // 8) + i // 32 * 8 + i % 8
    v = tile + 16 * D + ((i // 32 * 4 + slot // 8) * 16 + i % 16) * 16 + i // 16 % 2 * 8 + slot % 8
    at = (tile + 32 * D) // 2 + torch.arange(D // 32, device="cuda") * 32 + slot // 8 * 8 + torch.tensor(ORDER, device="cuda")[slot % 8]
    return k, v, at, at + D


def _rows_back(st):
    k, v, kd, vd = _addresses(st)
    halves = st["data"].view(torch.float16)

    def values(at, d):
        c = st["data"][at]
        c = torch.cat([c & 15, c >> 4], -1).reshape(*d.shape, 32)
        return ((c.float() - 8.0) * halves[d].float()[..., None]).reshape(st["n"], st["Hkv"], st["D"])

    return {"k": values(k, kd), "v": values(v, vd)}


def _rotate(x, angle, n_dims):
    """Pairs (i, i + n_dims / 2) turned in 64 bits, rounded once."""
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x[..., :n_dims // 2].double(), x[..., n_dims // 2:n_dims].double()
    return torch.cat([(a * c - b * s).float(), (a * s + b * c).float(), x[..., n_dims:]], -1)


def _append_plain(st):
    angle = _row_positions(st)[1].double()[:, None] * st["freqs"].double()
    kc, kd = _encode(_rotate(st["k"], angle, st["n_dims"]))
    vc, vd = _encode(st["v"])
    k, v, k_at, v_at = _addresses(st)
    st["data"][k], st["data"][v] = _nibbles(kc), _nibbles(vc)
    halves = st["data"].view(torch.float16)
    halves[k_at], halves[v_at] = kd, vd
    return {"q": _rotate(st["q"], angle, st["n_dims"]).half(), **_rows_back(st)}


def _attn_plain(st):
    D, Hkv, H, page, n = st["D"], st["Hkv"], st["H"], st["page"], st["n"]
    S, G, R = st["past"].numel(), H // Hkv, st["max_rows"]
    pages = st["pages"][:, :-(-st["max_keys"] // page)].long()
    tiles = st["data"].view(-1, Hkv, page // 32, 36 * D)[pages.clamp(min=0)]
    k, v = _unpack(tiles.transpose(1, 2).reshape(S, Hkv, -1, 36 * D))
    k, v = k.reshape(S, Hkv, -1, D), v.reshape(S, Hkv, -1, D)
    seq, pos = _row_positions(st)
    j = pos - st["past"][seq]
    q = torch.zeros((S, R, H, D), device="cuda")
    q[seq, j] = st["q"].float()
    q = q.view(S, R, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(S, Hkv, R * G, D)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * st["scale"]
    key = torch.arange(k.shape[2], device="cuda")
    at = (st["past"][:, None] + torch.arange(R, device="cuda"))[..., None]
    seen = key <= at
    if st["window"]:
        seen &= key > at - st["window"]
    s = s.view(S, Hkv, R, G, -1).masked_fill_(~seen[:, None, :, None], -math.inf).view(s.shape)
    s = torch.exp_(s.sub_(s.amax(-1, keepdim=True)))
    o = torch.matmul(s, v) / s.sum(-1, keepdim=True)
    return o.view(S, Hkv, R, G, D).permute(0, 2, 1, 3, 4).reshape(S, R, H, D)[seq, j]


# -------------------------------------------------------------------------------------- framework


def _handles(st):
    """What a user's program keeps beside the tensors: the cache and the batch (its lists of rows and pages)."""
    if "handles" not in st:
        path = os.path.join(os.getcwd(), "ggml-compiler_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        from ggml_compiler_amd import ops

        cache = ops.PagedCache(st["n_pages"], st["page"], st["Hkv"], st["D"], st["data"])
        st["handles"] = ops, cache, ops.PagedBatch(st["pages"], st["starts"], st["past"])
    return st["handles"]


def run(state):
    st = state
    if own:
        ops, cache, batch = _handles(st)
        if st["kind"] == "attn":
            return ops.paged_attn(cache, batch, st["q"], st["scale"], max_rows=st["max_rows"], window=st["window"])
        out = {}
        if st["kind"] == "append":
            out["q"] = ops.paged_append(cache, batch, st["k"], st["v"], q=st["q"], freqs=st["freqs"])
        out["k"], out["v"] = ops.paged_read(cache, batch, st["n"])
        return out
    if st["kind"] == "append":
        return _append_plain(st)
    return _rows_back(st) if st["kind"] == "read" else _attn_plain(st)


# ------------------------------------------------------------------- the definition, in 64 bits


def exact(case, seed):
    st = prepare(case, seed)
    D, Hkv, page = st["D"], st["Hkv"], st["page"]
    starts, past = st["starts"].tolist(), st["past"].tolist()
    if case["kind"] == "append":
        rows = torch.cat([torch.arange(p, p + b - a) for a, b, p in zip(starts, starts[1:], past)]).cuda()
        half = st["n_dims"] // 2
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), rows.double().outer(st["freqs"].double()))

        def turned(x):
            z = torch.complex(x[..., :half].double(), x[..., half:2 * half].double()) * turn[:, None]
            return torch.cat([z.real, z.imag, x[..., 2 * half:].double()], -1)

        def stored(x):  # the format's own steps in 32 bits, its value in 64
            b = x.unflatten(-1, (-1, 32))
            top, low = b.amax(-1), b.amin(-1)
            a = torch.maximum(top, -low)
            up, down = (b == a[..., None]).double(), (b == -a[..., None]).double()
            where = torch.arange(32, 0, -1, device="cuda", dtype=torch.float64)
            sign = torch.where((up * where).amax(-1) > (down * where).amax(-1), 1.0, -1.0).float()
            d = sign * a / -8.0
            inv = torch.where(d == 0, 0.0, torch.reciprocal(d))[..., None]
            code = torch.floor(b * inv + 8.5).clamp(0, 15).double()
            return ((code - 8) * d.half().double()[..., None]).flatten(-2)

        return {"q": turned(st["q"]), "k": stored(turned(st["k"]).float()), "v": stored(st["v"])}

    def sequence(s, length):
        """Keys and values of the first `length` positions, f64 [Hkv, length, D]."""
        p = torch.arange(length, device="cuda")
        i = torch.arange(D, device="cuda")
        tile = ((st["pages"][s].long()[p // page] * Hkv)[None] + torch.arange(Hkv, device="cuda")[:, None]) * (page // 32)
        tile = ((tile + (p % page // 32)) * (36 * D))[..., None]
        t, low, block = (p % 32)[:, None], i % (D // 2), i // 32
        kb = t * (D // 2) + low // 8 % 4 * (D // 8) + low // 32 * 8 + low % 8
        vb = 16 * D + low // 32 * 1024 + t // 8 * 256 + low % 16 * 16 + low // 16 % 2 * 8 + t % 8
        sb = block * 32 + t // 8 * 8 + torch.tensor(ORDER, device="cuda")[t % 8]
        shift = torch.where(i < D // 2, 0, 4).to(torch.uint8)
        halves = st["data"].view(torch.float16)

        def values(at, scale_at):
            c = (st["data"][tile + at] >> shift) & 15
            return (c.double() - 8) * halves[(tile + scale_at) // 2 + sb].double()

        return values(kb, 32 * D), values(vb, 34 * D)

    if case["kind"] == "read":
        kv = [sequence(s, p + starts[s + 1] - starts[s]) for s, p in enumerate(past)]
        return {n: torch.cat([x[i][:, p:].transpose(0, 1) for x, p in zip(kv, past)]) for i, n in enumerate("kv")}
    out, G = [], st["H"] // Hkv
    for s, p in enumerate(past):
        k, v = sequence(s, p + starts[s + 1] - starts[s])
        q = st["q"][starts[s]:starts[s + 1]].double()
        n, length = q.shape[0], k.shape[1]
        key, at = torch.arange(length, device="cuda")[None], torch.arange(p, p + n, device="cuda")[:, None]
        hidden = (key > at) | ((key <= at - st["window"]) if st["window"] else False)
        o = []
        for h in range(st["H"]):
            x = (q[:, h] @ k[h // G].T) * st["scale"]
            o.append(torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ v[h // G])
        out.append(torch.stack(o, 1))
    return torch.cat(out)
