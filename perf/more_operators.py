"""The operators of a step with drafted tokens as cases that can be prepared, run and checked: the masks and positions of
draft trees, appending their rows to the paged 4-bit cache, their attention over it, the drafts' verification, and moving the
accepted rows together.

A sequence's rows are a tree: row 0 is the last accepted token, every other row a drafted one, and its parent the number of
the earlier row of the sequence that it follows (rows without one follow the cached tokens). Row j lies in the cache at slot
past + j, its position is past + its depth, and it sees the past slots, its ancestors and itself. The cache's pool and batch:
[page][KV head][tile of 32 tokens][36 D bytes], keys and values as Q4_0 blocks (32 values: an f16 scale d and 32 codes of 4
bits, a code c standing for d (c - 8)); sequence s owns rows starts[s] .. starts[s + 1] - 1, slot p lies in page
pages[s][p / page], place p % page. A tile, for heads of D values, byte i of a token holding dim i in its low nibble and dim
i + D / 2 in its high one:
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
BELOW_ONE = 1.0 - 2.0 ** -24


def listed() -> list[dict]:
    return [
        # One conversation's tree of drafts: the smallest call, latency alone.
        _tree("tree_one", n_seq=1, rows=26, wide=4, past=(4000, 4000)),
        # A server's 64 conversations, large trees of odd sizes under a short window.
        _tree("tree_many", n_seq=64, rows=255, rows_min=40, wide=5, past=(1, 100000), window=4),
        # That one conversation's drafts into an 8B-shaped layer's cache.
        _append("append_one", H=32, Hkv=8, D=128, page=64, n_seq=1, rows=26, wide=4, past=(4000, 4000), n_dims=128),
        # 32 conversations' trees at once.
        _append("append_many", H=32, Hkv=8, D=128, page=64, n_seq=32, rows=64, rows_min=33, wide=4, past=(1, 100000), n_dims=128),
        # A short chain of drafts in a small model: 7 query heads per KV head of 64, sliding window.
        _attn("attn_chain", H=14, Hkv=2, D=64, page=32, n_seq=1, rows=6, wide=1, past=(1500, 1500), window=1024),
        # A serving step: 16 conversations of spread lengths, a tree of some 20 to 40 drafts each.
        _attn("attn_trees", H=32, Hkv=8, D=128, page=64, n_seq=16, rows=40, rows_min=20, wide=4, past=(200, 8191)),
        # One very long conversation and a wide tree.
        _attn("attn_long", H=32, Hkv=8, D=128, page=256, n_seq=1, rows=61, wide=4, past=(65000, 65000)),
        # Four drafts of one conversation against the drafter's own distributions.
        _verify("verify_chain", n_seq=1, rows=5, wide=1, V=128256, drawn=True),
        # The same for 64 conversations, some of them greedy.
        _verify("verify_chains", n_seq=64, rows=5, rows_min=2, wide=1, V=128256, drawn=True),
        # Trees of likely continuations (no distributions), 16 conversations.
        _verify("verify_trees", n_seq=16, rows=64, rows_min=40, wide=4, V=128256, drawn=False),
        # The accepted rows of one conversation, a small model's layers.
        _move("move_one", Hkv=2, D=64, page=32, n_seq=1, rows=26, wide=4, past=(900, 900), layers=4),
        # Those of 32 conversations in all of a large model's layers.
        _move("move_many", Hkv=8, D=128, page=64, n_seq=32, rows=64, rows_min=33, wide=3, past=(100, 2000), layers=32),
    ]


def draw(rng) -> dict:
    """One more case of the listed ranges: sizes spread over their logarithm."""
    kind = rng.choice(["tree", "append", "attn", "attn", "attn", "verify", "verify", "verify", "move"])
    wide, mix = rng.choice([1, 2, 3, 4, 4, 8]), rng.randrange(1 << 30)
    D = rng.choice([64, 128, 128, 128, 256])
    Hkv = rng.choice([1, 2, 4, 8, 8])
    H = Hkv * rng.choice([1, 2, 3, 4, 4, 7, 8, 12])
    page = rng.choice([32, 64, 64, 128, 256])
    window = rng.choice([0, 0, 0, _log_int(rng, 1, 4096)])
    n_seq = _log_int(rng, 1, 64)
    if kind == "tree":
        # (the plain form's seen rows are a square)
        rows = _log_int(rng, 1, min(1024, int(math.sqrt(64 * 255 * 255 / n_seq))))
        return _tree("", n_seq=n_seq, rows=rows, rows_min=_log_int(rng, 1, rows), wide=wide, past=(0, _log_int(rng, 1, 1 << 20)),
                     window=rng.choice([0, 0, _log_int(rng, 1, 16)]), mix=mix)
    if kind == "append":
        rows = _log_int(rng, 1, max(1, min(256, 32 * 64 * 48 * 128 // (n_seq * (H + 2 * Hkv) * D))))
        last = _log_int(rng, 1, min(1 << 17, (1 << 32) // (n_seq * Hkv * D)))
        return _append("", H=H, Hkv=Hkv, D=D, page=page, n_seq=n_seq, rows=rows, rows_min=_log_int(rng, 1, rows), wide=wide,
                       past=(_log_int(rng, 1, last) - 1, last - 1), n_dims=rng.choice([D, D, D // 2]), mix=mix)
    if kind == "move":
        layers = _log_int(rng, 1, 32)
        rows = _log_int(rng, 2, 256)
        last = _log_int(rng, 1, max(1, min(1 << 16, (1 << 31) // (n_seq * layers * Hkv * D) - rows)))
        while n_seq * layers * Hkv * D * _deep(rows, max(2, wide)) > 32 * 32 * 8 * 128 * _deep(64, 3):
            layers, n_seq = max(1, layers // 2), max(1, n_seq * 2 // 3)
        return _move("", Hkv=Hkv, D=D, page=page, n_seq=n_seq, rows=rows, rows_min=_log_int(rng, 1, rows), wide=max(2, wide),
                     past=(_log_int(rng, 1, last) - 1, last - 1), layers=layers, mix=mix)
    if kind == "verify":
        V = rng.choice([32000, 128256, _log_int(rng, 5, 200000), _log_int(rng, 5, 200000)])
        drawn, rows = rng.random() < 0.6, _log_int(rng, 1, 64)
        while n_seq * rows * V * (2 if drawn else 1) > 64 * 5 * 128256 * 2:
            n_seq, rows = max(1, n_seq * 2 // 3), max(1, rows * 4 // 5)
        return _verify("", n_seq=n_seq, rows=rows, rows_min=_log_int(rng, 1, rows), wide=min(wide, 4), V=V, drawn=drawn,
                       pad=rng.choice([0, 0, 1, 64]), mix=mix)
    rows = _log_int(rng, 1, 256)
    # (row, key) pairs, and keys of all sequences, no more than the largest listed case's; the plain form's scores fit besides
    while n_seq * rows * (rows + 32) * H * D > 61 * 65000 * 32 * 128 or n_seq * (rows + 32) * Hkv * D > 65000 * 8 * 128:
        n_seq, rows = max(1, n_seq * 2 // 3), max(1, rows * 3 // 4)
    limit = min(61 * 65000 * 32 * 128 // (n_seq * rows * H * D), (61 * 65000 * 8 * 128) // (n_seq * Hkv * D * 32), 100000) - rows
    last = _log_int(rng, 1, max(1, limit))
    return _attn("", H=H, Hkv=Hkv, D=D, page=page, n_seq=n_seq, rows=rows, rows_min=_log_int(rng, 1, rows), wide=wide,
                 past=(_log_int(rng, 1, last) - 1, last - 1), window=window, mix=mix)


def _case(kind, name, rows, past=(0, 0), rows_min=0, mix=7, **kw) -> dict:
    c = {"kind": kind, **kw, "rows": rows, "rows_min": rows_min or rows, "past_min": past[0], "past_max": past[1], "mix": mix}
    return {"name": name, **c} if name else c


def _tree(name, window=0, **kw) -> dict:
    return _case("tree", name, window=window, **kw)


def _append(name, **kw) -> dict:
    return _case("append", name, **kw)


def _attn(name, window=0, **kw) -> dict:
    return _case("attn", name, window=window, **kw)


def _verify(name, pad=0, **kw) -> dict:
    return _case("verify", name, pad=pad, **kw)


def _move(name, **kw) -> dict:
    return _case("move", name, **kw)


def _log_int(rng, lo: int, hi: int) -> int:
    lo, hi = max(1, lo), max(1, hi)
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _deep(rows: int, wide: int) -> int:
    """Levels of a tree of that many rows, about."""
    return 1 + int(math.log(rows) / math.log((1 + wide) / 2)) if wide > 1 else rows


def _trees(case) -> tuple[list[int], list[list[int]], list[int]]:
    """Rows, parents and past tokens of each sequence: trees laid out level by level, 1 to `wide` children to a row (chains: 1)."""
    rng = random.Random(case["mix"])
    rows = [_log_int(rng, case["rows_min"], case["rows"]) for _ in range(case["n_seq"])]
    parents = []
    for n in rows:
        tree, at = [-1], 0
        while len(tree) < n:
            tree += [at] * min(rng.randint(1, case["wide"]), n - len(tree))
            at += 1
        parents.append(tree)
    past = [_log_int(rng, case["past_min"] + 1, case["past_max"] + 1) - 1 for _ in rows]
    return rows, parents, past


def _depths(parents: list[int]) -> list[int]:
    d = []
    for a in parents:
        d.append(d[a] + 1 if a >= 0 else 0)
    return d


def _paths(case) -> list[list[int]]:
    """Rows that were accepted, one path from the root of each tree. No row is moved to where another is taken from, so that a move
    can be repeated."""
    rng, paths = random.Random(case["mix"] + 1), []
    for tree in _trees(case)[1]:
        path = [0]
        while rng.random() < 0.85:
            below = [c for c, a in enumerate(tree) if a == path[-1] and c]
            if not below:
                break
            path.append(rng.choice(below))
        while any(j != i and j < len(path) for i, j in enumerate(path)):
            path.pop()
        paths.append(path)
    return paths


def work(case) -> dict:
    rows, parents, past = _trees(case)
    n, kind = sum(rows), case["kind"]
    if kind == "tree":
        words = -(-max(rows) // 32)
        return {"bytes": n * (4 + 4 + 4 * words), "flops": n * words}
    if kind == "verify":
        # the rows on the paths: the root, and of a level below it a draft is accepted in some two of three times
        seen = sum(sum(0.67 ** d for d in range(max(_depths(t)) + 1)) for t in parents)
        return {"bytes": 4 * case["V"] * seen * (2 if case["drawn"] else 1), "flops": 8 * case["V"] * seen * (2 if case["drawn"] else 1)}
    D, Hkv = case["D"], case["Hkv"]
    q4 = D / 32 * 18
    if kind == "move":
        moved = sum(i != j for p in _paths(case) for i, j in enumerate(p))
        return {"bytes": 2 * moved * case["layers"] * 2 * Hkv * q4 + 4 * n, "flops": 0}
    H = case["H"]
    if kind == "append":  # q, k, v in; q out in f16; the rows written, read back and given out in f32
        return {"bytes": n * (4 * D * (H + 2 * Hkv) + 2 * D * H + 2 * Hkv * (2 * q4 + 4 * D)),
                "flops": n * D * (3 * (H + Hkv) + 2 * Hkv * 4)}
    pairs = keys = 0
    for r, tree, p in zip(rows, parents, past):
        w, depth = case["window"] or 1 << 40, _depths(tree)
        pairs += sum(min(p + d + 1, w) for d in depth)
        keys += min(p, w - 1) + r
    return {"bytes": keys * 2 * Hkv * q4 + n * H * D * (2 + 4), "flops": 4 * pairs * H * D}


# ------------------------------------------------------------------------------------------ inputs


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _int(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rows, parents, past = _trees(case)
    n, kind = sum(rows), case["kind"]
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    state = {"kind": kind, "n": n, "max_rows": max(rows), "starts": _int(starts), "parents": _int(sum(parents, []))}
    if kind == "verify":
        return state | _prepare_verify(case, g, parents, starts)
    state["past"] = _int(past)
    if kind == "tree":
        # (as many pages as the longest needs, though nothing here reads them)
        pages = _int([[0] * ((max(past) + max(rows)) // 64 + 1)] * len(rows))
        # other inputs for another seed: other lengths of the past
        state["past"] += torch.randint(0, 64, (len(rows),), generator=g, device="cuda", dtype=torch.int32)
        return state | {"pages": pages, "window": case["window"], "n_pages": 1, "page": 64}
    D, Hkv, page = case["D"], case["Hkv"], case["page"]
    need = [(p + r + page - 1) // page for p, r in zip(past, rows)]
    n_pages = sum(need) + 3  # (some pages belong to nobody)
    order = torch.randperm(n_pages, generator=g, device="cuda")
    table, at = torch.full((len(need), max(need) + 1), -1, dtype=torch.int32, device="cuda"), 0
    for s, m in enumerate(need):
        table[s, :m] = order[at:at + m].to(torch.int32)
        at += m
    state |= {"D": D, "Hkv": Hkv, "page": page, "n_pages": n_pages, "pages": table,
              "max_keys": max(p + r for p, r in zip(past, rows))}
    if kind == "move":
        paths = _paths(case)
        most = max(map(len, paths))
        size = n_pages * Hkv * (page // 32) * 36 * D
        return state | {"count": _int([len(p) for p in paths]), "rows": _int([p + [-1] * (most - len(p)) for p in paths]),
                        "data": [torch.randint(0, 256, (size,), generator=g, device="cuda", dtype=torch.uint8) for _ in range(case["layers"])]}
    depth = [_depths(t) for t in parents]
    state["positions"] = _int([p + d for p, t in zip(past, depth) for d in t])
    if kind == "append":
        # a layer's stacked projections of the rows, as a mat-mul leaves them
        H = case["H"]
        heads = _normal(g, n, (H + 2 * Hkv) * D).view(n, H + 2 * Hkv, D)
        half = case["n_dims"] // 2
        return state | {"H": H, "n_dims": case["n_dims"], "q": heads[:, :H], "k": heads[:, H:H + Hkv], "v": heads[:, H + Hkv:],
                        "freqs": torch.tensor([500000.0 ** (-i / half) for i in range(half)], dtype=torch.float32, device="cuda"),
                        "data": torch.zeros(n_pages * Hkv * (page // 32) * 36 * D, dtype=torch.uint8, device="cuda")}
    # a pool that appends have filled, and the step's tree, the same for all layers
    words, w, masks = -(-max(rows) // 32), case["window"] or 1 << 40, []
    for tree, d in zip(parents, depth):
        seen = []
        for j, a in enumerate(tree):
            seen.append((seen[a] if a >= 0 else 0) | 1 << j)
        for j, m in enumerate(seen):
            m = sum(1 << i for i in range(j + 1) if m >> i & 1 and d[j] - d[i] < w)
            masks.append([(m >> 32 * x & 0xffffffff) - (1 << 32 if m >> 32 * x + 31 & 1 else 0) for x in range(words)])
    T = n_pages * Hkv * (page // 32)
    k, v = _normal(g, T, 32, D), _normal(g, T, 32, D)
    state["data"] = _pack(*_encode(k), *_encode(v)).reshape(-1)
    return state | {"H": case["H"], "window": case["window"], "scale": D ** -0.5, "mask": _int(masks),
                    "q": (_normal(g, n, case["H"], D) * 1.5).half()}


def _prepare_verify(case, g, parents, starts):
    """Logits of a shape that language has: noise, and a few tokens far above it. The drafter's are the target's but for noise; its
    drafts are drawn from them (`drawn`), or the likeliest."""
    V, n, S = case["V"], starts[-1], len(parents)
    ld = V + case["pad"]
    temperature = torch.tensor([0.0, 0.7, 1.0, 1.3], device="cuda")[torch.randint(0, 4, (S,), generator=g, device="cuda")]
    logits, draft = (torch.empty(n, ld, device="cuda")[:, :V] for _ in range(2))
    flat = [(s, j, a) for s, t in enumerate(parents) for j, a in enumerate(t)]
    rank, rows_of = [0] * n, [[] for _ in range(n)]
    for r, (s, j, a) in enumerate(flat):
        if a >= 0:
            rank[r] = len(rows_of[starts[s] + a])
            rows_of[starts[s] + a].append(r)
    likely = min(V, max(map(len, rows_of), default=1) or 1)
    tops, step = [], max(1, (1 << 26) // V)
    for r in range(0, n, step):
        m = min(step, n - r)
        u = torch.rand(m, V, generator=g, device="cuda")
        logits[r:r + m] = _normal(g, m, V).mul_(2.0).add_(u.pow_(V / 32), alpha=14.0)
        draft[r:r + m] = _normal(g, m, V).mul_(0.7).add_(logits[r:r + m])
        tops.append(draft[r:r + m].topk(likely, -1).indices)
    tops = torch.cat(tops)
    node = torch.tensor([starts[s] + max(a, 0) for s, j, a in flat], device="cuda")
    tokens = tops[node, torch.tensor([k % likely for k in rank], device="cuda")]
    if case["drawn"]:
        seq = torch.tensor([s for s, j, a in flat], device="cuda")
        for r in range(0, n, step):
            t, at = temperature[seq[r:r + step], None], node[r:r + step]
            u = torch.rand(at.numel(), V, generator=g, device="cuda").clamp_(1e-30, 1.0)
            tokens[r:r + step] = torch.where(t[:, 0] > 0, (draft[at] / t.clamp(min=0.1) - u.log_().neg_().log_()).argmax(-1), tokens[r:r + step])
    coins = torch.rand(n, generator=g, device="cuda")
    return {"V": V, "logits": logits, "draft": draft if case["drawn"] else None, "temperature": temperature, "coins": coins,
            "tokens": tokens.to(torch.int32), "wide": max(map(len, rows_of)), "max_path": 1 + max(max(_depths(t)) for t in parents)}


# -------------------------------------------------------------------------------------- plain forms


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


def _rows_slots(st):
    """The sequence of each row, its number there and its slot."""
    r = torch.arange(st["n"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(st["starts"], r, right=True) - 1
    j = (r - st["starts"][seq]).long()
    return seq, j, st["past"][seq] + j


def _padded(x, seq, j, S, R, fill):
    out = torch.full((S, R), fill, device="cuda", dtype=torch.int64)
    out[seq, j] = x.long()
    return out


def _tree_plain(st):
    S, R = st["past"].numel(), st["max_rows"]
    seq, j, _ = _rows_slots(st)
    parent = _padded(st["parents"], seq, j, S, R, -1)
    at = torch.arange(R, device="cuda")
    parent = torch.where((parent >= 0) & (parent < at), parent, R)  # (R: a row that nobody is, its own parent)
    up = torch.cat([parent, torch.full((S, 1), R, device="cuda")], 1)
    seen = torch.eye(R + 1, R, device="cuda", dtype=torch.bool).expand(S, R + 1, R)
    for _ in range((R - 1).bit_length()):
        seen = seen | seen.gather(1, up[..., None].expand(S, R + 1, R))
        up = up.gather(1, up)
    seen = seen[:, :R]
    depth = seen.sum(-1) - 1
    if st["window"]:
        seen = seen & (depth[:, :, None] - depth[:, None] < st["window"])
    words = -(-R // 32)
    bits = torch.zeros(S, R, 32 * words, device="cuda", dtype=torch.int64)
    bits[..., :R] = seen
    bits = (bits.view(S, R, words, 32) << torch.arange(32, device="cuda")).sum(-1)
    mask = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32)
    return {"positions": st["past"][seq] + depth[seq, j].to(torch.int32), "mask": mask[seq, j]}


def _addresses(st):
    """Byte addresses of the rows' codes, [n, Hkv, D / 2] each, and f16 addresses of their scales, [n, Hkv, D / 32]."""
    D, Hkv, page = st["D"], st["Hkv"], st["page"]
    seq, _, pos = _rows_slots(st)
    return _slot_addresses(st["pages"][seq, pos // page].long(), pos, D, Hkv, page)


def _slot_addresses(entry, pos, D, Hkv, page):
    tile = (entry[:, None] * Hkv + torch.arange(Hkv, device="cuda")) * (page // 32)
    tile = (tile + (pos % page // 32)[:, None])[..., None] * (36 * D)
    slot = (pos % 32)[:, None, None]
    i = torch.arange(D // 2, device="cuda")
    k = tile + slot * (D // 2) + (i // 8 % 4) * (D // 8) + i // 32 * 8 + i % 8
    v = tile + 16 * D + ((i // 32 * 4 + slot // 8) * 16 + i % 16) * 16 + i // 16 % 2 * 8 + slot % 8
    at = (tile + 32 * D) // 2 + torch.arange(D // 32, device="cuda") * 32 + slot // 8 * 8 + torch.tensor(ORDER, device="cuda")[slot % 8]
    return k, v, at, at + D


def _rotate(x, angle, n_dims):
    """Pairs (i, i + n_dims / 2) turned in 64 bits, rounded once."""
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x[..., :n_dims // 2].double(), x[..., n_dims // 2:n_dims].double()
    return torch.cat([(a * c - b * s).float(), (a * s + b * c).float(), x[..., n_dims:]], -1)


def _append_plain(st):
    angle = st["positions"].double()[:, None] * st["freqs"].double()
    kc, kd = _encode(_rotate(st["k"], angle, st["n_dims"]))
    vc, vd = _encode(st["v"])
    k, v, k_at, v_at = _addresses(st)
    st["data"][k], st["data"][v] = _nibbles(kc), _nibbles(vc)
    halves = st["data"].view(torch.float16)
    halves[k_at], halves[v_at] = kd, vd

    def values(at, d):
        c = st["data"][at]
        c = torch.cat([c & 15, c >> 4], -1).reshape(*d.shape, 32)
        return ((c.float() - 8.0) * halves[d].float()[..., None]).reshape(st["n"], st["Hkv"], st["D"])

    return {"q": _rotate(st["q"], angle, st["n_dims"]).half(), "k": values(k, k_at), "v": values(v, v_at)}


def _attn_plain(st):
    D, Hkv, H, page = st["D"], st["Hkv"], st["H"], st["page"]
    S, G, R = st["past"].numel(), H // Hkv, st["max_rows"]
    pages = st["pages"][:, :-(-st["max_keys"] // page)].long()
    tiles = st["data"].view(-1, Hkv, page // 32, 36 * D)[pages.clamp(min=0)]
    k, v = _unpack(tiles.transpose(1, 2).reshape(S, Hkv, -1, 36 * D))
    k, v = k.reshape(S, Hkv, -1, D), v.reshape(S, Hkv, -1, D)
    seq, j, _ = _rows_slots(st)
    q = torch.zeros((S, R, H, D), device="cuda")
    q[seq, j] = st["q"].float()
    q = q.view(S, R, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(S, Hkv, R * G, D)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * st["scale"]
    key = torch.arange(k.shape[2], device="cuda")
    past = st["past"][:, None, None].long()
    seen = (key < past).expand(S, R, -1)
    if st["window"]:
        seen = seen & (key > _padded(st["positions"], seq, j, S, R, 0)[..., None] - st["window"])
    words = torch.zeros((S, R, st["mask"].shape[1]), device="cuda", dtype=torch.int64)
    words[seq, j] = st["mask"].long()
    i = (key - past).clamp(0, R - 1).expand(S, R, -1)
    seen = seen | (key >= past) & (key < past + R) & ((words.gather(2, i // 32) >> i % 32 & 1) > 0)
    s = s.view(S, Hkv, R, G, -1).masked_fill_(~seen[:, None, :, None], -math.inf).view(s.shape)
    s = torch.exp_(s.sub_(s.amax(-1, keepdim=True)))
    o = torch.matmul(s, v) / s.sum(-1, keepdim=True)
    return o.view(S, Hkv, R, G, D).permute(0, 2, 1, 3, 4).reshape(S, R, H, D)[seq, j]


def _verify_plain(st):
    """All sequences a level at a time, in 64 bits: a draft stands or falls by values next to a border."""
    V, P, starts = st["V"], st["max_path"], st["starts"].long()
    S, R = starts.numel() - 1, st["max_rows"]
    r = torch.arange(st["n"], device="cuda")
    seq = torch.searchsorted(starts, r, right=True) - 1
    parent = _padded(st["parents"], seq, r - starts[seq], S, R, -1)
    number, at = torch.arange(R, device="cuda"), torch.arange(V, device="cuda")
    parent = torch.where(number > 0, parent, -1)
    cur = torch.zeros(S, dtype=torch.int64, device="cuda")
    on = starts[1:] > starts[:-1]
    count, out_rows, out_tokens = cur.clone(), cur.new_full((S, P), -1), cur.new_full((S, P), -1)
    greedy, t = ~(st["temperature"] > 0), st["temperature"].double()
    t = torch.where(greedy, 1.0, t)[:, None]

    def softmax(x):
        x = x.double()
        e = torch.exp((x - x.amax(-1, keepdim=True)) / t)
        return e / e.sum(-1, keepdim=True)

    def first(x):
        return torch.where(x, at, V).amin(-1)

    for level in range(P):
        row = (starts[:-1] + cur).clamp(max=st["n"] - 1)
        x = st["logits"][row]
        top = first(x == x.amax(-1, keepdim=True))
        p = softmax(x)
        w, C, c = p, torch.zeros(S, 1, device="cuda", dtype=torch.float64), torch.ones(S, 1, device="cuda", dtype=torch.float64)
        q = softmax(st["draft"][row]) if st["draft"] is not None else None
        child = parent == cur[:, None]
        nth = child.cumsum(1)
        taken = torch.full_like(cur, -1)
        for b in range(st["wide"]):
            has = (child & (nth == b + 1)) & (taken < 0)[:, None]
            j = torch.where(has, number, R).amin(-1)
            has = j < R
            i = (starts[:-1] + j).clamp(max=st["n"] - 1)
            token = st["tokens"][i].long()
            good = (token >= 0) & (token < V)
            token = token.clamp(0, V - 1)[:, None]
            qt = q.gather(1, token) if q is not None else 1.0
            take = (st["coins"][i].double()[:, None] * c * qt < w.gather(1, token))[:, 0]
            take = has & good & torch.where(greedy, token[:, 0] == top, take)
            taken = torch.where(take, j, taken)
            less = (has & ~take)[:, None]
            if q is None:
                w = torch.where(less & good[:, None] & (at == token), 0.0, w)
            else:
                C = torch.where(less, C + c, C)
                w = torch.where(less, (p - C * q).clamp(min=0), w)
            c = torch.where(less, w.sum(-1, keepdim=True), c)
        w = torch.where(c > 0, w, p)
        sums = w.cumsum(-1)
        x = st["coins"][(starts[:-1]).clamp(max=st["n"] - 1)].double().clamp(0, BELOW_ONE)[:, None] * sums[:, -1:]
        sample = torch.where(greedy, top, first((sums > x) & (w > 0)))
        accepted = taken >= 0
        i = (starts[:-1] + taken.clamp(min=0)).clamp(max=st["n"] - 1)
        out_rows[:, level] = torch.where(on, cur, -1)
        out_tokens[:, level] = torch.where(on, torch.where(accepted, st["tokens"][i].long(), sample), -1)
        count += on
        on = on & accepted
        cur = torch.where(on, taken, cur)
    return {"count": count.to(torch.int32), "rows": out_rows.to(torch.int32), "tokens": out_tokens.to(torch.int32)}


def _move_plain(st):
    D, Hkv, page, P = st["D"], st["Hkv"], st["page"], st["rows"].shape[1]
    i = torch.arange(P, device="cuda")
    s, i = (i < st["count"][:, None]).nonzero(as_tuple=True)
    past, j = st["past"][s].long(), st["rows"][s, i].long()
    places = [_slot_addresses(st["pages"][s, x // page].long(), x, D, Hkv, page) for x in (past + j, past + i)]
    for data in st["data"]:
        halves = data.view(torch.float16)
        for n, (src, dst) in enumerate(zip(*places)):
            on = data if n < 2 else halves.view(torch.int16)
            on[dst] = on[src]
    return st["data"]


# -------------------------------------------------------------------------------------- framework


def _handles(st):
    """What a user's program keeps beside the tensors: the caches, the batch (its lists of rows and pages) and the step's tree."""
    if "handles" not in st:
        path = os.path.join(os.getcwd(), "ggml-compiler_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        from ggml_compiler_amd import ops

        h = {"ops": ops}
        if "pages" in st:
            h["batch"] = ops.PagedBatch(st["pages"], st["starts"], st["past"])
        if "data" in st:
            data = st["data"] if isinstance(st["data"], list) else [st["data"]]
            h["caches"] = [ops.PagedCache(st["n_pages"], st["page"], st["Hkv"], st["D"], d) for d in data]
        if "mask" in st:
            h["tree"] = ops.DraftTree(st["parents"], st["positions"], st["mask"])
        st["handles"] = h
    return st["handles"]


def _run_own(st):
    h = _handles(st)
    ops, kind = h["ops"], st["kind"]
    if kind == "tree":
        tree = ops.draft_tree(h["batch"], st["parents"], st["max_rows"], window=st["window"])
        return {"positions": tree.positions, "mask": tree.mask}
    if kind == "verify":
        path = ops.draft_verify(st["starts"], st["parents"], st["tokens"], st["logits"], st["coins"], draft_logits=st["draft"],
                                temperature=st["temperature"], max_rows=st["max_rows"], max_path=st["max_path"])
        return {"count": path.count, "rows": path.rows, "tokens": path.tokens}
    if kind == "move":
        ops.paged_move(h["caches"], h["batch"], st["count"], st["rows"])
        return st["data"]
    cache = h["caches"][0]
    if kind == "attn":
        return ops.paged_attn(cache, h["batch"], st["q"], st["scale"], max_rows=st["max_rows"], window=st["window"], tree=h["tree"])
    q = ops.paged_append(cache, h["batch"], st["k"], st["v"], q=st["q"], freqs=st["freqs"], positions=st["positions"])
    k, v = ops.paged_read(cache, h["batch"], st["n"])
    return {"q": q, "k": k, "v": v}


def run(state):
    if own:
        return _run_own(state)
    return {"tree": _tree_plain, "append": _append_plain, "attn": _attn_plain, "verify": _verify_plain,
            "move": _move_plain}[state["kind"]](state)


# ------------------------------------------------------------------- the definition, in 64 bits


def exact(case, seed):
    st = prepare(case, seed)
    starts = st["starts"].tolist()
    if case["kind"] == "verify":
        return _exact_verify(st, starts)
    past = st["past"].tolist()
    parents = st["parents"].tolist()
    lines = []  # each row's ancestors and itself, by number
    for a, b in zip(starts, starts[1:]):
        for j in range(b - a):
            up = parents[a + j]
            lines.append((lines[a + up] if 0 <= up < j else []) + [j])
    if case["kind"] == "tree":
        words, w = -(-st["max_rows"] // 32), case["window"] or len(lines) + 1
        mask = torch.zeros(len(lines), words, dtype=torch.int64)
        for r, line in enumerate(lines):
            for j in line[-w:]:
                mask[r, j // 32] += 1 << j % 32 if j % 32 < 31 else -(1 << 31)
        rows = [p for s, p in enumerate(past) for _ in range(starts[s + 1] - starts[s])]
        return {"positions": _int([p + len(line) - 1 for p, line in zip(rows, lines)]), "mask": mask.to(torch.int32).cuda()}
    D, Hkv, page = st["D"], st["Hkv"], st["page"]
    i = torch.arange(D, device="cuda")

    def places(s, slots):
        """Where the slots' values lie: bytes of keys, of values [Hkv, slots, D], and of their scales."""
        tile = ((st["pages"][s].long()[slots // page] * Hkv)[None] + torch.arange(Hkv, device="cuda")[:, None]) * (page // 32)
        tile = ((tile + (slots % page // 32)) * (36 * D))[..., None]
        t, low, block = (slots % 32)[:, None], i % (D // 2), i // 32
        kb = t * (D // 2) + low // 8 % 4 * (D // 8) + low // 32 * 8 + low % 8
        vb = 16 * D + low // 32 * 1024 + t // 8 * 256 + low % 16 * 16 + low // 16 % 2 * 8 + t % 8
        sb = 2 * (block * 32 + t // 8 * 8 + torch.tensor(ORDER, device="cuda")[t % 8])
        return tile + kb, tile + vb, tile + 32 * D + sb, tile + 34 * D + sb

    if case["kind"] == "move":
        count, rows = st["count"].tolist(), st["rows"].tolist()
        for data in st["data"]:
            old = data.clone()
            for s, m in enumerate(count):
                src = places(s, torch.tensor([past[s] + j for j in rows[s][:m]], device="cuda"))
                dst = places(s, torch.arange(past[s], past[s] + m, device="cuda"))
                for a, b in zip(src, dst):
                    data[b] = old[a]
                for a, b in zip(src[2:], dst[2:]):
                    data[b + 1] = old[a + 1]
        return st["data"]
    if case["kind"] == "append":
        depth = torch.tensor([len(line) - 1 for line in lines], device="cuda")
        first = torch.cat([torch.full((b - a,), p, device="cuda") for a, b, p in zip(starts, starts[1:], past)])
        half = st["n_dims"] // 2
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), (first + depth).double().outer(st["freqs"].double()))

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
    halves, out, G = st["data"].view(torch.float16), [], st["H"] // Hkv
    shift = torch.where(i < D // 2, 0, 4).to(torch.uint8)
    for s, p in enumerate(past):
        n = starts[s + 1] - starts[s]
        kb, vb, ks, vs = places(s, torch.arange(p + n, device="cuda"))
        k, v = ((((st["data"][c] >> shift) & 15).double() - 8) * halves[d // 2].double() for c, d in ((kb, ks), (vb, vs)))
        hidden = torch.ones(n, p + n, dtype=torch.bool)
        for j, line in enumerate(lines[starts[s]:starts[s + 1]]):
            keys = torch.cat([torch.arange(p), torch.tensor(line) + p])  # as many as its position, and itself
            hidden[j, keys[-case["window"]:] if case["window"] else keys] = False
        hidden, o = hidden.cuda(), []
        q = st["q"][starts[s]:starts[s + 1]].double()
        for h in range(st["H"]):
            x = (q[:, h] @ k[h // G].T) * st["scale"]
            o.append(torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ v[h // G])
        out.append(torch.stack(o, 1))
    return torch.cat(out)


def _exact_verify(st, starts):
    """One sequence after the other, what is left of the target's distribution renormalised after each draft that fell."""
    parents, tokens, coins = st["parents"].tolist(), st["tokens"].tolist(), st["coins"].tolist()
    P, count, rows, out = st["max_path"], [], [], []
    for a, b, t in zip(starts, starts[1:], st["temperature"].tolist()):
        path, said, at = [], [], 0 if b > a else None
        while at is not None and len(path) < P:
            path.append(at)
            below = [j for j in range(at + 1, b - a) if parents[a + j] == at]
            x = st["logits"][a + at].double()
            taken = None
            if t <= 0:
                best = int((x == x.max()).nonzero()[0, 0])
                taken = next((j for j in below if tokens[a + j] == best), None)
                said.append(best)
            else:
                left = torch.softmax(x / t, -1)
                q = torch.softmax(st["draft"][a + at].double() / t, -1) if st["draft"] is not None else None
                for j in below:
                    token = tokens[a + j]
                    if coins[a + j] * (1.0 if q is None else float(q[token])) < float(left[token]):
                        taken = j
                        said.append(token)
                        break
                    if q is None:
                        left[token] = 0.0
                    else:
                        left = (left - q).clamp(min=0)
                    left = left / left.sum()
                if taken is None:
                    sums = left.cumsum(0)
                    said.append(int(((sums > coins[a] * float(sums[-1])) & (left > 0)).nonzero()[0, 0]))
            at = taken
        count.append(len(path))
        rows.append(path + [-1] * (P - len(path)))
        out.append(said + [-1] * (P - len(said)))
    return {"count": _int(count), "rows": _int(rows), "tokens": _int(out)}
