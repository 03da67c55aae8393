"""Steps with drafted tokens (ops.draft_tree, paged_append with positions, paged_attn of a tree, draft_verify, paged_move)
against plain implementations: masks, positions, tokens and moved bytes equal, attention against float64, the drawn tokens'
distribution against the target's."""

import math

import numpy as np
import pytest
import torch
from test_gpu_paged import Case, check_attn, layout_bytes, q4_values, rotated

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------ helpers


def random_trees(rows, rng, near=4):
    """Parents of each sequence's rows: an earlier row, mostly a near one."""
    out = []
    for n in rows:
        out += [-1 if j == 0 else max(0, j - 1 - int(rng.integers(0, near))) for j in range(n)]
    return out


def lines_of(rows, parents):
    """Each row's ancestors and itself, by number."""
    lines, at = [], 0
    for n in rows:
        for j in range(n):
            p = parents[at + j]
            lines.append((lines[at + p] if 0 <= p < j else []) + [j])
        at += n
    return lines


def words_of(lines, words, window=0):
    m = np.zeros((len(lines), words), np.uint32)
    for r, line in enumerate(lines):
        for j in line[-window:] if window else line:
            m[r, j // 32] |= np.uint32(1 << j % 32)
    return m.view(np.int32)


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def batch_of(gops, rows, past, pages=1):
    starts = np.concatenate([[0], np.cumsum(rows)])
    return gops.PagedBatch(torch.zeros((len(rows), pages), dtype=torch.int32, device="cuda"), ints(starts), ints(past))


# ------------------------------------------------------------------------------------ trees


@pytest.mark.parametrize("rows,near", [([1], 1), ([7], 1), ([33], 40), ([64, 1, 0, 65, 17], 4), ([300], 3), ([1024], 1), ([1024], 1000),
                                       ([5] * 150, 2), ([257, 512], 8)])
@pytest.mark.parametrize("window", [0, 1, 3, 300])
def test_tree(gops, rows, near, window):
    rng = np.random.default_rng(sum(rows) + near)
    past = rng.integers(0, 1 << 20, len(rows))
    parents = random_trees(rows, rng, near)
    lines = lines_of(rows, parents)
    tree = gops.draft_tree(batch_of(gops, rows, past), ints(parents), max(rows), window=window)
    first = np.repeat(past, rows)
    assert tree.positions.tolist() == [int(p) + len(line) - 1 for p, line in zip(first, lines)]
    assert torch.equal(tree.mask, ints(words_of(lines, -(-max(rows) // 32), window)))


def test_tree_odd_parents_padding_and_wide_masks(gops):
    """Parents that are no earlier row's count as none; rows behind the last sequence and past max_rows stay as they are; a mask
    may be wider than the rows need."""
    rows, past = [6, 3, 8], [100, 0, 7]
    parents = [0, 5, 1, -7, 3, 99, 2, 0, -1, -1, 0, 1, 2, 3, 4, 5, 6] + [3, 3]
    parents[1] = 1  # itself
    lines = lines_of(rows, parents)
    tree = gops.DraftTree(ints(parents), torch.full((19,), 55, dtype=torch.int32, device="cuda"),
                          torch.full((19, 3), 55, dtype=torch.int32, device="cuda"))
    assert gops.draft_tree(batch_of(gops, rows, past), tree.parents, out=tree) is tree
    first = np.repeat(past, rows)
    assert tree.positions.tolist() == [int(p) + len(line) - 1 for p, line in zip(first, lines)] + [55, 55]
    assert torch.equal(tree.mask[:17], ints(words_of(lines, 3)))
    assert (tree.mask[17:] == 55).all()
    tree.positions.fill_(-9), tree.mask.fill_(-9)
    gops.draft_tree(batch_of(gops, rows, past), tree.parents, 6, out=tree)
    assert torch.equal(tree.mask[:15], ints(words_of(lines, 3))[:15])
    assert (tree.mask[15:] == -9).all() and (tree.positions[15:] == -9).all()


# ------------------------------------------------------------------------------------ append


@pytest.mark.parametrize("D,n_dims,H,Hkv,rows", [(128, 128, 4, 2, [5, 1, 9]), (64, 20, 6, 3, [3, 40]), (256, 256, 2, 1, [7]),
                                                 (128, 64, 32, 8, [150, 90]), (64, 64, 28, 4, [300, 250]), (256, 130, 16, 4, [200])])
def test_append_at_positions(gops, orc, D, n_dims, H, Hkv, rows):
    """Codes and scales of rows turned by positions that are not their slots, bit for bit, row by row and by eights."""
    past = [13 + 64 * s for s in range(len(rows))]
    c = Case(gops, rows, past, Hkv, D, 64, extra_rows=2)
    pos = c.rng.integers(0, 1 << 17, c.n).astype(np.int32)
    x = [c.rng.standard_normal((c.n, h, D)).astype(np.float32) for h in (H, Hkv, Hkv)]
    q, k, v = (torch.from_numpy(y).cuda() for y in x)
    freqs = gops.rope_freqs(n_dims, 10000.0)
    out = torch.full((c.n, H, D), 7.0, dtype=torch.float16, device="cuda")
    got = gops.paged_append(c.cache, c.batch(), k, v, q=q, freqs=freqs, q_out=out, positions=torch.from_numpy(pos).cuda())
    n = int(c.starts[-1])
    f = freqs.cpu().numpy()
    assert np.array_equal(got[:n].cpu().numpy(), rotated(x[0], pos, f)[:n].astype(np.float16)) and (out[n:] == 7).all()
    k2, v2 = gops.paged_read(c.cache, c.batch(), c.n)
    assert np.array_equal(k2[:n].cpu().numpy(), q4_values(orc, rotated(x[1], pos, f)[:n]))
    assert np.array_equal(v2[:n].cpu().numpy(), q4_values(orc, x[2][:n]))


def test_append_at_slots_is_append(gops):
    c = Case(gops, [5, 200], [77, 1], 8, 128, 64)
    k, v = (torch.randn(c.n, 8, 128, device="cuda") for _ in range(2))
    freqs = gops.rope_freqs(128, 500000.0)
    gops.paged_append(c.cache, c.batch(), k, v, freqs=freqs)
    want = c.cache.data.clone()
    c.cache.data.fill_(0xFF)
    pos = ints(np.concatenate([np.arange(77, 82), np.arange(1, 201)]))
    gops.paged_append(c.cache, c.batch(), k, v, freqs=freqs, positions=pos)
    assert torch.equal(c.cache.data, want)


# ------------------------------------------------------------------------------------ attention


def tree_reference(case, q, scale, lines, window=0, holes=(), max_rows=1 << 30):
    """float64, over the values that paged_read gave. lines: the rows of its sequence that each row sees."""
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    bound, G = 0.0, q.shape[1] // case.Hkv
    for s, (r, p) in enumerate(zip(case.rows, case.past)):
        if r == 0:
            continue
        k = case.k[case.key0[s]:case.key0[s + 1]].transpose(0, 1)
        v = case.v[case.key0[s]:case.key0[s + 1]].transpose(0, 1)
        rows = q[case.starts[s]:case.starts[s + 1]].double()
        seen = torch.zeros(r, p + r, dtype=torch.bool)
        for j, (at, line) in enumerate(lines[case.starts[s]:case.starts[s + 1]]):
            seen[j, max(0, at - window + 1) if window else 0:p] = True
            seen[j, [p + i for i in line if i < min(r, max_rows)]] = True
        for hs, pg in holes:
            if hs == s:
                seen[:, pg * case.page:(pg + 1) * case.page] = False
        seen = seen.cuda()
        v = torch.where(seen.any(0)[None, :, None], v, 0.0)
        for h in range(q.shape[1]):
            x = ((rows[:, h] @ k[h // G].T) * scale).masked_fill(~seen, -torch.inf)
            w = torch.exp(x - x.amax(-1, keepdim=True).nan_to_num(neginf=0.0))
            out[case.starts[s]:case.starts[s + 1], h] = w @ v[h // G] / w.sum(-1, keepdim=True).clamp(min=1e-300)
            bound = max(bound, float((rows[:, h].abs() @ torch.where(seen.any(0)[:, None], k[h // G], 0.0).abs().T).max()) * abs(scale))
    return out, bound


def run_tree(gops, case, G, parents=None, masks=None, positions=None, window=0, scale=None, holes=(), max_rows=None, seed=5, words=None):
    """Attention of trees, or of any masks (lists of the rows that each row sees), against float64."""
    H, D, n = G * case.Hkv, case.D, int(case.starts[-1])
    case.fill_past()
    q = (torch.randn(case.n, H, D, generator=torch.Generator().manual_seed(seed)) * 1.5).cuda().half()
    table = case.table.copy()
    for s, pg in holes:
        table[s, pg] = -1 if (s + pg) % 2 else case.n_pages
    batch = case.batch(table=table)
    first = np.repeat(case.past, case.rows)
    pad = [-1] * (case.n - n)
    if parents is not None:
        lines = lines_of(case.rows, parents)
        tree = gops.draft_tree(batch, ints(parents + pad), max(case.rows), window=window)
        positions = [int(p) + len(line) - 1 for p, line in zip(first, lines)]
        masks = [line[-window:] if window else line for line in lines]
    else:
        words = words or -(-max(case.rows) // 32)
        m = words_of(masks + [[]] * len(pad), words)
        positions = first if positions is None else positions
        tree = gops.DraftTree(ints([-1] * case.n), ints(list(positions) + pad), ints(m))
    scale = D ** -0.5 if scale is None else scale
    out = torch.full((case.n, H, D), 77.0, device="cuda")
    gops.paged_attn(case.cache, batch, q, scale, max_rows=max_rows, window=window, out=out, tree=tree)
    want, bound = tree_reference(case, q, scale, [(max(p, int(f)), m) for p, f, m in zip(positions, first, masks)], window, holes,
                                 max_rows or 1 << 30)
    assert (out[n:] == 77.0).all()  # rows of no sequence
    return out, want, bound


def check_tree(case, out, want, bound):
    n = int(case.starts[-1])
    check_attn(case, out[:n], want[:n], bound, max(p + r for r, p in zip(case.rows, case.past)))


@pytest.mark.parametrize("D,Hkv,G,rows,past,page", [
    (128, 2, 4, [26], [500], 64), (64, 2, 7, [6, 1, 33], [0, 31, 700], 32), (256, 1, 2, [9, 40], [100, 3], 128),
    (128, 8, 1, [64, 64, 5], [0, 1, 2], 64), (64, 1, 12, [130], [1000], 256), (128, 1, 3, [300], [37], 64),
    (256, 2, 4, [70, 1, 12], [2000, 5000, 0], 64), (128, 1, 4, [61], [9000], 256), (64, 2, 1, [1], [0], 32)])
@pytest.mark.parametrize("window", [0, 5, 400])
def test_attention_of_trees(gops, D, Hkv, G, rows, past, page, window):
    case = Case(gops, rows, past, Hkv, D, page, seed=D + sum(rows), extra_rows=2)
    out, want, bound = run_tree(gops, case, G, random_trees(rows, np.random.default_rng(len(rows)), 6), window=window)
    check_tree(case, out, want, bound)


def test_attention_of_a_chain_is_causal(gops):
    case = Case(gops, [9, 70, 1], [300, 64, 2000], 2, 128, 64)
    parents = [j - 1 for r in case.rows for j in range(r)]
    for window in (0, 50):
        out, want, bound = run_tree(gops, case, 4, parents, window=window)
        check_tree(case, out, want, bound)
        q = (torch.randn(case.n, 8, 128, generator=torch.Generator().manual_seed(5)) * 1.5).cuda().half()
        causal = gops.paged_attn(case.cache, case.batch(), q, 128 ** -0.5, window=window)
        check_attn(case, out, causal.double(), bound, 2100)


@pytest.mark.parametrize("D,G", [(128, 2), (64, 8), (256, 1)])
def test_attention_of_any_masks(gops, D, G):
    """Masks that are no tree's: rows seen ahead, rows that see no row, rows that see nothing at all (zeros), bits past the
    sequence's rows; rows that none sees are never appended and hold NaN scales."""
    rng = np.random.default_rng(D)
    rows, past = [40, 3, 1, 70], [0, 95, 0, 33]
    case = Case(gops, rows, past, 2, D, 32, seed=D)
    masks = []
    for s, r in enumerate(rows):
        hidden = {1, r - 2} if s in (0, 3) else set()
        for j in range(r):
            m = [i for i in range(r) if rng.random() < 0.3 and i not in hidden]
            masks.append([] if j % 5 == 2 or s == 2 else m + [r, r + 3, 95])
    spoil = [(s, i) for s in (0, 3) for i in (1, rows[s] - 2)]

    fill = case.fill_past

    def fill_and_spoil():
        fill()
        for s, i in spoil:
            case.cache.data[torch.from_numpy(layout_bytes(case, [(s, past[s] + i)])).cuda().flatten()] = 0xFF
    case.fill_past = fill_and_spoil
    out, want, bound = run_tree(gops, case, G, masks=masks, words=3)
    check_tree(case, out, want, bound)
    nothing = [r for r, m in enumerate(masks) if not m and (r < 40 or r == 43)]
    assert nothing and (out[nothing] == 0).all()


@pytest.mark.parametrize("window", [0, 70])
def test_attention_of_trees_missing_pages(gops, window):
    case = Case(gops, [20, 9], [200, 300], 2, 128, 32)
    out, want, bound = run_tree(gops, case, 4, random_trees(case.rows, np.random.default_rng(1)), window=window,
                                holes=[(0, 1), (0, 6), (1, 0), (1, 9)])
    check_tree(case, out, want, bound)


def test_attention_of_trees_positions_of_a_window(gops):
    """Positions that no tree of these rows has: below past (count as past), far ahead (nothing of the past is left)."""
    case = Case(gops, [4, 40], [90, 700], 1, 64, 32)
    positions = [0, 95, 1 << 30, 130] + [700 + 9 * j for j in range(40)]
    out, want, bound = run_tree(gops, case, 4, masks=[[j] for j in range(4)] + [[j] for j in range(40)], positions=positions, window=64)
    check_tree(case, out, want, bound)


def test_attention_of_trees_max_rows(gops):
    """Rows past max_rows are left as they are, and are not seen."""
    case = Case(gops, [40, 3], [100, 10], 2, 128, 64)
    out, want, bound = run_tree(gops, case, 2, masks=[list(range(j + 1)) for j in range(40)] + [[0, 1], [1, 2], [0]], max_rows=8, words=2)
    assert (out[8:40] == 77.0).all()
    keep = list(range(8)) + [40, 41, 42]
    check_attn(case, out[keep], want[keep], bound, 140)


@pytest.mark.parametrize("scale", [0.0, -0.09, 1e30])
def test_attention_of_trees_scales(gops, scale):
    case = Case(gops, [33, 2], [50, 0], 1, 64, 32)
    out, want, bound = run_tree(gops, case, 4, random_trees(case.rows, np.random.default_rng(2)), scale=scale)
    if scale == 1e30:  # the largest score alone
        assert torch.isfinite(out).all() and (out.double() - want).abs().max() <= 2.0 ** -18 * case.v.abs().max()
    else:
        check_tree(case, out, want, bound)


@pytest.mark.parametrize("window", [0, 6000])
@pytest.mark.parametrize("D,G", [(128, 4), (64, 8)])
def test_attention_of_trees_of_spread_lengths(gops, D, G, window):
    """Long splits of sequences of very different lengths, one of them without rows."""
    case = Case(gops, [40, 0, 33, 64, 1, 25, 40], [9000, 50, 300, 15000, 4000, 100, 9000], 8, D, 64, seed=D, extra_rows=1)
    out, want, bound = run_tree(gops, case, G, random_trees(case.rows, np.random.default_rng(G)), window=window)
    check_tree(case, out, want, bound)


def test_attention_of_a_long_tree(gops):
    """Past 2^16 keys, many splits, a tree over several of them."""
    case = Case(gops, [61], [70001], 1, 128, 256)
    out, want, bound = run_tree(gops, case, 4, random_trees(case.rows, np.random.default_rng(3)))
    check_tree(case, out, want, bound)


@pytest.mark.parametrize("D,Hkv,G,S,longest", [(64, 1, 2, 70, 3000), (128, 8, 2, 64, 1500), (128, 8, 4, 110, 1300), (256, 2, 1, 130, 200)])
def test_attention_of_more_trees_than_fit(gops, D, Hkv, G, S, longest):
    """More sequences than lanes, and more row tiles than workgroups that are resident at once; one of them long, so that some are split."""
    rng = np.random.default_rng(S)
    rows, past = [int(x) for x in rng.integers(0, 12, S)], [int(x) for x in rng.integers(0, 60, S)]
    rows[S // 2], past[S // 2] = 20, longest
    case = Case(gops, rows, past, Hkv, D, 64, seed=S, extra_rows=1)
    out, want, bound = run_tree(gops, case, G, random_trees(rows, rng), max_rows=20)
    check_tree(case, out, want, bound)


# ------------------------------------------------------------------------------------ verification


def reference(rows, parents, tokens, logits, coins, draft=None, temperature=None, max_path=None):
    """One sequence after the other in float64, what is left of the target's distribution renormalised after each draft that fell."""
    count, out_rows, out_tokens = [], [], []
    max_path, at0 = max_path or max(max(rows), 1), 0
    big = float(np.finfo(np.float32).max)

    def soft(x, t):
        x = np.minimum(np.where(np.isnan(x), -np.inf, x.astype(np.float64)), big)
        if x.max() == -np.inf:
            return np.zeros_like(x)
        with np.errstate(invalid="ignore"):
            w = np.where(x == -np.inf, 0.0, np.exp((x - x.max()) / t))
        return w / w.sum()

    for s, n in enumerate(rows):
        t = 1.0 if temperature is None else float(temperature[s])
        path, said, u = [], [], 0 if n else None
        while u is not None and len(path) < max_path:
            path.append(u)
            below = [j for j in range(u + 1, n) if parents[at0 + j] == u]
            x = logits[at0 + u]
            taken = token = None
            if not t > 0:
                y = np.minimum(np.where(np.isnan(x), -np.inf, x), big)
                token = int(y.argmax()) if y.max() > -np.inf else -1
                taken = next((j for j in below if tokens[at0 + j] == token), None) if token >= 0 else None
            else:
                p = soft(x, t)
                left, q = p.copy(), soft(draft[at0 + u], t) if draft is not None else None
                for j in below:
                    c = tokens[at0 + j]
                    good = 0 <= c < len(x)
                    if good and float(coins[at0 + j]) * (1.0 if q is None else q[c]) < left[c]:
                        taken, token = j, c
                        break
                    if q is not None:
                        left = np.maximum(left - q, 0)
                    elif good:
                        left[c] = 0
                    if left.sum() > 0:
                        left = left / left.sum()
                    elif q is None:
                        left = left * 0
                if taken is None:
                    left = left if left.sum() > 0 else p
                    sums = left.cumsum()
                    coin = min(max(float(coins[at0]), 0.0), 1 - 2.0 ** -24)
                    hit = np.flatnonzero((sums > coin * sums[-1]) & (left > 0))
                    token = int(hit[0]) if len(hit) else -1
            said.append(token)
            u = taken
        count.append(len(path))
        out_rows.append(path + [-1] * (max_path - len(path)))
        out_tokens.append(said + [-1] * (max_path - len(said)))
        at0 += n
    return count, out_rows, out_tokens


def peaked(rng, n, V):
    """Logits with a few tokens far ahead."""
    return (rng.standard_normal((n, V)) * 2 + 14 * rng.random((n, V)) ** (V / 8)).astype(np.float32)


def draws(rng, logits, t):
    """A token of each row's softmax(logits / t)."""
    z = logits / max(t, 0.05) - np.log(-np.log(rng.random(logits.shape).clip(1e-300, 1 - 1e-16)))
    return z.argmax(-1)


def make_verify(rows, V, drawn, near=3, seed=0, temps=(0.0, 0.7, 1.0, 1.3), noise=0.7):
    rng = np.random.default_rng(seed)
    n = sum(rows)
    parents = random_trees(rows, rng, near)
    temperature = rng.choice(temps, len(rows)).astype(np.float32)
    logits = peaked(rng, n, V)
    draft = (logits + noise * rng.standard_normal((n, V))).astype(np.float32)
    start = np.repeat(np.concatenate([[0], np.cumsum(rows)])[:-1], rows).astype(int)
    node = start + np.maximum(parents, 0)
    tokens = np.empty(n, np.int64)
    for r in range(n):
        t = temperature[np.searchsorted(np.cumsum(rows), r, side="right")]
        if drawn and t > 0:
            tokens[r] = draws(rng, draft[node[r]][None], t)[0]
        else:  # guesses: the likeliest, siblings different ones
            k = sum(1 for j in range(r) if node[j] == node[r] and j > node[r])
            tokens[r] = np.argsort(-draft[node[r]], kind="stable")[k % V]
    return parents, tokens, logits, rng.random(n).astype(np.float32), draft if drawn else None, temperature


def verify(gops, rows, parents, tokens, logits, coins, draft=None, temperature=None, max_rows=None, max_path=None, pad=0, extra=0):
    def rows_of(x):
        if x is None:
            return None
        y = torch.full((x.shape[0] + extra, x.shape[1] + pad), float("nan"), device="cuda")
        y[:x.shape[0], :x.shape[1]] = torch.from_numpy(x).cuda()
        return y[:, :x.shape[1]]
    more = lambda x, fill: ints(list(x) + [fill] * extra)  # noqa: E731
    path = gops.draft_verify(ints(np.concatenate([[0], np.cumsum(rows)])), more(parents, 0), more(tokens, 0), rows_of(logits),
                             torch.from_numpy(np.concatenate([coins, np.zeros(extra, np.float32)])).cuda(), draft_logits=rows_of(draft),
                             temperature=None if temperature is None else torch.from_numpy(temperature).cuda(), max_rows=max_rows,
                             max_path=max_path)
    return path.count.tolist(), path.rows.tolist(), path.tokens.tolist()


@pytest.mark.parametrize("rows,V,near", [([1], 1, 1), ([1], 5, 1), ([5], 7, 1), ([6, 1, 0, 9], 91, 3), ([4] * 3, 2048, 1), ([9, 20], 2049, 3),
                                         ([12, 5], 4096, 4), ([30, 7, 1], 32001, 4), ([5] * 12, 8191, 1), ([33], 16385, 30),
                                         ([3] * 150, 257, 2), ([70, 64, 65], 500, 3), ([2, 3], 128256, 1), ([40] * 9, 20000, 3)])
@pytest.mark.parametrize("drawn", [False, True])
def test_verify(gops, rows, V, near, drawn):
    a = make_verify(rows, V, drawn, near, seed=V + len(rows))
    assert verify(gops, rows, *a, pad=V % 3, extra=V % 2) == reference(rows, *a, max_path=sum(rows) + V % 2)


@pytest.mark.parametrize("drawn", [False, True])
def test_verify_paths_cut_short(gops, drawn):
    """max_path ends a path with the next draft's token; rows past max_rows are not looked at. (With fewer rows to a path than to a
    tree, sums of what is left go through several launches.)"""
    rows = [20, 7, 31, 1, 12]
    a = make_verify(rows, 40000, drawn, 3, seed=11, temps=(0.0, 0.9, 1.0), noise=0.9)
    for max_path in (1, 2, 3, 8, 30):
        assert verify(gops, rows, *a, max_path=max_path) == reference(rows, *a, max_path=max_path)
    cut = [min(r, 8) for r in rows]
    keep = np.concatenate([np.arange(r)[:8] + sum(rows[:s]) for s, r in enumerate(rows)])
    want = reference(cut, *[x[keep] if isinstance(x, np.ndarray) and len(x) == sum(rows) else [x[i] for i in keep] if isinstance(x, list)
                            else x for x in a], max_path=8)
    assert verify(gops, rows, *a, max_rows=8) == want


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("V", [60, 9000])
def test_verify_many_children(gops, drawn, V):
    """More children than lanes, most of which fall; drawn ones with the same token again and again."""
    rows = [200, 100, 3]
    rng = np.random.default_rng(V)
    n = sum(rows)
    logits = (rng.standard_normal((n, V)) * 0.5).astype(np.float32)
    draft = (rng.standard_normal((n, V)) * 0.5).astype(np.float32)
    parents = [-1] + [0] * 149 + [149] * 50 + [-1] + [0] * 99 + [-1, 0, 0]
    node = np.array([0] * 150 + [149] * 50 + [200] * 100 + [300] * 3)
    tokens = draws(rng, draft[node], 1.0) if drawn else rng.integers(-2, V + 2, n)
    coins = (1 - 0.3 * rng.random(n) ** 3).clip(0, 1 - 2.0 ** -24).astype(np.float32)
    a = (parents, tokens, logits, coins, draft if drawn else None)
    assert verify(gops, rows, *a, max_path=20) == reference(rows, *a, max_path=20)


def test_verify_long_chains(gops):
    """Paths of more rows than lanes: drafts that the target takes almost surely."""
    rows = [300, 1024, 65]
    rng = np.random.default_rng(4)
    n, V = sum(rows), 50
    logits = (rng.standard_normal((n, V))).astype(np.float32)
    parents = [j - 1 for r in rows for j in range(r)]
    tokens = rng.integers(0, V, n)
    logits[np.arange(n - 1), tokens[1:]] += 22
    logits[700, :] = 0
    coins = rng.random(n).astype(np.float32)
    coins[700] = 0.999
    a = (parents, tokens, logits, coins)
    want = reference(rows, *a)
    assert max(want[0]) > 64
    assert verify(gops, rows, *a, max_rows=1024) == want
    assert verify(gops, rows, *a, logits.copy(), max_rows=1024) == reference(rows, *a, logits)  # p == q: all stand


@pytest.mark.parametrize("drawn", [False, True])
def test_verify_special_logits(gops, drawn):
    """-inf (all but a few, all), NaN and +inf logits, the lowest float as a mask, huge and tiny temperatures, coins of 0 and next to 1,
    tokens that there are not."""
    V, inf, big = 3000, np.inf, float(np.finfo(np.float32).max)
    rng = np.random.default_rng(8)
    rows = [3] * 24
    parents, tokens, logits, coins, draft, _ = make_verify(rows, V, True, 1, seed=3)
    t = np.ones(24, np.float32)
    r = 3 * np.arange(24)
    logits[r[0]] = -inf
    logits[r[1], 5:] = -inf
    logits[r[2], :] = -inf
    logits[r[2], 2999] = -1e30
    logits[r[3], 100] = np.nan
    logits[r[4]] = np.nan
    logits[r[5], [7, 2500]] = inf
    logits[r[6]] = -big
    logits[r[6], 17] = -5.0
    logits[r[7]] = -big
    logits[r[8]] = -inf
    logits[r[8], [1, 2000]] = -big
    logits[r[9]] = rng.standard_normal(V) * 1e30
    t[9] = 1e29
    t[10], t[11], t[12], t[13], t[14], t[15] = 1e-30, 1e-38, inf, 1e30, -1.0, np.nan
    t[16] = 0.0
    logits[r[16], [40, 41]] = 100.0  # equals: the lowest
    t[17] = 0.0
    logits[r[17]] = np.nan
    coins[r[18]], coins[r[19]] = 0.0, 1 - 2.0 ** -24
    tokens[r[20] + 1], tokens[r[21] + 1] = -1, V
    draft[r[22]] = -inf
    draft[r[23], 10:] = -inf
    t[2] = 0.5
    logits[r[10], 3] = logits[r[10]].max() + 1
    logits[r[11], 3] = logits[r[11]].max() + 1
    a = (parents, tokens, logits, coins, draft if drawn else None, t)
    assert verify(gops, rows, *a, max_path=3) == reference(rows, *a)


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("V,rows", [(150001, [3, 6]), (700001, [5])])
def test_verify_large_vocabularies(gops, drawn, V, rows):
    """More parts than lanes: the total and the part are found 64 at a time, by coins from 0 to next to 1."""
    n = sum(rows)
    parents, tokens, logits, coins, draft, _ = make_verify(rows, V, True, 3, seed=V, temps=(1.0,))
    logits = logits * 0.3  # flat: any part may be the one
    draft = draft * 0.3
    for root in (0.0, 0.03, 0.5, 0.93, 1 - 2.0 ** -24):
        coins[np.cumsum([0] + rows[:-1])] = root
        a = (parents, tokens, logits, coins, draft if drawn else None)
        assert verify(gops, rows, *a, pad=3) == reference(rows, *a, max_path=n)
        assert verify(gops, rows, *a, max_path=2) == reference(rows, *a, max_path=2)


def test_verify_logits_past_32_bits(gops):
    """Rows of logits whose offsets pass 32 bits, and lie in one tensor with the drafter's."""
    rows, V, ld = [4, 2], 5000, 400_000_004
    a = make_verify(rows, V, True, 2, seed=21)
    n = sum(rows)
    both = torch.empty(n * ld, device="cuda").as_strided((n, ld), (ld, 1))
    logits, draft = both[:, 8:8 + V], both[:, 300_000_000:300_000_000 + V]
    logits.copy_(torch.from_numpy(a[2]))
    draft.copy_(torch.from_numpy(a[4]))
    path = gops.draft_verify(ints(np.concatenate([[0], np.cumsum(rows)])), ints(a[0]), ints(a[1]), logits, torch.from_numpy(a[3]).cuda(),
                             draft_logits=draft, temperature=torch.from_numpy(a[5]).cuda())
    assert (path.count.tolist(), path.rows.tolist(), path.tokens.tolist()) == reference(rows, *a, max_path=n)


def test_verify_what_is_left(gops):
    """Target and drafter far apart, equal, and equal but for one token: rows that fall until nothing or one token is left."""
    V, n = 1000, 12
    rng = np.random.default_rng(9)
    base = rng.standard_normal(V).astype(np.float32)
    rows = [4] * 3
    parents = [-1, 0, 0, 0] * 3
    logits, draft = np.tile(base, (n, 1)), np.tile(base, (n, 1))
    logits[0], draft[0] = base * 4, -base * 4
    draft[8, 123] += 3
    coins = np.full(n, 1 - 2.0 ** -24, np.float32)
    tokens = np.array([0, 5, 5, 7] * 2 + [0, 123, 123, 123])
    coins[[0, 4, 8]] = [0.3, 0.6, 0.9]
    a = (parents, tokens, logits, coins, draft)
    assert verify(gops, rows, *a, max_path=4) == reference(rows, *a)
    a = (parents, tokens, logits, coins, None)
    assert verify(gops, rows, *a, max_path=4) == reference(rows, *a)


def test_a_token_alone_is_the_inverse_of_the_distribution(gops):
    """One row a sequence and coins on a grid: each token as often as its probability, to one step of the grid a border."""
    V, N = 37, 1 << 14
    rng = np.random.default_rng(1)
    x = (rng.standard_normal(V) * 2).astype(np.float32)
    coins = ((np.arange(N) + 0.5) / N).astype(np.float32)
    logits = torch.from_numpy(x).cuda()[None].expand(N, V).contiguous()
    path = gops.draft_verify(ints(np.arange(N + 1)), ints([-1] * N), ints([0] * N), logits, torch.from_numpy(coins).cuda(), max_rows=1)
    p = np.exp(x.astype(np.float64) - x.max())
    p /= p.sum()
    got = np.bincount(path.tokens[:, 0].cpu().numpy(), minlength=V) / N
    assert np.abs(got - p).max() <= 1.01 / N and (path.count == 1).all()


@pytest.mark.parametrize("drawn,kids", [(True, 1), (True, 2), (False, 2)])
def test_tokens_are_distributed_as_the_target(gops, drawn, kids):
    """The first token after the root over all drafts (drawn ones by their probabilities) and a grid of coins: p, whatever q is.
    Each (draft, coin of the draft) cell of a G^(kids + 1) grid is off by a step a border: G drafts' borders and V tokens'."""
    V, G = 5, 24
    rng = np.random.default_rng(2)
    x, y = rng.standard_normal(V).astype(np.float32) * 1.5, rng.standard_normal(V).astype(np.float32) * 1.5
    p, q = np.exp(x.astype(np.float64)), np.exp(y.astype(np.float64))
    p, q = p / p.sum(), q / q.sum()
    tokens = [(c,) for c in range(V)] if kids == 1 else [(c, d) for c in range(V) for d in range(V)]
    weight = np.array([math.prod(q[c] for c in cs) for cs in tokens]) if drawn else None
    if not drawn:
        tokens = [(1, 3)]
        weight = np.ones(1)
    grid = (np.stack(np.meshgrid(*[np.arange(G)] * (kids + 1), indexing="ij"), -1).reshape(-1, kids + 1) + 0.5) / G
    S, n = len(tokens) * len(grid), kids + 1
    coins = np.tile(grid, (len(tokens), 1)).astype(np.float32).reshape(-1)
    toks = np.concatenate([[0, *cs] * len(grid) for cs in tokens])
    logits, draft = (torch.from_numpy(z).cuda()[None].expand(S * n, V).contiguous() for z in (x, y))
    path = gops.draft_verify(ints(n * np.arange(S + 1)), ints([-1] + [0] * kids).repeat(S), ints(toks), logits, torch.from_numpy(coins).cuda(),
                             draft_logits=draft if drawn else None, max_rows=n, max_path=2)
    got = np.zeros(V)
    np.add.at(got, path.tokens[:, 0].cpu().numpy(), np.repeat(weight, len(grid)) / len(grid))
    assert abs(got.sum() - 1) < 1e-9 and np.abs(got - p).max() <= (kids + 1) / G


def test_verify_more_sequences_than_a_list_of_lanes(gops):
    """Two thousand sequences, most with something left."""
    rows = [2] * 2000
    rng = np.random.default_rng(5)
    n, V = 4000, 300
    logits, draft = (rng.standard_normal((n, V)).astype(np.float32) * 2 for _ in range(2))
    parents = [-1, 0] * 2000
    tokens = np.repeat(draws(rng, draft[::2], 1.0), 2)
    a = (parents, tokens, logits, rng.random(n).astype(np.float32), draft)
    assert verify(gops, rows, *a, max_rows=2) == reference(rows, *a)


# ------------------------------------------------------------------------------------ move


@pytest.mark.parametrize("D,Hkv,page", [(64, 3, 32), (128, 2, 64), (256, 1, 128)])
def test_move(gops, D, Hkv, page):
    """Whole bytes, in every layer; entries below their own number, sources and targets without a page, and entries past count move
    nothing; sources are as before the call."""
    rows, past = [30, 5, 0, 12], [61, 0, 7, 95]
    case = Case(gops, rows, past, Hkv, D, page)
    table = case.table.copy()
    path = np.array([[0, 1, 5, 4, 5, 29], [2, 3, 4, 1, 9, 9], [1, 2, 3, 4, 5, 6], [0, 3, 4, 9, 10, 11]], np.int32)
    path[0, 4] = 3                                    # below its number
    path[3, 5] = 4000                                 # past the table
    count = np.array([6, 9, 0, 6], np.int32)          # more than there are columns
    table[3, (95 + 10) // page] = -1 if (95 + 10) // page != 95 // page else table[3, (95 + 10) // page]
    layers = [gops.PagedCache(case.n_pages, page, Hkv, D, torch.randint(0, 256, (case.cache.data.numel(),), dtype=torch.uint8, device="cuda"))
              for _ in range(3)]
    want = [c.data.clone() for c in layers]
    gops.paged_move(layers, case.batch(table=table), ints(count), ints(np.concatenate([path, path], 1))[:, :6])

    def there(s, slot):
        return slot // page < table.shape[1] and 0 <= table[s, slot // page] < case.n_pages

    for c, w in zip(layers, want):
        old = w.clone()
        for s in range(4):
            for i in range(min(count[s], 6)):
                src, dst = past[s] + int(path[s, i]), past[s] + i
                if path[s, i] >= i and there(s, src) and there(s, dst):
                    a, b = (torch.from_numpy(layout_bytes(case, [(s, x)])).cuda().flatten() for x in (src, dst))
                    w[b] = old[a]
        assert torch.equal(c.data, w)


def test_move_in_many_layers(gops):
    """More caches than a launch takes."""
    case = Case(gops, [9], [30], 1, 64, 32)
    layers = [gops.PagedCache(case.n_pages, 32, 1, 64, torch.randint(0, 256, (case.cache.data.numel(),), dtype=torch.uint8, device="cuda"))
              for _ in range(131)]
    want = [c.data.clone() for c in layers]
    gops.paged_move(layers, case.batch(), ints([2]), ints([[0, 8]]))
    a, b = (torch.from_numpy(layout_bytes(case, [(0, x)])).cuda().flatten() for x in (38, 31))
    for c, w in zip(layers, want):
        w[b] = w[a]
        assert torch.equal(c.data, w)


def test_step_in_a_cache_past_four_gigabytes(gops):
    """Append at positions, tree attention and move at page offsets past 32 bits: the bytes of a small cache."""
    D, Hkv, page, rows, past = 256, 8, 256, 40, 500
    size = page * Hkv * 288
    n_pages = (5 << 30) // size
    big, small = gops.PagedCache.new(n_pages, page, Hkv, D), gops.PagedCache.new(3, page, Hkv, D)
    assert big.data.numel() > 1 << 32
    at = [n_pages - 1, 3, n_pages - 2]
    starts, before = ints([0, rows]), ints([past])
    batches = gops.PagedBatch(ints([at]), starts, before), gops.PagedBatch(ints([[0, 1, 2]]), starts, before)
    parents = ints(random_trees([rows], np.random.default_rng(2)))
    g = torch.Generator().manual_seed(3)
    k0, v0 = (torch.randn((past, Hkv, D), generator=g).cuda() for _ in range(2))
    k, v = (torch.randn((rows, Hkv, D), generator=g).cuda() for _ in range(2))
    freqs, outs = gops.rope_freqs(D, 10000.0), []
    for cache, b in zip((big, small), batches):
        gops.paged_append(cache, gops.PagedBatch(b.pages, ints([0, past]), ints([0])), k0, v0)
        tree = gops.draft_tree(b, parents)
        q = gops.paged_append(cache, b, k, v, q=k, freqs=freqs, positions=tree.positions)
        outs.append(gops.paged_attn(cache, b, q, 1 / 16, tree=tree))
        gops.paged_move(cache, b, ints([5]), ints([[0, 2, 9, 30, 39]]))
    assert outs[0].isfinite().all() and torch.equal(*outs)
    for i, pg in enumerate(at):
        assert torch.equal(big.data[pg * size:(pg + 1) * size], small.data[i * size:(i + 1) * size])


# ------------------------------------------------------------------------------------ together


class Server:
    """Two layers of a toy model whose hidden rows are functions of token and position alone, so that a tree's rows can be had one by
    one as well."""

    def __init__(self, gops, S, V=64, D=64, Hkv=2, H=4, seed=0, page=32, n_pages=40):
        g = torch.Generator().manual_seed(seed)
        self.gops, self.S, self.V, self.D, self.Hkv, self.H = gops, S, V, D, Hkv, H
        self.emb = torch.randn(V, (H + 2 * Hkv) * D, generator=g).cuda()
        self.out = (torch.randn(H * D, V, generator=g) * 0.4).cuda()
        self.freqs = gops.rope_freqs(D, 10000.0)
        self.layers = [gops.PagedCache.new(n_pages, page, Hkv, D) for _ in range(2)]
        for c in self.layers:
            c.data.fill_(0xFF)
        self.pages = torch.randperm(n_pages, generator=g)[:S * (n_pages // S)].view(S, -1).to(torch.int32).cuda()

    def qkv(self, tokens):
        x = self.emb[tokens.long()].view(-1, self.H + 2 * self.Hkv, self.D)
        return x[:, :self.H], x[:, self.H:self.H + self.Hkv], x[:, self.H + self.Hkv:]

    def step(self, batch, tokens, tree=None, max_rows=None):
        """Logits of the rows."""
        total = 0
        for i, c in enumerate(self.layers):
            q, k, v = self.qkv((tokens + i) % self.V)
            q16 = self.gops.paged_append(c, batch, k, v, q=q, freqs=self.freqs, positions=None if tree is None else tree.positions)
            total = total + self.gops.paged_attn(c, batch, q16, self.D ** -0.5, max_rows=max_rows, tree=tree)
        return total.reshape(total.shape[0], -1) @ self.out


def test_drafted_decoding_equals_one_token_at_a_time(gops):
    """Greedy decoding of three sequences by trees of guesses, some of them right: the same tokens, and the same caches, as one token
    a step."""
    S, steps = 3, 14
    plain, fast = Server(gops, S), Server(gops, S)
    prompts = [[5, 9, 1, 33], [7], [60, 2, 2, 2, 8, 40]]
    prompt = ints(sum(prompts, []))
    starts = ints(np.concatenate([[0], np.cumsum([len(p) - 1 for p in prompts])]))
    keep = ints([t for p in prompts for t in p[:-1]])
    for m in (plain, fast):  # all but the last token of each prompt
        m.step(gops.PagedBatch(m.pages, starts, ints([0] * S)), keep)
    assert prompt.numel() == 11
    past = [len(p) - 1 for p in prompts]
    truth, cur, at = [[] for _ in range(S)], [p[-1] for p in prompts], list(past)
    ones = ints(np.arange(S + 1))
    for _ in range(steps + 8):
        logits = plain.step(gops.PagedBatch(plain.pages, ones, ints(at)), ints(cur), max_rows=1)
        cur = logits.argmax(-1).tolist()
        at = [a + 1 for a in at]
        for s in range(S):
            truth[s].append(cur[s])
    rng = np.random.default_rng(0)
    said, cur, at = [[] for _ in range(S)], [p[-1] for p in prompts], list(past)
    most = 0
    while min(len(x) for x in said) < steps:
        rows, parents, tokens = [], [], []
        for s in range(S):
            right = truth[s][len(said[s]):len(said[s]) + int(rng.integers(0, 4))]
            t, p = [cur[s]], [-1]
            node = 0
            for x in right:  # a wrong guess and the right one at each level
                t += [(x + 1) % 64, x]
                p += [node, node]
                node = len(t) - 1
            t += [3, 4]
            p += [node, node]
            rows.append(len(t)), parents.extend(p), tokens.extend(t)
        batch = gops.PagedBatch(fast.pages, ints(np.concatenate([[0], np.cumsum(rows)])), ints(at))
        tree = gops.draft_tree(batch, ints(parents), max(rows))
        logits = fast.step(batch, ints(tokens), tree, max(rows))
        path = gops.draft_verify(batch.starts, tree.parents, ints(tokens), logits, torch.zeros(sum(rows), device="cuda"),
                                 temperature=torch.zeros(S, device="cuda"), max_rows=max(rows))
        gops.paged_move(fast.layers, batch, path.count, path.rows)
        for s, n in enumerate(path.count.tolist()):
            new = path.tokens[s, :n].tolist()
            said[s] += new
            cur[s], at[s], most = new[-1], at[s] + n, max(most, n)
    assert most > 2
    for s in range(S):
        assert said[s][:steps] == truth[s][:steps]
        n = past[s] + steps - 1  # tokens whose keys both have
        b = [gops.PagedBatch(m.pages[s:s + 1], ints([0, n]), ints([0])) for m in (plain, fast)]
        for c0, c1 in zip(plain.layers, fast.layers):
            x, y = gops.paged_read(c0, b[0], n), gops.paged_read(c1, b[1], n)
            assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])


def test_captured_step_follows_its_inputs(gops):
    """A whole step in one graph: replayed over other trees, tokens, lengths and coins, with eager work between, each replay as the
    eager step. Two graphs share nothing but their inputs."""
    S, R, V = 3, 12, 3000
    m = Server(gops, S, V=V, seed=3)
    n = S * R
    starts, past, parents, tokens = ints([0] * (S + 1)), ints([0] * S), ints([-1] * n), ints([0] * n)
    coins, temperature = torch.zeros(n, device="cuda"), torch.ones(S, device="cuda")
    draft = torch.randn(n, V, device="cuda")
    batch = gops.PagedBatch(m.pages, starts, past)
    spare = [c.data.clone() for c in m.layers]

    def step(with_draft):
        tree = gops.draft_tree(batch, parents, R)
        logits = m.step(batch, tokens, tree, R)
        path = gops.draft_verify(starts, parents, tokens, logits, coins, draft_logits=draft if with_draft else None,
                                 temperature=temperature, max_rows=R, max_path=6)
        gops.paged_move(m.layers, batch, path.count, path.rows)
        return tree, logits, path

    def set_inputs(seed):
        rng = np.random.default_rng(seed)
        rows = [int(rng.integers(0, R + 1)) for _ in range(S)]
        p = random_trees(rows, rng, 3)
        pad = n - sum(rows)
        starts.copy_(ints(np.concatenate([[0], np.cumsum(rows)])))
        past.copy_(ints(rng.integers(0, 100, S)))
        parents.copy_(ints(p + [0] * pad))
        tokens.copy_(ints(rng.integers(0, V, n)))
        coins.copy_(torch.from_numpy((rng.random(n) ** 4).astype(np.float32)))
        temperature.copy_(torch.from_numpy(rng.choice([0.0, 0.8, 1.0], S).astype(np.float32)))
        draft.copy_(torch.from_numpy(rng.standard_normal((n, V)).astype(np.float32)))
        for c, d in zip(m.layers, spare):
            c.data.copy_(d)
        return sum(rows)

    # a past that is there: all slots appended once
    slots = m.pages.shape[1] * 32
    all_rows = gops.PagedBatch(m.pages, ints(slots * np.arange(S + 1)), ints([0] * S))
    m.step(all_rows, ints(np.random.default_rng(1).integers(0, V, slots * S)))
    for c, d in zip(m.layers, spare):
        d.copy_(c.data)
    graphs = []
    for with_draft in (False, True):
        set_inputs(0)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(with_draft)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(with_draft)
        graphs.append((g, out, with_draft))
    for seed in range(1, 8):
        for g, (tree, logits, path), with_draft in graphs:
            used = set_inputs(seed)
            g.replay()
            torch.cuda.synchronize()
            got = [tree.positions[:used].clone(), tree.mask[:used].clone(), logits[:used].clone(), path.count.clone(), path.rows.clone(),
                   path.tokens.clone(), *[c.data.clone() for c in m.layers]]
            set_inputs(seed)
            t2, l2, p2 = step(with_draft)
            want = [t2.positions[:used], t2.mask[:used], l2[:used], p2.count, p2.rows, p2.tokens, *[c.data for c in m.layers]]
            torch.cuda.synchronize()
            for x, y in zip(got, want):
                assert torch.equal(x, y)


def test_two_streams_at_once(gops):
    rows = [40] * 6
    cases = [make_verify(rows, 30000, True, 3, seed=s) for s in (1, 2)]
    want = [reference(rows, *a) for a in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    up = [[torch.from_numpy(np.asarray(x, np.int32 if i < 2 else np.float32)).cuda() for i, x in enumerate(a)] for a in cases]
    starts = ints(np.concatenate([[0], np.cumsum(rows)]))
    torch.cuda.synchronize()
    out = [[], []]
    for _ in range(5):
        for i, (s, (p, t, x, c, d, temp)) in enumerate(zip(streams, up)):
            with torch.cuda.stream(s):
                out[i].append(gops.draft_verify(starts, p, t, x, c, draft_logits=d, temperature=temp, max_rows=40))
    torch.cuda.synchronize()
    for got, w in zip(out, want):
        for path in got:
            assert (path.count.tolist(), path.rows.tolist(), path.tokens.tolist()) == w


def test_refusals_on_the_device(gops):
    c = Case(gops, [4, 3], [5, 0], 2, 64, 32)
    b = c.batch()
    k = torch.randn(7, 2, 64, device="cuda")
    with pytest.raises(ValueError, match="positions must be"):
        gops.paged_append(c.cache, b, k, k, positions=torch.zeros(7, device="cuda"))
    with pytest.raises(ValueError, match="positions must be contiguous"):
        gops.paged_append(c.cache, b, k, k, positions=ints([0] * 6))
    tree = gops.draft_tree(b, ints([-1, 0, 0, 1, -1, 0, 1]), 4)
    q = torch.zeros(8, 4, 64, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError, match="tree of 7 rows"):
        gops.paged_attn(c.cache, b, q, 0.1, tree=tree)
    with pytest.raises(ValueError, match="parents must be"):
        gops.draft_tree(b, torch.zeros(7, device="cuda"))
    with pytest.raises(ValueError, match="max_rows"):
        gops.draft_tree(b, ints([0] * 2000), 1025)
    with pytest.raises(ValueError, match="other parents"):
        gops.draft_tree(b, ints([0] * 7), out=tree)
    with pytest.raises(ValueError, match="window"):
        gops.draft_tree(b, tree.parents, 4, window=-1)
    with pytest.raises(gops.GcqError, match="past the mask's bits"):
        gops.paged_attn(c.cache, c.batch(), torch.zeros(40, 4, 64, dtype=torch.float16, device="cuda"), 0.1, max_rows=40, tree=gops.DraftTree(
            ints([0] * 40), ints([0] * 40), ints([[0]] * 40)))
    for bad in ((7, 0), (7, 33)):
        with pytest.raises(ValueError, match="1 to 32 words"):
            gops.DraftTree(tree.parents, tree.positions, torch.zeros(bad, dtype=torch.int32, device="cuda"))
    n = 7
    good = {"starts": ints([0, 4, 7]), "parents": tree.parents, "tokens": ints([0] * n), "logits": torch.zeros(n, 9, device="cuda"),
            "coins": torch.zeros(n, device="cuda")}
    for bad, text in (({"starts": ints([0])}, "starts"), ({"tokens": ints([0] * 6)}, "tokens"), ({"coins": torch.zeros(6, device="cuda")}, "coins"),
                      ({"logits": torch.zeros(9, n, device="cuda").T}, "logits"), ({"logits": torch.zeros(n, 9, device="cuda").half()}, "logits"),
                      ({"draft_logits": torch.zeros(n, 8, device="cuda")}, "draft_logits"), ({"draft_logits": torch.zeros(n, 9)}, "draft_logits"),
                      ({"temperature": torch.ones(3, device="cuda")}, "temperature"), ({"max_path": 0}, "max_path")):
        with pytest.raises(ValueError, match=text):
            gops.draft_verify(**(good | bad))
    with pytest.raises(gops.GcqError, match="max_rows"):
        gops.draft_verify(**(good | {"max_rows": 0, "max_path": 1}))
    with pytest.raises(ValueError, match="at least one cache"):
        gops.paged_move([], b, ints([1, 1]), ints([[0], [0]]))
    with pytest.raises(ValueError, match="count must be"):
        gops.paged_move(c.cache, b, ints([1]), ints([[0], [0]]))
    with pytest.raises(ValueError, match="rows must be"):
        gops.paged_move(c.cache, b, ints([1, 1]), ints([[0, 1]]))
    with pytest.raises(gops.GcqError, match="one shape"):
        gops.paged_move([c.cache, gops.PagedCache.new(1, 32, 2, 64)], b, ints([1, 1]), ints([[0], [0]]))


def test_nothing_to_do(gops):
    b = batch_of(gops, [0, 0], [3, 0])
    e = ints([]).to(torch.int32)
    tree = gops.draft_tree(b, e)
    assert tree.mask.shape == (0, 1)
    path = gops.draft_verify(b.starts, e, e, torch.zeros(0, 50, device="cuda"), torch.zeros(0, device="cuda"), max_path=3)
    assert path.count.tolist() == [0, 0] and (path.rows == -1).all() and (path.tokens == -1).all()


# ------------------------------------------------------------- long splits of several sequences


def check_long(gops, D, Hkv, G, rows, past, page=64, window=0):
    """Trees over long lines, their past drawn on the device."""
    case = Case(gops, rows, past, Hkv, D, page, seed=D)

    def fill():
        total = [p + r for p, r in zip(past, rows)]
        g = torch.Generator(device="cuda").manual_seed(D + sum(past))
        k, v = (torch.randn((sum(total), Hkv, D), generator=g, device="cuda") for _ in range(2))
        b = case.batch(total, [0] * len(total))
        gops.paged_append(case.cache, b, k, v)
        case.k, case.v = (x.double() for x in gops.paged_read(case.cache, b, sum(total)))
        case.key0 = np.concatenate([[0], np.cumsum(total)])
    case.fill_past = fill
    out, want, bound = run_tree(gops, case, G, random_trees(rows, np.random.default_rng(D)), window=window, max_rows=max(rows))
    assert not (out == 77.0).any()  # every row is written
    check_tree(case, out, want, bound)


@pytest.mark.parametrize("D,Hkv,G,rows,past,window", [
    (128, 4, 8, [32] * 5, [100000] * 4 + [1000], 0), (256, 8, 4, [32] * 7, [30000] + [200] * 6, 0),
    (128, 8, 4, [38, 20, 49, 35], [76116, 41908, 31893, 63026], 0), (256, 8, 2, [44, 40, 40, 37, 39], [1057, 44721, 28100, 7659, 16044], 0),
    (256, 2, 8, [42, 41, 41, 40], [4358, 4528, 4462, 3610], 4096), (256, 2, 8, [34, 22, 17, 23], [9014, 120, 45050, 31239], 20000)])
def test_attention_of_trees_nearly_as_many_as_fit(gops, D, Hkv, G, rows, past, window):
    """More workgroups than are resident at once, the last 256 of the grid not all there."""
    check_long(gops, D, Hkv, G, rows, past, window=window)


@pytest.mark.parametrize("D,Hkv,G,rows,past,window", [
    (128, 8, 4, [4, 4], [130000, 5000], 0), (128, 8, 4, [4, 4], [70000, 70000], 0), (256, 8, 4, [4, 4], [36000, 36000], 0),
    (64, 8, 1, [2, 2, 1], [67121, 68882, 79389], 0), (128, 8, 4, [1, 1], [84693, 96073], 0), (256, 8, 4, [4, 3, 4], [9028, 50329, 40970], 0),
    (128, 8, 4, [5, 5, 5], [90000, 100000, 110000], 60000)])
def test_attention_of_few_rows_behind_long_lines(gops, D, Hkv, G, rows, past, window):
    """More splits to a row tile than there are row tiles, their workgroups in either order."""
    check_long(gops, D, Hkv, G, rows, past, window=window)


# ------------------------------------------------------------- draws of many workgroups at once


@pytest.mark.parametrize("kids", [0, 2])
def test_draws_are_the_same_in_every_wavefront(gops, kids):
    """Flat distributions over many parts, which each wavefront of a draw's workgroup finds for itself: single rows and guesses that
    fall, more sequences than workgroups that are resident, beside a second stream's."""
    S, V = 700, 20011
    rng = np.random.default_rng(kids)
    rows = [1 + kids] * S
    parents = ([-1] + [0] * kids) * S
    tokens = rng.integers(0, V, S * (1 + kids))
    logits = np.repeat((rng.standard_normal((S, V)) * 0.5).astype(np.float32), 1 + kids, 0)
    coins = rng.random(len(tokens)).astype(np.float32)
    a = (parents, tokens, logits, coins)
    want = reference(rows, *a, max_path=1 + kids)
    up = [ints(np.concatenate([[0], np.cumsum(rows)])), ints(parents), ints(tokens), torch.from_numpy(logits).cuda(), torch.from_numpy(coins).cuda()]
    torch.cuda.synchronize()
    streams, out = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                out.append(gops.draft_verify(*up, max_rows=1 + kids))
    torch.cuda.synchronize()
    for path in out:
        assert (path.count.tolist(), path.rows.tolist(), path.tokens.tolist()) == want


@pytest.mark.parametrize("S,V", [(300, 5003), (40, 40000)])
def test_paths_that_go_on_behind_fallen_drafts(gops, S, V):
    """Drawn trees most of whose first children fall and a later one stands, so that paths go on, and end in rows without children, within
    the launches that draw: the same in every call, on two streams at once."""
    rng = np.random.default_rng(S)
    rows = [9] * S
    parents = [-1, 0, 0, 0, 0, 1, 2, 3, 4] * S  # four children, one more behind each
    start = 9 * np.repeat(np.arange(S), 9)
    base = (rng.standard_normal((S, V)) * 0.8).astype(np.float32)
    logits = np.repeat(base, 9, 0)
    draft = np.repeat((base + 1.2 * rng.standard_normal((S, V))).astype(np.float32), 9, 0)
    tokens = np.array([draws(rng, draft[r:r + 1], 1.0)[0] for r in start + np.maximum(parents, 0)])
    coins = np.where(np.tile(np.arange(9), S) < 3, 0.8 + 0.2 * rng.random(9 * S), 0.2 * rng.random(9 * S)).astype(np.float32)
    a = (parents, tokens, logits, coins, draft)
    want = reference(rows, *a, max_path=4)
    third = sum(r[1] >= 2 for r in want[1])  # behind a draft that fell
    assert third > S // 5 and sum(c == 3 for c in want[0]) > S // 8
    up = [ints(np.concatenate([[0], np.cumsum(rows)])), ints(parents), ints(tokens), torch.from_numpy(logits).cuda(), torch.from_numpy(coins).cuda()]
    more = torch.from_numpy(draft).cuda()
    torch.cuda.synchronize()
    streams, out = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                out.append(gops.draft_verify(*up, draft_logits=more, max_rows=9, max_path=4))
    torch.cuda.synchronize()
    for path in out:
        assert (path.count.tolist(), path.rows.tolist(), path.tokens.tolist()) == want


def test_verify_more_rows_than_threads_of_31_bits(gops):
    """A few trees before 2^25 rows of none: 64 threads a row pass 2^31."""
    rows, V, n = [3, 1, 0, 6] * 20, 5, (1 << 25) + 9
    a = make_verify(rows, V, False, 2, seed=6)
    up = []
    for x, dtype in ((a[0], torch.int32), (a[1], torch.int32), (a[2], torch.float32), (a[3], torch.float32)):
        x = torch.tensor(np.asarray(x), dtype=dtype, device="cuda")
        y = torch.zeros((n, *x.shape[1:]), dtype=dtype, device="cuda")
        y[:len(x)] = x
        up.append(y)
    path = gops.draft_verify(ints(np.concatenate([[0], np.cumsum(rows)])), *up, temperature=torch.from_numpy(a[5]).cuda(), max_rows=6, max_path=4)
    assert (path.count.tolist(), path.rows.tolist(), path.tokens.tolist()) == reference(rows, *a, max_path=4)


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("bits", [0x7fc00000, 0x7f800001, 0xff812345], ids=["quiet", "signalling", "signalling-payload"])
def test_verify_nans_beside_each_other(gops, bits, drawn):
    """NaNs of either kind in one, two, three and four of the columns that a thread has at a time, from the first ones to a row's last, of
    the target's rows and the drafter's: as -inf."""
    rng = np.random.default_rng(bits & 0xff)
    V, rows = 5001, [3] * 32
    parents, tokens, logits, coins, draft, t = make_verify(rows, V, True, 1, seed=31)
    nan = np.array([bits], np.uint32).view(np.float32)[0]

    def spoil(x):
        y = x.view(np.uint32)
        for r in range(len(x)):
            for at in [0, 4 * int(rng.integers(1, 900)), 4092, 5000 // 4 * 4 - 4]:
                cols = rng.permutation(4)[:1 + (r + at // 4) % 4]
                y[r, at + cols] = bits
        return x
    a = (parents, tokens, spoil(logits), coins, spoil(draft) if drawn else None, t)
    assert np.isnan(nan) and np.isnan(logits).sum() > 3 * len(logits)
    assert verify(gops, rows, *a, max_path=3) == reference(rows, *a, max_path=3)


def test_move_without_starts(gops):
    """Through the C call: a batch whose starts are NULL."""
    import ctypes

    from ggml_compiler_amd import _lib
    case = Case(gops, [9], [30], 1, 64, 32)
    cache = gops.PagedCache(case.n_pages, 32, 1, 64, torch.randint(0, 256, (case.cache.data.numel(),), dtype=torch.uint8, device="cuda"))
    batch, count, rows, want = case.batch(), ints([2]), ints([[0, 8]]), cache.data.clone()
    b = type(batch._c).from_buffer_copy(batch._c)
    b.starts = None
    at = (ctypes.c_void_p * 1)(cache._at)
    _lib.check(_lib.load().gcq_paged_move(at, 1, ctypes.addressof(b), count.data_ptr(), rows.data_ptr(), 2, 2,
                                          torch.cuda.current_stream().cuda_stream))
    x, y = (torch.from_numpy(layout_bytes(case, [(0, p)])).cuda().flatten() for p in (38, 31))
    want[y] = want[x]
    assert torch.equal(cache.data, want)


@pytest.mark.parametrize("drawn,kids,V,t,pad", [(True, 1, 5, 1.0, 0), (True, 1, 37, 0.7, 0), (True, 2, 6, 1.0, 0), (True, 2, 5, 1.6, 3), (False, 1, 11, 1.0, 2),
                                                (False, 2, 6, 0.8, 0)])
def test_tokens_are_distributed_as_the_target_sharply(gops, drawn, kids, V, t, pad):
    """The token after the root, over all drafts by their probabilities, is p to 1 / 512. Each child's chance to stand is measured by G coins
    of its own with those before it fallen, and the chances of the tokens that are drawn by G coins of the root's with all fallen. A border is
    off by half a step: a draft's 1 / 2G, a token's two 1 / G, products of probabilities by their sum at most. pad: rows without a parent behind the
    tree, whose tokens are none and whose logits are NaN, change nothing."""
    G = 1024
    rng = np.random.default_rng(V)
    x, y = rng.standard_normal(V).astype(np.float32) * 1.5, rng.standard_normal(V).astype(np.float32) * 1.5
    p, q = (np.exp(z.astype(np.float64) / t) for z in (x, y))
    p, q = p / p.sum(), q / q.sum()
    rows = 1 + kids + pad
    spoilt = [np.nan] * V
    logits, draft = (torch.tensor([z.tolist()] * (1 + kids) + [spoilt] * pad, dtype=torch.float32, device="cuda").repeat(G, 1) for z in (x, y))
    starts, parents = ints(rows * np.arange(G + 1)), ints([-1] + [0] * kids + [-1] * pad).repeat(G)
    grid, fallen = ((np.arange(G) + 0.5) / G).astype(np.float32), np.float32(1 - 2.0 ** -24)

    def sweep(drafts, which):
        """The child that stood (0: none) and the token, for G coins of row `which`."""
        coins = np.full((G, rows), fallen, np.float32)
        coins[:, which] = grid
        path = gops.draft_verify(starts, parents, ints([0, *drafts] + [-1] * pad).repeat(G), logits, torch.from_numpy(coins.reshape(-1)).cuda(),
                                 draft_logits=draft if drawn else None, temperature=torch.full((G,), t, device="cuda"), max_rows=rows, max_path=2)
        assert (path.count == (path.rows[:, 1] >= 0) + 1).all()
        return path.rows[:, 1].clamp(min=0).cpu().numpy(), path.tokens[:, 0].cpu().numpy()

    sets = [(c,) for c in range(V)] if kids == 1 else [(c, d) for c in range(V) for d in range(V)]
    weight = [math.prod(q[c] for c in cs) for cs in sets]
    if not drawn:
        sets, weight = [tuple(int(c) for c in rng.permutation(V)[:kids])], [1.0]
    got = np.zeros(V)
    for cs, w in zip(sets, weight):
        for i, c in enumerate(cs):
            child, token = sweep(cs, 1 + i)
            stands = child == 1 + i
            assert (token[stands] == c).all() and (child >= 1 + i).sum() + (child == 0).sum() == G
            got[c] += w * stands.mean()
            w *= 1 - stands.mean()
            if w == 0:  # it stands whatever its coin
                break
        else:
            child, token = sweep(cs, 0)
            assert (child == 0).all()
            got += w * np.bincount(token, minlength=V) / G
    assert np.abs(got - p).max() <= (kids / 2 + 1) / G + 1e-9
