"""The paged 4-bit cache (ops.paged_append, paged_read, paged_attn) against plain implementations in 64 bits: codes and
scales bit for bit (the oracle's Q4_0 encoder on rows rotated in float64), attention against float64 softmax over the values
the cache stands for."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

ORDER = [0, 2, 1, 3, 4, 6, 5, 7]


# ------------------------------------------------------------------------------------------ helpers


class Case:
    """A ragged batch over a pool with pages in random order; `holes`: table entries set out of range."""

    def __init__(self, gops, rows, past, Hkv, D, page, seed=0, extra_rows=0, spare_pages=2, extra_cols=1, fill=0xFF):
        self.gops, self.rows, self.past, self.Hkv, self.D, self.page = gops, rows, past, Hkv, D, page
        rng = np.random.default_rng(seed)
        need = [max(0, -(-(p + r) // page)) for r, p in zip(rows, past)]
        self.n_pages = sum(need) + spare_pages
        order = rng.permutation(self.n_pages)
        table = np.full((len(rows), max(need) + extra_cols), -1, np.int32)
        at = 0
        for s, m in enumerate(need):
            table[s, :m] = order[at:at + m]
            at += m
        self.table = table
        self.starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.n = int(self.starts[-1]) + extra_rows
        self.cache = gops.PagedCache.new(self.n_pages, page, Hkv, D)
        self.cache.data.fill_(fill)  # NaN scales wherever nothing is appended
        self.rng = rng

    def batch(self, rows=None, past=None, table=None):
        rows, past = self.rows if rows is None else rows, self.past if past is None else past
        starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        return self.gops.PagedBatch(torch.from_numpy(self.table if table is None else table).cuda(),
                                    torch.from_numpy(starts).cuda(), torch.tensor(past, dtype=torch.int32).cuda())

    def fill_past(self):
        """All tokens of every sequence, the new rows' among them, appended as one batch: float32 values in [-4, 4]."""
        rows = [p + r for r, p in zip(self.rows, self.past)]
        k, v = (torch.from_numpy(self.rng.standard_normal((sum(rows), self.Hkv, self.D)).astype(np.float32)).cuda()
                for _ in range(2))
        b = self.batch(rows, [0] * len(rows))
        self.gops.paged_append(self.cache, b, k, v)
        self.k, self.v = (x.double() for x in self.gops.paged_read(self.cache, b, sum(rows)))
        self.key0 = np.concatenate([[0], np.cumsum(rows)])


def q4_values(orc, x):
    """What ggml's Q4_0 encoder stores of f32 rows [.., D]."""
    flat = np.ascontiguousarray(x.reshape(-1, x.shape[-1]))
    return orc.dequantize(orc.quantize(flat, "q4_0"), "q4_0", x.shape[-1]).reshape(x.shape)


def rotated(x, pos, freqs, factor=1.0):
    """f32 [n, H, D] turned in float64, rounded once."""
    half = len(freqs)
    ang = np.asarray(pos, np.float64)[:, None] * freqs.astype(np.float64)
    c, s = np.cos(ang)[:, None] * np.float64(np.float32(factor)), np.sin(ang)[:, None] * np.float64(np.float32(factor))
    a, b = x[..., :half].astype(np.float64), x[..., half:2 * half].astype(np.float64)
    y = x.copy()
    y[..., :half] = (a * c - b * s).astype(np.float32)
    y[..., half:2 * half] = (a * s + b * c).astype(np.float32)
    return y


def positions(case):
    return np.concatenate([np.arange(p, p + r) for r, p in zip(case.rows, case.past)] or [[]]).astype(np.int64)


def attn_reference(case, q, scale, window=0, holes=()):
    """float64, over the values that paged_read gave; `holes`: (sequence, page) pairs that are not there."""
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    bound = 0.0
    G = q.shape[1] // case.Hkv
    for s, (r, p) in enumerate(zip(case.rows, case.past)):
        if r == 0:
            continue
        k = case.k[case.key0[s]:case.key0[s + 1]].transpose(0, 1)
        v = case.v[case.key0[s]:case.key0[s + 1]].transpose(0, 1)
        rows = q[case.starts[s]:case.starts[s + 1]].double()
        key, at = torch.arange(p + r, device="cuda")[None], torch.arange(p, p + r, device="cuda")[:, None]
        seen = key <= at
        if window:
            seen &= key > at - window
        for hs, pg in holes:
            if hs == s:
                seen &= key // case.page != pg
        for h in range(q.shape[1]):
            x = (rows[:, h] @ k[h // G].T) * scale
            x = x.masked_fill(~seen, -torch.inf)
            w = torch.exp(x - x.amax(-1, keepdim=True).nan_to_num(neginf=0.0))
            o = w @ v[h // G] / w.sum(-1, keepdim=True).clamp(min=1e-300)
            out[case.starts[s]:case.starts[s + 1], h] = o
            bound = max(bound, float((rows[:, h].abs() @ k[h // G].abs().T).max()) * abs(scale))
    return out, bound


def check_attn(case, got, want, bound, keys):
    """|error| <= max|v| (2 e_s + e_p): e_s, a score's, D products and sums in f32, each off by 2^-24 of sum |q k|
    (exponent and sum of blocks: 16 more); e_p, weights in two parts of 11 bits cut off (2^-19), exp2 and sums in f32.
    In the mean far less: errors of either sign, 2-norm within 2^-18."""
    eps = 2.0 ** -24
    most = float(case.v.abs().max()) if case.v.numel() else 1.0
    tol = most * (2 * (case.D + 16) * eps * bound + 2.0 ** -19 + (keys + 64) * eps)
    err = (got.double() - want).abs().max().item() if got.numel() else 0.0
    assert np.isfinite(err) and err <= tol, (err, tol)
    if got.numel():
        rel = ((got.double() - want).norm() / want.norm().clamp(min=1e-30)).item()
        assert rel <= 2.0 ** -18, rel


def run_attn(gops, case, G, window=0, scale=None, seed=5, max_rows=None, holes=(), q_scale=1.5):
    H, D = G * case.Hkv, case.D
    case.fill_past()
    q = torch.from_numpy(np.random.default_rng(seed).standard_normal((case.n, H, D)).astype(np.float32) * q_scale).cuda().half()
    table = case.table.copy()
    for s, pg in holes:
        table[s, pg] = -1 if (s + pg) % 2 else case.n_pages
    scale = D ** -0.5 if scale is None else scale
    out = torch.full((case.n, H, D), 77.0, device="cuda")
    gops.paged_attn(case.cache, case.batch(table=table), q, scale, max_rows=max_rows, window=window, out=out)
    want, bound = attn_reference(case, q, scale, window, holes)
    n = int(case.starts[-1])
    check_attn(case, out[:n], want[:n], bound, max([p + r for r, p in zip(case.rows, case.past)]))
    assert (out[n:] == 77.0).all()  # rows of no sequence
    return out, q


# ------------------------------------------------------------------------------------ append, read


@pytest.mark.parametrize("D,n_dims,page,H,Hkv", [(128, 128, 64, 32, 8), (64, 64, 32, 14, 2), (256, 256, 128, 8, 1),
                                                 (128, 64, 256, 6, 3), (64, 20, 64, 3, 3), (256, 130, 32, 5, 5)])
@pytest.mark.parametrize("rows,past", [([1], [0]), ([1, 1, 1, 1], [31, 32, 1000, 131071]), ([0, 37, 0, 5, 1], [9, 30, 0, 250, 3]),
                                       ([300], [17])])
def test_append_equals_the_encoder(gops, orc, D, n_dims, page, H, Hkv, rows, past):
    """Rotated rows, strided out of one stacked projection: q in f16, k and v as the oracle's Q4_0 encoder stores them."""
    c = Case(gops, rows, past, Hkv, D, page, seed=D + len(rows))
    x = c.rng.standard_normal((c.n, (H + 2 * Hkv) * D)).astype(np.float32)
    t = torch.from_numpy(x).cuda().view(c.n, H + 2 * Hkv, D)
    freqs = gops.rope_freqs(n_dims, 500000.0)
    q16 = gops.paged_append(c.cache, c.batch(), t[:, H:H + Hkv], t[:, H + Hkv:], q=t[:, :H], freqs=freqs, attn_factor=1.25)
    k, v = gops.paged_read(c.cache, c.batch(), c.n)
    x = x.reshape(c.n, H + 2 * Hkv, D)
    f = freqs.cpu().numpy()
    assert np.array_equal(q16.cpu().numpy(), rotated(x[:, :H], positions(c), f, 1.25).astype(np.float16))
    assert np.array_equal(k.cpu().numpy(), q4_values(orc, rotated(x[:, H:H + Hkv], positions(c), f, 1.25)))
    assert np.array_equal(v.cpu().numpy(), q4_values(orc, np.ascontiguousarray(x[:, H + Hkv:])))


def layout_bytes(c, slots):
    """Byte addresses of the (sequence, position) slots' codes and scales, from the documented layout."""
    D, at = c.D, []
    for s, p in slots:
        for h in range(c.Hkv):
            t0 = ((int(c.table[s, p // c.page]) * c.Hkv + h) * (c.page // 32) + p % c.page // 32) * 36 * D
            t = p % 32
            for i in range(D // 2):
                at.append(t0 + t * (D // 2) + i // 8 % 4 * (D // 8) + i // 32 * 8 + i % 8)
                at.append(t0 + 16 * D + ((i // 32 * 4 + t // 8) * 16 + i % 16) * 16 + i // 16 % 2 * 8 + t % 8)
            for b in range(D // 32):
                for base in (32 * D, 34 * D):
                    o = t0 + base + 2 * (32 * b + t // 8 * 8 + ORDER[t % 8])
                    at += [o, o + 1]
    return np.array(at)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_append_writes_its_slots_only(gops, D):
    c = Case(gops, [3, 0, 40], [30, 5, 62], 2, D, 32, seed=3, fill=0xA5)
    k, v = (torch.randn((c.n, 2, D), device="cuda") for _ in range(2))
    assert gops.paged_append(c.cache, c.batch(), k, v) is None
    got = c.cache.data.cpu().numpy()
    own = layout_bytes(c, [(0, p) for p in range(30, 33)] + [(2, p) for p in range(62, 102)])
    assert len(np.unique(own)) == len(own) == 43 * 2 * (D + D // 8)
    rest = np.ones(got.shape, bool)
    rest[own] = False
    assert (got[rest] == 0xA5).all()
    assert (got[own] != 0xA5).mean() > 0.9
    # a second append of the same rows changes nothing
    gops.paged_append(c.cache, c.batch(), k, v)
    assert np.array_equal(got, c.cache.data.cpu().numpy())


def test_append_far_positions(gops, orc):
    """Positions near 2^31 (few pages: all tokens dropped, the queries' rotation stays exact to f16)."""
    c = Case(gops, [2, 1], [0, 0], 1, 128, 32)
    past = [2147480000, 16777217]
    f = gops.rope_freqs(128, 10000.0)
    q = torch.randn((3, 4, 128), device="cuda")
    k = torch.randn((3, 1, 128), device="cuda")
    got = gops.paged_append(c.cache, c.batch(past=past), k, k, q=q, freqs=f)
    want = rotated(q.cpu().numpy(), [2147480000, 2147480001, 16777217], f.cpu().numpy())
    assert np.abs(got.float().cpu().numpy() - want).max() <= 2.0 ** -11 * np.abs(want).max()
    assert (c.cache.data == 0xFF).all()
    z, _ = gops.paged_read(c.cache, c.batch(past=past), 3)
    assert (z == 0).all()


def test_append_padded_batch_and_missing_pages(gops, orc):
    """Rows behind the last sequence write nothing; a token whose page is missing is dropped, its q still turned;
    reading gives zeros for it."""
    c = Case(gops, [40, 3], [0, 31], 2, 128, 32, extra_rows=6, seed=8)
    x = c.rng.standard_normal((c.n, 2, 128)).astype(np.float32)
    t = torch.from_numpy(x).cuda()
    table = c.table.copy()
    table[0, 0], table[1, 1] = -7, c.n_pages
    b = c.batch(table=table)
    q_out = torch.full((c.n, 2, 128), 5.0, dtype=torch.float16, device="cuda")
    before = c.cache.data.clone()
    gops.paged_append(c.cache, b, t, t, q=t, q_out=q_out)
    assert (q_out[43:] == 5.0).all() and np.array_equal(q_out[:43].cpu().numpy(), x[:43].astype(np.float16))
    own = layout_bytes(c, [(0, p) for p in range(32, 40)] + [(1, 31)])
    rest = np.ones(before.numel(), bool)
    rest[own] = False
    assert np.array_equal(before.cpu().numpy()[rest], c.cache.data.cpu().numpy()[rest])
    k = torch.full((c.n, 2, 128), 9.0, device="cuda")
    v = k.clone()
    gops.paged_read(c.cache, b, c.n, k=k, v=v)
    want = q4_values(orc, x)
    gone = np.r_[0:32, 41:43]
    want[gone] = 0.0
    for y in (k, v):
        assert np.array_equal(y[:43].cpu().numpy(), want[:43]) and (y[43:] == 9.0).all()


def test_append_special_values(gops, orc):
    """Zero blocks, ties of either sign, values whose scale is subnormal, too large or not finite, NaNs."""
    D = 64
    x = np.zeros((8, 1, D), np.float32)
    x[1, 0, 3], x[1, 0, 9], x[1, 0, 40], x[1, 0, 41] = 2.0, -2.0, -3.0, 3.0
    x[2] = np.random.default_rng(1).standard_normal((1, D)) * 1e-6
    x[3] = np.random.default_rng(2).standard_normal((1, D)) * 1e-42
    x[4, 0, :8] = [1e9, -3e38, 1.0, 65504.0, 65505.0, -7e5, 2.0, 6e4]
    x[5, 0, 5], x[5, 0, 6], x[5, 0, 33] = np.inf, 4.0, -np.inf
    x[6, 0, :40] = 1.0
    x[6, 0, 7], x[6, 0, 20] = np.nan, -2.0
    x[7] = np.nan
    c = Case(gops, [8], [0], 1, D, 32)
    t = torch.from_numpy(x).cuda()
    gops.paged_append(c.cache, c.batch(), t, t)
    k, v = gops.paged_read(c.cache, c.batch(), 8)
    clean = np.clip(np.nan_to_num(x, nan=0.0, posinf=65504.0, neginf=-65504.0), -65504.0, 65504.0)
    want = q4_values(orc, clean)
    assert np.isfinite(want).all()
    for y in (k, v):
        assert np.array_equal(y.cpu().numpy(), want)
    # ties go to the first: +2 at 3 makes its scale negative, -3 at 40 its own positive
    assert k[1, 0, 3] == 2.0 and k[1, 0, 40] == -3.0 and k[1, 0, 9] == -1.75 and k[1, 0, 41] == 2.625


# -------------------------------------------------------------------------------------- attention


@pytest.mark.parametrize("D,Hkv,G", [(64, 2, 7), (128, 2, 4), (256, 1, 2), (128, 1, 1), (64, 1, 16), (128, 1, 24), (256, 2, 8),
                                     (64, 3, 3)])
@pytest.mark.parametrize("rows,past,page", [
    ([1], [0], 32), ([1], [31], 32), ([1, 1, 1], [0, 63, 700], 64), ([0, 1, 0, 1], [5, 2048, 0, 33], 128),
    ([2, 5, 1, 8], [3, 100, 0, 256], 32), ([33], [0], 256), ([130, 1, 17], [65, 400, 0], 64), ([0, 0], [40, 3], 32)])
def test_attention(gops, D, Hkv, G, rows, past, page):
    run_attn(gops, Case(gops, rows, past, Hkv, D, page, seed=D + G, extra_rows=3), G)


@pytest.mark.parametrize("window", [1, 31, 32, 100, 4096])
@pytest.mark.parametrize("rows,past", [([1, 1], [500, 20]), ([4, 2], [300, 0]), ([150, 1, 40], [333, 900, 0])])
def test_attention_window(gops, window, rows, past):
    run_attn(gops, Case(gops, rows, past, 2, 128, 64, seed=window), 4, window=window)


@pytest.mark.parametrize("rows,past,window", [([1, 1, 1], [100, 40, 31], 0), ([5, 1], [300, 64], 40), ([140, 3], [200, 5], 0)])
def test_attention_missing_pages(gops, rows, past, window):
    """Pages taken out of the table: their keys are not seen, and a row left with none gives zeros."""
    c = Case(gops, rows, past, 2, 64, 32, seed=9)
    every = [(len(rows) - 1, p) for p in range(-(-(rows[-1] + past[-1]) // 32))]
    out, _ = run_attn(gops, c, 2, window=window, holes=[(0, 0), (0, 2), *every])
    assert (out[c.starts[-2]:c.starts[-1]] == 0).all()


@pytest.mark.parametrize("rows,past,G", [([1], [33000], 4), ([1, 1], [9000, 20000], 1), ([3], [12000], 8), ([200], [8000], 2)])
def test_attention_long(gops, rows, past, G):
    run_attn(gops, Case(gops, rows, past, 1, 128, 256, seed=11), G)


def test_attention_many_sequences(gops):
    """More sequences than lanes, lengths 0 to 400, some without rows."""
    rng = np.random.default_rng(4)
    rows = [int(r) for r in rng.integers(0, 4, 150)]
    past = [int(p) for p in rng.integers(0, 400, 150)]
    run_attn(gops, Case(gops, rows, past, 2, 64, 32, seed=12), 3, max_rows=3)


def test_attention_max_rows(gops):
    """Rows past max_rows are left as they are, the others are right."""
    c = Case(gops, [5, 2, 40], [10, 200, 3], 2, 128, 64, seed=13)
    full, q = run_attn(gops, c, 4)
    for m in (1, 2, 3, 39):
        out = torch.full_like(full, 77.0)
        gops.paged_attn(c.cache, c.batch(), q, 128 ** -0.5, max_rows=m, out=out)
        for s, r in enumerate(c.rows):
            a, b = c.starts[s], c.starts[s + 1]
            assert (out[a + m:b] == 77.0).all()
            assert (out[a:min(a + m, b)] - full[a:min(a + m, b)]).abs().max() < 2e-5


@pytest.mark.parametrize("scale", [0.0, -0.1, 1.0, 3.0])
@pytest.mark.parametrize("rows,past", [([1, 3], [200, 77]), ([100], [150])])
def test_attention_scales(gops, scale, rows, past):
    run_attn(gops, Case(gops, rows, past, 1, 64, 32, seed=14), 4, scale=scale)


def test_attention_large_scores(gops):
    """Scores in the thousands: one key takes all the weight; and cached values up to f16's largest."""
    c = Case(gops, [1, 70], [300, 10], 1, 128, 64, seed=15)
    run_attn(gops, c, 4, scale=5.0, q_scale=30.0)
    c = Case(gops, [1, 70], [300, 10], 1, 64, 64, seed=16)
    c.fill_past()
    b = c.batch([p + r for r, p in zip(c.rows, c.past)], [0, 0])
    gops.paged_append(c.cache, b, c.k.float(), c.v.float() * 30000.0)
    c.k, c.v = (x.double() for x in gops.paged_read(c.cache, b, int(c.key0[-1])))
    q = torch.randn((c.n, 2, 64), device="cuda").half()
    got = gops.paged_attn(c.cache, c.batch(), q, 0.125)
    want, bound = attn_reference(c, q, 0.125)
    check_attn(c, got, want, bound, 301)


def test_attention_huge_scores(gops):
    """Scores past 2^24, where f32 holds no fraction: the largest key takes all the weight unless another's score rounds to
    the same; NaN-free, and each output a mean of cached values of near-largest scores (within 2^-22 of them)."""
    c = Case(gops, [1, 70], [300, 10], 1, 128, 64, seed=26)
    c.fill_past()
    q = (torch.randn((c.n, 4, 128), device="cuda") * 3000).half()
    got = gops.paged_attn(c.cache, c.batch(), q, 2000.0).double()
    want, _ = attn_reference(c, q, 2000.0)
    for s in range(2):
        k, v = c.k[c.key0[s]:c.key0[s + 1], 0], c.v[c.key0[s]:c.key0[s + 1], 0]
        for r in range(c.rows[s]):
            for h in range(4):
                x = k[:c.past[s] + r + 1] @ q[c.starts[s] + r, h].double() * 2000.0
                near = x >= x.max() - x.abs().max() * 2.0 ** -20
                lo, hi = v[:len(x)][near].amin(0), v[:len(x)][near].amax(0)
                o = got[c.starts[s] + r, h]
                assert x.max() > 2.0 ** 24 or r < 4
                assert ((o >= lo - 1e-5) & (o <= hi + 1e-5)).all()


def test_attention_tiny_values(gops):
    """Cached values whose scales are f16 subnormals keep their bits."""
    c = Case(gops, [2, 64], [90, 0], 1, 128, 32, seed=17)
    c.fill_past()
    b = c.batch([p + r for r, p in zip(c.rows, c.past)], [0, 0])
    gops.paged_append(c.cache, b, c.k.float(), c.v.float() * 2.0 ** -20)
    c.k, c.v = (x.double() for x in gops.paged_read(c.cache, b, int(c.key0[-1])))
    q = torch.randn((c.n, 4, 128), device="cuda").half()
    got = gops.paged_attn(c.cache, c.batch(), q, 0.125)
    want, bound = attn_reference(c, q, 0.125)
    check_attn(c, got, want, bound, 92)


def test_nan_query_and_infinite_query_stay_in_their_rows(gops):
    c = Case(gops, [1, 90], [40, 0], 2, 128, 32, seed=18)
    full, q = run_attn(gops, c, 2)
    bad = q.clone()
    bad[0, 1, 5] = float("nan")
    bad[50, 2, 7] = float("inf")
    out = gops.paged_attn(c.cache, c.batch(), bad, 128 ** -0.5)
    assert torch.isnan(out[0, 1]).all()
    keep = torch.ones(out.shape[:2], dtype=torch.bool, device="cuda")
    keep[0, 1] = keep[50, 2] = False
    assert torch.equal(out[keep], full[keep])


def test_attention_strided_queries(gops):
    c = Case(gops, [1, 20], [70, 9], 2, 64, 32, seed=19)
    full, q = run_attn(gops, c, 3)
    wide = torch.zeros((c.n, 10, 80), dtype=torch.float16, device="cuda")
    wide[:, 2:8, 8:72] = q
    assert torch.equal(gops.paged_attn(c.cache, c.batch(), wide[:, 2:8, 8:72], 0.125), full)


def test_cache_past_four_gigabytes(gops):
    """Pages whose byte offsets pass 32 bits."""
    D, Hkv, page = 256, 8, 256
    n_pages = (5 << 30) // (page * Hkv * 288)
    cache = gops.PagedCache.new(n_pages, page, Hkv, D)
    assert cache.data.numel() > 1 << 32
    pages = torch.tensor([[n_pages - 1, 3, n_pages - 2]], dtype=torch.int32, device="cuda")
    n = 600
    b = gops.PagedBatch(pages, torch.tensor([0, n], dtype=torch.int32, device="cuda"),
                        torch.zeros(1, dtype=torch.int32, device="cuda"))
    k, v = (torch.randn((n, Hkv, D), device="cuda") for _ in range(2))
    q = gops.paged_append(cache, b, k, v, q=k)
    c = Case(gops, [n], [0], Hkv, D, page)
    c.k, c.v = (x.double() for x in gops.paged_read(cache, b, n))
    c.key0 = [0, n]
    assert ((c.k - k.double()).norm() / k.double().norm()) < 0.15
    for rows in (n, 1):
        b = gops.PagedBatch(pages, torch.tensor([0, rows], dtype=torch.int32, device="cuda"),
                            torch.tensor([n - rows], dtype=torch.int32, device="cuda"))
        c.rows, c.past, c.starts = [rows], [n - rows], np.array([0, rows])
        got = gops.paged_attn(cache, b, q[n - rows:], 1 / 16)
        want, bound = attn_reference(c, q[n - rows:], 1 / 16)
        check_attn(c, got, want, bound, n)


# ------------------------------------------------------------------------------------- run together


def test_serving_together(gops, orc):
    """Two prompts enter, then six steps that append and attend one token each while a third prompt joins: every output
    against float64 over what was appended, and a sequence read back into flash_attn_ext's contiguous f16 cache."""
    Hkv, G, D, page = 2, 4, 128, 32
    H = Hkv * G
    rng = np.random.default_rng(21)
    c = Case(gops, [70, 1, 40], [0, 0, 0], Hkv, D, page, seed=21)
    c.table = rng.permutation(24)[:18].reshape(3, 6).astype(np.int32)
    cache = gops.PagedCache.new(24, page, Hkv, D)
    freqs = gops.rope_freqs(D, 10000.0)
    kept = [[np.zeros((0, Hkv, D), np.float32)] * 2 for _ in range(3)]
    length = [0, 0, 0]
    for step, rows in enumerate([[70, 1, 0], [1, 1, 0], [1, 1, 40], [1, 1, 1], [1, 1, 1], [1, 1, 1], [1, 1, 1]]):
        n = sum(rows)
        x = rng.standard_normal((n, H + 2 * Hkv, D)).astype(np.float32)
        t = torch.from_numpy(x).cuda()
        b = c.batch(rows, length)
        q = gops.paged_append(cache, b, t[:, H:H + Hkv], t[:, H + Hkv:], q=t[:, :H], freqs=freqs)
        got = gops.paged_attn(cache, b, q, D ** -0.5, max_rows=max(rows))
        pos = np.concatenate([np.arange(p, p + r) for r, p in zip(rows, length)])
        kq = q4_values(orc, rotated(x[:, H:H + Hkv], pos, freqs.cpu().numpy()))
        vq = q4_values(orc, np.ascontiguousarray(x[:, H + Hkv:]))
        at = np.concatenate([[0], np.cumsum(rows)])
        for s in range(3):
            kept[s] = [np.concatenate([old, new[at[s]:at[s + 1]]]) for old, new in zip(kept[s], (kq, vq))]
        c.rows, c.past, c.starts = rows, list(length), at
        length = [p + r for p, r in zip(length, rows)]
        c.k, c.v = (torch.from_numpy(np.concatenate([kept[s][i] for s in range(3)])).cuda().double() for i in range(2))
        c.key0 = np.concatenate([[0], np.cumsum(length)])
        want, bound = attn_reference(c, q, D ** -0.5)
        check_attn(c, got, want, bound, max(length))
    # the first sequence, handed over: f16 rounds K and V (2^-11 of each), the output by two such steps and a score's
    b = gops.PagedBatch(torch.from_numpy(c.table[:1]).cuda(), torch.tensor([0, length[0]], dtype=torch.int32).cuda(),
                        torch.zeros(1, dtype=torch.int32).cuda())
    k, v = gops.paged_read(cache, b, length[0])
    assert np.array_equal(k.cpu().numpy(), kept[0][0]) and np.array_equal(v.cpu().numpy(), kept[0][1])
    o = gops.flash_attn_ext(q[:1].float().transpose(0, 1).contiguous(), k.half().transpose(0, 1).contiguous(),
                            v.half().transpose(0, 1).contiguous(), None, D ** -0.5)
    assert ((o - got[:1]).norm() / got[:1].norm()).item() < 2.0 ** -8


@pytest.mark.parametrize("n_max,max_rows", [(4, 1), (160, 160)])
def test_captured_step_follows_the_batch(gops, n_max, max_rows):
    """One captured append + attention, replayed over changing rows, lengths and pages (a padded batch), each replay
    against the eager calls, with eager work in between."""
    Hkv, G, D, page = 2, 4, 128, 64
    H = Hkv * G
    table = torch.from_numpy(np.random.default_rng(3).permutation(40).reshape(4, 10).astype(np.int32)).cuda()
    starts, past = torch.zeros(5, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    batch = gops.PagedBatch(table, starts, past)
    cache, other = (gops.PagedCache.new(40, page, Hkv, D) for _ in range(2))
    for cc in (cache, other):
        x = torch.randn((2400, Hkv, D), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
        full = gops.PagedBatch(table, torch.arange(0, 2401, 600, dtype=torch.int32, device="cuda"), torch.zeros_like(past))
        gops.paged_append(cc, full, x, x)
    freqs = gops.rope_freqs(D, 10000.0)
    t = torch.zeros((n_max, H + 2 * Hkv, D), device="cuda")
    q_out = torch.zeros((n_max, H, D), dtype=torch.float16, device="cuda")
    out = torch.zeros((n_max, H, D), device="cuda")

    def step(cc, qo, o):
        gops.paged_append(cc, batch, t[:, H:H + Hkv], t[:, H + Hkv:], q=t[:, :H], freqs=freqs, q_out=qo)
        gops.paged_attn(cc, batch, qo, D ** -0.5, max_rows=max_rows, out=o)

    step(cache, q_out, out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(cache, q_out, out)
    rng = np.random.default_rng(6)
    for rep in range(6):
        rows = rng.multinomial(rng.integers(0, n_max + 1), [0.25] * 4) if max_rows > 1 else rng.integers(0, 2, 4)
        starts.copy_(torch.from_numpy(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)))
        past.copy_(torch.from_numpy(rng.integers(0, 440, 4).astype(np.int32)))
        t.normal_()
        out.fill_(7.0)
        want_q, want = torch.zeros_like(q_out), torch.full_like(out, 7.0)
        q_out.zero_()
        torch.cuda.synchronize()
        g.replay()
        step(other, want_q, want)
        torch.cuda.synchronize()
        assert torch.equal(q_out, want_q) and torch.equal(out, want) and torch.equal(cache.data, other.data), rep
        assert (out[int(rows.sum()):] == 7.0).all()


def test_two_streams_at_once(gops):
    """The same cache read by two calls on streams of their own, interleaved; equal to one call after the other."""
    c = Case(gops, [1, 1, 1], [4000, 300, 9000], 2, 128, 64, seed=23)
    full, q = run_attn(gops, c, 4, max_rows=1)
    b = c.batch()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(gops.paged_attn(c.cache, b, q, 128 ** -0.5, max_rows=1))
    torch.cuda.synchronize()
    assert all(torch.equal(o, full) for o in outs)


def test_refusals_on_the_device(gops):
    cache = gops.PagedCache.new(4, 32, 2, 64)
    i32 = dict(dtype=torch.int32, device="cuda")
    batch = gops.PagedBatch(torch.zeros((2, 2), **i32), torch.zeros(3, **i32), torch.zeros(2, **i32))
    x, q = torch.zeros((4, 2, 64), device="cuda"), torch.zeros((4, 4, 64), dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError, match="contiguous bytes"):
        gops.PagedCache(4, 32, 2, 64, cache.data[:-1])
    with pytest.raises(ValueError, match="2 sequences need"):
        gops.PagedBatch(torch.zeros((2, 2), **i32), torch.zeros(2, **i32), torch.zeros(2, **i32))
    with pytest.raises(ValueError, match="rows overlap"):
        gops.PagedBatch(torch.zeros((1, 2), **i32).expand(2, 2), torch.zeros(3, **i32), torch.zeros(2, **i32))
    with pytest.raises(ValueError, match="torch.int32"):
        gops.PagedBatch(torch.zeros((2, 2), device="cuda", dtype=torch.int64), torch.zeros(3, **i32), torch.zeros(2, **i32))
    for bad in (x[:, :1], x[..., :32], x.half(), x.cpu(), x.transpose(1, 2).contiguous().transpose(1, 2)):
        with pytest.raises(ValueError):
            gops.paged_append(cache, batch, bad, x)
        with pytest.raises(ValueError):
            gops.paged_append(cache, batch, x, bad)
    with pytest.raises(ValueError, match="q_out without q"):
        gops.paged_append(cache, batch, x, x, q_out=q)
    with pytest.raises(gops.GcqError, match="n_dims"):
        gops.paged_append(cache, batch, x, x, freqs=torch.zeros(40, device="cuda"))
    with pytest.raises(gops.GcqError, match="multiple of n_head_kv"):
        gops.paged_attn(cache, batch, q[:, :3], 0.1)
    with pytest.raises(ValueError, match="torch.float16"):
        gops.paged_attn(cache, batch, q.float(), 0.1)
    for window in (-1, 1 << 31, 1 << 32):
        with pytest.raises(ValueError, match="window"):
            gops.paged_attn(cache, batch, q, 0.1, window=window)
    for bad in (x[0, 0, 0], x[0], x[None]):
        with pytest.raises(ValueError, match="must be"):
            gops.paged_append(cache, batch, bad, bad)
        with pytest.raises(ValueError, match="must be"):
            gops.paged_append(cache, batch, x, x, q=bad)
        with pytest.raises(ValueError, match="must be"):
            gops.paged_attn(cache, batch, bad.half(), 0.1)
    with pytest.raises(AttributeError):  # (its address is in the C structure)
        batch.past = batch.starts
    with pytest.raises(gops.GcqError, match="16-byte aligned"):
        gops.paged_read(cache, batch, 4, k=torch.zeros(4 * 2 * 64 + 1, device="cuda")[1:].view(4, 2, 64))
    with pytest.raises(gops.GcqError, match="max_rows"):
        gops.paged_attn(cache, batch, q, 0.1, max_rows=0)
    with pytest.raises(ValueError, match="contiguous"):
        gops.paged_attn(cache, batch, q, 0.1, out=torch.zeros((4, 4, 128), device="cuda")[..., ::2])
    assert gops.paged_attn(cache, batch, q[:0], 0.1).shape == (0, 4, 64)
    assert gops.paged_read(cache, batch, 0)[0].shape == (0, 2, 64)


@pytest.mark.parametrize("D,n_dims,Hkv", [(64, 64, 3), (128, 128, 4), (128, 72, 2), (256, 256, 2), (256, 64, 1)])
@pytest.mark.parametrize("rows,past", [([8], [0]), ([4], [30]), ([8, 9], [28, 31]), ([7, 9], [1, 2]),
                                       ([32, 64, 1, 31], [0, 32, 95, 33]), ([3, 200, 0, 95], [62, 33, 4, 1])])
def test_rows_by_eights_equal_rows_one_by_one(gops, D, n_dims, Hkv, rows, past):
    """A call that goes eight positions at a time and calls of a few rows each (strides that no 16-byte load takes among
    them) leave the same bytes, queries and rows read back; the rest of the pool stays as it is."""
    H = (1 << 20) // (D * sum(rows)) + 2  # (fewer values go row by row)
    c = Case(gops, rows, past, Hkv, D, 64, seed=31, extra_rows=2, fill=0xA5)
    x = torch.from_numpy(c.rng.standard_normal((c.n, H + 2 * Hkv, D)).astype(np.float32)).cuda()
    freqs = gops.rope_freqs(n_dims, 10000.0)
    odd = torch.zeros((c.n, H + 2 * Hkv, D + 1), device="cuda")
    odd[..., :D] = x
    q, k, v = x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
    q16 = torch.full((c.n, H, D), 5.0, dtype=torch.float16, device="cuda")
    gops.paged_append(c.cache, c.batch(), k, v, q=q, freqs=freqs, q_out=q16)
    once = c.cache.data.clone()
    c.cache.data.fill_(0xA5)
    o16 = torch.full_like(q16, 5.0)
    gops.paged_append(c.cache, c.batch(), odd[:, H:H + Hkv, :D], odd[:, H + Hkv:, :D], q=odd[:, :H, :D], freqs=freqs, q_out=o16)
    assert torch.equal(once, c.cache.data) and torch.equal(q16, o16)
    c.cache.data.fill_(0xA5)
    b = c.batch()
    got_k, got_v = gops.paged_read(gops.PagedCache(c.n_pages, 64, Hkv, D, once), b, c.n, *(torch.full_like(k, 3.0) for _ in range(2)))
    for s, (r, p) in enumerate(zip(rows, past)):
        for j in range(0, r, 5):
            m, at = min(5, r - j), int(c.starts[s]) + j
            one = gops.PagedBatch(b.pages[s:s + 1], torch.tensor([0, m], dtype=torch.int32).cuda(),
                                  torch.tensor([p + j], dtype=torch.int32).cuda())
            few = gops.paged_append(c.cache, one, k[at:at + m], v[at:at + m], q=q[at:at + m], freqs=freqs)
            assert torch.equal(few, q16[at:at + m])
            for y, w in zip(gops.paged_read(c.cache, one, m), (got_k, got_v)):
                assert torch.equal(y, w[at:at + m])
    assert torch.equal(once, c.cache.data)
    assert (got_k[-2:] == 3.0).all() and (got_v[-2:] == 3.0).all() and (q16[-2:] == 5.0).all()


def test_append_by_eights_special_values(gops):
    """Ties of either sign, zeros of either sign, NaNs, infinities and subnormal scales: by eights as one by one."""
    D = 64
    x = torch.zeros((32, 1, D), device="cuda")
    x[1, 0, 5], x[1, 0, 9] = -2.0, 2.0
    x[2, 0, 5], x[2, 0, 9] = 2.0, -2.0
    x[3, 0, 31], x[3, 0, 32], x[3, 0, 63] = 1.0, -1.0, 1.0
    x[4] = -0.0
    x[5, 0, 3], x[5, 0, 40] = float("nan"), float("nan")
    x[6, 0, 3], x[6, 0, 4], x[6, 0, 40] = float("inf"), 1.0, -float("inf")
    x[7] = 3e-7
    x[8, 0, ::3] = 1e-40
    x[9] = 3e38
    x[10, 0, :4], x[10, 0, 4:8] = 1.0, -1.0
    x[11, 0, 3], x[11, 0, 4] = -1.0, 1.0
    x[12, 0, 7], x[12, 0, 8] = 1.0, -1.0
    i32 = dict(dtype=torch.int32, device="cuda")
    a, b = (gops.PagedCache.new(1, 32, 1, D) for _ in range(2))
    page = torch.zeros((1, 1), **i32)
    whole = gops.PagedBatch(page, torch.tensor([0, 32], **i32), torch.tensor([0], **i32))
    q = gops.paged_append(a, whole, x, x, q=x.expand(32, 512, D))  # (512 heads: enough values to go by eights)
    assert torch.equal(q[:, 0].view(torch.int16), q[:, 511].view(torch.int16))
    for r in range(32):
        one = gops.PagedBatch(page, torch.tensor([0, 1], **i32), torch.tensor([r], **i32))
        o = gops.paged_append(b, one, x[r:r + 1], x[r:r + 1], q=x[r:r + 1])
        assert torch.equal(o[:, 0].view(torch.int16), q[r:r + 1, 0].view(torch.int16))
    assert torch.equal(a.data, b.data)


@pytest.mark.parametrize("rows", [[1, 2], [9, 90]])
def test_attention_largest_scale(gops, rows):
    """scale log2(e) past f32: queries of zeros still weigh all keys alike."""
    c = Case(gops, rows, [70, 3], 1, 64, 32, seed=33)
    run_attn(gops, c, 4, scale=3e38, q_scale=0.0)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rows,past,window,G", [([8] * 9, [500 * s for s in range(9)], 0, 4), ([8] * 9, [500 * s for s in range(9)], 700, 4),
                                                ([40] * 6 + [1], [9000, 0, 33, 64, 4000, 1, 7000], 0, 2),
                                                ([3, 1], [40000, 60000], 0, 8), ([3, 1], [40000, 60000], 2000, 8)])
def test_attention_both_row_tiles(gops, D, rows, past, window, G):
    """Sizes on either side of the choice between tiles of 16 and of 32 rows, in one and in several splits, the window
    moving it."""
    run_attn(gops, Case(gops, rows, past, 1 if max(past) > 30000 else 2, D, 64, seed=34), G, window=window, max_rows=max(rows))


def test_captured_long_step_follows_the_batch(gops):
    """As above where keys are split, rows go by eights and are read back: one captured append, attention and read."""
    Hkv, H, D, page, S, n = 2, 14, 128, 256, 3, 600
    rng = np.random.default_rng(41)
    table = torch.from_numpy(rng.permutation(80)[:72].reshape(S, 24).astype(np.int32)).cuda()
    starts, past = torch.zeros(S + 1, dtype=torch.int32, device="cuda"), torch.zeros(S, dtype=torch.int32, device="cuda")
    batch = gops.PagedBatch(table, starts, past)
    cache, other = (gops.PagedCache.new(80, page, Hkv, D) for _ in range(2))
    x = torch.randn((3 * 5000, Hkv, D), device="cuda")
    full = gops.PagedBatch(table, torch.arange(0, 15001, 5000, dtype=torch.int32, device="cuda"), torch.zeros_like(past))
    for c in (cache, other):
        gops.paged_append(c, full, x, x)
    qkv = torch.zeros((n, H + 2 * Hkv, D), device="cuda")
    freqs = gops.rope_freqs(D, 10000.0)
    q16 = torch.zeros((n, H, D), dtype=torch.float16, device="cuda")
    outs = [torch.zeros((n, H, D), device="cuda"), *(torch.zeros((n, Hkv, D), device="cuda") for _ in range(2))]

    def step(c, q16, out, k, v):
        gops.paged_append(c, batch, qkv[:, H:H + Hkv], qkv[:, H + Hkv:], q=qkv[:, :H], freqs=freqs, q_out=q16)
        gops.paged_attn(c, batch, q16, D ** -0.5, out=out)
        gops.paged_read(c, batch, n, k, v)

    step(cache, q16, *outs)  # (starts of zeros: nobody's rows)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(cache, q16, *outs)
    for rows, at in (([1, 1, 1], [4999, 10, 700]), ([600, 0, 0], [4300, 1, 2]), ([1, 0, 400], [5000, 0, 33]),
                     ([0, 2, 1], [0, 5100, 701]), ([100, 250, 250], [4950, 0, 3000]), ([1, 1, 1], [5050, 250, 3250])):
        qkv.copy_(torch.randn((n, H + 2 * Hkv, D), device="cuda"))
        starts.copy_(torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32))
        past.copy_(torch.tensor(at, dtype=torch.int32))
        for t in (q16, *outs):
            t.fill_(7.0)
        want = [t.clone() for t in (q16, *outs)]
        graph.replay()
        step(other, *want)
        torch.cuda.synchronize()
        for w, t in zip(want, (q16, *outs)):
            assert torch.equal(w, t)
        assert torch.equal(cache.data, other.data)
        assert not bool((outs[0][:sum(rows)] == 7.0).all()) and bool((outs[0][sum(rows):] == 7.0).all())


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("above", [10, 14, 17, 20, 24])
@pytest.mark.parametrize("keys,rows,S,G", [(1024, 1, 160, 4), (4096, 1, 160, 4), (16384, 1, 160, 1), (4096, 768, 1, 8), (16384, 384, 2, 8),
                                           (65536, 1, 1, 4)])
def test_attention_sink(gops, D, above, keys, rows, S, G):
    """One key `above` powers of two ahead of each other one, whose weights are log-normal, and values whose mean the first key's
    is far from: what the small weights lose together shows. Mostly one split (the sequences share their pages), all row tiles."""
    Hkv = 8 if rows == 1 else 2
    c = Case(gops, [keys], [0], Hkv, D, 256, seed=above + D)
    k = torch.from_numpy(c.rng.standard_normal((keys, Hkv, D)).astype(np.float32)).cuda() * 0.5
    v = torch.from_numpy(c.rng.standard_normal((keys, Hkv, D)).astype(np.float32)).cuda() + 1.0
    k[0], v[0] = above / (1.4426950408889634 * D ** 0.5), v[0] - 2.0  # (q's mean is 1: scale q K[0] = above ln 2)
    b = c.batch()
    gops.paged_append(c.cache, b, k, v)
    c.k, c.v = (x.double() for x in gops.paged_read(c.cache, b, keys))
    q = torch.from_numpy(c.rng.standard_normal((S * rows, G * Hkv, D)).astype(np.float32)).cuda().mul(0.5).add(1.0).half()
    out = gops.paged_attn(c.cache, c.batch([rows] * S, [keys - rows] * S, np.repeat(c.table, S, 0)), q, D ** -0.5, max_rows=rows)
    unseen = torch.arange(keys, device="cuda")[None] > torch.arange(keys - rows, keys, device="cuda").repeat(S)[:, None]
    want, bound = torch.empty(q.shape, dtype=torch.float64, device="cuda"), 0.0
    for h in range(G * Hkv):
        x, kh = q[:, h].double(), c.k[:, h // G]
        want[:, h] = torch.softmax((x @ kh.T * D ** -0.5).masked_fill(unseen, -torch.inf), -1) @ c.v[:, h // G]
        bound = max(bound, float((x.abs() @ kh.abs().T).max()) * D ** -0.5)
    check_attn(c, out, want, bound, keys)


def test_attention_scores_one_step_apart(gops):
    """Scores of 2^26 .. 2^27, whose f32 steps are 8: a later tile's key one step ahead of the first takes nearly all the weight."""
    D, n = 64, 160
    k, v = (torch.zeros((n, 1, D), device="cuda") for _ in range(2))
    k[0, 0, 0] = k[128, 0, 0] = 1.0
    k[128, 0, 32] = 2.0 ** -10
    v[0], v[128] = 1.0, -1.0
    c = Case(gops, [n], [0], 1, D, 32, seed=44)
    gops.paged_append(c.cache, c.batch(), k, v)
    q = torch.zeros((1, 1, D), dtype=torch.float16, device="cuda")
    q[0, 0, 0], q[0, 0, 32] = 2.0 ** 13, 1.0  # q K: 2^13, and 2^-23 of it more
    for i in range(24):
        got = gops.paged_attn(c.cache, c.batch([1], [n - 1]), q, 2.0 ** 13 / 1.4426950408889634 * (1 + i / 26))
        # 8 or more powers of two: at least 255 / 257 of the way, the weights' sums and product in f32
        assert bool(((got <= -253.0 / 257.0) & (got >= -1.0 - 2.0 ** -20)).all()), (i, got)


@pytest.mark.parametrize("D,G", [(64, 4), (128, 1), (256, 8)])
@pytest.mark.parametrize("rows,past,window", [([1, 1], [40, 0], 0), ([1], [40000], 0), ([3, 90], [700, 0], 0), ([40], [300], 33)])
def test_a_query_with_an_infinity_gives_nans(gops, D, G, rows, past, window):
    """softmax of scores among which are infinities is NaN, also where all of them are -inf; a row without keys gives zeros."""
    c = Case(gops, rows, past, 1, D, 32, seed=45)
    n_keys = [p + r for r, p in zip(rows, past)]
    b = c.batch(n_keys, [0] * len(rows))
    k = torch.rand((sum(n_keys), 1, D), device="cuda") + 0.5  # (positive, and no code stands for 0)
    gops.paged_append(c.cache, b, k, k)
    assert (gops.paged_read(c.cache, b, sum(n_keys))[0] > 0).all()
    q = torch.randn((c.n, G, D), device="cuda").half()
    table = c.table.copy()
    if len(rows) == 2:
        table[1] = -1
    b = c.batch(table=table)
    clean = gops.paged_attn(c.cache, b, q, 0.1, window=window)
    assert torch.isfinite(clean).all()
    bad = torch.zeros((c.n, G), dtype=torch.bool, device="cuda")
    for i, (r, h) in enumerate([(0, 0), (c.n - 1, G - 1), (c.n // 2, G // 2)]):
        bad[r, h] = True
        q[r, h, 7 * i + 5] = [-torch.inf, torch.inf, -torch.inf][i]
    keyless = torch.arange(c.n, device="cuda") >= rows[0] if len(rows) == 2 else torch.zeros(c.n, dtype=torch.bool, device="cuda")
    for scale in (0.1, -0.1, 0.0):
        want = clean if scale == 0.1 else gops.paged_attn(c.cache, b, q.masked_fill(bad[..., None], 0.0), scale, window=window)
        got = gops.paged_attn(c.cache, b, q, scale, window=window)
        assert torch.isnan(got[bad & ~keyless[:, None]]).all()
        assert (got[keyless] == 0).all()
        keep = ~bad & ~keyless[:, None]
        assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("scale", [1e25, 1e32, -1e36, 3e38, -3e38])
@pytest.mark.parametrize("D,G,rows,past", [(64, 4, [1, 1], [60, 0]), (128, 1, [70], [0]), (256, 8, [3, 20], [500, 0])])
def test_attention_scores_past_f32(gops, D, G, rows, past, scale):
    """Scores that f32 has no room for: still the largest key's values (of keys within 2^-20 of it, some mean), a single key's
    whatever its sign."""
    c = Case(gops, rows, past, 1, D, 32, seed=46)
    c.fill_past()
    q = torch.randn((c.n, G, D), device="cuda").half()
    got = gops.paged_attn(c.cache, c.batch(), q, scale).double()
    for s, (n, p) in enumerate(zip(rows, past)):
        k, v = c.k[c.key0[s]:c.key0[s + 1], 0], c.v[c.key0[s]:c.key0[s + 1], 0]
        for r in range(n):
            x = k[:p + r + 1] @ q[c.starts[s] + r].double().T * scale
            for h in range(G):
                near = x[:, h] >= x[:, h].max() - x[:, h].abs().max() * 2.0 ** -20
                o, u = got[c.starts[s] + r, h], v[:len(x)][near]
                assert ((o >= u.amin(0) - 1e-5) & (o <= u.amax(0) + 1e-5)).all()


@pytest.mark.parametrize("rows,past", [
    ([1] * 70 + [1, 2], [40 + s for s in range(70)] + [16000, 9000]),       # a few sequences split among many that are not
    ([300, 1, 1, 5], [10, 20000, 17, 12000]), ([1, 1], [0, 24000]), ([1] * 130, [2000 + s for s in range(130)]),
    ([17] * 40 + [1] * 3, [200] * 40 + [9000, 3, 15000]), ([1000, 700], [0, 9000])])
@pytest.mark.parametrize("D,Hkv,G", [(64, 2, 3), (128, 8, 4), (256, 1, 2)])
def test_attention_keeps_to_its_workspace(gops, D, Hkv, G, rows, past):
    """The bytes asked for, holding NaNs before, and none beyond them: sums of split row tiles beside tiles that are not split."""
    import ctypes

    from ggml_compiler_amd import _lib

    c = Case(gops, rows, past, Hkv, D, 256, seed=47)
    c.fill_past()
    q = torch.randn((c.n, G * Hkv, D), device="cuda").half()
    lib, b, most = _lib.load(), c.batch(), max(rows)
    wide = gops.PagedBatch(torch.nn.functional.pad(b.pages, (0, 1024), value=-1).contiguous(), b.starts, b.past)
    for batch in (b, wide):  # (a wider table: more workgroups than have work)
        at = ctypes.addressof(c.cache._c), ctypes.addressof(batch._c)
        n = lib.gcq_paged_attn_workspace(*at, c.n, G * Hkv, most)
        buf = torch.full(((n + 255) // 256 * 256 + 4096,), 0xFF, dtype=torch.uint8, device="cuda")
        out = torch.full((c.n, G * Hkv, D), 77.0, device="cuda")
        _lib.check(lib.gcq_paged_attn(*at, c.n, q.data_ptr(), q.stride(0), q.stride(1), G * Hkv, most, 0, D ** -0.5, out.data_ptr(),
                                      buf.data_ptr(), n, torch.cuda.current_stream().cuda_stream))
        assert bool((buf[n:] == 0xFF).all())
        want, bound = attn_reference(c, q, D ** -0.5)
        check_attn(c, out, want, bound, max(p + r for r, p in zip(rows, past)))


@pytest.mark.parametrize("S,most,H", [(65, 1, 4), (128, 1, 4), (200, 1, 4), (130, 9, 16), (70, 40, 16), (300, 5, 16)])
@pytest.mark.parametrize("D,n_dims", [(64, 64), (128, 40)])
def test_append_more_sequences_than_lanes(gops, orc, S, most, H, D, n_dims):
    """Rows one by one and by eights, some sequences without any: all that is held and given against the encoder, all else as it was."""
    rng = np.random.default_rng(S)
    rows = [1 if most == 1 else int(r) for r in rng.integers(max(1, most - 2), most + 1, S)]
    for s in (0, 3, 63, 64, S - 1):
        rows[s] = 0 if s != 64 else most
    past = [int(p) for p in rng.integers(0, 100, S)]
    c = Case(gops, rows, past, 2, D, 32, seed=S + D, extra_rows=2, fill=0xA5)
    x = c.rng.standard_normal((c.n, H + 4, D)).astype(np.float32)
    t = torch.from_numpy(x).cuda()
    freqs = gops.rope_freqs(n_dims, 10000.0)
    q_out = torch.full((c.n, H, D), 5.0, dtype=torch.float16, device="cuda")
    gops.paged_append(c.cache, c.batch(), t[:, H:H + 2], t[:, H + 2:], q=t[:, :H], freqs=freqs, q_out=q_out)
    k, v = gops.paged_read(c.cache, c.batch(), c.n)
    n, f = int(c.starts[-1]), freqs.cpu().numpy()
    assert np.array_equal(q_out[:n].cpu().numpy(), rotated(x[:n, :H], positions(c), f).astype(np.float16))
    assert (q_out[n:] == 5.0).all()
    assert np.array_equal(k[:n].cpu().numpy(), q4_values(orc, rotated(x[:n, H:H + 2], positions(c), f)))
    assert np.array_equal(v[:n].cpu().numpy(), q4_values(orc, np.ascontiguousarray(x[:n, H + 2:])))
    got = c.cache.data.cpu().numpy()
    rest = np.ones(got.shape, bool)
    rest[layout_bytes(c, [(s, past[s] + j) for s in range(S) for j in range(rows[s])])] = False
    assert (got[rest] == 0xA5).all()


@pytest.mark.parametrize("window", [0, 40, 3000])
def test_attention_of_rows_past_the_table(gops, window):
    """Rows at positions that the page table has no entry for see the keys it has, as far as the window reaches them."""
    Hkv, G, D, page, pages = 2, 4, 128, 32, 6
    rows, past = [1, 5, 1, 40, 1], [pages * page, pages * page + 20, 2000000000, pages * page - 10, 2500]
    c = Case(gops, [pages * page] * 5, [0] * 5, Hkv, D, page, seed=48, extra_cols=0)
    c.fill_past()
    q = torch.from_numpy(c.rng.standard_normal((sum(rows), G * Hkv, D)).astype(np.float32)).cuda().half()
    got = gops.paged_attn(c.cache, c.batch(rows, past), q, D ** -0.5, max_rows=40, window=window)
    at = 0
    for s, (r, p) in enumerate(zip(rows, past)):
        k, v = (x[c.key0[s]:c.key0[s + 1]] for x in (c.k, c.v))
        for j in range(r):
            pos = p + j
            lo, hi = max(0, pos - window + 1) if window else 0, min(pos + 1, pages * page)
            for h in range(G * Hkv):
                if lo >= hi:
                    assert (got[at, h] == 0).all()
                    continue
                w = torch.softmax(k[lo:hi, h // G] @ q[at, h].double() * D ** -0.5, 0)
                want = w @ v[lo:hi, h // G]
                assert ((got[at, h].double() - want).norm() <= 2.0 ** -18 * want.norm()).item()
            at += 1
