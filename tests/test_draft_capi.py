"""CPU-side checks of the C ABI for steps with drafted tokens (include/gcq_draft.h): symbols, sizes, and every refusal made on
the host before anything is launched; and the Python entry points' own refusals."""

import ctypes
import re

import pytest
import torch

from ggml_compiler_amd import _lib, ops
from test_paged_capi import P, _batch, _cache, _refused


def test_every_declared_symbol_is_exported():
    text = re.sub(r"#\s*define[^\n]*", "", _lib.DRAFT_HEADER.read_text())
    names = re.findall(r"GCQ_API[^;(]*?\b(\w+)\s*\(", text)
    assert len(names) == 6 and set(names) <= set(_lib.SIGNATURES)
    lib = _lib.load()
    assert all(hasattr(lib, n) for n in names)


def _tree(batch=None, **kw):
    a = {"n_rows": 5, "parents": P, "max_rows": 4, "window": 0, "positions": P, "mask": P, "ld_mask": 1, "stream": None} | kw
    b = batch or _batch()
    return _lib.load().gcq_draft_tree(ctypes.addressof(b), *a.values())


def _append(cache=None, batch=None, **kw):
    a = {"n_rows": 5, "positions": P, "k": P, "k_r": 256, "k_h": 128, "v": P, "v_r": 256, "v_h": 128, "q": P, "q_r": 512, "q_h": 128,
         "H": 4, "q_out": P, "freqs": P, "n_dims": 128, "attn_factor": 1.0, "stream": None} | kw
    c, b = cache or _cache(), batch or _batch()
    return _lib.load().gcq_paged_append_at(ctypes.addressof(c), ctypes.addressof(b), *a.values())


def _attn(cache=None, batch=None, **kw):
    a = {"n_rows": 5, "positions": P, "mask": P, "ld_mask": 1, "q": P, "q_r": 512, "q_h": 128, "H": 4, "max_rows": 2, "window": 0,
         "scale": 0.1, "out": P, "ws": P, "ws_size": 1 << 40, "stream": None} | kw
    c, b = cache or _cache(), batch or _batch()
    return _lib.load().gcq_paged_attn_tree(ctypes.addressof(c), ctypes.addressof(b), *a.values())


def _verify(**kw):
    a = {"starts": P, "n_seq": 3, "n_rows": 5, "parents": P, "tokens": P, "logits": P, "ld": 100, "draft_logits": P, "draft_ld": 100,
         "n_vocab": 100, "temperature": P, "coins": P, "max_rows": 4, "max_path": 4, "count": P, "rows": P, "tokens_out": P, "ws": P,
         "ws_size": 1 << 40, "stream": None} | kw
    return _lib.load().gcq_draft_verify(*a.values())


def _move(caches=None, batch=None, **kw):
    caches = [_cache()] if caches is None else caches
    a = {"count": P, "rows": P, "ld_rows": 4, "max_keep": 4, "stream": None} | kw
    at, b = (ctypes.c_void_p * max(1, len(caches)))(*[c and ctypes.addressof(c) for c in caches]), batch or _batch()
    return _lib.load().gcq_paged_move(at, len(caches), ctypes.addressof(b), *a.values())


def test_tree_refusals():
    _refused(_tree(_batch(n_seq=0)), "at least one sequence")
    _refused(_tree(n_rows=-1), "n_rows")
    _refused(_tree(n_rows=1 << 30), "n_rows")
    _refused(_tree(max_rows=0), "max_rows")
    _refused(_tree(ld_mask=0), "ld_mask")
    _refused(_tree(ld_mask=33), "ld_mask")
    _refused(_tree(n_rows=40, max_rows=33), "max_rows past the mask's bits")
    _refused(_tree(window=-1), "window")
    _refused(_tree(parents=None), "parents is NULL")
    _refused(_tree(positions=None), "positions is NULL")
    _refused(_tree(mask=P + 2), "mask must be 4-byte aligned")
    _refused(_tree(_batch(starts=None)), "starts is NULL")
    _refused(_tree(_batch(past=None)), "past is NULL")
    assert _tree(n_rows=0) == 0  # nothing to do


def test_append_at_refusals():
    _refused(_append(positions=None), "positions is NULL")
    _refused(_append(positions=P + 1), "4-byte aligned")
    _refused(_append(k=None), "k is NULL")
    _refused(_append(n_dims=130), "n_dims")
    _refused(_append(_cache(head_dim=96)), "pages of 32")
    _refused(_append(n_rows=-1), "n_rows")
    assert _append(n_rows=0, positions=None) == 0


def test_attn_tree_refusals():
    _refused(_attn(mask=None), "mask is NULL")
    _refused(_attn(mask=P + 2), "4-byte aligned")
    _refused(_attn(positions=None, window=8), "positions is NULL")
    _refused(_attn(ld_mask=0), "ld_mask")
    _refused(_attn(ld_mask=33), "ld_mask")
    _refused(_attn(n_rows=64, max_rows=33), "max_rows past the mask's bits")
    _refused(_attn(q=None), "q is NULL")
    _refused(_attn(H=3), "multiple of n_head_kv")
    _refused(_attn(max_rows=0), "max_rows")
    _refused(_attn(window=-1), "window")
    _refused(_attn(scale=float("inf")), "scale")
    _refused(_attn(ws_size=128), "workspace of 128 bytes")
    _refused(_attn(None, _batch(starts=None)), "starts is NULL")
    assert _attn(n_rows=0, mask=None) == 0


def test_verify_refusals():
    lib = _lib.load()
    assert lib.gcq_draft_verify_workspace(3, 5, 100, 4) >= 256
    for bad, text in (((0, 5, 100, 4), "sequence"), ((3, -1, 100, 4), "n_rows"), ((3, 5, 0, 4), "n_vocab"), ((3, 5, 1 << 30, 4), "n_vocab"),
                      ((3, 5, 100, 0), "max_rows"), ((3, 2000, 100, 1025), "max_rows"), ((1 << 30, 5, 100, 4), "sequence"),
                      ((1 << 29, 5, 1 << 29, 4), "too many")):
        assert lib.gcq_draft_verify_workspace(*bad) == 0
        assert text in lib.gcq_last_error().decode()
    assert lib.gcq_draft_verify_workspace(3, 5, 100, 5000) >= 256  # no more rows than there are
    for name in ("starts", "parents", "tokens", "logits", "coins", "count", "rows", "tokens_out"):
        _refused(_verify(**{name: None}), f"{name} is NULL")
        _refused(_verify(**{name: P + 2}), f"{name} must be 4-byte aligned")
    _refused(_verify(draft_logits=P + 2), "draft_logits must be")
    _refused(_verify(temperature=P + 2), "temperature must be")
    _refused(_verify(ld=99), "rows of logits overlap")
    _refused(_verify(draft_ld=99), "rows of draft_logits overlap")
    _refused(_verify(max_path=0), "max_path")
    _refused(_verify(ws=None), "workspace is NULL")
    _refused(_verify(ws=P + 128), "256-byte aligned")
    _refused(_verify(ws_size=100), "workspace of 100 bytes")


def test_move_refusals():
    _refused(_move([]), "at least one cache")
    _refused(_move([None]), "cache is NULL")
    _refused(_move([_cache(), _cache(page_size=32)]), "of one shape")
    _refused(_move([_cache(), _cache(n_pages=5)]), "of one shape")
    _refused(_move([_cache(data=None)]), "cache data is NULL")
    _refused(_move(count=None), "count is NULL")
    _refused(_move(rows=P + 2), "rows must be 4-byte aligned")
    _refused(_move(ld_rows=3), "max_keep")
    _refused(_move(max_keep=-1), "max_keep")
    _refused(_move(None, _batch(pages=None)), "pages is NULL")
    same = _cache()
    _refused(_move([same, same]), "caches overlap")
    _refused(_move([_cache(data=P + (1 << 40)), _cache(), _cache(data=P + 4096)]), "caches overlap")
    assert _move(max_keep=0) == 0
    assert _move([_cache(data=P + (1 << 40)), _cache(), _cache(data=P + (1 << 30))], max_keep=0) == 0


def test_python_refusals_without_a_device():
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="device tensor"):
        ops.DraftTree(i, i, i.view(4, 1))


def test_verify_refuses_what_cannot_be_launched():
    """Before anything is: the draws' workgroups, one to a sequence at the least, are counted first."""
    _refused(_verify(n_seq=1 << 23), "too many rows")
    _refused(_verify(n_seq=1 << 23, draft_logits=None), "too many rows")
    _refused(_verify(n_rows=1 << 26, max_rows=5), "too many rows")


def test_move_reads_pages_and_past_alone():
    """A batch without starts, or with any, is moved; pages and past are looked at."""
    assert _move(None, _batch(starts=None), max_keep=0) == 0
    assert _move(None, _batch(starts=P + 2), max_keep=0) == 0
    _refused(_move(None, _batch(starts=None, past=None)), "past is NULL")
    _refused(_move(None, _batch(past=P + 1)), "past must be 4-byte aligned")
    _refused(_move(None, _batch(pages=P + 2)), "pages must be 4-byte aligned")
    _refused(_move([_cache(data=P + 8)]), "cache data must be 16-byte aligned")
