"""CPU-side checks of the paged cache's C ABI (include/gcq_paged.h): symbols, sizes, and every refusal made on the host
before anything is launched; and the Python entry points' own refusals."""

import ctypes
import re

import pytest
import torch

from ggml_compiler_amd import _lib, ops


def test_every_declared_symbol_is_exported():
    text = re.sub(r"#\s*define[^\n]*", "", _lib.PAGED_HEADER.read_text())
    names = re.findall(r"GCQ_API[^;(]*?\b(\w+)\s*\(", text)
    assert len(names) == 5 and set(names) <= set(_lib.SIGNATURES)
    lib = _lib.load()
    assert all(hasattr(lib, n) for n in names)


def test_cache_sizes():
    size = _lib.load().gcq_paged_cache_size
    for D in (64, 128, 256):
        for page in (32, 64, 128, 256):
            # K and V: D / 2 code bytes and D / 32 f16 scales a token and head
            assert size(7, page, 3, D) == 7 * page * 3 * 2 * (D // 2 + D // 16)
    assert size(1 << 20, 256, 8, 256) == (1 << 20) * 256 * 8 * 288  # past 32 bits
    for bad in ((0, 64, 8, 128), (4, 16, 8, 128), (4, 48, 8, 128), (4, 512, 8, 128), (4, 64, 0, 128), (4, 64, 8, 96),
                (4, 64, 8, 0), (-1, 64, 8, 128), (4, 64, 65536, 128)):
        assert size(*bad) == 0
        assert "pages of 32" in _lib.load().gcq_last_error().decode()


P = 4096  # an address that nothing may read


def _cache(**kw):
    a = {"data": P, "n_pages": 4, "page_size": 64, "n_head_kv": 2, "head_dim": 128} | kw
    return _lib.PagedCache(*a.values())


def _batch(**kw):
    a = {"pages": P, "ld_pages": 4, "starts": P, "past": P, "n_seq": 3, "max_pages": 4} | kw
    return _lib.PagedBatch(*a.values())


def _refused(rc, text):
    assert rc == -1
    assert text in _lib.load().gcq_last_error().decode(), _lib.load().gcq_last_error().decode()


def _append(cache=None, batch=None, **kw):
    a = {"n_rows": 5, "k": P, "k_r": 256, "k_h": 128, "v": P, "v_r": 256, "v_h": 128, "q": P, "q_r": 512, "q_h": 128,
         "H": 4, "q_out": P, "freqs": P, "n_dims": 128, "attn_factor": 1.0, "stream": None} | kw
    c, b = cache or _cache(), batch or _batch()
    return _lib.load().gcq_paged_append(ctypes.addressof(c), ctypes.addressof(b), *a.values())


def _read(cache=None, batch=None, **kw):
    a = {"n_rows": 5, "k": P, "v": P, "stream": None} | kw
    c, b = cache or _cache(), batch or _batch()
    return _lib.load().gcq_paged_read(ctypes.addressof(c), ctypes.addressof(b), *a.values())


def _attn(cache=None, batch=None, **kw):
    a = {"n_rows": 5, "q": P, "q_r": 512, "q_h": 128, "H": 4, "max_rows": 2, "window": 0, "scale": 0.1, "out": P, "ws": P,
         "ws_size": 1 << 40, "stream": None} | kw
    c, b = cache or _cache(), batch or _batch()
    return _lib.load().gcq_paged_attn(ctypes.addressof(c), ctypes.addressof(b), *a.values())


@pytest.mark.parametrize("call", [_append, _read, _attn])
def test_cache_and_batch_refusals(call):
    _refused(call(_cache(data=None)), "cache data is NULL")
    _refused(call(_cache(data=P + 8)), "16-byte aligned")
    _refused(call(_cache(page_size=48)), "pages of 32")
    _refused(call(_cache(head_dim=80)), "pages of 32")
    _refused(call(_cache(n_pages=0)), "pages of 32")
    _refused(call(None, _batch(pages=None)), "pages is NULL")
    _refused(call(None, _batch(starts=None)), "starts is NULL")
    _refused(call(None, _batch(past=P + 2)), "past must be 4-byte aligned")
    _refused(call(None, _batch(n_seq=0)), "at least one sequence")
    _refused(call(None, _batch(max_pages=0)), "at least one sequence")
    _refused(call(None, _batch(ld_pages=3)), "ld_pages >= max_pages")
    _refused(call(n_rows=-1), "n_rows")
    _refused(call(n_rows=1 << 30), "n_rows")
    assert call(n_rows=0) == 0  # nothing to do


def test_append_refusals():
    _refused(_append(k=None), "k is NULL")
    _refused(_append(v=None), "v is NULL")
    _refused(_append(k=P + 2), "4-byte aligned")
    _refused(_append(k_r=-256), "negative strides")
    _refused(_append(q_out=None), "q_out is NULL")
    _refused(_append(H=0), "n_head")
    _refused(_append(n_dims=130), "n_dims")
    _refused(_append(n_dims=63), "n_dims")
    _refused(_append(n_dims=0), "n_dims")
    _refused(_append(attn_factor=float("inf")), "attn_factor")


def test_read_refusals():
    _refused(_read(k=None), "k is NULL")
    _refused(_read(v=P + 8), "16-byte aligned")


def test_attn_refusals():
    _refused(_attn(q=None), "q is NULL")
    _refused(_attn(q=P + 8), "16-byte aligned")
    _refused(_attn(out=None), "out is NULL")
    _refused(_attn(ws=P + 128), "256-byte aligned")
    _refused(_attn(H=3), "multiple of n_head_kv")
    _refused(_attn(H=0), "multiple of n_head_kv")
    _refused(_attn(q_r=516), "multiples of 8")
    _refused(_attn(q_h=-128), "multiples of 8")
    _refused(_attn(max_rows=0), "max_rows")
    _refused(_attn(window=-1), "window")
    _refused(_attn(scale=float("nan")), "scale")
    _refused(_attn(ws_size=128), "workspace of 128 bytes")
    lib, c, b = _lib.load(), _cache(), _batch()
    at = ctypes.addressof(c), ctypes.addressof(b)
    assert lib.gcq_paged_attn_workspace(*at, 5, 4, 2) >= 256
    assert lib.gcq_paged_attn_workspace(*at, 5, 3, 2) == 0
    assert lib.gcq_paged_attn_workspace(*at, 5, 4, 0) == 0
    assert lib.gcq_paged_attn_workspace(*at, -1, 4, 2) == 0


def test_python_refusals_without_a_device():
    with pytest.raises(ValueError, match="device tensor"):
        ops.PagedCache(1, 32, 1, 64, torch.zeros(1 * 32 * 72, dtype=torch.uint8))
    with pytest.raises(_lib.GcqError, match="pages of 32"):
        ops.PagedCache.new(1, 33, 1, 64)
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="device tensor"):
        ops.PagedBatch(i.view(1, 4), i[:2], i[:1])


def test_rope_freqs():
    f = ops.rope_freqs(8, 10000.0, 0.5, torch.tensor([1.0, 2.0, 4.0, 8.0]), device="cpu")
    want = [0.5 * 10000.0 ** (-i / 4) / 2 ** i for i in range(4)]
    assert f.dtype == torch.float32 and torch.equal(f, torch.tensor(want, dtype=torch.float64).float())


def test_hand_written_loads_declare_what_they_change():
    """An asm statement that sets m0 says so, and leaves the five wait states that a vector memory access needs behind a v_readlane
    which may have written its scalar base just before (the compiler counts none of them inside asm)."""
    found = 0
    for path in sorted((_lib.LIBRARY.parents[1] / "csrc").glob("*.h*")):
        text = path.read_text()
        for m in re.finditer(r"\basm\b(?:\s+volatile)?\s*\(((?:[^()\"]|\"(?:[^\"\\]|\\.)*\"|\([^()]*\))*)\)\s*;", text):
            code, *operands = re.split(r"(?<!:):(?!:)|::", m.group(1))
            if "m0" not in code:
                continue
            found += 1
            assert operands and '"m0"' in operands[-1], (path.name, m.group(0))
            assert "load" in code
            before = code[:code.index("load")].split("\\n\\t")
            states = sum(1 + int(i.split()[-1]) if "s_nop" in i else 1 for i in before[:-1])
            assert states >= 5, (path.name, m.group(0))
    assert found


def test_more_threads_than_a_launch_takes():
    """A launch of 2^32 threads or more is refused here, whatever the driver makes of it."""
    many = "too many rows and heads"
    _refused(_append(n_rows=1 << 27), many)                   # by eights
    _refused(_append(n_rows=1 << 26, k_r=255), many)          # row by row
    _refused(_read(n_rows=1 << 28), many)
    _refused(_read(_cache(n_head_kv=65535), n_rows=1 << 13), many)
    _refused(_attn(n_rows=1 << 28, max_rows=1 << 28, ws_size=1 << 62), many)
    _refused(_attn(_cache(head_dim=256), n_rows=1 << 28, max_rows=1 << 28, ws_size=1 << 62), many)


def test_attn_workspace_does_not_grow_with_the_rows():
    """Sums are kept of split row tiles alone, whose number the plan bounds; a note of 32 bytes for each workgroup besides."""
    lib, c = _lib.load(), _cache(n_head_kv=8, n_pages=1 << 20)
    b = _batch(max_pages=2048, ld_pages=2048, n_seq=1)
    at = ctypes.addressof(c), ctypes.addressof(b)
    for n in (8192, 65536):
        # a workgroup to 16 rows of a KV head; two times 1024 sums of 16 rows, or 768 of 32
        assert lib.gcq_paged_attn_workspace(*at, n, 32, n) <= n * 4 // 16 * 8 * 32 + 1024 * 32 + 2 * 768 * 32 * (128 * 4 + 8) + (1 << 20)
