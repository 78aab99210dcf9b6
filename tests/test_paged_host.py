"""CPU tests of the paged cache operators' boundary: the C entries refuse bad arguments with a message before touching the
device, the size query agrees with itself, empty batches are no error."""

from __future__ import annotations

import ctypes

import pytest


@pytest.fixture(scope="module")
def v():
    from vox_b200 import build

    build.build()
    import vox_b200

    return vox_b200


class Batch(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("page_table", "kv_len", "q_start")] + \
               [(n, ctypes.c_int64) for n in ("table_stride", "tokens")] + \
               [(n, ctypes.c_int32) for n in ("seqs", "table_width", "max_q", "max_kv")]


def cache(v, **k):
    d = dict(k=4096, v=4096, dtype=1, page_size=16, pages=8, kv_heads=2, head_dim=64, page_stride=16 * 128, row_stride=128, head_stride=64)
    d.update(k)
    return v._KvCache(*[d[n] for n, _ in v._KvCache._fields_])


def batch(**k):
    d = dict(page_table=4096, kv_len=4096, q_start=None, table_stride=4, tokens=3, seqs=3, table_width=4, max_q=0, max_kv=0)
    d.update(k)
    return Batch(*[d[n] for n, _ in Batch._fields_])


def size(v, c, b, heads=4, prefix=0, window=0, dtype=1):
    n = ctypes.c_size_t(12345)
    rc = v.lib.vox_cuda_attn_workspace(ctypes.byref(c), ctypes.byref(b), prefix, heads, window, dtype, ctypes.byref(n))
    return rc, n.value


BAD = [(dict(page_size=24), {}, -6, "page_size"), (dict(page_size=8), {}, -6, "page_size"), (dict(page_size=1 << 21), {}, -6, "page_size"),
       (dict(head_dim=96), {}, -8, "head_dim"), (dict(dtype=2), {}, -6, "f32 or bf16"), (dict(pages=0), {}, -6, "shape"),
       (dict(row_stride=130), {}, -6, "strides"), (dict(page_stride=0), {}, -6, "strides"), (dict(k=4100), {}, -6, "aligned"),
       (dict(k=None), {}, -6, "NULL"), ({}, dict(kv_len=None), -6, "NULL"), ({}, dict(page_table=None), -6, "NULL"),
       ({}, dict(tokens=4), -6, "multiple of seqs"), ({}, dict(seqs=-1), -6, "batch shape"), ({}, dict(table_stride=3), -6, "batch shape"),
       ({}, dict(table_width=1 << 28, table_stride=1 << 28), -6, "out of range"), ({}, dict(max_kv=-1), -6, "batch shape")]


@pytest.mark.parametrize("c,b,status,word", BAD)
def test_refusals(v, c, b, status, word):
    c, b = cache(v, **c), batch(**b)
    L = v.lib
    assert size(v, c, b)[0] == status and word in L.vox_cuda_last_error().decode()
    assert L.vox_cuda_attn_paged(ctypes.byref(c), ctypes.byref(b), 4096, 256, 8192, 256, 4, 0.1, 0, 1, None, 0, None) == status
    assert L.vox_cuda_attn_prefix(ctypes.byref(c), ctypes.byref(b), 4096, 10, 4096, 256, 8192, 256, 4, 0.1, 1, None, 0, None) == status
    assert L.vox_cuda_kv_append(ctypes.byref(c), ctypes.byref(b), 4096, 512, None, None, 4096, 64, 8192, 256, 4, 1e-6, 1, None) == status
    assert word in L.vox_cuda_last_error().decode()


def test_refusals_of_the_calls(v):
    c, b = cache(v), batch()
    L, C, B = v.lib, ctypes.byref(c), ctypes.byref(b)
    attend = lambda q=4096, qs=256, o=8192, os=256, heads=4, window=0, dt=1, ws=None, wb=0: \
        L.vox_cuda_attn_paged(C, B, q, qs, o, os, heads, 0.1, window, dt, ws, wb, None)  # noqa: E731
    for kw, word in ((dict(q=None), "NULL"), (dict(heads=3), "multiple of kv_heads"), (dict(qs=255), "aligned"), (dict(qs=128), "aligned"),
                     (dict(q=4100), "aligned"), (dict(window=-1), "window"), (dict(dt=2), "dtype")):
        assert attend(**kw) == -6 and word in L.vox_cuda_last_error().decode(), kw
    assert L.vox_cuda_attn_prefix(C, B, None, 10, 4096, 256, 8192, 256, 4, 0.1, 1, None, 0, None) == -6
    rc, need = size(v, c, b, prefix=4000)
    assert rc == 0 and need > 0
    assert L.vox_cuda_attn_prefix(C, B, 4096, 4000, 4096, 256, 8192, 256, 4, 0.1, 1, None, 0, None) == -6
    assert "workspace" in L.vox_cuda_last_error().decode()
    assert L.vox_cuda_attn_prefix(C, B, 4096, 4000, 4096, 256, 8192, 256, 4, 0.1, 1, 4096 + 16, need, None) == -6
    assert L.vox_cuda_attn_prefix(C, B, 4096, 4000, 4096, 256, 8192, 256, 4, 0.1, 1, 4096, need - 1, None) == -6
    app = lambda qs=512, q=8192, cs=4096, rows=64: L.vox_cuda_kv_append(C, B, 4096, qs, None, None, cs, rows, q, 256, 4, 1e-6, 1, None)  # noqa: E731
    for kw, word in ((dict(qs=256), "strides"), (dict(q=None), "NULL"), (dict(cs=4100), "aligned"), (dict(rows=0), "out of range")):
        assert app(**kw) == -6 and word in L.vox_cuda_last_error().decode(), kw


def test_empty_batches_need_nothing(v):
    c = cache(v)
    for b in (batch(seqs=0, tokens=0, page_table=None, kv_len=None), batch(tokens=0)):
        assert size(v, c, b) == (0, 0)
        assert v.lib.vox_cuda_attn_paged(ctypes.byref(c), ctypes.byref(b), None, 0, None, 0, 4, 0.1, 0, 1, None, 0, None) == 0
        assert v.lib.vox_cuda_kv_append(ctypes.byref(c), ctypes.byref(b), None, 0, None, None, None, 0, None, 0, 4, 1e-6, 1, None) == 0


def test_packed_batch_matches_the_header(v):
    raw = v._pack_batch(1, 2, 3, 4, 5, 6, 7, 8, 9)
    assert bytes(Batch(1, 2, 3, 4, 5, 6, 7, 8, 9)) == raw and len(raw) == ctypes.sizeof(Batch) == 56
    assert ctypes.sizeof(v._KvCache) == 64


def test_header_declares_and_library_exports_the_operators(v):
    from tests.test_abi import declared_functions

    for n in ("vox_cuda_kv_append", "vox_cuda_attn_paged", "vox_cuda_attn_prefix", "vox_cuda_attn_workspace"):
        assert n in declared_functions() and hasattr(v.lib, n)
