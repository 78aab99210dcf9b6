"""CPU tests of what the paged-cache calls promise beyond single bad arguments: batches whose parts contradict one another, and
what their documents say."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest
import torch

from tests.test_paged_host import batch, cache, size, v  # noqa: F401

ROOT = Path(__file__).resolve().parents[1]


def test_tokens_of_no_sequence_are_refused(v):  # noqa: F811
    """Tokens without a sequence would leave their rows of q and out unwritten."""
    c = cache(v)
    L = v.lib
    for b in (batch(seqs=0, tokens=3), batch(seqs=0, tokens=3, page_table=None, kv_len=None), batch(seqs=0, tokens=3, q_start=4096)):
        C, B = ctypes.byref(c), ctypes.byref(b)
        for rc in (size(v, c, b)[0],
                   L.vox_cuda_attn_paged(C, B, 4096, 256, 8192, 256, 4, 0.1, 0, 1, None, 0, None),
                   L.vox_cuda_attn_prefix(C, B, 4096, 10, 4096, 256, 8192, 256, 4, 0.1, 1, None, 0, None),
                   L.vox_cuda_kv_append(C, B, 4096, 512, None, None, 4096, 64, 8192, 256, 4, 1e-6, 1, None)):
            assert rc == -6
            assert "without a sequence" in L.vox_cuda_last_error().decode()


def test_documents_say_which_rotation_stands_behind_a_prefix(v):  # noqa: F811
    """The append rotates by the row in the sequence's own pages, so behind a shared prefix its table starts at row prefix_len.
    Whoever calls the two operators finds that at each of them, and the documented call does it."""
    header = (ROOT / "include" / "vox_cuda.h").read_text()
    at = {n: header.index("int " + n + "(") for n in ("vox_cuda_kv_append", "vox_cuda_attn_paged", "vox_cuda_attn_prefix", "vox_cuda_attn_workspace")}
    before = {"vox_cuda_kv_append": header.rindex("/*", 0, at["vox_cuda_kv_append"]), "vox_cuda_attn_prefix": at["vox_cuda_attn_paged"]}
    for n, start in before.items():
        text = " ".join(header[start:at[n]].replace("*", " ").split())
        assert "from row prefix_len on" in text, n
    seam = (ROOT / "include" / "vox_gpu_cuda.hpp").read_text()
    assert "from row prefix_len on" in " ".join(seam[:seam.index("bool gpu_attn_prefix(")].replace("//", " ").split())
    for f in (v.PagedKV.append, v.PagedKV.attend_prefix):
        assert "cs[prefix_len:]" in f.__doc__, f
    guide = (ROOT / "INTEGRATION.md").read_text()
    calls = re.findall(r"gpu_kv_append\(([^;]*)\);", guide)
    assert calls and all("prefix_len" in c for c in calls)


def test_size_query_names_all_that_it_depends_on(v):  # noqa: F811
    """The bytes follow from the whole description of the batch: with and without token offsets they differ, and so they do with the
    table's width where max_kv is left to it."""
    c = cache(v)
    big = dict(tokens=40, seqs=10, table_width=400, table_stride=400)
    need = [size(v, c, batch(**big), prefix=900), size(v, c, batch(q_start=4096, **big), prefix=900),
            size(v, c, batch(**{**big, "table_width": 1}), prefix=900)]
    assert all(rc == 0 for rc, _ in need) and len({n for _, n in need}) > 1
    header = (ROOT / "include" / "vox_cuda.h").read_text()
    end = header.index("int vox_cuda_attn_workspace(")
    text = " ".join(header[header.rindex("/*", 0, end):end].replace("*", " ").split())
    for word in ("q_start", "table_width", "current device", "not read", "NULL"):
        assert word in text, word
    assert "host arithmetic only" not in (ROOT / "INTEGRATION.md").read_text()


def test_bounds_that_do_not_fit_are_refused_in_the_library_s_manner(v):  # noqa: F811
    """max_q and max_kv are 32-bit numbers: others are an argument error of the library, not of the packing below it."""
    kv = v.PagedKV.__new__(v.PagedKV)
    kv._dev = -1  # host tensors stand in for a batch: nothing is called
    table, lens = torch.zeros((2, 3), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    assert len(kv._batch(2, table, lens, None, 1, 2 ** 31 - 1)) == 56
    for mq, mkv in ((2 ** 31, 0), (0, 2 ** 40), (0, -2 ** 31 - 1), (1.5, 0), (0, None)):
        with pytest.raises(v.VoxCudaError, match="max_q and max_kv"):
            kv._batch(2, table, lens, None, mq, mkv)
