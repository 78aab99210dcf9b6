"""CPU tests of what the paged-cache calls promise beyond single bad arguments: batches whose parts contradict one another, and
what their documents say."""

from __future__ import annotations

import ctypes

from tests.test_paged_host import batch, cache, size, v  # noqa: F401


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
