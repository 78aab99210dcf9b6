"""examples/paged_talker.py over more steps than its texts are long: the pool, the tables and the rotation table follow."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_paged_example import example, talk64

pytestmark = pytest.mark.gpu


def test_two_hundred_steps(vox):
    r = example().run(streams=8, steps=200, layers=1, dtype=torch.bfloat16)
    t = r["talker"]
    assert len(r["steps"]) == 200 and all(bool(torch.isfinite(y).all()) for _, y in r["steps"])
    # one stream against the model in 64 bits; the bound is test_gpu_paged_example.py's, of two layers
    n = r["texts"][0]
    h = torch.cat([r["voice"][0].double(), r["text"][0][:n].double()] + [x[:1].double().cpu() for x, _ in r["steps"]])
    want = talk64(t, h)[100 + n:]
    got = torch.cat([y[:1] for _, y in r["steps"]]).double().cpu()
    assert (got - want).pow(2).mean().sqrt() <= 0.08 * want.pow(2).mean().sqrt()
    assert vox.device_error() == 0
