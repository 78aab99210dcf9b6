"""CPU tests of examples/paged_talker.py's pool of pages: its size follows from the streams' lengths, and an empty pool or a full
table says so."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("paged_talker", ROOT / "examples" / "paged_talker.py")
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("texts", [[5], [5, 44, 16, 17], [44] * 8])
@pytest.mark.parametrize("steps", [0, 1, 200, 3000])
@pytest.mark.parametrize("voice", [1, 100, 128])
def test_pool_holds_every_step(example, page, texts, steps, voice):
    pages, width, positions = example.sizes(texts, steps, voice, page)
    pool = example.Pool(pages, page, len(texts), width)
    taken = set(pool.take(-(-voice // page)))
    lens = list(texts)
    pool.grow(lens)
    for _ in range(steps):
        lens = [n + 1 for n in lens]
        pool.grow(lens)
    assert positions >= voice + max(lens)
    for b, n in enumerate(lens):
        of = pool.table[b, :-(-n // page)].tolist()
        assert not taken & set(of) and len(set(of)) == len(of)
        taken |= set(of)
    assert len(taken) <= pages


def test_empty_pool_and_full_table_are_named(example):
    pool = example.Pool(3, 16, 1, 8)
    with pytest.raises(RuntimeError, match="page"):
        pool.grow([50])
    pool = example.Pool(9, 16, 1, 2)
    with pytest.raises(RuntimeError, match="table"):
        pool.grow([50])
    with pytest.raises(RuntimeError, match="page"):
        example.Pool(3, 16, 1, 8).take(4)
