"""Edges of the operators over a paged cache: padding pairs among forks."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from _ops64 import Pages
from llm_serving_runtime_b200 import DevicePages

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _pages_beside_the_plain_table(P, bs, S, M):
    return DevicePages(P, bs, S, M), Pages([[-1] * M for _ in range(S)], [0] * S, [0] * P, bs)


def _step(pages, table, name, *args):
    getattr(table, name)(*args)
    table.moves = []
    getattr(pages, name)(*[_i32(a) for a in args], validate=False)
    assert pages.read_errors() == table.flags
    table.flags = 0
    assert pages.block_tables.tolist() == table.tables
    assert pages.seq_lens.tolist() == table.lens and pages.ref_counts.tolist() == table.refs


def test_a_padding_pair_does_not_claim_its_child():
    """A pair without a parent is padding whatever its child is: a later pair may name it."""
    pages, table = _pages_beside_the_plain_table(20, 4, 6, 5)
    _step(pages, table, "reserve", [0, 1], [6, 9])
    _step(pages, table, "fork", [-1, 0, -1], [3, 3, 3])
    assert table.lens[3] == 6
    _step(pages, table, "fork", [-1, -1, 1, 1, 0], [4, 5, 5, 5, 4])  # 5 a second time is an error
    assert table.lens[4:] == [6, 9]


@pytest.mark.parametrize("seed", range(8))
def test_forks_among_padding_pairs(seed):
    rng = np.random.default_rng(seed)
    S = int(rng.integers(4, 1500))
    pages, table = _pages_beside_the_plain_table(4 * S, 3, S, 3)
    full = S // 3
    _step(pages, table, "reserve", list(range(full)), rng.integers(1, 7, full).tolist())
    for _ in range(4):
        n = int(rng.integers(2, S + 1))
        parents = np.where(rng.random(n) < 0.5, -1, rng.integers(0, full, n))
        children = rng.integers(full, S, n)
        _step(pages, table, "fork", parents.tolist(), children.tolist())
        _step(pages, table, "free", rng.permutation(np.arange(full, S))[: (S - full) // 2].tolist())
