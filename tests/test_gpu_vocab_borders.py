"""Operators along the vocabulary axis at the borders of their definitions, against the 64-bit oracle; tolerances as in test_gpu_vocab.py."""
import math

import pytest
import torch

from oracle import vocab as O
from test_gpu_vocab import DT, _check_distill, _logits, _teacher

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tag", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [3, 100, 300])   # slices of an eighth and a quarter of a row, whole rows
@pytest.mark.parametrize("tail", [False, True])
def test_distill_rows_with_a_few_logits_near_the_cap(tag, rows, tail):
    """Single lanes of a warp meet logits beyond three quarters of the cap (22.5 of 30) in slices long enough for batched loads; the
    first row has none, the second some in every slice, the third one alone."""
    g = torch.Generator().manual_seed(rows)
    V, K = 50304, 32
    x = _logits(g, rows, V, DT[tag])
    x.clamp_(-20.0, 20.0)
    x[1, torch.randint(0, V, (40,), generator=g)] = 27.0
    x[2, 40001] = -45.0
    values, ids, lse = _teacher(g, x[:4], K, 30.0, 1.0, tail, holes=False)
    values, ids, lse = (None if t is None else torch.cat([t, t[-1:].expand(rows - t.shape[0], *t.shape[1:])]) if rows > t.shape[0] else t for t in (values, ids, lse))
    _check_distill(x, values, ids, 30.0, 1.0, lse, torch.rand(rows, generator=g), only=slice(0, 4))
