"""Calls of the window-cache operators at the edges of what their documentation
allows, against their definitions in 64 bits (tests/cache_reference.py)."""
import itertools

import pytest
import torch

import cache_reference as ref
from streaming_transformer_b200.runtime import StreamError
from test_gpu_cache import TYPES, filled_cache, generator, normal, scales_of, starts_of, window_reference

pytestmark = pytest.mark.gpu

ops = pytest.importorskip("streaming_transformer_b200.attention")


@pytest.mark.parametrize("rows", [3, 40])
def test_more_sequences_than_half_of_the_integers(rows):
    # 2^30 + 2^27 sequences (4.8 GB of starts), all empty but two of the last ones
    sequences = 2 ** 30 + 2 ** 27
    starts = torch.zeros(sequences + 1, dtype=torch.int32, device="cuda")
    starts[sequences - 3:] = rows - 1
    starts[sequences] = rows
    g = generator(51)
    q, k, v = (normal(g, rows, h, 64, dtype=torch.bfloat16) for h in (4, 2, 2))
    got = ops.window_attention(q, k, v, window=7, sinks=1, starts=starts)
    for a, b, want, bound in window_reference(q, k, v, [0, rows - 1, rows], 7, 1, 0.125, torch.bfloat16):
        ref.check(got[a:b], want, bound, f"rows {a}..{b}")
