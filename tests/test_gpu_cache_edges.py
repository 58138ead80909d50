"""Calls of the window-cache operators at the edges of what their documentation
allows, against their definitions in 64 bits (tests/cache_reference.py)."""
import ctypes
import itertools

import pytest
import torch

import cache_reference as ref
from streaming_transformer_b200.runtime import StreamError
import test_cache_cpu as c_calls
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


def test_a_call_for_a_device_that_is_not_there_leaves_no_error_behind():
    lib, need, missing = c_calls.entry_points(), ctypes.c_size_t(), torch.cuda.device_count()
    cache, _ = filled_cache(generator(52), 1, 2, 9, 64, 0, "bf16")
    q = torch.ones(1, 4, 64, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([8], device="cuda")
    want = ops.cache_attention(q, *cache[:2], at)
    absent = c_calls.cache(device=missing)
    for call in (lambda: lib.st_cache_append(absent, c_calls.append(), None),
                 lambda: lib.st_cache_unpack(c_calls.cache(device=missing, **c_calls.FOUR), 2, c_calls.P, c_calls.P, None),
                 lambda: lib.st_cache_attention(absent, c_calls.attend(), None),
                 lambda: lib.st_window_attention(c_calls.window(device=missing), None)):
        assert call() == -3 and b"device" in lib.st_cache_error()
        assert torch.equal(ops.cache_attention(q, *cache[:2], at), want)
    lib.st_cache_attention_workspace(absent, 4, need)
    assert torch.equal(ops.cache_attention(q, *cache[:2], at), want)
