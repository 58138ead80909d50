"""Refusals of the window-cache operators that need no GPU: derivatives that a call
would drop, and C arguments that a kernel could not read."""
import pytest

torch = pytest.importorskip("torch")

from test_cache_cpu import FOUR, P, Rows, append as append_struct, attend as attend_struct, cache, entry_points, refused, rows, window as window_struct

from streaming_transformer_b200 import StreamError
from streaming_transformer_b200 import attention as ops


def append_arguments(four):
    """Names to tensors of one append; None where there is none."""
    row = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    cache = ops.new_cache(1, 1, 4, 64, mode="int4" if four else "bf16", device="cpu")
    return dict(zip(("keys", "values", "key_scales", "value_scales"), cache)) | dict(
        q=row.clone(), k=row.clone(), v=row.clone(), frequencies=ops.rotation_frequencies(64, device="cpu"),
        q_gain=torch.ones(64), k_gain=torch.ones(64), out=row.clone())


def append(t):
    return ops.cache_append(t["q"], t["k"], t["v"], t["keys"], t["values"], torch.zeros(1, dtype=torch.int64), t["frequencies"],
                            q_gain=t["q_gain"], k_gain=t["k_gain"], key_scales=t["key_scales"], value_scales=t["value_scales"],
                            out=t["out"])


def attend(t):
    return ops.cache_attention(t["q"], t["keys"], t["values"], torch.zeros(1, dtype=torch.int64), key_scales=t["key_scales"],
                               value_scales=t["value_scales"], out=t["out"])


def unpack(t):
    return ops.unpack_cache(t["keys"], t["values"], key_scales=t["key_scales"], value_scales=t["value_scales"])


def window(t):
    return ops.window_attention(t["q"], t["k"], t["v"], window=2, out=t["out"])


# every floating-point tensor of every call, with a cache of 16-bit or of 4-bit rows
DERIVATIVES = [(append, four, name) for four in (False, True) for name in ("q", "k", "v", "frequencies", "q_gain", "k_gain", "out")]
DERIVATIVES += [(append, False, "keys"), (append, False, "values"), (append, True, "key_scales"), (append, True, "value_scales")]
DERIVATIVES += [(attend, False, name) for name in ("q", "keys", "values", "out")]
DERIVATIVES += [(attend, True, name) for name in ("q", "key_scales", "value_scales", "out")]
DERIVATIVES += [(unpack, True, "key_scales"), (unpack, True, "value_scales")]
DERIVATIVES += [(window, False, name) for name in ("q", "k", "v", "out")]


@pytest.mark.parametrize("call,four,name", DERIVATIVES, ids=lambda v: v.__name__ if callable(v) else str(v))
def test_a_derivative_is_never_dropped(call, four, name):
    t = append_arguments(four)
    t[name].requires_grad_()
    with pytest.raises(StreamError, match="no backward pass"):
        call(t)
    with torch.no_grad(), pytest.raises(StreamError, match="expected a CUDA tensor"):   # past the gradients' check
        call(t)


@pytest.mark.parametrize("call,four,name", DERIVATIVES, ids=lambda v: v.__name__ if callable(v) else str(v))
def test_a_tangent_is_never_dropped(call, four, name):
    t = append_arguments(four)
    with torch.autograd.forward_ad.dual_level(), torch.no_grad():
        t[name] = torch.autograd.forward_ad.make_dual(t[name], torch.ones_like(t[name]))
        with pytest.raises(StreamError, match="no forward-mode derivative"):
            call(t)
    with pytest.raises(StreamError, match="expected a CUDA tensor"):
        call(append_arguments(four))


@pytest.mark.parametrize("name,by", [("positions", 4), ("positions", 1), ("starts", 2), ("frequencies", 4)])
@pytest.mark.parametrize("four", [False, True])
def test_misaligned_values_of_an_append_are_refused(name, by, four):
    # a kernel's load from such an address would fault
    change = {"starts": P, name: P + by}
    refused(entry_points().st_cache_append(cache(**(FOUR if four else {})), append_struct(**change), None), f"{name} must be on a boundary")


def test_misaligned_positions_and_starts_are_refused():
    lib = entry_points()
    for by in (1, 4):
        refused(lib.st_cache_attention(cache(), attend_struct(positions=P + by), None), "positions must be on a boundary")
    for by in (1, 2, 3):
        refused(lib.st_window_attention(window_struct(starts=P + by), None), "starts must be on a boundary")
    # frequencies that no pair uses are not read: what is refused here is the gain
    refused(lib.st_cache_append(cache(), append_struct(rotary=0, frequencies=P + 1, q_gain=P + 4), None), "gains")


def test_sinks_of_any_integer_type():
    import numpy as np
    t = append_arguments(False)
    positions = torch.zeros(1, dtype=torch.int64)

    def call(sinks):
        return ops.cache_append(t["q"], t["k"], t["v"], t["keys"], t["values"], positions, t["frequencies"], sinks=sinks)

    for sinks in (2, np.int64(2), np.int32(0), torch.tensor(1)):
        with pytest.raises(StreamError, match="expected a CUDA tensor"):     # past the integers' check
            call(sinks)
    for sinks in (1.0, np.float32(1), "1", None, torch.tensor(1.0)):
        with pytest.raises(StreamError, match="sinks: expected an integer"):
            call(sinks)
    for sinks in (-1, 2 ** 70, np.int64(-3)):
        with pytest.raises(StreamError, match="sinks.*out of range"):
            call(sinks)


@pytest.mark.parametrize("name", ["q", "k", "v"])
@pytest.mark.parametrize("mode", [1, 2])
def test_strides_that_no_tensor_map_takes_are_refused(name, mode):
    heads = 4 if name == "q" else 2
    for strides in ((2 ** 39, 64), (heads * 64, 2 ** 39)):
        refused(entry_points().st_window_attention(window_struct(mode=mode, **{name: Rows(P, *strides)}), None), f"{name}: strides of 16-bit")
    # along a dimension of one element a stride is never used: what is refused here is the next input
    one = window_struct(mode=mode, heads=1, kv_heads=1, q=Rows(P, 64, 2 ** 40), k=rows(1), v=Rows(P, 2 ** 39, 64))
    refused(entry_points().st_window_attention(one, None), "v: strides of 16-bit")
