"""Output buffers of KV8Store's attention without a GPU: what reaches the C entry (none of it runs)."""
import pytest
import torch

D = 128


class Reached(Exception):
    pass


def _store(batch, kv_heads):
    """A store whose calls end where the library's would begin."""
    from leankv_amd.kv8 import KV8Store

    store = KV8Store.__new__(KV8Store)
    store.batch, store.kv_heads, store.blocks, store.device = batch, kv_heads, 4, torch.device("cpu")
    store._queries = lambda q, dims, what: (q.shape[1], 1)
    store._ints = lambda t, what, name: 0
    store._workspace = lambda nbytes: None

    def call(name, *args):
        raise Reached([tuple(a) for a in args if hasattr(a, "_length_")])

    store._call = call
    return store


def _decode(out):
    B, H, _ = out.shape
    return _store(B, 1).decode_attention(torch.zeros(B, H, D, dtype=out.dtype), None, out=out)


def _prefill(out):
    B, H, S, _ = out.shape
    return _store(B, 1).prefill_attention(torch.zeros(B, H, S, D, dtype=out.dtype), None, out=out)


def _strided(shape, strides, dtype=torch.float16):
    n = 1 + sum((s - 1) * st for s, st in zip(shape, strides))
    return torch.zeros(n + 64, dtype=dtype).as_strided(shape, strides)


@pytest.mark.parametrize("shape,strides", [
    ((3, 4, D), (0, D, 1)), ((3, 4, D), (4 * D, 0, 1)),
    ((2, 4, D), (2 * D, D, 1)),                 # the second sequence over the first one's last heads
    ((2, 4, D), (4 * D, 64, 1)),                # rows half over each other
    ((3, 1, D), (120, 1000, 1)),
    ((1, 4, 5, D), (0, D, 0, 1)), ((2, 3, 5, D), (5 * D, D, D, 1)), ((1, 2, 7, D), (0, 256, 128, 1)),
    ((1, 3, 4, D), (0, 3 * D, 2 * D, 1))])      # rows 0 2 4 6, 3 5 7 9, 6 ...
def test_rows_over_each_other_are_refused(shape, strides):
    from leankv_amd._lib import LeanKVError

    with pytest.raises(LeanKVError, match="overlap"):
        (_decode if len(shape) == 3 else _prefill)(_strided(shape, strides))


@pytest.mark.parametrize("shape,strides", [
    ((2, 4, D), (4 * D, D, 1)), ((2, 4, D), (D, 2 * D, 1)), ((2, 4, D), (5 * D, D + 8, 1)), ((0, 4, D), (4 * D, D, 1)),
    ((2, 4, 3, D), (12 * D, D, 4 * D, 1)), ((2, 4, 3, D), (D, 6 * D, 2 * D, 1)),
    ((1, 3, 3, D), (0, 3 * D, 2 * D, 1))])      # rows 0 2 4, 3 5 7, 6 8 10: between each other, none twice
def test_rows_apart_are_taken(shape, strides):
    with pytest.raises(Reached):
        (_decode if len(shape) == 3 else _prefill)(_strided(shape, strides))


@pytest.mark.parametrize("shape,strides,passed", [
    ((1, 4, D), (1, D, 1), (0, D, 0)), ((3, 1, D), (2 * D, 3, 1), (2 * D, 0, 0)), ((1, 1, D), (7, 5, 1), (0, 0, 0)),
    ((1, 2, 1, D), (3, D, 5, 1), (0, D, 0))])
def test_strides_of_single_sizes_are_free(shape, strides, passed):
    with pytest.raises(Reached) as e:
        (_decode if len(shape) == 3 else _prefill)(_strided(shape, strides))
    assert e.value.args[0][-1] == passed
