"""What a StreamCache knows on the host: the end of the rotary table and of the
lengths' type. On the CPU, where a call that is not refused ends at the device."""
import pytest
import torch

from dfsattn_amd.streaming import StreamCache

BF = torch.bfloat16


def _table(rows, dim=64):
    return torch.ones(rows, dim // 2), torch.zeros(rows, dim // 2)


def _attend(cache, tokens, rows=16):
    x = torch.zeros(1, tokens, 1, cache.k.shape[3], dtype=BF)
    cache.attend(x, x, x, table=None if rows is None else _table(rows, cache.k.shape[3]))


def _reaches_the_device(cache, tokens, rows=16):
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        _attend(cache, tokens, rows)


@pytest.mark.parametrize("inference", [False, True])
def test_a_stream_ends_with_its_rotary_table(inference):
    with torch.inference_mode(inference):
        cache = StreamCache(1, 1, 64, 8, 6, 2, "cpu", BF)
        _reaches_the_device(cache, 6)
        cache.advance(6)
        cache.advance(6)
        _reaches_the_device(cache, 4)  # positions 12 to 15 of 16
        with pytest.raises(ValueError, match="table"):
            _attend(cache, 5)
        _reaches_the_device(cache, 5, rows=None)
        cache.advance(4)
        with pytest.raises(ValueError, match="table"):
            _attend(cache, 1)
        cache.reset()
        _reaches_the_device(cache, 6)
        assert int(cache.lens) == 0


def test_lengths_set_by_hand_are_not_second_guessed():
    """A caller who moves lens without advance keeps the device's behaviour
    (rows past the table are NaN) until reset."""
    cache = StreamCache(1, 1, 64, 8, 6, 2, "cpu", BF)
    cache.advance(6)
    cache.advance(6)
    cache.lens.fill_(2)  # rewound
    _reaches_the_device(cache, 6)
    cache.advance(6)
    _reaches_the_device(cache, 6)
    cache.lens = torch.zeros(1, dtype=torch.int32)
    _reaches_the_device(cache, 6)
    cache.reset()
    cache.advance(6)
    cache.advance(6)
    with pytest.raises(ValueError, match="table"):
        _attend(cache, 5)


def test_a_stream_ends_with_its_lengths_type():
    cache = StreamCache(1, 1, 16, 0, 1 << 18, 0, "cpu", BF)
    for _ in range((1 << 13) - 1):
        cache.advance(1 << 18)
    _reaches_the_device(cache, (1 << 18) - 256, rows=None)
    with pytest.raises(ValueError, match="2\\^31"):
        _attend(cache, (1 << 18) - 255, rows=None)
