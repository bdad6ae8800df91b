"""The oracle of the K/V pool in 4 bits against values worked out by hand."""
import math

import pytest
import torch

from oracle import mxfp4_oracle as mx


def _one(x):
    """Codes and the byte of one block of K (V is ones)."""
    k = torch.zeros(1, 1, 128, dtype=torch.float64)
    k[0, 0, : len(x)] = torch.tensor(x, dtype=torch.float64)
    codes, scales = mx.quantised(k, torch.ones_like(k))
    c = codes[0, 0, 0, :16]
    return torch.stack((c & 15, c >> 4), -1).flatten().tolist()[: len(x)], int(scales[0, 0, 0, 0])


def test_codes_are_nearest_and_halfway_goes_to_the_even_one():
    codes, byte = _one([6, 5, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25, 0.0, -0.5, -6, 5.01, 0.26])
    assert byte == 127
    assert codes == [7, 6, 6, 4, 4, 2, 2, 0, 0, 9, 15, 7, 1]


def test_the_factor_is_the_smallest_that_holds_the_block():
    assert _one([6.0])[1] == 127 and _one([6.0001])[1] == 128 and _one([3.0])[1] == 126 and _one([3.01])[1] == 127
    assert _one([0.0])[1] == 2 and _one([2.0 ** -140])[1] == 2 and _one([3.3e38])[1] == 252
    assert _one([3.3e38])[0] == [7]  # held at 6 * 2^125


def test_values_are_what_was_stored_and_never_beyond_half_a_step():
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(50, 2, 256, generator=g, dtype=torch.float64) for _ in range(2))
    codes, scales = mx.quantised(k, v)
    x = mx.values(codes, scales)
    factor = torch.ldexp(torch.ones((), dtype=torch.float64), scales.long() - 127).repeat_interleave(32, -1)
    y = torch.stack((k, v), 2)
    assert ((x - y).abs() <= factor).all()  # half the widest step, between 4 and 6
    again = mx.quantised(x[:, :, 0], x[:, :, 1])  # the factor may be smaller now, the values are the same
    assert torch.equal(mx.values(*again), x)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("of_v", [False, True])
def test_a_row_that_is_not_finite_marks_k(bad, of_v):
    k, v = torch.ones(2, 3, 128, dtype=torch.float64), torch.ones(2, 3, 128, dtype=torch.float64)
    (v if of_v else k)[1, 2, 77] = bad
    codes, scales = mx.quantised(k, v)
    assert (codes[1, 2] == 0).all() and (scales[1, 2, 0] == 255).all() and (scales[1, 2, 1] == 2).all()
    x = mx.values(codes, scales)
    assert torch.isnan(x[1, 2, 0]).all() and (x[1, 2, 1] == 0).all()
    assert torch.isfinite(x[0]).all() and torch.isfinite(x[1, :2]).all()


def test_attention_of_one_key_is_its_value_and_hidden_keys_do_not_count():
    codes, scales = mx.quantised(torch.ones(2, 1, 128, dtype=torch.float64), torch.full((2, 1, 128), 3.0, dtype=torch.float64))
    scales[1, :, 0] = 255
    ip = torch.tensor([0, 2], dtype=torch.int32)
    out, spread, _ = mx.attention(torch.ones(3, 2, 128), codes, scales, torch.tensor([0, 3]), ip, torch.tensor([0, 1]),
                                  torch.tensor([-1]), 0.1)
    assert (out[0] == 0).all() and (out[1] == 3).all() and torch.isnan(out[2]).all() and (spread[0] == 0).all()
