"""Decode in half precision over the K/V pool in 4 bits where half's own range ends: block bytes that no writer left, values and weights
that half rounds or does not reach."""
import math

import pytest
import torch

from _mxfp4_util import assert_within, indptr, pool, rows, tolerance
from oracle import mxfp4_oracle as mx

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def _decode(gpu, q, codes, scales, ip, idx, scale):
    from mini_sglang_amd_kernel import paged_decode_attention_mxfp4

    return paged_decode_attention_mxfp4(q.to(gpu), codes.to(gpu), scales.to(gpu), ip.to(gpu), idx.to(gpu), scale).cpu()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [128, 256])
def test_slots_that_nobody_stored(gpu, d, dtype):
    """Zeros, as the cache gives them out: alone, beside keys that were stored, and where an id outside the pool lands."""
    from mini_sglang_amd.kvcache import MXFP4KVCache

    cache = MXFP4KVCache(num_kv_heads=2, num_layers=1, head_dim=d, num_pages=300, dtype=dtype, device=gpu)
    stored = torch.arange(1, 200, 2, dtype=torch.int32)
    cache.store_kv(rows(100, 2, d, 1, dtype).to(gpu), rows(100, 2, d, 2, dtype).to(gpu), stored.to(gpu), 0)
    zeros = [0, 2, 250]
    ids = [zeros, list(range(200)), [7, 9, 298, 301, -1, 2 ** 31 - 1], [300], list(range(200, 300)) * 40]
    ip, idx = indptr([len(x) for x in ids]), torch.tensor([i for x in ids for i in x], dtype=torch.int32)
    q = rows(len(ids), 8, d, 3, dtype)
    codes, scales = cache.codes(0).cpu(), cache.scales(0).cpu()
    got = _decode(gpu, q, codes, scales, ip, idx, d ** -0.5)
    inside = torch.where((idx < 0) | (idx > 299), torch.full_like(idx, 299), idx)
    out, spread, score = mx.attention(q, codes, scales, None, ip, inside, None, d ** -0.5)
    assert (got[[0, 3, 4]] == 0).all() and (out[[0, 3, 4]] == 0).all()
    assert_within(got, out, spread, tolerance(spread, score, out, d, dtype))


def _bound(spread, score, out, d, largest, n=0):
    """As `tolerance` of half, with what half's range costs as it is: a weight is off by 2^-11 of itself or 2^-38 of the largest (`largest`: of
    the values that meet them, for `n` keys), a value by 2^-24, half of the step of V at half its size, and the result by half a step of its own, 2^-25 at the least."""
    half_step = 2.0 ** -11
    return (half_step * (1 + 2.0 ** -6) * (spread + out.abs()) + (half_step * out.abs()).clamp_min(2.0 ** -25) * (1 + half_step * 4) + n * 2.0 ** -37 * largest
            + 2.0 ** -24 + spread * (2 * (d + 2) * 2.0 ** -24 * score[..., None] + 2.0 ** -18))


@pytest.mark.parametrize("batch", [1, 600])
@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("n,above", [(2, 18), (33, 18), (700, 18), (2, 23), (700, 23)])
def test_weights_beside_one_that_is_far_larger(gpu, n, above, d, batch):
    """A key this much above the others in the exponent, whose V is zero: what is left is all of the others'.  600 requests, whose keys nobody cuts, and one."""
    k, v = torch.zeros(n, 2, d, dtype=F16), rows(n, 2, d, 1, F16, 2.0 ** 13)
    k[n // 2], v[n // 2] = 2.0, 0.0
    codes, scales = mx.quantised(k, v)
    q, idx, scale = torch.ones(1, 8, d, dtype=F16), torch.arange(n, dtype=torch.int32), above / (2 * d)
    out, spread, score = mx.attention(q, codes, scales, None, indptr([n]), idx, None, scale)
    assert float(score.max()) == above and float(out.abs().max()) > 2.0 ** -20
    got = _decode(gpu, q.expand(batch, 8, d), codes, scales, indptr([n] * batch), idx.repeat(batch), scale)
    assert torch.equal(got, got[:1].expand(batch, 8, d))
    assert_within(got[:1], out, spread, _bound(spread, score, out, d, float(v.abs().max()) * 4 / 3, n))


@pytest.mark.parametrize("d", [128, 256])
def test_the_lower_end_of_half(gpu, d):
    """Half has K and V at half their size: exact where a block's unit is 2^-22 or more, else off by 2^-24 at most."""
    q, idx, ip = rows(3, 8, d, 3, F16, 16.0), torch.arange(200, dtype=torch.int32), indptr([1, 99, 100])
    q_sum = q.double().abs().sum(-1)[..., None]
    for k_scale, v_scale in ((2.0 ** -12, 2.0 ** -12), (2.0 ** -19, 2.0 ** -19), (2.0 ** -22, 2.0 ** -22), (1.0, 2.0 ** -24)):
        codes, scales = mx.quantised(rows(200, 2, d, 1, F16, k_scale), rows(200, 2, d, 2, F16, v_scale))
        sm_scale = d ** -0.5 / 16 / k_scale
        k_off = sm_scale * q_sum * 2.0 ** -24 * float((scales[:, :, 0] < 127 - 22).any())
        out, spread, score = mx.attention(q, codes, scales, None, ip, idx, None, sm_scale)
        bound = _bound(spread, score, out, d, v_scale * 8, 200) + 2 * spread * torch.expm1(k_off)
        assert_within(_decode(gpu, q, codes, scales, ip, idx, sm_scale), out, spread, bound, f"{k_scale} {v_scale}")
