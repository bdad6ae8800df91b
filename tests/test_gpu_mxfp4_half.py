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
