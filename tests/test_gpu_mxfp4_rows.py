"""Writers and reader of the K/V pool in 4 bits: what they leave, bit for bit, against the definition in 64 bits."""
import math

import pytest
import torch

from _mxfp4_util import rows
from oracle import mxfp4_oracle as mx

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def _empty(num_slots, n_kv, d, device, wide=0):
    """A pool of bytes that nobody stores; `wide`: slots this much further apart."""
    codes = torch.full((num_slots, n_kv * d + wide), 0xA5, dtype=torch.uint8, device=device)
    scales = torch.full((num_slots, n_kv * d // 16 + wide // 2), 0x5A, dtype=torch.uint8, device=device)
    return (codes[:, : n_kv * d].view(num_slots, n_kv, 2, d // 2), scales[:, : n_kv * d // 16].view(num_slots, n_kv, 2, d // 32))


def _store(k, v, d, device, num_slots=None, wide=0, loc=None, **kw):
    from mini_sglang_amd_kernel import store_kv_cache_mxfp4

    n, n_kv = k.shape[:2]
    num_slots = num_slots or n + 5
    codes, scales = _empty(num_slots, n_kv, d, device, wide)
    if loc is None:
        loc = torch.randperm(num_slots, generator=torch.Generator().manual_seed(n))[:n].to(torch.int32)
    store_kv_cache_mxfp4(codes, scales, loc.to(device), k.to(device), v.to(device), **kw)
    return codes, scales, loc


def _check(codes, scales, loc, k, v):
    want_codes, want_scales = mx.quantised(k, v)
    at = loc.long()
    assert torch.equal(scales.cpu()[at], want_scales)
    assert torch.equal(codes.cpu()[at], want_codes)
    rest = torch.ones(codes.shape[0], dtype=torch.bool)
    rest[at] = False
    assert (codes.cpu()[rest] == 0xA5).all() and (scales.cpu()[rest] == 0x5A).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,n_kv,d", [(1, 1, 128), (1, 3, 256), (7, 8, 128), (33, 2, 256), (257, 5, 128), (100, 4, 256)])
def test_store_is_the_definition(gpu, n, n_kv, d, dtype):
    k, v = rows(n, n_kv, d, n, dtype), rows(n, n_kv, d, n + 1, dtype, 30.0)
    codes, scales, loc = _store(k, v, d, gpu)
    _check(codes, scales, loc, k, v)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_store_of_every_value_of_the_type(gpu, dtype):
    """All 65536 bit patterns, in blocks with a size of their own each; heads that are not finite are marked."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    k = bits.view(-1, 2, 128)
    v = bits.flip(0).view(-1, 2, 128)
    codes, scales, loc = _store(k, v, 128, gpu)
    _check(codes, scales, loc, k, v)


def test_store_at_the_borders_of_codes(gpu):
    """Halfway between codes, and the bf16 values on both sides, under many factors."""
    border = mx.BORDERS.float()
    x = torch.cat([border, border * (1 + 2.0 ** -7), border * (1 - 2.0 ** -8), torch.tensor([6.0])])
    x = torch.cat([x, -x])[:32]
    x[-1] = 6.0
    blocks = torch.stack([torch.ldexp(x, torch.tensor(e)) for e in range(-120, 121, 8)])
    k = blocks.repeat_interleave(4, 0).view(-1, 1, 128).to(BF16)
    codes, scales, loc = _store(k, k.flip(0), 128, gpu)
    _check(codes, scales, loc, k, k.flip(0))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_store_of_rows_that_are_not_finite(gpu, bad):
    for d in (128, 256):
        k, v = rows(9, 3, d, 5), rows(9, 3, d, 6)
        k[2, 1, 0], v[4, 2, d - 1], k[7, 0, d // 2], v[7, 0, 3] = bad, bad, bad, bad
        codes, scales, loc = _store(k, v, d, gpu)
        _check(codes, scales, loc, k, v)


@pytest.mark.parametrize("d", [128, 256])
def test_store_of_strided_rows_into_strided_pools(gpu, d):
    qkv = rows(21, 8 + 2 * 3, d, 8)
    k, v = qkv[:, 8:11], qkv[:, 11:]
    codes, scales, loc = _store(k.to(gpu), v.to(gpu), d, gpu, wide=64)
    _check(codes, scales, loc, k, v)
    g = qkv.to(gpu)
    codes, scales, loc = _store(g[:, 8:11], g[:, 11:], d, gpu)  # the views themselves
    _check(codes, scales, loc, k, v)
    odd = torch.empty(21 * 3 * d + 1, dtype=BF16, device=gpu)[1:].view(21, 3, d).copy_(k)  # not at 16 bytes
    codes, scales, loc = _store(odd, v.to(gpu), d, gpu)
    _check(codes, scales, loc, k, v)


def test_slots_outside_the_pool_store_nothing(gpu):
    k, v = rows(6, 2, 128, 1), rows(6, 2, 128, 2)
    loc = torch.tensor([3, -1, 0, 10, 2 ** 31 - 1, 9], dtype=torch.int32)
    codes, scales, _ = _store(k, v, 128, gpu, num_slots=10, loc=loc)
    keep = torch.tensor([0, 2, 5])
    _check(codes, scales, loc[keep], k[keep], v[keep])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,n_kv,d", [(1, 1, 128), (5, 3, 256), (300, 8, 128)])
def test_load_gives_the_values(gpu, n, n_kv, d, dtype):
    from mini_sglang_amd_kernel import load_kv_cache_mxfp4

    k, v = rows(n, n_kv, d, n, dtype), rows(n, n_kv, d, n + 1, dtype)
    if n > 1:
        k[1, 0, 5] = math.nan
    codes, scales, loc = _store(k, v, d, gpu, wide=32)
    order = torch.cat([loc.flip(0), loc[:1]])  # any order, one twice
    got = load_kv_cache_mxfp4(codes, scales, order.to(gpu), dtype=dtype)
    want = mx.values(codes.cpu()[order.long()], scales.cpu()[order.long()])
    for g, i in zip(got, (0, 1)):
        assert g.dtype is dtype and torch.equal(g.double().cpu().nan_to_num(nan=9e9), want[:, :, i].nan_to_num(nan=9e9))


def test_nothing_to_store_and_nothing_to_load(gpu):
    from mini_sglang_amd_kernel import load_kv_cache_mxfp4, qk_norm_rope_store_mxfp4, store_kv_cache_mxfp4

    codes, scales = _empty(4, 2, 128, gpu)
    none = torch.empty(0, dtype=torch.int32, device=gpu)
    x = torch.empty(0, 2, 128, dtype=BF16, device=gpu)
    w = torch.ones(128, dtype=BF16, device=gpu)
    store_kv_cache_mxfp4(codes, scales, none, x, x)
    k, v = load_kv_cache_mxfp4(codes, scales, none)
    assert k.shape == v.shape == (0, 2, 128)
    assert qk_norm_rope_store_mxfp4(x, x, x, w, w, none, none, codes, scales, eps=1e-6, rope_base=1e6).shape == (0, 2, 128)
    assert (codes == 0xA5).all() and (scales == 0x5A).all()




@pytest.mark.parametrize("n,n_q,n_kv,d", [(1, 1, 1, 128), (3, 16, 8, 128), (130, 32, 8, 128), (40, 24, 4, 256), (9, 5, 5, 256), (700, 16, 2, 128)])
@pytest.mark.parametrize("far", [0, 131072, 2 ** 30])
def test_norm_rope_store(gpu, n, n_q, n_kv, d, far):
    from mini_sglang_amd_kernel import qk_norm_rope_store_mxfp4

    g = torch.Generator().manual_seed(n + d)
    qkv = torch.randn(n, n_q + 2 * n_kv, d, generator=g).to(BF16)
    q, k, v = qkv[:, :n_q], qkv[:, n_q:n_q + n_kv], qkv[:, n_q + n_kv:]
    qw, kw = ((1 + 0.2 * torch.randn(d, generator=g)).to(BF16) for _ in range(2))
    positions = (far + torch.arange(n)).to(torch.int32)
    loc = torch.randperm(n + 3, generator=g)[:n].to(torch.int32)
    codes, scales = _empty(n + 3, n_kv, d, gpu)
    dev = qkv.to(gpu)
    out = qk_norm_rope_store_mxfp4(dev[:, :n_q], dev[:, n_q:n_q + n_kv], dev[:, n_q + n_kv:], qw.to(gpu), kw.to(gpu), positions.to(gpu),
                                   loc.to(gpu), codes, scales, eps=1e-6, rope_base=1e6)
    # q: roundings of 32 bits (six, of |a| + |b|), the rounding to bf16, and angles of 2^30 radians held to 2^30 2^-53 of 64 bits twice
    want = mx.norm_rope(q, qw, positions, 1e-6, 1e6)
    half = d // 2
    pair = (want[..., :half].square() + want[..., half:].square()).sqrt().repeat(1, 1, 2)
    slack = pair * (12 * 2.0 ** -24 + max(far, 1) * 2.0 ** -50)
    over = (out.double().cpu() - want).abs() / (want.abs() * 2.0 ** -8 + slack * (1 + 2.0 ** -8))
    assert float(over.max()) <= 1
    # k: codes of a value that lies within the slack of the one of 64 bits
    rotated = mx.norm_rope(k, kw, positions, 1e-6, 1e6)
    pair = (rotated[..., :half].square() + rotated[..., half:].square()).sqrt().repeat(1, 1, 2)
    slack = pair * (12 * 2.0 ** -24 + max(far, 1) * 2.0 ** -50)
    got_codes, got_scales = codes.cpu()[loc.long()], scales.cpu()[loc.long()]
    want_codes, want_scales = mx.quantised(rotated, v.double())
    assert torch.equal(got_codes[:, :, 1], want_codes[:, :, 1]) and torch.equal(got_scales[:, :, 1], want_scales[:, :, 1])
    low, _ = mx.quantised(rotated.sign() * (rotated.abs() - slack), v.double())
    high, _ = mx.quantised(rotated.sign() * (rotated.abs() + slack), v.double())
    same_factor = (got_scales[:, :, 0] == want_scales[:, :, 0]).repeat_interleave(32, -1)
    unpack = lambda c: torch.stack((c & 15, c >> 4), -1).flatten(-2)[:, :, 0]  # noqa: E731
    ok = (unpack(got_codes) == unpack(low)) | (unpack(got_codes) == unpack(high)) | (unpack(got_codes) == unpack(want_codes))
    tiny = rotated.abs() <= slack  # its sign is anybody's
    assert bool((ok | ~same_factor | tiny).all())
    # a factor can only be another where the block's largest value is on its border
    amax = rotated.unflatten(-1, (-1, 32)).abs().amax(-1)
    mantissa = torch.frexp(amax / 6)[0]
    on_border = (mantissa - 0.5).abs().minimum((mantissa - 1).abs()) < 1e-6 + max(far, 1) * 2.0 ** -48
    assert bool(((got_scales[:, :, 0] == want_scales[:, :, 0]) | on_border).all())


def test_norm_rope_store_of_rows_that_are_not_finite(gpu):
    from mini_sglang_amd_kernel import qk_norm_rope_store_mxfp4

    for d in (128, 256):
        q, k, v = rows(6, 4, d, 1), rows(6, 2, d, 2), rows(6, 2, d, 3)
        k[1, 0, 4], v[3, 1, d - 1], k[5, 1, 1] = math.nan, math.inf, -math.inf
        w = torch.ones(d, dtype=BF16)
        pos = torch.arange(6, dtype=torch.int32)
        codes, scales = _empty(8, 2, d, gpu)
        qk_norm_rope_store_mxfp4(*(t.to(gpu) for t in (q, k, v, w, w, pos, pos + 1)), codes, scales, eps=1e-6, rope_base=1e4)
        s, c = scales.cpu()[1:7], codes.cpu()[1:7]
        bad = torch.zeros(6, 2, dtype=torch.bool)
        bad[1, 0] = bad[3, 1] = bad[5, 1] = True
        assert ((s[:, :, 0] == 255).all(-1) == bad).all() and (s[:, :, 1] != 255).all() and (c[bad] == 0).all()
        good = mx.quantised(v.nan_to_num(0, 0, 0), v.nan_to_num(0, 0, 0))
        assert torch.equal(c[:, :, 1][~bad], good[0][:, :, 1][~bad])
        assert (scales.cpu()[0] == 0x5A).all() and (scales.cpu()[7] == 0x5A).all()


def test_norm_rope_store_slot_outside_still_gives_q(gpu):
    from mini_sglang_amd_kernel import qk_norm_rope_store_mxfp4

    q, k, v = rows(3, 4, 128, 1), rows(3, 2, 128, 2), rows(3, 2, 128, 3)
    w, pos = torch.ones(128, dtype=BF16), torch.arange(3, dtype=torch.int32)
    outs = []
    for loc in ([0, 1, 2], [-1, 5, 2]):
        codes, scales = _empty(4, 2, 128, gpu)
        loc = torch.tensor(loc, dtype=torch.int32)
        outs.append(qk_norm_rope_store_mxfp4(*(t.to(gpu) for t in (q, k, v, w, w, pos, loc)), codes, scales, eps=0.0, rope_base=1e4).cpu())
        untouched = [i for i in range(4) if i not in loc.tolist()]
        assert (codes.cpu()[untouched] == 0xA5).all()
    assert torch.equal(outs[0], outs[1])
