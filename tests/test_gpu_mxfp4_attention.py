"""Attention over the K/V pool in 4 bits against the definition in 64 bits, entry by entry within a bound on the roundings."""
import math

import pytest
import torch

from _mxfp4_util import assert_within, indptr, listed, pool, rows, tolerance
from oracle import mxfp4_oracle as mx

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def _decode(gpu, lens, n_q, n_kv, d, dtype=BF16, seed=1, start=0, num_slots=None, scale=None, **kw):
    from mini_sglang_amd_kernel import paged_decode_attention_mxfp4

    num_slots = num_slots or sum(lens) + 9
    codes, scales = pool(num_slots, n_kv, d, seed, dtype)
    idx = torch.cat([torch.full((start,), num_slots - 1, dtype=torch.int32), listed(lens, num_slots, seed)])
    q, ip, scale = rows(len(lens), n_q, d, seed + 1, dtype), indptr(lens, start), scale or d ** -0.5
    got = paged_decode_attention_mxfp4(q.to(gpu), codes.to(gpu), scales.to(gpu), ip.to(gpu), idx.to(gpu), scale, **kw)
    out, spread, score = mx.attention(q, codes, scales, None, ip, idx, None, scale)
    assert got.dtype is dtype and got.shape == q.shape
    assert_within(got, out, spread, tolerance(spread, score, out, d, dtype), f"{lens} {n_q}/{n_kv} x {d}")
    return got


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n_q,n_kv,d", [(1, 1, 128), (4, 1, 128), (32, 8, 128), (16, 8, 128), (15, 3, 128), (32, 2, 128), (6, 6, 256), (16, 2, 256),
                                        (24, 4, 256), (10, 5, 256)])
def test_decode(gpu, n_q, n_kv, d, dtype):
    _decode(gpu, [1, 2, 31, 32, 33, 63, 64, 65, 0, 100, 127, 128, 129, 500], n_q, n_kv, d, dtype)


@pytest.mark.parametrize("lens", [[1], [0], [0, 0, 0], [0, 1, 0, 1, 0], [3000], [1, 2047, 1], [17] * 200, [5000] + [1] * 70, [0] * 65 + [777]])
def test_decode_lengths(gpu, lens):
    _decode(gpu, lens, 8, 4, 128)


def test_decode_list_that_does_not_begin_at_zero(gpu):
    _decode(gpu, [40, 3, 200], 8, 2, 128, start=13)


def test_decode_large_scores(gpu):
    """Weights that are one key's alone, and a scale that is negative."""
    _decode(gpu, [70, 300, 1], 8, 2, 128, scale=4.0)
    _decode(gpu, [70, 300, 1], 8, 2, 128, scale=-0.3)


def test_decode_slots_that_requests_share(gpu):
    from mini_sglang_amd_kernel import paged_decode_attention_mxfp4

    codes, scales = pool(40, 2, 128, 3)
    idx = torch.tensor(list(range(30)) + list(range(30)) + [7] * 50, dtype=torch.int32)
    q, ip = rows(3, 8, 128, 4), indptr([30, 30, 50])
    q[1] = q[0]
    got = paged_decode_attention_mxfp4(q.to(gpu), codes.to(gpu), scales.to(gpu), ip.to(gpu), idx.to(gpu), 0.1)
    out, spread, score = mx.attention(q, codes, scales, None, ip, idx, None, 0.1)
    assert_within(got, out, spread, tolerance(spread, score, out, 128))
    assert_within(got[2:], mx.values(codes[7:8], scales[7:8])[:, :, 1].repeat_interleave(4, 1), spread[2:], tolerance(spread, score, out, 128)[2:])


def test_decode_pool_beyond_32_bits(gpu):
    """Slots whose bytes lie more than 4 GiB into the pool, which is wide and holds only those."""
    from mini_sglang_amd_kernel import paged_decode_attention_mxfp4, store_kv_cache_mxfp4

    n_kv, d, num_slots, stride = 2, 128, 5000, 1 << 20
    big = torch.empty(num_slots * stride, dtype=torch.uint8, device=gpu)
    codes = big.as_strided((num_slots, n_kv, 2, d // 2), (stride, d, d // 2, 1))
    scales = big.as_strided((num_slots, n_kv, 2, d // 32), (stride, d // 16, d // 32, 1), 4096)
    k, v = rows(300, n_kv, d, 1), rows(300, n_kv, d, 2)
    loc = torch.arange(4999, 4699, -1, dtype=torch.int32)
    store_kv_cache_mxfp4(codes, scales, loc.to(gpu), k.to(gpu), v.to(gpu))
    small_codes, small_scales = mx.quantised(k, v)
    q, ip = rows(2, 8, d, 3), indptr([100, 200])
    got = paged_decode_attention_mxfp4(q.to(gpu), codes, scales, ip.to(gpu), loc.to(gpu), d ** -0.5)
    out, spread, score = mx.attention(q, small_codes, small_scales, None, ip, torch.arange(300), None, d ** -0.5)
    assert_within(got, out, spread, tolerance(spread, score, out, d))


def test_decode_half_at_its_largest_values(gpu):
    """65504 in K and V of a float16 pool: the nearest value is 65536, which half itself has not."""
    from mini_sglang_amd_kernel import paged_decode_attention_mxfp4

    k = torch.full((3, 1, 128), 65504.0, dtype=F16)
    v = torch.full((3, 1, 128), 50000.0, dtype=F16)
    codes, scales = mx.quantised(k, v)
    q = torch.full((1, 4, 128), 2.0 ** -10, dtype=F16)
    idx, ip = torch.arange(3, dtype=torch.int32), indptr([3])
    got = paged_decode_attention_mxfp4(q.to(gpu), codes.to(gpu), scales.to(gpu), ip.to(gpu), idx.to(gpu), 1e-4)
    assert torch.equal(got.cpu(), torch.full_like(got.cpu(), 49152.0))


def test_decode_keys_that_are_not_finite(gpu):
    """A request that lists such a key has NaN in that head's rows, the others are as they were."""
    from mini_sglang_amd_kernel import paged_decode_attention_mxfp4

    for n, d, dtype in ((40, 128, BF16), (1, 128, BF16), (5000, 128, BF16), (40, 256, F16)):
        k, v = rows(2 * n, 4, d, 1, dtype), rows(2 * n, 4, d, 2, dtype)
        v[n // 2, 2, 5] = math.inf
        codes, scales = mx.quantised(k, v)
        q, ip, idx = rows(2, 8, d, 3, dtype), indptr([n, n]), torch.arange(2 * n, dtype=torch.int32)
        got = paged_decode_attention_mxfp4(q.to(gpu), codes.to(gpu), scales.to(gpu), ip.to(gpu), idx.to(gpu), d ** -0.5).cpu()
        bad = torch.isnan(got).all(-1)
        assert bad.tolist() == [[False] * 4 + [True] * 2 + [False] * 2, [False] * 8]
        assert torch.isfinite(got[~bad]).all()


# queries that a launch over the codes themselves takes (up to 64 columns of 128 dims, 32 of 256), and longer ones
SHORT = [(8, 2, 128, [1, 4, 3, 0, 2]), (32, 8, 128, [8, 8, 5]), (64, 1, 128, [1, 1]), (6, 2, 128, [11, 21, 1]), (8, 8, 256, [16, 1, 7]), (24, 4, 256, [5, 2]),
         (16, 2, 256, [2, 1, 4])]
LONG = [(32, 8, 128, [17, 300, 64, 0, 1]), (4, 4, 128, [65, 200]), (24, 4, 256, [6, 130, 33]), (16, 2, 256, [40, 0, 9]), (8, 1, 128, [513])]


def _extend(gpu, n_q, n_kv, d, new, cached, is_cross, window, seed=1, most=None, cut=None):
    from mini_sglang_amd_kernel import paged_prefill_attention_mxfp4

    lens = [c + e for c, e in zip(cached, new)]
    num_slots = sum(lens) + 11
    codes, scales = pool(num_slots, n_kv, d, seed)
    idx, q = listed(lens, num_slots, seed), rows(sum(new), n_q, d, seed + 1)
    qo, ip, prefix = indptr(new), indptr(lens), torch.tensor(cached, dtype=torch.int32)
    most = most or max(new)
    got = paged_prefill_attention_mxfp4(q.to(gpu), codes.to(gpu), scales.to(gpu), qo.to(gpu), ip.to(gpu), idx.to(gpu), prefix.to(gpu), d ** -0.5,
                                        most, is_cross_attention=is_cross, sliding_window_size=window)
    out, spread, score = mx.attention(q, codes, scales, qo, ip, idx, prefix, d ** -0.5, max_len_extend=most, is_cross=is_cross, window=window)
    cut = n_q // n_kv * most > (64 if d == 128 else 32)
    assert_within(got, out, spread, tolerance(spread, score, out, d, cut=cut), f"{n_q}/{n_kv} x {d}, {new} on {cached}")
    return got


@pytest.mark.parametrize("is_cross,window", [(False, 0), (True, 0), (False, 1), (False, 50), (True, 50)])
@pytest.mark.parametrize("n_q,n_kv,d,new", SHORT + LONG)
def test_extend(gpu, n_q, n_kv, d, new, is_cross, window):
    cached = [(37 * i * i + 90) % 301 for i in range(len(new))]
    _extend(gpu, n_q, n_kv, d, new, cached, is_cross, window)


@pytest.mark.parametrize("n_q,n_kv,d,new", SHORT + LONG)
def test_extend_of_prompts_and_of_long_prefixes(gpu, n_q, n_kv, d, new):
    _extend(gpu, n_q, n_kv, d, new, [0] * len(new), False, 0)
    _extend(gpu, n_q, n_kv, d, new, [2500] + [1] * (len(new) - 1), False, 700)


def test_extend_rows_beyond_the_longest_are_left(gpu):
    """max_len_extend below a request's rows: the first are computed."""
    for most in (2, 40):
        _extend(gpu, 8, 2, 128, [5, 60, 1], [10, 0, 70], False, 0, most=most)


def _prefixes(gpu, prefix, new, lens, is_cross=False, window=0, n_q=8, n_kv=2, d=128):
    """Requests whose first query is not where their keys end less their rows."""
    from mini_sglang_amd_kernel import paged_prefill_attention_mxfp4

    codes, scales = pool(sum(lens) + 3, n_kv, d, 2)
    idx, q = listed(lens, sum(lens) + 3, 5), rows(sum(new), n_q, d, 6)
    qo, ip, pl = indptr(new), indptr(lens), torch.tensor(prefix, dtype=torch.int32)
    got = paged_prefill_attention_mxfp4(q.to(gpu), codes.to(gpu), scales.to(gpu), qo.to(gpu), ip.to(gpu), idx.to(gpu), pl.to(gpu), d ** -0.5,
                                        max(new), is_cross_attention=is_cross, sliding_window_size=window)
    out, spread, score = mx.attention(q, codes, scales, qo, ip, idx, pl, d ** -0.5, is_cross=is_cross, window=window)
    assert_within(got, out, spread, tolerance(spread, score, out, d, cut=n_q // n_kv * max(new) > 64))


@pytest.mark.parametrize("new", [[3, 7, 16], [100, 3, 40]])
@pytest.mark.parametrize("window", [0, 20])
def test_extend_masks_that_leave_rows_empty(gpu, new, window):
    _prefixes(gpu, [-5, 0, 400], new, [90, 0, 120], window=window)  # before the first key, no key, behind the window of the last
    _prefixes(gpu, [10, 30, 64], new, [900, 200, 500], window=window)  # keys behind every query


@pytest.mark.parametrize("new,d", [([4, 4], 128), ([80, 90], 128), ([70, 66], 256), ([4, 4], 256)])
def test_extend_hidden_keys_that_are_not_finite(gpu, new, d):
    """Queries before such a key, or past it by the window, do not see it; whoever does has NaN."""
    from mini_sglang_amd_kernel import paged_prefill_attention_mxfp4

    n_q, n_kv, cached, window = 8, 2, 130, 60
    lens = [cached + e for e in new]
    for of_v in (False, True):
        for at in (cached + 2, 100):
            k, v = rows(sum(lens), n_kv, d, 1), rows(sum(lens), n_kv, d, 2)
            (v if of_v else k)[at, 1, 9] = math.nan
            codes, scales = mx.quantised(k, v)
            q, qo, ip = rows(sum(new), n_q, d, 3), indptr(new), indptr(lens)
            idx, prefix = torch.arange(sum(lens), dtype=torch.int32), torch.full((2,), cached, dtype=torch.int32)
            got = paged_prefill_attention_mxfp4(q.to(gpu), codes.to(gpu), scales.to(gpu), qo.to(gpu), ip.to(gpu), idx.to(gpu), prefix.to(gpu),
                                                d ** -0.5, max(new), sliding_window_size=window).cpu()
            position = cached + torch.arange(new[0])
            sees = torch.zeros(sum(new), n_q, dtype=torch.bool)
            sees[:new[0], n_q // 2:] = ((position >= at) & (at > position - window))[:, None]
            assert torch.equal(torch.isnan(got).all(-1), sees) and torch.isfinite(got[~sees]).all()
            clean_codes, clean_scales = mx.quantised(k.nan_to_num(0.0), v.nan_to_num(0.0))
            out, spread, score = mx.attention(q, clean_codes, clean_scales, qo, ip, idx, prefix, d ** -0.5, window=window)
            tol = tolerance(spread, score, out, d, cut=new[0] > 20)
            assert bool(((got.double() - out).abs() <= tol)[~sees].all())


def test_chunks_see_what_the_whole_prompt_sees(gpu):
    """A prompt in one call, in chunks, and its last token as a decode step: the same keys from the pool, so the same rows within their bounds."""
    from mini_sglang_amd_kernel import paged_decode_attention_mxfp4, paged_prefill_attention_mxfp4

    n, n_q, n_kv, d = 400, 8, 2, 128
    codes, scales = (t.to(gpu) for t in pool(n, n_kv, d, 1))
    idx, q = listed([n], n, 2).to(gpu), rows(n, n_q, d, 3).to(gpu)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    whole = paged_prefill_attention_mxfp4(q, codes, scales, i32(0, n), i32(0, n), idx, i32(0), d ** -0.5, n)
    out, spread, score = mx.attention(q.cpu(), codes.cpu(), scales.cpu(), indptr([n]), indptr([n]), idx.cpu(), torch.zeros(1), d ** -0.5)
    tol = tolerance(spread, score, out, d, cut=True)
    assert_within(whole, out, spread, tol)
    at = 0
    for e in (250, 140, 9, 1):
        part = paged_prefill_attention_mxfp4(q[at:at + e], codes, scales, i32(0, e), i32(0, at + e), idx[:at + e], i32(at), d ** -0.5, e)
        assert_within(part, out[at:at + e], spread[at:at + e], tol[at:at + e])
        at += e
    last = paged_decode_attention_mxfp4(q[-1:], codes, scales, i32(0, n), idx, d ** -0.5)
    assert_within(last, out[-1:], spread[-1:], tol[-1:])


def test_same_bits_every_time(gpu):
    a = _decode(gpu, [900, 40, 2000], 8, 4, 128)
    for _ in range(3):
        assert torch.equal(a, _decode(gpu, [900, 40, 2000], 8, 4, 128))


# launches whose requests are cut in every way: one head, two, four or eight to a workgroup, more requests than workgroups, more than stay in registers, one
# request alone with as many shares as there are, partials of more shares than one trip of the merge takes
CUTS = [([2000] * 40 + [37, 0, 4000] * 8, 32, 8, 128), ([300, 1, 900] * 90, 8, 8, 128), ([10] * 260 + [3000, 0, 0, 700], 8, 2, 128), ([0] * 300 + [5], 4, 1, 128), ([3, 0, 1, 40] * 300 + [2000, 0], 2, 2, 128), ([0] * 500 + [90, 1] * 200 + [0, 70], 4, 4, 256),
        ([30000], 32, 8, 128), ([20000, 1], 4, 1, 128), ([9000, 200, 4000, 1, 5000], 16, 16, 128), ([1500] * 12, 12, 4, 256), ([16000], 16, 2, 256),
        ([700 + 97 * i for i in range(30)], 10, 5, 256), ([1200 + 31 * i for i in range(66)], 16, 8, 128)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lens,n_q,n_kv,d", CUTS)
def test_decode_cuts(gpu, lens, n_q, n_kv, d, dtype):
    _decode(gpu, lens, n_q, n_kv, d, dtype)


# more columns than a workgroup's waves hold: up to three blocks of queries (eight at 256), the last of them short, and requests with nothing in the later ones
BLOCKS = [(64, 8, 128, [9, 16, 1, 0, 24]), (32, 8, 128, [48, 1]), (8, 1, 128, [24, 5, 9, 17]), (13, 13, 128, [130, 65, 64]), (16, 2, 256, [8, 3, 5, 1]),
          (64, 4, 256, [2, 16, 0]), (16, 2, 256, [32, 17, 1]), (4, 4, 256, [33, 200, 64]), (64, 1, 128, [1, 3, 2]), (32, 1, 256, [8, 1])]


@pytest.mark.parametrize("is_cross,window", [(False, 0), (True, 0), (False, 1), (False, 50), (True, 50)])
@pytest.mark.parametrize("n_q,n_kv,d,new", BLOCKS)
def test_extend_blocks_of_queries(gpu, n_q, n_kv, d, new, is_cross, window):
    from mini_sglang_amd_kernel import paged_prefill_attention_mxfp4

    cached = [(377 * i * i + 900) % 1601 for i in range(len(new))]
    lens = [c + e for c, e in zip(cached, new)]
    codes, scales = pool(sum(lens) + 1, n_kv, d, 3)
    idx, q = listed(lens, sum(lens) + 1, 4), rows(sum(new), n_q, d, 5)
    qo, ip, prefix = indptr(new), indptr(lens), torch.tensor(cached, dtype=torch.int32)
    got = paged_prefill_attention_mxfp4(q.to(gpu), codes.to(gpu), scales.to(gpu), qo.to(gpu), ip.to(gpu), idx.to(gpu), prefix.to(gpu), d ** -0.5,
                                        max(new), is_cross_attention=is_cross, sliding_window_size=window)
    out, spread, score = mx.attention(q, codes, scales, qo, ip, idx, prefix, d ** -0.5, is_cross=is_cross, window=window)
    assert_within(got, out, spread, tolerance(spread, score, out, d), f"{n_q}/{n_kv} x {d}, {new} on {cached}")


def test_extend_long_prefixes_of_many_shares(gpu):
    """Partials of wide launches: 64 columns and 32 of 256, four, eight and more shares to a request."""
    for n_q, n_kv, d, new, cached in ((32, 8, 128, [16, 2], [9000, 300]), (32, 8, 128, [8] * 5, [5000, 1, 900, 2500, 30]), (16, 2, 256, [4], [20000]),
                                      (16, 2, 256, [8, 8], [6000, 7000]), (64, 8, 128, [3] * 40, [500 + 60 * i for i in range(40)])):
        _extend(gpu, n_q, n_kv, d, new, cached, False, 0)


def test_scale_of_zero(gpu):
    """The mean of the visible values, infinite scores or none."""
    from mini_sglang_amd_kernel import paged_decode_attention_mxfp4, paged_prefill_attention_mxfp4

    lens, n_q, n_kv, d = [40, 0, 900, 1], 8, 2, 128
    codes, scales = pool(sum(lens), n_kv, d, 1)
    idx, ip, q = listed(lens, sum(lens), 2), indptr(lens), rows(4, n_q, d, 3)
    q[0] = math.inf
    got = paged_decode_attention_mxfp4(q.to(gpu), codes.to(gpu), scales.to(gpu), ip.to(gpu), idx.to(gpu), 0.0)
    out, spread, score = mx.attention(torch.zeros_like(q), codes, scales, None, ip, idx, None, 1.0)
    assert_within(got, out, spread, tolerance(spread, score, out, d))
    qo, prefix = indptr([1, 0, 2, 1]), torch.tensor([39, 0, 898, 0], dtype=torch.int32)
    got = paged_prefill_attention_mxfp4(q.to(gpu), codes.to(gpu), scales.to(gpu), qo.to(gpu), ip.to(gpu), idx.to(gpu), prefix.to(gpu), 0.0, 2)
    out, spread, score = mx.attention(torch.zeros_like(q), codes, scales, qo, ip, idx, prefix, 1.0)
    assert_within(got, out, spread, tolerance(spread, score, out, d))


@pytest.mark.parametrize("byte", [0x00, 0xff, 0x7f, 0x01])
def test_whatever_a_workspace_held(gpu, byte):
    """Memory that the allocator hands out again is full of something: counts and partials of an earlier life."""
    for lens, n_q, n_kv in (([3000, 40, 900], 16, 8), ([700] * 66, 8, 8)):
        want = _decode(gpu, lens, n_q, n_kv, 128)
        torch.cuda.synchronize()
        for size in (1 << 16, 1 << 20, 1 << 21, 1 << 22, 1 << 23, 1 << 24, 1 << 25):
            junk = [torch.full((size,), byte, dtype=torch.uint8, device=gpu) for _ in range(3)]
            del junk
        assert torch.equal(want, _decode(gpu, lens, n_q, n_kv, 128))
