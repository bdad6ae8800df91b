"""The K/V pool in 4 bits on every route that sizes choose: attention in each form of a launch (waves and kv heads of a workgroup, tiles of columns, past the
caches, offsets of 64 bits), unpacking in several trips, workspaces that hold NaN, norm + rotary + store of many tokens."""
import pytest
import torch

import test_gpu_mxfp4_rows as rows_tests
from _mxfp4_util import assert_within, indptr, listed, pool, rows, tolerance
from mini_sglang_amd_kernel import _lib
from oracle import mxfp4_oracle as mx

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def _far_apart(codes, scales, gpu):
    """The same pool with slots so far apart that it ends beyond 4 GiB."""
    n, n_kv, _, half = codes.shape
    stride = -(-(9 << 29) // n) // 256 * 256
    big = torch.empty(n * stride, dtype=torch.uint8, device=gpu)
    c = big.as_strided(codes.shape, (stride, 2 * half, half, 1))
    s = big.as_strided(scales.shape, (stride, half // 8, half // 16, 1), n_kv * 2 * half)
    assert n * stride > 1 << 32 and stride > n_kv * (2 * half + half // 8)
    return c.copy_(codes), s.copy_(scales)


# requests of few keys and of many, 120 of them: with kv heads as here the plan takes, in this order, 1, 2, 4 and 8 heads to a workgroup for one tile of
# columns; 8 waves of 2, 4 and 8 heads for two; 2 heads for four, and 4 with three times as many requests; 2 and 4 of head_dim 256 for one and for two
FORMS = [(2, 1, 128, 1, 1), (4, 4, 128, 1, 1), (8, 8, 128, 1, 1), (16, 16, 128, 1, 1), (16, 4, 128, 5, 1), (32, 8, 128, 5, 1), (64, 16, 128, 5, 1),
         (64, 4, 128, 5, 1), (128, 8, 128, 4, 1), (64, 4, 128, 5, 3), (4, 4, 256, 1, 1), (8, 8, 256, 1, 1), (16, 2, 256, 5, 1), (32, 4, 256, 5, 1)]


@pytest.mark.parametrize("far_apart", [False, True])
@pytest.mark.parametrize("n_q,n_kv,d,new,times", FORMS)
def test_forms_of_a_launch(gpu, tuning, n_q, n_kv, d, new, times, far_apart):
    from mini_sglang_amd_kernel import paged_decode_attention_mxfp4, paged_prefill_attention_mxfp4

    lens = ([100, 64, 33, 130] * 6 + [new, 1200 + new, 7 + new, 257]) * (4 * times) + [90, 31, 32, 96] * 2
    new_lens = [min(new, n) for n in lens]
    num_slots = sum(lens) + 3
    codes, scales = pool(num_slots, n_kv, d, new + d)
    idx, ip, qo = listed(lens, num_slots, 2), indptr(lens), indptr(new_lens)
    prefix, scale = torch.tensor([n - e for n, e in zip(lens, new_lens)], dtype=torch.int32), d ** -0.5
    q = rows(sum(new_lens), n_q, d, 4)
    out, spread, score = mx.attention(q, codes, scales, qo, ip, idx, prefix, scale)
    pools = _far_apart(codes, scales, gpu) if far_apart else (codes.to(gpu), scales.to(gpu))
    dev = [t.to(gpu) for t in (q, qo, ip, idx, prefix)]
    for kib in (-1, 1):  # by way of the caches, and past them
        tuning(_lib.TUNE_STREAM, kib)
        print(f"{n_q}/{n_kv} x {d}, {new} queries, far apart {far_apart}, stream {kib}", flush=True)
        if new == 1:
            got = paged_decode_attention_mxfp4(dev[0], *pools, dev[2], dev[3], scale)
        else:
            got = paged_prefill_attention_mxfp4(dev[0], *pools, *dev[1:], scale, new)
        assert_within(got, out, spread, tolerance(spread, score, out, d), f"stream {kib}")


@pytest.mark.parametrize("far_apart", [False, True])
@pytest.mark.parametrize("n_q,n_kv,d", [(16, 8, 128), (16, 2, 256)])
def test_half_past_the_caches_and_far_apart(gpu, tuning, n_q, n_kv, d, far_apart):
    from mini_sglang_amd_kernel import paged_decode_attention_mxfp4

    lens = [1500, 1, 0, 300, 64]
    codes, scales = pool(sum(lens), n_kv, d, 3, F16)
    q, ip, idx = rows(5, n_q, d, 5, F16), indptr(lens), listed(lens, sum(lens), 1)
    out, spread, score = mx.attention(q, codes, scales, None, ip, idx, None, d ** -0.5)
    pools = _far_apart(codes, scales, gpu) if far_apart else (codes.to(gpu), scales.to(gpu))
    for kib in (-1, 1):
        tuning(_lib.TUNE_STREAM, kib)
        got = paged_decode_attention_mxfp4(q.to(gpu), *pools, ip.to(gpu), idx.to(gpu), d ** -0.5)
        assert_within(got, out, spread, tolerance(spread, score, out, d, F16))


# ---- unpacked rows --------------------------------------------------------------------------------------
def _attention64(gpu, q, codes, scales, new, lens, idx, cached, scale, is_cross, window):
    """``mx.attention`` of long query blocks, a request and kv head at a time on the GPU."""
    n_kv, group, d = codes.shape[1], q.shape[1] // codes.shape[1], q.shape[2]
    out, spread = (torch.zeros(q.shape, dtype=torch.float64, device=gpu) for _ in range(2))
    score = torch.zeros(q.shape[:2], dtype=torch.float64, device=gpu)
    at = key_at = 0
    for e, n, c in zip(new, lens, cached):
        slots = idx[key_at:key_at + n].long()
        position, j = c + torch.arange(e, device=gpu)[:, None, None], torch.arange(n, device=gpu)[None, None]
        hidden = torch.zeros(e, 1, n, dtype=torch.bool, device=gpu)
        if not is_cross:
            hidden = hidden | (j > position)
        if window:
            hidden = hidden | (j <= position - window)
        hidden = hidden.expand(e, group, n).reshape(e * group, n)
        for h in range(n_kv if e and n else 0):
            x = mx.values(codes[slots, h], scales[slots, h]).to(gpu)
            k, v = x[:, 0], x[:, 1]
            qr = q[at:at + e, h * group:(h + 1) * group].to(gpu).double().reshape(e * group, d)
            w = torch.softmax((qr @ k.T.contiguous() * scale).masked_fill(hidden, -torch.inf), -1).nan_to_num(0.0)  # rows that see nothing
            at_rows = (slice(at, at + e), slice(h * group, (h + 1) * group))
            out[at_rows] = (w @ v).view(e, group, d)
            spread[at_rows] = (w @ v.abs()).view(e, group, d)
            score[at_rows] = ((qr.abs() @ k.abs().T.contiguous()) * scale).masked_fill(hidden, 0.0).amax(-1).view(e, group)
        at, key_at = at + e, key_at + n
    return out.cpu(), spread.cpu(), score.cpu()


# more rows of heads than the unpacking has workgroups for at once: 4096 of 32 rows (16 at head_dim 256) in all, their part of a request's under a window
@pytest.mark.parametrize("n_q,n_kv,d,new,cached,is_cross,window", [
    (8, 8, 128, [200, 3, 64], [14000, 6000, 100], False, 0), (8, 8, 128, [200, 3, 64], [14000, 6000, 100], True, 3000),
    (16, 8, 128, [100, 7] * 8, [6000, 4000] * 8, False, 3500), (4, 4, 256, [260, 5, 64], [15000, 4000, 0], False, 0),
    (8, 4, 256, [130, 9] * 8, [4000, 5000] * 8, False, 3000), (4, 4, 256, [260, 5], [9000, 8000], True, 0)])
def test_unpacking_in_several_trips(gpu, n_q, n_kv, d, new, cached, is_cross, window):
    from mini_sglang_amd_kernel import paged_prefill_attention_mxfp4

    lens = [c + e for c, e in zip(cached, new)]
    codes, scales = pool(sum(lens), n_kv, d, 1)
    idx, q = listed(lens, sum(lens), 2), rows(sum(new), n_q, d, 3)
    args = [t.to(gpu) for t in (q, codes, scales, indptr(new), indptr(lens), idx, torch.tensor(cached, dtype=torch.int32))]
    got = paged_prefill_attention_mxfp4(*args, d ** -0.5, max(new), is_cross_attention=is_cross, sliding_window_size=window)
    out, spread, score = _attention64(gpu, q, codes, scales, new, lens, idx, cached, d ** -0.5, is_cross, window)
    assert_within(got, out, spread, tolerance(spread, score, out, d, cut=True))


@pytest.mark.parametrize("is_cross,window", [(False, 0), (True, 0), (False, 1), (False, 50), (False, 700), (True, 50), (True, 700)])
@pytest.mark.parametrize("n_q,n_kv,d,new,cached", [
    (32, 8, 128, [17, 300, 64, 0, 1], [2000, 130, 1, 40, 900]), (4, 4, 128, [65, 200], [1000, 3001]), (8, 1, 128, [513], [777]),
    (24, 4, 256, [6, 130, 33], [1999, 64, 700]), (16, 2, 256, [40, 0, 9], [5000, 3, 1]), (32, 8, 128, [8, 3, 0, 1], [2000, 4, 1, 900]),
    (16, 2, 256, [4, 1], [3000, 127])])
def test_workspaces_and_rows_behind_the_last(gpu, n_q, n_kv, d, new, cached, is_cross, window):
    """What a workspace held (zeros, or NaN in all that lies before a window and is not unpacked) does not matter, and rows of the result that no request
    covers are left."""
    lib = _lib.load()
    lens = [c + e for c, e in zip(cached, new)]
    num_slots, n, behind = sum(lens) + 2, sum(new), 5
    codes, scales = pool(num_slots, n_kv, d, 3)
    idx, q = listed(lens, num_slots, 4), rows(n + behind, n_q, d, 5)
    dev = [t.to(gpu) for t in (q, codes, scales, indptr(new), indptr(lens), idx, torch.tensor(cached, dtype=torch.int32))]
    size = lib.msgl_paged_prefill_mxfp4_workspace_bytes(len(new), n + behind, sum(lens), n_q, n_kv, d, max(new))
    got = []
    for byte in (0x00, 0xff):
        ws, out = torch.full((size,), byte, dtype=torch.uint8, device=gpu), torch.full_like(dev[0], 7.0)
        print(f"{n_q}/{n_kv} x {d}, {new} on {cached}, cross {is_cross}, window {window}, workspace {size} of {byte}", flush=True)
        rc = lib.msgl_paged_prefill_attention_mxfp4(
            *(t.data_ptr() for t in dev), out.data_ptr(), ws.data_ptr(), size, len(new), n + behind, sum(lens), n_q, n_kv, d, num_slots,
            dev[1].stride(0), dev[2].stride(0), d ** -0.5, max(new), int(is_cross), window, 0, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        torch.cuda.synchronize()
        got.append(out)
    assert torch.equal(got[0], got[1]) and (got[0][n:] == 7.0).all()
    want, spread, score = _attention64(gpu, q[:n], codes, scales, new, lens, idx, cached, d ** -0.5, is_cross, window)
    assert_within(got[0][:n], want, spread, tolerance(spread, score, want, d, cut=True))


# ---- norm + rotary + store of many tokens: four to a workgroup from 2048 on ----------------------------------
@pytest.mark.parametrize("n,n_q,n_kv,d", [(2047, 3, 1, 128), (2048, 2, 2, 128), (2049, 5, 1, 128), (2051, 1, 1, 128), (2048, 1, 1, 256), (2049, 2, 2, 256),
                                          (2051, 3, 1, 256)])
@pytest.mark.parametrize("far", [0, 131072])
def test_norm_rope_store_of_many_tokens(gpu, n, n_q, n_kv, d, far):
    rows_tests.test_norm_rope_store(gpu, n, n_q, n_kv, d, far)


@pytest.mark.parametrize("n,d", [(2049, 128), (2050, 256), (4003, 128)])
def test_norm_rope_store_of_many_tokens_is_that_of_few(gpu, n, d):
    """The same bits in one call as in calls of 500, with rows that are not finite and slots outside the pool."""
    from mini_sglang_amd_kernel import qk_norm_rope_store_mxfp4

    n_q, n_kv, slots = 20, 18, n + 4  # heads beyond those of one trip
    qkv = rows(n, n_q + 2 * n_kv, d, n).to(gpu)
    for t, h in ((0, n_q), (n - 1, n_q + 2), (n - 2, n_q + n_kv + 1), (700, n_q + n_kv)):
        qkv[t, h, t % d] = float("nan") if t % 2 else float("inf")
    w = (1 + 0.1 * rows(2, 1, d, 1).view(2, d)).to(BF16).to(gpu)
    loc = torch.randperm(slots, generator=torch.Generator().manual_seed(n))[:n].to(torch.int32)
    loc[[3, n - 3]] = torch.tensor([-1, slots], dtype=torch.int32)
    loc, positions = loc.to(gpu), (torch.arange(n, dtype=torch.int32) * 37).to(gpu)
    results = []
    for step in (n, 500):
        codes = torch.full((slots, n_kv, 2, d // 2), 0xA5, dtype=torch.uint8, device=gpu)
        scales = torch.full((slots, n_kv, 2, d // 32), 0x5A, dtype=torch.uint8, device=gpu)
        q = torch.cat([qk_norm_rope_store_mxfp4(x[:, :n_q], x[:, n_q:n_q + n_kv], x[:, n_q + n_kv:], w[0], w[1], p, at, codes, scales, eps=1e-6, rope_base=1e6)
                       for x, p, at in zip(qkv.split(step), positions.split(step), loc.split(step))])
        results.append((q.view(torch.int16), codes, scales))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert int((results[0][2] == 255).any(-1).any(-1).sum()) == 4  # (token, head) pairs
