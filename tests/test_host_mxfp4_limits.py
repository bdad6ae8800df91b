"""The K/V pool in 4 bits on the host: sizes that its kernels' 32-bit numbers do not hold are refused before any launch."""
import ctypes

import pytest
import torch

BF16, F16, U8, I32 = torch.bfloat16, torch.float16, torch.uint8, torch.int32
FAKE, SHAPE = ctypes.c_void_p(0x1000), -9


def _entries(cs, ss):
    """Every C entry over a pool of 8 slots of 2 heads, `cs` and `ss` bytes from one to the next."""
    from mini_sglang_amd_kernel import _lib

    lib, f = _lib.load(), FAKE
    yield lib.msgl_store_kv_cache_mxfp4(f, f, f, f, f, 2, 2, 128, 8, cs, ss, 256, 256, 0, None)
    yield lib.msgl_load_kv_cache_mxfp4(f, f, f, f, f, 2, 2, 128, 8, cs, ss, 0, None)
    yield lib.msgl_qk_norm_rope_store_mxfp4(f, f, f, 512, 256, 256, f, f, f, f, f, f, f, cs, ss, 8, 2, 4, 2, 128, 1e-6, 1e4, 0, None)
    yield lib.msgl_paged_decode_attention_mxfp4(f, f, f, f, f, f, f, 1 << 40, 2, 100, 8, 2, 128, 8, cs, ss, 0.1, 0, None)
    for most in (4, 500):  # over the codes, over unpacked rows
        yield lib.msgl_paged_prefill_attention_mxfp4(f, f, f, f, f, f, f, f, f, 1 << 45, 2, 9, 100, 8, 2, 128, 8, cs, ss, 0.1, most, 0, 0, 0, None)


@pytest.mark.parametrize("cs,ss", [(1 << 32, 16), (256, 1 << 32), ((1 << 33) + 256, (1 << 33) + 16), (1 << 62, 16)])
def test_slots_four_gib_apart(cs, ss):
    """Attention multiplies slot ids by strides of 32 bits: what lies further apart would be written in one place and read in another."""
    assert list(_entries(cs, ss)) == [SHAPE] * 6


def test_slots_four_gib_apart_are_refused_with_the_reason():
    from mini_sglang_amd_kernel import load_kv_cache_mxfp4, paged_decode_attention_mxfp4

    far = torch.empty((1 << 32) + 4096, dtype=U8)  # never touched
    small = torch.zeros(2, 2, 2, 64, dtype=U8), torch.zeros(2, 2, 2, 4, dtype=U8)
    codes = far.as_strided((2, 2, 2, 64), (1 << 32, 128, 64, 1))
    scales = far.as_strided((2, 2, 2, 4), (1 << 32, 8, 4, 1))
    ids = torch.arange(2, dtype=I32)
    for c, s in ((codes, small[1]), (small[0], scales)):
        with pytest.raises(RuntimeError, match="less than 4 GiB apart"):
            load_kv_cache_mxfp4(c, s, ids)
        with pytest.raises(RuntimeError, match="less than 4 GiB apart"):
            paged_decode_attention_mxfp4(torch.zeros(1, 4, 128, dtype=BF16), c, s, ids, ids, 0.1)


def test_more_kv_heads_than_a_requests_partials_have_room_for():
    """A request's partials are addressed by 32 bits: the entries of attention take 2^15 kv heads at most."""
    from mini_sglang_amd_kernel import _lib

    lib, f = _lib.load(), FAKE
    for n_kv, group in (((1 << 15) + 1, 1), (1 << 17, 16), (1 << 20, 2)):
        n_q = n_kv * group
        for d in (128, 256):
            size = 1 << 60
            assert lib.msgl_paged_decode_attention_mxfp4(f, f, f, f, f, f, f, size, 2, 100, n_q, n_kv, d, 8, n_kv * d, n_kv * d // 16, 0.1, 0, None) == SHAPE
            for most in (2, 500):
                assert lib.msgl_paged_prefill_attention_mxfp4(f, f, f, f, f, f, f, f, f, size, 2, 9, 100, n_q, n_kv, d, 8, n_kv * d, n_kv * d // 16, 0.1, most,
                                                              0, 0, 0, None) == SHAPE


@pytest.mark.parametrize("pool,row", [(F16, BF16), (BF16, F16), (F16, torch.float32)])
def test_rows_of_another_type_than_the_caches(pool, row):
    """A cache's dtype is that of its rows: bf16 reaches values that a decode in half gives as infinities."""
    from types import SimpleNamespace

    from mini_sglang_amd.attention import AttnBackend
    from mini_sglang_amd.kvcache import MXFP4KVCache

    cache = MXFP4KVCache(num_kv_heads=2, num_layers=1, head_dim=128, num_pages=8, dtype=pool, device="cpu")
    right, wrong, loc = torch.zeros(3, 2, 128, dtype=pool), torch.zeros(3, 2, 128, dtype=row), torch.arange(3, dtype=I32)
    for k, v in ((wrong, wrong), (right, wrong), (wrong, right)):
        with pytest.raises(ValueError, match="store_kv: .*the cache's dtype"):
            cache.store_kv(k, v, loc, 0)
    backend = AttnBackend(SimpleNamespace(head_dim=128), cache, torch.zeros(2, 8, dtype=I32))
    with pytest.raises(ValueError, match="the cache's dtype"):
        backend.store_kv_only(wrong, wrong, loc, 0)
    batch = SimpleNamespace(out_loc=loc, attn_metadata=SimpleNamespace(positions=loc))
    with pytest.raises(ValueError, match="the cache's dtype"):
        backend.forward_fused_norm_rope(wrong, wrong, wrong, wrong[0, 0], wrong[0, 0], 0, batch, rms_norm_eps=1e-6, rope_base=1e4)
    with pytest.raises(RuntimeError, match="ROCm GPU device"):  # rows of the right type get as far as the operator
        cache.store_kv(right, right, loc, 0)
