"""The K/V pool in 4 bits on the host: what its entry points refuse, sizes of workspaces, and the pool's own arithmetic."""
import ctypes
from types import SimpleNamespace

import pytest
import torch

BF16, F16, U8, I32 = torch.bfloat16, torch.float16, torch.uint8, torch.int32


def _pool(pages=6, heads=2, d=128):
    return torch.zeros(pages, heads, 2, d // 2, dtype=U8), torch.zeros(pages, heads, 2, d // 32, dtype=U8)


def _ids(n):
    return torch.arange(n, dtype=I32)


def _refuses(text, call, *args, **kw):
    with pytest.raises(RuntimeError, match=text):
        call(*args, **kw)


def test_pool_forms_that_are_refused():
    from mini_sglang_amd_kernel import load_kv_cache_mxfp4

    codes, scales = _pool()
    no = lambda text, c, s: _refuses(text, load_kv_cache_mxfp4, c, s, _ids(2))  # noqa: E731
    no("must be 4D", codes[0], scales)
    no("must be 4D", codes, scales[0])
    no("must be uint8", codes.to(torch.int8), scales)
    no("must be uint8", codes, scales.to(BF16))
    no("head_dim must be 128 or 256", codes[..., :32], scales[..., :2])
    no("must be .num_pages, num_kv_heads, 2", codes, scales[:, :1])
    no("must be .num_pages, num_kv_heads, 2", codes, torch.zeros(6, 2, 2, 8, dtype=U8))
    no("as many pages", codes, scales[:5])
    no("must have a page", codes[:0], scales[:0])
    no("contiguous behind their first", torch.zeros(6, 2, 2, 128, dtype=U8)[..., ::2], scales)
    no("contiguous behind their first", torch.zeros(6, 4, 2, 64, dtype=U8)[:, ::2], scales)
    no("ROCm GPU device", codes, scales)
    _refuses("dtype must be", load_kv_cache_mxfp4, codes, scales, _ids(2), dtype=torch.float32)
    _refuses("indices must be 1D", load_kv_cache_mxfp4, codes, scales, _ids(2)[None])
    _refuses("indices must be int32", load_kv_cache_mxfp4, codes, scales, _ids(2).long())


def test_store_refusals():
    from mini_sglang_amd_kernel import store_kv_cache_mxfp4

    codes, scales = _pool()
    k = torch.zeros(3, 2, 128, dtype=BF16)
    no = lambda text, *a: _refuses(text, store_kv_cache_mxfp4, codes, scales, *a)  # noqa: E731
    no("indices must be 1D", _ids(3)[None], k, k)
    no("k and v must be 3D", _ids(3), k[0], k)
    no("k must be float16 or bfloat16", _ids(3), k.float(), k.float())
    no("same dtype", _ids(3), k, k.half())
    no("indices must be int32", _ids(3).long(), k, k)
    no("shape must be .length", _ids(2), k, k)
    no("shape must be .length", _ids(3), k, k[:, :1])
    no("must be .num_pages", _ids(3), k[:, :1], k[:, :1])
    no("ROCm GPU device", _ids(3), k, k)


def test_norm_rope_store_refusals():
    from mini_sglang_amd_kernel import qk_norm_rope_store_mxfp4

    codes, scales = _pool()
    q, k, w = torch.zeros(3, 4, 128, dtype=BF16), torch.zeros(3, 2, 128, dtype=BF16), torch.ones(128, dtype=BF16)

    def no(text, q=q, k=k, v=k, qw=w, kw=w, pos=_ids(3), loc=_ids(3)):
        _refuses(text, qk_norm_rope_store_mxfp4, q, k, v, qw, kw, pos, loc, codes, scales, eps=1e-6, rope_base=1e4)

    no("q must be 3D", q=q[0])
    no("q must be bfloat16", q=q.half())
    no("q must have a head", q=q[:, :0])
    no("k_weight must be bfloat16", kw=w.float())
    no("shape must be .tokens", k=k[:2], v=k[:2])
    no("shape must be .tokens", v=k[:, :1])
    no("q_weight and k_weight", qw=w[:64])
    no("positions must be int32", pos=_ids(3).long())
    no("length must match", loc=_ids(2))
    no("length must match", pos=_ids(3)[:, None])
    no("must be .num_pages", q=q, k=k[:, :1], v=k[:, :1])
    no("ROCm GPU device")


def test_attention_refusals():
    from mini_sglang_amd_kernel import paged_decode_attention_mxfp4, paged_prefill_attention_mxfp4

    codes, scales = _pool()
    q = torch.zeros(3, 4, 128, dtype=BF16)

    def dec(text, q=q, ip=_ids(4), ix=_ids(6), codes=codes, scales=scales):
        _refuses(text, paged_decode_attention_mxfp4, q, codes, scales, ip, ix, 0.1)

    dec("q must be 3D", q=q[0])
    dec("must be 1D", ip=_ids(4)[None])
    dec("multiple of num_kv_heads", q=q[:, :3])
    dec("multiple of num_kv_heads", q=q[:, :0])
    dec("<= 16", q=torch.zeros(3, 34, 128, dtype=BF16))
    dec("must be .num_pages", q=torch.zeros(3, 4, 256, dtype=BF16))
    dec("q must be float16 or bfloat16", q=q.float())
    dec("kv_indices must be int32", ix=_ids(6).long())
    dec("batch \\+ 1", ip=_ids(3))
    dec("ROCm GPU device")

    def pre(text, q=q, qo=_ids(2), ip=_ids(2), ix=_ids(6), pl=_ids(1), most=3, window=0):
        _refuses(text, paged_prefill_attention_mxfp4, q, codes, scales, qo, ip, ix, pl, 0.1, most, sliding_window_size=window)

    pre("q must be 3D", q=q[0])
    pre("must be 1D", pl=_ids(1)[None])
    pre("multiple of num_kv_heads", q=q[:, :3])
    pre("sliding_window_size must be >= 0", window=-1)
    pre("batch must be > 0", qo=_ids(1))
    pre("bfloat16 only", q=q.half())
    pre("prefix_lens must be int32", pl=_ids(1).long())
    pre("must match qo_indptr", ip=_ids(3))
    pre("fit 32 bits", most=1 << 31)
    pre("fit 32 bits", window=1 << 31)
    pre("ROCm GPU device")


def test_c_entries_refuse_before_any_launch():
    """Return codes of the C ABI: none of these calls gets as far as a launch."""
    from mini_sglang_amd_kernel import _lib

    lib, fake, odd = _lib.load(), ctypes.c_void_p(0x1000), ctypes.c_void_p(0x1004)

    def store(codes=fake, scales=fake, idx=fake, k=fake, n=2, heads=2, d=128, slots=8, cs=256, ss=16, ks=256, dtype=0):
        return lib.msgl_store_kv_cache_mxfp4(codes, scales, idx, k, fake, n, heads, d, slots, cs, ss, ks, ks, dtype, None)

    assert store(d=64) == -2 and store(dtype=2) == -5 and store(n=-1) == -9 and store(heads=0) == -9 and store(slots=0) == -9
    assert store(cs=255) == -9 and store(ss=8) == -9 and store(ks=128) == -9
    assert store(codes=None) == -1 and store(idx=None) == -1 and store(k=None) == -1
    assert store(codes=odd) == -10 and store(scales=odd) == -10 and store(k=odd) == -10 and store(cs=264) == -10 and store(ss=20) == -10
    assert store(n=0, codes=None, idx=None) == 0 and store(n=1 << 30) == -9

    def load(codes=fake, k=fake, n=2, d=128, dtype=0, slots=8):
        return lib.msgl_load_kv_cache_mxfp4(codes, fake, fake, k, fake, n, 2, d, slots, 256, 16, dtype, None)

    assert load(d=96) == -2 and load(dtype=3) == -5 and load(codes=None) == -1 and load(k=odd) == -10 and load(slots=0) == -9 and load(n=0) == 0

    def rope(q=fake, n=2, n_q=4, d=128, qs=512, eps=1e-6, base=1e4, dtype=0):
        return lib.msgl_qk_norm_rope_store_mxfp4(q, fake, fake, qs, 256, 256, fake, fake, fake, fake, fake, fake, fake, 256, 16, 8, n, n_q, 2, d,
                                                 eps, base, dtype, None)

    assert rope(d=64) == -2 and rope(dtype=1) == -5 and rope(n_q=0) == -9 and rope(qs=384) == -9 and rope(eps=-1.0) == -9
    assert rope(base=1.0) == -9 and rope(base=float("nan")) == -9 and rope(base=float("inf")) == -9 and rope(eps=float("nan")) == -9
    assert rope(q=None) == -1 and rope(q=odd) == -10 and rope(qs=516) == -10 and rope(n=0, q=None) == 0

    def dec(q=fake, ws=fake, size=1 << 40, batch=2, total=100, n_q=8, n_kv=2, d=128, dtype=0, idx=fake):
        return lib.msgl_paged_decode_attention_mxfp4(q, fake, fake, fake, idx, fake, ws, size, batch, total, n_q, n_kv, d, 8, n_kv * d, n_kv * d // 16,
                                                     0.1, dtype, None)

    assert dec(d=64) == -2 and dec(n_q=7) == -3 and dec(n_q=34) == -4 and dec(dtype=2) == -5 and dec(ws=None) == -8 and dec(size=64) == -8
    assert dec(q=None) == -1 and dec(idx=None) == -1 and dec(q=odd) == -10 and dec(batch=-1) == -9 and dec(total=1 << 31) == -9 and dec(total=(1 << 30) + 1) == -9 and dec(batch=0) == 0

    def pre(q=fake, ws=fake, size=1 << 45, batch=2, total_q=9, total=100, n_q=8, d=128, most=5, window=0, dtype=0, pl=fake):
        return lib.msgl_paged_prefill_attention_mxfp4(q, fake, fake, fake, fake, fake, pl, fake, ws, size, batch, total_q, total, n_q, 2, d, 8, 2 * d,
                                                      d // 8, 0.1, most, 0, window, dtype, None)

    assert pre(d=64) == -2 and pre(n_q=7) == -3 and pre(window=-1) == -7 and pre(batch=0) == -6 and pre(dtype=1) == -5
    assert pre(q=None) == -1 and pre(pl=None) == -1 and pre(q=odd) == -10 and pre(total_q=-1) == -9
    assert pre(ws=None) == -8 and pre(size=1 << 10) == -8 and pre(ws=None, most=500) == -8 and pre(size=1 << 10, most=500) == -8
    assert pre(total_q=0, q=None) == 0 and pre(most=0, q=None) == 0


def test_workspace_sizes():
    from mini_sglang_amd_kernel import _lib

    lib = _lib.load()
    dec, pre = lib.msgl_paged_decode_mxfp4_workspace_bytes, lib.msgl_paged_prefill_mxfp4_workspace_bytes
    assert dec(0, 10, 8, 2, 128) == 0 and dec(2, 10, 7, 2, 128) == 0 and dec(2, -1, 8, 2, 128) == 0
    assert 0 < dec(4, 2000, 16, 8, 128) < dec(64, 300000, 32, 8, 128) < 64 << 20
    assert pre(2, 10, 100, 7, 2, 128, 5) == 0 and pre(2, 10, 100, 8, 2, 128, 0) == 0
    # a long extend: K and V of every listed key in bf16, and their numbers
    assert pre(8, 4096, 65536, 32, 8, 128, 512) >= 65536 * (8 * 128 * 4 + 4)
    assert pre(8, 32, 65536, 32, 8, 128, 4) < 64 << 20  # a short one reads the codes


def test_pool_object():
    from mini_sglang_amd.kvcache import MHAKVCache, MXFP4KVCache, create_kvcache

    config = SimpleNamespace(num_kv_heads=4, num_layers=3, head_dim=256)
    cache = create_kvcache(config, 10, BF16, device="cpu", kv_format="mxfp4")
    assert type(cache) is MXFP4KVCache and type(create_kvcache(config, 10, BF16, device="cpu")) is MHAKVCache
    assert cache.pool_shape == (10, 4, 256) and cache.num_layers == 3 and cache.dtype is BF16
    assert cache.codes(1).shape == (10, 4, 2, 128) and cache.scales(2).shape == (10, 4, 2, 8)
    assert cache.k_cache(0).shape == cache.v_cache(0).shape == (10, 4, 128)
    assert cache.k_cache(1).data_ptr() == cache.codes(1).data_ptr()
    assert cache.nbytes * 64 == create_kvcache(config, 10, BF16, device="cpu").nbytes * 17  # 4.25 bits of 16
    with pytest.raises(KeyError, match="Unsupported KV format"):
        create_kvcache(config, 10, BF16, device="cpu", kv_format="int8")
    for bad in (dict(head_dim=64), dict(num_layers=0), dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            MXFP4KVCache(**{**dict(num_kv_heads=2, num_layers=1, head_dim=128, num_pages=4, dtype=BF16, device="cpu"), **bad})
    with pytest.raises(ValueError, match="slot ids"):
        cache.store_kv(torch.zeros(2, 4, 256), torch.zeros(3, 4, 256), torch.zeros(3, dtype=I32), 0)
