"""The K/V pool in 4 bits as a serving loop uses it: ``AttnBackend`` over an ``MXFP4KVCache``, step after step, and its calls on
streams, in graphs and with index checks on."""
from types import SimpleNamespace

import pytest
import torch

from _mxfp4_util import assert_within, indptr, listed, pool, rows, tolerance
from oracle import mxfp4_oracle as mx

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
N_Q, N_KV, D, PAGE = 8, 2, 128, 16


class _Server:
    """Two requests over shared layers: slots by page, the step's batch, and its outputs against the definition."""

    def __init__(self, gpu, layers=2, dtype=BF16):
        from mini_sglang_amd.attention import AttnBackend
        from mini_sglang_amd.kvcache import create_kvcache

        pages = torch.randperm(200, generator=torch.Generator().manual_seed(3)).view(2, 100)
        self.table = torch.zeros(3, 1600, dtype=torch.int32)
        self.table[:2] = (pages[:, :, None] * PAGE + torch.arange(PAGE)).reshape(2, -1)
        self.cache = create_kvcache(SimpleNamespace(num_kv_heads=N_KV, num_layers=layers, head_dim=D), 3200, dtype, device=gpu, kv_format="mxfp4")
        self.backend = AttnBackend(SimpleNamespace(head_dim=D), self.cache, self.table.to(gpu))
        self.gpu, self.layers, self.lens, self.seed, self.dtype = gpu, layers, [0, 0], 0, dtype

    def step(self, new, decode=False, fused=False, **mask):
        self.seed += 1
        cached, total = self.lens, [c + e for c, e in zip(self.lens, new)]
        self.lens = total
        reqs = [SimpleNamespace(table_idx=b, cached_len=c, device_len=t, extend_len=t - c) for b, (c, t) in enumerate(zip(cached, total))]
        loc = torch.cat([self.table[b, c:t] for b, (c, t) in enumerate(zip(cached, total))])
        batch = SimpleNamespace(reqs=reqs, padded_reqs=reqs, is_prefill=not decode, attn_metadata=None, out_loc=loc.to(self.gpu))
        self.backend.prepare_metadata(batch)
        for layer in range(self.layers):
            qkv = rows(sum(new), N_Q + 2 * N_KV, D, 100 * self.seed + layer, self.dtype).to(self.gpu)
            q, k, v = qkv[:, :N_Q], qkv[:, N_Q:N_Q + N_KV], qkv[:, N_Q + N_KV:]
            if fused:
                w = (1 + 0.1 * rows(1, 1, D, 5).view(D)).to(BF16).to(self.gpu)
                got = self.backend.forward_fused_norm_rope(q, k, v, w, w, layer, batch, rms_norm_eps=1e-6, rope_base=1e6, **mask)
                from mini_sglang_amd_kernel import qk_norm_rope_store_mxfp4

                codes, scales = torch.zeros_like(self.cache.codes(layer)), torch.zeros_like(self.cache.scales(layer))
                q = qk_norm_rope_store_mxfp4(q, k, v, w, w, batch.attn_metadata.positions, batch.out_loc, codes, scales, eps=1e-6, rope_base=1e6)
                assert torch.equal(codes[loc.long()], self.cache.codes(layer)[loc.long()])
            else:
                got = self.backend.forward(q.contiguous(), k, v, layer, batch, **mask)
                want = mx.quantised(k.cpu(), v.cpu())
                assert torch.equal(self.cache.codes(layer).cpu()[loc.long()], want[0])
                assert torch.equal(self.cache.scales(layer).cpu()[loc.long()], want[1])
            out, spread, score = mx.attention(
                q.cpu(), self.cache.codes(layer).cpu(), self.cache.scales(layer).cpu(), None if decode else indptr(new), indptr(total),
                torch.cat([self.table[b, :t] for b, t in enumerate(total)]), None if decode else torch.tensor(cached), D ** -0.5,
                is_cross=mask.get("is_cross_attention", False), window=mask.get("sliding_window_size", 0))
            cut = not decode and max(new) * (N_Q // N_KV) > 64
            assert_within(got, out, spread, tolerance(spread, score, out, D, self.dtype, cut), f"step {self.seed}")


@pytest.mark.parametrize("fused", [False, True])
def test_prompts_chunks_drafts_and_decode_steps(gpu, fused):
    s = _Server(gpu)
    s.step([300, 37], fused=fused)  # prompts
    s.step([1, 1], decode=True, fused=fused)
    s.step([64, 200], fused=fused)  # chunks on what is there
    s.step([5, 5], fused=fused)  # drafts
    s.step([5, 3], fused=fused, sliding_window_size=100)
    s.step([90, 1], fused=fused, sliding_window_size=50)
    s.step([4, 4], fused=fused, is_cross_attention=True)
    for _ in range(3):
        s.step([1, 1], decode=True, fused=fused)


def test_half_precision_decode_steps(gpu):
    s = _Server(gpu, layers=1, dtype=F16)
    for n in (40, 700):  # rows stored as a prompt's are, attended one by one
        loc = torch.cat([s.table[b, s.lens[b]:s.lens[b] + n] for b in range(2)]).to(gpu)
        s.cache.store_kv(rows(2 * n, N_KV, D, n, F16).to(gpu), rows(2 * n, N_KV, D, n + 1, F16).to(gpu), loc, 0)
        s.lens = [x + n for x in s.lens]
        s.step([1, 1], decode=True)
    with pytest.raises(RuntimeError, match="bfloat16 only"):
        s.step([2, 2])


def test_load_kv_of_the_cache(gpu):
    s = _Server(gpu, layers=2)
    s.step([20, 30])
    loc = s.table[1, :30]
    k, v = s.cache.load_kv(loc.to(gpu), 1)
    want = mx.values(s.cache.codes(1).cpu()[loc.long()], s.cache.scales(1).cpu()[loc.long()])
    assert torch.equal(k.double().cpu(), want[:, :, 0]) and torch.equal(v.double().cpu(), want[:, :, 1])


def _decode_args(gpu, lens, seed=1, n_q=32, n_kv=8, d=128):
    codes, scales = pool(sum(lens), n_kv, d, seed)
    return [t.to(gpu) for t in (rows(len(lens), n_q, d, seed), codes, scales, indptr(lens), listed(lens, sum(lens), seed))]


def test_a_decode_step_in_a_graph(gpu):
    """Captured once; replayed with new rows, queries and lengths, eager work in between, and every replay equal to the eager step."""
    from mini_sglang_amd_kernel import paged_decode_attention_mxfp4, qk_norm_rope_store_mxfp4

    lens, n_q, n_kv, d = [300, 1, 77, 1500], 16, 8, 128
    slots = sum(lens) + 40
    codes, scales = (t.to(gpu) for t in pool(slots, n_kv, d, 1))
    idx, ip = listed(lens, slots, 2).to(gpu), indptr(lens).to(gpu)
    loc, positions = idx[(ip[1:] - 1).long()].clone(), (ip[1:] - ip[:-1] - 1).clone()
    qkv, w = rows(4, n_q + 2 * n_kv, d, 3).to(gpu), torch.ones(d, dtype=BF16, device=gpu)

    def step(codes, scales):
        q = qk_norm_rope_store_mxfp4(qkv[:, :n_q], qkv[:, n_q:n_q + n_kv], qkv[:, n_q + n_kv:], w, w, positions, loc, codes, scales, eps=1e-6,
                                     rope_base=1e6)
        return paged_decode_attention_mxfp4(q, codes, scales, ip, idx, d ** -0.5)

    step(codes, scales)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(codes, scales)
    for i in range(6):
        qkv.copy_(rows(4, n_q + 2 * n_kv, d, 10 + i))
        if i >= 3:  # other lengths, no more keys than there were
            ip.copy_(indptr([250 - i, 0, 60, 900 + i]))
        graph.replay()
        eager = step(codes.clone(), scales.clone())
        assert torch.equal(out, eager), i
        torch.cuda.synchronize()


def test_two_graphs_of_extends(gpu):
    """A long and a short extend, captured each with a workspace of its own, replayed in turn."""
    from mini_sglang_amd_kernel import paged_prefill_attention_mxfp4

    calls = []
    for new, cached in (([70, 200], [130, 0]), ([3, 4], [500, 20])):
        lens = [c + e for c, e in zip(cached, new)]
        _, codes, scales, ip, idx = _decode_args(gpu, lens, sum(new))
        q = rows(sum(new), 32, 128, 9).to(gpu)
        args = (q, codes, scales, indptr(new).to(gpu), ip, idx, torch.tensor(cached, dtype=torch.int32, device=gpu), 128 ** -0.5, max(new))
        paged_prefill_attention_mxfp4(*args)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = paged_prefill_attention_mxfp4(*args)
        calls.append((graph, out, args))
    for i in range(4):
        for graph, out, args in calls:
            args[0].copy_(rows(args[0].shape[0], 32, 128, 20 + i))
            graph.replay()
        for graph, out, args in calls:
            assert torch.equal(out, paged_prefill_attention_mxfp4(*args))


def test_two_streams_at_once(gpu):
    from mini_sglang_amd_kernel import paged_decode_attention_mxfp4

    sets = [_decode_args(gpu, [2000, 500, 33], 1), _decode_args(gpu, [100] * 40, 2)]
    want = [paged_decode_attention_mxfp4(*a, 0.1) for a in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(gpu) for _ in sets]
    got = [[], []]
    for _ in range(10):
        for i, (s, a) in enumerate(zip(streams, sets)):
            got[i].append(paged_decode_attention_mxfp4(*a, 0.1, stream=s))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, w) for x in g)


def test_rows_on_a_stream_of_their_own(gpu):
    from mini_sglang_amd_kernel import load_kv_cache_mxfp4, store_kv_cache_mxfp4

    codes, scales = (t.to(gpu) for t in pool(500, 4, 128, 1))
    k, v, loc = rows(400, 4, 128, 2).to(gpu), rows(400, 4, 128, 3).to(gpu), torch.arange(400, dtype=torch.int32, device=gpu)
    s = torch.cuda.Stream(gpu)
    torch.cuda.synchronize()
    store_kv_cache_mxfp4(codes, scales, loc, k, v, stream=s)
    got = load_kv_cache_mxfp4(codes, scales, loc, stream=s)
    s.synchronize()
    want = mx.values(*mx.quantised(k.cpu(), v.cpu()))
    assert torch.equal(got[0].double().cpu(), want[:, :, 0]) and torch.equal(got[1].double().cpu(), want[:, :, 1])


def test_index_checks(gpu):
    from mini_sglang_amd_kernel import (load_kv_cache_mxfp4, paged_decode_attention_mxfp4, paged_prefill_attention_mxfp4,
                                        store_kv_cache_mxfp4)

    q, codes, scales, ip, idx = _decode_args(gpu, [5, 9])
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    assert torch.equal(paged_decode_attention_mxfp4(q, codes, scales, ip, idx, 0.1, validate=True), paged_decode_attention_mxfp4(q, codes, scales, ip, idx, 0.1))
    paged_prefill_attention_mxfp4(q, codes, scales, i32(0, 1, 2), ip, idx, i32(4, 8), 0.1, 1, validate=True)
    bad = idx.clone()
    bad[3] = 14
    k = rows(2, 8, 128, 1).to(gpu)
    for call in (lambda: paged_decode_attention_mxfp4(q, codes, scales, ip, bad, 0.1, validate=True),
                 lambda: paged_prefill_attention_mxfp4(q, codes, scales, i32(0, 1, 2), ip, bad, i32(4, 8), 0.1, 1, validate=True),
                 lambda: load_kv_cache_mxfp4(codes, scales, bad, validate=True),
                 lambda: store_kv_cache_mxfp4(codes, scales, i32(0, 14), k, k, validate=True)):
        with pytest.raises(RuntimeError, match="outside"):
            call()
    with pytest.raises(RuntimeError, match="duplicate"):
        store_kv_cache_mxfp4(codes, scales, i32(3, 3), k, k, validate=True)
    with pytest.raises(RuntimeError, match="non-decreasing"):
        paged_decode_attention_mxfp4(q, codes, scales, i32(0, 9, 4), idx, 0.1, validate=True)
