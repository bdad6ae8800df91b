"""The operators of the K/V pool in 4 bits, timed and compared with their plain form.

A pool holds, for every slot and kv head, K and V of ``d`` values as blocks of 32: two 4-bit floats (e2m1: 0, 0.5,
1, 1.5, 2, 3, 4, 6 and a sign) to a byte, the even dim in the low half, and one byte b to a block, whose values are
multiplied by 2^(b - 127).  b is the smallest with which no value of the block is beyond 6, held to [2, 252]; values go
to the nearest, halfway to the even code.  A row of K or V that is not finite leaves 255 in the block bytes of K, and
nothing else, so that whoever sees the key sees NaN.

Kinds of case, each one pass of

* ``store``   the rows of new tokens into the pool, and what it then holds for them read back as values;
* ``append``  the same with the norm of q and k and the rotary embedding in front;
* ``decode``  attention of one new token per request over the pool;
* ``extend``  attention of several new tokens per request under one of the masks.

Request lengths are uniform between the case's ``*_lo`` and ``*_hi``, drawn from its ``lens`` number, so that a case is
one set of shapes; the seed of ``prepare`` decides values, slots and page order.
"""
import math
import os
import random
import sys
from types import SimpleNamespace

import torch

# the package folder lies under the root this file is used from
sys.path.insert(1, os.path.abspath("mini-sglang-mlx_amd"))

own = False

PAGE = 16
BLOCK = 32
EPS = 1e-6
ROPE_BASE = 1e6
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _case(name, op, batch, heads, kv, ext=(1, 1), d=128, dtype="bf16", window=0, cross=False, lens=1):
    """``kv``: tokens in the cache before this step (shortest, longest request); ``ext``: new ones."""
    case = {"op": op, "batch": batch, "n_q": heads[0], "n_kv": heads[1], "d": d, "dtype": dtype, "kv_lo": kv[0], "kv_hi": kv[1],
            "ext_lo": ext[0], "ext_hi": ext[1], "window": window, "cross": cross, "lens": lens}
    return dict(case, name=name) if name else case


def listed():
    return [
        # the new tokens of four chats, half precision, head_dim 256: one round trip counts
        _case("store_few", "store", 4, (16, 2), (127, 4095), d=256, dtype="f16"),
        # fresh prompts of odd lengths whose keys are there already (a draft model's, a prefix moved between pools)
        _case("store_prompts", "store", 6, (32, 8), (0, 0), (237, 3333), lens=3),
        # one decode step of a loaded server, far into long documents
        _case("append_step", "append", 64, (32, 8), (1023, 131071)),
        # a chunk of a prefill: 512 new tokens each
        _case("append_chunks", "append", 8, (32, 8), (0, 16384), (512, 512)),
        # interactive use of a small model: four chats
        _case("decode_small", "decode", 4, (16, 8), (36, 1022)),
        # a loaded server in steady state: 64 requests of ordinary length
        _case("decode_batch", "decode", 64, (32, 8), (1023, 8191)),
        # long documents: 16 requests of 32 K to 128 K tokens, 64 query heads
        _case("decode_long", "decode", 16, (64, 8), (32767, 131071)),
        # the full-attention layer of a hybrid model: head_dim 256, few kv heads, half precision, short ragged chats
        _case("decode_d256_half", "decode", 24, (16, 2), (127, 4095), d=256, dtype="f16"),
        # speculative verify: eight draft tokens per request
        _case("verify", "extend", 32, (32, 8), (2048, 8192), (8, 8)),
        # the same on a sliding-window layer
        _case("verify_window", "extend", 32, (32, 8), (2048, 8192), (8, 8), window=1024),
        # chunked prefill: 512 new tokens each on cached prefixes of very different length
        _case("extend_chunks", "extend", 8, (32, 8), (0, 16384), (512, 512)),
        # prefill of the head_dim 256 layer, ragged
        _case("extend_d256", "extend", 4, (24, 4), (0, 8192), (237, 2048), d=256),
    ]


def _log(rng, lo, hi):
    """An integer in [lo, hi], its logarithm uniform."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(case):
    w = work(case)
    return w["bytes"] / 6e12 + w["flops"] / 1e15


def _padded(case):
    """Scores and keys of the plain form, in which every request is as long as the longest."""
    ext, cached = _lengths(case)
    keys = max(c + e for c, e in zip(cached, ext))
    return case["batch"] * keys * max(case["n_q"] * max(ext), case["n_kv"] * case["d"])


def draw(rng):
    most = {}
    for c in listed():
        most[c["op"]] = max(_cost(c), most.get(c["op"], 0.0))
    while True:
        op, lens = rng.choice(("store", "append", "decode", "decode", "verify", "extend")), rng.randrange(1 << 16)
        d = rng.choice((128, 128, 256))
        heads = rng.choice(((16, 8), (32, 8), (64, 8)) if d == 128 else ((16, 2), (16, 4), (24, 4), (32, 2)))
        half = rng.choice(("bf16", "bf16", "f16"))
        if op in ("store", "append"):
            new, cached = _log(rng, 1, 4096), _log(rng, 1, 131072)
            case = _case("", op, _log(rng, 1, 64), heads, (rng.randint(0, cached), cached), (_log(rng, 1, new), new), d,
                         half if op == "store" else "bf16", lens=lens)
        elif op == "decode":
            top = _log(rng, 64, 131071)
            case = _case("", "decode", _log(rng, 1, 256), heads, (_log(rng, max(1, top // 16), top), top), d=d, dtype=half, lens=lens)
        elif op == "verify":
            n, top = rng.randint(2, 16), _log(rng, 256, 16384)
            case = _case("", "extend", _log(rng, 1, 64), heads, (_log(rng, max(1, top // 16), top), top), (n, n), d,
                         window=rng.choice((0, 0, 1024)), lens=lens)
        else:
            new, cached = _log(rng, 16, 4096), rng.choice((0, _log(rng, 64, 131072)))
            # most layers are causal; some models have sliding windows, drafts see both sides
            window, cross = rng.choice(((0, False),) * 5 + ((1024, False), (0, True), (1024, True)))
            case = _case("", "extend", _log(rng, 1, 32), heads, (rng.randint(0, cached), cached), (_log(rng, 9, new) if new > 9 else new, new),
                         d, window=window, cross=cross, lens=lens)
        if _cost(case) <= most[case["op"]] and (case["op"] in ("store", "append") or _padded(case) <= 5 << 29):
            return case


def _lengths(case):
    r = random.Random(case["lens"])
    ext = [r.randint(case["ext_lo"], case["ext_hi"]) for _ in range(case["batch"])]
    return ext, [r.randint(case["kv_lo"], case["kv_hi"]) for _ in range(case["batch"])]


def _indptr(lens, dev):
    return torch.tensor([sum(lens[:b]) for b in range(len(lens) + 1)], dtype=torch.int32, device=dev)


# ---- the pool's format in elementary operations --------------------------------------------------
def _quantised(k, v):
    """The codes (rows, heads, 2, d / 2) and block bytes (rows, heads, 2, d / 32) of rows of k and v."""
    x = torch.stack((k, v), 2).float()
    rows, heads, _, d = x.shape
    fine = torch.isfinite(x).all(-1).all(-1)[:, :, None, None]
    x = torch.where(fine[..., None], x.view(rows, heads, 2, d // BLOCK, BLOCK), torch.zeros_like(x[:1, :1, :1, :1, None]))
    bits = x.abs().amax(-1).view(torch.int32)
    byte = ((bits >> 23) - 2 + ((bits & 0x7FFFFF) > 0x400000)).clamp(2, 252)
    y = x.abs() * ((254 - byte) << 23).view(torch.float32)[..., None]  # a power of two: exact
    code = (y > 0.25).int() + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5.0)
    code = (code + 8 * torch.signbit(x)).view(rows, heads, 2, d // 2, 2)
    of_k = torch.tensor([True, False], device=x.device)[None, None, :, None]
    return (code[..., 0] + 16 * code[..., 1]).to(torch.uint8), torch.where(of_k & ~fine, 255, byte).to(torch.uint8)


def _values(codes, scales):
    """What codes and block bytes stand for, in 32 bits: (..., d)."""
    code = torch.stack((codes & 15, codes >> 4), -1).int()
    x = torch.tensor(E2M1 + tuple(-y for y in E2M1), device=codes.device)[code].view(*codes.shape[:-1], -1, BLOCK)
    return (x * (scales.int() << 23).view(torch.float32)[..., None]).flatten(-2)


# ---- inputs ----------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    ext, cached = _lengths(case)
    total = [c + e for c, e in zip(cached, ext)]
    n_q, n_kv, d, dtype = case["n_q"], case["n_kv"], case["d"], DTYPES[case["dtype"]]
    s = SimpleNamespace(case=case, most_new=max(ext), most_keys=max(total))

    # slots: pages in random order, half as many again as the requests fill
    appends = case["op"] in ("store", "append")
    pages = [-(-t // PAGE) for t in (ext if appends else total)]  # of what is appended only the new tokens' slots matter
    order = torch.randperm(int(1.5 * sum(pages)) + 1, generator=g, device=dev).to(torch.int32)
    within, at, slots = torch.arange(PAGE, dtype=torch.int32, device=dev), 0, []
    for b, n in enumerate(pages):
        slots.append((order[at:at + n, None] * PAGE + within).view(-1)[:(ext if appends else total)[b]])
        at += n
    num_slots = order.numel() * PAGE
    s.kv_codes = torch.empty((num_slots, n_kv, 2, d // 2), dtype=torch.uint8, device=dev)
    s.kv_scales = torch.empty((num_slots, n_kv, 2, d // BLOCK), dtype=torch.uint8, device=dev)
    rand = lambda *shape: torch.randn(shape, generator=g, device=dev)  # noqa: E731
    slab = max(1, (1 << 26) // (n_kv * d))
    for i in range(0, num_slots, slab):  # what was stored before
        n = min(slab, num_slots - i)
        s.kv_codes[i:i + n], s.kv_scales[i:i + n] = _quantised(rand(n, n_kv, d).to(dtype), rand(n, n_kv, d).to(dtype))
    s.sm_scale = 1.0 / math.sqrt(d)
    if appends:
        s.out_loc = torch.cat(slots)
        s.positions = torch.cat([torch.arange(c, t, dtype=torch.int32, device=dev) for c, t in zip(cached, total)])
        # heads of q, k and v side by side, as one matrix product leaves them
        qkv = rand(sum(ext), n_q + 2 * n_kv, d).to(dtype)
        s.q, s.k, s.v = qkv[:, :n_q], qkv[:, n_q:n_q + n_kv], qkv[:, n_q + n_kv:]
        s.q_weight, s.k_weight = (1 + 0.1 * rand(2, d)).to(dtype)
    else:
        s.q = rand(sum(ext), n_q, d).to(dtype)
        s.kv_indices, s.kv_indptr, s.qo_indptr = torch.cat(slots), _indptr(total, dev), _indptr(ext, dev)
        s.prefix_lens = torch.tensor(cached, dtype=torch.int32, device=dev)
    return s


# ---- one pass ----------------------------------------------------------------------------------------
def run(state):
    s, op = state, state.case["op"]
    if own:
        from mini_sglang_amd_kernel import (load_kv_cache_mxfp4, paged_decode_attention_mxfp4, paged_prefill_attention_mxfp4,
                                            qk_norm_rope_store_mxfp4, store_kv_cache_mxfp4)
        if op == "store":
            store_kv_cache_mxfp4(s.kv_codes, s.kv_scales, s.out_loc, s.k, s.v)
            return load_kv_cache_mxfp4(s.kv_codes, s.kv_scales, s.out_loc, dtype=s.k.dtype)
        if op == "append":
            q = qk_norm_rope_store_mxfp4(s.q, s.k, s.v, s.q_weight, s.k_weight, s.positions, s.out_loc, s.kv_codes, s.kv_scales,
                                         eps=EPS, rope_base=ROPE_BASE)
            return q, *load_kv_cache_mxfp4(s.kv_codes, s.kv_scales, s.out_loc, dtype=s.k.dtype)
        if op == "decode":
            return paged_decode_attention_mxfp4(s.q, s.kv_codes, s.kv_scales, s.kv_indptr, s.kv_indices, s.sm_scale)
        return paged_prefill_attention_mxfp4(s.q, s.kv_codes, s.kv_scales, s.qo_indptr, s.kv_indptr, s.kv_indices, s.prefix_lens,
                                             s.sm_scale, s.most_new, is_cross_attention=s.case["cross"],
                                             sliding_window_size=s.case["window"])
    if op == "store":
        return _stored(s, s.k, s.v)
    if op == "append":
        angle = s.positions.double()[:, None] * _frequencies(s.case["d"], s.q.device)
        cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
        q, k = _rotated(s.q, s.q_weight, cos, sin), _rotated(s.k, s.k_weight, cos, sin)
        return q.to(s.q.dtype), *_stored(s, k, s.v)
    return _attention(s)


def _stored(s, k, v):
    s.kv_codes[s.out_loc], s.kv_scales[s.out_loc] = _quantised(k, v.to(k.dtype))
    x = _values(s.kv_codes[s.out_loc], s.kv_scales[s.out_loc]).to(s.k.dtype)
    return x[:, :, 0].contiguous(), x[:, :, 1].contiguous()


def _frequencies(d, dev):
    return ROPE_BASE ** (-torch.arange(d // 2, dtype=torch.float64, device=dev) / (d // 2))


def _rotated(x, weight, cos, sin):
    """Norm over the head and rotation of its halves.  A value next to the border of two codes of the pool falls by its last bit: the
    norm's factor and the angles are taken in 64 bits, each step from there is one rounding of 32."""
    factor = (1.0 / (x.double().square().mean(-1, keepdim=True) + EPS).sqrt()).float()
    y = weight.float() * (x.float() * factor)
    a, b = y.chunk(2, -1)
    return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)


def _attention(s):
    case, dev = s.case, s.q.device
    batch, n_q, n_kv, d, group = case["batch"], case["n_q"], case["n_kv"], case["d"], case["n_q"] // case["n_kv"]
    last = s.kv_indptr[1:, None] - 1
    key, new = torch.arange(s.most_keys, device=dev)[None], torch.arange(s.most_new, device=dev)[None]
    slots = s.kv_indices[torch.minimum(s.kv_indptr[:-1, None] + key, last).long()].long()
    x = _values(s.kv_codes[slots], s.kv_scales[slots])  # (batch, keys, heads, 2, d)
    k, v = x[:, :, :, 0].permute(0, 2, 3, 1), x[:, :, :, 1].transpose(1, 2)
    row = torch.minimum(s.qo_indptr[:-1, None] + new, s.qo_indptr[1:, None] - 1).long()
    q = s.q[row].float().view(batch, s.most_new, n_kv, group, d).permute(0, 2, 3, 1, 4).reshape(batch, n_kv, -1, d)
    position = (s.prefix_lens[:, None] + new)[:, :, None]
    seen = (key < s.kv_indptr[1:, None] - s.kv_indptr[:-1, None])[:, None]
    if not case["cross"]:
        seen = seen & (key[:, None] <= position)
    if case["window"]:
        seen = seen & (key[:, None] > position - case["window"])
    seen = seen.expand(batch, s.most_new, s.most_keys)[:, None, None]
    p = torch.matmul(q, k).mul_(s.sm_scale).view(batch, n_kv, group, s.most_new, -1).masked_fill_(~seen, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(batch, n_kv, group * s.most_new, -1), v).view(batch, n_kv, group, s.most_new, d)
    out = torch.where(total > 0, out / total, torch.zeros_like(out)).permute(0, 3, 1, 2, 4).reshape(batch, s.most_new, n_q, d)
    return out[new.expand(batch, -1) < (s.qo_indptr[1:, None] - s.qo_indptr[:-1, None])].to(s.q.dtype)


# ---- what a pass cannot do without ---------------------------------------------------------------------
def work(case):
    ext, cached = _lengths(case)
    n, n_q, n_kv, d = sum(ext), case["n_q"], case["n_kv"], case["d"]
    row = 2 * n_kv * d * 2  # a token's k and v in 16 bits
    held = 2 * n_kv * (d // 2 + d // BLOCK)  # and in the pool
    if case["op"] == "store":
        return {"bytes": n * (2 * row + held + 4), "flops": 4 * n * 2 * n_kv * d}
    if case["op"] == "append":
        return {"bytes": n * (2 * row + 2 * n_q * d * 2 + held + 8) + 4 * d, "flops": n * (8 * (n_q + n_kv) + 8 * n_kv) * d}
    keys = pairs = 0
    for c, e in zip(cached, ext):
        w = case["window"]
        keys += c + e - (max(0, c - w + 1) if w else 0)
        pairs += e * (c + e) if case["cross"] else e * c + e * (e + 1) // 2
        if w:  # less what lies before the window: key j of query i where j <= c + i - w
            first = max(0, w - c)  # the first query with such keys
            m = max(0, e - first)
            pairs -= m * (c + first - w) + m * (m + 1) // 2
    return {"bytes": keys * (held + 4) + 2 * n * n_q * d * 2 + 16 * case["batch"], "flops": 4 * d * n_q * pairs}


# ---- the definition in 64 bits ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("store", "append"):
        k, v, outs = s.k.double(), s.v.double(), ()
        if case["op"] == "append":
            outs, k = (_exact_rotated(s.q, s.q_weight, s.positions),), _exact_rotated(s.k, s.k_weight, s.positions)
        return outs + (_exact_held(k), _exact_held(v))
    return _exact_attention(s)


def _exact_held(x):
    """Every value at the nearest of its block's: the pool's values are in order, and halfway the even one is the nearer."""
    blocks = x.unflatten(-1, (-1, BLOCK))
    mantissa, exponent = torch.frexp(blocks.abs().amax(-1, keepdim=True) / 6.0)  # in [0.5, 1): the power above, but for 0.5 itself
    step = torch.ldexp(torch.ones_like(mantissa), (exponent - (mantissa == 0.5).to(exponent.dtype)).clamp(-125, 125))
    size = blocks.abs() / step
    best, held = torch.full_like(size, math.inf), torch.zeros_like(size)
    for value in (0.0, 1.0, 2.0, 4.0, 0.5, 1.5, 3.0, 6.0):  # the even codes first
        near = (size - value).abs()
        held = torch.where(near < best, value, held)
        best = torch.minimum(best, near)
    return (torch.copysign(held, blocks) * step).flatten(-2)


def _exact_rotated(x, weight, positions):
    x, half = x.double(), x.shape[-1] // 2
    y = weight.double() * x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
    i = torch.arange(half, dtype=torch.float64, device=x.device)
    turn = torch.polar(torch.ones(1, dtype=torch.float64, device=x.device), positions.double()[:, None] * torch.exp(-math.log(ROPE_BASE) * i / half))
    z = torch.complex(y[..., :half], y[..., half:]) * turn[:, None]
    return torch.cat((z.real, z.imag), -1)


def _exact_attention(s):
    case, dev = s.case, s.q.device
    n_q, n_kv, d = case["n_q"], case["n_kv"], case["d"]
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=dev)
    table = torch.tensor([m if c < 8 else -m for c in range(16) for m in (E2M1[c % 8],)], dtype=torch.float64, device=dev)
    first_row, first_key, cached = s.qo_indptr.tolist(), s.kv_indptr.tolist(), s.prefix_lens.tolist()
    for b in range(case["batch"]):
        slots = s.kv_indices[first_key[b]:first_key[b + 1]].long()
        rows = slice(first_row[b], first_row[b + 1])
        key = torch.arange(len(slots), device=dev)
        here = cached[b] + torch.arange(first_row[b + 1] - first_row[b], device=dev)[:, None]
        hidden = torch.zeros(len(here), len(slots), dtype=torch.bool, device=dev)
        if not case["cross"]:
            hidden |= key > here
        if case["window"]:
            hidden |= key <= here - case["window"]
        for h in range(n_kv):
            code = s.kv_codes[slots, h].int()
            x = torch.empty(len(slots), 2, d, dtype=torch.float64, device=dev)
            x[..., 0::2], x[..., 1::2] = table[code % 16], table[code // 16]
            x *= torch.ldexp(torch.ones((), dtype=torch.float64, device=dev), s.kv_scales[slots, h].int() - 127).repeat_interleave(BLOCK, -1)
            heads = slice(h * n_q // n_kv, (h + 1) * n_q // n_kv)
            p = torch.matmul(s.q[rows, heads].double().transpose(0, 1), x[:, 0].T.contiguous()) * s.sm_scale
            p = torch.softmax(p.masked_fill(hidden, -math.inf), -1)
            out[rows, heads] = torch.matmul(torch.nan_to_num(p), x[:, 1].contiguous()).transpose(0, 1)
    return out
