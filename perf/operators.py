"""What one decode step of a batch that shares a prompt is measured by: rotary positions with the store into
the key/value cache, attention over the shared prompt and each sequence's own keys, and the adjustment of the
logits; from a few tokens, where latency counts, to prompts and batches that fill the card.

`run` computes them with elementary torch operations; where `own` is set, with the library's calls.
"""
import math
import types

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
WIDTH = {"f32": 4, "bf16": 2, "f16": 2}
DEV = "cuda"
NULL_STREAM = 1  # hipStreamLegacy: what names the null stream, torch's default one, to the library
_backend = None


def listed():
    return [
        # one step of 16 sequences: rotate the new queries and keys, store keys and values in the cache
        {"name": "rope_16", "op": "rope", "tokens": 16, "q_heads": 32, "kv_heads": 8, "d": 128, "rot": 128, "layout": "half",
         "scaling": "none", "dtype": "bf16", "store": 4096, "padded": False, "inverse": False},
        # a prompt of 8192 tokens, angles scaled by parts for a long context
        {"name": "rope_8192", "op": "rope", "tokens": 8192, "q_heads": 32, "kv_heads": 8, "d": 128, "rot": 128, "layout": "half",
         "scaling": "parts", "dtype": "bf16", "store": 16384, "padded": False, "inverse": False},
        # the default element type, a quarter of an odd head, a padded batch
        {"name": "rope_777_part", "op": "rope", "tokens": 777, "q_heads": 12, "kv_heads": 4, "d": 80, "rot": 20, "layout": "interleaved",
         "scaling": "linear", "dtype": "f32", "store": 1000, "padded": True, "inverse": False},
        # the gradients of rotated queries and keys
        {"name": "rope_2048_gradient", "op": "rope", "tokens": 2048, "q_heads": 16, "kv_heads": 16, "d": 64, "rot": 64, "layout": "interleaved",
         "scaling": "base", "dtype": "f16", "store": 0, "padded": False, "inverse": True},
        # four answers to a short prompt: latency
        {"name": "sdpa_4x1024", "op": "sdpa", "batch": 4, "q_len": 1, "q_heads": 32, "kv_heads": 8, "d": 128, "prefix": 1024, "own": 128,
         "page": 0, "dtype": "bf16"},
        # a serving batch over a long system prompt, each sequence's own keys in pages of 16
        {"name": "sdpa_64x8192_paged", "op": "sdpa", "batch": 64, "q_len": 1, "q_heads": 32, "kv_heads": 8, "d": 128, "prefix": 8192,
         "own": 1024, "page": 16, "dtype": "bf16"},
        # questions on one very long document
        {"name": "sdpa_32x65536", "op": "sdpa", "batch": 32, "q_len": 1, "q_heads": 32, "kv_heads": 8, "d": 128, "prefix": 65536, "own": 512,
         "page": 64, "dtype": "f16"},
        # eight different questions of up to 256 tokens read on top of one prompt
        {"name": "sdpa_8x256_chunk", "op": "sdpa", "batch": 8, "q_len": 256, "q_heads": 16, "kv_heads": 4, "d": 64, "prefix": 4096, "own": 512,
         "page": 0, "dtype": "bf16"},
        # the default element type: three drafted tokens, odd heads, groups and lengths, small pages
        {"name": "sdpa_5x3_f32", "op": "sdpa", "batch": 5, "q_len": 3, "q_heads": 6, "kv_heads": 2, "d": 80, "prefix": 1001, "own": 77,
         "page": 8, "dtype": "f32"},
        # four rows of an odd vocabulary, a short history: latency
        {"name": "logits_4x50257", "op": "logits", "rows": 4, "vocab": 50257, "dtype": "f32", "out": "f32", "history": 200, "bias": 16},
        # a large batch over a large vocabulary, histories of a few thousand tokens
        {"name": "logits_256x131072", "op": "logits", "rows": 256, "vocab": 131072, "dtype": "bf16", "out": "f32", "history": 4000, "bias": 100},
        # histories as long as the vocabulary
        {"name": "logits_16x32000_long", "op": "logits", "rows": 16, "vocab": 32000, "dtype": "f16", "out": "f16", "history": 32768, "bias": 300},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _one(rng):
    op, dtype = rng.choice(["rope", "sdpa", "sdpa", "logits"]), rng.choice(["bf16", "f16", "f32"])
    if op == "logits":
        return {"op": op, "rows": _log(rng, 1, 256), "vocab": _log(rng, 1000, 131072), "dtype": dtype, "out": rng.choice([dtype, "f32"]),
                "history": _log(rng, 1, 32768), "bias": _log(rng, 1, 301) - 1}
    kv = rng.choice([1, 2, 3, 4, 8, 8, 16])
    heads = {"q_heads": kv * rng.choice([1, 2, 3, 4, 4, 8]), "kv_heads": kv}
    if op == "rope":
        d, tokens = rng.choice([32, 64, 80, 96, 128, 128, 256]), _log(rng, 1, 8192)
        rot = d if rng.random() < 0.6 else 2 * rng.randint(1, d // 2)
        return {"op": op, "tokens": tokens, **heads, "d": d, "rot": rot, "layout": rng.choice(["half", "interleaved"]),
                "scaling": rng.choice(["none", "linear", "base", "parts"]), "dtype": dtype, "store": rng.choice([0, tokens + rng.randint(1, 4096)]),
                "padded": rng.random() < 0.3, "inverse": rng.random() < 0.25}
    q_len = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 9, 512)])
    return {"op": op, "batch": _log(rng, 1, 128), "q_len": q_len, **heads, "d": rng.choice([32, 40, 64, 80, 96, 128, 128]),
            "prefix": _log(rng, 1, 65536), "own": q_len + _log(rng, 1, 2048) - 1, "page": rng.choice([0, 8, 16, 64]), "dtype": dtype}


def draw(rng):
    top = {op: [max(work(c)[k] for c in listed() if c["op"] == op) for k in ("bytes", "flops")] for op in ("rope", "sdpa", "logits")}
    while True:
        c = _one(rng)
        w = work(c)
        scores = c["batch"] * c["q_len"] * c["q_heads"] * (c["prefix"] + c["own"]) if c["op"] == "sdpa" else 0
        if w["bytes"] <= top[c["op"]][0] and w["flops"] <= top[c["op"]][1] and scores <= 1.5e8 and c.get("rows", 0) * c.get("history", 0) <= 1 << 20:
            return c


# ---- inputs ----


def _freqs(c):
    """Angular frequencies of a case's rotary pairs, in radians a position."""
    r, base, factor, length, low, high = c.rot, 10000.0, 8.0, 4096.0, 1.0, 4.0
    if c.scaling == "base" and r > 2:
        base *= factor ** (r / (r - 2))
    f = [base ** (-2.0 * i / r) for i in range(r // 2)]
    if c.scaling == "linear":
        f = [x / factor for x in f]
    if c.scaling == "parts":
        keep = [min(1.0, max(0.0, (length * x / (2 * math.pi) - low) / (high - low))) for x in f]
        f = [x * (g + (1 - g) / factor) for x, g in zip(f, keep)]
    return f


def _lengths(c):
    """Own lengths of a batch's sequences before they are shuffled: spread evenly up to the longest; a padding sequence in odd batches."""
    n = [c.q_len + (c.own - c.q_len) * (i + 1) // c.batch for i in range(c.batch)]
    if c.batch % 2 and c.batch > 2:
        n[0] = 0
    return n


def _ints(gen, lo, hi, shape):
    return torch.randint(lo, hi, shape, generator=gen, device=DEV, dtype=torch.int32)


def prepare(case, seed):
    c = types.SimpleNamespace(**case)
    gen = torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 23)

    def randn(*shape, dtype=None):
        return torch.randn(shape, generator=gen, device=DEV).to(dtype or TYPES[c.dtype])

    def shuffled(n):
        return torch.randperm(n, generator=gen, device=DEV).to(torch.int32)

    s = types.SimpleNamespace(c=c, call=None)
    if c.op == "rope":
        # the rows of one projection hold a token's queries, keys and values
        s.qkv = randn(c.tokens, (c.q_heads + 2 * c.kv_heads) * c.d)
        s.q = s.qkv[:, : c.q_heads * c.d].view(c.tokens, c.q_heads, c.d)
        s.k = s.qkv[:, c.q_heads * c.d : (c.q_heads + c.kv_heads) * c.d].view(c.tokens, c.kv_heads, c.d)
        s.v = s.qkv[:, (c.q_heads + c.kv_heads) * c.d :].view(c.tokens, c.kv_heads, c.d)
        start = _ints(gen, 0, 100000, (1,))
        s.positions = _ints(gen, 0, 131072, (c.tokens,)) if c.tokens <= 256 else start + torch.arange(c.tokens, device=DEV, dtype=torch.int32)
        s.rows = shuffled(c.store)[: c.tokens].contiguous() if c.store else None
        if c.padded and c.store:
            s.rows[-(-c.tokens * 7 // 8) :] = -1
        s.freqs = torch.tensor(_freqs(c), dtype=torch.float64, device=DEV)
        s.q_out = torch.empty((c.tokens, c.q_heads, c.d), dtype=TYPES[c.dtype], device=DEV)
        s.k_out = torch.zeros((c.store or c.tokens, c.kv_heads, c.d), dtype=TYPES[c.dtype], device=DEV)
        s.v_out = torch.zeros_like(s.k_out) if c.store else None
    elif c.op == "sdpa":
        n = torch.tensor(_lengths(c), dtype=torch.int32, device=DEV)
        s.lengths = n[shuffled(c.batch).long()].contiguous()
        s.q = randn(c.batch, c.q_len, c.q_heads, c.d) * 2
        s.pk, s.pv = randn(c.prefix, c.kv_heads, c.d), randn(c.prefix, c.kv_heads, c.d)
        per = -(-c.own // c.page) if c.page else 0  # pages a sequence
        rows = c.batch * (per * c.page if c.page else c.own)
        s.k, s.v = randn(rows, c.kv_heads, c.d), randn(rows, c.kv_heads, c.d)
        s.pages = shuffled(c.batch * per).view(c.batch, per).contiguous() if c.page else None
        s.out = torch.empty_like(s.q)
        s.lse = torch.empty((c.batch, c.q_len, c.q_heads), dtype=torch.float32, device=DEV)
        s.scale = 1 / math.sqrt(c.d)
    else:
        s.logits = (randn(c.rows, c.vocab, dtype=torch.float32) * 4).to(TYPES[c.dtype])
        s.tokens = _ints(gen, 0, c.vocab, (c.rows, c.history))
        s.tokens[:, ::3] %= max(1, c.vocab // 50)  # some tokens come often
        s.lengths = _ints(gen, (c.history + 1) // 2, c.history + 1, (c.rows,))
        s.prompt = (s.lengths.float() * torch.rand(c.rows, generator=gen, device=DEV)).to(torch.int32)
        s.repetition = 1 + torch.rand(c.rows, generator=gen, device=DEV)
        s.presence, s.frequency = torch.rand(c.rows, generator=gen, device=DEV), torch.rand(c.rows, generator=gen, device=DEV) * 0.1
        # each row's biases: ids of its own, spread over the vocabulary
        step = c.vocab // c.bias if c.bias else 1
        s.bias_ids = (_ints(gen, 0, step, (c.rows, c.bias)) + step * torch.arange(c.bias, device=DEV, dtype=torch.int32)).reshape(-1)
        s.bias_values = randn(c.rows * c.bias, dtype=torch.float32) * 5
        s.bias_offsets = torch.arange(c.rows + 1, device=DEV, dtype=torch.int32) * c.bias
        # the grammar's states, of which half the rows are in one, the others are free
        s.mask = torch.randint(-(1 << 31), 1 << 31, (max(1, c.rows // 2), -(-c.vocab // 32)), generator=gen, device=DEV).to(torch.int32)
        s.mask_rows = torch.where(torch.arange(c.rows, device=DEV) % 2 == 0, _ints(gen, 0, s.mask.shape[0], (c.rows,)), -1).to(torch.int32)
        s.out = torch.empty((c.rows, c.vocab), dtype=TYPES[c.out], device=DEV)
    return s


# ---- one pass ----


def run(s):
    if own:
        return _own(s)
    return {"rope": _rope, "sdpa": _sdpa, "logits": _logits}[s.c.op](s)


def _outputs(s):
    if s.c.op == "rope":
        return [s.q_out, s.k_out] + ([s.v_out] if s.c.store else [])
    return [s.out, s.lse] if s.c.op == "sdpa" else [s.out]


def _own(s):
    """The library's calls on the same buffers, on torch's current stream (whose inputs they read and whose work reads
    their outputs); a program keeps the block of arguments with its buffers."""
    global _backend
    import kurumi_amd as ku

    if _backend is None:
        _backend = ku.HipBackend()
    c = s.c
    if s.call is None:
        types_ = {"f32": ku.DType.F32, "bf16": ku.DType.BF16, "f16": ku.DType.F16}
        p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        if c.op == "rope":
            scaling = {"none": ku.ROPE_UNSCALED, "linear": ku.ROPE_LINEAR, "base": ku.ROPE_BASE, "parts": ku.ROPE_BY_PARTS}[c.scaling]
            args = ku.RopeArgs(
                dtype=types_[c.dtype], layout=ku.ROPE_HALF if c.layout == "half" else ku.ROPE_INTERLEAVED, inverse=int(c.inverse), scale=1.0,
                tokens=c.tokens, q_heads=c.q_heads, kv_heads=c.kv_heads, head_dim=c.d, rot_dim=c.rot, positions=p(s.positions),
                freqs=ku.rope_freqs(c.rot, 10000.0, scaling, factor=8.0, trained_len=4096.0, low=1.0, high=4.0),
                q=p(s.q), q_token_stride=s.q.stride(0), q_head_stride=s.q.stride(1), q_out=p(s.q_out), q_out_token_stride=s.q_out.stride(0),
                q_out_head_stride=s.q_out.stride(1), k=p(s.k), k_token_stride=s.k.stride(0), k_head_stride=s.k.stride(1), k_out=p(s.k_out),
                k_out_row_stride=s.k_out.stride(0), k_out_head_stride=s.k_out.stride(1))
            if c.store:
                args.v, args.v_token_stride, args.v_head_stride = p(s.v), s.v.stride(0), s.v.stride(1)
                args.v_out, args.v_out_row_stride, args.v_out_head_stride = p(s.v_out), s.v_out.stride(0), s.v_out.stride(1)
                args.rows, args.out_rows = p(s.rows), c.store
            else:
                args.out_rows = c.tokens
            s.call = (_backend.rope, args)
        elif c.op == "sdpa":
            s.call = (_backend.sdpa_prefix, ku.SdpaPrefixArgs(
                dtype=types_[c.dtype], scale=s.scale, batch=c.batch, q_len=c.q_len, q_heads=c.q_heads, kv_heads=c.kv_heads, head_dim=c.d,
                q=p(s.q), q_batch_stride=s.q.stride(0), q_token_stride=s.q.stride(1), q_head_stride=s.q.stride(2), out=p(s.out),
                out_batch_stride=s.out.stride(0), out_token_stride=s.out.stride(1), out_head_stride=s.out.stride(2), lse=p(s.lse),
                prefix_len=c.prefix, prefix_k=p(s.pk), prefix_v=p(s.pv), prefix_row_stride=s.pk.stride(0), prefix_head_stride=s.pk.stride(1),
                own_max=c.own, own_lens=p(s.lengths), own_k=p(s.k), own_v=p(s.v), own_row_stride=s.k.stride(0), own_head_stride=s.k.stride(1),
                own_rows=s.k.shape[0], own_seq_rows=0 if c.page else c.own, pages=p(s.pages), page_size=c.page,
                pages_per_seq=s.pages.shape[1] if c.page else 0))
        else:
            s.call = (_backend.logits_adjust, ku.LogitsArgs(
                dtype=types_[c.dtype], out_dtype=types_[c.out], rows=c.rows, vocab=c.vocab, logits=p(s.logits), logits_stride=s.logits.stride(0),
                out=p(s.out), out_stride=s.out.stride(0), history=c.history, tokens=p(s.tokens), tokens_stride=s.tokens.stride(0), lens=p(s.lengths),
                prompt_lens=p(s.prompt), repetition=p(s.repetition), presence=p(s.presence), frequency=p(s.frequency),
                bias_ids=p(s.bias_ids), bias_values=p(s.bias_values), bias_offsets=p(s.bias_offsets), bias_count=s.bias_ids.numel(), mask=p(s.mask),
                mask_rows=s.mask.shape[0], mask_stride=s.mask.stride(0), mask_index=p(s.mask_rows)))
    call, args = s.call
    # the handle by itself: torch.cuda.current_stream() makes an object around it, for 2.8 us
    call(args, torch._C._cuda_getCurrentRawStream(_outputs(s)[0].device.index) or NULL_STREAM)
    return _outputs(s)


def _rope(s):
    c, half = s.c, s.c.rot // 2
    turn = s.positions.double()[:, None] * s.freqs / (2 * math.pi)
    a = ((turn - turn.round()) * (2 * math.pi)).float()[:, None, :]
    cos, sin = a.cos(), -a.sin() if c.inverse else a.sin()

    def rotate(x):
        x = x.float()
        low, high = (x[..., :half], x[..., half : c.rot]) if c.layout == "half" else (x[..., 0 : c.rot : 2], x[..., 1 : c.rot : 2])
        y = (low * cos - high * sin, high * cos + low * sin)
        y = torch.cat(y, -1) if c.layout == "half" else torch.stack(y, -1).flatten(-2)
        return torch.cat((y, x[..., c.rot :]), -1).to(TYPES[c.dtype])

    s.q_out.copy_(rotate(s.q))
    if c.store:
        # a token without a row of the cache has row -1: it is left out by writing what is there already
        kept = (s.rows >= 0)[:, None, None]
        at = torch.where(s.rows >= 0, s.rows, s.rows[0]).long()
        k = rotate(s.k)
        s.k_out[at] = torch.where(kept, k, k[:1])
        s.v_out[at] = torch.where(kept, s.v, s.v[:1])
    else:
        s.k_out.copy_(rotate(s.k))
    return _outputs(s)


def _sdpa(s):
    c = s.c
    group = c.q_heads // c.kv_heads
    # [kv_heads, batch * q_len * group, d]: the queries of all sequences meet a shared key at once
    q = s.q.float().view(c.batch, c.q_len, c.kv_heads, group, c.d) * s.scale
    ps = torch.matmul(q.permute(2, 0, 1, 3, 4).reshape(c.kv_heads, -1, c.d), s.pk.float().permute(1, 2, 0).contiguous())
    j = torch.arange(c.own, device=DEV)
    at = s.pages.long()[:, j // c.page] * c.page + j % c.page if c.page else torch.arange(c.batch, device=DEV)[:, None] * c.own + j
    k, v = (x[at].float().permute(0, 2, 1, 3).contiguous() for x in (s.k, s.v))  # [batch, kv_heads, own, d]
    os_ = torch.matmul(q.permute(0, 2, 1, 3, 4).reshape(c.batch, c.kv_heads, -1, c.d), k.transpose(2, 3).contiguous())
    last = s.lengths[:, None] - (c.q_len - 1 - torch.arange(c.q_len, device=DEV))  # own keys that a query sees
    hidden = j >= last[:, :, None]
    os_ = os_.view(c.batch, c.kv_heads, c.q_len, group, c.own).masked_fill(hidden[:, None, :, None, :], -math.inf)
    ps = ps.view(c.kv_heads, c.batch, c.q_len * group, c.prefix)
    os_ = os_.permute(1, 0, 2, 3, 4).reshape(c.kv_heads, c.batch, c.q_len * group, c.own)
    top = torch.maximum(ps.amax(-1), os_.amax(-1))[..., None]
    ps, os_ = (ps - top).exp(), (os_ - top).exp()
    total = ps.sum(-1, keepdim=True) + os_.sum(-1, keepdim=True)
    o = torch.matmul(ps.view(c.kv_heads, -1, c.prefix), s.pv.float().permute(1, 0, 2).contiguous()).view(c.kv_heads, c.batch, -1, c.d)
    o = (o + torch.matmul(os_, v.permute(1, 0, 2, 3).contiguous())) / total
    shape = (c.kv_heads, c.batch, c.q_len, group)
    o = o.view(*shape, c.d).permute(1, 2, 0, 3, 4).reshape(s.q.shape).to(s.q.dtype)
    return [o, (top + total.log()).view(shape).permute(1, 2, 0, 3).reshape(s.lse.shape)]


def _logits(s):
    c = s.c
    x = s.logits.float()
    at = torch.arange(c.history, device=DEV)
    inside, new = at < s.lengths[:, None], at >= s.prompt[:, None]
    ids = s.tokens.long()
    seen = torch.zeros((c.rows, c.vocab), dtype=torch.int32, device=DEV).scatter_add_(1, ids, inside.int())
    count = torch.zeros((c.rows, c.vocab), dtype=torch.int32, device=DEV).scatter_add_(1, ids, (inside & new).int())
    r = s.repetition[:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - (s.frequency[:, None] * count + s.presence[:, None] * (count > 0))
    row = torch.arange(c.rows, device=DEV).repeat_interleave(c.bias)
    x.index_put_((row, s.bias_ids.long()), s.bias_values, accumulate=True)
    bits = (s.mask[:, :, None] >> torch.arange(32, device=DEV, dtype=torch.int32) & 1).view(s.mask.shape[0], -1)[:, : c.vocab]
    refused = (bits[s.mask_rows.clamp_min(0).long()] == 0) & (s.mask_rows >= 0)[:, None]
    return [x.masked_fill(refused, -math.inf).to(TYPES[c.out])]


# ---- what a pass cannot do without, and its results in 64 bits ----


def work(case):
    """Each input read once, each output written once; of a cache the rows that a pass reads or writes."""
    c = types.SimpleNamespace(**case)
    w = WIDTH[c.dtype]
    if c.op == "rope":
        stored = c.tokens - (c.tokens - -(-c.tokens * 7 // 8) if c.padded and c.store else 0)
        heads = 2 * c.q_heads * c.tokens + (4 if c.store else 2) * c.kv_heads * stored
        return {"bytes": w * c.d * heads + 4 * c.tokens * (2 if c.store else 1), "flops": 3 * c.rot * (c.q_heads * c.tokens + c.kv_heads * stored)}
    if c.op == "sdpa":
        n = _lengths(c)
        keys = sum(c.q_len * c.prefix + sum(max(0, m - i) for i in range(c.q_len)) for m in n)
        return {"bytes": w * (2 * c.batch * c.q_len * c.q_heads * c.d + 2 * c.kv_heads * c.d * (c.prefix + sum(n))) + 4 * c.batch * (c.q_len * c.q_heads + 1),
                "flops": 4 * c.d * c.q_heads * keys}
    return {"bytes": c.rows * (c.vocab * (w + WIDTH[c.out]) + 3 * c.history + 8 * c.bias + 24) + (c.rows + 1) // 2 * c.vocab // 8,
            "flops": 2 * c.rows * c.vocab}


def exact(case, seed):
    s = prepare(case, seed)
    c = s.c
    if c.op == "rope":
        i = torch.arange(c.rot // 2, device=DEV, dtype=torch.float64)
        base = 10000.0 * (8.0 ** (c.rot / (c.rot - 2)) if c.scaling == "base" and c.rot > 2 else 1.0)
        f = torch.exp(-2 * i / c.rot * math.log(base))
        if c.scaling == "linear":
            f = f / 8
        elif c.scaling == "parts":
            wave = 2 * math.pi / f
            f = torch.where(wave <= 4096 / 4, f, torch.where(wave >= 4096, f / 8, f / 8 + (f - f / 8) * (4096 / wave - 1) / 3))
        z = torch.polar(torch.ones_like(s.positions, dtype=torch.float64)[:, None] * torch.ones_like(f), s.positions.double()[:, None] * f)
        z = (z.conj() if c.inverse else z)[:, None, :]

        def turned(x):
            x = x.double()
            pairs = x[..., : c.rot].unflatten(-1, (2, -1)).transpose(-1, -2) if c.layout == "half" else x[..., : c.rot].unflatten(-1, (-1, 2))
            y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z)
            return torch.cat(((y.transpose(-1, -2) if c.layout == "half" else y).flatten(-2), x[..., c.rot :]), -1)

        if not c.store:
            return [turned(s.q), turned(s.k)]
        k, v = (torch.zeros(s.k_out.shape, dtype=torch.float64, device=DEV) for _ in range(2))
        there = s.rows >= 0
        k[s.rows[there].long()] = turned(s.k)[there]
        v[s.rows[there].long()] = s.v.double()[there]
        return [turned(s.q), k, v]
    if c.op == "sdpa":
        o, lse = torch.empty(s.q.shape, dtype=torch.float64, device=DEV), torch.empty(s.lse.shape, dtype=torch.float64, device=DEV)
        n, group = s.lengths.tolist(), c.q_heads // c.kv_heads
        if c.batch * c.kv_heads > 2048:
            return None
        for h in range(c.kv_heads):
            pk, pv = s.pk[:, h].double(), s.pv[:, h].double()
            for b in range(c.batch):
                if c.page:
                    rows = (s.pages[b].long()[:, None] * c.page + torch.arange(c.page, device=DEV)).reshape(-1)[: n[b]]
                else:
                    rows = b * c.own + torch.arange(n[b], device=DEV)
                k, v = torch.cat((pk, s.k[rows, h].double())), torch.cat((pv, s.v[rows, h].double()))
                q = s.q[b, :, h * group : (h + 1) * group].double().reshape(-1, c.d)
                x = (q @ k.T.contiguous()).view(c.q_len, group, -1) * s.scale
                ends = c.prefix + n[b] - c.q_len + 1 + torch.arange(c.q_len, device=DEV)
                gone = torch.arange(x.shape[-1], device=DEV) >= ends.clamp_min(c.prefix)[:, None]
                x = x.masked_fill(gone[:, None, :], -math.inf)
                o[b, :, h * group : (h + 1) * group] = (torch.softmax(x, -1).view(c.q_len * group, -1) @ v).view(c.q_len, group, c.d)
                lse[b, :, h * group : (h + 1) * group] = torch.logsumexp(x, -1)
        return [o, lse]
    y = s.logits.double()
    n, m = s.lengths.tolist(), s.prompt.tolist()
    for r in range(c.rows):
        t = s.tokens[r].long()
        count = torch.bincount(t[m[r] : n[r]], minlength=c.vocab).double()
        known = torch.bincount(t[: n[r]], minlength=c.vocab) > 0
        rep = s.repetition[r].double()
        y[r] = torch.where(known, y[r] * torch.where(y[r] > 0, 1 / rep, rep), y[r])
        y[r] -= s.frequency[r].double() * count + s.presence[r].double() * count.clamp(max=1)
        y[r, s.bias_ids.view(c.rows, -1)[r].long()] += s.bias_values.view(c.rows, -1)[r].double()
    words = s.mask.cpu().numpy().view("u1")
    allowed = torch.from_numpy(np.unpackbits(words, axis=1, bitorder="little")).to(DEV)[:, : c.vocab].bool()
    for r, at in enumerate(s.mask_rows.tolist()):
        if at >= 0:
            y[r, ~allowed[at]] = -math.inf
    return [y]
