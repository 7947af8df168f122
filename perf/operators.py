"""The 8-bit KV cache of a decode step and the rotary embedding in front of it: what is timed, and the plain forms.

Four operators that a serving step uses one after the other:

  rotary   rotary_embedding_positions  rotates q and k by their tokens' positions (both pair layouts, part of the head,
                                       frequencies scaled for long contexts)
  store    store_kvcache_q8            quantises new K/V rows into the paged 8-bit pool, one scale for each block and
                                       head: whole prompts ("prefill") or one token a sequence ("append")
  load     load_kvcache_q8             reads ranges of cached tokens back into contiguous rows of the model's type
  attn     paged_attention_q8          decode attention over the 8-bit pool, one query token a sequence

With ``own`` false ``run`` computes them with elementary torch operations in 32 bits (angles and quotients next to a
rounding border in 64); with ``own`` true it makes the package's calls.

The number format.  A block's scale for one head, over the block's tokens and the head's elements:
  int8   s = fl32(amax / 127), codes = round-half-even(x * fl32(1 / s))
  e4m3   s = 2^e with the smallest e for which amax <= 448 * s, codes = e4m3(x / s)
A scale below the smallest normal 32-bit number is 0 and its codes are 0.  An append into a block that already holds
tokens keeps the larger of the block's and the new token's scale; when that is the new token's, the codes already there
are rounded again: int8 codes q become round-half-even(q * fl32(s_old * fl32(1 / s_new))), e4m3 codes e4m3(q * s_old / s_new).
The first slot of a block starts from the new token alone.
"""
import math
import random
import types

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TINY = 2.0 ** -126      # smallest normal 32-bit number
LAYERS, LAYER = 2, 1    # the pools hold two layers, the second one is used: block and layer strides differ


# ---------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the tokens of one decode step, q and k as views of one fused projection; frequencies scaled by bands
        dict(name="rotary-decode", op="rotary", tokens=64, q_heads=32, kv_heads=8, head_dim=128, rotary_dim=128,
             interleaved=False, scaling="llama3", positions="decode", dtype="float16", fused=True),
        # a prefill batch of a model that pairs neighbours and rotates half of the head; odd token count
        dict(name="rotary-interleaved-part", op="rotary", tokens=4097, q_heads=64, kv_heads=8, head_dim=128,
             rotary_dim=64, interleaved=True, scaling="linear", positions="prefill", dtype="bfloat16", fused=False),
        # a large prefill batch (the prompt mix of the kv-prefill workload), contexts stretched by parts
        dict(name="rotary-prefill", op="rotary", tokens=49600, q_heads=32, kv_heads=8, head_dim=128, rotary_dim=128,
             interleaved=False, scaling="yarn", positions="prefill", dtype="float16", fused=True),
        # 64 prompts of up to 1536 tokens entering the cache at once
        dict(name="store-prefill", op="store", mode="prefill", code="int8", dtype="float16", batch=64, min_len=1,
             max_len=1536, kv_heads=8, head_dim=128, block_size=16, lens_seed=11),
        # the append of one decode step of the benchmark batch
        dict(name="store-append", op="store", mode="append", code="e4m3", dtype="float16", batch=256, min_len=1,
             max_len=1536, kv_heads=8, head_dim=128, block_size=16, lens_seed=12),
        # the append of three sequences: latency
        dict(name="store-append-small", op="store", mode="append", code="int8", dtype="bfloat16", batch=3, min_len=1,
             max_len=300, kv_heads=32, head_dim=128, block_size=16, lens_seed=13),
        # cached prefixes of a batch read back for a prefill attention that wants contiguous rows
        dict(name="load-prefixes", op="load", code="e4m3", dtype="bfloat16", batch=32, min_len=1, max_len=2048,
             kv_heads=8, head_dim=128, block_size=16, lens_seed=14, begins=True),
        # one short prefix: latency
        dict(name="load-small", op="load", code="int8", dtype="float16", batch=1, min_len=100, max_len=100,
             kv_heads=8, head_dim=128, block_size=16, lens_seed=15, begins=False),
        # few short sequences: latency
        dict(name="attn-small", op="attn", code="int8", dtype="float16", batch=8, min_len=1, max_len=2048, q_heads=32,
             kv_heads=8, head_dim=128, block_size=16, lens_seed=16),
        # the benchmark's grouped-query batch
        dict(name="attn-gqa", op="attn", code="int8", dtype="float16", batch=256, min_len=1, max_len=1536, q_heads=32,
             kv_heads=8, head_dim=128, block_size=16, lens_seed=17),
        # the benchmark's multi-head batch
        dict(name="attn-mha", op="attn", code="e4m3", dtype="bfloat16", batch=64, min_len=1, max_len=768, q_heads=32,
             kv_heads=32, head_dim=128, block_size=16, lens_seed=18),
        # a few long contexts, groups of eight
        dict(name="attn-long", op="attn", code="e4m3", dtype="float16", batch=8, min_len=8192, max_len=32768, q_heads=64,
             kv_heads=8, head_dim=128, block_size=16, lens_seed=19),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["rotary", "store", "load", "attn", "attn"])
    if op == "rotary":
        q_heads, kv_heads = rng.choice([(8, 8), (14, 2), (16, 16), (28, 4), (32, 8), (64, 8), (5, 1)])
        head_dim = rng.choice([64, 80, 112, 128, 128, 256])
        rotary_dim = head_dim if rng.random() < 0.6 else rng.choice([head_dim // 2, head_dim // 4, 3 * head_dim // 4])
        most = max(1, min(49600, 49600 * 40 * 128 // ((q_heads + kv_heads) * head_dim)))
        return dict(op="rotary", tokens=_log_int(rng, 1, most), q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim,
                    rotary_dim=rotary_dim - rotary_dim % 2, interleaved=rng.random() < 0.5,
                    scaling=rng.choice(["none", "linear", "ntk", "llama3", "yarn"]),
                    positions=rng.choice(["decode", "prefill"]),
                    dtype=rng.choice(["float16", "bfloat16"]), fused=rng.random() < 0.5)
    code, dtype = rng.choice(list(CODES)), rng.choice(["float16", "bfloat16"])
    kv_heads = rng.choice([1, 2, 4, 5, 8, 8, 32])
    lens_seed = rng.randrange(1 << 20)
    if op == "attn":
        group = rng.choice([1, 2, 4, 4, 5, 8, 16])
        head_dim = rng.choice([64, 128, 128, 128])
        room = 8 * 32768 * 8 * 128 // (kv_heads * head_dim)          # tokens, padded, that cost no more than attn-long
        batch = _log_int(rng, 1, 256)
        max_len = _log_int(rng, 1, max(1, min(32768, room // batch)))
        return dict(op="attn", code=code, dtype=dtype, batch=batch, min_len=rng.choice([1, max(1, max_len // 2)]),
                    max_len=max_len, q_heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim,
                    block_size=rng.choice([16, 16, 32]), lens_seed=lens_seed)
    head_dim = rng.choice([64, 80, 112, 128, 128, 256])
    block_size = rng.choice([8, 16, 16, 32])
    room = 64 * 1536 * 8 * 128 // (kv_heads * head_dim)
    batch = _log_int(rng, 1, 256)
    max_len = _log_int(rng, 1, max(1, min(4096, room // batch)))
    case = dict(op=op, code=code, dtype=dtype, batch=batch, min_len=rng.choice([1, max(1, max_len // 2)]),
                max_len=max_len, kv_heads=kv_heads, head_dim=head_dim, block_size=block_size, lens_seed=lens_seed)
    if op == "store":
        case["mode"] = rng.choice(["prefill", "append"])
    else:
        case["begins"] = rng.random() < 0.5
    return case


def _lengths(case):
    """The sequences' lengths: part of the case, the same for every seed."""
    r = random.Random(case["lens_seed"])
    return [r.randint(case["min_len"], case["max_len"]) for _ in range(case["batch"])]


def _ranges(case):
    """(first, behind last) cached token that a load reads, for each sequence."""
    r = random.Random(case["lens_seed"] + 1)
    return [(r.randint(0, n - 1) if case["begins"] else 0, n) for n in _lengths(case)]


def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "rotary":
        n = case["tokens"] * (case["q_heads"] + case["kv_heads"])
        # every element is read and written once; a pair takes four products and two sums; one sine and cosine for
        # each token and frequency
        return {"bytes": 2 * e * n * case["head_dim"] + 4 * case["tokens"],
                "flops": 3 * n * case["rotary_dim"] + 10 * case["tokens"] * case["rotary_dim"]}
    heads, dim, bs = case["kv_heads"], case["head_dim"], case["block_size"]
    lens = _lengths(case)
    if case["op"] == "attn":
        tokens, blocks = sum(lens), sum(-(-n // bs) for n in lens)
        rows = case["batch"] * case["q_heads"] * dim
        return {"bytes": 2 * heads * (tokens * dim + 4 * blocks) + 2 * e * rows + 4 * blocks,
                "flops": 4 * tokens * case["q_heads"] * dim}
    if case["op"] == "load":
        ranges = _ranges(case)
        tokens, blocks = sum(b - a for a, b in ranges), sum(-(-b // bs) - a // bs for a, b in ranges)
        return {"bytes": 2 * heads * (tokens * dim * (1 + e) + 4 * blocks) + 4 * blocks, "flops": 2 * heads * tokens * dim}
    # store: the new rows are read, their codes and scales written, and the touched blocks' tokens come back as values
    if case["mode"] == "prefill":
        new, back, blocks = sum(lens), sum(lens), sum(-(-n // bs) for n in lens)
    else:
        new, back, blocks = len(lens), sum((n - 1) % bs + 1 for n in lens), len(lens)
    return {"bytes": 2 * heads * (new * dim * (1 + e) + back * dim * e + 4 * blocks) + 4 * blocks,
            "flops": 2 * heads * dim * (3 * new + back)}


# --------------------------------------------------------------------------------------------------------- inputs
def _inv_freq(case):
    """Radians a position for each pair, in 64 bits: base 10000 (500000 where scaled by bands), scaled as the name says."""
    dim, kind = case["rotary_dim"], case["scaling"]
    factor, original = 8.0, 8192
    base = 500000.0 if kind == "llama3" else 10000.0
    if kind == "ntk":
        base *= factor ** (dim / max(dim - 2, 1))
    inv = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    turns = original * inv / (2 * math.pi)                      # turns over the original context
    if kind == "linear":
        inv = inv / factor
    elif kind == "llama3":                                      # keep above 4 turns, divide below 1, blend between
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        inv = inv * keep + inv / factor * (1 - keep)
    elif kind == "yarn":                                        # keep above 32 turns, divide below 1, ramp by index
        index = [dim * math.log(original / (n * 2 * math.pi)) / (2 * math.log(base)) for n in (32.0, 1.0)]
        low, high = max(math.floor(index[0]), 0), min(math.ceil(index[1]), dim - 1)
        ramp = ((torch.arange(dim // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
        inv = inv / factor * ramp + inv * (1 - ramp)
    return inv, (0.1 * math.log(factor) + 1.0 if kind == "yarn" else 1.0)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)

    s = types.SimpleNamespace(case=dict(case), op=case["op"])
    if case["op"] == "rotary":
        t, hq, hkv, d = case["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"]
        if case["fused"]:       # q | k | v of a token side by side, as one projection leaves them
            qkv = normal(t, hq + 2 * hkv, d).to(dtype)
            s.q, s.k = qkv[:, :hq], qkv[:, hq:hq + hkv]
        else:
            s.q, s.k = normal(t, hq, d).to(dtype), normal(t, hkv, d).to(dtype)
        s.q_out, s.k_out = torch.empty((t, hq, d), dtype=dtype, device="cuda"), torch.empty((t, hkv, d), dtype=dtype, device="cuda")
        if case["positions"] == "decode":
            s.positions = torch.randint(0, 65536, (t,), generator=gen, device="cuda", dtype=torch.int32)
        else:                   # prompts of one length behind a cached prefix each
            at = torch.arange(t, device="cuda", dtype=torch.int32)
            first = torch.randint(0, 4096, (t // 1000 + 1,), generator=gen, device="cuda", dtype=torch.int32)
            s.positions = at % 1000 + first[(at // 1000).long()]
        inv, s.attention_scale = _inv_freq(case)
        s.inv_freq = inv.cuda()
        return s

    lens, bs, hkv, d = _lengths(case), case["block_size"], case["kv_heads"], case["head_dim"]
    batch = len(lens)
    need = [-(-n // bs) for n in lens]
    blocks, width = sum(need) + 8, max(need) + 1
    rows = batch + 3            # block-table rows; the batch uses some of them in any order
    r = random.Random(int(seed))
    order = r.sample(range(rows), batch)
    ids = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32)
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    need_t = torch.tensor(need, dtype=torch.int64, device="cuda")
    s.seq_ids = torch.tensor(order, dtype=torch.int32, device="cuda")
    s.block_table = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
    col = torch.arange(width, device="cuda")[None]
    used = col < need_t[:, None]
    slot = (torch.cumsum(need_t, 0) - need_t)[:, None] + col
    s.block_table[s.seq_ids.long()] = torch.where(used, ids[slot.clamp(max=blocks - 1)], -1)
    # a pool in use: normal values whose extremes sit at the top of the code range, and every block's own scale
    shape = (blocks, LAYERS, hkv)
    code = CODES[case["code"]]
    for name in ("k", "v"):
        if case["code"] == "int8":
            codes = (normal(*shape, bs, d) * 36.0).round_().clamp_(-127, 127).to(code)
            scale = (normal(*shape).abs() * 0.005 + 0.02)
        else:
            codes = (normal(*shape, bs, d) * 110.0).clamp_(-448, 448).to(code)
            scale = torch.exp2(torch.randint(-8, -5, shape, generator=gen, device="cuda").float())
        setattr(s, name + "_cache", codes)
        setattr(s, name + "_scale", scale)
    s.model_config = types.SimpleNamespace(num_layers=LAYERS, num_q_heads=case.get("q_heads", hkv), num_kv_heads=hkv, head_dim=d)
    s.engine_config = types.SimpleNamespace(block_size=bs, max_blocks_per_seq=width)
    prefill = case["op"] == "store" and case["mode"] == "prefill"
    starts = torch.cumsum(lens_t, 0, dtype=torch.int32) - lens_t
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    s.infer_state = types.SimpleNamespace(
        batch_size=batch, num_tokens=sum(lens) if prefill else batch, seq_ids=s.seq_ids, softmax_scale=d ** -0.5,
        num_prefill_seqs=batch if prefill else 0, num_prefill_tokens=sum(lens) if prefill else 0,
        prefill_seq_start_locs=starts if prefill else none, prefill_seq_lens=lens_t if prefill else none,
        max_prefill_len=max(lens) if prefill else 0, num_decoding_seqs=0 if prefill else batch,
        decoding_seq_lens=none if prefill else lens_t, max_decoding_len=0 if prefill else max(lens),
        num_blocks_org=blocks, kv_cache_new_block_size=0, ignore_kvcache=False)
    s.lens, s.width = lens_t, max(need)
    if case["op"] == "attn":
        s.q = normal(batch, case["q_heads"], d).to(dtype)
        s.o = torch.empty((batch, case["q_heads"] * d), dtype=dtype, device="cuda")
        return s
    if case["op"] == "load":
        begins, ends = zip(*_ranges(case))
    elif prefill:
        begins, ends = [0] * batch, lens
    else:                       # an append comes back as its sequences' last blocks
        begins, ends = [(n - 1) // bs * bs for n in lens], lens
    s.max_len = max(b - a for a, b in zip(begins, ends))
    s.begins = torch.tensor(begins, dtype=torch.int32, device="cuda")
    s.ends = torch.tensor(ends, dtype=torch.int32, device="cuda")
    count = s.ends - s.begins
    s.start_locs = torch.cumsum(count, 0, dtype=torch.int32) - count
    s.back = sum(b - a for a, b in zip(begins, ends))
    s.k_rows = torch.empty((s.back, hkv, d), dtype=dtype, device="cuda")
    s.v_rows = torch.empty_like(s.k_rows)
    if case["op"] == "store":
        n = sum(lens) if prefill else batch
        # tokens of unequal size, so that appended ones raise some blocks' scales
        size = torch.exp(normal(n, 1, 1) * 0.3)
        s.k, s.v = (normal(n, hkv, d) * size).to(dtype), (normal(n, hkv, d) * size).to(dtype)
    return s


# ---------------------------------------------------------------------------------------------------- plain forms
def _rotary_plain(s):
    """y = x rotated: pairs (a, b) become (a cos - b sin, a sin + b cos) at the angle position * inv_freq."""
    angle = s.positions.double()[:, None] * s.inv_freq[None]
    cos = (angle.cos() * s.attention_scale).float()[:, None]
    sin = (angle.sin() * s.attention_scale).float()[:, None]
    rd, half = s.case["rotary_dim"], s.case["rotary_dim"] // 2

    def rotate(x, out):
        y = x.float()
        a, b = (y[..., 0:rd:2], y[..., 1:rd:2]) if s.case["interleaved"] else (y[..., :half], y[..., half:rd])
        c, d = a * cos - b * sin, a * sin + b * cos
        turned = torch.stack((c, d), -1).flatten(-2) if s.case["interleaved"] else torch.cat((c, d), -1)
        out.copy_(torch.cat((turned, y[..., rd:]), -1))
        return out

    return rotate(s.q, s.q_out), rotate(s.k, s.k_out)


def _scale_plain(amax, code):
    """The scale that holds values of up to `amax` (32 bits)."""
    if code == "int8":
        scale = (amax.double() / 127.0).float()
    else:
        part, exponent = torch.frexp(amax)                      # amax = part * 2^exponent, part in [0.5, 1)
        scale = torch.exp2((exponent - 9 + (part > 0.875)).double()).float()
    return torch.where(scale < TINY, 0.0, scale)


def _inverse_plain(scale):
    return torch.where(scale > 0, (1.0 / scale.double()).float(), 0.0)


def _quantise_plain(x, inverse, code):
    exact = x.double() * inverse.double()
    return exact.round().to(torch.int8) if code == "int8" else exact.float().to(torch.float8_e4m3fn)


def _prefill_plain(s):
    code, bs = s.case["code"], s.case["block_size"]
    count = s.lens.long()
    seq = torch.repeat_interleave(torch.arange(len(count), device="cuda"), count, output_size=s.k.shape[0])
    pos = torch.arange(s.k.shape[0], device="cuda") - (torch.cumsum(count, 0) - count)[seq]
    block = s.block_table[s.seq_ids.long()[seq], pos // bs].long()
    for x, cache, scale in ((s.k, s.k_cache, s.k_scale), (s.v, s.v_cache, s.v_scale)):
        y = x.float()
        peak = torch.full(scale[:, LAYER].shape, -1.0, device="cuda")
        peak.scatter_reduce_(0, block[:, None].expand(-1, y.shape[1]), y.abs().amax(-1), "amax")
        new = torch.where(peak >= 0, _scale_plain(peak.clamp(min=0), code), scale[:, LAYER])
        scale[:, LAYER] = new
        cache[:, LAYER].view(torch.int8)[block, :, pos % bs] = _quantise_plain(y, _inverse_plain(new)[block][..., None], code).view(torch.int8)


def _append_plain(s):
    code, bs = s.case["code"], s.case["block_size"]
    pos = s.lens.long() - 1
    block, slot = s.block_table[s.seq_ids.long(), pos // bs].long(), pos % bs
    held = (torch.arange(bs, device="cuda")[None] < slot[:, None])[:, None, :, None]
    here = (torch.arange(bs, device="cuda")[None] == slot[:, None])[:, None, :, None]
    for x, cache, scale in ((s.k, s.k_cache, s.k_scale), (s.v, s.v_cache, s.v_scale)):
        y = x.float()
        old = scale[block, LAYER]
        mine = _scale_plain(y.abs().amax(-1), code)
        new = torch.where((slot > 0)[:, None], torch.maximum(old, mine), mine)
        inverse = _inverse_plain(new)
        codes = cache[:, LAYER].view(torch.int8)[block].view(CODES[code])
        ratio = (old * inverse)[..., None, None]
        again = torch.where(held & (new > old)[..., None, None], _quantise_plain(codes.float(), ratio, code).float(), codes.float())
        fresh = _quantise_plain(y, inverse[..., None], code).float()[:, :, None]
        cache[:, LAYER].view(torch.int8)[block] = torch.where(here, fresh, again).to(CODES[code]).view(torch.int8)
        scale[block, LAYER] = new


def _load_plain(s):
    bs = s.case["block_size"]
    count = (s.ends - s.begins).long()
    seq = torch.repeat_interleave(torch.arange(len(count), device="cuda"), count, output_size=s.back)
    pos = torch.arange(s.back, device="cuda") - s.start_locs.long()[seq] + s.begins.long()[seq]
    block = s.block_table[s.seq_ids.long()[seq], pos // bs].long()
    for out, cache, scale in ((s.k_rows, s.k_cache, s.k_scale), (s.v_rows, s.v_cache, s.v_scale)):
        codes = cache[:, LAYER].view(torch.int8)[block, :, pos % bs].view(cache.dtype).float()
        out.copy_(codes * scale[block, LAYER][..., None])


def _attn_plain(s):
    bs, hkv, d = s.case["block_size"], s.case["kv_heads"], s.case["head_dim"]
    batch, group = s.case["batch"], s.case["q_heads"] // s.case["kv_heads"]
    block = s.block_table[s.seq_ids.long(), :s.width].long().clamp(min=0)

    def values(cache, scale):       # [batch, head, token, dim], padded to the longest sequence
        x = cache[:, LAYER].view(torch.int8)[block].view(cache.dtype).float() * scale[block, LAYER][..., None, None]
        return x.transpose(1, 2).reshape(batch, hkv, s.width * bs, d)

    q = s.q.float().view(batch, hkv, group, d)
    score = torch.matmul(q, values(s.k_cache, s.k_scale).transpose(-1, -2)) * s.infer_state.softmax_scale
    score.masked_fill_(torch.arange(s.width * bs, device="cuda") >= s.lens[:, None, None, None], -math.inf)
    weight = torch.exp(score - score.amax(-1, keepdim=True))
    weight /= weight.sum(-1, keepdim=True)
    s.o.copy_(torch.matmul(weight, values(s.v_cache, s.v_scale)).reshape(batch, -1))
    return s.o


def run(s):
    if own:
        import morphserve_b200 as mk

        pool = (s.k_cache, s.v_cache, s.k_scale, s.v_scale, [], [], [], []) if s.op != "rotary" else ()
        if s.op == "rotary":
            mk.rotary_embedding_positions(s.q, s.k, s.positions, s.inv_freq, interleaved=s.case["interleaved"],
                                          attention_scale=s.attention_scale, q_out=s.q_out, k_out=s.k_out)
            return s.q_out, s.k_out
        if s.op == "attn":
            mk.paged_attention_q8(s.q, *pool, s.block_table, s.model_config, s.engine_config, s.infer_state, LAYER, s.o)
            return s.o
        if s.op == "store":
            mk.store_kvcache_q8(s.k, s.v, *pool, s.block_table, s.model_config, s.engine_config, s.infer_state, LAYER)
        mk.load_kvcache_q8(s.k_rows, s.v_rows, *pool, s.block_table, s.model_config, s.engine_config, s.seq_ids,
                           s.begins, s.ends, s.start_locs, s.max_len, LAYER)
    elif s.op == "rotary":
        return _rotary_plain(s)
    elif s.op == "attn":
        return _attn_plain(s)
    else:
        if s.op == "store":
            (_prefill_plain if s.case["mode"] == "prefill" else _append_plain)(s)
        _load_plain(s)
    return (s.k_rows, s.v_rows, s.k_scale, s.v_scale) if s.op == "store" else (s.k_rows, s.v_rows)


# -------------------------------------------------------------------------------------------------- in 64 bits
def _exact_rotary(s):
    turn = torch.polar(torch.full((), s.attention_scale, dtype=torch.float64, device="cuda"),
                       s.positions.double().unsqueeze(1) * s.inv_freq).unsqueeze(1)
    n = s.inv_freq.numel()

    def rotated(x):
        y = x.double()
        first = slice(0, 2 * n, 2) if s.case["interleaved"] else slice(0, n)
        second = slice(1, 2 * n, 2) if s.case["interleaved"] else slice(n, 2 * n)
        z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn
        y = y.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    return rotated(s.q), rotated(s.k)


def _exact_scale(peak, code):
    """peak: 64-bit.  The stored (32-bit) scale, as 64-bit numbers."""
    if code == "int8":
        scale = (peak / 127).float().double()
    else:
        scale = 2.0 ** torch.ceil(torch.log2(peak.clamp(min=2.0 ** -300)) - math.log2(448.0))
        scale = torch.where(peak > 448 * scale, 2 * scale, torch.where(peak <= 224 * scale, scale / 2, scale))
    return torch.where(scale < TINY, 0.0, scale)


def _exact_codes(x, inverse, code):
    y = x * inverse
    if code == "int8":
        return torch.round(y)
    step = 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)     # e4m3: three bits behind the first
    return torch.round(y / step) * step


def _exact_inverse(scale):
    return torch.where(scale > 0, (1.0 / scale).float().double(), 0.0)


def exact(case, seed):
    s = prepare(case, seed)
    if s.op == "rotary":
        return _exact_rotary(s)
    bs, code, hkv = case["block_size"], case["code"], case["kv_heads"]
    lens = _lengths(case)
    table = s.block_table[s.seq_ids.long()].long()
    k, v = (c[:, LAYER].double() for c in (s.k_cache, s.v_cache)) if s.op != "attn" else (None, None)
    ks, vs = (c[:, LAYER].double() for c in (s.k_scale, s.v_scale))
    if s.op == "attn":
        out = torch.empty((case["batch"], case["q_heads"], case["head_dim"]), dtype=torch.float64, device="cuda")
        for i, n in enumerate(lens):
            b = table[i, :-(-n // bs)]
            keys, vals = ((c[b, LAYER].double() * t[b][..., None, None]).permute(1, 0, 2, 3).flatten(1, 2)[:, :n]
                          for c, t in ((s.k_cache, ks), (s.v_cache, vs)))
            q = s.q[i].double().view(hkv, -1, case["head_dim"])
            p = torch.softmax(q @ keys.mT * s.infer_state.softmax_scale, -1)
            out[i] = (p @ vals).flatten(0, 1)
        return out.view(case["batch"], -1)
    if s.op == "store" and case["mode"] == "prefill":
        at = 0
        for i, n in enumerate(lens):
            b = table[i, :-(-n // bs)]
            for x, cache, scale in ((s.k, k, ks), (s.v, v, vs)):
                y = torch.zeros((len(b) * bs, hkv, case["head_dim"]), dtype=torch.float64, device="cuda")
                y[:n] = x[at:at + n].double()
                y = y.view(len(b), bs, hkv, -1).transpose(1, 2)
                scale[b] = _exact_scale(y.abs().amax((-1, -2)), code)
                new = _exact_codes(y, _exact_inverse(scale[b])[..., None, None], code)
                last = n - (len(b) - 1) * bs
                cache[b[:-1]] = new[:-1]
                cache[b[-1], :, :last] = new[-1, :, :last]
            at += n
    elif s.op == "store":
        for i, n in enumerate(lens):
            b, j = table[i, (n - 1) // bs], (n - 1) % bs
            for x, cache, scale in ((s.k, k, ks), (s.v, v, vs)):
                y = x[i].double()
                mine, was = _exact_scale(y.abs().amax(-1), code), scale[b].clone()
                scale[b] = torch.maximum(mine, was) if j else mine
                inverse = _exact_inverse(scale[b])
                ratio = (was * inverse).float().double()
                again = _exact_codes(cache[b, :, :j], ratio[:, None, None], code)
                cache[b, :, :j] = torch.where((scale[b] > was)[:, None, None], again, cache[b, :, :j])
                cache[b, :, j] = _exact_codes(y, inverse[:, None], code)
    rows = [[], []]
    for i, (first, behind) in enumerate(zip(s.begins.tolist(), s.ends.tolist())):
        b = table[i, first // bs:-(-behind // bs)]
        for out, cache, scale in ((rows[0], k, ks), (rows[1], v, vs)):
            x = (cache[b] * scale[b][..., None, None]).transpose(1, 2).flatten(0, 1)
            out.append(x[first - first // bs * bs:][:behind - first])
    back = torch.cat(rows[0]), torch.cat(rows[1])
    if s.op == "load":
        return back
    whole = [c.double() for c in (s.k_scale, s.v_scale)]
    whole[0][:, LAYER], whole[1][:, LAYER] = ks, vs
    return back + tuple(whole)
