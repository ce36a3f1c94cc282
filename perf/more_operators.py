"""Operators around a paged KV cache that is held in 8 bits, as workloads: inputs, a plain form
in elementary torch operations, a 64-bit form from the definitions, and the calls a user makes.

Four operators, the steps of a decode or a prompt over such a cache:

* ``norm_rotary``: an RMSNorm of every head of Q and K and their rotary positions;
* ``append``: the same on the way into the cache, K and V quantised to e4m3 as they are
  written, with a power of two as the scale of each block of tokens and head; and the blocks
  that were written read back;
* ``read``: a cached stretch of every sequence as dense rows of 16 bits;
* ``attention``: a tree of drafted tokens per sequence over the 8-bit cache.

``run`` computes the plain form, or with ``own`` set calls the framework's operators.
"""
import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
SIZES = {"bf16": 2, "f32": 4}
EPS = 1e-5
THETA = 5e5
LOWEST, HIGHEST = -40, 40  # exponents of a scale
LARGEST = 448.0            # of e4m3


# --------------------------------------------------------------------------
# Cases
# --------------------------------------------------------------------------

def _named(name, **case):
    return dict(case, name=name) if name else case


def _norm_rotary(rows, hq, hkv, hd, rotary_dim, pairs, max_pos, dtype, name=None):
    return _named(name, op="norm_rotary", rows=rows, hq=hq, hkv=hkv, hd=hd, rotary_dim=rotary_dim, pairs=pairs,
                  max_pos=max_pos, dtype=dtype)


def _append(batch, tokens, ctx, tree, norm, hq, hkv, hd, rotary_dim, pairs, page, block, dtype, name=None):
    return _named(name, op="append", batch=batch, tokens=tokens, ctx=ctx, tree=tree, norm=norm, hq=hq, hkv=hkv, hd=hd,
                  rotary_dim=rotary_dim, pairs=pairs, page=page, block=block, dtype=dtype)


def _read(batch, lo, hi, hkv, hd, page, block, dtype, name=None):
    return _named(name, op="read", batch=batch, lo=lo, hi=hi, hkv=hkv, hd=hd, page=page, block=block, dtype=dtype)


def _attention(batch, ctx_lo, ctx_hi, tokens, ragged, hq, hkv, hd, page, block, dtype, name=None):
    return _named(name, op="attention", batch=batch, ctx_lo=ctx_lo, ctx_hi=ctx_hi, tokens=tokens, ragged=ragged, hq=hq,
                  hkv=hkv, hd=hd, page=page, block=block, dtype=dtype)


def listed():
    return [
        # one decode step of 64 sequences at the Llama-3-8B shape: latency counts
        _norm_rotary(64, 32, 8, 128, 128, "half", 8192, "bf16", "norm-rotary-decode"),
        # a prompt batch at the 70B shape
        _norm_rotary(16384, 64, 8, 128, 128, "half", 32768, "bf16", "norm-rotary-prompt"),
        # the tinyllama shape in 32 bits, interleaved pairs on half of each head, an odd number of rows
        _norm_rotary(1001, 6, 6, 48, 24, "interleaved", 4096, "f32", "norm-rotary-f32"),
        # one new token of each of 64 sequences, normed and rotated on the way
        _append(64, 1, 500, False, True, 32, 8, 128, 128, "half", 16, 16, "bf16", "append-decode"),
        # four prompts of 8192 tokens at the 70B shape, scales for 64 tokens
        _append(4, 8192, 0, False, True, 64, 8, 128, 128, "half", 64, 64, "bf16", "append-prompt"),
        # trees of 25 drafted tokens at the tinyllama shape, pages that are no power of two, no norm
        _append(8, 25, 100, True, False, 6, 6, 48, 48, "half", 24, 8, "f32", "append-tree-f32"),
        # one short prefix taken out of the cache
        _read(1, 300, 300, 8, 128, 16, 16, "bf16", "read-one"),
        # cached prefixes of 16 sequences, handed on in 16 bits
        _read(16, 1000, 8192, 8, 128, 64, 64, "bf16", "read-batch"),
        # one user's sequence: 12 drafted tokens behind 8000 cached ones
        _attention(1, 8000, 8000, 12, False, 32, 8, 128, 16, 16, "bf16", "attention-one"),
        # a serving batch of uneven sequences, up to 8 drafted tokens each
        _attention(64, 1, 8192, 8, True, 32, 8, 128, 16, 16, "bf16", "attention-batch"),
        # wide trees over long contexts at the 70B shape: products count as much as bytes
        _attention(16, 4096, 8192, 64, False, 64, 8, 128, 64, 64, "bf16", "attention-wide"),
        # the tinyllama shape in 32 bits
        _attention(32, 0, 230, 25, True, 6, 6, 48, 16, 4, "f32", "attention-f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_rotary", "append", "append", "read", "attention", "attention", "attention"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    hd = rng.choice([48, 64, 128, 128, 256])
    hkv = rng.choice([1, 2, 6, 8])
    hq = hkv * rng.choice([1, 2, 4, 7, 8])
    pairs = rng.choice(["half", "interleaved"])
    part = rng.choice([hd, hd, hd // 2, 24])
    page = rng.choice([8, 16, 24, 32, 64, 100, 128, 256])
    block = rng.choice([n for n in (1, 4, 8, 16, 32, 64, page, page) if page % n == 0])
    if op == "norm_rotary":
        rows = max(1, min(_log(rng, 1, 16384), 16384 * 72 * 128 * 2 // ((hq + hkv) * hd * SIZES[dtype])))
        return _norm_rotary(rows, hq, hkv, hd, part, pairs, _log(rng, max(64, rows // 4), 131072), dtype)
    if op == "append":
        tree = rng.random() < 0.4
        tokens = rng.randint(1, 64) if tree else _log(rng, 1, 4096)
        batch = max(1, min(_log(rng, 1, 64), 16384 // tokens))
        return _append(batch, tokens, _log(rng, 1, 2000), tree, rng.random() < 0.5, hq, hkv, hd, part, pairs, page, block,
                       dtype)
    if op == "read":
        hi = _log(rng, 1, 8192)
        batch = max(1, min(_log(rng, 1, 64), 16 * 4096 * 8 * 128 // (hi * hkv * hd)))
        return _read(batch, rng.choice([0, hi // 2, hi]), hi, hkv, hd, page, block, dtype)
    hi = _log(rng, 16, 8192)
    if dtype == "f32":
        hi, tokens = min(hi, 2048), rng.randint(1, 25)
    else:
        tokens = _log(rng, 1, 64)
    # no more products than the largest listed case, and no more cached values
    room = min(16 * 6144 * 64 * 64 * 128 // (hi * tokens * hq * hd), 64 * 4096 * 8 * 128 // (hi * hkv * hd))
    if dtype == "f32":
        room //= 16
    batch = max(1, min(_log(rng, 1, 64), room))
    return _attention(batch, rng.choice([0, hi // 2, hi]), hi, tokens, rng.random() < 0.6, hq, hkv, hd, page, block, dtype)


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------

def _frequencies(dim):
    """The inverse frequency of each pair, in 64 bits."""
    return THETA ** (-2.0 * torch.arange(dim // 2, dtype=torch.float64) / dim)


def _table(max_pos, dim):
    """[max_pos][dim / 2][2] of (cos, sin), from 64-bit angles, as a server keeps it."""
    a = torch.arange(max_pos, dtype=torch.float64, device=DEVICE)[:, None] * _frequencies(dim).to(DEVICE)[None, :]
    return torch.stack([torch.cos(a), torch.sin(a)], dim=-1).float()


def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32) * scale).to(dtype)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _starts(counts):
    return [0] + np.cumsum(counts, dtype=np.int64).tolist()


def _pages(rng, lens, page):
    """A page table [batch][most pages of a sequence] of distinct pages in random order."""
    need = [-(-n // page) for n in lens]
    ids = list(range(sum(need) + 3))
    rng.shuffle(ids)
    width = max(max(need), 1)
    table, at = [], 0
    for n in need:
        table.append(ids[at:at + n] + [0] * (width - n))
        at += n
    return table, len(ids)


def _trees(rng, sizes):
    """A random parent (an earlier node, or -1: the context) for every node of every tree."""
    return [[rng.randint(max(-1, j - 6), j - 1) for j in range(n)] for n in sizes]


def _lens(case):
    """(context length, drafted tokens) of each sequence: part of the case, whatever the seed."""
    rng = random.Random("%d %d %d %d" % (case["batch"], case["ctx_lo"], case["ctx_hi"], case["tokens"]))
    out = []
    for _ in range(case["batch"]):
        n = rng.randint(1, case["tokens"]) if case["ragged"] else case["tokens"]
        out.append((rng.randint(case["ctx_lo"], case["ctx_hi"]), n))
    return out


def _read_lens(case):
    """(first slot, slots) of each sequence: part of the case, whatever the seed."""
    rng = random.Random("%d %d %d" % (case["batch"], case["lo"], case["hi"]))
    out = []
    for _ in range(case["batch"]):
        n = rng.randint(max(1, case["lo"]), case["hi"])
        first = rng.choice([0, rng.randint(0, n - 1)])
        out.append((first, n - first))
    return out


def _append_ctx(case):
    rng = random.Random("%d %d %d" % (case["batch"], case["tokens"], case["ctx"]))
    return [case["ctx"] - rng.randint(0, case["ctx"] // 2) for _ in range(case["batch"])]


def _masks(parents):
    """Ancestors-and-self bits of every node, 64 to a word."""
    rows, words = [], 1
    for tree in parents:
        words = max(words, -(-len(tree) // 64))
    for tree in parents:
        bits = []
        for j, p in enumerate(tree):
            bits.append((1 << j) | (bits[p] if p >= 0 else 0))
        rows += bits
    signed = lambda w: w - (1 << 64) if w >= 1 << 63 else w  # noqa: E731
    return torch.tensor([[signed((b >> (64 * w)) & ((1 << 64) - 1)) for w in range(words)] for b in rows],
                        dtype=torch.int64, device=DEVICE)


def _cache(g, s, case, count):
    """Pages as earlier steps left them: e4m3 values, and for each block of tokens and head a
    power of two near 2^-7, so that K and V are about as large as a normed head's."""
    for name in ("k", "v"):
        values = _randn(g, count, case["hkv"], case["page"], case["hd"], scale=100.0).clamp_(-LARGEST, LARGEST)
        s[name + "_pages"] = values.to(torch.float8_e4m3fn)
        exponents = torch.randint(-8, -5, (count, case["hkv"], case["page"] // case["block"]), generator=g, device=DEVICE)
        s[name + "_scales"] = (exponents + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _handle(s, case):
    from baremetalinferenceengine_b200 import ops

    return ops.PagedKV8(s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"], s["page_table"])


def _rope_table(max_pos, dim):
    from baremetalinferenceengine_b200 import ops

    return ops.RopeTable(max_pos, dim, THETA, DEVICE)


def prepare(case, seed):
    g, rng, dt, hd = _generator(seed), random.Random(seed), DTYPES[case["dtype"]], case["hd"]
    s = {"case": case}
    if case["op"] in ("norm_rotary", "append"):
        rows = case["rows"] if case["op"] == "norm_rotary" else case["batch"] * case["tokens"]
        qkv = _randn(g, rows, case["hq"] + 2 * case["hkv"], hd, dtype=dt)  # one projection's output, side by side
        s["q"], s["k"], s["v"] = qkv.split([case["hq"], case["hkv"], case["hkv"]], 1)
        s["q_out"] = torch.empty(rows, case["hq"], hd, dtype=dt, device=DEVICE)
        norm = case.get("norm", True)
        s["q_weight"], s["k_weight"] = ((1.0 + _randn(g, hd, scale=0.2)).to(dt) if norm else None for _ in range(2))
    if case["op"] == "norm_rotary":
        s["positions"] = torch.randint(0, case["max_pos"], (rows,), generator=g, device=DEVICE, dtype=torch.int32)
        s["k_out"] = torch.empty(rows, case["hkv"], hd, dtype=dt, device=DEVICE)
        s["table"] = (_rope_table if own else _table)(case["max_pos"], case["rotary_dim"])
        return s
    if case["op"] == "append":
        batch, n, block = case["batch"], case["tokens"], case["block"]
        ctx = _append_ctx(case)
        rng.shuffle(ctx)
        depth = []
        for tree in _trees(rng, [n] * batch) if case["tree"] else [range(-1, n - 1)] * batch:
            d = []
            for p in tree:
                d.append(d[p] + 1 if p >= 0 else 0)
            depth.append(d)
        s["positions"] = _i32([c + x for c, d in zip(ctx, depth) for x in d])
        s["ctx_lens"], s["q_starts"] = _i32(ctx), _i32(_starts([n] * batch))
        first = [c // block * block for c in ctx]  # the blocks that the new tokens meet, from their beginnings
        s["first"], s["read_starts"] = _i32(first), _i32(_starts([c + n - f for c, f in zip(ctx, first)]))
        s["read_rows"], s["read_most"] = (f([c + n - f0 for c, f0 in zip(ctx, first)]) for f in (sum, max))
        table, count = _pages(rng, [c + n for c in ctx], case["page"])
        s["page_table"] = _i32(table)
        _cache(g, s, case, count)
        s["table"] = (_rope_table if own else _table)(case["ctx"] + n, case["rotary_dim"])
        for name in ("k_read", "v_read"):
            s[name] = torch.empty(s["read_rows"], case["hkv"], hd, dtype=torch.bfloat16, device=DEVICE)
        if own:
            s["cache"] = _handle(s, case)
        return s
    if case["op"] == "read":
        lens = _read_lens(case)
        rng.shuffle(lens)
        s["first"], s["read_starts"] = _i32([f for f, _ in lens]), _i32(_starts([n for _, n in lens]))
        s["read_rows"], s["read_most"] = sum(n for _, n in lens), max(n for _, n in lens)
        table, count = _pages(rng, [f + n for f, n in lens], case["page"])
        s["page_table"] = _i32(table)
        _cache(g, s, case, count)
        for name in ("k_read", "v_read"):
            s[name] = torch.empty(s["read_rows"], case["hkv"], hd, dtype=dt, device=DEVICE)
        if own:
            s["cache"] = _handle(s, case)
        return s
    lens = _lens(case)
    rng.shuffle(lens)
    s["lens"] = lens
    total = sum(n for _, n in lens)
    s["q"] = _randn(g, total, case["hq"], hd, dtype=dt, scale=2.0)
    table, count = _pages(rng, [c + n for c, n in lens], case["page"])
    s["page_table"] = _i32(table)
    _cache(g, s, case, count)
    s["parents"] = _trees(rng, [n for _, n in lens])
    s["mask"] = _masks(s["parents"])
    s["ctx_lens"], s["q_starts"] = _i32([c for c, _ in lens]), _i32(_starts([n for _, n in lens]))
    s["most"] = max(c + n for c, n in lens)
    s["widest"] = max(n for _, n in lens)
    s["out"] = torch.empty_like(s["q"])
    if own:
        from baremetalinferenceengine_b200 import ops

        s["cache"] = _handle(s, case)
        s["workspace"] = ops.paged_kv8_tree_attention_workspace(s["q"], s["cache"], case["batch"], case["ctx_hi"],
                                                                case["tokens"])
    return s


# --------------------------------------------------------------------------
# The plain forms
# --------------------------------------------------------------------------

def _power(exponents):
    """2^e in 32 bits, exactly, from its bits."""
    return ((exponents.to(torch.int32) + 127) << 23).view(torch.float32)


def _exponents(scales):
    return scales.view(torch.uint8).to(torch.int32) - 127


def _normed(x, weight):
    x = x.float()
    if weight is None:
        return x
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()


def _rotated(x, positions, table, dim, pairs):
    """x [rows, heads, hd] in 32 bits, the first `dim` elements of each head rotated."""
    cs = table[positions.long()][:, None]  # [rows, 1, dim / 2, 2]
    c, s = cs[..., 0], cs[..., 1]
    out = x.clone()
    if pairs == "half":
        a, b = x[..., :dim // 2], x[..., dim // 2:dim]
        out[..., :dim // 2] = a * c - b * s
        out[..., dim // 2:dim] = b * c + a * s
    else:
        a, b = x[..., 0:dim:2], x[..., 1:dim:2]
        out[..., 0:dim:2] = a * c - b * s
        out[..., 1:dim:2] = b * c + a * s
    return out


def _places(s, case, starts, first, rows):
    """(page, slot in it, sequence, slot) of dense rows: sequence b's are starts[b]: and on, from slot first[b]."""
    row = torch.arange(rows, device=DEVICE)
    seq = torch.searchsorted(starts.long(), row, right=True) - 1
    slot = first.long()[seq] + row - starts.long()[seq]
    return s["page_table"].long()[seq, slot // case["page"]], slot % case["page"], seq, slot


def _plain_read(s, case):
    page, off, _, _ = _places(s, case, s["read_starts"], s["first"], s["read_rows"])
    for name in ("k", "v"):
        codes = s[name + "_pages"].view(torch.uint8)[page, :, off].view(torch.float8_e4m3fn).float()
        scale = _power(_exponents(s[name + "_scales"])[page, :, off // case["block"]])
        s[name + "_read"].copy_(codes * scale[..., None])
    return [s["k_read"], s["v_read"]]


def _plain_append(s, case):
    rot = s["positions"], s["table"], case["rotary_dim"], case["pairs"]
    s["q_out"].copy_(_rotated(_normed(s["q"], s["q_weight"]), *rot))
    new = {"k": _rotated(_normed(s["k"], s["k_weight"]), *rot), "v": s["v"].float()}
    # every slot of the blocks that the new tokens meet
    rows, block, hkv = s["read_rows"], case["block"], case["hkv"]
    page, off, seq, slot = _places(s, case, s["read_starts"], s["first"], rows)
    ctx = s["ctx_lens"].long()[seq]
    row = (s["q_starts"].long()[seq] + slot - ctx).clamp(min=0)
    is_new = (slot >= ctx)[:, None]
    place = page * (case["page"] // block) + off // block  # of the block among all blocks
    kept_block = (slot // block * block < ctx)[:, None]    # it has slots of earlier calls
    blocks = s["k_pages"].shape[0] * (case["page"] // block)
    for name in ("k", "v"):
        pages, scales = s[name + "_pages"].view(torch.uint8), s[name + "_scales"]
        x = new[name][row]
        amax = torch.where(is_new, x.abs().amax(-1), 0.0)
        most = torch.zeros(blocks, hkv, device=DEVICE).scatter_reduce_(0, place[:, None].expand(-1, hkv), amax, "amax")[place]
        m, e = torch.frexp(most)  # most = m 2^e, m in [0.5, 1): of 448 = 0.875 * 2^9
        e = torch.where(most > 0, torch.where(m <= 0.875, e - 9, e - 8), LOWEST).clamp(LOWEST, HIGHEST)
        before = _exponents(scales)[page, :, off // block]
        e = torch.where(kept_block, torch.maximum(e, before), e)
        kept = pages[page, :, off].view(torch.float8_e4m3fn).float() * _power(before - e)[..., None]
        codes = torch.where(is_new[..., None], x * _power(-e)[..., None], kept).clamp(-LARGEST, LARGEST)
        pages[page, :, off] = codes.to(torch.float8_e4m3fn).view(torch.uint8)
        scales.view(torch.uint8)[page, :, off // block] = (e + 127).to(torch.uint8)
    return [s["q_out"]] + _plain_read(s, case)


def _plain_attention(s, case):
    hd, hkv, page, block, most, widest = case["hd"], case["hkv"], case["page"], case["block"], s["most"], s["widest"]
    hq, batch, group = case["hq"], case["batch"], case["hq"] // case["hkv"]
    ctx, starts = s["ctx_lens"].long(), s["q_starts"].long()
    slot = torch.arange(most, device=DEVICE)
    ids = s["page_table"].long()[:, slot // page]                              # [batch, most]
    k, v = ((s[name + "_pages"].view(torch.uint8)[ids, :, slot % page].view(torch.float8_e4m3fn).float()
             * _power(_exponents(s[name + "_scales"])[ids, :, slot % page // block])[..., None]).transpose(1, 2)
            for name in ("k", "v"))                                            # [batch, hkv, most, hd]
    i = torch.arange(widest, device=DEVICE)
    n = starts[1:] - starts[:-1]
    row = (starts[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)               # [batch, widest]
    q = s["q"][row].float().reshape(batch, widest, hkv, group, hd).permute(0, 2, 3, 1, 4)
    score = torch.matmul(q.reshape(batch, hkv, group * widest, hd), k.transpose(-1, -2)) * hd ** -0.5
    j = slot[None, :] - ctx[:, None]                                           # drafted slot, [batch, most]
    word = (j.clamp(0, 64 * s["mask"].shape[1] - 1) // 64)[:, None].expand(-1, widest, -1)
    seen = (s["mask"][row].gather(2, word) >> (j.clamp(min=0) % 64)[:, None]) & 1  # [batch, widest, most]
    seen = (j < 0)[:, None] | ((j < n[:, None])[:, None] & (seen != 0))
    score = score.view(batch, hkv, group, widest, most).masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    o = torch.matmul(p.view(batch, hkv, group * widest, most), v).view(batch, hkv, group, widest, hd) / p.sum(-1, keepdim=True)
    token = torch.arange(s["q"].shape[0], device=DEVICE)
    at = torch.searchsorted(starts, token, right=True) - 1
    s["out"].copy_(o[at, :, :, token - starts[at]].reshape(-1, hq, hd))
    return s["out"]


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------

def run(s):
    case = s["case"]
    inter = case.get("pairs") == "interleaved"
    if own:
        from baremetalinferenceengine_b200 import ops

        if case["op"] == "norm_rotary":
            return list(ops.qk_norm_rotary(s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"], s["table"],
                                           eps=EPS, interleaved=inter, q_out=s["q_out"], k_out=s["k_out"]))
        if case["op"] == "append":
            ops.paged_kv8_append(s["q"], s["k"], s["v"], s["cache"], s["ctx_lens"], s["q_starts"], case["tokens"],
                                 positions=s["positions"], table=s["table"], q_weight=s["q_weight"],
                                 k_weight=s["k_weight"], eps=EPS, interleaved=inter, q_out=s["q_out"])
        if case["op"] in ("append", "read"):
            ops.paged_kv8_read(s["cache"], s["first"], s["read_starts"], s["read_rows"], s["read_most"],
                               k_out=s["k_read"], v_out=s["v_read"])
            return ([s["q_out"]] if case["op"] == "append" else []) + [s["k_read"], s["v_read"]]
        return ops.paged_kv8_tree_attention(s["q"], s["cache"], s["ctx_lens"], s["q_starts"], case["ctx_hi"],
                                            case["tokens"], tree_mask=s["mask"], out=s["out"], workspace=s["workspace"])
    if case["op"] == "norm_rotary":
        rot = s["positions"], s["table"], case["rotary_dim"], case["pairs"]
        s["q_out"].copy_(_rotated(_normed(s["q"], s["q_weight"]), *rot))
        s["k_out"].copy_(_rotated(_normed(s["k"], s["k_weight"]), *rot))
        return [s["q_out"], s["k_out"]]
    if case["op"] == "append":
        return _plain_append(s, case)
    if case["op"] == "read":
        return _plain_read(s, case)
    return _plain_attention(s, case)


def work(case):
    es, hd, hkv = SIZES[case["dtype"]], case["hd"], case["hkv"]
    if case["op"] == "norm_rotary":
        heads = case["hq"] + hkv
        angles = min(case["rows"], case["max_pos"]) * case["rotary_dim"] * 4
        return {"bytes": case["rows"] * (2 * heads * hd * es + 4) + angles,
                "flops": case["rows"] * heads * (4 * hd + 3 * case["rotary_dim"])}
    if case["op"] == "append":
        rows, block = case["batch"] * case["tokens"], case["block"]
        kept = sum(c % block for c in _append_ctx(case))
        angles = min(rows, case["ctx"] + case["tokens"]) * case["rotary_dim"] * 4
        # Q in and out, K and V in, their 8 bits written, kept ones read; and the blocks as 16 bits
        size = rows * (2 * (case["hq"] + hkv) * es + 2 * hkv) * hd + kept * 2 * hkv * hd + (rows + kept) * 4 * hkv * hd
        return {"bytes": size + 4 * rows + angles, "flops": rows * (case["hq"] + 2 * hkv) * (7 if case["norm"] else 3) * hd}
    if case["op"] == "read":
        rows = sum(n for _, n in _read_lens(case))
        return {"bytes": rows * 2 * hkv * hd * (1 + es) + rows * 2 * hkv // case["block"], "flops": rows * 2 * hkv * hd}
    read = flops = rows = 0
    for ctx, n in _lens(case):
        rows += n
        read += (ctx + n) * 2 * hkv * hd + (ctx + n) * 2 * hkv // case["block"] + 4 * (-(-(ctx + n) // case["page"]))
        flops += 4 * hd * case["hq"] * n * (ctx + (n + 1) / 2)
    return {"bytes": read + rows * 2 * case["hq"] * hd * es + 8 * rows, "flops": flops}


# --------------------------------------------------------------------------
# The definitions in 64 bits
# --------------------------------------------------------------------------

def _exact_turned(x, weight, positions, dim, pairs):
    """Heads divided by their root mean square, then each pair as a complex number times e^(i p f)."""
    x = x.double()
    if weight is not None:
        x = x / ((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * weight.double()
    angle = positions.double()[:, None, None] * _frequencies(dim).to(x.device)
    turn = torch.polar(torch.ones_like(angle), angle)
    head, rest = x[..., :dim], x[..., dim:]
    if pairs == "half":
        z = torch.complex(head[..., :dim // 2].contiguous(), head[..., dim // 2:].contiguous()) * turn
        return torch.cat([z.real, z.imag, rest], -1)
    z = torch.view_as_complex(head.reshape(*head.shape[:-1], dim // 2, 2).contiguous()) * turn
    return torch.cat([torch.view_as_real(z).flatten(-2), rest], -1)


#: The 256 values of e4m3: sign, four bits of exponent (bias 7), three of mantissa.
_E4M3 = np.array([(-1.0) ** (b >> 7) * (math.nan if b & 127 == 127 else (b & 7) * 2.0 ** -9 if b & 120 == 0
                                        else (8 + (b & 7)) * 2.0 ** ((b >> 3 & 15) - 10)) for b in range(256)])


def _to_e4m3(x):
    """The nearest value of e4m3, of two the one with an even last bit; larger ones end at 448."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(2.0 ** -6, LARGEST))) - 3)
    return (torch.round(x / step) * step).clamp(-LARGEST, LARGEST)


def _exact_values(s, name):
    """(values of the pages, exponents of their scales)."""
    codes = torch.from_numpy(_E4M3).to(DEVICE)[s[name + "_pages"].view(torch.uint8).int()]
    return codes, s[name + "_scales"].view(torch.uint8).double() - 127


def _exact_places(s, case, first, counts):
    pages = s["page_table"].cpu().numpy()
    at = [(pages[b, t // case["page"]], t % case["page"]) for b, (f, n) in enumerate(zip(first, counts)) for t in range(f, f + n)]
    at = torch.tensor(np.array(at, dtype=np.int64).reshape(-1, 2), device=DEVICE)
    return at[:, 0], at[:, 1]


def _exact_append(s, case):
    turn = lambda x, w: _exact_turned(x, w, s["positions"], case["rotary_dim"], case["pairs"])  # noqa: E731
    n, block, out = case["tokens"], case["block"], [turn(s["q"], s["q_weight"])]
    ctx = s["ctx_lens"].cpu().tolist()
    for name in ("k", "v"):
        new = (turn(s["k"], s["k_weight"]) if name == "k" else s["v"].double()).reshape(case["batch"], n, case["hkv"], case["hd"])
        codes, exponents = _exact_values(s, name)
        values = []
        for b, c in enumerate(ctx):
            first = c // block * block
            blocks = -(-(c + n - first) // block)
            page, off = _exact_places(s, case, [0] * b + [first], [0] * b + [c - first])
            x = torch.zeros(blocks * block, case["hkv"], case["hd"], dtype=torch.float64, device=DEVICE)
            x[c - first:c - first + n] = new[b]
            e = torch.ceil(torch.log2(x.reshape(blocks, block, case["hkv"], -1).abs().amax((1, 3)) / LARGEST)).clamp(LOWEST, HIGHEST)
            if c > first:
                was = exponents[page[0], :, off[0] // block]
                e[0] = torch.maximum(e[0], was)
                x[:c - first] = codes[page, :, off] * torch.exp2(was)[None, :, None]
            scale = torch.exp2(e).repeat_interleave(block, 0)[..., None]
            values.append((_to_e4m3(x / scale) * scale)[:c - first + n])
        out.append(torch.cat(values))
    return out


def _exact_attention(s, case):
    hd, page, block, out, row = case["hd"], case["page"], case["block"], [], 0
    (kc, ke), (vc, ve) = _exact_values(s, "k"), _exact_values(s, "v")
    for b, (ctx, n) in enumerate(s["lens"]):
        slot = torch.arange(ctx + n, device=DEVICE)
        ids = s["page_table"][b].long()[slot // page]
        k, v = ((c[ids, :, slot % page] * torch.exp2(e[ids, :, slot % page // block])[..., None]).repeat_interleave(
            case["hq"] // case["hkv"], 1) for c, e in ((kc, ke), (vc, ve)))
        seen = np.zeros((n, ctx + n), dtype=bool)
        seen[:, :ctx] = True
        for i in range(n):
            j = i
            while j >= 0:
                seen[i, ctx + j] = True
                j = s["parents"][b][j]
        score = torch.einsum("nhd,shd->hns", s["q"][row:row + n].double(), k) * hd ** -0.5
        score = torch.where(torch.from_numpy(seen).to(DEVICE)[None], score, -math.inf)
        out.append(torch.einsum("hns,shd->nhd", torch.softmax(score, -1), v))
        row += n
    return torch.cat(out)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm_rotary":
        return [_exact_turned(s[x], s[x + "_weight"], s["positions"], case["rotary_dim"], case["pairs"]) for x in ("q", "k")]
    if case["op"] == "append":
        return _exact_append(s, case)
    if case["op"] == "read":
        starts = s["read_starts"].cpu().numpy()
        page, off = _exact_places(s, case, s["first"].cpu().tolist(), (starts[1:] - starts[:-1]).tolist())
        return [codes[page, :, off] * torch.exp2(e[page, :, off // case["block"]])[..., None]
                for codes, e in (_exact_values(s, name) for name in ("k", "v"))]
    return _exact_attention(s, case)
