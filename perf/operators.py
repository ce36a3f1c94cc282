"""The serving operators around a paged KV cache, as workloads: inputs, a plain form in
elementary torch operations, a 64-bit form from the definitions, and the calls a user makes.

Four operators, which make one step of a batch that decodes with drafted tokens:

* ``rotary``: rotary positions on Q and K, half or interleaved pairs, part of the head,
  frequencies scaled for long contexts;
* ``append``: K rotated and V copied into the pages of a paged cache, Q rotated;
* ``attention``: a tree of drafted tokens per sequence over the paged cache;
* ``sample``: temperature, top-k, top-p and min-p, from given uniform numbers.

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


# --------------------------------------------------------------------------
# Cases
# --------------------------------------------------------------------------

def _rotary(rows, hq, hkv, hd, rotary_dim, pairs, scaling, max_pos, dtype, name=None):
    return dict(op="rotary", rows=rows, hq=hq, hkv=hkv, hd=hd, rotary_dim=rotary_dim, pairs=pairs, scaling=scaling,
                max_pos=max_pos, dtype=dtype, **({"name": name} if name else {}))


def _append(batch, tokens, ctx, tree, hq, hkv, hd, rotary_dim, pairs, page, dtype, name=None):
    return dict(op="append", batch=batch, tokens=tokens, ctx=ctx, tree=tree, hq=hq, hkv=hkv, hd=hd,
                rotary_dim=rotary_dim, pairs=pairs, page=page, dtype=dtype, **({"name": name} if name else {}))


def _attention(batch, ctx_lo, ctx_hi, tokens, ragged, hq, hkv, hd, page, dtype, name=None):
    return dict(op="attention", batch=batch, ctx_lo=ctx_lo, ctx_hi=ctx_hi, tokens=tokens, ragged=ragged, hq=hq,
                hkv=hkv, hd=hd, page=page, dtype=dtype, **({"name": name} if name else {}))


def _sample(rows, vocab, filters, dtype, name=None):
    return dict(op="sample", rows=rows, vocab=vocab, filters=filters, dtype=dtype, **({"name": name} if name else {}))


def listed():
    return [
        # one decode step of 64 sequences at the Llama-3-8B shape: latency counts
        _rotary(64, 32, 8, 128, 128, "half", "bands", 8192, "bf16", "rotary-decode"),
        # a prompt batch at the 70B shape, interleaved pairs on half of each head, a stretched context
        _rotary(16384, 64, 8, 128, 64, "interleaved", "yarn", 32768, "bf16", "rotary-prompt"),
        # one new token of each of 64 sequences
        _append(64, 1, 500, False, 32, 8, 128, 128, "half", 16, "bf16", "append-decode"),
        # four prompts of 8192 tokens at the 70B shape
        _append(4, 8192, 0, False, 64, 8, 128, 128, "half", 64, "bf16", "append-prompt"),
        # trees of 25 drafted tokens at the tinyllama shape, pages that are no power of two
        _append(8, 25, 100, True, 6, 6, 48, 48, "half", 24, "f32", "append-tree-f32"),
        # one user's sequence: 12 drafted tokens behind 8000 cached ones
        _attention(1, 8000, 8000, 12, False, 32, 8, 128, 16, "bf16", "tree-one"),
        # a serving batch of uneven sequences, up to 8 drafted tokens each
        _attention(64, 1, 8192, 8, True, 32, 8, 128, 16, "bf16", "tree-batch"),
        # wide trees over long contexts at the 70B shape: products count as much as bytes
        _attention(16, 4096, 8192, 64, False, 64, 8, 128, 64, "bf16", "tree-wide"),
        # the tinyllama shape in 32 bits
        _attention(32, 0, 230, 25, True, 6, 6, 48, 16, "f32", "tree-f32"),
        # one user's token from a small vocabulary
        _sample(1, 32000, "nucleus", "f32", "sample-one"),
        # a decode step of 64 requests with settings of their own
        _sample(64, 128256, "mixed", "f32", "sample-mixed"),
        # a large batch, every filter but top-k, bf16 logits
        _sample(256, 128256, "nucleus", "bf16", "sample-nucleus"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attention", "attention", "sample", "sample"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    hd = rng.choice([48, 64, 128, 128, 256])
    hkv = rng.choice([1, 2, 6, 8])
    hq = hkv * rng.choice([1, 2, 4, 7, 8])
    pairs = rng.choice(["half", "interleaved"])
    part = rng.choice([hd, hd, hd // 2, 24])
    page = rng.choice([8, 16, 24, 32, 64, 100, 128, 256])
    if op == "rotary":
        rows = max(1, min(_log(rng, 1, 16384), 16384 * 72 * 128 * 2 // ((hq + hkv) * hd * SIZES[dtype])))
        return _rotary(rows, hq, hkv, hd, part, pairs, rng.choice(["none", "linear", "ntk", "bands", "yarn"]),
                       _log(rng, max(64, rows // 4), 131072), dtype)
    if op == "append":
        tree = rng.random() < 0.4
        tokens = rng.randint(1, 64) if tree else _log(rng, 1, 4096)
        batch = max(1, min(_log(rng, 1, 64), 16384 // tokens))
        return _append(batch, tokens, _log(rng, 1, 2000), tree, hq, hkv, hd, part, pairs, page, dtype)
    if op == "attention":
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
        return _attention(batch, rng.choice([0, hi // 2, hi]), hi, tokens, rng.random() < 0.6, hq, hkv, hd, page, dtype)
    vocab = rng.choice([1000, 32000, 50257, 128256, _log(rng, 300, 131072), _log(rng, 300, 131072)])
    return _sample(_log(rng, 1, 256), vocab, rng.choice(["plain", "nucleus", "topk", "mixed", "mixed"]), dtype)


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------

THETA = 5e5
SCALINGS = {
    "none": dict(kind="none"),
    "linear": dict(kind="linear", factor=4.0),
    "ntk": dict(kind="ntk", factor=4.0),
    "bands": dict(kind="bands", factor=8.0, original_max_pos=8192, low_freq_factor=1.0, high_freq_factor=4.0),
    "yarn": dict(kind="yarn", factor=8.0, original_max_pos=4096, beta_fast=32.0, beta_slow=1.0),
}


def _frequencies(dim, theta, s):
    """(inverse frequency of each pair, in 64 bits; factor of cos and sin)."""
    i = torch.arange(dim // 2, dtype=torch.float64)
    kind = s["kind"]
    if kind == "none":
        return theta ** (-2.0 * i / dim), 1.0
    if kind == "linear":
        return theta ** (-2.0 * i / dim) / s["factor"], 1.0
    if kind == "ntk":
        return (theta * s["factor"] ** (dim / (dim - 2.0))) ** (-2.0 * i / dim), 1.0
    f = theta ** (-2.0 * i / dim)
    if kind == "bands":
        turns = s["original_max_pos"] * f / (2 * math.pi)  # full turns within the original context
        keep = ((turns - s["low_freq_factor"]) / (s["high_freq_factor"] - s["low_freq_factor"])).clamp(0.0, 1.0)
        return f / s["factor"] * (1.0 - keep) + f * keep, 1.0
    edge = [dim * math.log(s["original_max_pos"] / (b * 2 * math.pi)) / (2 * math.log(theta))
            for b in (s["beta_fast"], s["beta_slow"])]
    low, high = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), dim - 1)
    ramp = ((i - low) / (max(high - low, 0.001))).clamp(0.0, 1.0)
    return f / s["factor"] * ramp + f * (1.0 - ramp), 0.1 * math.log(s["factor"]) + 1.0


def _table(max_pos, dim, scaling):
    """[max_pos][dim / 2][2] of (cos, sin), from 64-bit angles, as a server keeps it."""
    f, m = _frequencies(dim, THETA, SCALINGS[scaling])
    a = torch.arange(max_pos, dtype=torch.float64, device=DEVICE)[:, None] * f.to(DEVICE)[None, :]
    return torch.stack([m * torch.cos(a), m * torch.sin(a)], dim=-1).float()


def _rope_table(max_pos, dim, scaling):
    from baremetalinferenceengine_b200 import ops

    s = SCALINGS[scaling]
    return ops.RopeTable(max_pos, dim, THETA, DEVICE,
                         scaling=None if s["kind"] == "none" else ops.RopeScaling(**s))


def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32) * scale).to(dtype)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


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
    out = []
    for n in sizes:
        out.append([rng.randint(max(-1, j - 6), j - 1) for j in range(n)])
    return out


def _lens(case):
    """(context length, drafted tokens) of each sequence: part of the case, whatever the seed."""
    rng = random.Random("%d %d %d %d" % (case["batch"], case["ctx_lo"], case["ctx_hi"], case["tokens"]))
    out = []
    for _ in range(case["batch"]):
        n = rng.randint(1, case["tokens"]) if case["ragged"] else case["tokens"]
        out.append((rng.randint(case["ctx_lo"], case["ctx_hi"]), n))
    return out


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


def prepare(case, seed):
    g, rng, dt = _generator(seed), random.Random(seed), DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "rotary":
        rows, hd = case["rows"], case["hd"]
        qkv = _randn(g, rows, case["hq"] + 2 * case["hkv"], hd, dtype=dt)  # one projection's output: q, k and v side by side
        s["q"], s["k"] = qkv[:, :case["hq"]], qkv[:, case["hq"]:case["hq"] + case["hkv"]]
        s["positions"] = torch.randint(0, case["max_pos"], (rows,), generator=g, device=DEVICE, dtype=torch.int32)
        s["table"] = (_rope_table if own else _table)(case["max_pos"], case["rotary_dim"], case["scaling"])
        s["q_out"] = torch.empty(rows, case["hq"], hd, dtype=dt, device=DEVICE)
        s["k_out"] = torch.empty(rows, case["hkv"], hd, dtype=dt, device=DEVICE)
        return s
    if case["op"] == "append":
        batch, n, hd, page = case["batch"], case["tokens"], case["hd"], case["page"]
        rows = batch * n
        s["q"] = _randn(g, rows, case["hq"], hd, dtype=dt)
        s["k"] = _randn(g, rows, case["hkv"], hd, dtype=dt)
        s["v"] = _randn(g, rows, case["hkv"], hd, dtype=dt)
        lens = random.Random("%d %d %d" % (batch, n, case["ctx"]))  # part of the case, whatever the seed
        ctx = [case["ctx"] - lens.randint(0, case["ctx"] // 2) for _ in range(batch)]
        rng.shuffle(ctx)
        depth = []
        for tree in _trees(rng, [n] * batch) if case["tree"] else [range(-1, n - 1)] * batch:
            d = []
            for p in tree:
                d.append(d[p] + 1 if p >= 0 else 0)
            depth.append(d)
        s["positions"] = _i32([c + x for c, d in zip(ctx, depth) for x in d])
        s["slots"] = _i32([c + j for c in ctx for j in range(n)]) if case["tree"] else None
        s["seq_ids"] = _i32([b for b in range(batch) for _ in range(n)])
        table, count = _pages(rng, [c + n for c in ctx], page)
        s["page_table"] = _i32(table)
        for name in ("k_pages", "v_pages"):
            s[name] = _randn(g, count, case["hkv"], page, hd, dtype=dt)
        s["table"] = (_rope_table if own else _table)(case["ctx"] + n, case["rotary_dim"], "none")
        s["q_out"] = torch.empty_like(s["q"])
        if own:
            from baremetalinferenceengine_b200 import ops

            s["cache"] = ops.PagedKV(s["k_pages"], s["v_pages"], s["page_table"])
        return s
    if case["op"] == "attention":
        hd, page = case["hd"], case["page"]
        lens = _lens(case)
        rng.shuffle(lens)
        s["lens"] = lens
        total = sum(n for _, n in lens)
        s["q"] = _randn(g, total, case["hq"], hd, dtype=dt, scale=2.0)
        table, count = _pages(rng, [c + n for c, n in lens], page)
        s["page_table"] = _i32(table)
        for name in ("k_pages", "v_pages"):
            s[name] = _randn(g, count, case["hkv"], page, hd, dtype=dt)
        s["parents"] = _trees(rng, [n for _, n in lens])
        s["mask"] = _masks(s["parents"])
        s["ctx_lens"] = _i32([c for c, _ in lens])
        starts = [0]
        for _, n in lens:
            starts.append(starts[-1] + n)
        s["q_starts"] = _i32(starts)
        s["out"] = torch.empty_like(s["q"])
        if own:
            from baremetalinferenceengine_b200 import ops

            s["cache"] = ops.PagedKV(s["k_pages"], s["v_pages"], s["page_table"])
            s["workspace"] = ops.paged_tree_attention_workspace(s["q"], s["cache"], case["batch"], case["ctx_hi"],
                                                                case["tokens"])
        return s
    rows, vocab = case["rows"], case["vocab"]
    spread = 1.0 + 4.0 * torch.rand(rows, 1, generator=g, device=DEVICE)  # from flat rows to peaked ones
    s["logits"] = (torch.randn(rows, vocab, generator=g, device=DEVICE) * spread).to(dt)
    s["uniforms"] = torch.rand(rows, generator=g, device=DEVICE)
    f = case["filters"]
    s["temperature"] = 0.5 + torch.rand(rows, generator=g, device=DEVICE)
    s["top_k"] = s["top_p"] = s["min_p"] = None
    pick = lambda values: [rng.choice(values) for _ in range(rows)]  # noqa: E731
    real = lambda values: torch.tensor(values, dtype=torch.float32, device=DEVICE)  # noqa: E731
    if f == "mixed":  # greedy requests among the others
        s["temperature"] = s["temperature"] * real(pick([0.0, 1.0, 1.0, 1.0, 1.0]))
    if f in ("topk", "mixed"):
        s["top_k"] = _i32(pick([0, 1, 20, 50, 200] if f == "mixed" else [5, 20, 50, 1000]))
    if f in ("nucleus", "mixed"):
        s["top_p"] = real(pick([0.5, 0.9, 0.95, 1.0]))
        s["min_p"] = real(pick([0.0, 0.0, 0.02, 0.1]))
    return s


# --------------------------------------------------------------------------
# The plain forms
# --------------------------------------------------------------------------

def _rotated(x, positions, table, dim, pairs):
    """x [rows, heads, hd] in 32 bits, the first `dim` elements of each head rotated."""
    x = x.float()
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


def _plain_append(s, case):
    rot = case["rotary_dim"], case["pairs"]
    dt = s["q"].dtype
    s["q_out"].copy_(_rotated(s["q"], s["positions"], s["table"], *rot).to(dt))
    slots = (s["slots"] if s["slots"] is not None else s["positions"]).long()
    page = s["page_table"][s["seq_ids"].long(), slots // case["page"]].long()
    off = slots % case["page"]
    s["k_pages"][page, :, off] = _rotated(s["k"], s["positions"], s["table"], *rot).to(dt)
    s["v_pages"][page, :, off] = s["v"]
    return [s["q_out"], s["k_pages"], s["v_pages"]]


def _plain_attention(s, case):
    hd, hkv, page = case["hd"], case["hkv"], case["page"]
    group = case["hq"] // hkv
    row = 0
    for b, (ctx, n) in enumerate(s["lens"]):
        ids = s["page_table"][b, :-(-(ctx + n) // page)].long()
        k, v = (s[name][ids].transpose(0, 1).reshape(hkv, -1, hd)[:, :ctx + n].float()
                for name in ("k_pages", "v_pages"))
        q = s["q"][row:row + n].float().reshape(n, hkv, group, hd).permute(1, 2, 0, 3)  # [hkv, group, n, hd]
        score = torch.matmul(q, k[:, None].transpose(-1, -2)) / math.sqrt(hd)
        j = torch.arange(n, device=k.device)
        seen = (s["mask"][row:row + n][:, j // 64] >> (j % 64)) & 1
        score[..., ctx:].masked_fill_(seen == 0, -math.inf)
        p = torch.exp(score - score.amax(-1, keepdim=True))
        o = torch.matmul(p, v[:, None]) / p.sum(-1, keepdim=True)
        s["out"][row:row + n] = o.permute(2, 0, 1, 3).reshape(n, case["hq"], hd).to(s["out"].dtype)
        row += n
    return s["out"]


def _plain_sample(s):
    x = s["logits"].double()
    rows, vocab = x.shape
    temp = s["temperature"].double()[:, None]
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)  # ties: the lowest index first
    w = torch.exp((x - x[:, :1]) / torch.where(temp > 0, temp, 1.0))
    rank = torch.arange(vocab, device=x.device)[None]
    if s["top_k"] is not None:
        k = s["top_k"].long()[:, None]
        w = torch.where((k <= 0) | (rank < k), w, 0.0)
    first = w[:, :1].clone()
    if s["top_p"] is not None:
        before = torch.cumsum(w, -1) - w
        p = s["top_p"].double()[:, None]
        w = torch.where((p >= 1) | (rank == 0) | (before < p * w.sum(-1, keepdim=True)), w, 0.0)
    if s["min_p"] is not None:
        w = torch.where(w >= s["min_p"].double()[:, None] * first, w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)  # back to the order of the vocabulary
    c = torch.cumsum(w, -1)
    token = (c <= s["uniforms"].double()[:, None] * c[:, -1:]).sum(-1)
    last = vocab - 1 - torch.argmax((w > 0).flip(-1).to(torch.int8), -1)
    token = torch.minimum(token, last)
    return torch.where(temp[:, 0] > 0, token, order[:, 0]).to(torch.int32)


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------

def run(s):
    case = s["case"]
    if own:
        from baremetalinferenceengine_b200 import ops

        if case["op"] == "rotary":
            return list(ops.rotary(s["q"], s["k"], s["positions"], s["table"],
                                   interleaved=case["pairs"] == "interleaved", q_out=s["q_out"], k_out=s["k_out"]))
        if case["op"] == "append":
            ops.paged_kv_append(s["q"], s["k"], s["v"], s["positions"], s["cache"], table=s["table"],
                                seq_ids=s["seq_ids"], slots=s["slots"], interleaved=case["pairs"] == "interleaved",
                                q_out=s["q_out"])
            return [s["q_out"], s["k_pages"], s["v_pages"]]
        if case["op"] == "attention":
            return ops.paged_tree_attention(s["q"], s["cache"], s["ctx_lens"], s["q_starts"], case["ctx_hi"],
                                            case["tokens"], tree_mask=s["mask"], out=s["out"],
                                            workspace=s["workspace"])
        return ops.sample(s["logits"], s["uniforms"], temperature=s["temperature"], top_k=s["top_k"],
                          top_p=s["top_p"], min_p=s["min_p"])
    if case["op"] == "rotary":
        for x, o in ((s["q"], s["q_out"]), (s["k"], s["k_out"])):
            o.copy_(_rotated(x, s["positions"], s["table"], case["rotary_dim"], case["pairs"]).to(o.dtype))
        return [s["q_out"], s["k_out"]]
    if case["op"] == "append":
        return _plain_append(s, case)
    if case["op"] == "attention":
        return _plain_attention(s, case)
    return _plain_sample(s)


def work(case):
    if case["op"] == "sample":
        values = case["rows"] * case["vocab"]
        return {"bytes": values * SIZES[case["dtype"]] + 24 * case["rows"], "flops": 4 * values}
    es, hd, hq, hkv = SIZES[case["dtype"]], case["hd"], case["hq"], case["hkv"]
    if case["op"] == "rotary":
        row = (hq + hkv) * hd
        angles = min(case["rows"], case["max_pos"]) * case["rotary_dim"] * 4
        return {"bytes": case["rows"] * (2 * row * es + 4) + angles,
                "flops": 3 * case["rows"] * (hq + hkv) * case["rotary_dim"]}
    if case["op"] == "append":
        rows = case["batch"] * case["tokens"]
        angles = min(rows, case["ctx"] + case["tokens"]) * case["rotary_dim"] * 4
        return {"bytes": rows * ((2 * hq + 4 * hkv) * hd * es + 16) + angles,
                "flops": 3 * rows * (hq + hkv) * case["rotary_dim"]}
    read = flops = rows = 0
    for ctx, n in _lens(case):
        rows += n
        read += (ctx + n) * 2 * hkv * hd * es + 4 * (-(-(ctx + n) // case["page"]))
        flops += 4 * hd * hq * n * (ctx + (n + 1) / 2)
    return {"bytes": read + rows * 2 * hq * hd * es + 8 * rows, "flops": flops}


# --------------------------------------------------------------------------
# The definitions in 64 bits
# --------------------------------------------------------------------------

def _exact_rotated(x, positions, dim, pairs, scaling):
    """Each pair as a complex number times mscale * e^(i p f), in 64 bits."""
    f, m = _frequencies(dim, THETA, SCALINGS[scaling])
    angle = positions.double()[:, None, None] * f.to(x.device)
    turn = torch.polar(torch.full_like(angle, m), angle)
    x = x.double()
    head, rest = x[..., :dim], x[..., dim:]
    if pairs == "half":
        z = torch.complex(head[..., :dim // 2].contiguous(), head[..., dim // 2:].contiguous()) * turn
        return torch.cat([z.real, z.imag, rest], -1)
    z = torch.view_as_complex(head.reshape(*head.shape[:-1], dim // 2, 2).contiguous()) * turn
    return torch.cat([torch.view_as_real(z).flatten(-2), rest], -1)


def _exact_attention(s, case):
    hd, hkv, page = case["hd"], case["hkv"], case["page"]
    out, row = [], 0
    for b, (ctx, n) in enumerate(s["lens"]):
        slot = torch.arange(ctx + n, device=s["q"].device)
        ids = s["page_table"][b].long()[slot // page]
        k, v = (s[name][ids, :, slot % page].double() for name in ("k_pages", "v_pages"))  # [slots, hkv, hd]
        k, v = (t.repeat_interleave(case["hq"] // hkv, 1) for t in (k, v))
        seen = np.zeros((n, ctx + n), dtype=bool)
        seen[:, :ctx] = True
        for i in range(n):
            j = i
            while j >= 0:
                seen[i, ctx + j] = True
                j = s["parents"][b][j]
        q = s["q"][row:row + n].double()
        score = torch.einsum("nhd,shd->hns", q, k) * hd ** -0.5
        score = torch.where(torch.from_numpy(seen).to(q.device)[None], score, -math.inf)
        out.append(torch.einsum("hns,shd->nhd", torch.softmax(score, -1), v))
        row += n
    return torch.cat(out)


def _exact_sample(s, case):
    value = lambda name, r: None if s[name] is None else s[name][r].item()  # noqa: E731
    logits, tokens = s["logits"].float().cpu().numpy().astype(np.float64), []
    for r in range(case["rows"]):
        x = logits[r]
        if value("temperature", r) == 0:
            tokens.append(int(np.argmax(x)))
            continue
        order = np.argsort(-x, kind="stable")
        w = np.exp((x[order] - x[order[0]]) / value("temperature", r))
        keep = len(w)
        if value("top_k", r):
            keep = min(keep, value("top_k", r))
        p = value("top_p", r)
        if p is not None and p < 1:
            c = np.cumsum(w[:keep])
            keep = 1 + int(np.searchsorted(c[:-1], p * c[-1], side="left")) if keep > 1 else keep
        if value("min_p", r):
            keep = int(np.count_nonzero(w[:keep] >= value("min_p", r)))
        chosen = np.sort(order[:keep])
        c = np.cumsum(np.exp((x[chosen] - x[order[0]]) / value("temperature", r)))
        tokens.append(int(chosen[min(np.searchsorted(c, value("uniforms", r) * c[-1], side="right"), keep - 1)]))
    return torch.tensor(tokens, dtype=torch.int32)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s, case)
    if case["op"] == "attention":
        return _exact_attention(s, case)
    if case["op"] == "rotary":
        return [_exact_rotated(s[name], s["positions"], case["rotary_dim"], case["pairs"], case["scaling"])
                for name in ("q", "k")]
    turn = lambda x: _exact_rotated(x, s["positions"], case["rotary_dim"], case["pairs"], "none")  # noqa: E731
    k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    slots = (s["slots"] if s["slots"] is not None else s["positions"]).cpu().tolist()
    pages, k, v = s["page_table"].cpu().numpy(), turn(s["k"]), s["v"].double()
    seqs = s["seq_ids"].cpu().tolist()
    page = torch.tensor([int(pages[b, t // case["page"]]) for b, t in zip(seqs, slots)], device=k.device)
    off = torch.tensor([t % case["page"] for t in slots], device=k.device)
    k_pages.transpose(1, 2)[page, off] = k
    v_pages.transpose(1, 2)[page, off] = v
    return [turn(s["q"]), k_pages, v_pages]
