"""64-bit plain forms of the paged-cache serving operators, on the CPU, one element or
row at a time from the definitions, and their tolerances.

Tolerances count roundings: storing a value in type t is off by at most
torch.finfo(t).eps / 2 of it (bf16 2^-8, fp32 2^-24)."""
from __future__ import annotations

import math

import numpy as np
import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def frequencies(dim, theta, kind="none", factor=1.0, original_max_pos=0, low=1.0, high=4.0):
    out = []
    for i in range(dim // 2):
        base = theta * factor ** (dim / (dim - 2.0)) if kind == "ntk" else theta
        f = base ** (-2.0 * i / dim)
        if kind == "linear":
            f /= factor
        elif kind == "bands":
            wave = 2 * math.pi / f
            if wave > original_max_pos / low:
                f /= factor
            elif wave >= original_max_pos / high:
                smooth = (original_max_pos / wave - low) / (high - low)
                f = (1 - smooth) * f / factor + smooth * f
        elif kind == "yarn":
            def edge(turns):
                return dim * math.log(original_max_pos / (turns * 2 * math.pi)) / (2 * math.log(theta))

            a, b = max(math.floor(edge(low)), 0), min(math.ceil(edge(high)), dim - 1)
            r = min(max((i - a) / max(b - a, 0.001), 0.0), 1.0)
            f = (1 - r) * f + r * f / factor
        out.append(f)
    return np.array(out)


def rotated(x, positions, freq, mscale, interleaved):
    """(rotated x in 64 bits, |a| + |b| of each element's pair: 0 where it is copied)."""
    x = x.detach().cpu().double().numpy()
    out, pair = x.copy(), np.zeros_like(x)
    half = len(freq)
    angle = np.asarray(positions, dtype=np.float64)[:, None] * freq[None]
    c, s = mscale * np.cos(angle)[:, None], mscale * np.sin(angle)[:, None]
    i, j = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    a, b = x[..., i], x[..., j]
    out[..., i], out[..., j] = a * c - b * s, b * c + a * s
    pair[..., i] = pair[..., j] = np.abs(a) + np.abs(b)
    return out, pair


def rotation_tolerance(want, pair, mscale, dtype):
    """The table's fp32 rounding (2^-24 of |c| and |s| <= mscale), one rounded product, one
    fused multiply-add: at most 3 * 2^-24 mscale (|a| + |b|); a factor of 4 covers the
    products of these and 64-bit angles up to 2^20 (2^-32). Then the storage rounding;
    copied elements are exact."""
    moved = pair > 0
    return np.where(moved, HALF[dtype] * np.abs(want) * (1 + 2.0 ** -7) + 4 * 2.0 ** -24 * mscale * pair + 2.0 ** -32, 0.0)


def tree_bits(parents, words):
    """int64 [n, words]: bit j of row i is set for i's ancestors j and i itself."""
    out = np.zeros((len(parents), words), dtype=np.uint64)
    for i in range(len(parents)):
        j = i
        while j >= 0:
            out[i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
            j = parents[j]
    return torch.from_numpy(out.view(np.int64).copy())


def attention(q, k_pages, v_pages, page_table, seqs, ctxs, starts, mask, scale, dtype, tensor_cores):
    """(out, tolerance) in 64 bits, rows outside every sequence zero; mask: bool function
    (row, i, j)."""
    rows, hq, hd = q.shape
    hkv, page = k_pages.shape[1], k_pages.shape[2]
    group = hq // hkv
    out, tol = np.zeros((rows, hq, hd)), np.zeros((rows, hq, hd))
    q = q.detach().cpu().double().numpy()
    k_pages, v_pages = (t.detach().cpu().double() for t in (k_pages, v_pages))
    page_table = page_table.cpu().numpy()
    for b, ctx in enumerate(ctxs):
        n = starts[b + 1] - starts[b]
        if n == 0:
            continue
        slots = np.arange(ctx + n)
        ids = torch.from_numpy(page_table[seqs[b]][slots // page].astype(np.int64))
        off = torch.from_numpy(slots % page)
        k, v = (t[ids, :, off].numpy() for t in (k_pages, v_pages))  # [slots, hkv, hd]
        seen = np.zeros((n, ctx + n), dtype=bool)
        seen[:, :ctx] = True
        for i in range(n):
            for j in range(n):
                seen[i, ctx + j] = mask(starts[b] + i, i, j)
        for h in range(hq):
            kh, vh = k[:, h // group], v[:, h // group]
            qh = q[starts[b]:starts[b] + n, h]
            s = np.where(seen, qh @ kh.T * scale, -np.inf)
            size = np.abs(qh) @ np.abs(kh).T * scale
            top = s.max(-1, keepdims=True, initial=-np.inf)
            p = np.where(seen, np.exp(s - np.where(np.isfinite(top), top, 0.0)), 0.0)
            total = p.sum(-1, keepdims=True)
            p = np.divide(p, total, out=np.zeros_like(p), where=total > 0)
            o = p @ vh
            # A score is a sum of hd fp32 products (q times scale rounded first): off by at
            # most (hd + 2) 2^-24 of its absolute terms; weights and sums of len terms by
            # 2^-21 and len 2^-24 of themselves; bf16 weights by half a step each.
            ds = (hd + 2) * 2.0 ** -24 * size.max(-1, keepdims=True, initial=0.0)
            rel = 2 * ds + 2.0 ** -21 + (ctx + n) * 2.0 ** -24 + (HALF[torch.bfloat16] if tensor_cores else 0.0)
            out[starts[b]:starts[b] + n, h] = o
            tol[starts[b]:starts[b] + n, h] = rel * (p @ np.abs(vh)) * 1.01 + HALF[dtype] * np.abs(o) * 1.01
    return out, tol


def sample(logits, uniforms, temperature, top_k, top_p, min_p):
    """The tokens, one row at a time in 64 bits."""
    out = []
    x_all = logits.detach().cpu().float().double().numpy()
    for r in range(x_all.shape[0]):
        x = np.where(np.isnan(x_all[r]), -np.inf, x_all[r])
        t, k, p, m, u = (None if a is None else a[r].item() for a in (temperature, top_k, top_p, min_p, uniforms))
        t = 1.0 if t is None else t
        if not t >= 0 or not 0 <= u < 1 or (p is not None and p != p) or (m is not None and m != m):
            out.append(-1)
            continue
        order = np.argsort(-x, kind="stable")
        top = x[order[0]]
        if top == -np.inf:
            out.append(-1)
            continue
        if t == 0:
            out.append(int(order[0]))
            continue
        with np.errstate(invalid="ignore", over="ignore"):
            w = np.where(x == top, 1.0, np.where((x == -np.inf) | (top == np.inf), 0.0, np.exp((x - top) / t)))[order]
        keep = len(w)
        if k is not None and 0 < k < keep:
            keep = k
        if p is not None and p < 1:
            total, run = math.fsum(w[:keep]), 0.0
            for i in range(keep):
                if i > 0 and not run < p * total:
                    keep = i
                    break
                run = math.fsum((run, w[i])) if keep < 2000 else run + w[i]
        if m is not None and m > 0:
            keep = max(1, int(np.count_nonzero(w[:keep] >= min(m, 1.0))))
        index = np.argsort(order[:keep])
        chosen, weights = order[:keep][index], w[:keep][index]
        c = np.cumsum(weights)
        at = int(np.searchsorted(c, u * c[-1], side="right"))
        out.append(int(chosen[min(at, keep - 1)]))
    return out
