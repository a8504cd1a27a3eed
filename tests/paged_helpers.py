"""Paged caches with known contents, and their operators by definition in 64 bits."""
import math

import torch

from dawn_srw_b200.ops import paged as P

KINDS = ("bf16", "e4m3", "int8")


def make_cache(kind, lengths, H, dh, page, device, seed=0, spare=3, width=None, garbage=True, least_pages=0):
    """Pages of sequences of the given lengths at shuffled places of the pool.  Slots behind a length and spare
    pages hold NaN (8-bit kinds: any codes under a NaN scale), table entries behind it name no page."""
    gen = torch.Generator().manual_seed(seed)
    used = [-(-n // page) for n in lengths]
    n_pages = max(sum(used) + spare, least_pages)
    order = torch.randperm(n_pages, generator=gen)
    width = width if width is not None else max(used + [0]) + 1
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = order[at: at + u].int()
        at += u
    c = {"table": table.to(device), "lengths": torch.tensor(lengths, dtype=torch.int32).to(device)}
    live = torch.zeros(n_pages, page, dtype=torch.bool)
    for b, n in enumerate(lengths):
        for i in range(used[b]):
            live[table[b, i].long(), : max(0, min(page, n - i * page))] = True
    live = live[:, None, :, None].to(device)
    g = torch.Generator(device=device).manual_seed(seed + 1)
    for name in ("k", "v"):
        x = torch.randn(n_pages, H, page, dh, generator=g, device=device) * (1.3 if name == "k" else 0.8)
        codes, scale = P.encode_rows(x, P.PAGE_DTYPES[kind])
        if garbage and kind == "bf16":
            codes = torch.where(live, codes, torch.full_like(codes, math.nan))
        elif garbage:
            scale = torch.where(live[..., 0], scale, torch.full_like(scale, math.nan))
        c[name + "_pages"], c[name + "_scale"] = codes.contiguous(), None if scale is None else scale.contiguous()
    return c


def starts_of(new, device):
    return torch.tensor([0] + list(new)).cumsum(0).to(torch.int32).to(device)


def args(c):
    return [c[k] for k in ("k_pages", "v_pages", "table", "lengths")]


def scales(c):
    return {k: c[k] for k in ("k_scale", "v_scale")}


def held64(c, b, n, name):
    """Positions 0..n-1 of sequence b in 64 bits: [n, H, dh]."""
    pages, scale = c[name + "_pages"], c[name + "_scale"]
    page = pages.shape[2]
    pos = torch.arange(n, device=pages.device)
    ids = c["table"][b].long()[pos // page].clamp(min=0)
    raw = pages.view(torch.uint8 if pages.element_size() == 1 else torch.int16)[ids, :, pos % page].view(pages.dtype)
    x = raw.double()
    return x if scale is None else x * scale[ids, :, pos % page].double()[..., None]


def attention64(q, c, new, window=None, sinks=0, scale=None):
    """(result, sum of p |v|) of every packed row, by definition; rows without a key are zero."""
    N, Hq, dh = q.shape
    H = c["k_pages"].shape[1]
    out = torch.zeros(N, Hq, dh, dtype=torch.double, device=q.device)
    mag = torch.zeros_like(out)
    scale = 1.0 / math.sqrt(dh) if scale is None else scale
    at = 0
    for b, n in enumerate(new):
        length = int(c["lengths"][b])
        k, v = held64(c, b, length, "k"), held64(c, b, length, "v")
        for i in range(n):
            p = length - n + i
            if p >= 0:
                j = torch.arange(p + 1, device=q.device)
                keep = torch.ones_like(j, dtype=torch.bool) if window is None else (j > p - window) | (j < sinks)
                kk, vv = k[j[keep]], v[j[keep]]                               # [n, H, dh]
                s = torch.einsum("hgd,nhd->hgn", q[at + i].double().view(H, Hq // H, dh), kk) * scale
                w = torch.softmax(s, -1)
                out[at + i] = torch.einsum("hgn,nhd->hgd", w, vv).reshape(Hq, dh)
                mag[at + i] = torch.einsum("hgn,nhd->hgd", w, vv.abs()).reshape(Hq, dh)
        at += n
    return out, mag


def largest_score(q, c, new, scale=None):
    """The largest scale * sum |q| |k| of any row and any position of its sequence."""
    H, G = c["k_pages"].shape[1], q.shape[1] // c["k_pages"].shape[1]
    scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else abs(scale)
    most, at = 0.0, 0
    for b, n in enumerate(new):
        if n and int(c["lengths"][b]):
            k = held64(c, b, int(c["lengths"][b]), "k").abs()
            s = torch.einsum("rhgd,nhd->rhgn", q[at: at + n].double().abs().view(n, H, G, -1), k)
            most = max(most, float(s.max()) * scale)
        at += n
    return most


def assert_attention(got, ref, mag, rounded_scores=0.0):
    """A bf16 result of bf16 operands: each weight is rounded to bf16 once (2^-8 of it at most, so 2^-8 of
    sum p |v|), the result once (2^-8 of it); what is left is fp32 (scores of magnitude below 100 from sums of
    at most 128 products: below 2^-12 of a weight).

    Over 8-bit pages the weights are fp16 (2^-11), and a chunk's int8 keys and values, code * scale, are rounded
    to fp16 too: 2^-11 of sum p |v| for the values, and a score moves by 2^-11 of scale * sum |q| |k| =: A at most,
    a weight by that and, through the sum of all, by that again.  2^-11 (2 + 2 A) is within the 2^-8 above while
    A <= 3 even if all roundings have one sign; rows of random numbers, whose roundings have not, stay far below it
    at A of 10.  Where scores are made large on purpose, ``rounded_scores`` = A adds the term 2 * 2^-11 A, with
    another 1 + 2^-11 A for the exponential's second order (A below 100)."""
    assert got.dtype == torch.bfloat16
    err = (got.double() - ref).abs()
    tol = ref.abs() * 2.0 ** -8 + mag * (2.0 ** -8 + 2.0 ** -12) * (1 + 2.0 ** -8)
    tol = tol + mag * 2.0 ** -10 * rounded_scores * (1 + 2.0 ** -11 * rounded_scores)
    bad = ~(err <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float((err - tol)[bad].max()), bad.nonzero()[:4].tolist())
