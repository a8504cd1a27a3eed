"""Paged key/value cache in plain PyTorch: the definition that the kernels of
``csrc/paged_kernels.cu`` are tested against, and the path of CPU runs.

Pages of keys and values are ``[n_pages, H, page, dh]``: bf16, or 8-bit codes (``float8_e4m3fn``,
``int8``) with fp32 scales ``[n_pages, H, page]``, one for each position and head.  ``table [B, width]``
(int32) names the page of positions ``i * page .. (i + 1) * page`` of a sequence, ``lengths [B]`` (int32)
its positions, new tokens included.  The new tokens of all sequences are packed: rows ``starts[b] ..
starts[b + 1]`` (ascending) are the last tokens of sequence ``b``; ``starts`` is None where every sequence
has one.  Sequences may share pages that they read.  No two rows that one call writes may have one place: the
plain path refuses them, the kernels do not look and would mix the two.

A row of keys or values is stored with one rounding: bf16; e4m3 after division by the smallest power of
two that brings the row's largest magnitude to 448 or less; or int8, ``round(x * (127 / largest))`` with
the scale ``largest / 127``.  A row whose values are all below 2^-100 is stored as zeros with scale 1, a
row with a NaN or an infinity as zeros with scale NaN (it reads back as NaN).

The reference's caches are dense, fp32 and of one length for the whole batch
(models/dawn_spatial_v41_exp.py:1772-1957); they have no counterpart of this.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

PAGE_DTYPES = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
SMALLEST = 2.0 ** -100


def _refuse_unless(ok: bool, msg: str) -> None:
    if not ok:
        raise ValueError("paged cache: " + msg)


def check_cache(k_pages, v_pages, table, lengths, starts, k_scale, v_scale, rows: int) -> None:
    """What the kernels' bindings check too, but for the head dimensions, sizes (more than 65535 sequences or
    heads, 2^30 rows or positions) and pages or scales off a 16-byte border that only they cannot take."""
    _refuse_unless(k_pages.dim() == 4 and k_pages.shape == v_pages.shape and k_pages.dtype == v_pages.dtype,
                   "k and v pages must have one shape [n_pages, heads, page, dim] and one type")
    _refuse_unless(k_pages.is_contiguous() and v_pages.is_contiguous(), "pages must be contiguous")
    _refuse_unless(k_pages.dtype in PAGE_DTYPES.values(), "pages must be bfloat16, float8_e4m3fn or int8")
    page = k_pages.shape[2]
    _refuse_unless(16 <= page <= 256 and page & (page - 1) == 0,
                   f"page size {page} is not a power of two from 16 to 256")
    scaled = k_pages.dtype != torch.bfloat16
    _refuse_unless((k_scale is not None) == scaled and (v_scale is not None) == scaled,
                   "8-bit pages come with k_scale and v_scale, bf16 pages without")
    for s in (k_scale, v_scale) if scaled else ():
        _refuse_unless(s.dtype == torch.float32 and s.is_contiguous() and s.shape == k_pages.shape[:3]
                       and s.device == k_pages.device,
                       "scales must be contiguous float32 [n_pages, heads, page] on the pages' device")
    _refuse_unless(table.dim() == 2 and table.dtype == torch.int32 and table.is_contiguous(),
                   "table must be a contiguous int32 [sequences, pages]")
    B = table.shape[0]
    _refuse_unless(lengths.shape == (B,) and lengths.dtype == torch.int32 and lengths.is_contiguous(),
                   "lengths must be a contiguous int32 [sequences]")
    if starts is not None:
        _refuse_unless(starts.shape == (B + 1,) and starts.dtype == torch.int32 and starts.is_contiguous()
                       and starts.device == k_pages.device,
                       "starts must be a contiguous int32 [sequences + 1] on the pages' device")
    else:
        _refuse_unless(rows == B, f"without starts every sequence has one new token: {rows} rows for {B} sequences")
    _refuse_unless(k_pages.device == v_pages.device == table.device == lengths.device,
                   "pages, table and lengths must be on one device")


def _check_rows(x, pages, name: str) -> None:
    _refuse_unless(x.dim() == 3 and x.shape[2] == pages.shape[3],
                   f"{name} must be [rows, heads, dim] with the pages' head dimension")
    _refuse_unless(x.dtype in (torch.float32, torch.bfloat16), f"{name} must be float32 or bfloat16")
    _refuse_unless(x.device == pages.device, f"{name} must be on the pages' device")


def encode_rows(x: torch.Tensor, dtype: torch.dtype) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(codes, scales) of rows x [..., dh] as pages of ``dtype`` hold them; no scales for bf16."""
    x = x.float()
    if dtype == torch.bfloat16:
        return x.to(dtype), None
    amax = x.abs().amax(-1, keepdim=True)                    # NaN where a value is
    odd = ~torch.isfinite(amax)
    some = ~odd & (amax >= SMALLEST)
    one = torch.ones_like(amax)
    if dtype == torch.float8_e4m3fn:
        m, e = torch.frexp(torch.where(some, amax, one))
        scale = torch.where(some, torch.ldexp(one, torch.where(m <= 0.875, e - 9, e - 8)), one)
        codes = torch.where(odd, 0.0, x / scale).to(dtype)
    else:
        most = torch.full_like(amax, 127.0)                  # a tensor: torch multiplies by a number's reciprocal
        scale = torch.where(some, amax / most, one)
        inv = torch.where(some, most / amax, one)
        codes = torch.where(odd, 0.0, x * inv).round().to(dtype)
    return codes, torch.where(odd, math.nan, scale)[..., 0]


def decode_rows(codes: torch.Tensor, scale: Optional[torch.Tensor]) -> torch.Tensor:
    """The fp32 values that codes [..., dh] with scales [...] stand for."""
    return codes.float() if scale is None else codes.float() * scale.unsqueeze(-1)


def _raw(pages):
    """Indexing works on integers of the same width for every type."""
    return pages.view(torch.uint8 if pages.element_size() == 1 else torch.int16)


def _valid_lengths(table, lengths, page: int):
    return lengths.long().clamp(0, table.shape[1] * page)


def _places(table, lengths, starts, rows: int, page: int):
    """(sequence, position) of every packed row; position -1 for a row of no sequence or before its first position."""
    row = torch.arange(rows, device=table.device)
    if starts is None:
        seq, back = row, torch.ones_like(row)
    else:
        s = starts.long().clamp(0, rows)
        seq = torch.searchsorted(s, row, right=True) - 1
        inside = (seq >= 0) & (seq < table.shape[0])
        seq = torch.where(inside, seq, torch.full_like(seq, -1))
        back = s[(seq + 1).clamp(max=len(s) - 1)] - row
    at = _valid_lengths(table, lengths, page)
    pos = at[seq.clamp(min=0)] - back if len(at) else torch.full_like(row, -1)
    return seq, torch.where(seq >= 0, pos, torch.full_like(pos, -1)).clamp(min=-1)


def write(k, v, k_pages, v_pages, table, lengths, starts=None, k_scale=None, v_scale=None) -> None:
    _refuse_unless(k_pages.dim() == 4, "pages must be [n_pages, heads, page, dim]")
    _check_rows(k, k_pages, "k")
    _check_rows(v, k_pages, "v")
    _refuse_unless(k.shape == v.shape and k.dtype == v.dtype and k.shape[1] == k_pages.shape[1],
                   "k and v must have one type and one shape with the pages' heads")
    check_cache(k_pages, v_pages, table, lengths, starts, k_scale, v_scale, k.shape[0])
    page = k_pages.shape[2]
    seq, pos = _places(table, lengths, starts, k.shape[0], page)
    there = pos >= 0
    seq, pos = seq[there], pos[there]
    ids = table[seq, pos // page].long()
    _refuse_unless(bool(((ids >= 0) & (ids < k_pages.shape[0])).all()), "a table entry names no page")
    slot = pos % page
    _refuse_unless(len((ids * page + slot).unique()) == len(ids), "two rows have one place")
    for x, pages, scales in ((k, k_pages, k_scale), (v, v_pages, v_scale)):
        codes, scale = encode_rows(x[there], pages.dtype)
        _raw(pages)[ids, :, slot] = _raw(codes)
        if scale is not None:
            scales[ids, :, slot] = scale


def _dense(k_pages, v_pages, table, lengths, k_scale, v_scale, max_len: int):
    page, B = k_pages.shape[2], table.shape[0]
    n = _valid_lengths(table, lengths, page)
    pos = torch.arange(max_len, device=table.device)
    there = pos < n[:, None]                                            # [B, max_len]
    used = table[:, : -(-max_len // page)].long()
    named = there[:, ::page][:, : used.shape[1]]                         # a page counts if its first position does
    _refuse_unless(bool((~named | ((used >= 0) & (used < k_pages.shape[0]))).all()), "a table entry names no page")
    ids = torch.where(named, used, torch.zeros_like(used))
    out = []
    for pages, scales in ((k_pages, k_scale), (v_pages, v_scale)):
        x = k_pages.new_zeros((B, pages.shape[1], max_len, pages.shape[3]), dtype=torch.float32)
        if ids.numel() and pages.shape[0]:
            got = _raw(pages)[ids].view(pages.dtype)
            g = decode_rows(got, None if scales is None else scales[ids])
            g = g.transpose(1, 2).flatten(2, 3)[:, :, :max_len]
            x[:, :, : g.shape[2]] = torch.where(there[:, None, : g.shape[2], None], g, 0.0)
        out.append(x)
    return out


def read(k_pages, v_pages, table, lengths, max_len: int, k_scale=None, v_scale=None, dtype=torch.float32):
    _refuse_unless(max_len >= 0, f"max_len {max_len}")
    _refuse_unless(dtype in (torch.float32, torch.bfloat16), "dtype must be float32 or bfloat16")
    check_cache(k_pages, v_pages, table, lengths, None, k_scale, v_scale, table.shape[0] if table.dim() == 2 else 0)
    return tuple(t.to(dtype) for t in _dense(k_pages, v_pages, table, lengths, k_scale, v_scale, max_len))


def attention(q, k_pages, v_pages, table, lengths, starts=None, k_scale=None, v_scale=None, *,
              max_new: Optional[int] = None, window: Optional[int] = None, sinks: int = 0,
              scale: Optional[float] = None) -> torch.Tensor:
    """fp32 in, q's type out; a sequence at a time (padded to nothing)."""
    _refuse_unless(k_pages.dim() == 4, "pages must be [n_pages, heads, page, dim]")
    _check_rows(q, k_pages, "q")
    Hq, H = q.shape[1], k_pages.shape[1]
    _refuse_unless(Hq >= 1 and H >= 1 and Hq % H == 0, f"{Hq} query heads are no multiple of the pages' {H} heads")
    _refuse_unless(window is None or window >= 1, "window must be at least 1 (None: no window)")
    _refuse_unless(sinks >= 0, "sinks must not be negative")
    _refuse_unless(max_new is None or max_new >= 0, "max_new must not be negative")
    check_cache(k_pages, v_pages, table, lengths, starts, k_scale, v_scale, q.shape[0])
    seq, pos = _places(table, lengths, starts, q.shape[0], k_pages.shape[2])
    scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float32, device=q.device)
    G = Hq // H
    for b in seq[pos >= 0].unique().tolist():
        mine = (seq == b) & (pos >= 0)
        p, n = pos[mine], int(pos[mine].max()) + 1
        key = torch.arange(n, device=q.device)
        sees = key <= p[:, None]
        used = torch.ones(n, dtype=torch.bool, device=q.device)
        if window is not None:
            sees &= (key > p[:, None] - window) | (key < sinks)
            used = sees.any(0)
        # pages that no row sees may be gone from the table
        page = k_pages.shape[2]
        first = torch.where(used, key, torch.zeros_like(key))
        ids = table[b].long()[first // page]
        _refuse_unless(bool((~used | ((ids >= 0) & (ids < k_pages.shape[0]))).all()), "a table entry names no page")
        ids, slot = torch.where(used, ids, torch.zeros_like(ids)), first % page
        kv = []
        for pages, scales in ((k_pages, k_scale), (v_pages, v_scale)):
            x = decode_rows(_raw(pages)[ids, :, slot].view(pages.dtype), None if scales is None else scales[ids, :, slot])
            kv.append(torch.where(used[:, None, None], x, 0.0).transpose(0, 1))          # [H, n, dh]
        rows = q[mine].float().view(len(p), H, G, -1).transpose(0, 1)                   # [H, rows, G, dh]
        s = torch.einsum("hrgd,hnd->hrgn", rows, kv[0]) * scale
        s = s.masked_fill(~sees[None, :, None], -math.inf)
        w = torch.softmax(s, -1)
        # a weight of zero does not keep a value that is no number away from a row that does not see it
        odd = ~torch.isfinite(kv[1])
        o = torch.einsum("hrgn,hnd->hrgd", w, torch.where(odd, 0.0, kv[1]))
        for j in odd.any(-1).any(0).nonzero().flatten().tolist():
            part = w[..., j, None] * kv[1][:, None, None, j]
            o += torch.where(odd[:, None, None, j] & sees[None, :, None, j, None], part, 0.0)
        out[mine] = o.transpose(0, 1).reshape(len(p), Hq, -1)
    return out.to(q.dtype)
