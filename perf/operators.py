"""The operators of the paged key/value cache, as timed cases.

A serving process keeps the keys and values of its sequences in pages ``[n_pages, H, page, dh]`` (bf16,
or 8-bit codes with one fp32 scale per position and head ``[n_pages, H, page]``), which page holds which
positions in a table ``[B, P]``, and the lengths ``[B]`` of the sequences, new tokens included.  New
tokens come packed: those of sequence ``b`` are rows ``starts[b] .. starts[b + 1]`` and the last ones of
its length (``starts`` is None where every sequence has exactly one).

* write: keys and values ``[N, H, dh]`` go into their pages, rounded to the pages' type;
* read: pages come back as dense ``[B, H, max_len, dh]``, zeros behind a length;
* attend: softmax(scale q k^T) v of the new tokens over the pages, causal, with an optional window and
  first positions that stay visible (sinks).

``run`` computes them in plain torch, or, with ``own``, by the framework's backend.
"""
import functools
import math
import random

import torch

own = False

BYTES = {"bf16": 2, "e4m3": 1, "int8": 1}
CODES = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
PLAIN = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _case(name, op, kv, batch, heads, dim, page, ctx, new=(1, 1), group=1, window=0, sinks=0, io="bf16"):
    """``ctx``, ``new``: smallest and largest length and number of new tokens of a sequence; ``heads``:
    heads of the cache, each read by ``group`` query heads; ``io``: type of what is written or read."""
    return dict(name=name, op=op, kv=kv, batch=batch, heads=heads, group=group, dim=dim, page=page,
                ctx_lo=ctx[0], ctx_hi=ctx[1], new_lo=new[0], new_hi=new[1], window=window, sinks=sinks, io=io)


def listed():
    return [
        # one user's newest token on the smallest model (6 heads of 64): latency
        _case("write_40M_1", "write", "bf16", 1, 6, 64, 16, (290, 290), io="fp32"),
        # the prompts of a batch on the largest model (16 heads of 128), stored in 8 bits and read back
        _case("write_1B_prompts", "write", "e4m3", 24, 16, 128, 32, (37, 512), (37, 512), io="fp32"),
        # a few sequences of the flagship model (16 heads of 80) back into dense fp32 caches
        _case("read_400M_5", "read", "bf16", 5, 16, 80, 16, (60, 512), io="fp32"),
        # many longer ones, kept in 8 bits
        _case("read_1B_40", "read", "int8", 40, 16, 128, 64, (100, 2000), io="bf16"),
        # single tokens: one user on the smallest model, a serving batch on the largest one
        _case("decode_40M_1", "attend", "bf16", 1, 6, 64, 16, (290, 290)),
        _case("decode_1B_32", "attend", "bf16", 32, 16, 128, 16, (100, 512)),
        # ragged long contexts in 8 bits on the flagship's heads
        _case("decode_400M_long", "attend", "e4m3", 6, 16, 80, 64, (2000, 32000)),
        # shared heads, a window and sinks over contexts of up to 40 k positions
        _case("decode_shared_window", "attend", "int8", 16, 4, 128, 64, (1000, 40000), group=8, window=4096, sinks=4),
        # a handful of drafted tokens to verify per sequence
        _case("verify_5", "attend", "bf16", 8, 8, 64, 16, (200, 6000), (5, 5), group=2),
        # prompts: a chunk over what is cached of it, a ragged batch of whole ones, a long one under a window
        _case("chunk_400M_512", "attend", "e4m3", 1, 16, 80, 64, (2100, 2100), (512, 512)),
        _case("prompts_1B_ragged", "attend", "bf16", 5, 16, 128, 32, (301, 2048), (301, 2048)),
        _case("chunk_shared_window", "attend", "int8", 1, 4, 64, 64, (16000, 16000), (4099, 4099), group=4,
              window=6000, sinks=64),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["write", "read", "decode", "decode", "verify", "chunk", "chunk"])
    kv = rng.choice(["bf16", "e4m3", "int8"])
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128])
    heads, group = rng.choice([(6, 1), (16, 1), (16, 1), (8, 2), (4, 8), (3, 5), (8, 4)])
    page = rng.choice([16, 32, 64, 128])
    batch = _log_int(rng, 1, 48)
    hi = _log_int(rng, 16, {"write": 4000, "read": 4000, "verify": 30000, "decode": 40000, "chunk": 16000}[kind])
    lo = _log_int(rng, 1, hi)
    new = (1, 1)
    if kind == "verify":
        new = (rng.randint(1, 3), rng.randint(3, 12))
    elif kind == "chunk" or (kind == "write" and rng.random() < 0.7):
        n = _log_int(rng, 8, min(hi, 4099))
        new = (rng.choice([0, 1, n // 3, n]), n)
    window = sinks = 0
    if kind not in ("write", "read") and rng.random() < 0.4:
        window, sinks = _log_int(rng, 5, 8000), rng.choice([0, 1, 4, 100])
    case = _case("", "attend", kv, batch, heads, dim, page, (lo, hi), new, group, window, sinks,
                 rng.choice(["bf16", "fp32"]))
    case["op"] = kind if kind in ("write", "read") else "attend"
    if case["op"] == "attend":
        case["io"] = "bf16"
    else:
        case["group"] = 1
    while _cost(case) > 1.0:                       # fewer, then shorter sequences
        if case["batch"] > 1:
            case["batch"] = case["batch"] // 2
        else:
            for key in ("ctx_lo", "ctx_hi", "new_lo", "new_hi"):
                case[key] = (case[key] + 1) // 2
    del case["name"]
    return case


def _cost(case):
    """Share of the largest listed case, in work and in what the plain form needs room for."""
    w = work(case)
    total, new = _lengths(case)
    rows = max(new) * case["heads"] * case["group"] if case["op"] == "attend" else 0
    room = 4 * case["batch"] * max(total) * max(rows, 4 * case["heads"] * case["dim"])
    return max(w["bytes"] / 1e9, w["flops"] / 1.2e11, room / 6e9)


def _lengths(case):
    """(length, new tokens) of every sequence: spread over the logarithm, the first the longest."""
    r = random.Random(repr((case["batch"], case["ctx_lo"], case["ctx_hi"], case["new_lo"], case["new_hi"])))
    lo, hi = min(case["ctx_lo"], case["ctx_hi"]), case["ctx_hi"]
    total = [hi] + [_log_int(r, max(1, lo), hi) for _ in range(case["batch"] - 1)]
    a, b = min(case["new_lo"], case["new_hi"]), case["new_hi"]
    new = [min(t, n) for t, n in zip(total, [b] + [r.randint(a, b) for _ in range(case["batch"] - 1)])]
    whole = b > 1 and (a, b) == (lo, hi)           # prompts of which nothing is cached yet
    return total, list(total) if whole else new


def _visible(t, n, window, sinks):
    """(pairs, keys): how many (token, key) pairs the last ``n`` of ``t`` positions see, and how many keys any does."""
    if n == 0:
        return 0, 0
    if not window:
        return n * (t - n) + n * (n + 1) // 2, t
    pairs = sum(min(p + 1, window) + min(sinks, max(0, p + 1 - window)) for p in range(t - n, t))
    low = max(0, t - n - window + 1)
    return pairs, (t - low) + min(sinks, low)


def work(case):
    total, new = _lengths(case)
    H, dh, size = case["heads"], case["dim"], BYTES[case["kv"]]
    row = H * (dh * size + (4 if size == 1 else 0)) * 2            # keys, values and scales of a position
    io = H * dh * (4 if case["io"] == "fp32" else 2) * 2
    if case["op"] == "write":
        n = sum(new)
        back = case["batch"] * max(total) * H * dh * 4 + row * n if size == 1 else 0
        return {"bytes": n * (row + io) + back, "flops": 0}
    if case["op"] == "read":
        return {"bytes": sum(total) * row + case["batch"] * max(total) * io, "flops": 0}
    seen = [_visible(t, n, case["window"], case["sinks"]) for t, n in zip(total, new)]
    heads = H * case["group"]
    return {"bytes": sum(k for _, k in seen) * row + sum(new) * heads * dh * 4,
            "flops": 4 * heads * dh * sum(p for p, _ in seen)}


# ---------------------------------------------------------------------------
def _encode(x, kv):
    """Rows of x in the pages' type, and their scales (None for bf16): one step's rounding from x.
    e4m3: the smallest power of two that brings the largest value to 448 or less; int8: largest / 127."""
    x = x.float()
    if kv == "bf16":
        return x.to(torch.bfloat16), None
    amax = x.abs().amax(-1, keepdim=True)
    if kv == "e4m3":
        m, e = torch.frexp(amax)
        scale = torch.ldexp(torch.ones_like(amax), torch.where(m <= 0.875, e - 9, e - 8))
        scale = torch.where(amax > 0, scale, torch.ones_like(amax))
        return (x / scale).to(torch.float8_e4m3fn), scale[..., 0]
    some = amax > 0
    scale = torch.where(some, amax / 127, torch.ones_like(amax))
    inv = torch.where(some, 127 / amax, torch.ones_like(amax))
    return (x * inv).round().to(torch.int8), scale[..., 0]


def _decode(codes, scale):
    return codes.float() if scale is None else codes.float() * scale.unsqueeze(-1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)
    total, new = _lengths(case)
    B, H, dh, page, kv = case["batch"], case["heads"], case["dim"], case["page"], case["kv"]
    width = -(-max(total) // page) + 1
    used = [-(-t // page) for t in total]
    n_pages = sum(used) + 3
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed), dtype=torch.int32)
    ids = torch.zeros(B, width, dtype=torch.int32)
    at = 0
    for b, u in enumerate(used):                          # pages of a sequence are anywhere in the pool
        ids[b, :u] = order[at:at + u]
        at += u
    ends = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    ints = lambda v: torch.as_tensor(v, dtype=torch.int32).cuda()
    # keys have channels that stand out, values do not; recycled pages hold what was there before
    k, v = rn(n_pages, H, page, dh), rn(n_pages, H, page, dh)
    k[..., : dh // 16] *= 3.0
    (kp, ks), (vp, vs) = _encode(k, kv), _encode(v, kv)
    del k, v
    s = dict(case=case, table=ids.cuda(), lengths=ints(total), max_len=max(total), max_new=max(new),
             starts=None if new == [1] * B else ends.cuda(), k_pages=kp, v_pages=vp, k_scale=ks, v_scale=vs)
    io, N = PLAIN[case["io"]], sum(new)
    if case["op"] == "write":
        s["k"], s["v"] = rn(N, H, dh).to(io), (rn(N, H, dh) * 0.7).to(io)
    elif case["op"] == "attend":
        # scores with a standard deviation of about one and a half
        s["q"] = (rn(N, H * case["group"], dh) * 1.3).to(io)
    return s


# ---------------------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _backend():
    from dawn_srw_b200.ops.backend import default_backend
    return default_backend("cuda")


def run(state):
    op = state["case"]["op"]
    if op == "write":
        return _write(state)
    if op == "read":
        return _read(state, PLAIN[state["case"]["io"]])
    return _attend(state)


def _write(s):
    if own:
        _backend().paged_write(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["starts"],
                               s["k_scale"], s["v_scale"])
    else:
        seq, pos = _places(s, s["k"].shape[0])
        page = s["k_pages"].shape[2]
        ids, slot = s["table"][seq, pos // page].long(), pos % page
        for x, pages, scales in ((s["k"], s["k_pages"], s["k_scale"]), (s["v"], s["v_pages"], s["v_scale"])):
            codes, scale = _encode(x, s["case"]["kv"])
            if scale is not None:
                scales[ids, :, slot] = scale
                codes, pages = codes.view(torch.uint8), pages.view(torch.uint8)
            pages[ids, :, slot] = codes
    if s["k_scale"] is None:
        return s["k_pages"], s["v_pages"]
    return _read(s, torch.bfloat16)


def _read(s, dtype):
    if own:
        return _backend().paged_read(s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["max_len"],
                                     s["k_scale"], s["v_scale"], dtype)
    return tuple(t.to(dtype) for t in _dense(s))


def _attend(s):
    c = s["case"]
    if own:
        return _backend().paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["starts"],
                                          s["k_scale"], s["v_scale"], max_new=s["max_new"],
                                          window=c["window"] or None, sinks=c["sinks"])
    q = s["q"]
    N, Hq, dh = q.shape
    B, H, G, n = c["batch"], c["heads"], c["group"], s["max_new"]
    k, v = _dense(s)                                                     # [B, H, S, dh]
    seq, pos = _places(s, N)
    first = _index(s, N)
    rows = torch.zeros(B, n, Hq, dh, device=q.device)
    rows[seq, first] = q.float()
    at = torch.full((B, n), -1, dtype=torch.long, device=q.device)
    at[seq, first] = pos
    rows = rows.view(B, n, H, G, dh).transpose(1, 2).reshape(B, H, n * G, dh)
    score = (rows @ k.transpose(-1, -2)) / math.sqrt(dh)                 # [B, H, n G, S]
    key = torch.arange(k.shape[2], device=q.device)
    sees = key <= at[..., None]                                          # [B, n, S]
    if c["window"]:
        sees &= (key > at[..., None] - c["window"]) | (key < c["sinks"])
    sees = sees.repeat_interleave(G, dim=1).unsqueeze(1)
    score.masked_fill_(~sees, float("-inf"))
    top = score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    e = score.sub_(top).exp_()
    o = (e @ v) / e.sum(-1, keepdim=True).clamp(min=1e-30)
    return o.view(B, H, n, G, dh).transpose(1, 2).reshape(B, n, Hq, dh)[seq, first].to(torch.bfloat16)


def _counts(s):
    """New tokens of every sequence."""
    return torch.ones_like(s["lengths"]).long() if s["starts"] is None else s["starts"].diff().long()


def _sequence(s, N):
    """Which sequence each of the N new tokens belongs to."""
    row = torch.arange(N, device="cuda")
    return row if s["starts"] is None else torch.searchsorted(s["starts"].long(), row, right=True) - 1


def _index(s, N):
    """Which of its sequence's new tokens each is."""
    row, seq = torch.arange(N, device="cuda"), _sequence(s, N)
    return torch.zeros_like(row) if s["starts"] is None else row - s["starts"].long()[seq]


def _places(s, N):
    """(sequence, position) of the N new tokens."""
    seq = _sequence(s, N)
    return seq, (s["lengths"].long() - _counts(s))[seq] + _index(s, N)


def _dense(s):
    """Keys and values [B, H, max_len, dh] in fp32, zeros behind a length."""
    page, n = s["k_pages"].shape[2], s["max_len"]
    ids = s["table"][:, : -(-n // page)].long()
    there = (torch.arange(n, device="cuda") < s["lengths"][:, None])[:, None, :, None]
    out = []
    for pages, scales in ((s["k_pages"], s["k_scale"]), (s["v_pages"], s["v_scale"])):
        got = pages.view(torch.uint8 if pages.element_size() == 1 else torch.int16)[ids].view(pages.dtype)
        x = _decode(got, None if scales is None else scales[ids])
        x = x.transpose(1, 2).flatten(2, 3)[:, :, :n]
        out.append(torch.where(there, x, 0.0))
    return out


# ---------------------------------------------------------------------------
def exact(case, seed):
    """The same by definition, sequence by sequence, in 64 bits."""
    s = prepare(case, seed)
    total, new = _lengths(case)
    table, page = s["table"].cpu(), case["page"]
    value = lambda codes, scale: codes.double() if scale is None else codes.double() * scale.double()[..., None]

    def held(b, name):                                   # [H, length, dh]
        ids = table[b, : -(-total[b] // page)].long().cuda()
        pages, scales = s[name + "_pages"], s[name + "_scale"]
        raw = pages.view(torch.uint8 if pages.element_size() == 1 else torch.int16)[ids].view(pages.dtype)
        x = value(raw, None if scales is None else scales[ids])
        return x.permute(1, 0, 2, 3).reshape(x.shape[1], -1, x.shape[3])[:, : total[b]]

    if case["op"] == "write":
        results = []
        for name in ("k", "v"):
            x, at = s[name].double(), 0
            stored = _stored64(x, case["kv"])
            if case["kv"] == "bf16":
                pages = s[name + "_pages"].double()
                for b in range(case["batch"]):
                    p = torch.arange(total[b] - new[b], total[b])
                    pages[table[b].long()[p // page].cuda(), :, (p % page).cuda()] = stored[at: at + new[b]]
                    at += new[b]
                results.append(pages)
            else:
                dense = torch.zeros(case["batch"], x.shape[1], max(total), x.shape[2], dtype=torch.double, device="cuda")
                for b in range(case["batch"]):
                    dense[b, :, : total[b]] = held(b, name)
                    dense[b, :, total[b] - new[b]: total[b]] = stored[at: at + new[b]].transpose(0, 1)
                    at += new[b]
                results.append(dense)
        return tuple(results)
    if case["op"] == "read":
        results = []
        for name in ("k", "v"):
            dense = torch.zeros(case["batch"], case["heads"], max(total), case["dim"], dtype=torch.double, device="cuda")
            for b in range(case["batch"]):
                dense[b, :, : total[b]] = held(b, name)
            results.append(dense)
        return tuple(results)
    q, at, G = s["q"].double(), 0, case["group"]
    out = torch.zeros_like(q)
    for b in range(case["batch"]):
        k, v = held(b, "k"), held(b, "v")
        for i in range(0, new[b], 256):                  # 256 tokens at a time
            n = min(256, new[b] - i)
            p = total[b] - new[b] + i + torch.arange(n, device="cuda")
            j = torch.arange(total[b], device="cuda")
            mask = j[None] <= p[:, None]
            if case["window"]:
                mask &= (j[None] > p[:, None] - case["window"]) | (j[None] < case["sinks"])
            for h in range(case["heads"]):
                rows = q[at + i: at + i + n, h * G: (h + 1) * G]                     # [n, G, dh]
                a = torch.einsum("ngd,sd->ngs", rows, k[h]) / math.sqrt(case["dim"])
                a = torch.softmax(a.masked_fill(~mask[:, None], -math.inf), -1)
                out[at + i: at + i + n, h * G: (h + 1) * G] = torch.einsum("ngs,sd->ngd", a, v[h])
        at += new[b]
    return out


def _stored64(x, kv):
    """The values that rows of x stand for once they are held in the pages' type."""
    if kv == "bf16":
        return x.float().to(torch.bfloat16).double()
    amax = x.abs().amax(-1, keepdim=True)
    if kv == "e4m3":
        scale = torch.exp2(torch.ceil(torch.log2(amax / 448)))
        return (x / scale).float().to(torch.float8_e4m3fn).double() * scale
    return torch.round(x / amax * 127) * (amax / 127)
