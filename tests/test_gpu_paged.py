"""Kernels of the paged key/value cache against the plain definition in 64 bits."""
import math

import pytest
import torch

from dawn_srw_b200.ops import paged as P
from paged_helpers import KINDS, args, assert_attention, attention64, largest_score, make_cache, scales, starts_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cb():
    from dawn_srw_b200.ops import cuda_backend
    cuda_backend.check_status()
    return cuda_backend


@pytest.fixture(scope="module")
def be(cb):
    return cb.CudaBackend()


def _rand(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


# ---------------------------------------------------------------- storage
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("src", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,dh,page,lengths,new", [
    (6, 64, 16, [290], [1]),
    (2, 80, 32, [33, 0, 16, 1], [33, 1, 5, 1]),                 # sequence 1: a slot without positions
    (3, 128, 256, [700, 3], [600, 3]),
    (1, 16, 64, [64, 65, 63], [1, 65, 0]),
    (5, 112, 128, [129], [129]),
])
def test_write_and_read(cb, be, kind, src, H, dh, page, lengths, new):
    """Bit by bit what the plain path stores (the same roundings in the same order), and nothing else moves."""
    c = make_cache(kind, lengths, H, dh, page, "cuda", seed=dh)
    n = sum(new) + 2                                            # two rows behind the last sequence
    k, v = (_rand(n, H, dh, seed=s) * 10.0 ** (s - 4) for s in (3, 5))
    k[0, 0], v[0, -1] = 0.0, 2.0 ** -110
    k, v = k.to(src), v.to(src)
    starts = starts_of(new, "cuda")
    want = {x: (t.clone() if t is not None else None) for x, t in c.items()}
    P.write(k, v, *args(want), starts, **scales(want))
    be.paged_write(k, v, *args(c), starts, **scales(c))
    raw = lambda t: t.view(torch.uint8 if t.element_size() == 1 else torch.int16)
    for name in ("k", "v"):
        assert torch.equal(raw(c[name + "_pages"]), raw(want[name + "_pages"]))
        if kind != "bf16":
            assert torch.equal(c[name + "_scale"].view(torch.int32), want[name + "_scale"].view(torch.int32))
    for dtype in (torch.float32, torch.bfloat16):
        for max_len in (0, 1, max(lengths), max(lengths) + 70):
            got = be.paged_read(*args(c), max_len, **scales(c), dtype=dtype)
            ref = P.read(*args(c), max_len, **scales(c), dtype=dtype)
            assert all(torch.equal(a, b) and a.dtype == dtype for a, b in zip(got, ref)), (dtype, max_len)
    cb.check_status()


@pytest.mark.parametrize("kind", KINDS)
def test_write_of_strided_and_unaligned_rows(cb, be, kind):
    c = make_cache(kind, [5, 40], 4, 32, 16, "cuda")
    wide = _rand(45, 3 * 4 * 32 + 1, seed=9)
    views = {"one projection": [wide[:, i * 128: (i + 1) * 128].view(45, 4, 32) for i in (0, 2)],
             "off by one": [wide[:, 1 + i * 128: 1 + (i + 1) * 128].view(45, 4, 32) for i in (0, 2)],
             "heads first": [wide[:, i * 128: (i + 1) * 128].reshape(45, 4, 32).transpose(0, 1).contiguous().transpose(0, 1)
                             for i in (0, 2)],
             "inner stride": [wide[:, i: i + 256: 2].reshape(45, 4, 32) for i in (0, 1)]}
    views["inner stride"] = [torch.stack([x, x], -1)[..., 0] for x in views["inner stride"]]
    starts = starts_of([5, 40], "cuda")
    for name, (k, v) in views.items():
        be.paged_write(k, v, *args(c), starts, **scales(c))
        got = be.paged_read(*args(c), 40, **scales(c))
        for x, y in zip((k, v), got):
            want = P.decode_rows(*P.encode_rows(x, c["k_pages"].dtype)).transpose(0, 1)
            assert torch.equal(y[0, :, :5], want[:, :5]) and torch.equal(y[1], want[:, 5:]), name


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_every_code_reads_as_its_value(be, kind):
    codes = torch.arange(256, dtype=torch.uint8, device="cuda")
    if kind == "e4m3":
        codes[[0x7f, 0xff]] = 0                                  # the NaN codes, which are never written
    kp = codes.view(P.PAGE_DTYPES[kind]).view(1, 1, 16, 16).contiguous()
    s = _rand(1, 1, 16, seed=1).abs() + 0.1
    k, v = be.paged_read(kp, kp.clone(), torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                         torch.tensor([16], dtype=torch.int32, device="cuda"), 16, s, s)
    assert torch.equal(k, P.decode_rows(kp, s)) and torch.equal(v, k)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("odd", [math.nan, math.inf, -math.inf])
def test_rows_that_hold_no_number(be, kind, odd):
    c = make_cache(kind, [1, 1], 2, 64, 16, "cuda")
    k = _rand(2, 2, 64)
    k[1, 0, 63] = odd
    be.paged_write(k, k, *args(c), **scales(c))
    got = be.paged_read(*args(c), 1, **scales(c))[0]
    assert bool(got[1, 0].isnan().all()) and bool(got[1, 1].isfinite().all()) and bool(got[0].isfinite().all())


# ---------------------------------------------------------------- attention
def _check(cb, be, kind, H, G, dh, page, lengths, new, window=None, sinks=0, seed=0, max_new=None, extra=0, **kw):
    c = make_cache(kind, lengths, H, dh, page, "cuda", seed=seed)
    N = sum(new)
    q = _rand(N + extra, H * G, dh, seed=seed + 7, dtype=torch.bfloat16)
    starts = None if new == [1] * len(new) and extra == 0 else starts_of(new, "cuda")
    got = be.paged_attention(q, *args(c), starts, **scales(c), max_new=max_new, window=window, sinks=sinks, **kw)
    ref, mag = attention64(q[:N], c, new, window, sinks, kw.get("scale"))
    assert_attention(got[:N], ref, mag)
    assert not bool(got[N:].any())                              # rows of no sequence
    cb.check_status()
    return c, q, starts, got


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,G,dh,page", [(6, 1, 64, 16), (16, 1, 80, 32), (2, 8, 128, 64), (3, 5, 96, 16), (1, 1, 16, 256),
                                         (2, 2, 32, 16), (1, 12, 112, 128), (1, 40, 48, 16)])
def test_single_tokens(cb, be, kind, H, G, dh, page):
    """Lengths around the tiles of every kernel, from none (a slot without positions) to several thousand."""
    lengths = [290, 0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 1000, 4097]
    _check(cb, be, kind, H, G, dh, page, lengths, [1] * len(lengths), seed=dh)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 0), (64, 4), (100, 1), (128, 130), (5000, 0), (3, 5000), (1, 1)])
def test_single_tokens_under_a_window(cb, be, kind, window, sinks):
    lengths = [0, 1, 5, 8, 64, 70, 129, 200, 1025, 3000]
    _check(cb, be, kind, 2, 4, 64, 16, lengths, [1] * len(lengths), window, sinks, seed=window)
    _check(cb, be, kind, 3, 1, 128, 64, lengths, [1] * len(lengths), window, sinks, seed=window)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,G,dh,page,lengths,new", [
    (8, 2, 64, 16, [200, 6, 900, 5], [5, 5, 5, 5]),                      # drafted tokens
    (2, 1, 80, 32, [9, 300, 0, 77], [2, 9, 0, 1]),
    (1, 1, 128, 16, [130, 64], [130, 64]),                               # whole prompts
    (2, 3, 32, 64, [257, 128, 1, 500], [257, 100, 1, 43]),
    (1, 8, 96, 128, [400, 20], [33, 20]),
    (2, 1, 64, 16, [1000], [513]),
    (1, 1, 16, 16, [3, 2], [5, 2]),                                      # more new tokens than positions
])
def test_chunks(cb, be, kind, H, G, dh, page, lengths, new):
    _check(cb, be, kind, H, G, dh, page, lengths, new, seed=dh, extra=3)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (50, 0), (128, 4), (200, 129), (7, 1000), (100000, 3)])
def test_chunks_under_a_window(cb, be, kind, window, sinks):
    _check(cb, be, kind, 2, 2, 64, 16, [700, 130, 260, 0], [300, 130, 1, 0], window, sinks, seed=window)
    _check(cb, be, kind, 1, 1, 128, 32, [515], [515], window, sinks, seed=window)


@pytest.mark.parametrize("max_new", [None, 0, 1, 5, 100, 100000])
def test_the_hint_only_chooses_the_kernel(cb, be, max_new):
    """Also where it is wrong."""
    _check(cb, be, "bf16", 2, 2, 64, 16, [300, 40, 17], [140, 1, 17], seed=3, max_new=max_new)
    _check(cb, be, "int8", 2, 2, 80, 16, [300, 40, 17], [1, 1, 1], seed=3, max_new=max_new)


def test_scales_of_the_scores(cb, be):
    for s in (0.01, 1.0, 3.0):
        _check(cb, be, "bf16", 2, 1, 64, 16, [300, 77], [1, 1], scale=s)
        _check(cb, be, "e4m3", 2, 1, 64, 16, [300, 77], [200, 77], scale=s)
    _check(cb, be, "bf16", 1, 1, 64, 16, [300], [300], scale=0.0)
    _check(cb, be, "bf16", 1, 1, 64, 16, [300], [300], scale=-0.1)


@pytest.mark.parametrize("new", [[1, 1], [200, 3]])
def test_scores_far_apart_and_infinite(cb, be, new):
    """Keys whose scores rise, fall and reach -inf over the context: the running maximum moves at every tile."""
    lengths = [900, 333]
    c = make_cache("bf16", lengths, 2, 64, 16, "cuda", garbage=False)
    ramp = torch.linspace(-30, 30, 16, device="cuda").repeat_interleave(64)
    for b in range(2):
        for i in range(-(-lengths[b] // 16)):
            page = int(c["table"][b, i])
            c["k_pages"][page, :, :, 0] = (ramp[i * 16: i * 16 + 16] if b == 0 else -ramp[i * 16: i * 16 + 16]).bfloat16()
    c["k_pages"][int(c["table"][0, 3]), :, 2, 1] = -math.inf
    q = _rand(sum(new), 2, 64, dtype=torch.bfloat16, seed=2).abs() + 0.5
    got = be.paged_attention(q, *args(c), None if new == [1, 1] else starts_of(new, "cuda"))
    ref, mag = attention64(q, c, new)
    assert bool(ref.isfinite().all())
    assert_attention(got, ref, mag)


@pytest.mark.parametrize("kind", KINDS)
def test_strided_queries_and_types(cb, be, kind):
    c = make_cache(kind, [50, 20, 300], 2, 80, 16, "cuda")
    wide = _rand(3, 2 * 320 + 8, seed=4, dtype=torch.bfloat16)
    ref, mag = attention64(wide[:, 160: 480].view(3, 4, 80), c, [1, 1, 1])
    views = [wide[:, 160:480].view(3, 4, 80), wide[:, 160:480].float().view(3, 4, 80),
             torch.cat([wide[:, :1], wide[:, 160:480]], 1)[:, 1:].view(3, 4, 80),
             wide[:, 160:480].view(3, 4, 80).transpose(0, 1).contiguous().transpose(0, 1)]
    for q in views:
        assert_attention(be.paged_attention(q, *args(c), **scales(c)), ref, mag)


@pytest.mark.parametrize("kind", KINDS)
def test_nothing_to_do(be, kind):
    c = make_cache(kind, [0, 0], 2, 64, 16, "cuda")
    q = _rand(2, 2, 64, dtype=torch.bfloat16)
    assert not bool(be.paged_attention(q, *args(c), **scales(c)).any())
    e = make_cache(kind, [], 2, 64, 16, "cuda")
    assert be.paged_attention(q[:0], *args(e), **scales(e)).shape == (0, 2, 64)
    be.paged_write(q[:0], q[:0], *args(e), **scales(e))
    assert be.paged_read(*args(e), 5, **scales(e))[0].shape == (0, 2, 5, 64)
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert not bool(be.paged_attention(q, *args(e), none, **scales(e)).any())     # two rows, no sequence


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bad", [-1, -2 ** 31, 10 ** 6, 2 ** 31 - 1])
def test_pages_outside_the_pool_are_reported_and_not_read(cb, be, kind, bad):
    """The positions of such a page count as absent; the status word tells of it."""
    lengths = [100, 30]
    c = make_cache(kind, lengths, 2, 64, 16, "cuda")
    q = _rand(2, 2, 64, dtype=torch.bfloat16)
    fine = be.paged_attention(q, *args(c), **scales(c))
    chunk = _rand(100, 2, 64, dtype=torch.bfloat16)
    starts = starts_of([99, 1], "cuda")
    cb.check_status()
    c["table"][0, 2] = bad
    got = be.paged_attention(q, *args(c), **scales(c))
    with pytest.raises(RuntimeError, match="status 4"):
        cb.check_status()
    assert torch.equal(got[1], fine[1]) and bool(got.isfinite().all())
    assert bool(be.paged_attention(chunk, *args(c), starts, **scales(c)).isfinite().all())
    with pytest.raises(RuntimeError, match="status 4"):
        cb.check_status()
    dense = be.paged_read(*args(c), 100, **scales(c))[0]
    with pytest.raises(RuntimeError, match="status 4"):
        cb.check_status()
    assert not bool(dense[0, :, 32:48].any()) and bool(dense[0, :, 31].any())
    before = c["k_pages"].clone()
    c["lengths"][0] = 40                                         # the newest position is in that page
    be.paged_write(q, q, *args(c), **scales(c))
    with pytest.raises(RuntimeError, match="status 4"):
        cb.check_status()
    raw = lambda t: t.view(torch.uint8 if t.element_size() == 1 else torch.int16)
    changed = (raw(before) != raw(c["k_pages"])).any(-1).any(1).sum()
    assert int(changed) == 1                                     # the other sequence's slot alone
    c["lengths"][0] = 10 ** 6                                    # more positions than the table has room for
    be.paged_attention(q, *args(c), **scales(c))
    with pytest.raises(RuntimeError, match="status 4"):
        cb.check_status()


@pytest.mark.parametrize("new", [[1, 1], [70, 200]])
def test_windows_forget_pages(cb, be, new):
    """Table entries of pages that no new token sees are not looked at."""
    c = make_cache("e4m3", [1000, 500], 2, 64, 16, "cuda")
    q = _rand(sum(new), 2, 64, dtype=torch.bfloat16)
    starts = None if new == [1, 1] else starts_of(new, "cuda")
    kw = dict(window=100, sinks=5, **scales(c))
    want = be.paged_attention(q, *args(c), starts, **kw)
    for b, t in enumerate((1000, 500)):
        first = max(0, t - new[b] - 100 + 1) // 16
        c["table"][b, 1:first] = -1
    assert torch.equal(be.paged_attention(q, *args(c), starts, **kw), want)
    cb.check_status()


@pytest.mark.parametrize("kind,heads", [("int8", 64), ("bf16", 32)])
def test_offsets_beyond_32_bits(cb, be, kind, heads):
    """A pool of more than 2^32 elements, the sequence in its last pages."""
    c = make_cache(kind, [70], heads, 128, 256, "cuda", garbage=False, least_pages=1)
    n = 2 ** 32 // (heads * 256 * 128) + 2
    for name in ("k", "v"):
        pool = torch.zeros(n, *c[name + "_pages"].shape[1:], dtype=c[name + "_pages"].dtype, device="cuda")
        at = int(c["table"][0, 0])
        raw = lambda t: t.view(torch.uint8 if t.element_size() == 1 else torch.int16)
        raw(pool)[n - 1] = raw(c[name + "_pages"])[at]
        if kind != "bf16":
            s = torch.ones(n, *c[name + "_scale"].shape[1:], device="cuda")
            s[n - 1] = c[name + "_scale"][at]
            c[name + "_scale"] = s
        c[name + "_pages"] = pool
    c["table"][0, 0] = n - 1
    for new in ([1], [70]):
        q = _rand(new[0], heads, 128, dtype=torch.bfloat16)
        starts = starts_of(new, "cuda")
        ref, mag = attention64(q, c, new)
        assert_attention(be.paged_attention(q, *args(c), starts, **scales(c)), ref, mag)
        be.paged_write(q, q, *args(c), starts, **scales(c))
        got = be.paged_read(*args(c), 70, **scales(c))[0][0, :, 70 - new[0]:].transpose(0, 1)
        assert torch.equal(got, P.decode_rows(*P.encode_rows(q, c["k_pages"].dtype)))
    cb.check_status()


# ---------------------------------------------------------------- streams and graphs
def test_captured_steps_follow_their_inputs(cb, be):
    """Write and attention of a step captured once; lengths, table and rows change between replays.  Two graphs
    whose replays interleave on two streams do not disturb each other."""
    def step(c, q, k):
        be.paged_write(k, k, *args(c), **scales(c))
        return be.paged_attention(q, *args(c), **scales(c))
    runs = []
    for seed, kind in ((1, "bf16"), (2, "int8")):
        c = make_cache(kind, [600, 30, 200], 4, 64, 16, "cuda", seed=seed, width=64)
        c["lengths"] -= 20
        q, k = _rand(3, 4, 64, seed=seed, dtype=torch.bfloat16), _rand(3, 4, 64, seed=seed + 9)
        step(c, q, k)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(c, q, k)
        runs.append((c, q, k, graph, out, torch.cuda.Stream()))
    for i in range(15):
        torch.cuda.synchronize()
        for c, q, k, *_ in runs:
            c["lengths"] += 1
            q.copy_(_rand(3, 4, 64, seed=50 + i))
            k.copy_(_rand(3, 4, 64, seed=90 + i))
        torch.cuda.synchronize()
        for _ in range(3):
            for *_, graph, _out, stream in runs:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for c, q, k, _, out, _ in runs:
            ref, mag = attention64(q, c, [1, 1, 1])
            assert_attention(out, ref, mag)
    cb.check_status()


def test_calls_on_another_stream(cb, be):
    c = make_cache("e4m3", [5000, 70], 2, 128, 32, "cuda")
    q = _rand(300, 4, 128, dtype=torch.bfloat16)
    starts = starts_of([250, 50], "cuda")
    want = be.paged_attention(q, *args(c), starts, **scales(c))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(be.paged_attention(q, *args(c), starts, **scales(c)))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)                # sums in a fixed order


@pytest.mark.parametrize("kind", KINDS)
def test_a_prompt_in_chunks_then_tokens(cb, be, kind):
    """The operators together, as a session uses them: two prompts enter by chunks, then token by token; every
    step's attention is that of the cache as it then stands, and the dense form reads back what was stored."""
    H, dh, page, total = 3, 64, 16, [90, 61]
    c = make_cache(kind, total, H, dh, page, "cuda", spare=1)
    k, v, q = ([_rand(t, H, dh, seed=10 * i + b) for b, t in enumerate(total)] for i in (1, 2, 3))
    done = [0, 0]
    for new in ([40, 7], [33, 50], [1, 1], [1, 0], [14, 3], [1, 0]):
        sl = [slice(d, d + n) for d, n in zip(done, new)]
        done = [d + n for d, n in zip(done, new)]
        c["lengths"].copy_(torch.tensor(done, dtype=torch.int32))
        cat = lambda xs: torch.cat([x[s] for x, s in zip(xs, sl)])
        starts = starts_of(new, "cuda")
        be.paged_write(cat(k), cat(v), *args(c), starts, **scales(c))
        qq = cat(q).bfloat16()
        ref, mag = attention64(qq, c, new)
        assert_attention(be.paged_attention(qq, *args(c), starts, **scales(c)), ref, mag)
    assert done == total
    dense = be.paged_read(*args(c), max(total), **scales(c))
    for x, got in zip((k, v), dense):
        for b, t in enumerate(total):
            want = P.decode_rows(*P.encode_rows(x[b], c["k_pages"].dtype)).transpose(0, 1)
            assert torch.equal(got[b, :, :t], want) and not bool(got[b, :, t:].any())
    cb.check_status()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dh", [48, 80, 128])
@pytest.mark.parametrize("new", [[1, 1], [300, 40]])
def test_the_running_maximum_moves_in_every_tile(cb, be, kind, dh, new):
    """Scores that rise (first sequence) or fall along the context, by several powers of two from tile to tile."""
    lengths = [1100, 333]
    c = make_cache(kind, lengths, 2, dh, 16, "cuda", garbage=False)
    for b, up in enumerate((1.0, -1.0)):
        for i in range(-(-lengths[b] // 16)):
            page = int(c["table"][b, i])
            x = torch.randn(2, 16, dh, device="cuda", generator=torch.Generator("cuda").manual_seed(i)) * 0.1
            x[..., 0] += up * (i - 30)
            codes, scale = P.encode_rows(x, P.PAGE_DTYPES[kind])
            c["k_pages"][page] = codes
            if scale is not None:
                c["k_scale"][page] = scale
    q = _rand(sum(new), 4, dh, dtype=torch.bfloat16, seed=5)
    q[..., 0] = q[..., 0].abs() + 2.0
    starts = None if new == [1, 1] else starts_of(new, "cuda")
    got = be.paged_attention(q, *args(c), starts, **scales(c))
    for _ in range(30):                                           # the order of a block's warps changes nothing
        assert torch.equal(be.paged_attention(q, *args(c), starts, **scales(c)), got)
    ref, mag = attention64(q, c, new)
    assert_attention(got, ref, mag, largest_score(q, c, new) if kind == "int8" and new != [1, 1] else 0.0)
    cb.check_status()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [[1, 1], [40, 3]])
def test_a_pool_without_pages(cb, be, kind, new):
    c = make_cache(kind, [0, 0], 2, 64, 16, "cuda", spare=0)
    assert c["k_pages"].shape[0] == 0
    q = _rand(sum(new), 2, 64, dtype=torch.bfloat16)
    starts = None if new == [1, 1] else starts_of(new, "cuda")
    assert not bool(be.paged_attention(q, *args(c), starts, **scales(c)).any())
    be.paged_write(q, q, *args(c), starts, **scales(c))
    assert not bool(be.paged_read(*args(c), 9, **scales(c))[0].any())
    cb.check_status()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dh,G", [(64, 1), (128, 2), (112, 3)])
def test_chunks_of_many_shapes(cb, be, kind, dh, G):
    """Runs of one tile, of a few and of many, units that blocks share, row tiles with and without work."""
    gen = torch.Generator().manual_seed(dh)
    for i in range(6):
        B = int(torch.randint(1, 5, (1,), generator=gen))
        lengths = torch.randint(1, (64, 500, 1500)[i % 3], (B,), generator=gen).tolist()
        new = [int(torch.randint(1, min(n, 400) + 1, (1,), generator=gen)) for n in lengths]
        window = (None, 150, 33)[(i // 2) % 3]
        _check(cb, be, kind, 2, G, dh, (16, 64, 256)[i % 3], lengths, new, window, 0 if window is None else 5, seed=i,
               max_new=1000)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("window", [None, 100])
def test_many_sequences_without_work_between_others(cb, be, kind, dh, window):
    """Runs of units that have rows and no positions, longer than what a block plans ahead, behind a unit with some."""
    lengths = [1, 79, 1, 0, 1, 300, 0, 1, 0, 1, 200, 0, 0, 0, 40]
    new = [0, 50, 1, 1, 1, 262, 0, 3, 1, 4, 200, 2, 1, 9, 40]
    _check(cb, be, kind, 8, 8, dh, 16, lengths, new, window, extra=3)
    _check(cb, be, kind, 8, 1, dh, 16, lengths, [min(n, 1) for n in new], window, extra=1)
