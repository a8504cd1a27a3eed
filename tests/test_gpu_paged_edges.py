"""Paged attention where keys, values or scales are extreme or no numbers, against the definition in 64 bits."""
import math

import pytest
import torch

from dawn_srw_b200.ops import paged as P
from paged_helpers import KINDS, args, assert_attention, attention64, held64, make_cache, scales, starts_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cb():
    from dawn_srw_b200.ops import cuda_backend
    cuda_backend.check_status()
    return cuda_backend


@pytest.fixture(scope="module")
def be(cb):
    return cb.CudaBackend()


def _rand(*shape, seed=0, dtype=torch.bfloat16):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


def _at(c, b, pos):
    """(page, slot) of a position."""
    page = c["k_pages"].shape[2]
    return int(c["table"][b, pos // page]), pos % page


def _run(be, c, q, new, **kw):
    starts = None if new == [1] * len(new) else starts_of(new, "cuda")
    return be.paged_attention(q, *args(c), starts, **scales(c), **kw)


def smallest_weights(q, c, new, window=None, sinks=0):
    """What the fp16 weights of 8-bit pages may add to a result.  A weight goes to fp16 as p_j S_j, S_j being the power
    of two next to (in a chunk: at) the largest scale of the values among 32 positions, p_j the softmax; the
    row's largest, W, stands at 2^6 or more.  A weight below fp16's normal numbers is off by half of its smallest step,
    2^-25, which is 2^-31 W: by sum_j 2^-31 W |v_j| / S_j in all, and S_j is more than half of the scale of j.  In a
    chunk a value next to a larger scale is off by half of that step too, 2^-25 S_j (none where the scales of 32
    positions are more than 2^20, for int8 2^13, apart: the work is done in fp32): by sum_j p_j 2^-25 S_j; and a key in the same way,
    which moves a score by scale |q|_1 2^-25 S'_j, a weight by that and the sum of weights by as much again."""
    out = torch.zeros(q.shape, dtype=torch.double, device=q.device)
    if c["v_scale"] is None:
        return out
    H, G = c["k_pages"].shape[1], q.shape[1] // c["k_pages"].shape[1]
    at = 0
    for b, n in enumerate(new):
        length = int(c["lengths"][b])
        k, v = held64(c, b, length, "k"), held64(c, b, length, "v")
        pos = torch.arange(length, device=q.device)
        ids = c["table"][b].long()[pos // c["k_pages"].shape[2]]
        groups = {}
        for name, x64 in (("v", v), ("k", k)):
            s = c[name + "_scale"][ids, :, pos % c["k_pages"].shape[2]].double()              # [length, H]
            s = torch.where((x64 == 0).all(-1) | ~s.isfinite(), torch.zeros_like(s), s)
            group = torch.zeros_like(s)
            for x in range(0, length, 32):
                top, least = s[x: x + 32].amax(0), torch.where(s > 0, s, torch.full_like(s, math.inf))[x: x + 32].amin(0)
                near = top <= 2.0 ** (14 if c["k_pages"].dtype == torch.int8 else 21) * least
                group[x: x + 32] = torch.where(near, top, s[x: x + 32])
            groups[name] = s, group
        (s, group), (_, kgroup) = groups["v"], groups["k"]
        codes = torch.where(s[..., None] > 0, v.abs() / s[..., None], torch.zeros_like(v)).nan_to_num(0.0)
        for i in range(n):
            p = length - n + i
            j = torch.arange(max(p, -1) + 1, device=q.device)
            if window is not None:
                j = j[(j > p - window) | (j < sinks)]
            if not len(j):
                continue
            a = torch.einsum("hgd,nhd->hgn", q[at + i].double().view(H, G, -1), k[j]) / math.sqrt(q.shape[2])
            w = torch.softmax(a, -1)
            most = (w * group[j].T[:, None]).amax(-1)                                   # [H, G]
            step = 2.0 ** -25 * (w * group[j].T[:, None]).sum(-1)
            moved = 2.0 ** -24 / math.sqrt(q.shape[2]) * q[at + i].double().abs().sum(-1).view(H, G) * kgroup[j].amax(0)[:, None]
            mag = torch.einsum("hgn,nhd->hgd", w, v[j].abs())
            slack = 2.0 ** -30 * most[..., None] * codes[j].sum(0)[:, None] + step[..., None] + moved[..., None] * mag
            out[at + i] = slack.reshape(q.shape[1:])
        at += n
    return out.nan_to_num(0.0)


def _compare(cb, be, c, q, new, window=None, sinks=0, nan_rows=False):
    """Finite results as the definition has them, the others where it has them and of the same kind; with ``nan_rows``
    a row with one that is not finite is NaN throughout."""
    got = _run(be, c, q, new, window=window, sinks=sinks)
    ref, mag = attention64(q, c, new, window, sinks)
    if nan_rows:
        assert torch.equal(ref.isnan().any(-1), ref.isnan().all(-1))
    fine = ref.isfinite()
    assert torch.equal(got.isfinite(), fine)
    assert torch.equal(got.isnan(), ref.isnan())
    assert torch.equal(got[~fine].nan_to_num(0.0).double(), ref[~fine].bfloat16().nan_to_num(0.0).double())
    zero = torch.zeros_like
    mag = mag + 2.0 ** 8 * smallest_weights(q, c, new, window, sinks)                   # assert_attention takes 2^-8 of it
    assert_attention(torch.where(fine, got, zero(got)), torch.where(fine, ref, zero(ref)), torch.where(fine, mag, zero(mag)))
    cb.check_status()
    return ref


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("q_mag,k_mag", [(-60, -60), (-20, -90), (-100, -20)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (50, 2)])
def test_small_queries_and_keys(cb, be, kind, dh, q_mag, k_mag, window, sinks):
    """Products far below the smallest fp32 number: all scores are nearly alike, hidden ones stay hidden."""
    for new in ([200, 77], [5, 5], [1, 1]):
        c = make_cache(kind, [300, 77], 2, dh, 16, "cuda", seed=dh)
        c["k_scale"] *= 2.0 ** k_mag
        q = _rand(sum(new), 4, dh, seed=3) * 2.0 ** q_mag
        ref = _compare(cb, be, c, q, new, window, sinks)
        assert bool(ref.isfinite().all())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dh", [64, 80, 128])
@pytest.mark.parametrize("odd", [math.nan, math.inf])
@pytest.mark.parametrize("at", [0, 5, 6, 31, 37, 64, 69, 100])
def test_a_key_that_is_no_number(cb, be, kind, dh, odd, at):
    """NaN for the rows that see it, wherever it stands in a tile, and nothing for those that do not."""
    for lengths, new, window in (([220, 40], [180, 40], None), ([220, 40], [180, 40], 60), ([104, 40], [5, 3], None),
                                 ([220, 40], [1, 1], None), ([220, 40], [1, 1], 30)):
        c = make_cache(kind, lengths, 2, dh, 16, "cuda", seed=at)
        page, slot = _at(c, 0, at)
        if kind == "bf16":
            c["k_pages"][page, 0, slot, 0] = odd
        else:                                                    # as a row with such a value is stored
            c["k_scale"][page, 0, slot] = math.nan
        q = _rand(sum(new), 4, dh, seed=at + 1)
        q[..., 0] = q[..., 0].abs() + 0.1
        ref = _compare(cb, be, c, q, new, window, 0, nan_rows=True)
        sees = torch.tensor([p >= at and (window is None or at > p - window) for p in range(lengths[0] - new[0], lengths[0])])
        assert torch.equal(ref[: new[0], 0, 0].isnan().cpu(), sees)


@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("lengths,new,window", [([1, 30], [1, 1], None), ([1, 9], [1, 9], None), ([40, 300], [40, 300], None),
                                                ([40, 300], [40, 300], 1), ([4, 300], [4, 290], 3), ([40, 20], [3, 1], 2)])
def test_rows_that_see_only_scores_of_minus_infinity(cb, be, dh, lengths, new, window):
    """Nothing over nothing: NaN by the definition, unlike a row that sees no key."""
    c = make_cache("bf16", lengths, 2, dh, 16, "cuda")
    for b, pos in ((0, 0), (0, lengths[0] - 1), (1, 0), (1, lengths[1] - 1)):
        page, slot = _at(c, b, pos)
        c["k_pages"][page, 0, slot, 3] = -math.inf
    q = _rand(sum(new), 4, dh, seed=2)
    q[..., 3] = q[..., 3].abs() + 0.1
    _compare(cb, be, c, q, new, window, nan_rows=True)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("dh", [64, 80, 128])
@pytest.mark.parametrize("odd", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 0), (70, 20)])
def test_a_value_that_is_no_number(cb, be, kind, dh, odd, window, sinks):
    """It reaches the rows that see it, in its column, and no other."""
    for lengths, new, at in (([220, 40], [180, 40], 100), ([220, 40], [180, 40], 10), ([600, 40], [500, 30], 333),
                             ([104, 40], [5, 3], 102), ([105, 40], [9, 3], 40), ([300, 40], [8, 3], 256)):
        c = make_cache(kind, lengths, 2, dh, 16, "cuda", seed=at)
        page, slot = _at(c, 0, at)
        if kind == "bf16":
            c["v_pages"][page, 0, slot, 7] = odd
        else:
            c["v_pages"].view(torch.uint8)[page, 0, slot, 7] = 0x7f if odd > 0 or odd != odd else 0xff     # both are NaN
        q = _rand(sum(new), 4, dh, seed=at + 1)
        ref = _compare(cb, be, c, q, new, window, sinks)
        bad = (~ref.isfinite()).nonzero()
        assert bool((bad[:, 2] == 7).all()) and bool((bad[:, 1] < 2).all())


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("window,sinks", [(None, 0), (20000, 3)])
def test_a_value_that_is_no_number_in_a_long_context(cb, be, kind, window, sinks):
    """Drafted tokens whose warps take equal runs of all units, and leave pieces."""
    lengths, new = [40000, 300, 7, 1000, 9, 70, 200, 1], [5, 3, 5, 1, 4, 0, 5, 1]
    for at in (39997, 39999, 20000, 19998, 5):
        c = make_cache(kind, lengths, 8, 64, 64, "cuda", seed=at)
        for b, pos in ((0, at), (2, 4)):
            page, slot = _at(c, b, pos)
            if kind == "bf16":
                c["v_pages"][page, 0, slot, 7] = math.inf
            else:
                c["v_pages"].view(torch.uint8)[page, 0, slot, 7] = 0x7f
        q = _rand(sum(new), 16, 64, seed=at + 1) * 0.2
        _compare(cb, be, c, q, new, window, sinks)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("which,mag", [("v", 30), ("v", -40), ("v", 19), ("v", -12), ("k", 26), ("k", 18), ("k", -14),
                                       ("v zero", -40), ("k zero", -20)])
def test_neighbours_of_another_magnitude(cb, be, kind, dh, which, mag):
    """Keys or values whose scales differ by much, some by more than fp16 numbers do, beside each other in a tile; rows
    before the large one do not see it.  ``zero``: rows of zeros, which are stored under a scale of 1, among small ones."""
    for lengths, new, at in (([200, 30], [200, 30], 150), ([700, 30], [400, 30], 500), ([155, 30], [8, 3], 150)):
        c = make_cache(kind, lengths, 2, dh, 16, "cuda", seed=at)
        name = which[0]
        page, slot = _at(c, 0, at)
        q = _rand(sum(new), 4, dh, seed=at + 1)
        if which.endswith("zero"):
            c[name + "_scale"] *= 2.0 ** mag
            c[name + "_scale"][page, :, slot] = 1.0
            c[name + "_pages"].view(torch.uint8)[page, :, slot] = 0
            if name == "k":
                q = q * 2.0 ** -mag
        else:
            c[name + "_scale"][page, :, slot] *= 2.0 ** mag
        ref = _compare(cb, be, c, q, new)
        assert bool(ref.isfinite().all())


def test_nan_codes_read_back_as_nan(cb, be):
    """0x7f and 0xff of e4m3, which no write here makes but a page may hold."""
    c = make_cache("e4m3", [20], 2, 64, 16, "cuda", garbage=False)
    raw = c["k_pages"].view(torch.uint8)
    raw[:, 0, 3, 5], raw[:, 1, 2, 63] = 0x7f, 0xff
    for dtype in (torch.float32, torch.bfloat16):
        got, want = be.paged_read(*args(c), 20, **scales(c), dtype=dtype)[0], P.read(*args(c), 20, **scales(c), dtype=dtype)[0]
        assert int(want.isnan().sum()) == 4 and torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(), want.nan_to_num())
    cb.check_status()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [[180, 40], [5, 3]])
def test_captured_calls_follow_values_that_come_and_go(cb, be, kind, new):
    """A call captured over an ordinary cache, replayed on two streams in turn while a value is no number, or a scale far
    from the others, and when all is well again."""
    lengths, at = [220, 40], 217
    c = make_cache(kind, lengths, 2, 64, 16, "cuda", seed=3)
    q, starts, page_slot = _rand(sum(new), 4, 64, seed=9), starts_of(new, "cuda"), _at(c, 0, at)
    call = lambda: be.paged_attention(q, *args(c), starts, **scales(c))
    first = call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    page, slot = page_slot
    keep = {n: None if c[n] is None else c[n].clone() for n in ("v_pages", "v_scale")}
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(6):
        odd = i % 2 == 1
        if odd and kind == "bf16":
            c["v_pages"][page, 0, slot, 7] = math.inf
        elif odd:
            c["v_scale"][page, 0, slot] *= 2.0 ** 30
        elif kind == "bf16":
            c["v_pages"].copy_(keep["v_pages"])
        else:
            c["v_scale"].copy_(keep["v_scale"])
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[i // 2 % 2]):
            graph.replay()
        torch.cuda.synchronize()
        eager = call()
        assert torch.equal(out.nan_to_num(), eager.nan_to_num()) and torch.equal(out.isnan(), eager.isnan())
        if odd:
            _compare(cb, be, c, q, new)
        else:
            assert torch.equal(out, first)
    cb.check_status()
