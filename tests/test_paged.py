"""Paged key/value cache on the CPU: the plain definition, and what both backends refuse."""
import math

import pytest
import torch

from dawn_srw_b200.ops import paged as P
from dawn_srw_b200.ops.backend import ReferenceBackend

from paged_helpers import KINDS, args, attention64, held64, make_cache, scales, starts_of

CPU = torch.device("cpu")


@pytest.mark.parametrize("dtype", list(P.PAGE_DTYPES.values()))
def test_rows_are_stored_with_one_rounding(dtype):
    """e4m3: half a step is 2^-4 of a value, and never less than 2^-10 of the scale (half the smallest step);
    int8: half a step of the scale, plus the fp32 roundings of 127 / largest, the product and the scale
    (3 * 2^-24 of at most 127 steps)."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(500, 64, generator=g) * torch.exp2(torch.randint(-20, 20, (500, 1), generator=g).float())
    x[7] = 0.0
    x[8] = 2.0 ** -120
    codes, scale = P.encode_rows(x, dtype)
    y, x64 = P.decode_rows(codes, scale).double(), x.double()
    if dtype == torch.bfloat16:
        assert scale is None and bool(((y - x64).abs() <= x64.abs() * 2.0 ** -8).all())
        return
    s = scale.double()[:, None]
    assert bool((scale[7:9] == 1).all()) and bool((y[7:9] == 0).all())
    live = torch.ones(500, dtype=torch.bool)
    live[8] = False
    if dtype == torch.float8_e4m3fn:
        ok = (y - x64).abs() <= torch.maximum(x64.abs() * 2.0 ** -4, s * 2.0 ** -10)
        m, _ = torch.frexp(scale)
        assert bool((m == 0.5).all())                                     # powers of two
        top = x.abs().amax(-1) / scale
        top = top[(x.abs().amax(-1) >= P.SMALLEST)]
        assert bool((top <= 448).all()) and bool((top > 224).all())
    else:
        ok = (y - x64).abs() <= s * (0.5 + 127 * 3 * 2.0 ** -24)
        assert int(codes.long().abs().max()) == 127
    assert bool(ok[live].all())


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("odd", [math.nan, math.inf, -math.inf])
def test_a_row_with_a_value_that_is_no_number_reads_back_as_nan(dtype, odd):
    x = torch.ones(3, 16)
    x[1, 5] = odd
    codes, scale = P.encode_rows(x, dtype)
    y = P.decode_rows(codes, scale)
    assert bool(y[1].isnan().all()) and bool((y[[0, 2]] == 1).all())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,G,dh,page,lengths,new", [
    (2, 1, 8, 16, [5, 33, 16], [1, 1, 1]),
    (1, 3, 16, 32, [40, 3, 0, 70], [7, 3, 0, 0]),
    (2, 2, 24, 16, [1, 17], [1, 17]),
])
def test_reference_attention_against_the_definition(kind, H, G, dh, page, lengths, new):
    """fp32 throughout on the plain path: sums of at most 70 terms, 1e-5 of the sum of magnitudes."""
    be = ReferenceBackend()
    c = make_cache(kind, lengths, H, dh, page, CPU, seed=sum(lengths))
    q = torch.randn(sum(new), H * G, dh, generator=torch.Generator().manual_seed(1))
    starts = None if new == [1] * len(new) else starts_of(new, CPU)
    for window, sinks in ((None, 0), (4, 0), (6, 2), (1, 0), (1000, 3)):
        ref, mag = attention64(q, c, new, window, sinks)
        got = be.paged_attention(q, *args(c), starts, **scales(c), window=window, sinks=sinks)
        assert bool(((got.double() - ref).abs() <= 1e-5 * mag + 1e-12).all()), (window, sinks)


@pytest.mark.parametrize("kind", KINDS)
def test_reference_write_then_read(kind):
    be = ReferenceBackend()
    lengths, new, H, dh = [20, 0, 37, 16], [20, 1, 5, 16], 2, 16           # sequence 1: a slot without positions
    c = make_cache(kind, lengths, H, dh, 16, CPU)
    before = be.paged_read(*args(c), 37, **scales(c))
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(sum(new) + 3, H, dh, generator=g) for _ in range(2))          # three rows of no sequence
    be.paged_write(k, v, *args(c), starts_of(new, CPU), **scales(c))
    after = be.paged_read(*args(c), 37, **scales(c))
    at = 0
    for b, (t, n) in enumerate(zip(lengths, new)):
        for x, old, got in ((k, before[0], after[0]), (v, before[1], after[1])):
            if t:
                want = P.decode_rows(*P.encode_rows(x[at: at + n], c["k_pages"].dtype))
                assert torch.equal(got[b, :, t - n: t], want.transpose(0, 1))
                assert torch.equal(got[b, :, : t - n], old[b, :, : t - n])
            assert not bool(got[b, :, t:].any())
        at += n
    for name, dense in (("k", after[0]), ("v", after[1])):
        assert torch.equal(held64(c, 2, 37, name).float(), dense[2].transpose(0, 1))


def test_reference_windows_forget_pages():
    """A page that no new token sees may be gone from the table; one that is seen may not."""
    be = ReferenceBackend()
    c = make_cache("bf16", [100], 1, 16, 16, CPU)
    q = torch.randn(1, 1, 16, generator=torch.Generator().manual_seed(1))
    want = be.paged_attention(q, *args(c), window=20, sinks=3)
    c["table"][0, 1:5] = -1                                  # positions 16..79; the window starts at 80
    assert torch.equal(be.paged_attention(q, *args(c), window=20, sinks=3), want)
    c["table"][0, 5] = -1
    with pytest.raises(ValueError, match="names no page"):
        be.paged_attention(q, *args(c), window=20, sinks=3)


# ---- refusals: the same calls are refused by the plain path and by the kernels' bindings
def _good(page=16, dh=16, kind="int8"):
    c = make_cache(kind, [20, 7], 2, dh, page, CPU, garbage=False)
    return dict(k_pages=c["k_pages"], v_pages=c["v_pages"], table=c["table"], lengths=c["lengths"],
                k_scale=c["k_scale"], v_scale=c["v_scale"])


def _drop(name):
    return lambda a: a.update({name: None})


def _make(name, f):
    return lambda a: a.update({name: f(a[name])})


BAD_CACHES = {
    "page size": lambda a: a.update(_good(page=16), k_pages=torch.zeros(3, 2, 24, 16, dtype=torch.int8),
                                    v_pages=torch.zeros(3, 2, 24, 16, dtype=torch.int8),
                                    k_scale=torch.zeros(3, 2, 24), v_scale=torch.zeros(3, 2, 24)),
    "k and v pages": _make("v_pages", lambda t: t[:-1]),
    "one type": _make("v_pages", lambda t: t.view(torch.float8_e4m3fn)),
    "must be contiguous": lambda a: a.update(k_pages=a["k_pages"].transpose(0, 1).contiguous().transpose(0, 1)),
    "pages must be bfloat16": lambda a: a.update(k_pages=a["k_pages"].float(), v_pages=a["v_pages"].float()),
    "8-bit pages come with": _drop("k_scale"),
    "bf16 pages without": lambda a: a.update(k_pages=a["k_pages"].bfloat16(), v_pages=a["v_pages"].bfloat16()),
    "scales must be": _make("v_scale", lambda t: t[:, :1]),
    "scales must be contiguous": _make("v_scale", lambda t: t.double()),
    "table must be": _make("table", lambda t: t.long()),
    "table must be a": _make("table", lambda t: t[0]),
    "lengths must be": _make("lengths", lambda t: t.long()),
    "lengths must be a": _make("lengths", lambda t: t[:1]),
    "starts must be": lambda a: a.update(starts=torch.zeros(2, dtype=torch.int32)),
    "starts must be a": lambda a: a.update(starts=torch.zeros(3, dtype=torch.int64)),
}


def _backends():
    from dawn_srw_b200.ops.cuda_backend import CudaBackend
    return [ReferenceBackend(), CudaBackend()]


def _calls(be, a, rows=2, heads=2, dim=16, **kw):
    q = torch.zeros(rows, heads, dim)
    starts = a.pop("starts", None)
    rest = [a[n] for n in ("k_pages", "v_pages", "table", "lengths")]
    sc = [a["k_scale"], a["v_scale"]]
    return {"write": lambda: be.paged_write(q, q, *rest, starts, *sc),
            "read": lambda: be.paged_read(*rest, 20, *sc),
            "attention": lambda: be.paged_attention(q, *rest, starts, *sc, **kw)}


@pytest.mark.parametrize("why", list(BAD_CACHES))
@pytest.mark.parametrize("which", [0, 1])
def test_refused_caches(why, which):
    be = _backends()[which]
    for op in ("write", "read", "attention"):
        a = _good()
        BAD_CACHES[why](a)
        if "starts" in a and op == "read":
            continue
        with pytest.raises(ValueError, match=why):
            _calls(be, a)[op]()


@pytest.mark.parametrize("which", [0, 1])
def test_refused_rows(which):
    be = _backends()[which]
    z = torch.zeros
    a = _good()
    rest, sc = [a[n] for n in ("k_pages", "v_pages", "table", "lengths")], [a["k_scale"], a["v_scale"]]
    with pytest.raises(ValueError, match="one new token"):
        be.paged_write(z(3, 2, 16), z(3, 2, 16), *rest, None, *sc)
    with pytest.raises(ValueError, match="pages' heads"):
        be.paged_write(z(2, 4, 16), z(2, 4, 16), *rest, None, *sc)
    with pytest.raises(ValueError, match="one type"):
        be.paged_write(z(2, 2, 16), z(2, 2, 16).bfloat16(), *rest, None, *sc)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        be.paged_write(z(2, 2, 16).half(), z(2, 2, 16).half(), *rest, None, *sc)
    with pytest.raises(ValueError, match="head dimension"):
        be.paged_attention(z(2, 2, 8), *rest, None, *sc)
    with pytest.raises(ValueError, match="no multiple"):
        be.paged_attention(z(2, 3, 16), *rest, None, *sc)
    with pytest.raises(ValueError, match="window"):
        be.paged_attention(z(2, 2, 16), *rest, None, *sc, window=0)
    with pytest.raises(ValueError, match="sinks"):
        be.paged_attention(z(2, 2, 16), *rest, None, *sc, window=3, sinks=-1)
    with pytest.raises(ValueError, match="max_new"):
        be.paged_attention(z(2, 2, 16), *rest, None, *sc, max_new=-1)
    with pytest.raises(ValueError, match="max_len"):
        be.paged_read(*rest, -1, *sc)
    with pytest.raises(ValueError, match="dtype"):
        be.paged_read(*rest, 5, *sc, dtype=torch.float16)


def test_kernels_refuse_what_only_they_cannot_take():
    be = _backends()[1]
    for dh in (8, 24, 144):
        for op in ("write", "read", "attention"):
            with pytest.raises(ValueError, match="not supported by the kernels"):
                _calls(be, _good(dh=dh), dim=dh)[op]()
    for op in ("write", "read", "attention"):
        with pytest.raises(ValueError, match="CUDA tensors"):
            _calls(be, _good())[op]()
