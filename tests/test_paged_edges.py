"""Paged key/value cache at the edges of its range, on the CPU: alignment, and values that are no numbers."""
import ctypes
import math

import pytest
import torch

from dawn_srw_b200.ops import build
from dawn_srw_b200.ops.backend import ReferenceBackend
from dawn_srw_b200.ops.cuda_backend import CudaBackend

from paged_helpers import args, attention64, make_cache, scales, starts_of

CPU = torch.device("cpu")


def off_a_border(t):
    """A contiguous copy of t that starts four bytes behind a 16-byte border."""
    room = torch.zeros(t.numel() * t.element_size() + 16, dtype=torch.uint8)
    at = 4 + -room.data_ptr() % 16
    moved = room[at: at + t.numel() * t.element_size()].view(t.dtype).view(t.shape)
    moved.copy_(t)
    assert moved.data_ptr() % 16 == 4 and moved.is_contiguous()
    return moved


@pytest.mark.parametrize("kind,what", [("bf16", "k_pages"), ("int8", "v_pages"), ("int8", "k_scale"), ("e4m3", "v_scale")])
def test_pages_and_scales_off_a_border_are_refused(kind, what):
    """The kernels read pages and scales in words of 16 bytes."""
    be = CudaBackend()
    c = make_cache(kind, [20, 7], 2, 16, 16, CPU, garbage=False)
    c[what] = off_a_border(c[what])
    q = torch.zeros(2, 2, 16)
    for call in (lambda: be.paged_write(q, q, *args(c), **scales(c)), lambda: be.paged_read(*args(c), 20, **scales(c)),
                 lambda: be.paged_attention(q, *args(c), **scales(c))):
        with pytest.raises(ValueError, match="16-byte aligned"):
            call()


class DsbPaged(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("k", "v", "k_scale", "v_scale", "table", "lengths", "starts", "status")]
                + [(n, ctypes.c_int) for n in ("kind", "n_pages", "H", "page", "dh", "B", "width", "N")])


def c_view(**kw):
    """One int8 sequence of one page at addresses that nothing reads."""
    at = dict(k=4096, v=4096, k_scale=4096, v_scale=4096, table=4096, lengths=4096, starts=None, status=4096)
    return DsbPaged(**{**at, **dict(kind=2, n_pages=1, H=1, page=16, dh=64, B=1, width=1, N=1), **kw})


def c_calls(c, out=4096):
    """The return codes of the C entry points; a refused call touches none of the addresses, and without a GPU no
    other call does."""
    lib = ctypes.CDLL(str(build.PLAIN_SO_PATH))
    p, n, ll, i = ctypes.c_void_p, ctypes.byref(c), ctypes.c_longlong, ctypes.c_int
    return {"write": lib.dsb_paged_write(n, p(4096), p(4096), i(1), ll(64), ll(64), ll(64), ll(64), p(0)),
            "read": lib.dsb_paged_read(n, p(out), p(out), i(1), i(16), p(0)),
            "attention": lib.dsb_paged_attention(n, p(4096), ll(64), ll(64), p(out), i(1), i(1), i(0), i(0),
                                                 ctypes.c_float(1.0), p(0), p(0))}


@pytest.mark.skipif(torch.cuda.is_available(), reason="what is not refused would be launched")
@pytest.mark.parametrize("what", ["k", "v", "k_scale", "v_scale"])
def test_c_entry_points_refuse_addresses_off_a_border(what):
    assert c_calls(c_view(**{what: 4100})) == {"write": 930, "read": 934, "attention": 940}


@pytest.mark.skipif(torch.cuda.is_available(), reason="what is not refused would be launched")
def test_c_entry_points_refuse_results_off_a_border():
    """Reading back stores words of 16 bytes, the attention of 32; a result on a border gets as far as the launch, or
    the want of a workspace."""
    c = c_view()
    assert c_calls(c, out=4100)["read"] == 934 and c_calls(c, out=4104)["read"] == 934
    assert c_calls(c, out=4100)["attention"] == 941 and c_calls(c, out=4096 + 16)["attention"] == 941
    assert c_calls(c, out=4096 + 16)["read"] == 936
    assert c_calls(c)["attention"] not in (0, 940, 941)


@pytest.mark.parametrize("odd", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("window,sinks", [(None, 0), (4, 0), (5, 2)])
def test_a_value_that_is_no_number_reaches_the_rows_that_see_it(odd, window, sinks):
    """The plain path, fp32 throughout: 1e-5 of the sum of magnitudes."""
    c = make_cache("bf16", [20, 5], 2, 16, 16, CPU)
    c["v_pages"][int(c["table"][0, 0]), 1, 9, 3] = odd
    new = [18, 5]
    q = torch.randn(23, 4, 16, generator=torch.Generator().manual_seed(1))
    got = ReferenceBackend().paged_attention(q, *args(c), starts_of(new, CPU), window=window, sinks=sinks)
    ref, mag = attention64(q, c, new, window, sinks)
    fine = ref.isfinite()
    assert int((~fine).sum()) == 2 * (11 if window is None else window)              # two query heads of the group, a column
    assert torch.equal(got.isfinite(), fine) and torch.equal(got[~fine].double().nan_to_num(), ref[~fine].float().double().nan_to_num())
    assert bool(((got.double() - ref).abs() <= 1e-5 * mag + 1e-12)[fine].all())


def test_two_rows_with_one_place_are_refused_by_the_plain_path():
    c = make_cache("int8", [20, 7], 2, 16, 16, CPU, garbage=False)
    c["table"][1, 0] = c["table"][0, 0]                          # a page that both read is fine
    x = torch.zeros(2, 2, 16)
    ReferenceBackend().paged_write(x, x, *args(c), **scales(c))
    c["lengths"][:] = 7
    with pytest.raises(ValueError, match="one place"):
        ReferenceBackend().paged_write(x, x, *args(c), **scales(c))
