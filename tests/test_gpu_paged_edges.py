"""Paged attention where keys, values or scales are extreme or no numbers, against the definition in 64 bits."""
import math

import pytest
import torch

from dawn_srw_b200.ops import paged as P
from paged_helpers import KINDS, args, assert_attention, attention64, make_cache, scales, starts_of

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
