"""Sequences of their own lengths over a paged cache: chunks, single tokens, windows, pages that come and go."""
import math

import pytest
import torch

from dawn_srw_b200.models import inference as I
from dawn_srw_b200.models.baseline import VanillaTransformer
from dawn_srw_b200.models.dawn import DAWN
from dawn_srw_b200.ops import paged as P
from dawn_srw_b200.ops.backend import ReferenceBackend

KW = dict(vocab_size=200, d_model=32, n_layers=2, n_heads=4, max_seq_len=90)


def _model(kind):
    torch.manual_seed(0)
    if kind == "dense":
        m = VanillaTransformer(**KW, d_ff=64)
        with torch.no_grad():
            for p in m.parameters():
                p.add_(0.05 * torch.randn(p.shape))
    else:
        m = DAWN(**KW, d_route=8, n_qk=24, n_v=30, n_know=50, dropout_rate=0.0, router_dropout=0.0, model_version=kind, seed=1)
    return m.eval()


class RoundedBackend(ReferenceBackend):
    """Dense attention over keys and values as the pages hold them."""

    def __init__(self, kv, window=None, sinks=0):
        super().__init__(torch.float32)
        self.dtype, self.window, self.sinks = P.PAGE_DTYPES[kv], window, sinks

    def attention(self, q, k, v, dropout_p, training):
        k, v = (P.decode_rows(*P.encode_rows(t, self.dtype)) for t in (k, v))
        i = torch.arange(q.shape[2])
        seen = i[None] <= i[:, None]
        if self.window is not None:
            seen &= (i[None] > i[:, None] - self.window) | (i[None] < self.sinks)
        s = (q @ k.transpose(-1, -2) / math.sqrt(q.shape[-1])).masked_fill(~seen, -math.inf)
        return torch.softmax(s, -1) @ v


def _expected(model, ids, kv, window=None, sinks=0):
    """Logits [S, V] of every position of one sequence."""
    be, old = RoundedBackend(kv, window, sinks), model._backend
    model._backend = lambda device: be
    model._inference_pools = None
    try:
        return I.prefill(model, ids[None])[0][0]
    finally:
        model._backend = old
        model._inference_pools = None


def _close(a, b):
    """The same fp32 arithmetic in another order, over two layers of width 32; where a value falls next to a
    rounding border of the 8-bit types its code may differ by a step, which moves a logit by less than this."""
    return torch.allclose(a, b, atol=5e-3, rtol=1e-3) and float((a - b).abs().median()) < 1e-5


@pytest.mark.parametrize("kind", ["spatial-r1-v4.1", "spatial-r1-v3.9.4", "dense"])
@pytest.mark.parametrize("kv", ["bf16", "e4m3", "int8"])
@pytest.mark.parametrize("window,sinks", [(None, 0), (9, 2)])
def test_chunks_and_tokens_give_the_logits_of_the_whole(kind, kv, window, sinks):
    m = _model(kind)
    g = torch.Generator().manual_seed(1)
    ids = [torch.randint(1, 200, (n,), generator=g) for n in (60, 37, 17)]
    want = [_expected(m, i, kv, window, sinks) for i in ids]
    s = I.PagedSession(m, 4, kv_dtype=kv, window=window, sinks=sinks)
    a, b = s.open(), s.open()
    lg = s.extend({b: ids[1][:20], a: ids[0][:33]})
    assert _close(lg[0], want[1][19]) and _close(lg[1], want[0][32])
    c = s.open()
    parts = s.extend({a: ids[0][33:40], c: ids[2][:16], b: ids[1][20:21]}, all_logits=True)
    assert _close(parts[0], want[0][33:40]) and _close(parts[1], want[2][:16]) and _close(parts[2], want[1][20:21])
    for t in range(40, 60):
        step = {a: ids[0][t]}
        if t < 55:
            step[b] = ids[1][t - 19]
        if t == 50:
            step[c] = ids[2][16]
        lg = s.step(step)
        assert _close(lg[0], want[0][t])
        if t < 55:
            assert _close(lg[1], want[1][t - 19])
        if t == 50:
            assert _close(lg[2], want[2][16])
    assert s.lengths[:3] == [60, 36, 17]


def test_a_slot_is_used_again_and_pages_are_given_back():
    m = _model("spatial-r1-v4.1")
    s = I.PagedSession(m, 2, n_pages=6)
    g = torch.Generator().manual_seed(2)
    ids = torch.randint(1, 200, (40,), generator=g)
    want = _expected(m, ids, "bf16")
    a = s.open()
    s.extend({a: ids})
    b = s.open()
    with pytest.raises(RuntimeError, match="full"):
        s.extend({b: torch.cat([ids, ids])})
    assert len(s.free_pages) == 3 and s.lengths == [40, 0]            # the refused call changed nothing
    assert _close(s.extend({b: ids[:30]})[0], want[29])
    with pytest.raises(RuntimeError, match="all 2 sequences"):
        s.open()
    s.close(a)
    assert len(s.free_pages) == 4
    a = s.open()
    assert _close(s.extend({a: ids[:39]})[0], want[38])
    lg = s.step({a: ids[39], b: ids[30]})
    assert _close(lg[0], want[39]) and _close(lg[1], want[30])


def test_pages_behind_a_window_go_back():
    m = _model("dense")
    s = I.PagedSession(m, 1, n_pages=3, window=16, sinks=3)           # 48 positions at a time, for 90
    ids = torch.randint(1, 200, (90,), generator=torch.Generator().manual_seed(3))
    want = _expected(m, ids, "bf16", 16, 3)
    a = s.open()
    s.extend({a: ids[:30]})
    for t in range(30, 90):
        assert _close(s.step({a: ids[t]})[0], want[t])
    assert s.pages[a][0] >= 0 and s.pages[a][1:4] == [-1, -1, -1]
    with pytest.raises(ValueError, match="gone"):
        s.dense([a])
    with pytest.raises(ValueError, match="max_seq_len"):
        s.step({a: 1})


def test_dense_caches_of_a_session_go_on_in_a_dense_one():
    m = _model("spatial-r1-v4.0.1")
    ids = torch.randint(1, 200, (2, 20), generator=torch.Generator().manual_seed(4))
    s = I.PagedSession(m, 2)
    a, b = s.open(), s.open()
    s.extend({a: ids[0, :19], b: ids[1, :19]})
    ck, cv = s.dense([a, b])
    assert ck.shape == (2, 2, 4, 90, 8) and not bool(ck[:, :, :, 19:].any()) and not bool(cv[:, :, :, 19:].any())
    dense, *_ = I.decode_step(m, ids[:, 19], ck, cv, 19)
    paged = s.step({a: ids[0, 19], b: ids[1, 19]})
    # the dense step keeps its own newest key and value in fp32, the paged one in bf16: 2^-8 of one of twenty of them
    assert torch.allclose(dense, paged, atol=2e-2)


def test_a_write_to_a_parameter_is_seen():
    m = _model("spatial-r1-v4.1")
    ids = torch.randint(1, 200, (20,), generator=torch.Generator().manual_seed(5))
    s = I.PagedSession(m, 1)
    a = s.open()
    s.extend({a: ids})
    before = s.step({a: 3})
    s.close(a)
    with torch.no_grad():
        m.neuron_pool.know_write.mul_(1.5)
        m.layers[0].attn.expand_O.weight.mul_(0.5)
    a = s.open()
    s.extend({a: ids})
    after = s.step({a: 3})
    want = _expected(m, torch.cat([ids, torch.tensor([3])]), "bf16")
    assert _close(after[0], want[20]) and not torch.allclose(before, after, atol=1e-3)


def test_generate_with_paged_caches():
    m = _model("spatial-r1-v4.1")
    ids = torch.randint(1, 200, (2, 7), generator=torch.Generator().manual_seed(6))
    seq, info = I.generate(m, ids, max_new_tokens=5, temperature=0.0, kv_dtype="bf16")
    assert seq.shape == (2, 12) and info["new_tokens"] == 5
    for b in range(2):
        for t in range(7, 12):
            assert int(seq[b, t]) == int(_expected(m, seq[b, :t], "bf16")[-1].argmax())
    seq, _ = I.generate(m, ids, max_new_tokens=4, temperature=0.0, window=4, sinks=1)
    assert int(seq[0, 10]) == int(_expected(m, seq[0, :10], "bf16", 4, 1)[-1].argmax())
    with pytest.raises(ValueError, match="sinks"):
        I.generate(m, ids, max_new_tokens=2, sinks=1)


def test_refusals():
    m = _model("dense")
    for kw in (dict(kv_dtype="fp32"), dict(page_size=24), dict(page_size=8), dict(window=0), dict(sinks=-1)):
        with pytest.raises(ValueError):
            I.PagedSession(m, 2, **kw)
    with pytest.raises(ValueError):
        I.PagedSession(m, 0)
    s = I.PagedSession(m, 2)
    with pytest.raises(ValueError, match="not open"):
        s.extend({0: torch.tensor([1])})
    with pytest.raises(ValueError, match="not open"):
        s.close(1)
    a = s.open()
    for bad in ({}, {a: torch.zeros(0, dtype=torch.long)}):
        with pytest.raises(ValueError):
            s.extend(bad)
    with pytest.raises(ValueError):
        s.step({})
    with pytest.raises(ValueError, match="max_seq_len"):
        s.extend({a: torch.ones(91, dtype=torch.long)})
    assert s.lengths == [0, 0] and len(s.free_pages) == 12


@pytest.mark.parametrize("bad", [-1, 200, 2 ** 40])
def test_ids_outside_the_vocabulary_are_refused(bad):
    m = _model("dense")
    s = I.PagedSession(m, 2)
    a, b = s.open(), s.open()
    with pytest.raises(ValueError, match="vocabulary"):
        s.extend({a: torch.tensor([5]), b: torch.tensor([3, bad, 4])})
    with pytest.raises(ValueError, match="vocabulary"):
        s.step({a: 7, b: bad})
    assert s.lengths == [0, 0] and s.pages[a] == s.pages[b] == []
    assert s.extend({a: torch.tensor([0, 199])}).shape == (1, 200)
