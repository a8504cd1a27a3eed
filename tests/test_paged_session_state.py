"""What a paged session keeps between calls: parameters that change under it, calls that fail, refused settings."""
import copy

import pytest
import torch

from dawn_srw_b200.models import inference as I

from test_paged_session import _close, _expected, _model

IDS = torch.randint(1, 200, (20,), generator=torch.Generator().manual_seed(5))


def _other(m):
    """A model of the same shape with other weights."""
    o = copy.deepcopy(m)
    with torch.no_grad():
        for p in o.parameters():
            p.mul_(1.0 + 0.3 * torch.randn(p.shape, generator=torch.Generator().manual_seed(p.numel())))
    return o


def _point_elsewhere(m, o, names):
    for (n, p), q in zip(m.named_parameters(), o.parameters()):
        if any(x in n for x in names):
            p.data = q.detach().clone()


CHANGES = {
    "a pool's data": lambda m, o: _point_elsewhere(m, o, ["know_write"]),
    "a later layer's data": lambda m, o: _point_elsewhere(m, o, ["layers.1.attn"]),
    "all data": lambda m, o: _point_elsewhere(m, o, [""]),
    "parameters assigned": lambda m, o: m.load_state_dict(o.state_dict(), assign=True),
    "a layer replaced": lambda m, o: m.layers.__setitem__(1, o.layers[1]),
}


def _logits(s, m):
    a = s.open()
    s.extend({a: IDS})
    got = s.step({a: 3})
    s.close(a)
    return got


@pytest.mark.parametrize("kind,change", [(k, c) for k in ("spatial-r1-v4.1", "dense") for c in CHANGES
                                         if k != "dense" or c != "a pool's data"])
def test_parameters_that_are_pointed_elsewhere_or_replaced(kind, change):
    m = _model(kind)
    s = I.PagedSession(m, 1)
    before = _logits(s, m)
    watched = s._watched
    _logits(s, m)
    assert s._watched is watched                                  # nothing changed: a captured step stays
    CHANGES[change](m, _other(m))
    after = _logits(s, m)
    assert s._watched is not watched                              # a captured step is captured again
    want = _expected(m, torch.cat([IDS, torch.tensor([3])]), "bf16")
    assert _close(after[0], want[20]) and not torch.allclose(before, after, atol=1e-3)


class Failing:
    """A backend whose n-th call of an operator from now on fails."""

    def __init__(self, be, name, n):
        self._be, self._name, self._left = be, name, n

    def __getattr__(self, name):
        f = getattr(self._be, name)
        if name != self._name:
            return f

        def call(*a, **kw):
            self._left -= 1
            if self._left == 0:
                raise RuntimeError("out of memory")
            return f(*a, **kw)
        return call


@pytest.mark.parametrize("name,n", [("paged_write", 1), ("paged_attention", 2), ("logits", 1), ("layer_norm", 3)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (9, 2)])
def test_a_call_that_fails_changes_nothing(name, n, window, sinks):
    """Lengths, pages and what is free stay, and the call made again gives the logits of a session without the failure."""
    m = _model("spatial-r1-v4.1")
    ids = torch.randint(1, 200, (60,), generator=torch.Generator().manual_seed(7))
    s = I.PagedSession(m, 2, window=window, sinks=sinks)
    a, b = s.open(), s.open()
    s.extend({a: ids[:30], b: ids[:16]})
    be, state = s.be, lambda: (list(s.lengths), copy.deepcopy(s.pages), list(s.free_pages))
    for new in (lambda: s.extend({b: ids[16:50], a: ids[30:33]}), lambda: s.extend({a: ids[33:35], b: ids[50:51]}, all_logits=True),
                lambda: s.step({a: ids[35], b: ids[51]})):
        before = state()
        s.be = Failing(be, name, n)
        with pytest.raises(RuntimeError, match="out of memory"):
            new()
        assert state() == before
        s.be = be
        last = new()
    assert s.lengths == [36, 52]
    assert _close(last[0], _expected(m, ids[:36], "bf16", window, sinks)[35])
    assert _close(last[1], _expected(m, ids[:52], "bf16", window, sinks)[51])


def test_sinks_without_a_window_are_refused():
    """As with dense caches; they were left out without a word."""
    m = _model("dense")
    with pytest.raises(ValueError, match="sinks belong to a window"):
        I.PagedSession(m, 1, sinks=2)
    with pytest.raises(ValueError, match="sinks belong to a window"):
        I.generate(m, IDS[None], max_new_tokens=2, kv_dtype="bf16", sinks=1)


@pytest.mark.parametrize("d_model,heads", [(32, 4), (96, 4), (320, 2)])
def test_heads_that_the_kernels_cannot_take_are_refused_by_the_constructor(d_model, heads):
    """Of 8, 24 and 160; the plain path takes them."""
    from dawn_srw_b200.models.baseline import VanillaTransformer
    from dawn_srw_b200.ops.cuda_backend import CudaBackend
    m = VanillaTransformer(vocab_size=50, d_model=d_model, n_layers=1, n_heads=heads, max_seq_len=40, d_ff=16).eval()
    I.PagedSession(m, 1)
    m.backend = CudaBackend()
    with pytest.raises(ValueError, match="not supported by the kernels"):
        I.PagedSession(m, 1)
    with pytest.raises(ValueError, match="too many"):
        m.backend.paged_supported(2, 64, 65536, 512)


class Reporting(Failing):
    """A backend that counts how often its failures are asked for, and can have one to report."""
    failure = None

    def __init__(self, be):
        super().__init__(be, "", 0)
        self.steps = self.runs = 0

    def finish_step(self):
        self.steps += 1
        if self.failure:
            raise RuntimeError(self.failure)

    def finish_run(self):
        self.runs += 1


def test_failures_of_kernels_are_asked_for():
    m = _model("dense")
    s = I.PagedSession(m, 1)
    s.be = Reporting(s.be)
    a = s.open()
    s.extend({a: IDS})
    s.step({a: 3})
    assert (s.be.steps, s.be.runs) == (2, 0)
    s.be.failure = "status 4"
    for call in (lambda: s.step({a: 3}), lambda: s.extend({a: IDS})):
        with pytest.raises(RuntimeError, match="status 4"):
            call()
        assert s.lengths == [21]
    s.check()
    assert s.be.runs == 1
    m.backend = Reporting(m._backend(torch.device("cpu")))
    for kw in ({}, {"kv_dtype": "int8"}):
        runs = m.backend.runs
        I.generate(m, IDS[None], max_new_tokens=2, **kw)
        assert m.backend.runs == runs + 1
