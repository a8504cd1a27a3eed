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


@pytest.mark.parametrize("change", list(CHANGES))
@pytest.mark.parametrize("kind", ["spatial-r1-v4.1", "dense"])
def test_parameters_that_are_pointed_elsewhere_or_replaced(kind, change):
    if kind == "dense" and change == "a pool's data":
        pytest.skip("no pools")
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
