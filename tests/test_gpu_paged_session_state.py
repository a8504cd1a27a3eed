"""Captured steps of paged sessions: what they follow, and what a failed capture leaves behind."""
import copy

import pytest
import torch

from dawn_srw_b200.models import inference as I

from test_gpu_paged_session import _model

pytestmark = pytest.mark.gpu


def _logits(s, ids):
    a = s.open()
    s.extend({a: ids})
    got = s.step({a: 3})
    s.close(a)
    return got


def test_a_captured_step_follows_weights_that_are_pointed_elsewhere():
    m = _model("dense")
    ids = torch.arange(1, 40)
    s = I.PagedSession(m, 1)
    before = _logits(s, ids)
    for p in (m.layers[1].ffn.w_up.weight, m.layers[1].norm1.weight, m.layers[1].attn.q_proj.bias):
        p.data = p.data * 1.5 + 0.1
    after = _logits(s, ids)
    want = _logits(I.PagedSession(copy.deepcopy(m), 1, use_graph=False), ids)
    assert torch.equal(after, want) and not torch.allclose(before, after, atol=1e-2)
    s.be.finish_run()


def test_a_failed_capture_leaves_no_graph():
    m = _model("dense")
    ids = torch.arange(1, 40)
    s = I.PagedSession(m, 1)
    a = s.open()
    s.extend({a: ids})
    forward, calls = s._forward, []

    def failing(*args):
        calls.append(torch.cuda.is_current_stream_capturing())
        if calls[-1]:
            raise RuntimeError("no room")                        # on the host, while nothing has been launched
        return forward(*args)
    s._forward = failing
    with pytest.raises(RuntimeError, match="no room"):
        s.step({a: 3})
    assert calls[-1] and s._graph is None and s.lengths == [39]
    s._forward = forward
    got = s.step({a: 3})
    assert s._graph is not None and s.lengths == [40]
    assert torch.equal(got, _logits(I.PagedSession(m, 1, use_graph=False), ids))
    s.be.finish_run()


@pytest.mark.parametrize("use_graph", [True, False])
def test_a_page_outside_the_pool_is_reported_to_the_caller(use_graph):
    m = _model("dense")
    s = I.PagedSession(m, 1, use_graph=use_graph)
    a = s.open()
    s.extend({a: torch.arange(1, 40)})
    s.step({a: 3})
    s.check()
    good, s.pages[a][1] = s.pages[a][1], 10 ** 6                 # counts as absent; the status word tells of it
    s.step({a: 3})
    with pytest.raises(RuntimeError, match="status 4"):
        s.step({a: 3})
    assert s.lengths == [41]
    s.pages[a][1] = good
    try:
        s.check()                                                # of the step that raised, which ran all the same
    except RuntimeError:
        pass
    s.step({a: 3})
    s.check()
    s.pages[a][1] = 10 ** 6
    s.extend({a: torch.arange(1, 20)})
    with pytest.raises(RuntimeError, match="status 4"):
        s.check()
