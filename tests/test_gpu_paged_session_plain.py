"""A session on the kernels against whole prompts through dense attention in plain torch, over keys and values as the
pages hold them: everything between the model and the operators (layers, scales, windows, positions) is compared."""
import math

import pytest
import torch

from dawn_srw_b200.models import inference as I
from dawn_srw_b200.models.baseline import VanillaTransformer
from dawn_srw_b200.models.dawn import DAWN
from dawn_srw_b200.ops import paged as P
from dawn_srw_b200.ops.cuda_backend import CudaBackend

pytestmark = pytest.mark.gpu


def _model(kind):
    torch.manual_seed(0)
    kw = dict(vocab_size=512, d_model=128, n_layers=3, n_heads=2, max_seq_len=400)
    if kind == "dense":
        m = VanillaTransformer(**kw, d_ff=256)
    else:
        m = DAWN(**kw, d_route=64, n_qk=600, n_v=600, n_know=1100, dropout_rate=0.0, router_dropout=0.0,
                 model_version=kind, seed=1)
    with torch.no_grad():
        for p in m.parameters():                                 # no two layers alike, biases and gains neither
            p.add_(0.02 * torch.randn(p.shape))
    return m.cuda().eval()


class PlainAttention(CudaBackend):
    """The kernels' backend with attention in plain torch.  ``off``: results off by up to that share of sum p |v|, of
    either sign, as a measure of what such errors come to in the logits."""

    def __init__(self, kv, window, sinks, off=0.0, seed=0):
        super().__init__()
        self.kv, self.window, self.sinks, self.off = P.PAGE_DTYPES[kv], window, sinks, off
        self.gen = torch.Generator("cuda").manual_seed(seed)

    @property
    def prompt_attention(self):
        raise AttributeError                                     # prompts go through attention

    def attention(self, q, k, v, dropout_p, training):
        k, v = (P.decode_rows(*P.encode_rows(t.contiguous(), self.kv)) for t in (k, v))
        i = torch.arange(q.shape[2], device=q.device)
        seen = i[None] <= i[:, None]
        if self.window is not None:
            seen &= (i[None] > i[:, None] - self.window) | (i[None] < self.sinks)
        w = torch.softmax((q.bfloat16().double() @ k.double().transpose(-1, -2) / math.sqrt(q.shape[-1])).masked_fill(~seen, -math.inf), -1)
        o, mag = w @ v.double(), w @ v.double().abs()
        if self.off:
            o = o + self.off * mag * (2 * torch.rand(o.shape, device=o.device, generator=self.gen) - 1).sign()
        return o.float().bfloat16()


def _whole(m, ids, *args, **kw):
    old, m.backend = m.backend, PlainAttention(*args, **kw)
    m._inference_pools = None
    try:
        return I.prefill(m, ids[None].cuda())[0][0]
    finally:
        m.backend, m._inference_pools = old, None


@pytest.mark.parametrize("kind", ["dense", "spatial-r1-v4.0.1", "spatial-r1-v4.1", "spatial-r1-v3.9.4"])
@pytest.mark.parametrize("kv,window,sinks", [("bf16", None, 0), ("e4m3", None, 0), ("int8", 50, 4), ("bf16", 33, 1)])
def test_a_session_gives_the_logits_of_the_whole(kind, kv, window, sinks):
    """The kernels' attention is within 2^-7 of sum p |v| of the definition: weights and result are rounded to bf16 or
    finer, 2^-8 each.  What errors of that size, all at the bound and of random signs, come to in the logits is the
    measure, root mean square over all of them; the kernels' own errors are mostly far below the bound.  A window
    or sinks off by one position come to more."""
    m = _model(kind)
    g = torch.Generator().manual_seed(1)
    ids = [torch.randint(1, 512, (n,), generator=g) for n in (230, 90)]
    s = I.PagedSession(m, 3, kv_dtype=kv, window=window, sinks=sinks)
    a, b = s.open(), s.open()
    got = {a: [], b: []}
    for chunk in ({a: 100, b: 17}, {b: 1, a: 5}, {a: 120}, {b: 60}):
        parts = s.extend({k: ids[k][sum(map(len, got[k])): sum(map(len, got[k])) + n] for k, n in chunk.items()}, all_logits=True)
        for k, part in zip(chunk, parts):
            got[k].append(part)
    while sum(map(len, got[a])) < 230 or sum(map(len, got[b])) < 90:
        now = [k for k in (a, b) if sum(map(len, got[k])) < len(ids[k])]
        lg = s.step({k: int(ids[k][sum(map(len, got[k]))]) for k in now})
        for k, row in zip(now, lg):
            got[k].append(row[None])
    s.check()
    for k in (a, b):
        have, want = torch.cat(got[k]), _whole(m, ids[k], kv, window, sinks)
        rms = lambda x: float((x - want).double().square().mean().sqrt())
        slack = min(rms(_whole(m, ids[k], kv, window, sinks, off=2.0 ** -7, seed=x)) for x in range(3))
        assert rms(have) <= slack
        if window is not None:
            assert all(rms(_whole(m, ids[k], kv, *w)) > slack for w in ((window + 1, sinks), (window, sinks + 1)))
