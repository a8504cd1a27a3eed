"""bf16 compute copies that the kernels' backend keeps of weights."""
import torch

from dawn_srw_b200.ops.cuda_backend import CudaBackend


def test_a_weight_that_is_pointed_elsewhere_is_cast_again():
    be, w = CudaBackend(), torch.nn.Parameter(torch.randn(8, 8))
    first = be._w(w)
    assert be._w(w) is first
    version = w._version
    w.data = w.data + 1.0
    assert w._version == version
    assert torch.equal(be._w(w), w.detach().bfloat16())
