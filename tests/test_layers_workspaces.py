"""CPU-only: what the Python wrappers of the operators around a layer take as a workspace."""
import pytest
import torch

import fbcuda_amd as F


def test_a_workspace_lies_on_the_gpu():
    assert F._space(None) == (None, 0)
    assert F._space(torch.empty(0)) == (None, 0)  # where none is needed
    with pytest.raises(ValueError):
        F._space(torch.empty(1 << 20, dtype=torch.uint8))


class OnGpu:
    """What of a GPU tensor a wrapper looks at."""
    is_cuda = True

    def __init__(self, t):
        self.t = t

    def __getattr__(self, name):
        return getattr(self.t, name)


def test_a_workspace_is_no_larger_than_its_memory():
    whole = torch.empty(4096, dtype=torch.float32)
    for t, size in ((whole, 16384), (whole[1024:], 12288), (whole[:1].expand(1 << 30), 4096 * 4), (whole[4095:].expand(1 << 30), 4),
                    (whole.view(64, 64)[:, :32], 8192), (torch.empty(1, dtype=torch.uint8).expand(1 << 40), 1)):
        assert F._space(OnGpu(t)) == (t.data_ptr(), size)
