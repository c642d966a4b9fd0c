"""CPU checks of what the Python entry points of the paged cache refuse: tensors of
the host, or of a GPU that is not the current one (a fake here)."""
import pytest
import torch

from spindle_b200 import kv4


class OnGpu(torch.Tensor):
    """A tensor that says it lies on a GPU."""
    where = 0

    def get_device(self):
        return self.where


def on(where, *n, dtype=torch.float32):
    t = torch.zeros(*n, dtype=dtype).as_subclass(OnGpu)
    t.where = where
    return t


def test_host_tensors():
    with pytest.raises(ValueError):
        kv4.logprobs(torch.zeros(2, 10))
    with pytest.raises(ValueError):
        kv4._dev(torch.zeros(2), "x")
    with pytest.raises(TypeError):
        kv4._i32(torch.zeros(2, dtype=torch.int32), "x", 0)
    with pytest.raises(ValueError):
        kv4._tables(torch.zeros(2, 2, dtype=torch.int32), 2, 0)


def test_a_gpu_that_is_not_the_current_one(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    assert kv4._dev(on(0, 3), "x") == 0
    with pytest.raises(ValueError):
        kv4._dev(on(1, 3), "x")
    with pytest.raises(ValueError):
        kv4.logprobs(on(1, 2, 10))
    with pytest.raises(TypeError):
        kv4._i32(on(1, 3, dtype=torch.int32), "x", 0)
    with pytest.raises(ValueError):
        kv4._tables(on(1, 2, 2, dtype=torch.int32), 2, 0)
