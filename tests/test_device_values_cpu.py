"""The operations on float64 matrices refuse values of another type before anything reads them: stand-ins for CUDA tensors, and
no library behind them."""
import pytest
import torch


class OnDevice:
    """What the device layer asks of a CUDA tensor."""

    def __init__(self, dtype, *shape):
        self.dtype, self.shape, self.is_cuda, self.device = dtype, shape, True, "cpu"

    def is_contiguous(self):
        return True

    def dim(self):
        return len(self.shape)

    def stride(self, i):
        return self.shape[1] if i == 0 and len(self.shape) > 1 else 1

    def data_ptr(self):
        return 4096


@pytest.fixture
def calls(monkeypatch):
    from comet_b200 import device
    made = []
    monkeypatch.setattr(device, "_call", lambda name, *args: made.append(name))
    monkeypatch.setattr(device, "_stream", lambda: 0)
    return made


def matrix(values):
    from comet_b200 import device
    return device.DeviceCSR(3, 3, OnDevice(torch.int64, 4), OnDevice(torch.int64, 5), OnDevice(values, 5))


def operations(A, dense=torch.float64, out=torch.float64):
    from comet_b200 import device
    f64 = matrix(torch.float64)
    return [lambda: device.spmv(A, OnDevice(dense, 3), OnDevice(out, 3)),
            lambda: device.spmm(A, OnDevice(dense, 3, 2), OnDevice(out, 3, 2)),
            lambda: device.sddmm(A, OnDevice(dense, 3, 2), OnDevice(torch.float64, 3, 2), OnDevice(out, 5)),
            lambda: device.sddmm(A, OnDevice(torch.float64, 3, 2), OnDevice(dense, 3, 2), OnDevice(out, 5)),
            lambda: device.spgemm_symbolic(A, f64), lambda: device.spgemm_symbolic(f64, A)]


def test_float64_goes_through(calls):
    for op in operations(matrix(torch.float64)):
        op()
    assert len(calls) == 6


@pytest.mark.parametrize("values", [torch.float32, torch.float16, torch.bfloat16, torch.int64])
def test_matrices_of_other_values_are_refused(calls, values):
    """top_entries makes a matrix of float32 values."""
    for op in operations(matrix(values)):
        with pytest.raises(ValueError, match="float64"):
            op()
    assert not calls


def test_dense_operands_of_other_values_are_refused(calls):
    for op in operations(matrix(torch.float64), dense=torch.float32)[:4] + operations(matrix(torch.float64), out=torch.float32)[:4]:
        with pytest.raises(ValueError, match="float64"):
            op()
    assert not calls


def test_results_of_other_values_are_refused(calls):
    from comet_b200 import device
    with pytest.raises(ValueError, match="float64"):
        device.spgemm_numeric(1, 5, "cuda", crd=OnDevice(torch.int64, 5), val=OnDevice(torch.float32, 5))
    assert not calls


def test_a_count_does_not_ask_for_values(calls):
    from comet_b200 import device
    A = matrix(torch.float32)
    device.masked_pair_count(A, A, A, out=OnDevice(torch.int64, 1))
    assert len(calls) == 1
