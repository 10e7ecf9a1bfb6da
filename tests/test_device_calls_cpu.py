"""What the device layer hands to the C entries of log probabilities and of a router's experts, and what it refuses: CPU tensors take the place of CUDA ones (the
current device is made to be theirs), and a stand-in takes the call."""
import gc
import weakref

import pytest
import torch


@pytest.fixture
def calls(monkeypatch):
    """The calls that are made, and what else is to happen inside one."""
    from comet_b200 import device

    class Calls(list):
        inside = staticmethod(lambda *args: None)

    made = Calls()

    def call(name, *args):
        made.append((name, args))
        made.inside(*args)

    monkeypatch.setattr(device, "_call", call)
    monkeypatch.setattr(device, "_stream", lambda: 0)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: -1, raising=False)     # what get_device() says of a CPU tensor
    monkeypatch.setattr(device, "_check_logits", lambda what, X: (X.shape[0], X.shape[1], X.stride(0)))
    return made


def pattern(rows=3, cols=40, nnz=3):
    from comet_b200 import device
    return device.DeviceCSR(rows, cols, torch.arange(rows + 1), torch.arange(nnz), None)


def log_probs_calls():
    from comet_b200 import device
    X = torch.zeros(3, 40)
    return [lambda t: device.log_probs(pattern(), X, temperature=t, top=2),
            lambda t: device.log_probs_grad(pattern(), X, torch.zeros(3, 2), torch.zeros(3), temperature=t)]


@pytest.mark.parametrize("which", [0, 1])
def test_a_temperature_lives_until_its_call_returns(calls, which):
    """Another thread's calls, at other temperatures, may clear what the layer remembers of them while the C function reads this one."""
    from comet_b200 import device
    alive = []

    def others(*args):
        own = weakref.ref(device._numbers[(0.749,)][1])
        for i in range(300):
            device._floats(1000.0 + i)
        gc.collect()
        alive.append(own() is not None)
        assert (0.749,) not in device._numbers

    calls.inside = others
    log_probs_calls()[which](0.749)
    assert alive == [True]
