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


class Elsewhere:
    """A tensor as another one, but on another device."""

    def __init__(self, like):
        self._like = like

    def get_device(self):
        return 1

    def __getattr__(self, name):
        return getattr(self._like, name)


def experts_calls(G):
    """Each of the four operations on 6 tokens with 2 of 4 experts, width 64 and inner 48."""
    from comet_b200 import device
    new = lambda *shape: torch.zeros(shape, dtype=torch.bfloat16)                   # noqa: E731
    X, W, H, V = new(6, 64), new(4, 96, 64), new(12, 48), new(4, 64, 48)
    return [lambda: device.gated_experts(G, X, W), lambda: device.gated_experts_grad(G, X, W, H), lambda: device.combine_experts(G, H, V),
            lambda: device.combine_experts_grad(G, H, V, X)]


def choices():
    from comet_b200 import device
    S = device.DeviceCSR(6, 4, torch.arange(0, 13, 2), torch.arange(12) % 4, torch.ones(12))
    return S, device.group_entries


@pytest.fixture
def groups(calls):
    """group_entries asks for a CUDA matrix: EntryGroups as it makes them."""
    from comet_b200 import device
    S, _ = choices()
    plan = torch.zeros(16 + 4 + 8 + 8 + 256 * 5, dtype=torch.int32)
    return device.EntryGroups(S, plan, 128 * 5)


@pytest.mark.parametrize("which", range(4))
def test_groups_of_the_current_device_go_through(calls, groups, which):
    experts_calls(groups)[which]()
    assert len(calls) == 1


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("part", ["plan", "pos", "crd", "val"])
def test_groups_of_another_device_are_refused(calls, groups, part, which):
    """Their addresses are of another device's memory."""
    if part == "plan":
        groups.plan = Elsewhere(groups.plan)
    else:
        setattr(groups.S, part, Elsewhere(getattr(groups.S, part)))
    if part == "val" and which < 2:                                                 # not looked at
        experts_calls(groups)[which]()
        return
    with pytest.raises(ValueError, match="device"):
        experts_calls(groups)[which]()
    assert not calls


def sums_of(buffer):
    from comet_b200 import device
    return lambda: device.log_probs_grad(pattern(), torch.zeros(3, 40), buffer, torch.zeros(3))


def test_sums_at_an_odd_address_are_refused(calls):
    """Kernels read both numbers of a row at once.  So are sums that are not contiguous, whatever their strides."""
    room = torch.zeros(32)
    assert room.data_ptr() % 8 == 0
    for bad in (room[1:7].view(3, 2), room[:6].view(2, 3).t(), room[:12].view(3, 4)[:, :2], room[:6].double().view(3, 2), room[:6]):
        with pytest.raises(ValueError, match="sums"):
            sums_of(bad)()
    assert not calls
    for good in (room[2:8].view(3, 2), room[:6].view(3, 2)):
        sums_of(good)()
    assert len(calls) == 2
