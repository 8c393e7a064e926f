"""Host side of the serving calls without a GPU: the native module is replaced by one that records its calls, or that
computes the turn with torch."""
import contextlib
import types

import pytest

torch = pytest.importorskip("torch")


class Recorder:
    """The native module: the calls that reached it, and torch's current stream then."""

    def __init__(self):
        self.calls, self.stream = [], None

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, self.stream))
            return (None,) * 5
        return call


@pytest.fixture
def native(pkg, monkeypatch):
    pkg.rotary  # noqa: B018  (loads the module)
    module = Recorder()
    monkeypatch.setattr(pkg.serving, "_module", module)

    class External:
        def __init__(self, handle, device=None):
            self.cuda_stream, self.device = handle, torch.device("cuda", 0) if device is None else torch.device(device)

    @contextlib.contextmanager
    def current(stream):
        module.stream, before = (stream.cuda_stream, stream.device), module.stream
        yield
        module.stream = before

    monkeypatch.setattr(torch.cuda, "ExternalStream", External)
    monkeypatch.setattr(torch.cuda, "stream", current)
    return module


def operand(device):
    return types.SimpleNamespace(device=torch.device(device), requires_grad=False, shape=(1,) * 4)


def calls(pkg, x, stream):
    table = pkg.RotaryTable(x, x, False)
    return {"plan": lambda: pkg.cache_plan(x, x, x, x, x, 16, 4, stream=stream),
            "append": lambda: pkg.cache_append(x, x, x, x, x, stream=stream),
            "rotate": lambda: pkg.rotary(x, None, x, table, stream=stream),
            "rotate k": lambda: pkg.rotary(None, x, x, table, stream=stream),
            "tree": lambda: pkg.fused_tree(x, x, x, x, x, x, x, x, 0.1, stream=stream)}


@pytest.mark.parametrize("name", ["plan", "append", "rotate", "rotate k", "tree"])
def test_a_raw_stream_belongs_to_the_operands_device(pkg, native, name):
    """Not to the current one, where the call would run on another stream than the caller's."""
    for device in ("cuda:0", "cuda:1"):
        calls(pkg, operand(device), 0x1234)[name]()
        assert native.calls.pop() == (name.split()[0], (0x1234, torch.device(device)))
    assert native.stream is None


@pytest.mark.parametrize("name", ["plan", "append", "rotate", "rotate k", "tree"])
def test_a_stream_of_another_device_is_refused(pkg, native, name):
    stream = torch.cuda.ExternalStream(0x1234, device="cuda:1")
    with pytest.raises(pkg.VerifyError, match="stream must belong to cuda:0"):
        calls(pkg, operand("cuda:0"), stream)[name]()
    calls(pkg, operand("cuda:1"), stream)[name]()
    assert native.calls == [(name.split()[0], (0x1234, torch.device("cuda:1")))]


def test_host_operands_reach_the_checks_of_the_call(pkg, native):
    calls(pkg, operand("cpu"), 0x1234)["tree"]()
    assert native.calls == [("tree", None)]
