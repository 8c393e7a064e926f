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

    def dual(self, q, k):
        return False

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


# ------------------------------------------------------------------ derivatives of the turn
@pytest.fixture
def turning(pkg, monkeypatch):
    """The native module's turn on CPU tensors, by the plain statement, with its own look for tangents."""
    import serving_ref as ref
    pkg.rotary  # noqa: B018

    class Module:
        dual = staticmethod(pkg.serving._native().dual)

        def rotate(self, q, k, positions, freqs, axes, neighbours, inverse):
            return tuple(None if x is None else ref.rotary(x, positions, freqs, axes, neighbours, inverse).to(x.dtype)
                         for x in (q, k))

    monkeypatch.setattr(pkg.serving, "_module", Module())
    return lambda q, k, pos, table, **kw: pkg.rotary(q, k, pos, table, **kw)


def operands(T=6, D=10, dtype=torch.float64):
    g = torch.Generator().manual_seed(3)
    q, k, tq, tk = (torch.randn(T, h, D, generator=g, dtype=dtype) for h in (3, 2, 3, 2))
    return q, k, tq, tk, torch.arange(2 * T).view(2, T) * 5


@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
def test_tangents_turn_as_the_values_do(pkg, turning, neighbours, inverse):
    q, k, tq, tk, pos = operands()
    table = pkg.rotary_table(8, [2, 2], neighbours=neighbours, device="cpu")
    want = turning(tq, tk, pos, table, inverse=inverse)
    values = turning(q, k, pos, table, inverse=inverse)
    fw = torch.autograd.forward_ad
    with fw.dual_level():
        a, b = turning(fw.make_dual(q, tq), fw.make_dual(k, tk), pos, table, inverse=inverse)
        for x, value, t in ((a, values[0], want[0]), (b, values[1], want[1])):
            assert torch.equal(fw.unpack_dual(x).primal, value) and torch.equal(fw.unpack_dual(x).tangent, t)
        # one operand has a tangent, the other none (or is not there, or wants a gradient)
        a, none = turning(fw.make_dual(q, tq), None, pos, table, inverse=inverse)
        assert none is None and torch.equal(fw.unpack_dual(a).tangent, want[0])
        a, b = turning(q, fw.make_dual(k, tk), pos, table, inverse=inverse)
        assert torch.equal(fw.unpack_dual(b).tangent, want[1])
        left = fw.unpack_dual(a).tangent
        assert left is None or not left.any()
        wants = q.clone().requires_grad_()
        a, b = turning(wants, fw.make_dual(k, tk), pos, table, inverse=inverse)
        assert torch.equal(fw.unpack_dual(b).tangent, want[1])
        with torch.no_grad():
            a, _ = turning(fw.make_dual(q, tq), None, pos, table, inverse=inverse)
            assert torch.equal(fw.unpack_dual(a).tangent, want[0])


def test_derivatives_against_differences(pkg, turning):
    q, k, _, _, pos = operands(3)
    table = pkg.rotary_table(8, [3, 1], device="cpu")
    q.requires_grad_(), k.requires_grad_()
    run = lambda a, b: turning(a, b, pos, table)  # noqa: E731
    assert torch.autograd.gradcheck(run, (q, k), check_forward_ad=True)
    assert torch.autograd.gradgradcheck(run, (q, k), check_fwd_over_rev=True)


def test_transforms_are_refused_not_ignored(pkg, turning):
    q, _, tq, _, pos = operands()
    table = pkg.rotary_table(8, device="cpu")
    run = lambda x: turning(x, None, pos[:1], table)[0]  # noqa: E731
    with pytest.raises(RuntimeError, match="setup_context"):
        torch.func.jvp(run, (q,), (tq,))
    with pytest.raises(RuntimeError, match="setup_context"):
        torch.func.grad(lambda x: run(x).sum())(q)


def test_fused_with_a_turn_refuses_what_it_cannot_differentiate(pkg):
    """Before anything else is looked at: a gradient that never arrives is worse than an error."""
    table, pos = pkg.rotary_table(8, device="cpu"), torch.arange(4)
    fw = torch.autograd.forward_ad
    for i in range(3):
        x = [torch.randn(4, 8) for _ in range(3)]
        x[i].requires_grad_()
        with pytest.raises(pkg.VerifyError, match="fused has no backward"):
            pkg.fused(*x, 0.1, rotary=table, positions=pos)
        with torch.no_grad(), pytest.raises(pkg.VerifyError, match="CUDA"):
            pkg.fused(*x, 0.1, rotary=table, positions=pos)
        x[i] = x[i].detach()
        with fw.dual_level(), pytest.raises(pkg.VerifyError, match="fused has no forward-mode"):
            pkg.fused(*(fw.make_dual(y, y) if j == i else y for j, y in enumerate(x)), 0.1, rotary=table, positions=pos)


# ------------------------------------------------------------------ what a call would write twice
@pytest.mark.parametrize("kw", [{"k_cache_stride": [0, 1024, 64]}, {"v_cache_stride": [2048, 0, 64]},
                                {"k_cache_stride": [2048, 1024, 0]}, {"v_cache_stride": [2048, 32, 64]}])
def test_a_cache_whose_rows_overlap_is_refused(pkg, kw):
    from test_serving import _append
    assert _append(pkg, **kw) == -3 and "overlap" in pkg.last_error()


@pytest.mark.parametrize("kw", [{"o_stride": [0, 128]}, {"o_stride": [1024, 0]}, {"o_stride": [1024, 64]}])
def test_a_result_whose_rows_overlap_is_refused(pkg, kw):
    from test_serving import _tree
    assert _tree(pkg, **kw) == -3 and "overlap" in pkg.last_error()


@pytest.mark.parametrize("strides", [[0, 0, 128], [0, 64, 0], [0, 32, 128]])
def test_a_turn_whose_rows_overlap_is_refused(pkg, strides):
    import ctypes
    for heads, field in (("Hq", "qo_stride"), ("Hk", "ko_stride")):
        d = pkg.AttnRotary()
        d.dtype, d.num_axes, d.B, d.N, d.D, d.R = pkg.ATTN_BF16, 1, 1, 4, 64, 64
        setattr(d, heads, 2)
        for f in ("q", "k", "qo", "ko", "positions", "freqs"):
            setattr(d, f, 0x10000)
        getattr(d, field)[:] = strides
        assert pkg.lib().attn_rotary(ctypes.byref(d), None) == -3 and "overlap" in pkg.last_error()


def test_the_c_library_builds_without_torch():
    """Its entries need none: only the calls on torch tensors are left out."""
    import os
    import subprocess
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlir-flashattention_b200", "csrc")
    plans = [subprocess.run(["make", "-C", csrc, "-n", "-B", *more], capture_output=True, text=True, check=True).stdout
             for more in ([], ["PYTHON=false"])]
    assert all("libattnrt.so" in x for x in plans)
    assert "torch_binding.cpp" in plans[0] and "torch_binding.cpp" not in plans[1]
