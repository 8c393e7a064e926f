"""GPU: how the serving calls are made - streams, derivatives, calls back to back, extreme sizes."""

import pytest

torch = pytest.importorskip("torch")

from test_gpu_serving import BF16, F32, Tree, check_rotary, ints

pytestmark = pytest.mark.gpu


def test_calls_on_a_raw_stream_handle(pkg):
    """Behind what that stream still has to do, the turn in front of the attention that reads it."""
    t = Tree(BF16, BF16, 8, 2, 128, 16, [500, 30], [3, 2], None, seed=51)
    t.run(pkg).check(pkg)
    table, pos = pkg.rotary_table(128), ints(range(t.q.shape[0]))
    q, k, v = (x.cuda().nan_to_num(0) for x in (t.q, t.k, t.v))
    want = pkg.rotary(q, k, pos, table)
    whole = [x.transpose(0, 1)[None].contiguous() for x in (q, k, v)]
    fused = pkg.fused(*whole, 0.1, causal=True, rotary=table, positions=pos)
    s = torch.cuda.Stream()
    late = [torch.zeros_like(x) for x in (q, k)]
    o, cache = torch.zeros_like(q), [x.cuda() for x in (t.kc, t.vc, t.table)] + [ints(t.held), ints(t.starts)]
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        late[0].copy_(q)
        late[1].copy_(k)
    got = pkg.rotary(*late, pos, table, stream=s.cuda_stream)
    pkg.fused_tree(late[0], k, v, *cache, t.scale, max_new=t.max_new, output=o, stream=s.cuda_stream)
    again = pkg.fused(*whole, 0.1, causal=True, rotary=table, positions=pos, stream=s.cuda_stream)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(again, fused)
    assert torch.equal(o[:t.rows], t.o[:t.rows])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_tangents_of_a_turn(pkg, dtype):
    """The map is linear: the tangent is the turned tangent."""
    T, D = 33, 64
    table, pos = pkg.rotary_table(48, [12, 12]), torch.randint(0, 5000, (2, T), device="cuda")
    q, k, tq, tk = (torch.randn(T, h, D, device="cuda").to(dtype) for h in (3, 2, 3, 2))
    fw = torch.autograd.forward_ad
    with fw.dual_level():
        a, b = pkg.rotary(fw.make_dual(q, tq), fw.make_dual(k, tk), pos, table)
        check_rotary(pkg, tq, fw.unpack_dual(a).tangent, pos, table)
        check_rotary(pkg, tk, fw.unpack_dual(b).tangent, pos, table)
        check_rotary(pkg, q, fw.unpack_dual(a).primal, pos, table)
        a, b = pkg.rotary(q, fw.make_dual(k, tk.mT.contiguous().mT), pos, table)  # a tangent of other strides
        check_rotary(pkg, tk, fw.unpack_dual(b).tangent, pos, table)
    with pytest.raises(RuntimeError, match="setup_context"):
        torch.func.jvp(lambda x: pkg.rotary(x, None, pos, table)[0], (q,), (tq,))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda x: pkg.rotary(x, None, pos, table)[0])(q[None])
    pkg.check_status(0)


def test_derivatives_that_are_refused(pkg):
    """No operand's gradient or tangent is dropped in silence."""
    t = Tree(BF16, BF16, 2, 1, 64, 16, [5], [1], tail=0)
    ops = [x.cuda().nan_to_num(0) for x in (t.q, t.k, t.v, t.kc, t.vc)]
    rest = (t.table.cuda(), ints(t.held), ints(t.starts), 1.0)
    slots = ints([3], torch.int64)
    fw = torch.autograd.forward_ad
    for i in range(5):
        other = list(ops)
        other[i] = ops[i].clone().requires_grad_()
        with pytest.raises(pkg.VerifyError, match="no backward"):
            pkg.fused_tree(*other, *rest)
        if i:
            with pytest.raises(pkg.VerifyError, match="no backward"):
                pkg.cache_append(*other[1:], slots)
        with torch.no_grad():
            pkg.fused_tree(*other, *rest)
        with fw.dual_level(), torch.no_grad():
            other[i] = fw.make_dual(ops[i], torch.ones_like(ops[i]))
            with pytest.raises(pkg.VerifyError, match="forward-mode"):
                pkg.fused_tree(*other, *rest)
            if i:
                with pytest.raises(pkg.VerifyError, match="forward-mode"):
                    pkg.cache_append(*other[1:], slots)
    pkg.check_status(0)
