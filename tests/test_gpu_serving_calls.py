"""GPU: how the serving calls are made - streams, derivatives, calls back to back, extreme sizes."""

import pytest

torch = pytest.importorskip("torch")

from test_gpu_serving import BF16, Tree, ints

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
