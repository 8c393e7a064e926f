"""GPU: how the serving calls are made - streams, derivatives, calls back to back, extreme sizes."""

import math
import threading
import time

import pytest

torch = pytest.importorskip("torch")

from test_gpu_serving import BF16, E4M3, F16, F32, Tree, check_rotary, ints

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


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("Hq,H,new,tree", [(8, 8, 1, False), (8, 8, 12, True), (32, 1, 20, True), (16, 2, 40, False)])
def test_calls_back_to_back(pkg, cache, Hq, H, new, tree):
    """A step's calls for many layers without a pause, each reading at once what the one before wrote - q and the new
    keys and values, the lengths, tables and starts of the plan, the pages: the same bits as with a wait after each, and
    from a captured graph."""
    B, D, page, pages, layers = 3, 128, 16, 200, 6
    table = pkg.rotary_table(D)
    d = 1.0 if cache is BF16 else 0.05
    g = torch.Generator(device="cuda").manual_seed(52)
    T = B * new
    x0 = torch.randn(T, Hq, D, generator=g, device="cuda").to(BF16)
    kv = [torch.randn(T, H, D, generator=g, device="cuda").to(BF16) for _ in range(2)]
    filled = [torch.randn(pages, H, page, D, generator=g, device="cuda").to(cache) for _ in range(2)]
    mask = torch.rand(T, new, generator=g, device="cuda") < 0.5 if tree else None
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)

    def fresh():
        blocks = torch.full((B, 60), -1, dtype=torch.int32, device="cuda")
        held = [700, 5, 16]
        at = 0
        for b, n in enumerate(held):
            blocks[b, :-(-n // page)] = order[at:at - (-n // page)]
            at -= -n // page
        free = torch.cat([order[at:], order.new_full((at,), -1)])
        return [x.clone() for x in filled], ints(held), blocks, free, ints([pages - at]), x0.clone()

    def steps(state, pause):
        (kc, vc), lengths, blocks, free, count, x = state
        lse = []
        for _ in range(2):
            want = lengths + new
            plan = pkg.cache_plan(lengths, want, blocks, free, count, page, T)
            pause()
            for _ in range(layers):
                q, k = pkg.rotary(x, kv[0], plan.positions, table)
                pause()
                lse.append(torch.empty(T, Hq, device="cuda"))
                pkg.fused_tree(q, k, kv[1], kc, vc, blocks, lengths, plan.starts, 0.1, mask=mask, max_new=new, output=x,
                               lse=lse[-1], k_descale=d, v_descale=d)
                pause()
                x = pkg.fused_tree(x, k, x[:, :H], kc, vc, blocks, lengths, plan.starts, 0.1, mask=mask, max_new=new,
                                   k_descale=d, v_descale=d)
                pause()
                pkg.cache_append(k, kv[1], kc, vc, plan.slots, k_descale=d, v_descale=d)
                pause()
            lengths, count = plan.lengths, plan.free_count
        return [x, *lse, kc.view(torch.uint8), vc.view(torch.uint8), blocks, free]

    want = steps(fresh(), torch.cuda.synchronize)
    pkg.check_status(0)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(steps(fresh(), lambda: None), want))
    state = fresh()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = steps(state, lambda: None)
    again = fresh()
    for _ in range(2):
        for a, b in zip([*state[0], *state[1:]], [*again[0], *again[1:]]):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    pkg.check_status(0)


def test_plan_with_as_many_tokens_as_there_may_be(pkg):
    """A padded call of 2^31 - 1 tokens: indexes that step past 2^31 end the loop."""
    tokens = (1 << 31) - 1
    blocks, free = ints([[3, -1], [-1, -1]]), ints([9, 8, 7])
    lengths = ints([10, 0])
    slots = torch.full((tokens,), 5, dtype=torch.int64, device="cuda")
    plan = pkg.cache_plan(lengths, ints([20, 5]), blocks, free, ints([3]), 16, tokens, slots=slots)
    pkg.check_status(0)
    want = [58, 59, 60, 61, 62, 63, 112, 113, 114, 115, 128, 129, 130, 131, 132]  # pages 3 and 7, then 8
    assert slots[:15].tolist() == want and plan.starts.tolist() == [0, 10, 15]
    assert plan.positions[:15].tolist() == [*range(10, 20), *range(5)] and blocks.tolist() == [[3, 7], [8, -1]]
    for at in range(15, tokens, 1 << 28):
        assert bool((slots[at:at + (1 << 28)] == -1).all()) and not plan.positions[at:at + (1 << 28)].any()


@pytest.mark.parametrize("new", [1, 60])
def test_a_request_as_long_as_there_may_be(pkg, new):
    """2^31 - 16 cached tokens, one page over and over: the number of key tiles is taken past 2^31.

    Each of a share's four warps (60 rows: each share's two accumulators) adds 2^31 / (296 * 4) keys, 16 to 128 at a
    time, one after another in 32 bits: 1.2e5 additions off by 2^-23 of the sum at most in the products, 4 a lane in the
    weights: 4.6e5 by 2^-24, below 3 % in all, of both the sums that O divides; 0.03 in LSE."""
    W, page, D = (1 << 27) - 1, 16, 64
    g = torch.Generator().manual_seed(53)
    q, k, v = (torch.randn(new, 1, D, generator=g).to(F16) for _ in range(3))
    kc, vc = (torch.randn(1, 1, page, D, generator=g).to(F16) for _ in range(2))
    o, lse = torch.empty(new, 1, D, dtype=F16, device="cuda"), torch.empty(new, 1, device="cuda")
    pkg.fused_tree(q.cuda(), k.cuda(), v.cuda(), kc.cuda(), vc.cuda(), torch.zeros(1, W, dtype=torch.int32, device="cuda"),
                   ints([W * page]), ints([0, new]), 0.1, max_new=new, output=o, lse=lse)
    pkg.check_status(0)
    s = q[:, 0].double() @ kc[0, 0].double().T * 0.1  # the new keys weigh 2^-27 of these
    want, size = torch.softmax(s, 1) @ vc[0, 0].double(), torch.softmax(s, 1) @ vc[0, 0].double().abs()
    assert bool(((o.cpu().double()[:, 0] - want).abs() <= 0.06 * size).all())
    assert bool(((lse.cpu().double()[:, 0] - torch.logsumexp(s, 1) - 27 * 0.6931471805599453).abs() <= 0.03).all())


@pytest.mark.parametrize("name", ["plan", "append", "rotary", "tree"])
def test_other_threads_run_while_a_call_waits_for_the_queue(pkg, name):
    """A call that finds the launch queue full waits for the GPU without the interpreter's lock."""
    t = Tree(BF16, BF16, 2, 1, 64, 16, [30], [2], None, seed=54, tail=0)
    q, k, v, kc, vc, blocks = (x.cuda().nan_to_num(0) for x in (t.q, t.k, t.v, t.kc, t.vc, t.table))
    held, starts, slots, table = ints(t.held), ints(t.starts), ints([16, 17], torch.int64), pkg.rotary_table(64)
    free, count, pos = ints([0, 1]), ints([2]), ints([3, 4])
    calls = {"plan": lambda: pkg.cache_plan(held, held, blocks, free, count, 16, 2),
             "append": lambda: pkg.cache_append(k, v, kc, vc, slots),
             "rotary": lambda: pkg.rotary(q, k, pos, table),
             "tree": lambda: pkg.fused_tree(q, k, v, kc, vc, blocks, held, starts, 0.1, max_new=2)}
    calls[name]()
    torch.cuda.synchronize()
    ticks, done = [], threading.Event()

    def tick():
        while not done.wait(0.001):
            ticks.append(time.perf_counter())

    other = threading.Thread(target=tick)
    other.start()
    try:
        torch.cuda._sleep(1_500_000_000)  # about 0.8 s
        begin = time.perf_counter()
        for _ in range(3000):
            calls[name]()
        took = time.perf_counter() - begin
    finally:
        done.set()
        other.join()
    torch.cuda.synchronize()
    pkg.check_status(0)
    assert took > 0.4, "the queue never filled"
    inside = [x for x in ticks if begin < x < begin + took]
    assert max(b - a for a, b in zip([begin, *inside], [*inside, begin + took])) < 0.2


def test_what_a_call_writes_is_known_to_autograd(pkg):
    """Positions that a turn saved for its gradient and a later plan overwrites: an error, not another gradient."""
    x, table = torch.randn(2, 1, 64, device="cuda", requires_grad=True), pkg.rotary_table(64)
    lengths, blocks, free = ints([3]), ints([[1, -1]]), ints([0])
    plan = pkg.cache_plan(lengths, ints([5]), blocks, free, ints([1]), 16, 2)
    y, _ = pkg.rotary(x, None, plan.positions, table)
    pkg.cache_plan(ints([5]), ints([7]), blocks, free, ints([1]), 16, 2, positions=plan.positions)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    t = Tree(BF16, BF16, 2, 1, 64, 16, [5], [1], None, seed=55, tail=0)
    q, k, v, kc, vc = (z.cuda().nan_to_num(0) for z in (t.q, t.k, t.v, t.kc, t.vc))
    lse, o = torch.empty(1, 2, device="cuda"), torch.empty_like(q)
    before = [z._version for z in (q, k, v, kc, vc, o, lse)]
    pkg.fused_tree(q, k, v, kc, vc, t.table.cuda(), ints(t.held), ints(t.starts), 0.1, output=o, lse=lse)
    pkg.cache_append(k, v, kc, vc, ints([8], torch.int64))
    assert [z._version - n for z, n in zip((q, k, v, kc, vc, o, lse), before)] == [0, 0, 0, 1, 1, 1, 1]
    with torch.inference_mode():  # tensors that count no versions
        made = [z.clone() for z in (q, k, v, kc, vc)]
    pkg.cache_append(*made[1:], ints([8], torch.int64))
    pkg.fused_tree(*made, t.table.cuda(), ints(t.held), ints(t.starts), 0.1, output=made[0])
    pkg.check_status(0)


def test_threads_call_at_once(pkg):
    """Each on a stream of its own, refused calls among them: the bits of a call alone, and each thread its own error."""
    shapes = [(8, 2, 128, [3000, 7], [1, 1], None), (32, 1, 128, [500], [40], "tree"), (4, 4, 64, [0, 900], [9, 3], None)]
    trees = [Tree(BF16, BF16, *s[:3], 16, *s[3:], seed=56) for s in shapes]
    want = [(t.run(pkg).o.clone(), t.lse.clone()) for t in trees]
    dev = [[x.cuda() for x in (t.q, t.k, t.v, t.kc, t.vc, t.table)] + [ints(t.held), ints(t.starts)] for t in trees]
    masks = [None if t.mask is None else t.mask.cuda() for t in trees]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            t = trees[i]
            refused, why = ({"k_descale": 2.0}, "descales apply") if i == 1 else ({"scale": math.nan}, "scale must be finite")
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(60):
                    o, lse = torch.full_like(want[i][0], 7), torch.full_like(want[i][1], 7)
                    args = {"scale": t.scale, "mask": masks[i], "max_new": t.max_new, "output": o, "lse": lse}
                    pkg.fused_tree(*dev[i], **args)
                    with pytest.raises(pkg.AttentionError, match=why):
                        pkg.fused_tree(*dev[i], **{**args, **refused})
                    torch.cuda.current_stream().synchronize()
                    if not (torch.equal(o, want[i][0]) and torch.equal(lse, want[i][1])):
                        wrong.append(i)
        except BaseException as e:  # noqa: BLE001
            wrong.append((i, repr(e)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    pkg.check_status(0)
    assert not wrong
