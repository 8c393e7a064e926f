"""GPU parity of the serving calls against plain 64-bit statements (serving_ref.py).

Tolerances, with u = eps / 2 of a type (half a step, relative):
* copies, page lists and e4m3 codes are exact (one correctly rounded division);
* rotary: |out - ref| <= u |ref| + 2^-21 (|x| + |y|): one rounding of the output; cos, sin and the two products in 32
  bits, the reduced angle (a fraction of a turn below 1/2) being off by 2^-26 turns = 2^-23.3 radians;
* attention: |O - ref| <= u |ref| + 1.1 u A + 1e-6 max A with A = sum p |v| of the row: one rounding of O, one of every
  weight p to the operands' type (an e4m3 cache is met in f16 or finer), and a tenth for scores and exponentials in
  32 bits;
* LSE: N 2^-24 + 2^-17 for N keys: a serial 32-bit sum, and scores below 32 in 32 bits.
"""
import math
import random

import pytest

torch = pytest.importorskip("torch")

import serving_ref as ref

pytestmark = pytest.mark.gpu

BF16, F16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


# ------------------------------------------------------------------ planner
def check_plan(pkg, lengths, targets, table, free, count, page, tokens, in_place=False):
    tl, tt, ttab, tf, tc = (ints(x) for x in (lengths, targets, table, free, [count]))
    ttab = ttab.reshape(len(lengths), -1)
    kw = {"lengths_out": tl, "free_count_out": tc} if in_place else {}
    r = pkg.cache_plan(tl, tt, ttab, tf, tc, page, tokens, **kw)
    want = ref.plan(lengths, targets, table, free, count, page, tokens)
    got = (r.slots.tolist(), r.positions.tolist(), r.starts.tolist(), r.lengths.tolist(), ttab.tolist(), tf.tolist(),
           r.free_count.tolist()[0])
    for g, w, name in zip(got, want[:7], ("slots", "positions", "starts", "lengths", "table", "free", "count")):
        assert g == w, name
    if want[7]:
        pkg.check_status(0)
    else:
        with pytest.raises(pkg.AttentionError):
            pkg.check_status(0)
    if not in_place:
        assert tl.tolist() == list(lengths) and tc.tolist() == [count]
    return got


def random_plan(rng, B, page, most, tokens_slack=3):
    width = -(-most // page) + 1
    lengths = [rng.choice([0, rng.randrange(most + 1), page * rng.randrange(most // page + 1)]) for _ in range(B)]
    targets = [rng.choice([n, min(most, n + 1), 0, rng.randrange(most + 1)]) for n in lengths]
    used = sum(-(-n // page) for n in lengths)
    need = sum(max(0, -(-t // page) + -(-n // -page)) for n, t in zip(lengths, targets))
    order = list(range(used + need + 5))
    rng.shuffle(order)
    table, at = [], 0
    for n in lengths:
        k = -(-n // page)
        table.append(order[at:at + k] + [-7] * (width - k))
        at += k
    free = order[used:] + [-9] * used
    new = sum(max(0, t - n) for n, t in zip(lengths, targets))
    return lengths, targets, table, free, len(order) - used, page, new + rng.randrange(tokens_slack + 1)


@pytest.mark.parametrize("B,page,most", [(1, 16, 100), (3, 16, 40), (33, 64, 1000), (256, 16, 300), (257, 32, 500),
                                         (1025, 1024, 5000), (3000, 16, 64), (8192, 16, 40)])
def test_plan_matches_lists(pkg, B, page, most):
    rng = random.Random(B + page)
    for in_place in (False, True):
        check_plan(pkg, *random_plan(rng, B, page, most), in_place=in_place)


def test_plan_long_prompts_use_many_blocks(pkg):
    check_plan(pkg, [0, 5, 7000], [40000, 20005, 0], [[-1] * 2500, [9] + [-1] * 2499, list(range(10, 448)) + [-1] * 2062],
               list(range(500, 4700)) + [-1] * 600, 4200, 16, 61000)


def test_plan_takes_pages_given_back_in_the_same_call(pkg):
    got = check_plan(pkg, [32, 0, 16], [0, 64, 0], [[3, 4, -1, -1], [-1] * 4, [5, -1, -1, -1]], [9, 8, -1, -1, -1], 2, 16,
                     64)
    assert got[4][1] == [5, 4, 3, 8]


def test_plan_is_all_or_nothing(pkg):
    table = [[1, -1], [2, -1]]
    check_plan(pkg, [16, 16], [32, 33], table, [7, 8], 2, 16, 40)     # a table row too short
    check_plan(pkg, [16, 16], [32, 32], table, [7], 1, 16, 40)        # a page too few
    check_plan(pkg, [16, 16], [32, 32], table, [7, 8], 2, 16, 31)     # a slot too few
    check_plan(pkg, [16, -1], [32, 32], table, [7, 8], 2, 16, 40)     # lengths that cannot be
    check_plan(pkg, [16, 40], [32, 32], table, [7, 8], 2, 16, 40)
    check_plan(pkg, [16, 16], [32, -3], table, [7, 8], 2, 16, 40)
    check_plan(pkg, [16, 16], [32, 32], table, [7, 8], 2, 16, 40)     # and the next call runs
    tl = ints([16, 16])
    pkg.cache_plan(tl, ints([32, 32]), ints(table), ints([7, 8]), ints([3]), 16, 40)  # a count past the stack
    with pytest.raises(pkg.AttentionError, match="invalid"):
        pkg.check_status(0)


def test_plan_without_requests_or_tokens(pkg):
    r = pkg.cache_plan(ints([]), ints([]), torch.empty(0, 4, dtype=torch.int32, device="cuda"), ints([1, 2]), ints([2]), 16,
                       3)
    assert r.slots.tolist() == [-1] * 3 and r.starts.tolist() == [0] and r.free_count.tolist() == [2]
    check_plan(pkg, [5], [2], [[4]], [-1], 0, 16, 0)


def test_plan_in_a_graph_decodes_step_by_step(pkg):
    """lengths, targets and the count updated in place by replays of one captured step."""
    page, B = 16, 5
    lengths, targets = ints([0, 3, 15, 16, 31]), ints([1, 4, 16, 17, 32])
    table = torch.full((B, 6), -1, dtype=torch.int32, device="cuda")
    table[1, 0], table[2, 0], table[3, 0], table[4, 0], table[4, 1] = 20, 21, 22, 23, 24
    free, count = ints(list(range(20)) + [-1] * 5), ints([20])
    state = [x.tolist() for x in (lengths, targets, table, free)] + [20]
    out = [torch.empty(B, dtype=torch.int64, device="cuda"), torch.empty(B, dtype=torch.int32, device="cuda"),
           torch.empty(B + 1, dtype=torch.int32, device="cuda")]

    def step():
        pkg.cache_plan(lengths, targets, table, free, count, page, B, lengths_out=lengths, free_count_out=count,
                       slots=out[0], positions=out[1], starts=out[2])
        targets.add_(1)

    check_plan(pkg, [5], [2], [[4]], [-1], 0, 16, 0)  # a device's first call is made outside capture
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for _ in range(40):
        g.replay()
        torch.cuda.synchronize()
        n, t, tab, fr, c = state
        want = ref.plan(n, t, tab, fr, c, page, B)
        assert out[0].tolist() == want[0] and out[1].tolist() == want[1]
        assert table.tolist() == want[4] and count.tolist() == [want[6]] and lengths.tolist() == want[3]
        state = [want[3], [x + 1 for x in want[3]], want[4], want[5], want[6]]
    pkg.check_status(0)


# ------------------------------------------------------------------ writer
def fp8_of(x, descale):
    return (x.float() / descale).clamp(-448, 448).to(E4M3)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("cache", [None, E4M3])
@pytest.mark.parametrize("T,H,D,page", [(1, 1, 16, 16), (7, 3, 64, 32), (300, 8, 128, 16), (5000, 2, 128, 1024)])
def test_append_matches_indexing(pkg, dtype, cache, T, H, D, page):
    gen = torch.Generator().manual_seed(T + D)
    kind = cache or dtype
    pages = -(-T // page) + 3
    k, v = (torch.randn(T, H, D, generator=gen).to(dtype) * 3 for _ in range(2))
    k[0, 0, 0], v[0, 0, 1] = float("inf"), float("nan")
    slots = torch.randperm(pages * page, generator=gen)[:T]
    slots[torch.rand(T, generator=gen) < 0.3] = -1
    rows = torch.randint(0, T, (T,), generator=gen, dtype=torch.int32)
    heads = torch.rand(H, generator=gen) + 0.01
    old = [torch.randn(pages, H, page, D, generator=gen).to(kind) for _ in range(2)]
    for r in (None, rows):
        for kd, vd in ([(1.0, 1.0)] if cache is None else [(0.02, 0.5), (heads, 0.3)]):
            kc, vc = (x.cuda() for x in old)
            dev = lambda x: x.cuda() if isinstance(x, torch.Tensor) else x  # noqa: E731
            pkg.cache_append(k.cuda(), v.cuda(), kc, vc, slots.cuda(), rows=dev(r) if r is not None else None,
                             k_descale=dev(kd), v_descale=dev(vd))
            pkg.check_status(0)
            for x, got, before, d in ((k, kc, old[0], kd), (v, vc, old[1], vd)):
                want = before.clone()
                d = d[:, None] if isinstance(d, torch.Tensor) else d
                src = x if r is None else x[r.long()]
                put = fp8_of(src, d) if cache else src
                at = slots >= 0
                want.view(torch.uint8 if cache else torch.int16)[slots[at] // page, :, slots[at] % page] = \
                    put[at].view(torch.uint8 if cache else torch.int16)
                same = got.cpu().view(torch.uint8 if cache else torch.int16) == want.view(torch.uint8 if cache else torch.int16)
                nan = got.cpu().float().isnan() & want.float().isnan()  # any NaN code
                assert bool((same | nan).all())


def test_append_strides_and_wrong_slots(pkg):
    T, H, D, page, pages = 9, 2, 64, 16, 4
    qkv = torch.randn(T, 4 + 2 * H, D, device="cuda").to(BF16)
    k, v = qkv[:, 4:4 + H], qkv[:, 4 + H:]
    kc = torch.zeros(pages, page, H, D, dtype=BF16, device="cuda")  # tokens outside heads
    vc = torch.zeros(H, pages, page, D, dtype=BF16, device="cuda")
    slots = ints([3, 17, -1, 63, 64, -5, 40, 1 << 40, 41], torch.int64)
    pkg.cache_append(k, v, kc.transpose(1, 2), vc.transpose(0, 1), slots)
    with pytest.raises(pkg.AttentionError, match="invalid"):
        pkg.check_status(0)
    for i, s in ((0, 3), (1, 17), (3, 63), (6, 40), (8, 41)):
        assert torch.equal(kc[s // page, s % page], k[i]) and torch.equal(vc[:, s // page, s % page], v[i])
    assert int((kc != 0).any(-1).any(-1).sum()) == 5
    rows = ints([0, 9, -1])
    pkg.cache_append(k, v, kc.transpose(1, 2), vc.transpose(0, 1), ints([0, 1, 2], torch.int64), rows=rows)
    with pytest.raises(pkg.AttentionError, match="invalid"):
        pkg.check_status(0)
    assert torch.equal(kc[0, 0], k[0]) and not kc[0, 1].any() and not kc[0, 2].any()


def test_append_past_32_bits(pkg):
    """A cache of more than 2^32 elements."""
    H, page, D = 8, 1024, 128
    pages = (1 << 32) // (H * page * D) + 3
    kc, vc = (torch.empty(pages, H, page, D, dtype=E4M3, device="cuda") for _ in range(2))
    k = torch.randn(3, H, D, device="cuda").to(BF16)
    slots = [pages * page - 1, 5, (pages - 2) * page]
    pkg.cache_append(k, -k, kc, vc, ints(slots, torch.int64), k_descale=0.1, v_descale=0.1)
    pkg.check_status(0)
    for i, s in enumerate(slots):
        want = fp8_of(k[i].cpu(), 0.1)
        assert torch.equal(kc[s // page, :, s % page].cpu().view(torch.uint8), want.view(torch.uint8))
        assert torch.equal(vc[s // page, :, s % page].cpu().float(), -want.float())


# ------------------------------------------------------------------ rotary
def check_rotary(pkg, x, got, positions, table, inverse=False):
    """x, got [T, H, D]."""
    want = ref.rotary(x.cpu(), positions.cpu(), table.freqs.cpu(), table.axes.cpu(), table.neighbours, inverse)
    x64, half = x.cpu().double(), len(table.freqs)
    size = x64.abs()
    turned = size[..., :2 * half]
    pair = turned[..., 0::2] + turned[..., 1::2] if table.neighbours else turned[..., :half] + turned[..., half:]
    both = torch.stack([pair, pair], -1).flatten(-2) if table.neighbours else torch.cat([pair, pair], -1)
    tol = half_step(x.dtype) * want.abs()
    tol[..., :2 * half] += 2.0 ** -21 * both
    assert bool(((got.detach().cpu().double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("T,Hq,Hk,D,dim,sections", [
    (1, 1, 1, 64, 64, None), (5, 12, 2, 128, 128, [24, 20, 20]), (130, 4, 4, 64, 32, [8, 8]), (33, 3, 1, 80, 40, [7, 7, 6]),
    (1000, 2, 1, 18, 6, [1, 1, 1]), (17, 1, 1, 7, 2, None), (9, 2, 1, 256, 256, [64, 32, 32])])
def test_rotary_matches(pkg, dtype, neighbours, T, Hq, Hk, D, dim, sections):
    gen = torch.Generator(device="cuda").manual_seed(T * D)
    q, k = (torch.randn(T, h, D, generator=gen, device="cuda").to(dtype) for h in (Hq, Hk))
    for interleaved in (False, True):
        table = pkg.rotary_table(dim, sections, interleaved=interleaved, neighbours=neighbours)
        pos = torch.randint(-50, 1 << 20, (len(sections or [1]), T), generator=gen, device="cuda", dtype=torch.int32)
        a, b = pkg.rotary(q, k, pos, table)
        check_rotary(pkg, q, a, pos, table)
        check_rotary(pkg, k, b, pos, table)
        only, none = pkg.rotary(q, None, pos.long(), table.freqs, table.axes, neighbours=neighbours, inverse=True)
        assert none is None
        check_rotary(pkg, q, only, pos, table, inverse=True)
    pkg.check_status(0)


def test_rotary_far_positions_and_layouts(pkg):
    """[B, H, N, D] with batched positions near 2^31, from a fused projection whose rows are not 16-byte aligned."""
    B, N, Hq, Hk, D = 2, 37, 3, 2, 64
    table = pkg.rotary_table(D, [16, 8, 8], 1e6)
    pos = (2 ** 31 - 1 - torch.arange(3 * B * N, device="cuda").reshape(3, B, N) * 977).to(torch.int32)
    for pad in (0, 3):
        x = torch.randn(B, N, (Hq + Hk) * D + pad, device="cuda").to(BF16)
        q = x[..., :Hq * D].view(B, N, Hq, D).transpose(1, 2) if not pad else \
            x.as_strided((B, Hq, N, D), (N * x.shape[2], D, x.shape[2], 1))
        k = x.as_strided((B, Hk, N, D), (N * x.shape[2], D, x.shape[2], 1), Hq * D + pad)
        a, b = pkg.rotary(q, k, pos, table)
        assert a.shape == q.shape
        for i in range(B):
            check_rotary(pkg, q[i].transpose(0, 1), a[i].transpose(0, 1), pos[:, i], table)
            check_rotary(pkg, k[i].transpose(0, 1), b[i].transpose(0, 1), pos[:, i], table)
        c, _ = pkg.rotary(q, None, pos[:, 0], table)  # the same positions for every batch
        check_rotary(pkg, q[1].transpose(0, 1), c[1].transpose(0, 1), pos[:, 0], table)
    pkg.check_status(0)


def test_rotary_wrong_axis_is_recorded(pkg):
    x = torch.randn(4, 1, 8, device="cuda")
    pkg.rotary(x, None, ints([[1, 2, 3, 4]]), torch.ones(4, dtype=torch.float64, device="cuda"), ints([0, 1, 0, -1]))
    with pytest.raises(pkg.AttentionError, match="invalid"):
        pkg.check_status(0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("neighbours", [False, True])
def test_rotary_gradient(pkg, dtype, neighbours):
    """Against the formula (the transpose of a turn is the turn back) and against differences of a loss."""
    T, Hq, Hk, D = 11, 3, 2, 32
    table = pkg.rotary_table(24, [6, 3, 3], neighbours=neighbours)
    pos = torch.randint(0, 5000, (3, T), device="cuda")
    q, k = (torch.randn(T, h, D, device="cuda").to(dtype).requires_grad_() for h in (Hq, Hk))
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    a, b = pkg.rotary(q, k, pos, table)
    dq, dk = torch.autograd.grad((a, b), (q, k), (gq, gk))
    check_rotary(pkg, gq, dq, pos, table, inverse=True)
    check_rotary(pkg, gk, dk, pos, table, inverse=True)
    a, b = pkg.rotary(q, k, pos, table)
    (only,) = torch.autograd.grad(a, (q,), gq)  # K unused
    assert torch.equal(only, dq)
    (wide,) = torch.autograd.grad(pkg.rotary(q, None, pos, table)[0].sum(), (q,))  # an expanded gradient
    check_rotary(pkg, torch.ones_like(q), wide, pos, table, inverse=True)
    if dtype == F32:  # the map is linear: a difference over any step is the derivative
        step = torch.randn_like(q)
        with torch.no_grad():
            rise = ((pkg.rotary(q + step, None, pos, table)[0] - pkg.rotary(q, None, pos, table)[0]).double() * gq).sum()
        # 2^-22 per value for each of the two outputs and the sum q + step, values and gradients of order 1
        assert abs(float(rise - (dq.double() * step).sum())) <= 8 * 2.0 ** -22 * q.numel() * 4
        assert torch.autograd.gradcheck(lambda x: _second(pkg, x, pos, table, gq), (q,), eps=0.5, atol=1e-3, rtol=1e-3)


def _second(pkg, x, pos, table, g):
    return (pkg.rotary(x, None, pos, table)[0] * g).sum(-1)


def test_rotary_backward_in_a_graph(pkg):
    T, H, D = 16, 4, 64
    table = pkg.rotary_table(D)
    pos = torch.arange(T, device="cuda")
    q = torch.randn(T, H, D, device="cuda", requires_grad=True)
    g = torch.randn(T, H, D, device="cuda")
    want = torch.autograd.grad(pkg.rotary(q, None, pos, table)[0], q, g)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(pkg.rotary(q, None, pos, table)[0], q, g)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(pkg.rotary(q, None, pos, table)[0], q, g)[0]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_fused_turns_q_and_k(pkg):
    B, Hq, Hk, N, D = 2, 4, 2, 200, 64
    q, k, v = (torch.randn(B, h, N, D, device="cuda").to(BF16) for h in (Hq, Hk, Hk))
    table = pkg.rotary_table(D, [16, 8, 8])
    pos = torch.randint(0, 300, (3, B, N), device="cuda")
    got = pkg.fused(q, k, v, 0.125, causal=True, rotary=table, positions=pos)
    a, b = pkg.rotary(q, k, pos, table)
    assert torch.equal(got, pkg.fused(a, b, v, 0.125, causal=True))
    one = pkg.fused(q[0, 0], k[0, 0], v[0, 0], 0.125, rotary=table, positions=pos[:, 0])
    a, b = pkg.rotary(q[:1, :1], k[:1, :1], pos[:, 0], table)
    assert torch.equal(one, pkg.fused(a, b, v[:1, :1], 0.125)[0, 0])


# ------------------------------------------------------------------ attention
class Tree:
    """One call: ragged requests over shuffled pages, everything that must not be read poisoned with NaN."""

    def __init__(self, dtype, cache, Hq, H, D, page, held, new, mask=None, seed=0, tail=3, std=1.0):
        g = torch.Generator().manual_seed(seed)
        rng = random.Random(seed)
        counts = [-(-n // page) for n in held]
        pages, width = sum(counts) + 2, max(counts, default=0) + 1
        order = list(range(pages))
        rng.shuffle(order)
        self.table = torch.full((len(held), width), -1, dtype=torch.int32)
        nan = float("nan")
        self.kc, self.vc = (torch.full((pages, H, page, D), nan).to(cache) for _ in range(2))
        at = 0
        for b, (n, c) in enumerate(zip(held, counts)):
            ids = order[at:at + c]
            at += c
            self.table[b, :c] = torch.tensor(ids, dtype=torch.int32)
            for x in (self.kc, self.vc):
                rows = (torch.randn(n, H, D, generator=g) * std).to(cache)
                for j in range(c):
                    part = rows[j * page:(j + 1) * page].transpose(0, 1)
                    x.view(torch.uint8 if cache is E4M3 else cache)[ids[j], :, :part.shape[1]] = \
                        part.view(torch.uint8 if cache is E4M3 else cache)
        self.held, self.starts = list(held), [sum(new[:b]) for b in range(len(new) + 1)]
        self.rows = self.starts[-1]
        T = self.rows + tail  # rows behind the last request
        self.q, self.k, self.v = (torch.randn(T, h, D, generator=g).mul_(std).to(dtype) for h in (Hq, H, H))
        for x in (self.q, self.k, self.v):
            x[self.rows:] = nan
        self.max_new, self.mask = max(new, default=0), None
        if mask is not None:
            self.mask = torch.ones(T, self.max_new + 5, dtype=torch.bool)
            for b, n in enumerate(new):
                for i in range(n):
                    if mask == "tree":
                        parent = rng.randrange(-1, i) if i else -1
                        if parent >= 0:
                            self.mask[self.starts[b] + i] = self.mask[self.starts[b] + parent]
                        self.mask[self.starts[b] + i, i] = False
                    elif mask == "random":
                        self.mask[self.starts[b] + i, :n] = torch.rand(n, generator=g) < 0.6
                    # "empty": nothing of the new tokens is seen
        self.kd, self.vd = (1.0, 1.0) if cache is not E4M3 else (0.7, 1.3)
        self.scale = 1.0 / math.sqrt(D)

    def run(self, pkg, **kw):
        d = lambda x: x.cuda() if isinstance(x, torch.Tensor) else x  # noqa: E731
        self.o = torch.full(self.q.shape, 7.0, dtype=self.q.dtype, device="cuda")
        self.lse = torch.full(self.q.shape[:2], 7.0, device="cuda")
        args = dict(mask=None if self.mask is None else d(self.mask), max_new=self.max_new, output=self.o, lse=self.lse,
                    k_descale=d(self.kd), v_descale=d(self.vd))
        args.update(kw)
        pkg.fused_tree(d(self.q), d(self.k), d(self.v), d(self.kc), d(self.vc), d(self.table), ints(self.held),
                       ints(self.starts), self.scale, **args)
        return self

    def check(self, pkg):
        pkg.check_status(0)
        n = self.rows
        o, lse, a = ref.tree(self.q[:n], self.k[:n], self.v[:n], self.kc, self.vc, self.table, self.held, self.starts,
                             self.scale, self.mask, self.kd, self.vd)
        got, glse, u = self.o.cpu().double(), self.lse.cpu().double(), half_step(self.q.dtype)
        assert bool((got[n:] == 7).all()) and bool((glse[n:] == 7).all()), "rows behind the last request"
        if n == 0:
            return self
        tol = u * o.abs() + 1.1 * u * a + 1e-6 * a.amax(-1, keepdim=True)
        off = (got[:n] - o).abs()
        assert bool((off <= tol).all()), f"O off by up to {float((off / tol.clamp(min=1e-30)).max()):.2f} tolerances"
        empty = lse == -math.inf
        assert torch.equal(glse[:n] == -math.inf, empty) and not got[:n][empty].any()
        keys = max(self.held, default=0) + self.max_new
        assert bool(((glse[:n] - lse)[~empty].abs() <= keys * 2.0 ** -24 + 2.0 ** -17).all())
        return self


TYPES = [(BF16, BF16), (F16, F16), (BF16, E4M3), (F16, E4M3)]


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("Hq,H,D", [(4, 4, 64), (8, 1, 128), (7, 1, 64), (6, 2, 128), (16, 1, 128), (40, 2, 64)])
def test_decode(pkg, dtype, cache, Hq, H, D):
    if cache is E4M3 and D == 64:
        D = 128
    for page in (16, 64, 256):
        Tree(dtype, cache, Hq, H, D, page, [0, 1, 15, 16, 63, 64, 65, 127, 128, 129, 300, 1000], [1] * 12,
             seed=page).run(pkg).check(pkg)


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("mask", [None, "tree", "random", "empty"])
@pytest.mark.parametrize("Hq,H,D", [(2, 2, 64), (4, 1, 128), (6, 2, 128), (8, 1, 64)])
def test_trees(pkg, dtype, cache, mask, Hq, H, D):
    if cache is E4M3 and D == 64:
        D = 128
    for new in ([2, 0, 1, 3, 2], [17, 16, 5, 0, 64], [1, 65, 33, 40, 100]):
        Tree(dtype, cache, Hq, H, D, 32, [0, 200, 31, 129, 500], new, mask, seed=len(new) + sum(new)).run(pkg).check(pkg)


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_chunks(pkg, dtype, cache):
    """Chunks of prompts: several tiles of queries and of new keys, with and without a cached part."""
    Tree(dtype, cache, 4, 2, 128, 64, [0, 700, 128], [400, 257, 128], seed=5).run(pkg).check(pkg)
    Tree(dtype, cache, 3, 1, 128, 16, [0, 50], [130, 300], "random", seed=6).run(pkg).check(pkg)
    if cache is not E4M3:
        Tree(dtype, cache, 2, 2, 64, 128, [1000], [513], seed=7).run(pkg).check(pkg)


def test_long_request_is_split_and_joined(pkg):
    """One request over many blocks, its weight moving along the keys, and a batch as ragged as can be."""
    for dtype, cache, H, D in ((BF16, BF16, 1, 128), (F16, F16, 2, 64), (BF16, E4M3, 1, 128)):
        t = Tree(dtype, cache, 4 * H, H, D, 64, [9000], [1], seed=8)
        rise = torch.linspace(0.1, 3.0, 9000)
        for i in range(9000):
            row = t.kc[t.table[0, i // 64].item(), :, i % 64]
            row.copy_((row.float() * rise[i]).to(cache))
        t.run(pkg).check(pkg)
        Tree(dtype, cache, 4 * H, H, D, 16, [5000] + [3] * 40 + [0, 0, 2500], [1, 9] + [2] * 42, "tree", seed=9).run(pkg) \
            .check(pkg)


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("Hq,H,new", [(8, 8, 1), (8, 8, 30), (32, 8, 8), (32, 8, 20), (24, 8, 60)])
def test_blocks_take_several_tiles_and_items(pkg, dtype, cache, Hq, H, new):
    """More work than blocks: pieces of many tiles, shares that begin and end inside items."""
    held = [3000, 1, 2048, 2900, 700, 127, 1500]
    Tree(dtype, cache, Hq, H, 128, 64, held, [new, 1, new, max(1, new // 2), new, 1, new],
         "tree" if new > 1 else None, seed=new).run(pkg).check(pkg)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("Hq,H,new,B", [(16, 4, 12, 40), (4, 4, 44, 37), (4, 4, 48, 3), (5, 1, 9, 150), (16, 4, 10, 40)])
def test_rows_between_the_kernels(pkg, dtype, Hq, H, new, B):
    """33 to 48 rows at D = 64, with items for every SM and with few."""
    rng = random.Random(new)
    held = [rng.randrange(0, 200) for _ in range(B)]
    news = [rng.randrange(0, new + 1) for _ in range(B - 1)] + [new]
    Tree(dtype, dtype, Hq, H, 64, 16, held, news, "tree", seed=27).run(pkg).check(pkg)
    Tree(dtype, dtype, Hq, H, 64, 32, held, news, None, seed=28).run(pkg).check(pkg)
    Tree(dtype, dtype, Hq, H, 64, 32, [9000] + held[1:], news, "empty", seed=29).run(pkg).check(pkg)


def test_long_chunks(pkg):
    """Chains of many row tiles: more items than blocks, accumulators whose keys end at different tiles."""
    Tree(BF16, BF16, 16, 4, 128, 128, [300, 0], [1300, 900], seed=22).run(pkg).check(pkg)
    Tree(F16, F16, 8, 8, 64, 64, [600], [2000], seed=23).run(pkg).check(pkg)


def test_many_small_requests(pkg):
    Tree(BF16, BF16, 4, 2, 128, 16, [i % 50 for i in range(700)], [i % 3 for i in range(700)], seed=10).run(pkg).check(pkg)
    Tree(F16, F16, 2, 1, 64, 16, [0] * 300, [1] * 300, seed=11).run(pkg).check(pkg)


def test_large_scores_and_negative_scale(pkg):
    """A softmax that a few keys win, scores of several hundred, and a scale below 0 or of 0."""
    t = Tree(BF16, BF16, 4, 1, 128, 32, [500, 90], [9, 40], "tree", seed=12, std=3.0)
    t.scale = 0.3  # scores to about 300: 32-bit scores are off by 300 2^-22, so weights by 2^-13, inside the tenth of u
    u = half_step(BF16)
    t.run(pkg)
    pkg.check_status(0)
    n = t.rows
    o, lse, a = ref.tree(t.q[:n], t.k[:n], t.v[:n], t.kc, t.vc, t.table, t.held, t.starts, t.scale, t.mask)
    assert bool(((t.o.cpu().double()[:n] - o).abs() <= u * o.abs() + 1.1 * u * a + 1e-6 * a.amax(-1, keepdim=True)).all())
    assert bool(((t.lse.cpu().double()[:n] - lse).abs() <= 300 * 2.0 ** -20).all())
    for scale in (-0.1, 0.0):
        t = Tree(F16, F16, 4, 2, 64, 32, [100, 0], [1, 20], seed=13)
        t.scale = scale
        t.run(pkg).check(pkg)


def test_infinite_and_nan_keys_under_the_mask(pkg):
    """A drafted token whose K is NaN or infinite, seen by itself alone, spoils no other row."""
    for Hq, H in ((4, 2), (32, 2)):
        t = Tree(BF16, BF16, Hq, H, 128, 16, [40], [8], "tree", seed=14)
        t.mask[:, 5] = True
        t.mask[5, 5] = False
        for bad in (float("nan"), float("inf"), torch.finfo(BF16).min):
            t.k[5] = bad
            keep = [i for i in range(8) if i != 5]
            t.run(pkg)
            pkg.check_status(0)
            o, lse, a = ref.tree(t.q[:8], t.k[:8].nan_to_num(0, 0, 0), t.v[:8], t.kc, t.vc, t.table, t.held, t.starts,
                                 t.scale, t.mask)
            u = half_step(BF16)
            tol = u * o.abs() + 1.1 * u * a + 1e-6 * a.amax(-1, keepdim=True)
            assert bool(((t.o.cpu().double()[:8] - o).abs() <= tol)[keep].all())


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("Hq,H,new,held", [(4, 2, 8, 40), (16, 2, 8, 300), (32, 2, 8, 40), (32, 1, 40, 3000), (4, 4, 8, 9000)])
def test_values_under_the_mask(pkg, dtype, cache, Hq, H, new, held):
    """A drafted token's value that is infinite or no number reaches the rows that see it and no others, in items that
    one block takes whole and in items cut between blocks."""
    for mask in ("tree", None):
        t = Tree(dtype, cache, Hq, H, 128, 16, [held, 3], [new, 2], mask, seed=24)
        n = t.rows
        t.v[5, 0, 3], t.v[5, 0, 70], t.v[5, H - 1, 127] = float("inf"), float("nan"), -float("inf")
        t.run(pkg)
        pkg.check_status(0)
        clean = t.v[:n].nan_to_num(0, 0, 0)
        o, _, a = ref.tree(t.q[:n], t.k[:n], clean, t.kc, t.vc, t.table, t.held, t.starts, t.scale, t.mask, t.kd, t.vd)
        got = t.o.cpu().double()[:n]
        for i in range(new):
            if (t.mask is None and i >= 5) or (t.mask is not None and not t.mask[i, 5]):
                for x in range(Hq // H):
                    o[i, x, 3] = float("inf")
                    o[i, x, 70] = float("nan")
                    o[i, (H - 1) * (Hq // H) + x, 127] = -float("inf")
        odd = ~o.isfinite()
        assert torch.equal(got.isnan(), o.isnan()) and torch.equal(got[odd & ~o.isnan()], o[odd & ~o.isnan()])
        u = half_step(dtype)
        tol = u * o.abs() + 1.1 * u * a + 1e-6 * a.amax(-1, keepdim=True)
        assert bool(((got - o).abs() <= tol)[~odd].all())


def test_layouts(pkg):
    """Q, K, V from one fused projection, tokens outside heads in the cache, a padded table and mask."""
    t = Tree(BF16, BF16, 6, 2, 128, 32, [100, 33, 260], [3, 1, 9], "tree", seed=15)
    T = t.q.shape[0]
    qkv = torch.cat([t.q, t.k, t.v], 1).cuda()
    q, k, v = qkv[:, :6], qkv[:, 6:8], qkv[:, 8:]
    kc, vc = (x.transpose(1, 2).contiguous().cuda().transpose(1, 2) for x in (t.kc, t.vc))
    table = torch.full((3, 40), 12345, dtype=torch.int32)
    table[:, :t.table.shape[1]] = t.table
    mask = torch.ones(T, 301, dtype=torch.uint8)
    mask[:, :t.mask.shape[1]] = t.mask
    out = torch.full((T, 10, 128), 7.0, dtype=BF16, device="cuda")
    t.lse = torch.full((T, 6), 7.0, device="cuda")
    pkg.fused_tree(q, k, v, kc, vc, table.cuda()[:, :20], ints(t.held), ints(t.starts), t.scale, mask=mask.cuda()[:, 0:],
                   max_new=9, output=out[:, 2:8], lse=t.lse)
    t.o = out[:, 2:8]
    t.check(pkg)
    assert bool((out[:, :2] == 7).all()) and bool((out[:, 8:] == 7).all())


@pytest.mark.parametrize("Hq,H,new,held", [(8, 2, 1, 9000), (16, 2, 5, 100), (32, 1, 40, 3000), (64, 8, 30, 50)])
def test_output_over_q(pkg, Hq, H, new, held):
    """The result may take q's place, whole items and cut ones, with the same bits."""
    t = Tree(BF16, BF16, Hq, H, 128, 16, [held, 3, 70], [new, 1, new], "tree" if new > 1 else None, tail=0, seed=25).run(pkg)
    q = t.q.cuda()
    pkg.fused_tree(q, t.k.cuda(), t.v.cuda(), t.kc.cuda(), t.vc.cuda(), t.table.cuda(), ints(t.held),
                   ints(t.starts), t.scale, mask=None if t.mask is None else t.mask.cuda(), max_new=t.max_new, output=q)
    assert torch.equal(q.view(torch.int16), t.o.view(torch.int16))
    t.check(pkg)


def test_after_a_refused_plan_nothing_is_written(pkg):
    """starts of 0, as a refused plan leaves them: no row belongs to a request."""
    t = Tree(BF16, BF16, 8, 2, 128, 16, [40, 3], [3, 2], None, seed=26)
    t.starts = [0, 0, 0]
    t.run(pkg)
    pkg.check_status(0)
    assert bool((t.o == 7).all()) and bool((t.lse == 7).all())


def test_descales_per_head(pkg):
    t = Tree(BF16, E4M3, 8, 4, 128, 16, [200, 10], [1, 7], seed=16)
    t.kd, t.vd = torch.tensor([0.5, 1.0, 0.1, 2.0]), torch.tensor([3.0, 0.2, 1.0, 0.6])
    t.run(pkg).check(pkg)
    t = Tree(F16, E4M3, 64, 1, 128, 16, [200, 10], [1, 7], seed=16)
    t.kd, t.vd = torch.tensor([0.5]), torch.tensor([3.0])
    t.run(pkg).check(pkg)


def test_cache_past_32_bits(pkg):
    """Pages whose elements lie past 2^32."""
    H, page, D = 8, 128, 128
    pages = (1 << 32) // (H * page * D) + 8
    t = Tree(BF16, E4M3, 16, H, D, page, [1000], [1], seed=17)
    kc, vc = (torch.empty(pages, H, page, D, dtype=E4M3, device="cuda") for _ in range(2))
    n = t.kc.shape[0]
    kc.view(torch.uint8)[-n:] = t.kc.view(torch.uint8).cuda()
    vc.view(torch.uint8)[-n:] = t.vc.view(torch.uint8).cuda()
    t.lse, t.o = torch.empty(t.q.shape[:2], device="cuda").fill_(7), torch.full(t.q.shape, 7.0, dtype=BF16, device="cuda")
    table = torch.where(t.table >= 0, t.table + pages - n, t.table).cuda()
    pkg.fused_tree(t.q.cuda(), t.k.cuda(), t.v.cuda(), kc, vc, table, ints(t.held), ints(t.starts), t.scale, max_new=1,
                   output=t.o, lse=t.lse, k_descale=t.kd, v_descale=t.vd)
    t.check(pkg)


def test_what_the_device_refuses(pkg):
    """Lengths and starts that cannot be: that request is skipped and recorded, the others are computed."""
    for change in ("length", "page", "new"):
        t = Tree(BF16, BF16, 4, 2, 128, 16, [30, 40, 50], [2, 2, 2], seed=18, tail=0)
        if change == "length":
            t.held[1] = 10000
        elif change == "page":
            t.table[1, 1] = 10 ** 6
        t.run(pkg, max_new=1 if change == "new" else 2)
        with pytest.raises(pkg.AttentionError, match="invalid"):
            pkg.check_status(0)
        if change == "new":
            assert bool((t.o == 7).all())
            continue
        got = t.o.cpu()
        t.held[1], t.table[1] = 40, t.table[2]
        o, _, a = ref.tree(t.q, t.k, t.v, t.kc.nan_to_num(0), t.vc.nan_to_num(0), t.table, t.held, t.starts, t.scale)
        u = half_step(BF16)
        for b in (0, 2):
            s = slice(2 * b, 2 * b + 2)
            assert bool(((got[s].double() - o[s]).abs() <= u * o[s].abs() + 1.1 * u * a[s] + 1e-6 * a[s].max()).all())


def test_calls_repeat_exactly_and_overlap(pkg):
    """Two streams at once, a captured and replayed call beside an eager one: each as a call alone, bit for bit."""
    calls = [Tree(BF16, BF16, 8, 2, 128, 64, [5000, 70], [1, 1], seed=19), Tree(F16, F16, 16, 2, 64, 32, [4000], [48], "tree", seed=20)]
    alone = []
    for t in calls:
        t.run(pkg)
        alone.append((t.o.clone(), t.lse.clone()))
    dev = [[x.cuda() for x in (t.q, t.k, t.v, t.kc, t.vc, t.table)] + [ints(t.held), ints(t.starts)] for t in calls]
    masks = [None if t.mask is None else t.mask.cuda() for t in calls]

    def run(i, **kw):
        lse = torch.full_like(alone[i][1], 7)
        o = torch.full_like(alone[i][0], 7)
        return pkg.fused_tree(*dev[i], calls[i].scale, mask=masks[i], max_new=calls[i].max_new, lse=lse, output=o, **kw), lse

    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run(i)
        graphs.append((g, out))
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, run(i)))
                graphs[1 - i][0].replay()
    torch.cuda.synchronize()
    pkg.check_status(0)
    for i, (o, lse) in got + [(i, graphs[i][1]) for i in range(2)]:
        assert torch.equal(o, alone[i][0]) and torch.equal(lse, alone[i][1])
    s = torch.cuda.Stream()
    o, lse = run(0, stream=s)
    s.synchronize()
    assert torch.equal(o, alone[0][0])


def test_grad_is_refused(pkg):
    t = Tree(BF16, BF16, 2, 1, 64, 16, [5], [1])
    q = t.q.cuda().requires_grad_()
    with pytest.raises(pkg.VerifyError, match="no backward"):
        pkg.fused_tree(q, t.k.cuda(), t.v.cuda(), t.kc.cuda(), t.vc.cuda(), t.table.cuda(), ints(t.held), ints(t.starts), 1.0)


# ------------------------------------------------------------------ a run of them together
@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_serving_loop(pkg, cache):
    """Prompts, decoded tokens, a drafted tree with some accepted, a request that ends: planner, rotary, attention and
    writer in turn, against whole-sequence attention in 64 bits over what each request has seen."""
    g = torch.Generator().manual_seed(21)
    B, Hq, H, D, page, W = 3, 8, 2, 128, 16, 20
    table = pkg.rotary_table(D, [32, 16, 16])
    pages = 40
    kc, vc = (torch.full((pages, H, page, D), float("nan"), device="cuda").to(cache) for _ in range(2))
    kd, vd = (0.05, 0.05) if cache is E4M3 else (1.0, 1.0)
    blocks = torch.full((B, W), -1, dtype=torch.int32, device="cuda")
    free, count, lengths = ints(list(range(pages))), ints([pages]), ints([0] * B)
    past = [[torch.zeros(0, H, D, dtype=torch.float64) for _ in range(2)] for _ in range(B)]

    def stored(x, d):
        return fp8_of(x, d).double() * d if cache is E4M3 else x.double()

    def step(new, parents=None, accept=None):
        nonlocal lengths, count
        T = sum(new)
        starts_list = [sum(new[:b]) for b in range(B + 1)]
        q, k, v = (torch.randn(T, h, D, generator=g).to(BF16).cuda() for h in (Hq, H, H))
        held = lengths.tolist()
        depth, mask = [], None
        if parents is not None:
            mask = torch.ones(T, max(new), dtype=torch.bool)
            for b, n in enumerate(new):
                for i in range(n):
                    p = parents[i]
                    depth.append(held[b] if p < 0 else depth[starts_list[b] + p] + 1)
                    if p >= 0:
                        mask[starts_list[b] + i] = mask[starts_list[b] + p]
                    mask[starts_list[b] + i, i] = False
        else:
            depth = [held[b] + i for b, n in enumerate(new) for i in range(n)]
        pos = ints([depth] * 3)
        q, k = pkg.rotary(q, k, pos, table)
        lse = torch.empty(T, Hq, device="cuda")
        o = pkg.fused_tree(q, k, v, kc, vc, blocks, lengths, ints(starts_list), D ** -0.5,
                           mask=None if mask is None else mask.cuda(), max_new=max(new), lse=lse, k_descale=kd, v_descale=vd)
        # 64-bit attention over what each request has stored and its new tokens
        u = half_step(BF16)
        for b, n in enumerate(new):
            s = slice(starts_list[b], starts_list[b] + n)
            seen = torch.ones(n, n, dtype=torch.bool).tril() if mask is None else ~mask[s, :n]
            seen = torch.cat([torch.ones(n, len(past[b][0]), dtype=torch.bool), seen], 1)
            for h in range(Hq):
                kk = torch.cat([past[b][0][:, h // (Hq // H)], k[s, h // (Hq // H)].cpu().double()])
                vv = torch.cat([past[b][1][:, h // (Hq // H)], v[s, h // (Hq // H)].cpu().double()])
                p = torch.softmax((q[s, h].cpu().double() @ kk.T * D ** -0.5).masked_fill(~seen, -math.inf), 1)
                want, a = p @ vv, p @ vv.abs()
                tol = u * want.abs() + 1.1 * u * a + 1e-6 * a.max() if n else a
                assert bool(((o[s, h].cpu().double() - want).abs() <= tol).all())
        take = [list(range(n)) for n in new] if accept is None else [accept[:n] for n in new]
        rows = [starts_list[b] + i for b in range(B) for i in take[b]]
        targets = ints([held[b] + len(take[b]) for b in range(B)])
        plan = pkg.cache_plan(lengths, targets, blocks, free, count, page, T)
        padded = ints(rows + [0] * (T - len(rows)))
        pkg.cache_append(k, v, kc, vc, plan.slots, rows=padded, k_descale=kd, v_descale=vd)
        pkg.check_status(0)
        lengths, count = plan.lengths, plan.free_count
        assert plan.positions.tolist()[:len(rows)] == [held[b] + i for b in range(B) for i in range(len(take[b]))]
        for b in range(B):
            pick = [starts_list[b] + i for i in take[b]]
            past[b][0] = torch.cat([past[b][0], stored(k[pick].cpu(), kd)])
            past[b][1] = torch.cat([past[b][1], stored(v[pick].cpu(), vd)])

    step([37, 5, 90])
    for _ in range(3):
        step([1, 1, 1])
    step([6, 6, 6], parents=[-1, 0, 0, 1, 2, 3], accept=[0, 1, 3, 5])
    step([1, 1, 1])
    # request 1 ends, and a new prompt takes its place and its pages
    ended = lengths.clone()
    ended[1] = 0
    plan = pkg.cache_plan(lengths, ended, blocks, free, count, page, 0, lengths_out=lengths, free_count_out=count)
    assert count.tolist() == [pages - sum(-(-n // page) for n in lengths.tolist())] and plan.starts.tolist() == [0] * 4
    past[1] = [x[:0] for x in past[1]]
    step([1, 50, 1])
    step([3, 3, 3], parents=[-1, 0, 0], accept=[0, 2])
