"""GPU: queries, keys and values that are infinite or no numbers in the attention over a paged cache, against the
definition in 64 bits.  A row that sees no key gives 0 and a log-sum-exp of -inf; any other row is what its softmax is,
also where that is no number.  Tolerances of the other rows: those of test_gpu_serving.py."""
import math

import pytest

torch = pytest.importorskip("torch")

from test_gpu_serving import BF16, E4M3, F16, TYPES, Tree, half_step

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


def definition(t):
    """(O, LSE, A) of a Tree's rows in 64 bits, A = sum p |v|."""
    T, Hq, D = t.rows, *t.q.shape[1:]
    H, page = t.kc.shape[1:3]
    o, a = torch.zeros(T, Hq, D, dtype=torch.float64), torch.zeros(T, Hq, D, dtype=torch.float64)
    lse = torch.full((T, Hq), -INF, dtype=torch.float64)
    for b, n in enumerate(t.held):
        rows = slice(t.starts[b], t.starts[b + 1])
        m = rows.stop - rows.start
        ids = t.table[b, :-(-n // page)].long()
        seen = torch.ones(m, m, dtype=torch.bool).tril() if t.mask is None else ~t.mask[rows, :m]
        seen = torch.cat([torch.ones(m, n, dtype=torch.bool), seen], 1)
        some = seen.any(1)
        for x in range(Hq):
            h = x // (Hq // H)
            k = torch.cat([t.kc[ids, h].double().flatten(0, 1)[:n] * t.kd, t.k[rows, h].double()])
            v = torch.cat([t.vc[ids, h].double().flatten(0, 1)[:n] * t.vd, t.v[rows, h].double()])
            s = (t.q[rows, x].double() @ k.T * t.scale).masked_fill(~seen, -INF)
            p = torch.where(some[:, None], torch.softmax(s, 1), 0.0)
            o[rows, x], a[rows, x] = p @ v, p @ v.abs()
            lse[rows, x] = torch.logsumexp(s, 1)
    return o, lse, a


def check(pkg, t):
    pkg.check_status(0)
    o, lse, a = definition(t)
    got, glse, u = t.o.cpu().double()[:t.rows], t.lse.cpu().double()[:t.rows], half_step(t.q.dtype)
    assert torch.equal(got.isnan(), o.isnan()) and torch.equal(glse.isnan(), lse.isnan())
    assert torch.equal(glse == -INF, lse == -INF)
    fine = o.isfinite().all(-1)
    tol = u * o.abs() + 1.1 * u * a + 1e-6 * a.amax(-1, keepdim=True)
    assert bool(((got - o).abs() <= tol)[fine].all())
    fine = lse.isfinite()
    assert bool(((glse - lse).abs() <= (max(t.held) + t.max_new) * 2.0 ** -24 + 2.0 ** -17)[fine].all())
    return o, lse


# Items that one block takes whole and items cut between blocks, of one 16-row tile, two, three and a tcgen05 tile.
SHAPES = [(8, 2, 64, [9000], [1], None), (8, 2, 128, [9000, 30], [1, 1], None), (8, 8, 128, [50] * 80, [1] * 80, None),
          (32, 2, 128, [5000, 0], [2, 2], "tree"), (4, 4, 64, [200] * 37, [44] * 37, "tree"),
          (4, 4, 64, [6000], [45], None), (32, 1, 128, [3000], [40], "tree"), (32, 1, 64, [3000, 7], [40, 3], None),
          (32, 8, 128, [20] * 40, [30] * 40, "tree"), (8, 1, 64, [0, 500], [100, 70], None)]


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("Hq,H,D,held,new,mask", SHAPES)
def test_a_query_that_is_no_number(pkg, dtype, cache, Hq, H, D, held, new, mask):
    """One NaN in q: O and LSE of that row and head are no numbers, all others as ever."""
    t = Tree(dtype, cache, Hq, H, 128 if cache is E4M3 else D, 16, held, new, mask, seed=41)
    t.q[0, Hq - 1, 5] = NAN
    t.q[t.rows - 1, 0, 0] = NAN
    o, lse = check(pkg, t.run(pkg))
    assert int(lse.isnan().sum()) == 2 and int(o.isnan().all(-1).sum()) == 2


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("Hq,H,D,held,new,mask", [SHAPES[0], SHAPES[3], SHAPES[5], SHAPES[6], SHAPES[7]])
def test_keys_that_are_no_numbers(pkg, dtype, cache, Hq, H, D, held, new, mask):
    """One cached key, then a run of them long enough to be a block's whole piece: all rows that share the head."""
    for first, last in ((77, 78), (1000, 2900)):
        t = Tree(dtype, cache, Hq, H, 128 if cache is E4M3 else D, 16, held, new, mask, seed=42)
        for i in range(first, last):
            t.kc.view(torch.uint8 if cache is E4M3 else cache)[t.table[0, i // 16], 0, i % 16, 3] = \
                0x7f if cache is E4M3 else NAN
        o, lse = check(pkg, t.run(pkg))
        assert bool(lse[:new[0], :Hq // H].isnan().all()) and bool(lse[:, Hq // H:].isfinite().all())


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("Hq,H,D,held,new,mask", SHAPES)
def test_scores_that_are_all_minus_infinity(pkg, dtype, cache, Hq, H, D, held, new, mask):
    """0 / 0, not the 0 of a row that sees nothing."""
    t = Tree(dtype, cache, Hq, H, 128 if cache is E4M3 else D, 16, held, new, mask, seed=43)
    for x in (t.kc, t.k):
        if x.dtype is E4M3:
            x.view(torch.uint8)[..., 0] = 0x38  # 1
        else:
            x[..., 0] = 1.0
    t.q[0, Hq - 1, 0] = -INF
    o, lse = check(pkg, t.run(pkg))
    assert bool(o[0, Hq - 1].isnan().all()) and float(lse[0, Hq - 1]) == -INF


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("Hq,H,D,new", [(4, 2, 128, 6), (16, 2, 64, 6), (32, 1, 128, 40)])
def test_rows_that_see_nothing_beside_scores_of_minus_infinity(pkg, dtype, Hq, H, D, new):
    """Without cached keys: a row whose mask leaves nothing, one that sees keys of score -inf, one of both kinds."""
    t = Tree(dtype, dtype, Hq, H, D, 16, [0, 0], [new, 1], "tree", seed=44)
    t.k[..., 0] = 1.0
    t.q[:3, :, 0] = -INF
    t.mask[0] = True            # nothing
    t.mask[1, :2], t.mask[1, 2:] = False, True
    t.mask[2] = True
    t.mask[2, new - 1] = False  # the last new token alone
    t.mask[3] = True            # nothing, with finite scores
    o, lse = check(pkg, t.run(pkg))
    assert not o[0].any() and not o[3].any() and bool(o[1:3].isnan().all())
    assert bool((lse[:4] == -math.inf).all())


def values_definition(t):
    """O where new values are no numbers: the sum over the finite ones, and by each row and column what the others that
    the row sees make of it (weights are above 0)."""
    n = t.rows
    fine, t.v = t.v, t.v.clone()
    t.v[:n] = t.v[:n].nan_to_num(0, 0, 0)
    o, _, a = definition(t)
    t.v = fine
    Hq, H = t.q.shape[1], t.v.shape[1]
    for b in range(len(t.held)):
        rows = slice(t.starts[b], t.starts[b + 1])
        m = rows.stop - rows.start
        seen = torch.ones(m, m, dtype=torch.bool).tril() if t.mask is None else ~t.mask[rows, :m]
        v = t.v[rows].double()
        odd = torch.where(v.isfinite(), 0.0, v)
        for h in range(H):
            hit = [seen.double() @ kind.double() > 0 for kind in (odd[:, h] == INF, odd[:, h] == -INF, odd[:, h].isnan())]
            add = hit[0].double().masked_fill(hit[0], INF) + hit[1].double().masked_fill(hit[1], -INF) + \
                hit[2].double().masked_fill(hit[2], NAN)
            o[rows, h * (Hq // H):(h + 1) * (Hq // H)] += add[:, None]
    return o, a


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("mask", [None, "tree", "random"])
@pytest.mark.parametrize("Hq,H,D,held,new", [(8, 2, 128, [40, 0, 300], [300, 1, 129]), (4, 4, 64, [9000, 5], [7, 160]),
                                             (5, 1, 128, [0] * 200, [3] * 200)])
def test_many_values_that_are_no_numbers(pkg, dtype, cache, mask, Hq, H, D, held, new):
    """Infinities of both signs and NaN in many rows: whole columns, a few a column, both signs in one column."""
    t = Tree(dtype, cache, Hq, H, 128 if cache is E4M3 else D, 16, held, new, mask, seed=45)
    g, n = torch.Generator().manual_seed(46), t.rows
    t.v[:n, :, 0], t.v[:n, 0, 1], t.v[:n, H - 1, 2] = NAN, INF, -INF
    pick = torch.rand(n, H, generator=g)
    t.v[:n, :, 3] = torch.where(pick < 0.01, INF, torch.where(pick > 0.99, -INF, 1.0)).to(dtype)
    t.v[:n, :, 4] = torch.where(pick < 0.3, INF, torch.where(pick > 0.98, NAN, 1.0)).to(dtype)
    t.v[n - 1, 0, 5], t.v[0, H - 1, 6] = -INF, INF
    t.run(pkg)
    pkg.check_status(0)
    o, a = values_definition(t)
    got, u = t.o.cpu().double()[:n], half_step(dtype)
    fine = o.isfinite()
    assert torch.equal(got.isnan(), o.isnan()) and torch.equal(got[~fine & ~o.isnan()], o[~fine & ~o.isnan()])
    tol = u * o.abs() + 1.1 * u * a + 1e-6 * a.amax(-1, keepdim=True)
    assert bool(((got - o).abs() <= tol)[fine].all())


@pytest.mark.parametrize("mask", [False, True])
@pytest.mark.parametrize("what", [NAN, INF])
def test_a_chunk_of_values_that_are_no_numbers_takes_no_longer(pkg, mask, what):
    """All values of a chunk of 2048 tokens: milliseconds (an update for every pair of a row and a key it sees, one
    after another, would take seconds)."""
    T, Hq, H, D = 2048, 32, 8, 128
    q, k = (torch.randn(T, h, D, device="cuda").to(BF16) for h in (Hq, H))
    v = torch.full((T, H, D), what, device="cuda").to(BF16)
    cache = torch.zeros(1, H, 16, D, dtype=BF16, device="cuda")
    args = (q, k, v, cache, cache, torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
            torch.zeros(1, dtype=torch.int32, device="cuda"), torch.tensor([0, T], dtype=torch.int32, device="cuda"), 0.1)
    hide = torch.ones(T, T, dtype=torch.bool, device="cuda").triu(1) if mask else None
    pkg.fused_tree(*args, mask=hide)
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    o = pkg.fused_tree(*args, mask=hide)
    end.record()
    end.synchronize()
    pkg.check_status(0)
    assert bool(o.isnan().all() if what != what else (o == INF).all())
    assert begin.elapsed_time(end) < 100
