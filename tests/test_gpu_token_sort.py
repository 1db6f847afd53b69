"""Pairs sorted by expert, tokens gathered and rows combined on the GPU, against
plain arithmetic in 64 bits.

Tolerances: a sum of n fp32 products in order is off by n 2^-24 of the sum of
their magnitudes, the result rounds once by half a step of its type."""
import math

import pytest
import torch

from ftmoe.engine import MoeGraphRunner
from ftmoe.moe.token_sort import TokenSort, combine_tokens, gather_tokens, sort_tokens

pytestmark = pytest.mark.gpu
DTYPES = (torch.bfloat16, torch.float16, torch.float32)
U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def routing(T, k, E, seed, lo=0, hi=None, dtype=torch.int32):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(lo, E if hi is None else hi, (T, k), generator=g).to(dtype)


def exact_sort(ids, E):
    ids = ids.cpu().reshape(-1).long()
    T_k = ids.numel()
    key = torch.where((ids < 0) | (ids >= E), E, ids)
    order = torch.sort(key, stable=True).indices
    offsets = torch.searchsorted(key[order].contiguous(), torch.arange(E + 1))
    row = torch.empty(T_k, dtype=torch.long)
    row[order] = torch.arange(T_k)
    n = int(offsets[E])
    here = key < E
    used = torch.arange(T_k) < n
    return offsets, torch.where(here, row, ~row), torch.where(used, order, ~order), used


def check_sort(sort, ids, E):
    T, k = ids.shape
    off, row, pair, used = exact_sort(ids, E)
    assert torch.equal(sort.offsets.cpu().long(), off)
    assert torch.equal(sort.row_of_pair.cpu().long(), row.reshape(T, k))
    assert torch.equal(sort.pair_of_row.cpu().long(), pair)
    assert torch.equal(sort.token_of_row.cpu().long(), torch.where(used, pair // k, -1))


@pytest.mark.parametrize("T,k,E", [(1, 1, 1), (1, 8, 256), (3, 2, 5), (16, 8, 256), (63, 1, 7), (64, 1, 512), (65, 3, 512),
                                   (1023, 8, 64), (1024, 8, 128), (1025, 8, 511), (2048, 8, 128), (4096, 8, 256),
                                   (9000, 6, 512), (100000, 8, 60), (70000, 16, 512)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_sort(gpu, T, k, E, dtype):
    ids = routing(T, k, E, T + k, dtype=dtype)
    check_sort(sort_tokens(ids.to(gpu), E), ids, E)


@pytest.mark.parametrize("T,k,E", [(5, 2, 4), (700, 8, 32), (3000, 4, 100)])
def test_sort_ids_without_an_expert(gpu, T, k, E):
    """Negative ids and ids past the experts, in 64 bits too; every pair without one; one
    expert for all; the same expert twice for a token."""
    ids = routing(T, k, E, 1, lo=-E, hi=2 * E)
    check_sort(sort_tokens(ids.to(gpu), E), ids, E)
    wide = ids.long()
    wide[::3, 0] = 2 ** 40 + 1
    wide[1::3, 0] = -(2 ** 40)
    check_sort(sort_tokens(wide.to(gpu), E), wide, E)
    for v in (-1, 0, E - 1, E):
        same = torch.full((T, k), v, dtype=torch.int32)
        check_sort(sort_tokens(same.to(gpu), E), same, E)


def test_sort_layouts_and_refusals(gpu):
    ids = routing(40, 6, 9, 2).to(gpu)
    for v in (ids.t().contiguous().t(), ids[:, ::2], ids[::3]):
        check_sort(sort_tokens(v, 9), v, 9)
    empty = sort_tokens(ids[:0], 9)
    assert not empty.offsets.any() and empty.row_of_pair.shape == (0, 6) and empty.pair_of_row.shape == (0,)
    for err, a in ((TypeError, (ids.float(), 9)), (TypeError, (ids.to(torch.int16), 9)), (ValueError, (ids[0], 9)),
                   (ValueError, (ids, 0)), (ValueError, (ids, 513)), (ValueError, (ids[:, :0], 9))):
        with pytest.raises(err):
            sort_tokens(*a)


# ------------------------------------------------------------------ rows out of tokens
@pytest.mark.parametrize("dtype", [*DTYPES, torch.int8, torch.int32])
@pytest.mark.parametrize("T,k,E,H", [(1, 1, 1, 1), (5, 3, 8, 64), (33, 8, 16, 2880), (700, 4, 64, 33), (17, 2, 8, 5000)])
def test_gather(gpu, dtype, T, k, E, H):
    ids = routing(T, k, E, 3, lo=-1).to(gpu)
    x = torch.randint(-100, 100, (T, H), generator=torch.Generator().manual_seed(4)).to(gpu).to(dtype)
    sort = sort_tokens(ids, E)
    got = gather_tokens(x, sort)
    t = sort.token_of_row.long()
    ref = torch.where((t >= 0)[:, None], x[t.clamp_min(0)], torch.zeros_like(x[:1]))
    assert got.dtype == dtype and torch.equal(got, ref)


def test_gather_strides_and_refusals(gpu):
    sort = sort_tokens(routing(20, 3, 8, 5).to(gpu), 8)
    big = torch.randn(40, 300, device=gpu).to(torch.bfloat16)
    t = sort.token_of_row.long()
    for x in (big[:20, 16:144], big[::2, 3:50], big[:20].t().contiguous().t(), big[:1, :64].expand(20, 64), big[:20, :1]):
        assert torch.equal(gather_tokens(x, sort), x[t])
    x = big[:20, :64]
    for err, a in ((ValueError, big[:19]), (ValueError, big[0]), (TypeError, x.double()),
                   (TypeError, x.to(torch.complex64))):
        with pytest.raises(err):
            gather_tokens(a, sort)
    bad = TokenSort(8, sort.offsets, sort.row_of_pair.long(), sort.pair_of_row, sort.token_of_row)
    with pytest.raises(ValueError):
        gather_tokens(x, bad)
    assert gather_tokens(x[:, :0], sort).shape == (60, 0)


# ------------------------------------------------------------------ rows back into tokens
def exact_combine(rows, w, sort):
    """(sum, sum of magnitudes) in 64 bits, from the definition."""
    r = sort.row_of_pair.long()
    v = torch.where((r >= 0)[..., None], rows.double()[r.clamp_min(0)], torch.zeros((), dtype=torch.float64, device=rows.device))
    if w is not None:
        v = v * w.double()[..., None]
    return v.sum(dim=1), v.abs().sum(dim=1)


def within(got, ref, mag, n, dtype):
    assert got.dtype == dtype and got.shape == ref.shape
    err = (got.double() - ref).abs()
    bound = n * U * mag * (1 + half_step(dtype)) + half_step(dtype) * ref.abs() + tiny(dtype)
    assert (err <= bound).all(), float((err - bound).max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,E,H", [(1, 1, 1, 8), (5, 3, 8, 64), (33, 8, 16, 2880), (700, 4, 64, 33), (17, 9, 20, 2056),
                                     (40, 17, 32, 128)])
@pytest.mark.parametrize("wdt", [None, *DTYPES])
def test_combine(gpu, dtype, T, k, E, H, wdt):
    g = torch.Generator(device=gpu).manual_seed(6)
    sort = sort_tokens(routing(T, k, E, 7, lo=-1).to(gpu), E)
    rows = torch.randn(T * k, H, generator=g, device=gpu).to(dtype)
    w = None if wdt is None else torch.rand(T, k, generator=g, device=gpu).to(wdt)
    ref, mag = exact_combine(rows, w, sort)
    within(combine_tokens(rows, w, sort), ref, mag, k, dtype)
    if dtype == torch.float32:
        for od in DTYPES:
            within(combine_tokens(rows, w, sort, out_dtype=od), ref, mag, k, od)


def test_combine_reads_no_row_without_an_expert(gpu):
    """NaN and infinities in the rows of no expert (and in their weights) stay there; a token
    without any expert becomes zeros."""
    T, k, E, H = 30, 4, 8, 96
    ids = routing(T, k, E, 8)
    ids[::2, 1] = -1
    ids[5] = -1
    sort = sort_tokens(ids.to(gpu), E)
    rows = torch.randn(T * k, H, device=gpu)
    w = torch.rand(T, k, device=gpu)
    ref = combine_tokens(rows, w, sort)
    n = int(sort.offsets[-1])
    rows[n:], rows[n + 1:] = math.nan, math.inf
    w[ids.to(gpu) < 0] = math.nan
    got = combine_tokens(rows, w, sort)
    assert torch.equal(got, ref) and not got[5].any()
    rows[int(sort.row_of_pair[7, 0])] = math.inf  # a row of an expert does count
    assert torch.isinf(combine_tokens(rows, w, sort)[7]).all()


def test_combine_strides_and_refusals(gpu):
    T, k, H = 20, 3, 64
    sort = sort_tokens(routing(T, k, 8, 9).to(gpu), 8)
    big = torch.randn(T * k, 3 * H, device=gpu).to(torch.bfloat16)
    w = torch.rand(k, T, device=gpu).t()
    for rows in (big[:, H:2 * H], big[:, 5:40], big.t().contiguous().t(), big[:1, :H].expand(T * k, H)):
        assert torch.equal(combine_tokens(rows, w, sort), combine_tokens(rows.contiguous(), w.contiguous(), sort))
    rows = big[:, :H]
    assert combine_tokens(rows[:, :0], w, sort).shape == (T, 0)
    for err, a, kw in ((ValueError, (rows[:-1], w, sort), {}), (ValueError, (rows, w[:-1], sort), {}),
                       (TypeError, (rows.double(), w, sort), {}), (TypeError, (rows, w.double(), sort), {}),
                       (TypeError, (rows, w, sort), dict(out_dtype=torch.float32)),
                       (TypeError, (rows.float(), w, sort), dict(out_dtype=torch.float64)),
                       (RuntimeError, (rows, w.cpu(), sort), {})):
        with pytest.raises(err):
            combine_tokens(*a, **kw)


# ------------------------------------------------------------------ gradients
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,E,H", [(1, 1, 1, 8), (9, 3, 8, 64), (50, 8, 16, 2880), (300, 4, 64, 33), (17, 9, 20, 2056)])
def test_gather_gradient(gpu, dtype, T, k, E, H):
    sort = sort_tokens(routing(T, k, E, 10, lo=-1).to(gpu), E)
    x = torch.randn(T, H, device=gpu).to(dtype).requires_grad_()
    g = torch.randn(T * k, H, device=gpu).to(dtype)
    gather_tokens(x, sort).backward(g)
    ref, mag = exact_combine(g, None, sort)
    within(x.grad, ref, mag, k, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,E,H", [(1, 1, 1, 8), (9, 3, 8, 64), (50, 8, 16, 2880), (300, 4, 64, 33), (17, 9, 20, 2056),
                                     (5, 17, 32, 128)])
@pytest.mark.parametrize("wdt", DTYPES)
def test_combine_gradient(gpu, dtype, T, k, E, H, wdt):
    """grad_rows = w g is one product, rounded once more to a 16-bit type; grad_w is a sum of
    H products (in any order)."""
    gen = torch.Generator(device=gpu).manual_seed(11)
    sort = sort_tokens(routing(T, k, E, 12, lo=-1).to(gpu), E)
    for od in (DTYPES if dtype == torch.float32 else (dtype,)):
        rows = torch.randn(T * k, H, generator=gen, device=gpu).to(dtype).requires_grad_()
        w = torch.rand(T, k, generator=gen, device=gpu).to(wdt).requires_grad_()
        g = torch.randn(T, H, generator=gen, device=gpu).to(od)
        gr, gw = torch.autograd.grad(combine_tokens(rows, w, sort, out_dtype=od), (rows, w), g)
        r = sort.row_of_pair.long()
        here = r >= 0
        ref = torch.zeros(T * k, H, dtype=torch.float64, device=gpu)
        ref[r[here]] = (w.detach().double()[..., None] * g.double()[:, None])[here]
        within(gr, ref, ref.abs(), 1, dtype)
        prod = torch.where(here[..., None], rows.detach().double()[r.clamp_min(0)] * g.double()[:, None], 0.0)
        within(gw, prod.sum(dim=2), prod.abs().sum(dim=2), H, wdt)
        assert not gw[~here].any()


def test_combine_gradient_by_differences(gpu):
    """The sum is linear in rows and in weights: over a step of either the scalar <g, out>
    moves by <gradient, step>, up to the fp32 rounding of both outputs."""
    T, k, E, H = 40, 4, 16, 96
    gen = torch.Generator(device=gpu).manual_seed(13)
    sort = sort_tokens(routing(T, k, E, 14, lo=-1).to(gpu), E)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=gpu)  # noqa: E731
    rows, w, g = rnd(T * k, H).requires_grad_(), rnd(T, k).requires_grad_(), rnd(T, H)
    gr, gw = torch.autograd.grad(combine_tokens(rows, w, sort), (rows, w), g)

    def f(r, v):
        return (combine_tokens(r, v, sort).double() * g.double()).sum()

    dr, dw = rnd(T * k, H), rnd(T, k)
    with torch.no_grad():
        base = f(rows, w)
        # every |term| sums to less than T k H 5^3; each of the two outputs and the gradient
        # is off by less than (k + 1) 2^-24 of that
        tol = 3 * (k + 1) * U * T * k * H * 125
        assert abs((f(rows + dr, w) - base) - (gr.double() * dr.double()).sum()) < tol
        assert abs((f(rows, w + dw) - base) - (gw.double() * dw.double()).sum()) < tol
        x = rnd(T, H)
    xg = x.requires_grad_()
    gg = rnd(T * k, H)
    (gx,) = torch.autograd.grad(gather_tokens(xg, sort), xg, gg)
    dx = rnd(T, H)
    with torch.no_grad():
        d = ((gather_tokens(x + dx, sort).double() - gather_tokens(x, sort).double()) * gg.double()).sum()
        assert abs(d - (gx.double() * dx.double()).sum()) < tol


@pytest.mark.parametrize("needs", [(True, False), (False, True)])
def test_combine_gradient_of_one_input(gpu, needs):
    T, k, H = 12, 3, 40
    sort = sort_tokens(routing(T, k, 6, 15).to(gpu), 6)
    rows, w = torch.randn(T * k, H, device=gpu), torch.rand(T, k, device=gpu)
    both = torch.autograd.grad(combine_tokens(rows.requires_grad_(), w.requires_grad_(), sort).sum(), (rows, w))
    rows, w = rows.detach().requires_grad_(needs[0]), w.detach().requires_grad_(needs[1])
    one = torch.autograd.grad(combine_tokens(rows, w, sort).sum(), rows if needs[0] else w)[0]
    assert torch.equal(one, both[0] if needs[0] else both[1])
    ones = combine_tokens(rows.detach().requires_grad_(), None, sort)
    assert torch.equal(torch.autograd.grad(ones.sum(), ones.grad_fn.next_functions[0][0].variable)[0],
                       torch.ones_like(rows))


def test_gradients_of_broadcast_outputs(gpu):
    """An expanded upstream gradient (of a sum) and one that is transposed."""
    T, k, H = 14, 3, 64
    sort = sort_tokens(routing(T, k, 6, 16, lo=-1).to(gpu), 6)
    x = torch.randn(T, H, device=gpu, requires_grad=True)
    gather_tokens(x, sort).sum().backward()
    assert torch.equal(x.grad, (sort.row_of_pair >= 0).sum(dim=1, keepdim=True).float().expand(T, H))
    rows, w = torch.randn(T * k, H, device=gpu, requires_grad=True), torch.rand(T, k, device=gpu, requires_grad=True)
    g = torch.randn(H, T, device=gpu).t()
    a = torch.autograd.grad(combine_tokens(rows, w, sort), (rows, w), g)
    b = torch.autograd.grad(combine_tokens(rows, w, sort), (rows, w), g.contiguous())
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    with pytest.raises(RuntimeError):  # no second derivative
        (gx,) = torch.autograd.grad(gather_tokens(x, sort).pow(2).sum(), x, create_graph=True)
        gx.sum().backward()


def test_rows_past_32_bits(gpu):
    """More than 2^32 bytes of rows, tokens and gradients: the last tokens against the same alone."""
    T, k, H, E = 300000, 2, 8192, 9
    ids = torch.arange(T * k, device=gpu).reshape(T, k) % E
    sort = sort_tokens(ids, E)
    x = torch.zeros(T, H, device=gpu, dtype=torch.bfloat16)
    x[-9:] = torch.randn(9, H, generator=torch.Generator(device=gpu).manual_seed(4), device=gpu).to(torch.bfloat16)
    rows = gather_tokens(x, sort)
    at = sort.row_of_pair[-9:].reshape(-1).long()
    assert torch.equal(rows[at], x[-9:].repeat_interleave(k, 0))
    w = torch.rand(T, k, device=gpu)
    small = sort_tokens(ids[-9:], E)
    sr, sw = gather_tokens(x[-9:], small).requires_grad_(), w[-9:].clone().requires_grad_()
    ref = combine_tokens(sr, sw, small)
    rows.requires_grad_(), w.requires_grad_()
    out = combine_tokens(rows, w, sort)
    assert torch.equal(out[-9:], ref)
    gr, gw = torch.autograd.grad(out, (rows, w), x)
    sgr, sgw = torch.autograd.grad(ref, (sr, sw), x[-9:])
    assert torch.equal(gw[-9:], sgw) and torch.equal(gr[at], sgr[small.row_of_pair.reshape(-1).long()])


def test_more_tokens_than_one_grid_dimension(gpu):
    """2^24 tokens and more, a workgroup each."""
    T, H, E = 2**24 + 70, 8, 4
    ids = (torch.arange(T, device=gpu)[:, None] * 7 // 3) % E
    sort = sort_tokens(ids, E)
    x = torch.randn(T, H, generator=torch.Generator(device=gpu).manual_seed(6), device=gpu).to(torch.bfloat16)
    rows = gather_tokens(x, sort)
    assert torch.equal(rows, x[sort.token_of_row.long()])
    w = torch.rand(T, 1, device=gpu)
    rows.requires_grad_(), w.requires_grad_()
    out = combine_tokens(rows, w, sort)
    assert torch.equal(out.detach(), (x.float() * w.detach()).to(torch.bfloat16))
    gr, gw = torch.autograd.grad(out, (rows, w), x)
    assert torch.equal(gr, (x.float() * w.detach()).to(torch.bfloat16)[sort.token_of_row.long()])
    ref = x.double().pow(2).sum(1, keepdim=True)
    assert ((gw.double() - ref).abs() <= 9 * U * ref).all()


def test_gradient_after_the_order_changed(gpu):
    """A write to the order between forward and backward is refused, not used."""
    sort = sort_tokens(routing(8, 2, 4, 3).to(gpu), 4)
    x = torch.randn(8, 16, device=gpu, requires_grad=True)
    rows = gather_tokens(x, sort)
    out = combine_tokens(rows, torch.rand(8, 2, device=gpu), sort)
    sort.row_of_pair.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


# ------------------------------------------------------------------ together
def test_training_step(gpu):
    """Tokens out, a dense expert each, rows back: values and gradients of tokens, router
    weights and experts against autograd over the same definition in 64 bits."""
    T, k, E, H = 60, 2, 4, 48
    gen = torch.Generator(device=gpu).manual_seed(17)
    ids = routing(T, k, E, 18, lo=-1).to(gpu)
    sort = sort_tokens(ids, E)
    x0 = torch.randn(T, H, generator=gen, device=gpu)
    w0 = torch.rand(T, k, generator=gen, device=gpu)
    m0 = torch.randn(E, H, H, generator=gen, device=gpu) / math.sqrt(H)
    ends = sort.offsets.tolist()

    x, w, m = (v.clone().requires_grad_() for v in (x0, w0, m0))
    rows = gather_tokens(x, sort)
    y = torch.cat([rows[ends[e]:ends[e + 1]] @ m[e] for e in range(E)] + [rows[ends[E]:]])
    out = combine_tokens(y, w, sort)
    out.pow(2).sum().backward()

    xd, wd, md = (v.double().requires_grad_() for v in (x0, w0, m0))
    ref = torch.zeros(T, H, dtype=torch.float64, device=gpu)
    for e in range(E):
        t, j = (ids == e).nonzero(as_tuple=True)
        ref = ref.index_add(0, t, (xd[t] @ md[e]) * wd[t, j][:, None])
    ref.pow(2).sum().backward()
    # sums of at most 4 H = 192 products, each of at most three such sums: 3 * 192 * 2^-24 of the largest magnitudes
    for got, want in ((out, ref), (x.grad, xd.grad), (w.grad, wd.grad), (m.grad, md.grad)):
        assert ((got.double() - want).norm() / want.norm()).item() <= 3 * 4 * H * U


def test_same_bits_every_time_and_on_streams(gpu):
    T, k, E, H = 3000, 8, 64, 128
    ids = routing(T, k, E, 19, lo=-1).to(gpu)
    x = torch.randn(T, H, device=gpu).to(torch.bfloat16)
    w = torch.rand(T, k, device=gpu)

    def step():
        sort = sort_tokens(ids, E)
        rows = gather_tokens(x, sort)
        return sort.row_of_pair, rows, combine_tokens(rows, w, sort)

    ref = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=gpu) for _ in range(2)]
    got = []
    for s in streams * 3:
        with torch.cuda.stream(s):
            got.append(step())
    torch.cuda.synchronize()
    for o in got:
        assert all(torch.equal(a, b) for a, b in zip(o, ref))


def test_forward_and_backward_in_a_graph(gpu):
    """A step with its gradients captured (its leaves made in it) and replayed over new
    inputs, eager steps over the same buffers in between."""
    T, k, E, H = 1500, 8, 32, 64
    ids = routing(T, k, E, 20).to(gpu)
    x, w, g = torch.randn(T, H, device=gpu), torch.rand(T, k, device=gpu), torch.randn(T, H, device=gpu)

    def step():
        xl, wl = x.detach().requires_grad_(), w.detach().requires_grad_()
        sort = sort_tokens(ids, E)
        out = combine_tokens(gather_tokens(xl, sort), wl, sort)
        return (out.detach(), *torch.autograd.grad(out, (xl, wl), g))

    eager = step()  # its graph is gone; a captured one must not depend on it
    run = MoeGraphRunner()
    captured = run.capture(step)
    for seed in range(3):
        ids.copy_(routing(T, k, E, 21 + seed, lo=-1))
        x.normal_(), w.uniform_(), g.normal_()
        run.replay()
        torch.cuda.synchronize()
        eager = step()
        assert all(torch.equal(a, b) for a, b in zip(captured, eager)), seed


# ------------------------------------------------------------------ many pairs
@pytest.mark.parametrize("T,k,E", [(131072 + 9, 8, 60), (300000, 8, 1), (300000, 7, 511), (2**20 + 5, 8, 512)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_sort_of_many_workgroups(gpu, T, k, E, dtype):
    """More workgroups than read one another's counts."""
    ids = routing(T, k, E, T + k, lo=-1, dtype=dtype)
    check_sort(sort_tokens(ids.to(gpu), E), ids, E)


def test_sort_time_is_proportional_to_the_pairs(gpu):
    """Eight times the pairs of 4 M take about eight times as long (a cost for every two
    workgroups would take 64 times): 24 leaves room for what the smaller one's caches gain."""
    E, times = 64, []
    for T in (2**19, 2**22):
        ids = torch.arange(T * 8, device=gpu, dtype=torch.int32).reshape(T, 8).remainder_(E)
        sort_tokens(ids, E)
        best = math.inf
        for _ in range(5):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            torch.cuda.synchronize()
            start.record()
            sort_tokens(ids, E)
            end.record()
            torch.cuda.synchronize()
            best = min(best, start.elapsed_time(end))
        times.append(best)
    assert times[1] < 24 * times[0], times
