"""Every kernel of the long-context attention, with its positions whole and split: which one a call gets goes by its expected time, and the
shapes of small tests would leave some of them out. The contexts here name the kernel; the cases and their bounds are those of
test_attention_long.py."""
import contextlib
import os

import pytest

import test_attention_long as T

torch = T.torch
pytestmark = pytest.mark.gpu

# kind of cache, kernel, splits (r: joined through records, in the kernel for few rows; without it by a cluster)
KERNELS = [("f32", "few", "1"), ("f32", "few", "3"), ("f32", "tiles", "1"), ("f32", "tiles", "3")] + [
    (kind, *which) for kind in ("f16", "q4") for which in (("few", "1"), ("few", "3"), ("few", "3r"), ("tiles", "1"), ("tiles", "3"))]


@contextlib.contextmanager
def context(kernel, splits):
    """A context on the current stream whose attention runs in the named kernel."""
    from rllama_b200 import Cuda
    names = {"RLB_ATTN_LONG": kernel, "RLB_ATTN_LONG_SPLITS": splits}
    before = {name: os.environ.get(name) for name in names}
    os.environ.update(names)
    try:
        cl = Cuda(stream=torch.cuda.current_stream().cuda_stream)
    finally:
        for name, value in before.items():
            os.environ.pop(name) if value is None else os.environ.__setitem__(name, value)
    yield cl
    torch.cuda.synchronize()
    cl.close()


@pytest.fixture(params=KERNELS, ids="-".join)
def on(request):
    kind, kernel, splits = request.param
    with context(kernel, splits) as cl:
        yield kind, cl


@pytest.mark.parametrize("kind", ["f32", "f16", "q4"])
def test_the_context_chooses(kind):
    """One launch, or two where records are joined; and the two kernels differ in their last bits."""
    q, k, v = T.normal(T.gen(0), 40, 8 * 128), T.normal(T.gen(1), 2, 500, 128), T.normal(T.gen(2), 2, 500, 128)
    results = {}
    for which in [(kernel, splits) for x, kernel, splits in KERNELS if x == kind]:
        with context(*which) as cl:
            before = cl.kernel_launches()
            results[which] = T.attend(cl, q, k, v, 8, 2, 128, 460, 1000, 0, kind, 500)[0]
            cluster = which == ("few", "3") and kind != "f32"
            assert cl.kernel_launches() - before == (kind == "q4") + (1 if which[1] == "1" or cluster else 2)
    assert not torch.equal(results["few", "1"], results["tiles", "1"])


def test_shapes(on):
    for shape in T.SHAPES:
        T.check_attention(on[1], *shape, on[0])


def test_long_contexts(on):
    for shape in T.LONG:
        T.check_attention(on[1], *shape, on[0])


@pytest.mark.parametrize("window", [0, 1, 31, 32, 33, 64, 65, 127, 128, 129])
def test_window_and_tile_edges(on, window):
    T.test_attention_window_and_tile_edges(on[1], on[0], window)


def test_random_shapes(on):
    import random
    for seed in range(20):
        r = random.Random(100 + seed)
        kv = r.choice([1, 2, 3, 5, 8])
        heads, n = kv * r.choice([1, 1, 2, 3, 7, 8, 16]), r.choice([1, 1, 2, 7, 20, 55, 100, 190, 333])
        start = int(2 ** r.uniform(0, 11.5)) - 1
        T.check_attention(on[1], heads, kv, r.choice([64, 128]), n, start, r.choice([10 ** 9, r.randrange(1, start + n + 1), r.randrange(1, start + n + 1)]),
                          r.choice([0, 0, 1, 4, 50, 10 ** 9]), on[0], seed=seed, max_seq=start + n + r.randrange(3))


def test_strided_rows(on):
    T.test_attention_strided_rows(on[1], on[0])


@pytest.mark.parametrize("n", [1, 3, 150, 300])
def test_rows_that_see_nothing_are_zero(on, n):
    T.test_attention_rows_that_see_nothing_are_zero(on[1], on[0], n)


@pytest.mark.parametrize("n,start,window,sinks", [(1, 900, 100, 4), (5, 900, 100, 4), (200, 700, 64, 3), (300, 0, 40, 0)])
def test_unseen_rows_may_hold_anything(on, n, start, window, sinks):
    T.test_attention_unseen_rows_may_hold_anything(on[1], on[0], n, start, window, sinks)


@pytest.mark.parametrize("on", [x for x in KERNELS if x[0] != "q4"], ids="-".join, indirect=True)
@pytest.mark.parametrize("n", [4, 40, 200])
def test_a_bad_row_reaches_only_the_rows_that_see_it(on, n):
    T.test_attention_a_bad_row_reaches_only_the_rows_that_see_it(on[1], on[0], n)


@pytest.mark.parametrize("on", [x for x in KERNELS if x[0] == "q4"], ids="-".join, indirect=True)
@pytest.mark.parametrize("n", [4, 40, 200, 300])
def test_a_bad_group_of_a_4_bit_row_reaches_only_the_rows_that_see_it(on, n):
    from rllama_b200 import Cache4
    cl = on[1]
    heads, kv, hd, start, window, sinks = 2, 1, 64, 50, 13, 2
    total, at = start + n, start + n // 2
    g = T.gen(6)
    q, k, v = T.normal(g, n, heads * hd), T.normal(g, total, hd), T.normal(g, total, hd)
    want, spread, top = T.attention64(q, *(T.values4(x).view(1, total, hd) for x in (k, v)), heads, kv, hd, start, window, sinks)
    tol = T.tolerance(want, spread, top, torch.float16, hd, window + sinks)
    sees = T.visible(start, n, window, sinks, total)[:, at]
    for which in (0, 1):
        parts = T.empty_cache4(kv, total, hd)
        cache, out = Cache4.wrap(cl, *parts, kv, total, hd), torch.empty(n, heads * hd, dtype=torch.float16, device=T.DEV)
        cache.append(cl.wrap(k), cl.wrap(v), 0)
        parts[1 + 2 * which][at, 1] = float("nan")
        cache.attention(cl.wrap(out), cl.wrap(q), heads, start, window, sinks)
        bad = out.view(n, heads, 2, 32)[sees].isnan()
        assert bad[:, :, 1].all() and (which == 1 or bad.all())
        assert ((out[~sees].double() - want[~sees]).abs() <= tol[~sees]).all()
        if which == 1:   # the other half of the result is that of the other values
            good = torch.zeros(n, heads, hd, dtype=torch.bool, device=T.DEV)
            good[..., :32] = True
            good = good.view(n, -1)
            assert ((out.double() - want).abs() <= tol)[good].all()


@pytest.mark.parametrize("n", [1, 6, 140, 300])
def test_flat_and_sharp(on, n):
    for q_scale in (1e-6, 30.0):
        T.test_attention_flat_and_sharp(on[1], on[0], n, q_scale)


@pytest.mark.parametrize("n", [1, 140, 300])
def test_magnitudes(on, n):
    T.test_attention_magnitudes(on[1], on[0], n)


@pytest.mark.parametrize("n", [5, 150])
def test_a_bad_query_reaches_only_its_row(on, n):
    T.test_attention_a_bad_query_reaches_only_its_row(on[1], on[0], n)


def check_best_row(cl, kind, n, size):
    """One-hot queries whose scores lie further apart than f32 can weigh: the result is the value of the largest score, or the mean of equal ones.
    (c of them: each weight may be rounded to f16 after it was added to their sum, 2^-11; the sum of c, the division and a product are c + 8 half steps
    of f32; the result is rounded to its type.)"""
    heads, kv, hd, start, window, total = 2, 1, 64, 200 - n, 90, 200
    g = T.gen(17)
    key = torch.arange(total, device=T.DEV)[torch.randperm(total, generator=g, device=T.DEV)]
    k, v = torch.zeros(kv, total, hd, device=T.DEV), T.normal(g, kv, total, hd)
    k[0, :, 0] = torch.where(key < 128, 1 + key / 128, 2 + (key - 128) / 64)
    q = torch.zeros(n, heads, hd, device=T.DEV)
    q[:, 0, 0], q[:, 1, 0] = size, -size
    out, k, v = T.attend(cl, q.view(n, -1), k, v, heads, kv, hd, start, window, 3, kind, total + 10)
    sees = T.visible(start, n, window, 3, total)
    half, weight = torch.finfo(out.dtype).eps / 2, 0.0 if kind == "f32" else 2.0 ** -11
    for h, sign in ((0, 1), (1, -1)):
        s = (sign * k[0, :, 0].double()).expand(n, total).masked_fill(~sees, -float("inf"))
        best = (s == s.amax(1, keepdim=True)).double()
        count = best.sum(1, keepdim=True)
        want, spread = (best @ x / count for x in (v[0].double(), v[0].double().abs()))
        off = (out.view(n, heads, hd)[:, h].double() - want).abs()
        assert (off <= half * want.abs() * (1 + weight) + (weight + (count + 8) * 2.0 ** -24) * spread + 2.0 ** -25).all()


@pytest.mark.parametrize("on", [x for x in KERNELS if x[1] == "few"], ids="-".join, indirect=True)
@pytest.mark.parametrize("n", [1, 5, 150])
@pytest.mark.parametrize("size", [1e30, 1e33, 1e34, 1e36, 1e37])
def test_queries_next_to_the_largest_f32(on, n, size):
    """Scores that f32 can still hold are computed without a step that it cannot."""
    check_best_row(on[1], on[0], n, size)


@pytest.mark.parametrize("n", [1, 5, 150])
@pytest.mark.parametrize("size", [1e6, 1e7, 1e8, 1e9, 3e9, 1e10, 1e11, 1e20, 1e30, 1e36])
def test_huge_queries_find_the_best_row(on, n, size):
    """Scores whose rounding in f32 is larger than the steps of an exponential: the largest one still weighs something."""
    check_best_row(on[1], on[0], n, size)


@pytest.mark.parametrize("n", [1, 40, 150])
def test_large_scores_of_full_queries(on, n):
    """The same with queries that are not one-hot, at magnitudes where scores pass 2^23 units: every row is a mean of values, never zero or NaN, and
    where the largest score leads by more than all roundings together it is that row's value."""
    kind, cl = on
    heads, kv, hd, start = 2, 1, 128, 300
    total = start + n
    for seed, size in enumerate((1e5, 1e7, 1e8, 1e9, 1e11)):
        g = T.gen(30 + seed)
        q, k, v = T.normal(g, n, heads * hd, scale=size), T.normal(g, kv, total, hd), T.normal(g, kv, total, hd)
        out, k, v = T.attend(cl, q, k, v, heads, kv, hd, start, 200, 3, kind, total + 3)
        sees = T.visible(start, n, 200, 3, total)
        assert torch.isfinite(out).all() and (out.view(n, heads, hd) != 0).any(-1).all()
        for h in range(heads):
            qq = q[:, h * hd:(h + 1) * hd].double()
            s = (qq @ k[0].double().T / hd ** 0.5).masked_fill(~sees, -float("inf"))
            size_of = torch.where(sees, qq.abs() @ k[0].double().abs().T / hd ** 0.5, 0.0).amax(-1)
            two = s.topk(2, -1)
            # scores off by 2^-11 (f16 queries) and (hd + 8) 2^-24 of their terms each; a lead of 20 beyond that leaves 1e-8 of the weight to the others
            sure = two.values[:, 0] - two.values[:, 1] > 2 * (2.0 ** -11 + (hd + 8) * 2.0 ** -24) * size_of + 20
            want = v[0].double()[two.indices[:, 0]]
            off = (out.view(n, heads, hd)[:, h].double() - want).abs()
            tol = torch.finfo(out.dtype).eps / 2 * want.abs() + (2.0 ** -11 * (kind != "f32") + 16 * 2.0 ** -24 + 1e-6) * (want.abs() + 10) + 2.0 ** -25
            assert sure.any() and (off <= tol)[sure].all()


def milliseconds(call):
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    times = []
    for _ in range(4):
        start.record()
        call()
        end.record()
        torch.cuda.synchronize()
        times.append(start.elapsed_time(end))
    return min(times[1:])


@pytest.mark.parametrize("kind,kernel", [("f32", "tiles"), ("f16", "few"), ("f16", "tiles"), ("q4", "few"), ("q4", "tiles")])
def test_rows_that_see_a_bad_position_cost_no_more(kind, kernel):
    """A row's result is not a number because of what it sees: nothing is to be gained from another pass over its positions. (Such passes made 128 rows
    after 4000 positions a hundred times slower.)"""
    from rllama_b200 import Cache4
    heads, hd, n, start = 8, 128, 128, 4000
    total, dt = start + n, torch.float32 if kind == "f32" else torch.float16
    g = T.gen(21)
    q, k, v = T.normal(g, n, heads * hd), T.normal(g, total, heads * hd), T.normal(g, total, heads * hd)
    out = torch.empty(n, heads * hd, dtype=dt, device=T.DEV)
    with context(kernel, "1") as cl:
        if kind == "q4":
            parts = T.empty_cache4(heads, total, hd)
            cache = Cache4.wrap(cl, *parts, heads, total, hd)
            cache.append(cl.wrap(k), cl.wrap(v), 0)
            places = [parts[1].view(heads, total, -1)[:, 100, 2]]       # K's scales; a V group cannot hold an infinity
            call = lambda: cache.attention(cl.wrap(out), cl.wrap(q), heads, start)
        else:
            kc, vc = (x.view(total, heads, hd).transpose(0, 1).reshape(heads * total, hd).to(dt) for x in (k, v))
            places = [x.view(heads, total, hd)[:, 100, 3] for x in (kc, vc)]
            call = lambda: cl.wrap(out).attention_window(cl.wrap(q), cl.wrap(kc), cl.wrap(vc), heads, heads, total, start, total)
        clean = milliseconds(call)
        for which, place in enumerate(places):
            before = place.clone()
            place.fill_(float("inf") if which else float("nan"))
            bad = milliseconds(call)
            o = out.view(n, heads, hd)
            assert bool((o[..., 3] == float("inf")).all()) if which else o.isnan().all()
            assert which == 0 or torch.isfinite(o[..., 4:]).all()
            assert bad < 4 * clean + 0.05, (clean, bad)
            place.copy_(before)
        q[:, 5] = float("nan")   # head 0 of every row
        bad = milliseconds(call)
        assert out.view(n, heads, hd)[:, 0].isnan().all() and torch.isfinite(out.view(n, heads, hd)[:, 1:]).all() and bad < 4 * clean + 0.05, (clean, bad)


@pytest.mark.parametrize("on", [x for x in KERNELS if x[0] != "f32"], ids="-".join, indirect=True)
@pytest.mark.parametrize("n", [1, 9, 300])
def test_values_next_to_the_largest_f16(on, n):
    """A mean of values is never beyond the largest of them: weights that were rounded up do not make an infinity of 65504 (4 bits: 65408)."""
    kind, cl = on
    heads, kv, hd, start = 8, 2, 128, 500
    total = start + n
    for seed in range(4):
        g = T.gen(40 + seed)
        q, k = T.normal(g, n, heads * hd, scale=1.0 + seed), T.normal(g, kv, total, hd)
        v = (65504.0 * torch.where(torch.arange(hd, device=T.DEV) % 3 == 0, -1.0, 1.0)).expand(kv, total, hd)
        out, k, v = T.attend(cl, q, k, v, heads, kv, hd, start, 300, 2, kind, total + 3)
        want = v[0, 0].repeat(heads).double()
        assert ((out.double() - want).abs() <= 2 * 2.0 ** -11 * want.abs()).all() and (out.double().abs() <= 65504).all()


@pytest.mark.parametrize("n", [1, 5, 40, 300])
def test_queries_keep_their_low_halves(on, n):
    """Two kinds of keys whose scores differ by what f16 queries would lose: every kernel holds 22 bits of them and tells them apart."""
    kind, cl = on
    heads, kv, hd, start = 4, 2, 128, 300
    total = start + n
    q = torch.full((n, heads, hd), 8.0, device=T.DEV)
    q[..., hd // 2:] *= 1 + 0.98 * 2.0 ** -11                       # rounds down to 8 in f16
    k = torch.zeros(kv, total, hd, device=T.DEV)
    k[:, ::2, :hd // 2] = k[:, 1::2, hd // 2:] = 1.4140625
    v = torch.ones(kv, total, hd, device=T.DEV)
    v[:, 1::2] = -1.0
    q = q.view(n, -1)
    out, k, v = T.attend(cl, q, k, v, heads, kv, hd, start, 200, 3, kind, total + 3)
    want, spread, top = T.attention64(q, k, v, heads, kv, hd, start, 200, 3)
    # queries 2^-22; products summed by additions that may cut off, a whole step each, with 4 bits of codes up to 15 where the values are 7; weights as
    # everywhere (2^-11 in f16, sums of 203)
    e = (2.0 ** -22 + 2 * (hd + 8) * 2.0 ** -24) * top * (15 / 7 if kind == "q4" else 1) + (211 + 8) * 2.0 ** -24 + (0 if kind == "f32" else 2.0 ** -11)
    tol = 1.1 * 2 * e * spread + torch.finfo(out.dtype).eps / 2 * want.abs() + 2.0 ** -25
    assert ((out.double() - want).abs() <= tol).all()
    short = T.attention64(q.half().float(), k, v, heads, kv, hd, start, 200, 3)[0]
    assert ((short - want).abs() > 2 * tol).all()   # (what a lost low half looks like)
