"""The long-context operators: rotation and append, the 4-bit cache, attention with a window and first tokens kept, over f16,
f32 and 4-bit caches. Each is compared with its formula in float64; the bounds are counted in roundings (below)."""
import ctypes
import math

import pytest

from rllama_b200 import _ffi

torch = pytest.importorskip("torch")
DEV = "cuda"
HALF = {torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}   # half a step, relative to the value


# ------------------------------------------------------------------------------------------- refusals that need no device
def test_null_handles_are_errors_not_crashes():
    lib = _ffi.lib()
    out = ctypes.c_void_p()
    assert lib.rlb_ctx_create_on_stream(0, 0, None, None) == 1
    assert lib.rlb_tensor_wrap(None, None, 1, 8, 8, 0, ctypes.byref(out)) == 1
    assert lib.rlb_rope_table(None, 4, 64, ctypes.byref(out)) == 1
    assert lib.rlb_norm_rope_append(None, None, None, None, None, None, None, None, 0.0, None, 1, 1, 1, 0) == 1
    assert lib.rlb_attention_window(None, None, None, None, 1, 1, 1, 0, 1, 0) == 1
    assert lib.rlb_cache4_create(None, 1, 1, 64, ctypes.byref(out)) == 1
    assert lib.rlb_cache4_wrap(None, None, None, None, None, 1, 1, 64, ctypes.byref(out)) == 1
    assert lib.rlb_cache4_append(None, None, None, 0) == 1
    assert lib.rlb_cache4_read(None, None, None, 0) == 1
    assert lib.rlb_cache4_attention(None, None, None, 1, 0, 1, 0) == 1
    assert lib.rlb_cache4_norm_rope_append(None, None, None, None, None, None, None, 0.0, None, 1, 0) == 1
    assert lib.rlb_cache4_free(None) == 0


def test_no_device_no_context_on_a_stream():
    lib = _ffi.lib()
    n = ctypes.c_int(-1)
    lib.rlb_device_count(ctypes.byref(n))
    if n.value > 0:
        pytest.skip("a CUDA device is present")
    h = ctypes.c_void_p()
    assert lib.rlb_ctx_create_on_stream(0, 0, None, ctypes.byref(h)) == 3 and not h.value


# ------------------------------------------------------------------------------------------- helpers
@pytest.fixture(scope="module")
def cl():
    from rllama_b200 import Cuda
    return Cuda(stream=torch.cuda.current_stream().cuda_stream)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV) * scale


def empty_cache4(kv, max_seq, hd):
    return [torch.zeros(kv * max_seq, w, dtype=t, device=DEV) for t, w in ((torch.uint8, hd // 2), (torch.float16, hd // 32)) * 2]


def values4(x):
    """The 4-bit format's values of rows x (rows, hd), in its own arithmetic on f32."""
    g = x.float().reshape(x.shape[0], -1, 32)
    d = (g.abs().amax(-1, keepdim=True).clamp(max=65504.0) * (1.0 / 7.0)).to(torch.bfloat16).to(torch.float16).float()
    u = torch.where(d > 0, (g / torch.where(d > 0, d, torch.ones_like(d))).clamp(-7, 7).round(), torch.zeros_like(g))
    return (u * d).reshape(x.shape)


def visible(start, n, window, sinks, total):
    row = torch.arange(start, start + n, device=DEV)[:, None]
    t = torch.arange(total, device=DEV)[None]
    return (t <= row) & ((t > row - window) | (t < sinks))


def attention64(q, k, v, heads, kv, hd, start, window, sinks):
    """float64 attention of rows q over k, v (kv, total, hd), and the largest error that the roundings allow.

    A weight exp(s) whose s is off by d_s and which is rounded with relative error r is off by at most E = d_s + r
    (first order; a factor of 1.1 below covers the rest, E < 0.1), numerator and denominator together move the result by at
    most 2 E sum p|v| / sum p, and its own rounding adds half a step of it."""
    n, total = q.shape[0], k.shape[1]
    seen = visible(start, n, window, sinks, total)
    out = torch.zeros(n, heads, hd, dtype=torch.float64, device=DEV)
    spread, top = torch.zeros_like(out), torch.zeros(n, heads, 1, dtype=torch.float64, device=DEV)
    for h in range(heads):
        kk, vv = k[h // (heads // kv)].double(), v[h // (heads // kv)].double()
        qq = q[:, h * hd:(h + 1) * hd].double()
        s = torch.where(seen, qq @ kk.T / math.sqrt(hd), -math.inf)
        p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
        out[:, h], spread[:, h] = p @ vv, p @ vv.abs()
        top[:, h] = torch.where(seen, qq.abs() @ kk.abs().T / math.sqrt(hd), 0.0).amax(-1, keepdim=True)
    return out.reshape(n, -1), spread.reshape(n, -1), top.expand(n, heads, hd).reshape(n, -1)


def tolerance(out, spread, top, dtype, hd, seen):
    f32 = 2.0 ** -24
    # scores: products of hd terms summed in f32, the exponential's argument and the exponential itself a few steps of f32;
    # weights summed over `seen` positions. An f16 output's weights and queries may be f16 tensor-core operands.
    e = (hd + 8) * f32 * top + 8 * f32 + (seen + 8) * f32
    if dtype == torch.float16:
        e = e + 2.0 ** -11 * top + 2.0 ** -11
    return 1.1 * 2 * e * spread + HALF[dtype] * out.abs() + (2.0 ** -25 if dtype == torch.float16 else 1e-37)


def attend(cl, q, k, v, heads, kv, hd, start, window, sinks, kind, max_seq, poison=True, out_pad=0, q_pad=0):
    """The framework's result on caches that hold k, v (kv, total, hd); rows behind `total` hold NaN. Also the caches' values."""
    from rllama_b200 import Cache4
    n, total = q.shape[0], k.shape[1]
    dt = torch.float32 if kind == "f32" else torch.float16
    wide = torch.full((n, heads * hd + out_pad), 7.0, dtype=dt, device=DEV)
    out = wide[:, :heads * hd]
    if q_pad:
        room = torch.full((n, heads * hd + q_pad), math.nan, device=DEV)
        room[:, :heads * hd] = q
        q = room[:, :heads * hd]
    if kind == "q4":
        parts = empty_cache4(kv, max_seq, hd)
        cache = Cache4.wrap(cl, *parts, kv, max_seq, hd)
        rows = [x.transpose(0, 1).reshape(total, kv * hd).contiguous() for x in (k, v)]
        cache.append(*(cl.wrap(x) for x in rows), 0)
        if poison:
            for s in (parts[1], parts[3]):
                s.view(kv, max_seq, -1)[:, total:] = math.nan
        k, v = (values4(x.reshape(-1, hd)).reshape(kv, total, hd) for x in (k, v))
        cache.attention(cl.wrap(out), cl.wrap(q), heads, start, window, sinks)
    else:
        kc, vc = (torch.full((kv, max_seq, hd), math.nan if poison else 0.0, dtype=dt, device=DEV) for _ in range(2))
        kc[:, :total], vc[:, :total] = k, v
        k, v = kc[:, :total].clone(), vc[:, :total].clone()
        cl.wrap(out).attention_window(cl.wrap(q), cl.wrap(kc.view(-1, hd)), cl.wrap(vc.view(-1, hd)), heads, kv, max_seq, start, window, sinks)
    cl.flush()  # raises if a kernel gave up on a wait
    if out_pad:
        assert (wide[:, heads * hd:] == 7.0).all(), "the padding of out was written"
    return out, k, v


def check_attention(cl, heads, kv, hd, n, start, window, sinks, kind, seed=0, max_seq=None, q_scale=1.5, **more):
    g = gen(seed)
    total = start + n
    q, k, v = normal(g, n, heads * hd, scale=q_scale), normal(g, kv, total, hd), normal(g, kv, total, hd)
    out, k, v = attend(cl, q, k, v, heads, kv, hd, start, window, sinks, kind, max_seq or total + 5, **more)
    want, spread, top = attention64(q, k, v, heads, kv, hd, start, window, sinks)
    tol = tolerance(want, spread, top, out.dtype, hd, min(total, window + sinks))
    off = (out.double() - want).abs()
    assert torch.isfinite(out).all()
    assert (off <= tol).all(), "worst %.3g of the bound at %s" % ((off / tol).max().item(), divmod((off / tol).argmax().item(), heads * hd))


# ------------------------------------------------------------------------------------------- rotation and append
@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,heads,kv,start,dtype,norm,pad", [(1, 4, 4, 0, "f16", True, 0), (1, 32, 32, 383, "f16", False, 0), (7, 6, 2, 5, "f32", True, 4),
                                                            (65, 13, 13, 1000, "f16", True, 8), (130, 5, 1, 29999, "f32", True, 0)])
def test_norm_rope_append(cl, n, heads, kv, start, dtype, norm, pad, hd):
    g = gen(1)
    max_seq, eps = start + n + 3, 1e-5
    dt = torch.float16 if dtype == "f16" else torch.float32
    q, k, v = (normal(g, n, h * hd + pad, scale=2.0)[:, :h * hd] for h in (heads, kv, kv))
    gains = [1 + normal(g, 1, hd, scale=0.2) for _ in range(2)] if norm else [None, None]
    kc, vc = (torch.full((kv * max_seq, hd), 7.0, dtype=dt, device=DEV) for _ in range(2))
    q_out = torch.empty(n, heads * hd, device=DEV)
    table = cl.rope_table(max_seq, hd)
    W = cl.wrap
    W(q_out).norm_rope_append(W(kc), W(vc), W(q), W(k), W(v), table, heads, kv, max_seq, start, *(W(x) if norm else None for x in gains), eps)

    pos = torch.arange(start, start + n, dtype=torch.float64, device=DEV)[:, None, None]
    ang = pos * 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=DEV) / hd)

    def turned(x, gain):
        x = x.double().reshape(n, -1, hd)
        if gain is not None:
            x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * gain.double()
        a, b = x[..., 0::2], x[..., 1::2]
        y = torch.stack([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()], -1).reshape(n, -1, hd)
        size = (a.abs() + b.abs()).repeat_interleave(2, -1)
        return y, size

    # f32 steps: the norm's sum (hd terms, in a tree: log2 of them and the lane's own four), division, root, reciprocal and two
    # products: 16; cos and sin one each, product and sum: 4
    f32 = 20 * 2.0 ** -24
    y, size = turned(q, gains[0])
    assert ((q_out.double().reshape(n, heads, hd) - y).abs() <= f32 * size).all()
    y, size = turned(k, gains[1])
    rows = kc.view(kv, max_seq, hd)
    got = rows[:, start:start + n].transpose(0, 1).double()
    assert ((got - y).abs() <= f32 * size + HALF[dt] * (y.abs() + f32 * size) + 2.0 ** -25 * (dt == torch.float16)).all()
    assert torch.equal(vc.view(kv, max_seq, hd)[:, start:start + n], v.reshape(n, kv, hd).transpose(0, 1).to(dt))
    for c in (rows, vc.view(kv, max_seq, hd)):  # the other rows of the caches stay as they were
        assert (c[:, :start] == 7.0).all() and (c[:, start + n:] == 7.0).all()


@pytest.mark.gpu
def test_norm_rope_append_in_place_and_without_rows(cl):
    g = gen(2)
    q, k = normal(g, 3, 128), normal(g, 3, 128)
    kc, vc = torch.zeros(2 * 8, 64, device=DEV), torch.zeros(2 * 8, 64, device=DEV)
    table = cl.rope_table(8, 64)
    W = cl.wrap
    q_out = torch.empty_like(q)
    W(q_out).norm_rope_append(W(kc), W(vc), W(q), W(k), W(k), table, 2, 2, 8, 2)
    wq = W(q)
    wq.norm_rope_append(W(kc), W(vc), wq, W(k), W(k), table, 2, 2, 8, 2)
    assert torch.equal(q, q_out)
    before = kc.clone()
    none = W(torch.empty(0, 128, device=DEV))
    none.norm_rope_append(W(kc), W(vc), none, none, none, table, 2, 2, 8, 8)
    assert torch.equal(kc, before)


# ------------------------------------------------------------------------------------------- the 4-bit cache
@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,kv,start,dtype,pad", [(1, 1, 0, "f32", 0), (1, 40, 639, "f16", 0), (3, 2, 5, "f32", 4), (77, 13, 1000, "f16", 8), (300, 4, 0, "f32", 0)])
def test_cache4_append_and_read(cl, n, kv, start, dtype, pad, hd):
    from rllama_b200 import Cache4
    g = gen(3)
    max_seq = start + n + 2
    dt = torch.float16 if dtype == "f16" else torch.float32
    k, v = (normal(g, n, kv * hd + pad, scale=s).to(dt)[:, :kv * hd] for s in (1.0, 1e-3))
    parts = empty_cache4(kv, max_seq, hd)
    for p in parts:
        p.fill_(9)
    cache, W = Cache4.wrap(cl, *parts, kv, max_seq, hd), cl.wrap
    cache.append(W(k), W(v), start)
    for out_dt in (torch.float16, torch.float32):
        ko, vo = (torch.empty(n, kv * hd, dtype=out_dt, device=DEV) for _ in range(2))
        cache.read(W(ko), W(vo), start)
        for x, got in ((k, ko), (v, vo)):
            want = values4(x.reshape(-1, hd)).reshape(n, kv * hd)
            assert torch.equal(got.float(), want)               # every value is an f16 number: no rounding anywhere
            group = x.float().reshape(n, -1, 32)
            step = group.abs().amax(-1, keepdim=True) / 7       # half a step, and what the scale's rounding (2^-9, or f16's smallest) takes
            off = (got.float().reshape(n, -1, 32) - group).abs()
            assert (off <= step * (0.5 + 7 * 2.0 ** -8) + 7 * 2.0 ** -25).all()
        only = torch.empty(n, kv * hd, dtype=out_dt, device=DEV)
        cache.read(None, W(only), start)
        assert torch.equal(only, vo)
    for p in parts:  # the other rows stay as they were
        rows = p.view(kv, max_seq, -1)
        assert (rows[:, :start] == 9).all() and (rows[:, start + n:] == 9).all()


def empty_like_cache(cl, kv, max_seq, hd):
    from rllama_b200 import Cache4
    parts = empty_cache4(kv, max_seq, hd)
    for p in parts:
        p.fill_(9)
    return parts, Cache4.wrap(cl, *parts, kv, max_seq, hd)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,heads,kv,start,norm,pad", [(1, 1, 1, 0, True, 0), (1, 40, 40, 383, False, 0), (5, 6, 2, 7, True, 4), (70, 3, 33, 500, True, 8),
                                                       (130, 34, 1, 29999, False, 0)])
def test_cache4_norm_rope_append(cl, n, heads, kv, start, norm, pad, hd):
    g = gen(19)
    max_seq, eps = start + n + 3, 1e-5
    q, k, v = (normal(g, n, h * hd + pad, scale=2.0)[:, :h * hd] for h in (heads, kv, kv))
    gains = [1 + normal(g, 1, hd, scale=0.2) for _ in range(2)] if norm else [None, None]
    table, W = cl.rope_table(max_seq, hd), cl.wrap
    wg = [W(x) if norm else None for x in gains]
    parts, cache = empty_like_cache(cl, kv, max_seq, hd)
    q_out = torch.empty(n, heads * hd, device=DEV)
    cache.norm_rope_append(W(q_out), W(q), W(k), W(v), table, heads, start, *wg, eps)
    # the two steps one after the other
    kc, vc = (torch.empty(kv * max_seq, hd, device=DEV) for _ in range(2))
    parts2, cache2 = empty_like_cache(cl, kv, max_seq, hd)
    q2 = torch.empty_like(q_out)
    W(q2).norm_rope_append(W(kc), W(vc), W(q), W(k), W(v), table, heads, kv, max_seq, start, *wg, eps)
    rows = [c.view(kv, max_seq, hd)[:, start:start + n].transpose(0, 1).reshape(n, kv * hd) for c in (kc, vc)]
    cache2.append(W(rows[0]), W(rows[1]), start)
    assert torch.equal(parts[2], parts2[2]) and torch.equal(parts[3], parts2[3])
    if not norm:   # (the norm's sums are taken in another order)
        assert torch.equal(q_out, q2) and torch.equal(parts[0], parts2[0]) and torch.equal(parts[1], parts2[1])
    pos = torch.arange(start, start + n, dtype=torch.float64, device=DEV)[:, None, None]
    ang = pos * 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=DEV) / hd)

    def turned(x, gain):
        x = x.double().reshape(n, -1, hd)
        if gain is not None:
            x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * gain.double()
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()], -1).reshape(n, -1, hd), (a.abs() + b.abs()).repeat_interleave(2, -1)

    # f32 steps: the norm's sum (eight terms one after the other, up to four groups, eight threads: at most 14 roundings, of which the root keeps half), division, sum with
    # eps, root, reciprocal, two products: 13; cos and sin one each, product and sum: 4
    f32 = 20 * 2.0 ** -24
    y, size = turned(q, gains[0])
    assert ((q_out.double().reshape(n, heads, hd) - y).abs() <= f32 * size).all()
    ko = torch.empty(n, kv * hd, device=DEV)
    cache.read(W(ko), None, start)
    y, size = turned(k, gains[1])
    y, size = y.reshape(n, -1, 32), size.reshape(n, -1, 32)
    step = (y.abs() + f32 * size).amax(-1, keepdim=True) / 7   # as for the append alone, of the rotated row's f32
    assert ((ko.double().reshape(n, -1, 32) - y).abs() <= step * (0.5 + 7 * 2.0 ** -8) + 7 * 2.0 ** -25 + f32 * size).all()
    for p in parts:
        held = p.view(kv, max_seq, -1)
        assert (held[:, :start] == 9).all() and (held[:, start + n:] == 9).all()
    wq = W(q)
    cache.norm_rope_append(wq, wq, W(k), W(v), table, heads, start, *wg, eps)   # in place
    assert torch.equal(q, q_out)


@pytest.mark.gpu
def test_cache4_norm_rope_append_refusals(cl):
    from rllama_b200 import Cuda, RllamaError
    W, f16 = cl.wrap, torch.float16
    cache, table = empty_like_cache(cl, 2, 10, 64)[1], cl.rope_table(10, 64)

    def t(r, c, dt=torch.float32, on=cl):
        return on.wrap(torch.zeros(r, c, dtype=dt, device=DEV))

    def call(q_out=None, q=None, k=None, v=None, tab=table, heads=4, start=3, qg=None, kg=None, eps=1e-6):
        cache.norm_rope_append(q_out or t(2, 256), q or t(2, 256), k or t(2, 128), v or t(2, 128), tab, heads, start, qg, kg, eps)

    call()
    call(q_out=t(0, 256), q=t(0, 256), k=t(0, 128), v=t(0, 128), start=10)
    other = Cuda(stream=torch.cuda.current_stream().cuda_stream)
    for bad in (dict(start=9), dict(start=-1), dict(heads=3), dict(heads=0), dict(q=t(3, 256)), dict(q_out=t(2, 128)), dict(q_out=t(2, 256, f16)), dict(q=t(2, 256, f16)),
                dict(k=t(2, 64)), dict(k=t(3, 128)), dict(k=t(2, 128, f16)), dict(v=t(2, 128, f16)), dict(v=t(2, 256)), dict(tab=cl.rope_table(4, 64)),
                dict(tab=cl.rope_table(10, 128)), dict(qg=t(1, 128)), dict(kg=t(2, 64)), dict(kg=t(1, 64, f16)), dict(eps=-1.0), dict(eps=math.nan),
                dict(q=t(2, 256, on=other)), dict(k=t(2, 128, on=other)), dict(qg=t(1, 64, on=other)), dict(tab=other.rope_table(10, 64))):
        with pytest.raises(RllamaError) as e:
            call(**bad)
        assert e.value.status == 1


@pytest.mark.gpu
def test_cache4_special_values(cl):
    from rllama_b200 import Cache4
    x = torch.zeros(8, 64, device=DEV)
    x[1, :32], x[1, 32:] = 3.0, -1.0
    x[2, 5], x[2, 40] = math.nan, math.inf
    x[3, 0], x[3, 33] = -math.inf, 1e-9
    x[4, 0], x[4, 63] = 1e30, 6e-8
    x[5] = torch.linspace(-1, 1, 64, device=DEV)
    x[6, :32] = torch.linspace(-3.5, 3.5, 32, device=DEV)   # exact halves of a step: ties
    x[6, 31] = 7.0
    x[7] = 65504.0
    cache, W = Cache4(cl, 1, 8, 64), cl.wrap
    cache.append(W(x), W(x), 0)
    out = torch.empty(8, 64, dtype=torch.float16, device=DEV)
    cache.read(W(out), None, 0)
    assert (out[0] == 0).all()
    assert torch.equal(out[1].float(), values4(x[1:2])[0]) and out[1, 0] > 0 > out[1, 63]
    assert torch.isnan(out[2, :32]).all() and out[2, 40] == 65408.0 and (out[2, 32:40] == 0).all()
    assert out[3, 0] == -65408.0 and (out[3, 32:] == 0).all()
    assert out[4, 0] == 65408.0 and (out[4, 1:32] == 0).all()
    for r in (4, 5, 6, 7):
        assert torch.equal(out[r].float(), values4(x[r:r + 1])[0])
    cache.free()


# ------------------------------------------------------------------------------------------- attention
SHAPES = [
    # heads, kv, hd, n, start, window, sinks
    (2, 2, 128, 1, 0, 1, 0),            # one position
    (4, 4, 64, 1, 96, 1000, 0),         # one row, everything
    (4, 2, 128, 1, 383, 100, 3),
    (8, 1, 128, 1, 5000, 700, 5),       # eight heads share
    (20, 1, 64, 1, 333, 334, 0),        # more heads share than a fragment holds
    (3, 3, 128, 1, 40, 1, 7),           # itself and the first
    (3, 1, 64, 1, 700, 300, 450),       # the runs meet
    (2, 2, 128, 2, 0, 1, 1),
    (6, 2, 128, 5, 61, 33, 2),
    (5, 5, 64, 16, 100, 40, 0),
    (4, 4, 128, 33, 0, 8, 1),
    (2, 1, 128, 77, 300, 100, 3),
    (3, 3, 64, 128, 0, 500, 0),
    (2, 2, 128, 129, 0, 64, 130),
    (1, 1, 128, 300, 513, 257, 4),
    (8, 2, 64, 200, 1, 90, 17),
    (3, 1, 128, 257, 255, 2000, 0),     # three heads in a row tile
    (2, 2, 64, 640, 0, 128, 129),
    (1, 1, 128, 5, 20, 0, 3),           # nothing but the first
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "q4"])
@pytest.mark.parametrize("heads,kv,hd,n,start,window,sinks", SHAPES)
def test_attention(cl, heads, kv, hd, n, start, window, sinks, kind):
    check_attention(cl, heads, kv, hd, n, start, window, sinks, kind)


LONG = [
    # enough positions that a row's splits are joined by a second kernel, or within a cluster, or not at all
    (2, 1, 128, 1, 40000, 100000, 0),
    (3, 1, 64, 3, 50000, 45000, 9),
    (16, 2, 128, 1, 30000, 29000, 70),
    (6, 6, 128, 1, 2000, 3000, 0),
    (40, 40, 128, 1, 1500, 3000, 0),
    (2, 1, 128, 150, 9000, 100000, 0),
    (8, 8, 64, 70, 6000, 5000, 40),
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "q4"])
@pytest.mark.parametrize("heads,kv,hd,n,start,window,sinks", LONG)
def test_attention_long_contexts(cl, heads, kv, hd, n, start, window, sinks, kind):
    check_attention(cl, heads, kv, hd, n, start, window, sinks, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "q4"])
@pytest.mark.parametrize("window", [0, 1, 31, 32, 33, 64, 65, 127, 128, 129])
def test_attention_window_and_tile_edges(cl, kind, window):
    """Windows, first tokens and row counts around the kernels' tiles of 16, 32, 64 and 128."""
    for i, (n, start, sinks) in enumerate([(1, 128, 0), (8, 56, 1), (9, 0, 16), (63, 1, 31), (64, 64, 32), (65, 63, 33), (127, 130, 64), (128, 0, 65),
                                           (129, 127, 128), (256, 0, 129)]):
        if window or sinks:
            check_attention(cl, 2, 1 + i % 2, 64 if i % 3 else 128, n, start, window, sinks, kind, seed=i)


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(24))
def test_attention_random_shapes(cl, seed):
    import random
    r = random.Random(seed)
    kv = r.choice([1, 2, 3, 5, 8])
    heads, n = kv * r.choice([1, 1, 2, 3, 7, 8, 16]), r.choice([1, 1, 2, 7, 20, 55, 100, 190, 333])
    start = int(2 ** r.uniform(0, 11.5)) - 1
    check_attention(cl, heads, kv, r.choice([64, 128]), n, start, r.choice([10 ** 9, r.randrange(1, start + n + 1), r.randrange(1, start + n + 1)]),
                    r.choice([0, 0, 1, 4, 50, 10 ** 9]), r.choice(["f16", "q4", "f32"]), seed=seed, max_seq=start + n + r.randrange(3))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "q4"])
def test_attention_strided_rows(cl, kind):
    for n in (1, 40, 200):
        check_attention(cl, 4, 2, 64, n, 30, 90, 2, kind, out_pad=16, q_pad=8)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "q4"])
@pytest.mark.parametrize("n", [1, 3, 150])
def test_attention_rows_that_see_nothing_are_zero(cl, kind, n):
    g = gen(4)
    q, k, v = normal(g, n, 256), normal(g, 2, n + 9, 128), normal(g, 2, n + 9, 128)
    out, _, _ = attend(cl, q, k, v, 2, 2, 128, 9, 0, 0, kind, n + 20)
    assert (out == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "q4"])
@pytest.mark.parametrize("n,start,window,sinks", [(1, 900, 100, 4), (5, 900, 100, 4), (200, 700, 64, 3), (300, 0, 40, 0)])
def test_attention_unseen_rows_may_hold_anything(cl, kind, n, start, window, sinks):
    """NaN and infinities in every cache row that no query sees, and the same finite result bit for bit."""
    from rllama_b200 import Cache4
    heads, kv, hd, total = 4, 2, 128, start + n
    g = gen(5)
    q, k, v = normal(g, n, heads * hd), normal(g, kv, total, hd), normal(g, kv, total, hd)
    clean, _, _ = attend(cl, q, k, v, heads, kv, hd, start, window, sinks, kind, total + 40, poison=False)
    low = max(0, start + 1 - window)
    for bad in (math.nan, math.inf, -math.inf):
        k2, v2 = k.clone(), v.clone()
        k2[:, sinks:low], v2[:, sinks:low] = bad, bad
        out, _, _ = attend(cl, q, k2, v2, heads, kv, hd, start, window, sinks, kind, total + 40)
        assert torch.equal(out, clean)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("n", [4, 40, 200])
def test_attention_a_bad_row_reaches_only_the_rows_that_see_it(cl, kind, n):
    heads, kv, hd, start, window, sinks = 2, 1, 64, 50, 13, 2
    total = start + n
    g = gen(6)
    q, k, v = normal(g, n, heads * hd), normal(g, kv, total, hd), normal(g, kv, total, hd)
    clean, k, v = attend(cl, q, k, v, heads, kv, hd, start, window, sinks, kind, total)
    want, spread, top = attention64(q, k, v, heads, kv, hd, start, window, sinks)
    tol = tolerance(want, spread, top, clean.dtype, hd, window + sinks)
    for which in (0, 1):
        at = start + n // 2
        k2, v2 = k.clone(), v.clone()
        (k2, v2)[which][:, at] = math.nan if which == 0 else math.inf
        out, _, _ = attend(cl, q, k2, v2, heads, kv, hd, start, window, sinks, kind, total)
        sees = visible(start, n, window, sinks, total)[:, at]
        assert not torch.isfinite(out[sees]).any()
        assert torch.isfinite(out[~sees]).all()
        # The formula's result for rows that do not see it has not changed, so the bound of every result holds for theirs, whichever way they
        # were computed. (Two ways differ by up to the sum of their bounds, in f32 hd + 8 steps times the scores' terms among them, not by the four
        # steps of the result that this test asked for at first.)
        assert ((out[~sees].double() - want[~sees]).abs() <= tol[~sees]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "q4"])
@pytest.mark.parametrize("n", [1, 6, 140])
@pytest.mark.parametrize("q_scale", [1e-6, 30.0])
def test_attention_flat_and_sharp(cl, kind, n, q_scale):
    check_attention(cl, 2, 2, 128, n, 600, 500, 2, kind, q_scale=q_scale)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "q4"])
@pytest.mark.parametrize("n", [1, 140])
def test_attention_magnitudes(cl, kind, n):
    """Queries beyond f16's range against tiny keys, and tiny values: nothing is lost on the way."""
    g = gen(7)
    heads, kv, hd, start = 2, 2, 128, 300
    total = start + n
    q, k, v = normal(g, n, heads * hd, scale=1e6), normal(g, kv, total, hd, scale=2e-3) * 1e-3, normal(g, kv, total, hd, scale=1e-3)
    k = (k * 1024).half().float() if kind == "f16" else k * 1024
    q = q / 1024
    out, k, v = attend(cl, q, k, v, heads, kv, hd, start, 200, 3, kind, total)
    want, spread, top = attention64(q, k, v, heads, kv, hd, start, 200, 3)
    assert ((out.double() - want).abs() <= tolerance(want, spread, top, out.dtype, hd, 203)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "q4"])
@pytest.mark.parametrize("n", [1, 5, 150])
@pytest.mark.parametrize("size", [1e30, 1e36])
def test_attention_of_huge_queries_is_the_best_row(cl, kind, n, size):
    """Scores further apart than f32 can weigh: the result is the value of the largest score, or the mean of equal ones."""
    heads, kv, hd, start, window = 2, 1, 64, 200 - n, 90
    g = gen(17)
    key = torch.arange(200, device=DEV)[torch.randperm(200, generator=g, device=DEV)]
    k, v = torch.zeros(kv, 200, hd, device=DEV), normal(g, kv, 200, hd)
    k[0, :, 0] = torch.where(key < 128, 1 + key / 128, 2 + (key - 128) / 64)
    q = torch.zeros(n, heads, hd, device=DEV)
    q[:, 0, 0], q[:, 1, 0] = size, -size
    out, k, v = attend(cl, q.view(n, -1), k, v, heads, kv, hd, start, window, 3, kind, 210)
    sees = visible(start, n, window, 3, 200)
    # In 4 bits neighbours from 1.75 on can share a scale (the step of an eight-bit scale next to 1/4 is 2^-9, theirs 2^-7 / 7): equal rows have equal
    # scores and weigh the same. The sum of c of them and the division are off by c + 2 half steps of f32, the result by half a step of its type.
    half = torch.finfo(out.dtype).eps / 2
    for h, sign in ((0, 1), (1, -1)):
        s = (sign * k[0, :, 0].double()).expand(n, 200).masked_fill(~sees, -math.inf)
        best = (s == s.amax(1, keepdim=True)).double()
        count = best.sum(1, keepdim=True)
        want, size = (best @ x / count for x in (v[0].double(), v[0].double().abs()))
        off = (out.view(n, heads, hd)[:, h].double() - want).abs()
        assert (off <= half * want.abs() + (count + 2) * 2.0 ** -24 * size + 2.0 ** -25).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "q4"])
@pytest.mark.parametrize("n", [5, 150])
def test_attention_a_bad_query_reaches_only_its_row(cl, kind, n):
    heads, kv, hd, start, window, sinks = 4, 2, 128, 30, 60, 2
    total = start + n
    g = gen(18)
    q, k, v = normal(g, n, heads * hd), normal(g, kv, total, hd), normal(g, kv, total, hd)
    bad = q.clone()
    bad[1, 3], bad[3, 2 * hd + 5] = math.nan, math.inf   # rows 1 and 3, heads 0 and 2
    out, k, v = attend(cl, bad, k, v, heads, kv, hd, start, window, sinks, kind, total)
    want, spread, top = attention64(q, k, v, heads, kv, hd, start, window, sinks)
    good = torch.ones(n, heads, dtype=torch.bool, device=DEV)
    good[1, 0] = good[3, 2] = False
    good = good.repeat_interleave(hd, 1)
    assert out[~good].isnan().all()
    assert ((out.double() - want).abs() <= tolerance(want, spread, top, out.dtype, hd, window + sinks))[good].all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f16", "q4"])
def test_attention_offsets_beyond_32_bits(cl, kind):
    """A cache whose last head starts past 2^32 elements (f16: past 2^33 bytes)."""
    heads = kv = 40
    hd, max_seq, n, start, window = 128, 1_000_003, 2, 1_000_000, 300
    from rllama_b200 import Cache4
    g = gen(8)
    q = normal(g, n, heads * hd)
    k, v = (normal(g, kv, window + n, hd).half() for _ in range(2))
    low = start + n - (window + n)
    out = torch.empty(n, heads * hd, dtype=torch.float16, device=DEV)
    W = cl.wrap
    if kind == "q4":
        cache = Cache4(cl, kv, max_seq, hd)
        rows = [x.transpose(0, 1).reshape(window + n, kv * hd).contiguous() for x in (k, v)]
        cache.append(W(rows[0]), W(rows[1]), low)
        cache.attention(W(out), W(q), heads, start, window)
        k, v = (values4(x.reshape(-1, hd)).reshape(x.shape) for x in (k, v))
        torch.cuda.synchronize()
        cache.free()
    else:
        kc, vc = (torch.zeros(kv, max_seq, hd, dtype=torch.float16, device=DEV) for _ in range(2))
        kc[:, low:start + n], vc[:, low:start + n] = k, v
        W(out).attention_window(W(q), W(kc.view(-1, hd)), W(vc.view(-1, hd)), heads, kv, max_seq, start, window)
    want, spread, top = attention64(q, k, v, heads, kv, hd, window, window, 0)
    assert ((out.double() - want).abs() <= tolerance(want, spread, top, out.dtype, hd, window)).all()


@pytest.mark.gpu
def test_attention_equals_the_framework_s_own_over_everything(cl):
    """Without a window and without shared heads: the same function as attention_decode and attention_prefill."""
    g = gen(9)
    heads, hd, max_seq = 4, 128, 300
    kc, vc = (normal(g, heads * max_seq, hd).half() for _ in range(2))
    for n, start in ((1, 250), (120, 60)):
        q = normal(g, n, heads * hd)
        a, b = (torch.empty(n, heads * hd, dtype=torch.float16, device=DEV) for _ in range(2))
        W = cl.wrap
        W(a).attention_window(W(q), W(kc), W(vc), heads, heads, max_seq, start, max_seq)
        if n == 1:
            W(b).attention_decode(W(q), W(kc), W(vc), heads, max_seq, start, 3)
        else:
            W(b).attention_prefill(W(q), W(kc), W(vc), heads, max_seq, start)
        k, v = (x.view(heads, max_seq, hd)[:, :start + n] for x in (kc, vc))
        want, spread, top = attention64(q, k, v, heads, heads, hd, start, max_seq, 0)
        tol = tolerance(want, spread, top, a.dtype, hd, start + n)
        assert ((a.double() - want).abs() <= tol).all() and ((b.double() - want).abs() <= tol).all()


# ------------------------------------------------------------------------------------------- the chain
@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f16", "f32", "q4"])
def test_a_prompt_and_tokens_one_by_one_agree(cl, kind):
    """rotate + append + attend, a prompt at once and then token by token, against the same chain in float64: what the K/V rows
    went through (rounding, or the 4-bit cache) is read back, the rest follows the formula."""
    from rllama_b200 import Cache4
    heads, kv, hd, max_seq, prompt, steps, window, sinks = 6, 3, 64, 200, 70, 5, 40, 2
    g = gen(10)
    W, dt = cl.wrap, torch.float32 if kind == "f32" else torch.float16
    table = cl.rope_table(max_seq, hd)
    gq, gk = 1 + normal(g, 1, hd, scale=0.1), 1 + normal(g, 1, hd, scale=0.1)
    # the rotated rows pass through an f32 or f16 cache; for the 4-bit one an f32 cache of one chunk hands them on
    kc, vc = (torch.zeros(kv * max_seq, hd, dtype=torch.float32 if kind == "q4" else dt, device=DEV) for _ in range(2))
    cache = Cache4(cl, kv, max_seq, hd) if kind == "q4" else None
    pos = 0
    for n in [prompt] + [1] * steps:
        q, k, v = normal(g, n, heads * hd), normal(g, n, kv * hd), normal(g, n, kv * hd)
        qr, out = torch.empty_like(q), torch.empty(n, heads * hd, dtype=dt, device=DEV)
        W(qr).norm_rope_append(W(kc), W(vc), W(q), W(k), W(v), table, heads, kv, max_seq, pos, W(gq), W(gk), 1e-6)
        if cache is not None:
            rows = [c.view(kv, max_seq, hd)[:, pos:pos + n].transpose(0, 1).reshape(n, kv * hd) for c in (kc, vc)]
            cache.append(W(rows[0]), W(rows[1]), pos)
            cache.attention(W(out), W(qr), heads, pos, window, sinks)
            held = [torch.empty(pos + n, kv * hd, dtype=torch.float32, device=DEV) for _ in range(2)]
            cache.read(W(held[0]), W(held[1]), 0)
            ck, cv = (h.reshape(pos + n, kv, hd).transpose(0, 1) for h in held)
        else:
            W(out).attention_window(W(qr), W(kc), W(vc), heads, kv, max_seq, pos, window, sinks)
            ck, cv = (c.view(kv, max_seq, hd)[:, :pos + n] for c in (kc, vc))
        want, spread, top = attention64(qr, ck, cv, heads, kv, hd, pos, window, sinks)
        assert ((out.double() - want).abs() <= tolerance(want, spread, top, out.dtype, hd, window + sinks)).all()
        pos += n


# ------------------------------------------------------------------------------------------- streams, graphs, devices
@pytest.mark.gpu
def test_context_on_a_stream_of_its_own_and_on_the_caller_s(cl):
    from rllama_b200 import Cuda
    g = gen(11)
    heads, hd, max_seq = 4, 128, 5000
    q, kc, vc = normal(g, 1, heads * hd), normal(g, heads * max_seq, hd).half(), normal(g, heads * max_seq, hd).half()
    want = torch.empty(1, heads * hd, dtype=torch.float16, device=DEV)
    W = cl.wrap
    W(want).attention_window(W(q), W(kc), W(vc), heads, heads, max_seq, 4999, 4000, 4)
    torch.cuda.synchronize()
    own = Cuda()
    a = torch.zeros_like(want)
    wa = own.wrap(a)
    wa.attention_window(own.wrap(q), own.wrap(kc), own.wrap(vc), heads, heads, max_seq, 4999, 4000, 4)
    wa.wait_until_ready()
    assert torch.equal(a, want) and (wa.to_numpy() == want.cpu().numpy()).all()
    side = torch.cuda.Stream()
    on = Cuda(stream=side.cuda_stream)
    b = torch.zeros_like(want)
    with torch.cuda.stream(side):
        q2 = q * 2                       # queued on the stream: the op must follow it ...
        on.wrap(b).attention_window(on.wrap(q2 / 2), on.wrap(kc), on.wrap(vc), heads, heads, max_seq, 4999, 4000, 4)
        c = b + 0                        # ... and come before this
    side.synchronize()
    assert torch.equal(c, want)
    own.close()
    on.close()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f16", "f32", "q4"])
def test_two_captured_graphs_side_by_side(kind):
    """Captured calls own their scratch: two graphs replayed on two streams at once, after a larger eager call in between."""
    from rllama_b200 import Cache4, Cuda
    side = torch.cuda.Stream()
    on = Cuda(stream=side.cuda_stream)
    heads, kv, hd, max_seq = 8, 2, 128, 20000
    g = gen(12)
    dt = torch.float32 if kind == "f32" else torch.float16
    if kind == "q4":
        cache = Cache4(on, kv, max_seq, hd)
        rows = [normal(g, max_seq, kv * hd) for _ in range(2)]
        torch.cuda.synchronize()
        cache.append(on.wrap(rows[0]), on.wrap(rows[1]), 0)
    else:
        kc, vc = (normal(g, kv * max_seq, hd).to(dt) for _ in range(2))
    qs = [normal(g, n, heads * hd) for n in (1, 1, 24)]
    outs = [torch.empty(q.shape, dtype=dt, device=DEV) for q in qs]
    starts = (19999, 15000, 12000)

    def call(i):
        if kind == "q4":
            cache.attention(on.wrap(outs[i]), on.wrap(qs[i]), heads, starts[i])
        else:
            on.wrap(outs[i]).attention_window(on.wrap(qs[i]), on.wrap(kc), on.wrap(vc), heads, kv, max_seq, starts[i], max_seq)

    torch.cuda.synchronize()
    for i in range(2):
        call(i)
    side.synchronize()
    want = [o.clone() for o in outs[:2]]
    graphs = []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call(i)
        graphs.append(graph)
    call(2)  # may replace the context's scratch
    side.synchronize()
    other = torch.cuda.Stream()
    for _ in range(20):
        for o in outs[:2]:
            o.fill_(math.nan)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    del graphs
    on.close()


@pytest.mark.gpu
def test_a_captured_step_follows_its_inputs():
    """rotate, append to both kinds of cache, read back and attend, in one graph that is replayed with new inputs in place."""
    from rllama_b200 import Cache4, Cuda
    side = torch.cuda.Stream()
    on = Cuda(stream=side.cuda_stream)
    heads, kv, hd, max_seq, pos = 8, 2, 64, 3000, 2900
    g = gen(15)
    q, k, v = normal(g, 1, heads * hd), normal(g, 1, kv * hd), normal(g, 1, kv * hd)
    kc, vc = (normal(g, kv * max_seq, hd).half() for _ in range(2))
    qr, q4, out, out4 = torch.empty_like(q), torch.empty_like(q), torch.empty(1, heads * hd, dtype=torch.float16, device=DEV), torch.empty(1, heads * hd, dtype=torch.float16, device=DEV)
    held = [torch.empty(1, kv * hd, device=DEV) for _ in range(2)]
    torch.cuda.synchronize()
    table, cache, W = on.rope_table(max_seq, hd), Cache4(on, kv, max_seq, hd), on.wrap

    def step():
        W(qr).norm_rope_append(W(kc), W(vc), W(q), W(k), W(v), table, heads, kv, max_seq, pos)
        W(out).attention_window(W(qr), W(kc), W(vc), heads, kv, max_seq, pos, 2500, 4)
        cache.append(W(k), W(v), pos)
        cache.read(W(held[0]), W(held[1]), pos)
        cache.norm_rope_append(W(q4), W(q), W(k), W(v), table, heads, pos)
        cache.attention(W(out4), W(q4), heads, pos, 5)

    step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for _ in range(3):
        for x in (q, k, v):
            x.copy_(normal(g, *x.shape))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (qr, q4, out, *held, out4)]
        with torch.cuda.stream(side):
            step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (qr, q4, out, *held, out4))) and torch.equal(qr, q4)
        assert torch.equal(held[0], values4(k.view(-1, hd)).view(1, -1)) and torch.equal(held[1], values4(v.view(-1, hd)).view(1, -1))
    del graph
    cache.free()
    on.close()


@pytest.mark.gpu
def test_two_threads_on_one_context(cl):
    """Calls from two host threads: each thread's results are those of its own inputs."""
    import threading
    g = gen(16)
    heads, kv, hd, max_seq = 8, 1, 128, 20000
    kc, vc = (normal(g, kv * max_seq, hd).half() for _ in range(2))
    qs = [normal(g, n, heads * hd) for n in (1, 40)]
    outs = [[torch.empty(q.shape, dtype=torch.float16, device=DEV) for _ in range(20)] for q in qs]
    W = cl.wrap
    args = [[(W(o), W(q)) for o in os] for os, q in zip(outs, qs)]
    wk, wv = W(kc), W(vc)
    torch.cuda.synchronize()

    def work(i):
        for o, q in args[i]:
            o.attention_window(q, wk, wv, heads, kv, max_seq, 19000 - i * 7000, 18000, 3)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        k, v = (x.view(kv, max_seq, hd)[:, :19000 - i * 7000 + len(qs[i])] for x in (kc, vc))
        want, spread, top = attention64(qs[i], k, v, heads, kv, hd, 19000 - i * 7000, 18000, 3)
        tol = tolerance(want, spread, top, torch.float16, hd, 18003)
        for o in outs[i]:
            assert ((o.double() - want).abs() <= tol).all() and torch.equal(o, outs[i][0])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 300])
def test_two_streams_at_once(n):
    """Contexts on two streams, whose kernels share the SMs (and their tensor memory): each has the results that it has alone."""
    from rllama_b200 import Cache4, Cuda
    heads, kv, hd, max_seq = 8, 4, 128, 6000
    start = max_seq - n
    g = gen(20)
    q = normal(g, n, heads * hd)
    kc, vc = (normal(g, kv * max_seq, hd).half() for _ in range(2))
    rows = [normal(g, max_seq, kv * hd) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    ons = [Cuda(stream=s.cuda_stream) for s in streams]
    outs = [[torch.empty(n, heads * hd, dtype=torch.float16, device=DEV) for _ in range(12)] for _ in range(2)]
    torch.cuda.synchronize()
    cache = Cache4(ons[1], kv, max_seq, hd)
    cache.append(*(ons[1].wrap(x) for x in rows), 0)
    calls = [lambda o: ons[0].wrap(o).attention_window(ons[0].wrap(q), ons[0].wrap(kc), ons[0].wrap(vc), heads, kv, max_seq, start, 4000, 4),
             lambda o: cache.attention(ons[1].wrap(o), ons[1].wrap(q), heads, start)]
    alone = []
    for call in calls:
        o = torch.empty(n, heads * hd, dtype=torch.float16, device=DEV)
        torch.cuda.synchronize()
        call(o)
        torch.cuda.synchronize()
        alone.append(o)
    for i in range(12):
        for k in range(2):
            calls[k](outs[k][i])
    torch.cuda.synchronize()
    for k in range(2):
        assert torch.isfinite(alone[k]).all() and all(torch.equal(o, alone[k]) for o in outs[k])
    cache.free()
    for on in ons:
        on.close()


@pytest.mark.gpu
def test_ops_with_scratch_of_the_context_refuse_capture():
    from rllama_b200 import Cuda, RllamaError
    side = torch.cuda.Stream()
    on = Cuda(stream=side.cuda_stream)
    q, kc = torch.zeros(1, 256, device=DEV), torch.zeros(2 * 64, 128, dtype=torch.float16, device=DEV)
    out, w = torch.zeros(1, 256, dtype=torch.float16, device=DEV), torch.zeros(32, 128, dtype=torch.float16, device=DEV)
    c = torch.zeros(32, 128, dtype=torch.float16, device=DEV)
    T = [on.wrap(x) for x in (q, kc, out, w, c)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out.fill_(1.0)
        for call in (lambda: T[2].attention_decode(T[0], T[1], T[1], 2, 64, 5, 2), lambda: T[2].attention_decode_static(T[0], T[1], T[1], 2, 64, 5, 2),
                     lambda: T[4].matrix_mul_inplace_transposed(T[3], T[1])):
            with pytest.raises(RllamaError) as e:
                call()
            assert e.value.status == 5
    graph.replay()
    torch.cuda.synchronize()
    assert (out == 1.0).all()
    del graph
    with pytest.raises(RllamaError) as e:
        from rllama_b200 import DataSettings, Transformer
        Transformer(64, 1, 1, 64, 64, 8, 1e-6, DataSettings(cl=on))
    assert e.value.status == 5


@pytest.mark.gpu
def test_results_do_not_change_from_call_to_call(cl):
    g = gen(13)
    heads, kv, hd, max_seq = 8, 2, 128, 9000
    kc, vc = normal(g, kv * max_seq, hd).half(), normal(g, kv * max_seq, hd).half()
    for n, start in ((1, 8999), (9, 8000), (500, 3000)):
        q = normal(g, n, heads * hd)
        first = None
        for _ in range(6):
            out = torch.empty(n, heads * hd, dtype=torch.float16, device=DEV)
            cl.wrap(out).attention_window(cl.wrap(q), cl.wrap(kc), cl.wrap(vc), heads, kv, max_seq, start, 6000, 4)
            first = out if first is None else first
            assert torch.equal(out, first)


# ------------------------------------------------------------------------------------------- wrapped tensors and refusals
@pytest.mark.gpu
def test_wrapped_tensors_in_the_older_ops(cl):
    """Views of wider tensors: what lies between their rows is neither read nor written."""
    g = gen(14)
    for dt, tol in ((torch.float16, 2.0 ** -10), (torch.float32, 1e-5)):
        for rows in (1, 5, 40):
            t = torch.full((rows, 64), 7.0, dtype=dt, device=DEV)
            part = t[:, :21]
            part.copy_(normal(g, rows, 21))
            before = part.clone()
            cl.wrap(part).silu_inplace()
            cl.wrap(part).hadamard_product_inplace(cl.wrap(part))
            want = torch.nn.functional.silu(before.double()).to(dt).double().square()
            assert ((part.double() - want).abs() <= 4 * tol * (1 + want.abs())).all() and (t[:, 21:] == 7.0).all()
            wide = torch.full((rows, 64), math.nan, dtype=dt, device=DEV)
            x = wide[:, :19]
            x.copy_(normal(g, rows, 19))
            wide_w = torch.full((24, 48), math.nan, dtype=dt, device=DEV)
            w = wide_w[:, :19]
            w.copy_(normal(g, 24, 19))
            for m in (24, 21):   # rows of w, i.e. columns of the product
                y = torch.full((rows, 32), 7.0, dtype=dt, device=DEV)
                cl.wrap(y[:, :m]).matrix_mul_inplace_transposed(cl.wrap(x), cl.wrap(w[:m]))
                want = x.double() @ w[:m].double().T
                assert ((y[:, :m].double() - want).abs() <= tol * (1 + want.abs()) * 4).all()
                assert (y[:, m:] == 7.0).all()
            assert (cl.wrap(x).to_numpy() == x.cpu().numpy()).all()


@pytest.mark.gpu
def test_refusals(cl):
    from rllama_b200 import Cache4, Cuda, RllamaError
    W = cl.wrap
    f16, f32 = torch.float16, torch.float32

    def t(r, c, dt=f32):
        return torch.zeros(r, c, dtype=dt, device=DEV)

    def refused(call, status=1):
        with pytest.raises(RllamaError) as e:
            call()
        assert e.value.status == status

    q, out, kc = W(t(2, 256)), W(t(2, 256, f16)), W(t(2 * 10, 128, f16))
    att = lambda o=out, qq=q, k=kc, v=kc, h=2, kv=2, m=10, s=3, w=4, z=1: o.attention_window(qq, k, v, h, kv, m, s, w, z)
    att()
    refused(lambda: att(s=9))                       # past the cache
    refused(lambda: att(s=-1))
    refused(lambda: att(w=-1))
    refused(lambda: att(z=-1))
    refused(lambda: att(h=3))                       # heads no multiple, q of another width
    refused(lambda: att(h=4))
    refused(lambda: att(kv=1))                      # caches of another size
    refused(lambda: att(kv=0))
    refused(lambda: att(m=11))
    refused(lambda: att(o=W(t(2, 256))))            # out's dtype
    refused(lambda: att(o=W(t(1, 256, f16))))
    refused(lambda: att(qq=W(t(2, 256, f16))))
    refused(lambda: att(v=W(t(20, 128))))           # K and V of two dtypes
    refused(lambda: att(k=W(t(20, 96, f16)), v=W(t(20, 96, f16)), qq=W(t(2, 192)), o=W(t(2, 192, f16))))  # head_dim
    k32 = W(t(20, 128))
    refused(lambda: att(o=q, k=k32, v=k32))         # out is q
    other = Cuda(stream=0)
    refused(lambda: att(qq=other.wrap(t(2, 256))))  # another context
    cache = Cache4(cl, 2, 10, 128)
    cat = lambda o=out, qq=q, h=2, s=3, w=4, z=1: cache.attention(o, qq, h, s, w, z)
    cat()
    refused(lambda: cat(s=9))
    refused(lambda: cat(h=3))
    refused(lambda: cat(w=-2))
    refused(lambda: cat(o=W(t(2, 256))))
    refused(lambda: cat(o=other.wrap(t(2, 256, f16)), qq=other.wrap(t(2, 256))))
    refused(lambda: cache.append(q, out, 0))        # two dtypes
    refused(lambda: cache.append(q, W(t(3, 256)), 0))
    refused(lambda: cache.append(W(t(2, 128)), W(t(2, 128)), 0))
    refused(lambda: cache.append(q, q, 9))
    refused(lambda: cache.append(q, q, -1))
    refused(lambda: cache.read(None, None, 0))
    refused(lambda: cache.read(q, None, 9))
    refused(lambda: cache.read(q, out, 0))
    refused(lambda: Cache4(cl, 0, 10, 128))
    refused(lambda: Cache4(cl, 2, 0, 128))
    refused(lambda: Cache4(cl, 2, 10, 96))
    with pytest.raises(ValueError):
        Cache4.wrap(cl, *empty_cache4(2, 10, 128)[::-1], 2, 10, 128)
    parts = empty_cache4(2, 10, 128)
    with pytest.raises(ValueError):
        Cache4.wrap(cl, *parts, 2, 11, 128)

    table = cl.rope_table(10, 128)
    x = W(t(2, 256))
    rot = lambda o=x, k_c=kc, v_c=kc, qq=q, k=q, v=q, tab=table, h=2, kv=2, m=10, s=3, g=None, e=1e-6: o.norm_rope_append(k_c, v_c, qq, k, v, tab, h, kv, m, s, g, None, e)
    rot()
    refused(lambda: rot(s=9))
    refused(lambda: rot(s=-1))
    refused(lambda: rot(h=3))
    refused(lambda: rot(kv=1))
    refused(lambda: rot(m=9))
    refused(lambda: rot(o=out))
    refused(lambda: rot(k=W(t(3, 256))))
    refused(lambda: rot(v=out))
    refused(lambda: rot(tab=cl.rope_table(4, 128)))  # too short
    refused(lambda: rot(tab=cl.rope_table(10, 64)))
    refused(lambda: rot(g=W(t(1, 64))))
    refused(lambda: rot(e=-1.0))
    refused(lambda: rot(e=math.nan))
    refused(lambda: rot(v_c=k32))
    refused(lambda: cl.rope_table(0, 128))
    refused(lambda: cl.rope_table(4, 6))

    for bad in (torch.zeros(4, 8, device=DEV, dtype=torch.int32), torch.zeros(4, 8), torch.zeros(8, device=DEV), torch.zeros(8, 8, device=DEV).T[:, ::2]):
        with pytest.raises(ValueError):
            cl.wrap(bad)
    base = torch.zeros(8, 20, device=DEV)
    refused(lambda: cl.wrap(base[:, 1:9]))          # 16-byte alignment
    refused(lambda: cl.wrap(torch.zeros(3, 9, device=DEV)))
    lib, h = _ffi.lib(), ctypes.c_void_p()
    host = torch.zeros(64)
    assert lib.rlb_tensor_wrap(cl._h, ctypes.c_void_p(host.data_ptr() // 16 * 16), 1, 8, 8, 0, ctypes.byref(h)) == 1  # host memory
    here = ctypes.c_void_p(base.data_ptr())
    assert lib.rlb_tensor_wrap(cl._h, here, 1 << 44, 8, 8, 0, ctypes.byref(h)) == 1   # an end that is no memory
    assert lib.rlb_tensor_wrap(cl._h, here, 1 << 62, 8, 8, 0, ctypes.byref(h)) == 1
    assert lib.rlb_cache4_wrap(cl._h, here, here, here, here, 60000, 1 << 30, 128, ctypes.byref(h)) == 1
    assert lib.rlb_cache4_create(cl._h, 1, (1 << 30) + 1, 128, ctypes.byref(h)) == 7
    refused(lambda: Cache4(cl, 65536, 1 << 30, 128), 4)   # more than there is
    assert torch.zeros(4, device=DEV).add_(1).sum().item() == 4   # none of these is an error of the caller's next call


@pytest.mark.gpu
def test_handles_may_outlive_their_context():
    from rllama_b200 import Cache4, Cuda
    on = Cuda(stream=torch.cuda.current_stream().cuda_stream)
    table, cache, view, zeros = on.rope_table(16, 64), Cache4(on, 1, 16, 64), on.wrap(torch.zeros(4, 8, device=DEV)), on.zeros(4, 8, 0)
    on.close()
    for x in (table, cache, view, zeros):
        x.free()
    assert torch.zeros(4, device=DEV).add_(1).sum().item() == 4


@pytest.mark.gpu
def test_a_call_without_rows_does_nothing(cl):
    from rllama_b200 import Cache4
    W = cl.wrap
    q, out, kc = W(torch.empty(0, 256, device=DEV)), W(torch.empty(0, 256, dtype=torch.float16, device=DEV)), W(torch.zeros(20, 128, dtype=torch.float16, device=DEV))
    out.attention_window(q, kc, kc, 2, 2, 10, 10, 4, 1)
    cache = Cache4(cl, 2, 10, 128)
    cache.append(q, q, 10)
    cache.read(out, out, 10)
    cache.attention(out, q, 2, 10)


@pytest.mark.gpu
def test_the_current_device_and_stream_stay_the_caller_s(cl):
    before = torch.cuda.current_device()
    check_attention(cl, 2, 2, 64, 1, 10, 5, 1, "f16")
    assert torch.cuda.current_device() == before
