"""The rotation into an f16 or f32 cache and the one into a 4-bit cache are documented as one computation: the same bits."""
import pytest

import test_attention_long as T

torch = T.torch


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,heads,kv,start,pad", [(1, 1, 1, 0, 0), (1, 40, 40, 383, 0), (5, 6, 2, 7, 4), (70, 3, 33, 500, 8), (131, 64, 8, 2999, 0)])
def test_both_rotations_agree_bit_for_bit(n, heads, kv, start, pad, hd):
    from rllama_b200 import Cuda
    cl = Cuda(stream=torch.cuda.current_stream().cuda_stream)
    g = T.gen(50)
    max_seq = start + n + 1
    q, k, v = (T.normal(g, n, h * hd + pad, scale=2.0)[:, :h * hd] for h in (heads, kv, kv))
    gains = [1 + T.normal(g, 1, hd, scale=0.2) for _ in range(2)]
    W, table = cl.wrap, cl.rope_table(max_seq, hd)
    kc, vc = (torch.zeros(kv * max_seq, hd, device=T.DEV) for _ in range(2))
    a, b = torch.empty(n, heads * hd, device=T.DEV), torch.empty(n, heads * hd, device=T.DEV)
    W(a).norm_rope_append(W(kc), W(vc), W(q), W(k), W(v), table, heads, kv, max_seq, start, *map(W, gains), 1e-5)
    parts, cache = T.empty_like_cache(cl, kv, max_seq, hd)
    cache.norm_rope_append(W(b), W(q), W(k), W(v), table, heads, start, *map(W, gains), 1e-5)
    assert torch.equal(a, b)
    rows = [c.view(kv, max_seq, hd)[:, start:start + n].transpose(0, 1).reshape(n, kv * hd) for c in (kc, vc)]
    parts2, cache2 = T.empty_like_cache(cl, kv, max_seq, hd)
    cache2.append(W(rows[0]), W(rows[1]), start)
    assert all(torch.equal(x, y) for x, y in zip(parts, parts2))
    for m, c in zip((0, 1), (kc, vc)):   # and an f16 cache holds the f32 one's rows, rounded
        half = [torch.zeros(kv * max_seq, hd, dtype=torch.float16, device=T.DEV) for _ in range(2)]
        W(a).norm_rope_append(W(half[0]), W(half[1]), W(q), W(k), W(v), table, heads, kv, max_seq, start, *map(W, gains), 1e-5)
        assert torch.equal(half[m], c.half())
    cl.flush()


@pytest.mark.gpu
def test_shared_heads_cost_what_their_bytes_do():
    """64 query heads on 8 K/V heads move 0.53 of the bytes of 64 on 64 (the K/V planes of the grid once worked on as many heads as q's)."""
    from rllama_b200 import Cuda
    cl = Cuda(stream=torch.cuda.current_stream().cuda_stream)
    n, heads, hd, max_seq, W = 1792, 64, 128, 2048, cl.wrap
    table, gain, us = cl.rope_table(max_seq, hd), torch.ones(1, hd, device=T.DEV), {}
    for kv in (64, 8):
        sets = []
        for _ in range(4):   # more than the L2 cache holds
            q, k, v = (torch.ones(n, h * hd, device=T.DEV) for h in (heads, kv, kv))
            sets.append([W(x) for x in (torch.empty_like(q), q, k, v)] + [T.empty_like_cache(cl, kv, max_seq, hd)[1]])
        best = []
        for _ in range(6):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            for i in range(20):
                q_out, q, k, v, cache = sets[i % 4]
                cache.norm_rope_append(q_out, q, k, v, table, heads, 0, W(gain), W(gain))
            end.record()
            torch.cuda.synchronize()
            best.append(start.elapsed_time(end))
        us[kv] = min(best[1:]) * 50
    assert us[8] < 0.72 * us[64], us
