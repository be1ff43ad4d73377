"""Arguments of the long-context operators' Python forms that the library's 32 bits cannot hold, and handles that are gone."""
import sys

import pytest

from rllama_b200 import F32, Cache4, Cuda, CudaTensor, RllamaError

BEYOND = [2 ** 31, 2 ** 32, 2 ** 32 + 3, 2 ** 40, sys.maxsize, -2 ** 31 - 1, -2 ** 32]


@pytest.fixture
def bare(monkeypatch):
    """Objects without a device: every call ends in the library's refusal of null handles, unless it is refused before."""
    cl = Cuda.__new__(Cuda)
    import ctypes
    cl._h = ctypes.c_void_p()
    cache = Cache4.__new__(Cache4)
    cache._h, cache.max_seq_len = ctypes.c_void_p(), 8
    return cl, CudaTensor(cl, 1, 64, 64, F32), cache


@pytest.mark.parametrize("bad", BEYOND)
def test_numbers_beyond_32_bits_are_refused(bare, bad):
    cl, t, c = bare
    for call in (lambda x: t.norm_rope_append(t, t, t, t, t, t, x, 1, 1, 0), lambda x: t.norm_rope_append(t, t, t, t, t, t, 1, x, 1, 0),
                 lambda x: t.norm_rope_append(t, t, t, t, t, t, 1, 1, x, 0), lambda x: t.norm_rope_append(t, t, t, t, t, t, 1, 1, 1, x),
                 lambda x: t.attention_window(t, t, t, x, 1, 1, 0, 1), lambda x: t.attention_window(t, t, t, 1, x, 1, 0, 1),
                 lambda x: t.attention_window(t, t, t, 1, 1, x, 0, 1), lambda x: t.attention_window(t, t, t, 1, 1, 1, x, 1),
                 lambda x: c.append(t, t, x), lambda x: c.read(None, None, x), lambda x: c.attention(t, t, x, 0), lambda x: c.attention(t, t, 1, x),
                 lambda x: c.norm_rope_append(t, t, t, t, t, x, 0), lambda x: c.norm_rope_append(t, t, t, t, t, 1, x),
                 lambda x: cl.rope_table(x, 64), lambda x: cl.rope_table(4, x), lambda x: Cache4(cl, x, 1, 64), lambda x: Cache4(cl, 1, x, 64),
                 lambda x: Cache4(cl, 1, 1, x)):
        with pytest.raises(OverflowError):
            call(bad)
        for fits in (0, 1, -1, 2 ** 31 - 1, -2 ** 31):
            with pytest.raises(RllamaError) as e:   # it reaches the library
                call(fits)
            assert e.value.status == 1


def test_a_window_or_first_tokens_beyond_32_bits_are_all_there_is(bare):
    t, c = bare[1:]
    for x in BEYOND:
        for call in (lambda: t.attention_window(t, t, t, 1, 1, 1, 0, x), lambda: t.attention_window(t, t, t, 1, 1, 1, 0, 1, x), lambda: c.attention(t, t, 1, 0, x),
                     lambda: c.attention(t, t, 1, 0, 1, x)):
            with pytest.raises(RllamaError if x > 0 else OverflowError):
                call()


def test_a_freed_gain_is_not_a_missing_one(bare):
    cl, t, c = bare
    gone = CudaTensor(cl, 1, 64, 64, F32)
    for call in (lambda: t.norm_rope_append(t, t, t, t, t, t, 1, 1, 1, 0, gone), lambda: t.norm_rope_append(t, t, t, t, t, t, 1, 1, 1, 0, None, gone),
                 lambda: c.norm_rope_append(t, t, t, t, t, 1, 0, gone), lambda: c.read(gone, None, 0), lambda: c.read(None, gone, 0)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "q4"])
def test_results_with_a_window_or_first_tokens_beyond_32_bits(kind):
    import test_attention_long as T
    torch = T.torch
    cl = Cuda(stream=torch.cuda.current_stream().cuda_stream)
    for x in [b for b in BEYOND if b > 0]:
        T.check_attention(cl, 4, 2, 64, 3, 200, x, 0, kind)
        T.check_attention(cl, 4, 2, 64, 3, 200, 5, x, kind)


@pytest.mark.gpu
def test_rows_wider_than_31_bits_are_refused():
    """Columns are counted in 32 bits inside the kernels. (Without rows no memory is needed: the widths are checked first.)"""
    import test_attention_long as T
    torch, cl = T.torch, Cuda(stream=T.torch.cuda.current_stream().cuda_stream)
    W, heads = cl.wrap, 2 ** 25
    for h, status in ((heads, 7), (heads - 1, 0)):
        wide = [W(torch.empty(0, h * 64, dtype=dt, device=T.DEV)) for dt in (torch.float32, torch.float32, torch.float16)]
        row = [W(torch.zeros(1, 64, device=T.DEV)) for _ in range(2)]
        half = [W(torch.zeros(1, 64, dtype=torch.float16, device=T.DEV)) for _ in range(2)]
        none, table = W(torch.empty(0, 64, device=T.DEV)), cl.rope_table(1, 64)
        for call in (lambda: wide[0].attention_window(wide[1], *row, h, 1, 1, 0, 1), lambda: wide[2].attention_window(wide[0], *half, h, 1, 1, 0, 1),
                     lambda: wide[0].norm_rope_append(*row, wide[1], none, none, table, h, 1, 1, 0),
                     lambda: Cache4(cl, 1, 1, 64).attention(wide[2], wide[0], h, 0)):
            if status:
                with pytest.raises(RllamaError) as e:
                    call()
                assert e.value.status == status
            else:
                call()
