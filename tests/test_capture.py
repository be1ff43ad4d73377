"""What a caller may do with a context while its stream is captured into a CUDA graph: calls that cannot be part of a graph say so and leave the
capture as it is, and handles may be dropped."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture
def on():
    from rllama_b200 import Cuda
    side = torch.cuda.Stream()
    cl = Cuda(stream=side.cuda_stream)
    yield cl, side
    cl.close()


def captured(on, during):
    """x + 1 as a graph, with `during` called in between; x after three replays."""
    cl, side = on
    x = torch.zeros(4, 8, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        x.add_(1)
        during(cl.wrap(x))
        x.add_(1)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    return x


@pytest.mark.parametrize("what", ["zeros", "upload", "rope_table", "flush", "wait", "download", "cache4"])
def test_calls_that_cannot_be_captured_leave_the_capture_alone(on, what):
    from rllama_b200 import Cache4, RllamaError
    cl = on[0]
    calls = {"zeros": lambda x: cl.zeros(4, 8, 0), "upload": lambda x: cl.upload(np.zeros((4, 8), np.float32)), "rope_table": lambda x: cl.rope_table(8, 64),
             "flush": lambda x: cl.flush(), "wait": lambda x: x.wait_until_ready(), "download": lambda x: x.to_numpy(), "cache4": lambda x: Cache4(cl, 1, 8, 64)}

    def during(x):
        with pytest.raises(RllamaError) as e:
            calls[what](x)
        assert e.value.status == 5

    assert (captured(on, during) == 6).all()
    if what != "flush":
        calls[what](cl.wrap(torch.zeros(4, 8, device="cuda")))   # outside a capture all is well


def test_handles_may_be_dropped_during_a_capture(on):
    """As by a garbage collector: freeing them must not break the capture, and their memory comes back."""
    from rllama_b200 import Cache4
    cl = on[0]
    before = torch.cuda.mem_get_info()[0]
    room = 1 << 26
    drop = [cl.zeros(16, room, 0), cl.rope_table(64, 64), Cache4(cl, 64, 1 << 16, 128), cl.wrap(torch.zeros(4, 8, device="cuda"))]
    cl.flush()
    held = torch.cuda.mem_get_info()[0]
    assert before - held > 1 << 30

    def during(x):
        while drop:
            drop.pop().free()

    assert (captured(on, during) == 6).all()
    assert torch.cuda.mem_get_info()[0] - held > 1 << 30


def test_another_context_works_during_a_capture(on, monkeypatch):
    """A context on another stream may be made, allocate, run and go while this one's stream is captured (as by a second thread)."""
    from rllama_b200 import Cache4, Cuda
    monkeypatch.setenv("RLB_ATTN_LONG_SPLITS", "3r")   # scratch for records
    side = torch.cuda.Stream()
    q, kc = torch.ones(1, 256, device="cuda"), torch.ones(2 * 300, 128, dtype=torch.float16, device="cuda")
    outs = [torch.zeros(1, 256, dtype=torch.float16, device="cuda") for _ in range(3)]
    torch.cuda.synchronize()

    def during(x):
        other = Cuda(stream=side.cuda_stream)
        W = other.wrap
        W(outs[0]).attention_window(W(q), W(kc), W(kc), 2, 2, 300, 299, 300)
        table, cache, zeros = other.rope_table(300, 128), Cache4(other, 2, 300, 128), other.zeros(300, 256, 0)
        cache.append(zeros, zeros, 0)
        cache.attention(W(outs[1]), W(q), 2, 299)
        W(outs[2]).attention_decode(W(q), W(kc), W(kc), 2, 300, 299, 40)
        assert (W(outs[0]).to_numpy() == 1).all()
        other.flush()
        for t in (table, cache, zeros):
            t.free()
        other.close()

    outs[1].fill_(1)
    assert (captured(on, during) == 6).all()
    assert (outs[0] == 1).all() and (outs[1] == 0).all() and (outs[2] == 1).all()
