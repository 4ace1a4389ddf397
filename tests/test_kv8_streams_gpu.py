"""A context whose stream is not torch's current one: what a call takes from the allocator belongs to the context's stream, so that
neither the current stream's kernels nor what is allocated there later meets it."""
import pytest
import torch

import cuda_ltc_b200 as ltc
from test_kv8_gpu import device_cache, filled, ints, queries
from util import randn

pytestmark = pytest.mark.gpu

B, H, G, S, D = 2, 2, 2, 20000, 64                      # steps that many warps share: the call needs scratch


@pytest.fixture(scope="module")
def given():
    cache = device_cache(filled(B, H, S, D, 64, 3))
    return cache, queries(B, H * G, 1, D, "bf16", 4), ints([S, S - 77])


@pytest.fixture
def aside():
    """A context on a stream of its own, and that stream."""
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    c = ltc.Context(0, stream)
    yield c, stream
    torch.cuda.synchronize()
    assert c.device_status() == 0
    c.close()


def busy(stream):
    """Some ten milliseconds of nothing."""
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)


CALLS = {
    "decode": lambda c, cache, q, n: c.kv8_decode(q, cache, kv_len=n),
    "read": lambda c, cache, q, n: c.kv8_read(cache, kv_len=n, count=128),
    "select": lambda c, cache, q, n: (c.kv8_select(q, cache, n, 9),),
    "forward": lambda c, cache, q, n: c.attn_fwd(q, q, q),
}


@pytest.mark.parametrize("name", list(CALLS))
def test_results_that_are_let_go_early(given, aside, name):
    """The call waits behind its own stream's work; its results are dropped, and tensors of their sizes made on the current stream
    keep what is written to them."""
    c, stream = aside
    sizes = [(t.shape, t.dtype) for t in CALLS[name](c, *given)]
    torch.cuda.synchronize()
    for _ in range(3):
        busy(stream)
        CALLS[name](c, *given)
        kept = [torch.full(shape, 7, dtype=dtype, device="cuda") for shape, dtype in sizes for _ in range(4)]
        torch.cuda.synchronize()
        assert all((t == 7).all().item() for t in kept)


@pytest.mark.parametrize("name", list(CALLS))
def test_results_where_the_current_stream_has_yet_to_write(given, aside, name):
    """Blocks that the current stream has given back and still writes to later are not what the call gets."""
    c, stream = aside
    want = [t.clone() for t in CALLS[name](c, *given)]
    torch.cuda.synchronize()
    for _ in range(3):
        busy(torch.cuda.current_stream())
        let_go = [torch.full(t.shape, 7, dtype=t.dtype, device="cuda") for t in want for _ in range(4)]
        del let_go
        got = CALLS[name](c, *given)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_results_and_scratch_in_a_captured_graph(given, aside):
    """Captured on the context's stream while another one of the capture is current."""
    c, stream = aside
    want = [t.clone() for t in CALLS["decode"](c, *given)]
    torch.cuda.synchronize()
    graph, main = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=main):
        stream.wait_stream(main)
        got = CALLS["decode"](c, *given)
        main.wait_stream(stream)
    others = [torch.full(t.shape, 7, dtype=t.dtype, device="cuda") for t in want for _ in range(4)]
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and all((t == 7).all().item() for t in others)


@pytest.mark.parametrize("bounds", [False, True])
def test_a_new_cache_is_written_behind_its_making(aside, bounds):
    """The current stream is busy when the cache is made: what is appended right after stays."""
    c, stream = aside
    k, v = (torch.from_numpy(randn((2, 2, 70, 64), i)).cuda().bfloat16() for i in range(2))
    n = ints([70, 33])
    want = c.kv8_cache(2, 2, 70, 64, bounds=bounds)
    c.kv8_append(want, k, v, n)
    torch.cuda.synchronize()
    for _ in range(3):
        busy(torch.cuda.current_stream())
        cache = c.kv8_cache(2, 2, 70, 64, bounds=bounds)
        c.kv8_append(cache, k, v, n)
        torch.cuda.synchronize()
        for a, b in zip(cache[:5], want[:5]):
            assert a is b is None or torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_the_stream_is_the_contexts_own_whoever_sets_it(aside):
    import ctypes as C
    c, stream = aside
    at = C.c_void_p()
    for s in (stream, torch.cuda.Stream(), torch.cuda.current_stream()):
        c.lib.ltca_ctx_set_stream(c.handle, C.c_void_p(s.cuda_stream))
        assert c.lib.ltca_ctx_get_stream(c.handle, C.byref(at)) == 0 and (at.value or 0) == s.cuda_stream
        assert c.stream().cuda_stream == s.cuda_stream
    assert c.lib.ltca_ctx_get_stream(None, C.byref(at)) == -1 and c.lib.ltca_ctx_get_stream(c.handle, None) == -1
