"""Operators called from several threads and streams."""
import ctypes as C
import threading

import pytest
import torch

from auratensor_b200 import _lib
from auratensor_b200.core import context
from auratensor_b200.kvblock import BlockKvCache, TokenBatch

pytestmark = pytest.mark.gpu


def stream_of(ctx):
    s = C.c_void_p()
    _lib.call("at_ctx_stream", ctx, C.byref(s))
    return s.value


def in_threads(*steps):
    """Runs lists of callables, one list per thread, step by step in turn; raises what they raise."""
    barrier, errors = threading.Barrier(len(steps), timeout=60), []

    def work(i):
        try:
            for j in range(max(map(len, steps))):
                for who in range(len(steps)):
                    barrier.wait()
                    if who == i and j < len(steps[i]):
                        steps[i][j]()
        except BaseException as e:  # noqa: BLE001
            errors.append(e)
            barrier.abort()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(steps))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for e in errors:
        if not isinstance(e, threading.BrokenBarrierError):
            raise e


def test_a_context_is_bound_per_thread(cuda):
    """Thread B's call does not move thread A's launches to B's stream."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    seen = {}

    def bind(i):
        with torch.cuda.stream(streams[i]):
            context(0)

    def look(i):
        seen[i] = stream_of(context_of)

    context_of = context(0)
    in_threads(*[[lambda i=i: bind(i), lambda i=i: look(i)] for i in range(2)])
    assert seen == {i: streams[i].cuda_stream for i in range(2)}


def test_a_thread_that_never_bound_the_context_takes_the_last_binding(cuda):
    s, seen = torch.cuda.Stream(), []
    with torch.cuda.stream(s):
        ctx = context(0)
    t = threading.Thread(target=lambda: seen.append(stream_of(ctx)))
    t.start()
    t.join()
    assert seen == [s.cuda_stream]
    context(0)


def test_a_direct_binding_does_not_outlast_the_next_call(cuda):
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(a):
        ctx = context(0)
        _lib.call("at_ctx_set_stream", ctx, b.cuda_stream)
        assert stream_of(ctx) == b.cuda_stream
        context(0)
        assert stream_of(ctx) == a.cuda_stream
    context(0)


def test_clashing_bindings_heal(cuda):
    """Many rebindings at once: afterwards each thread still launches on its own stream."""
    streams = [torch.cuda.Stream() for _ in range(4)]
    wrong = []

    def work(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(3000):
                if stream_of(context(0)) != streams[i].cuda_stream:
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def split_batch(cuda, seed):
    """A cache whose one long sequence is split over blocks that a second kernel joins (a workspace), and its query."""
    cache = BlockKvCache.allocate(1, 150, 1, 64, 1, 150, 64, torch.float32)
    g = torch.Generator(device=cuda).manual_seed(seed)
    k, v = (torch.randn((9001, 1, 64), generator=g, device=cuda) for _ in range(2))
    cache.reserve(0, 9001)
    cache.append(0, TokenBatch.of([0], [0], [9001]), k, v)
    batch = TokenBatch.of([0], [9000], [1])
    need = C.c_size_t()
    _lib.call("at_kvb_attention_workspace", context(0), cache._refs[0], batch._ref, 4, 0, C.byref(need))
    assert need.value > 0
    return cache, batch, [torch.randn((1, 4, 64), generator=g, device=cuda) for _ in range(4)]


def test_threads_on_one_stream_do_not_share_a_workspace(cuda):
    """A call launches two kernels; another thread's may come between them."""
    cache, batch, qs = split_batch(cuda, 1)
    at = {}
    stream = torch.cuda.current_stream().cuda_stream

    def note(i):
        at[i] = cache._workspace(stream, 1 << 16).data_ptr()

    in_threads([lambda: note(0), lambda: note(0)], [lambda: note(1), lambda: note(1)])
    assert at[0] != at[1]


def test_attention_from_several_threads(cuda):
    cache, batch, qs = split_batch(cuda, 2)
    want = [cache.attention(0, batch, q) for q in qs]
    torch.cuda.synchronize()
    got = [[] for _ in qs]

    def work(i):
        for _ in range(300):
            got[i].append(cache.attention(0, batch, qs[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(qs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for w, ys in zip(want, got):
        assert len(ys) == 300 and all(torch.equal(w, y) for y in ys)


def test_split_attention_on_several_streams(cuda):
    """Different data on each stream: a workspace that two streams shared would mix them."""
    cache, batch, qs = split_batch(cuda, 3)
    want = [cache.attention(0, batch, q) for q in qs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in qs], []
    for _ in range(50):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, cache.attention(0, batch, qs[i])))
    torch.cuda.synchronize()
    assert all(torch.equal(want[i], y) for i, y in got)


def test_captured_split_attention_keeps_its_workspace(cuda):
    """Calls outside the graph, and memory freed and taken again after the capture, do not touch the graph's workspace."""
    cache, batch, qs = split_batch(cuda, 4)
    want = [cache.attention(0, batch, q) for q in qs]
    q = qs[0].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = cache.attention(0, batch, q)
    side = torch.cuda.Stream()
    for i in range(40):
        j = i % 4
        q.copy_(qs[j])
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            other = cache.attention(0, batch, qs[(j + 1) % 4])
            del_me = torch.full((1 << 20,), float("nan"), device=cuda)
        torch.cuda.synchronize()
        assert torch.equal(y, want[j]) and torch.equal(other, want[(j + 1) % 4])
        del del_me
