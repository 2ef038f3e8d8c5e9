"""The ragged step's split operators in CUDA graphs: every graph's workspace is its own and is
zeroed by the graph, so graphs captured on one stream may be replayed in any order, at the
same time on two streams, and beside eager calls on the stream that they were captured on."""
import gc

import pytest
import torch

from gqa_kernels import check_device_error, paged_ragged_attention, verify_drafts, verify_drafts_greedy
from tests._serving import cu_of, paged_batch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib_ready(cuda_lib):
    check_device_error()
    yield
    torch.cuda.synchronize()
    assert check_device_error() == (0, 0)


def attention_call(reqs, seed):
    q, kc, vc, bt, cu, lens = paged_batch(reqs, 8, 2, 128, 64, torch.bfloat16, seed)
    out = torch.empty_like(q)
    bounds = dict(max_query_len=max(x for x, _ in reqs), max_seq_len=max(sum(r) for r in reqs))
    return lambda: paged_ragged_attention(q, kc, vc, bt, cu, lens, out=out, **bounds), [out]


def verify_call(n, k, vocab, greedy, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    target = torch.rand(n * (k + 1), vocab, generator=g, device="cuda")
    drafts = torch.randint(0, vocab, (n, k), generator=g, device="cuda", dtype=torch.int32)
    uniforms = torch.rand(n, k, generator=g, device="cuda")
    expo = torch.empty(n, vocab, device="cuda").exponential_(generator=g)
    out = (torch.empty(n, k + 1, dtype=torch.int32, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda"))
    cu = cu_of([k + 1] * n)
    if greedy:
        return lambda: verify_drafts_greedy(drafts, target, cu, out=out), list(out)
    return lambda: verify_drafts(drafts, target, None, uniforms, expo, cu, out=out), list(out)


# Split keys in the streaming form, in the tcgen05 form, in both at once, and the two verifications.
CALLS = [lambda: attention_call([(1, 9000), (3, 4100)], 1), lambda: attention_call([(40, 16000)], 2),
         lambda: attention_call([(1, 12000), (7, 3000), (300, 2000)], 3), lambda: verify_call(3, 4, 50000, False, 4),
         lambda: verify_call(2, 3, 90000, True, 5)]


def wipe(outs):
    for o in outs:
        o.fill_(-7)


def dirty_pool():
    """A graph memory pool whose free memory holds 0xff bytes."""
    pool = torch.cuda.graph_pool_handle()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, pool=pool):
        for size in (1 << 16, 1 << 20, 64 << 20):
            torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    graph.replay()
    torch.cuda.synchronize()
    return pool, graph


@pytest.mark.parametrize("first", range(len(CALLS)))
@pytest.mark.parametrize("second", range(len(CALLS)))
def test_the_graph_captured_second_is_replayed_first(first, second):
    pool, keep = dirty_pool()
    calls = [CALLS[first](), CALLS[second]()]
    want, graphs = [], []
    for call, outs in calls:
        call()
        want.append([o.clone() for o in outs])
        wipe(outs)
    for call, _ in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=pool):
            call()  # once: a second call of the same shape would join the first one's partials
    for i in (1, 0, 0, 1):
        graphs[i].replay()
        assert all(torch.equal(o, w) for o, w in zip(calls[i][1], want[i])), i
        wipe(calls[i][1])


def test_two_graphs_of_one_stream_at_the_same_time():
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    calls = [attention_call([(1, 16000)] * 6, 6), attention_call([(1, 16000)] * 6, 7)]
    want, graphs = [], []
    for call, outs in calls:
        call()
        want.append(outs[0].clone())
        wipe(outs)
    torch.cuda.synchronize()
    for call, _ in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            for _ in range(8):
                call()
    for _ in range(10):
        with torch.cuda.stream(side):
            graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
        torch.cuda.synchronize()
        for (_, outs), w in zip(calls, want):
            assert torch.equal(outs[0], w)
            wipe(outs)
        torch.cuda.synchronize()


def test_eager_calls_on_a_stream_that_was_captured():
    """The first call on a stream is captured; eager ones follow on it before any replay, then
    both in turn, after the graph is gone too."""
    pool, keep = dirty_pool()
    side = torch.cuda.Stream()
    call, outs = CALLS[2]()
    call()
    want = outs[0].clone()
    wipe(outs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, pool=pool, stream=side):
        call()
    with torch.cuda.stream(side):
        for replay in (False, False, True, False, True):
            if replay:
                graph.replay()
            else:
                call()
            assert torch.equal(outs[0], want)
            wipe(outs)
        side.synchronize()
        del graph
        gc.collect()
        for _ in range(2):
            call()
            assert torch.equal(outs[0], want)
            wipe(outs)


def test_workspaces_of_graphs_that_are_gone_are_freed():
    """Capturing again and again does not keep memory: a graph's workspace goes with it."""
    call, outs = attention_call([(1, 16000)] * 8, 8)  # more than 4 MB of partials
    call()
    torch.cuda.synchronize()
    used = []
    for _ in range(12):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        graph.replay()
        torch.cuda.synchronize()
        del graph
        gc.collect()
        torch.cuda.synchronize()
        call()  # frees what the graphs have left
        torch.cuda.synchronize()
        used.append(torch.cuda.memory_allocated())
    assert used[-1] <= used[3]


def test_a_forked_capture_has_a_workspace_per_stream():
    fork = torch.cuda.Stream()
    calls = [attention_call([(1, 16000)] * 6, 9), attention_call([(40, 16000)], 10)]
    want = []
    for call, outs in calls:
        call()
        want.append(outs[0].clone())
        wipe(outs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fork.wait_stream(torch.cuda.current_stream())
        for _ in range(6):
            calls[0][0]()
            with torch.cuda.stream(fork):
                calls[1][0]()
        torch.cuda.current_stream().wait_stream(fork)
    for _ in range(5):
        graph.replay()
        torch.cuda.synchronize()
        for (_, outs), w in zip(calls, want):
            assert torch.equal(outs[0], w)
            wipe(outs)
