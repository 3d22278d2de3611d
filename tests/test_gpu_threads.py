"""GPU: calls of several host threads, each on its own stream."""
import threading

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _in_thread(f):
    out = []
    t = threading.Thread(target=lambda: out.append(f()))
    t.start()
    t.join()
    return out[0]


@pytest.fixture
def no_follow(gpu):
    """Calls go to the stream that set_stream selected, not to torch's current one."""
    gpu.follow_torch_stream(False)
    yield gpu
    gpu.follow_torch_stream(True)
    gpu.set_stream(None)


def _operands():
    import torch

    rng = np.random.default_rng(0)
    x = torch.from_numpy(rng.standard_normal((2, 256)).astype(np.float32)).cuda()
    return rng, x, torch.zeros((2, 64), device="cuda")


@pytest.mark.parametrize("kind", ["4-bit linear", "linear"])
def test_a_call_runs_on_the_stream_its_thread_selected(no_follow, kind):
    """Another thread selects its stream between this thread's selection and its call.  The call is
    captured by this thread's stream: one that went elsewhere would have run at once."""
    import torch

    gpu = no_follow
    rng, x, y = _operands()
    w = rng.standard_normal((64, 256)).astype(np.float32)
    if kind == "linear":
        W, go = gpu.Weight(w), lambda: gpu.linear(y, x, W, sync=False)
    else:
        W = gpu.Q4Weight(*gpu.quantize_q4(w, 64), K=256, group=64)
        go = lambda: gpu.linear_q4(y, x, W, sync=False)  # noqa: E731
    mine, other = torch.cuda.Stream(), torch.cuda.Stream()
    gpu.set_stream(mine.cuda_stream)
    go()  # workspaces are there before the capture
    mine.synchronize()
    want = y.cpu().numpy()
    y.zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=mine):
        gpu.set_stream(mine.cuda_stream)
        _in_thread(lambda: gpu.set_stream(other.cuda_stream))
        go()
    torch.cuda.synchronize()
    assert (y.cpu().numpy() == 0).all()
    graph.replay()
    torch.cuda.synchronize()
    assert np.array_equal(y.cpu().numpy(), want) and np.abs(want).max() > 0


def test_a_thread_without_a_selection_uses_the_last_one(no_follow):
    import torch

    gpu = no_follow
    rng, x, y = _operands()
    W = gpu.Q4Weight(*gpu.quantize_q4(rng.standard_normal((64, 256)).astype(np.float32), 64), K=256, group=64)
    mine = torch.cuda.Stream()
    gpu.set_stream(mine.cuda_stream)
    gpu.linear_q4(y, x, W)  # the kernel is loaded before the capture
    y.zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=mine):
        gpu.set_stream(mine.cuda_stream)
        _in_thread(lambda: gpu.linear_q4(y, x, W, sync=False))
    torch.cuda.synchronize()
    assert (y.cpu().numpy() == 0).all()
    graph.replay()
    torch.cuda.synchronize()
    assert np.abs(y.cpu().numpy()).max() > 0


def test_threads_with_streams_of_their_own_get_their_results(gpu):
    """Chains of calls of four threads, interleaved: each equals the same chain alone, bit for bit."""
    import torch

    rng = np.random.default_rng(1)
    n, steps = 512, 40
    W = gpu.Q4Weight(*gpu.quantize_q4((rng.standard_normal((n, n)) / n ** 0.5).astype(np.float32), 128), K=n, group=128)
    start = [torch.from_numpy(rng.standard_normal((3, n)).astype(np.float32)).cuda() for _ in range(4)]

    def chain(x):
        with torch.cuda.stream(torch.cuda.Stream()) as _:
            s = torch.cuda.current_stream()
            y = torch.empty_like(x)
            a, b = x.clone(), y
            for _ in range(steps):
                gpu.linear_q4(b, a, W, sync=False)
                a, b = b, a
            s.synchronize()
            return a.cpu().numpy()

    torch.cuda.synchronize()
    alone = [chain(x) for x in start]
    got = [None] * 4
    threads = [threading.Thread(target=lambda i=i: got.__setitem__(i, chain(start[i]))) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(alone, got):
        assert np.isfinite(a).all() and np.array_equal(a, b)


def test_operands_have_to_live_where_the_library_runs(gpu):
    L = gpu.lib()
    assert L.envg_use_device(0, 0, None) == gpu.OK
    for device in (1, -1):
        assert L.envg_use_device(device, 1, None) == gpu.ERR_ARG and "device" in gpu.last_error()
