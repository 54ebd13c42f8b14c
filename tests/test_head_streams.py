"""One ``UnembedHead`` on several streams and threads: a layout that one stream still makes is waited for by the calls of the
others, and a layout waits for the calls that still use the last one (``tsc_unembed_*``, ``lm_head.model_head``).

A stream is kept busy in front of a layout, so that a call that did not wait would find memory that nothing has been laid out in."""
import threading

import pytest
import torch

from test_lm_head import model_of, tokens_of
from test_unembed import DEV, make, run

TICKS = []
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def keep_busy(ms=100.0):
    """The current stream waits for about that long (a warm call takes 50 us, making a head some milliseconds)."""
    if not TICKS:
        torch.cuda._sleep(1000)
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        torch.cuda._sleep(1_000_000)
        end.record()
        end.synchronize()
        TICKS.append(1_000_000 / begin.elapsed_time(end))
    torch.cuda._sleep(int(ms * TICKS[0]))


def same(got, want):
    assert set(got) == set(want)
    for k in want:
        assert torch.equal(got[k], want[k]), k


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tied", [False, True])
def test_a_new_head_on_another_stream(tied, dtype):
    import tsc_hip

    x, W, b, t, dloss = make(100, 72, 1999, dtype, tied=tied, ignored=0.1, seed=61)
    run(x, W * 2, b, t, dloss)  # (the kernels are loaded)
    a, c = torch.cuda.Stream(), torch.cuda.Stream()
    keep_busy(1)
    torch.cuda.synchronize()
    with torch.cuda.stream(a):
        keep_busy()
        head = tsc_hip.UnembedHead(W, b)
        laid = torch.cuda.Event()
        laid.record()
    with torch.cuda.stream(c):
        got = run(x, W, b, t, dloss, head=head)
    assert not laid.query(), "the layout was to be under way"
    torch.cuda.synchronize()
    same(got, run(x, W, b, t, dloss))
    with torch.cuda.stream(c):
        same(run(x, W, b, t, dloss, head=head), got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_weights_changed_on_a_third_stream(dtype):
    import tsc_hip

    x, W, b, t, dloss = make(100, 72, 1999, dtype, seed=62)
    head = tsc_hip.UnembedHead(W, b)
    run(x, W, b, t, dloss, head=head)
    torch.cuda.synchronize()
    change, *users = [torch.cuda.Stream() for _ in range(4)]
    for k in (0.5, 1.75):
        with torch.cuda.stream(change):
            for u in users:  # they still read W
                change.wait_stream(u)
            keep_busy()
            W.mul_(k)
            b.add_(k)
        got = []
        for u in users:
            u.wait_stream(change)
            with torch.cuda.stream(u):
                got.append(run(x, W, b, t, dloss, head=head))
        torch.cuda.synchronize()
        want = run(x, W, b, t, dloss)
        for g in got:
            same(g, want)


@pytest.mark.gpu
def test_a_layout_waits_for_the_calls_before_it():
    import tsc_hip

    x, W, b, t, dloss = make(100, 72, 1999, torch.float32, seed=63)
    head = tsc_hip.UnembedHead(W, b)
    want = run(x, W, b, t, dloss)
    a, c = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    used = torch.cuda.Event()
    with torch.cuda.stream(c):
        keep_busy()
        got = run(x, W, b, t, dloss, head=head)
        used.record()
    with torch.cuda.stream(a):
        head.refresh()
    assert not used.query(), "the call was to be under way"
    a.synchronize()
    assert used.query()
    same(got, want)


@pytest.mark.gpu
def test_threads_with_streams_of_their_own():
    import tsc_hip

    x, W, b, t, dloss = make(100, 72, 1999, torch.float32, seed=64)
    head = tsc_hip.UnembedHead(W, b)
    start, failed = threading.Barrier(4), []
    got = [None] * 4

    def work(i):
        try:
            stream = torch.cuda.Stream()
            for k in range(3):
                start.wait(30)
                if i == 0:
                    keep_busy()
                    W.mul_(0.9)
                    torch.cuda.synchronize()
                start.wait(30)
                with torch.cuda.stream(stream):
                    got[i] = run(x, W, b, t, dloss, head=head)
                stream.synchronize()
                start.wait(30)
                if i == 0:
                    want = run(x, W, b, t, dloss)
                    for g in got:
                        same(g, want)
        except BaseException as e:  # noqa: BLE001 -- told by the main thread
            failed.append(e)
            start.abort()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join(60)
    real = [e for e in failed if not isinstance(e, threading.BrokenBarrierError)]
    assert not failed, real or failed


@pytest.mark.gpu
def test_a_model_on_several_streams():
    m = model_of(DEV)
    tok = tokens_of(m)
    for _ in range(2):
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(3)]
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                if i == 0:
                    keep_busy()
                got.append(m(tok, return_type="loss", loss_per_token=True))
        torch.cuda.synchronize()
        want = m(tok, return_type="loss", loss_per_token=True)
        assert all(torch.equal(g, want) for g in got)
        torch.cuda.synchronize()
        m.W_U.mul_(1.25)


@pytest.mark.gpu
def test_a_capture_while_the_layout_runs_is_refused():
    import tsc_hip

    x, W, b, t, dloss = make(100, 72, 1999, torch.bfloat16, seed=65)
    a, c = torch.cuda.Stream(), torch.cuda.Stream()
    head = tsc_hip.UnembedHead(W, b)
    keep_busy(1)  # (not measured inside a capture)
    some = torch.zeros(4, device=DEV)
    for call in (lambda: head.loss(x, t), lambda: head.loss_backward(dloss, x, t, dloss), head.refresh):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(c):
            g.capture_begin()
            try:
                some.add_(1)
                with torch.cuda.stream(a):  # eager work beside the capture (whose beginning may take longer than the wait)
                    keep_busy()
                    head.refresh()
                with pytest.raises(tsc_hip.TscError, match="synchronize"):
                    call()
            finally:
                g.capture_end()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):  # (which synchronizes)
        out = run(x, W, b, t, dloss, head=head)
    want = run(x, W, b, t, dloss)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        same(out, want)


@pytest.mark.gpu
def test_streams_that_are_not_torchs_are_not_kept():
    """Their owner may destroy them; a torch stream is there for good."""
    import tsc_hip

    x, W, b, t, dloss = make(100, 72, 1999, torch.float32, seed=66)
    head = tsc_hip.UnembedHead(W, b)
    want = run(x, W, b, t, dloss)
    pooled = torch.cuda.Stream()
    outside = torch.cuda.ExternalStream(torch.cuda.Stream().cuda_stream)
    torch.cuda.synchronize()
    for s, kept in ((torch.cuda.current_stream(), True), (pooled, True), (outside, False)):
        with torch.cuda.stream(s):
            same(run(x, W, b, t, dloss, head=head), want)
        assert (s.cuda_stream in head._users) == kept
    head.refresh()
    assert not head._users
    same(run(x, W, b, t, dloss, head=head), want)
