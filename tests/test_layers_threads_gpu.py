"""The layers called from several host threads."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def _in_thread(fn):
    """fn() on a new host thread; its result, or its exception here."""
    out = {}

    def work():
        try:
            out["value"] = fn()
        except BaseException as e:   # pylint: disable=broad-except
            out["error"] = e

    t = threading.Thread(target=work)
    t.start()
    t.join()
    if "error" in out:
        raise out["error"]
    return out["value"]


@pytest.mark.parametrize("m", [1, 24, 100, 300])
def test_first_cuda_call_of_a_host_thread(cuda, m):
    """Nothing has bound a context to the thread: its memory comes out of torch's cache."""
    from aimet_b200._lib import lib
    from aimet_b200.v2.nn import linear
    g = torch.Generator(device="cuda").manual_seed(101)
    n, k = 256, 512
    x = torch.randn(m, k, device=cuda, generator=g).bfloat16()
    w = torch.randn(n, k, device=cuda, generator=g).bfloat16()
    with torch.no_grad():
        want = linear(x, w)
        y = torch.empty_like(want)
        stream = torch.cuda.current_stream().cuda_stream
        assert _in_thread(lambda: lib.aq_linear_forward(x.data_ptr(), k, w.data_ptr(), k, None, None, 0, y.data_ptr(), n, None, 0, 2,
                                                        m, n, k, 0, stream)) == 0
        torch.cuda.synchronize()
        assert torch.equal(y, want)
    assert torch.equal(_in_thread(lambda: linear(x, w)), want)


def _race(jobs, calls):
    """Every job on a thread and a stream of its own; the foreign calls release the interpreter's lock."""
    gate = threading.Barrier(len(jobs))
    failed = []

    def work(job):
        stream = torch.cuda.Stream()
        gate.wait()
        for i in range(calls):
            rc = job(stream.cuda_stream)
            if rc:
                failed.append((i, rc))
                break
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(job,)) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return failed


def _check_race(jobs, outs):
    stream = torch.cuda.current_stream().cuda_stream
    want = []
    for job, out in zip(jobs, outs):
        assert job(stream) == 0
        want.append(out.clone())
    torch.cuda.synchronize()
    assert _race(jobs, 20000) == []
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("m", [64, 100])
def test_products_from_two_threads(cuda, m):
    """One kernel, called with its deep pipeline by one thread and with its shallow one by the other."""
    from aimet_b200._lib import lib
    g = torch.Generator(device="cuda").manual_seed(89)
    jobs, outs = [], []
    for n, k in ((512, 512), (25600, 64)):
        x = torch.randn(m, k, device=cuda, generator=g).bfloat16()
        w = torch.randn(n, k, device=cuda, generator=g).bfloat16()
        y = torch.empty(m, n, device=cuda, dtype=torch.bfloat16)

        def job(stream, x=x, w=w, n=n, k=k, y=y):
            return lib.aq_linear_forward(x.data_ptr(), k, w.data_ptr(), k, None, None, 0, y.data_ptr(), n, None, 0, 2, m, n, k, 0,
                                         stream)

        jobs.append(job)
        outs.append(y)
    _check_race(jobs, outs)


def test_norm_backward_from_two_threads(cuda):
    """One kernel on rows of different lengths."""
    from aimet_b200._lib import lib
    g = torch.Generator(device="cuda").manual_seed(97)
    jobs, outs = [], []
    for rows, dim in ((16, 2064), (16, 4096)):
        x, dy = (torch.randn(rows, dim, device=cuda, generator=g).bfloat16() for _ in range(2))
        mean, rstd = x.float().mean(1).contiguous(), x.float().var(1, unbiased=False).rsqrt().contiguous()
        dx = torch.empty(rows, dim, device=cuda, dtype=torch.bfloat16)

        def job(stream, x=x, dy=dy, mean=mean, rstd=rstd, rows=rows, dim=dim, dx=dx):
            return lib.aq_layer_norm_backward(x.data_ptr(), dim, dy.data_ptr(), dim, None, mean.data_ptr(), rstd.data_ptr(),
                                              dx.data_ptr(), None, None, 2, rows, dim, None, 0, stream)

        jobs.append(job)
        outs.append(dx)
    _check_race(jobs, outs)


def test_no_wait_ran_out_here(cuda):
    from aimet_b200.v2.nn import wait_ran_out
    assert wait_ran_out() is False and wait_ran_out(cuda) is False


def test_other_threads_run_while_launches_wait(cuda):
    """A call whose launch waits for room in the stream's queue does not keep the interpreter's lock."""
    import time
    from aimet_b200.v2.nn import layer_norm, linear
    x, w = torch.randn(4, 64, device=cuda), torch.randn(64, 64, device=cuda)
    with torch.no_grad():
        for fn in (lambda: linear(x, w), lambda: layer_norm(x, 64)):
            fn()
            torch.cuda.synchronize()
            done = threading.Event()
            gaps = []

            def tick(done=done, gaps=gaps):
                last = time.perf_counter()
                while not done.is_set():
                    time.sleep(0.001)
                    now = time.perf_counter()
                    gaps.append(now - last)
                    last = now

            t = threading.Thread(target=tick)
            t.start()
            start = time.perf_counter()
            torch.cuda._sleep(1_000_000_000)   # about half a second; the queue fills after some 1000 launches
            for _ in range(4000):
                fn()
            blocked = time.perf_counter() - start
            done.set()
            t.join()
            torch.cuda.synchronize()
            assert blocked > 0.3, "the queue never filled"
            assert max(gaps) < 0.3, max(gaps)


def test_saved_tensor_hooks_in_python(cuda):
    """Code in Python that a call reaches: what packs and unpacks the tensors kept for the backward pass."""
    from aimet_b200.v2.nn import layer_norm, linear
    x = torch.randn(20, 64, device=cuda, requires_grad=True)
    w = torch.randn(24, 64, device=cuda, requires_grad=True)
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(tuple(t.shape)) or t.cpu(), lambda t: t.to(cuda)):
        y = linear(layer_norm(x, 64), w, activation="gelu")
    got = torch.autograd.grad(y.sum(), (x, w))
    y = linear(layer_norm(x, 64), w, activation="gelu")
    assert len(seen) >= 5
    assert all(torch.equal(a, b) for a, b in zip(got, torch.autograd.grad(y.sum(), (x, w))))


def test_wait_ran_out_waits_for_every_stream(cuda):
    """torch's streams do not wait for the default one, nor it for them."""
    from aimet_b200.v2.nn import linear, wait_ran_out
    x, w = torch.randn(20, 64, device=cuda).half(), torch.randn(24, 64, device=cuda).half()
    stream = torch.cuda.Stream()
    linear(x, w)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(1_000_000_000)
        linear(x, w)
    assert not stream.query()
    assert wait_ran_out() is False
    assert stream.query()
