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
