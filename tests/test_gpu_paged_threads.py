"""The paged cache's calls from one thread while another asks for what has been reported."""
import threading

import pytest
import torch

import lloom_amd as L

from . import paged_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, F32 = torch.float16, torch.float32


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("shape", [([30000], [2], 64, 1, 4, 64), ([6000], [90], 64, 2, 2, 64)])
def test_a_check_beside_calls_leaves_their_splits_alone(shape, act):
    """Calls whose requests are split among workgroups, on a stream of their own, with checks all the while."""
    s = R.case(*shape, act, device=DEV)

    def call():
        return L.paged_attention(s["q"], s["k"], s["v"], s["t_tables"], s["t_start"], s["t_lens"], out=torch.full_like(s["q"], 7.0))

    want = call()
    torch.cuda.synchronize()
    wrong, done = [], threading.Event()

    def serve():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    outs = [call() for _ in range(20)]
                    wrong.extend(i for i, o in enumerate(outs) if not torch.equal(o, want))
        except Exception as e:  # noqa: BLE001
            wrong.append(e)
        finally:
            done.set()

    thread = threading.Thread(target=serve)
    thread.start()
    checks = 0
    while not done.is_set():
        L.paged_check()
        checks += 1
    thread.join()
    assert not wrong and checks > 0
    assert torch.equal(call(), want)
