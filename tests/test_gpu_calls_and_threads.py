"""Calls of the operators around the attention leave other threads free: a launch that waits for room in a full queue
holds nothing that they need."""
import threading
import time

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["gated_ffn", "qk_norm_rope", "pack8"])
def test_a_full_launch_queue_does_not_stop_other_threads(name):
    import dsalt_b200 as D
    x, w = torch.ones(4, 64, device="cuda"), torch.ones(64, 64, device="cuda")
    q, t = torch.ones(4, 1, 64, device="cuda"), torch.ones(4, 64, device="cuda")
    call = {"gated_ffn": lambda: D.gated_ffn(x, w, w, w), "qk_norm_rope": lambda: D.qk_norm_rope(q, q, t, t),
            "pack8": lambda: D.pack8(x)}[name]
    call()
    torch.cuda.synchronize()
    start = torch.cuda.Event()

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            torch.cuda._sleep(1_200_000_000)  # some 0.6 s on the device
            start.record()
            for _ in range(3000):             # more launches than the queue holds
                call()

    worker = threading.Thread(target=work)
    last, longest = time.perf_counter(), 0.0
    worker.start()
    while worker.is_alive():
        time.sleep(0.001)
        now = time.perf_counter()
        longest, last = max(longest, now - last), now
    worker.join()
    torch.cuda.synchronize()
    assert longest < 0.2, f"another thread stood still for {longest:.2f} s"


def test_calls_reach_what_is_written_in_python():
    """Without the lock: anomaly detection, hooks on saved tensors and a mode that sees every operation take it themselves."""
    import dsalt_b200 as D
    from torch.utils._python_dispatch import TorchDispatchMode
    x = torch.randn(40, 64, device="cuda").bfloat16().requires_grad_(True)
    w = [torch.randn(64, 64, device="cuda").bfloat16().mul_(0.1).requires_grad_(True) for _ in range(3)]
    n = torch.ones(64, device="cuda", requires_grad=True)
    t = torch.randn(40, 64, device="cuda")

    def step():
        y = D.gated_ffn(x, *w, keep="8bit").view(40, 1, 64)
        q, k = D.qk_norm_rope(y, y, t, t, q_weight=n, k_weight=n)
        return [q.detach(), *torch.autograd.grad((q, k), [x, *w, n], (q.detach(), k.detach()))]

    class Seen(TorchDispatchMode):
        names = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(str(func))
            return func(*args, **(kwargs or {}))

    ref = step()
    packed = []
    with torch.autograd.detect_anomaly(check_nan=False):
        runs = [step()]
    with torch.autograd.graph.saved_tensors_hooks(lambda s: packed.append(s) or s, lambda s: s):
        runs.append(step())
    with Seen():
        runs.append(step())
    assert packed and Seen.names
    for got in runs:
        assert all(torch.equal(a, b) for a, b in zip(got, ref))
    with pytest.raises(D.DsaltError):
        D.qk_norm_rope(torch.ones(4, 1, 20, device="cuda"), torch.ones(4, 1, 20, device="cuda"), t[:4, :20], t[:4, :20])


def test_two_threads_at_once():
    import dsalt_b200 as D

    def inputs(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        new = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16().mul_(0.2).requires_grad_(True)  # noqa: E731
        T = 300 + 200 * seed
        return [new(T, 128), new(264, 128), new(264, 128), new(64, 264)], torch.ones(64, device="cuda"), torch.randn(T, 64, device="cuda")

    def step(leaves, n, t):
        y = D.gated_ffn(*leaves).view(-1, 1, 64)
        q, k = D.qk_norm_rope(y, y, t, t, q_weight=n, k_weight=n)
        with torch.no_grad():
            z = D.gated_ffn(*leaves)
        return [q.detach(), z, *torch.autograd.grad((q, k), leaves, (q.detach(), k.detach())), *D.pack8(z)]

    sets = [inputs(i) for i in range(2)]
    ref = [step(*s) for s in sets]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                if not all(torch.equal(a, b) for a, b in zip(step(*sets[i]), ref[i])):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and D.device_status() == 0
