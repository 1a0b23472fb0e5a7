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
