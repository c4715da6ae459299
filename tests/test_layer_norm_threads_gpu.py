"""Layer norm's backward called from several host threads, with widths that share a kernel instance."""
import threading

import pytest
import torch

from subq_audio import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,widths", [(torch.float32, (3200, 3584, 4096)), (torch.float32, (1280, 1536)), (torch.bfloat16, (4352, 6144)),
                                          (torch.float32, (4104, 8192))])
def test_two_widths_of_one_instance_at_once(dtype, widths):
    """The kernels ask for different amounts of shared memory: no call may lower the limit that another one needs."""
    g = torch.Generator(device="cuda").manual_seed(widths[0])
    jobs = []
    for D in widths + widths:
        x, dy = (torch.randn(8, D, generator=g, device="cuda").to(dtype) for _ in range(2))
        jobs.append((dy, x, torch.randn(D, generator=g, device="cuda")))
    want = [ops.layer_norm_backward(*job) for job in jobs]
    torch.cuda.synchronize()
    errors, start = [], threading.Barrier(len(jobs))

    def work(i):
        start.wait()
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for n in range(1500):
                    got = ops.layer_norm_backward(*jobs[i], need_dweight=n % 3 > 0, need_dbias=n % 3 > 0)
                    if n % 100 < 2:
                        assert all(a is None or torch.equal(a, b) for a, b in zip(got, want[i]))
        except Exception as e:  # noqa: BLE001 (reported by the test's own thread)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors[:3]
