"""Calls of the low-rank adapters from several host threads."""

import threading

import pytest
import torch

from aihwkit_b200 import _cabi
from tests.test_digital_gpu import rand

pytestmark = pytest.mark.gpu


def test_launches_of_two_threads_do_not_disturb_each_other():
    """Calls of one kernel with more and with less shared memory, issued by two host threads at once."""
    lib = _cabi.lib()
    rows, k, n = 64, 64, 64
    failed = []

    def work(rank):
        x, y = rand((rows, k), torch.float32, rank), torch.zeros(rows, n, device="cuda")
        a, b = rand((1, rank, k), torch.float32, 1), rand((1, rank, n), torch.float32, 2)
        scale, ids = torch.ones(1, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
        starts = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        for i in range(3000):
            code = lib.ab200_low_rank_apply(x.data_ptr(), k, None, 0, y.data_ptr(), n, a.data_ptr(), b.data_ptr(), scale.data_ptr(),
                                            ids.data_ptr(), starts.data_ptr(), 1, rows, k, n, rank, 1, 0, None, stream.cuda_stream)
            if code != 0:
                failed.append((rank, i, lib.ab200_last_error().decode()))
                return
            if i % 500 == 499:
                stream.synchronize()

    threads = [threading.Thread(target=work, args=(rank,)) for rank in (40, 256)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
