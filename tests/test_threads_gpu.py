"""Calls from threads that have made no CUDA call of their own."""
import threading

import pytest
import torch

from dice_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("call", ["grouped_gemm", "grouped_dgrad", "grouped_wgrad", "grouped_ffn_train"])
def test_first_cuda_call_of_a_thread(cuda_device, call):
    """Autograd runs backward passes in a thread of its own, and memory comes from torch's cache: the kernel's tensor maps
    may be the thread's first contact with the driver."""
    x = torch.randn(300, 128, device=cuda_device, dtype=torch.bfloat16)
    w = torch.randn(1, 128, 128, device=cuda_device, dtype=torch.bfloat16)
    seg = torch.tensor([0, 300], dtype=torch.int32, device=cuda_device)
    status = ops.device_status(cuda_device)
    calls = {
        "grouped_gemm": lambda: ops.grouped_gemm(x, w, seg, ops.EPI_STORE, 128, status),
        "grouped_dgrad": lambda: ops.grouped_dgrad(x, w, seg),
        "grouped_wgrad": lambda: ops.grouped_wgrad(x, x, seg),
        "grouped_ffn_train": lambda: ops.grouped_ffn_train(x, w, w, seg, "gelu_tanh", 128)[0],
    }
    want = calls[call]()
    torch.cuda.synchronize()
    got = []

    def work():
        try:
            got.append(calls[call]())
        except Exception as e:  # carried to the test's thread
            got.append(e)

    for _ in range(2):  # the second thread finds the first one's memory in the cache
        thread = threading.Thread(target=work)
        thread.start()
        thread.join()
        if isinstance(got[-1], Exception):
            raise got[-1]
        assert torch.equal(got.pop(), want)
