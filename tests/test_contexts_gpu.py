"""Entry points that build tensor maps leave the calling thread's CUDA context as they find it."""
import ctypes as C
import threading

import pytest
import torch

from lego_b200 import _abi, ops

pytestmark = pytest.mark.gpu


def _refused_at_the_tensor_maps(x):
    """The status of a call that gets as far as building its tensor maps and is refused there: a stride of 2^41
    bytes is past what they hold (of an axis of one, so that no address follows from it).  Nothing is launched."""
    d = _abi.Attention(dtype=_abi.F16, batch=1, q_len=4, k_len=4, q_heads=1, k_heads=1, head_dim=64, scale=0.1)
    for s in (d.q_stride, d.k_stride, d.v_stride):
        s[:] = (1 << 40, 64, 64)
    return _abi.lib().lego_attention_fwd(C.byref(d), *(x.data_ptr(),) * 4, None, x.data_ptr(), x.data_ptr(), 4096, None)


def test_a_context_of_the_callers_own_stays_current():
    x = torch.zeros(256, 256, device="cuda", dtype=torch.float16)
    ops.matmul(x, x)                            # the device's workspace is there
    torch.cuda.synchronize()
    assert _refused_at_the_tensor_maps(x) == -8
    cu = C.CDLL("libcuda.so.1")
    seen = {}

    def work():
        own, now, dev = C.c_void_p(), C.c_void_p(), C.c_int()
        seen["made"] = cu.cuDeviceGet(C.byref(dev), torch.cuda.current_device()) or cu.cuCtxCreate_v2(C.byref(own), 0, dev)
        if seen["made"]:
            return
        try:
            seen["status"] = _refused_at_the_tensor_maps(x)
            cu.cuCtxGetCurrent(C.byref(now))
            seen["kept"] = now.value == own.value
        finally:
            cu.cuCtxDestroy_v2(own)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert seen["made"] == 0 and seen["status"] == -8
    assert seen["kept"]
    torch.cuda.synchronize()


def test_a_thread_without_a_context_gets_the_primary_one():
    x = torch.zeros(256, 256, device="cuda", dtype=torch.float16)
    ops.matmul(x, x)
    torch.cuda.synchronize()
    got = []
    t = threading.Thread(target=lambda: got.append(_refused_at_the_tensor_maps(x)))
    t.start()
    t.join()
    assert got == [-8]
