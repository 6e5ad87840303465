"""The bounded waits of the kernels' roles (csrc/tc_ptx.cuh): they end when their
barrier completes, after some 2 s when it never does, and soon after another
role of the CTA has failed; a warp's not while another has announced work."""

import pytest
import torch

from moe_fused_inference_b200 import _lib

pytestmark = pytest.mark.gpu


def test_waits_are_bounded_by_the_clock_and_by_the_cta():
    out = torch.zeros(16, dtype=torch.int64, device="cuda")
    lib = _lib.load()
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.mfi_selftest_waits(out.data_ptr(), stream) == 0, lib.mfi_last_error()
    torch.cuda.synchronize()
    for ok, ns, late, late_ns, failed, failed_ns, code in out[:14].view(2, 7).tolist():
        assert ok == 1 and ns < 10 ** 8
        assert late == 0 and code == 3 and 2 * 10 ** 9 <= late_ns < 3 * 10 ** 9
        assert failed == 0 and failed_ns < 5 * 10 ** 8
    ok, ns = out[14:].tolist()        # longer than the limit, while another role has work
    assert ok == 1 and 29 * 10 ** 8 <= ns < 4 * 10 ** 9
    assert _lib.device_error(clear=True) == 0
    assert lib.mfi_selftest_waits(None, stream) == 1
    assert lib.mfi_selftest_waits(out.data_ptr() + 4, stream) == 1
