"""What a stream's workspace takes of the device's free memory, as hipMemGetInfo reports it."""
from __future__ import annotations

import ctypes

import pytest

import flash_attention_amd as fa
from test_zz_no_alloc import PAIRS, _tensors, _workspace

pytestmark = pytest.mark.gpu


def hip_runtime():
    """The HIP runtime that this process has loaded."""
    with open("/proc/self/maps") as f:
        return ctypes.CDLL(next(line.split()[-1] for line in f if "libamdhip64" in line))


def test_a_workspace_takes_its_size_whatever_was_allocated_before():
    """The free memory that is reported falls by a workspace's size at least, also where the report is a unit of
    2 MiB short (once in 1000 MiB of allocations of 50 MiB).  Other allocations in steps of 40 MiB, smaller than the
    workspace of 48.25 MiB, move it over more than 1000 MiB."""
    import torch

    fa.init()
    variant, bh, sq, sk, d, causal, path, splits = case = PAIRS[2][0]
    q, k, v = _tensors(bh, sq, sk, d, 1)
    out, ws = torch.empty(bh * sq * d, device="cuda"), _workspace(*case)
    hip, ballast, stream = hip_runtime(), [], torch.cuda.current_stream().cuda_stream

    def run():
        fa.attention_device(variant, q.data_ptr(), k.data_ptr(), v.data_ptr(), 1, bh, sq, sk, d, causal, out.data_ptr(),
                            stream, path=path, num_splits=splits)
        torch.cuda.synchronize()

    run()
    falls = []
    try:
        for _ in range(27):
            fa.release_stream_workspace(stream)
            p = ctypes.c_void_p()
            assert hip.hipMalloc(ctypes.byref(p), ctypes.c_size_t(40 << 20)) == 0
            ballast.append(p)
            before = torch.cuda.mem_get_info()[0]
            run()
            falls.append(before - torch.cuda.mem_get_info()[0])
    finally:
        for p in ballast:
            assert hip.hipFree(p) == 0
    print(f"workspace {ws}: free memory fell by {sorted(set(falls))}", flush=True)
    assert min(falls) >= ws
