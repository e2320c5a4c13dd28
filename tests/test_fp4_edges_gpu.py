"""The 4-bit KV pool at the ends of its ranges: signed zeros, infinite and NaN queries, pool scales and
work lists far from the usual.
"""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from helpers import HeadConfig, rand, to_dev, torch_dtype
from minisgl_b200 import workloads as W
from oracle import fp4 as F

pytestmark = pytest.mark.gpu


def _device_error() -> int:
    import torch

    from minisgl_b200 import _native as nat

    code = ctypes.c_int(-1)
    nat.call("b2a_device_error", torch.cuda.current_stream().cuda_stream, ctypes.byref(code))
    return code.value


def _i32(a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_negative_zero_keeps_its_sign(dtype):
    """-0.0 beside values of any size, and negative values whose code is zero, have code 8."""
    from minisgl_b200 import FP4KVCache

    x = np.zeros((6, 1, 64), np.float32)
    x[:, 0, ::3] = -0.0
    for t, top in enumerate((6.0, -1.0, 0.01, 448.0, 2688.0, 0.0)):  # the last row has no live block
        x[t, 0, 1::16] = top
        x[t, 0, 2::16] = -abs(top) * 2.0 ** -9
    c = FP4KVCache(1, 6, 1, 64, torch_dtype(dtype), "cuda")
    kd = to_dev(x, dtype)
    c.store_kv(kd, -kd, _i32(np.arange(6)), 0)
    k = kd.double().cpu().numpy()
    assert np.signbit(k[k == 0]).sum() > 100
    np.testing.assert_array_equal(c.rows(0).cpu().numpy(), F.pack_rows(k, -k))
    assert _device_error() == 0
