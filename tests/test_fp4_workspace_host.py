"""CPU tests of the workspace that an extend over the 4-bit pool asks for."""

from __future__ import annotations

import numpy as np
import pytest

from minisgl_b200 import _native as nat

MB = 1 << 20


def _plan(keys, Hkv, sms=148):
    """run_keys and n_split as b2a_fp4_extend_runs proposes them on a GPU of ``sms`` SMs, restated."""
    nb = np.maximum(1, -(-np.asarray(keys) // 128))
    slots = sms // Hkv
    if slots <= len(nb) or nb.max() <= 4:
        return 0, 1
    run = max(4, -(-int(nb.sum()) // slots), -(-int(nb.max()) // 64))
    while run < nb.max() and (-(-nb // run)).sum() > slots:
        run += 1
    return (run * 128, int(-(-nb.max() // run))) if run < nb.max() else (0, 1)


@pytest.mark.parametrize("Hkv,keys", [(1, [300] * 83 + [32768]), (2, [300] * 36 + [16384]), (8, [100] * 9 + [16000])])
@pytest.mark.parametrize("D,dtype", [(128, 1), (256, 1), (64, 0), (128, 0)])
def test_one_long_request_among_short_ones(Hkv, keys, D, dtype):
    """The batch's own runs fill the SMs once; the workspace holds those, not every item's longest cut."""
    run_keys, n_split = _plan(keys, Hkv)
    assert n_split > 1
    got = nat.fp4_extend_workspace(np.array(keys), len(keys), run_keys, n_split, Hkv, D, dtype)
    rows = 256 if dtype == 1 and D <= 128 else 128
    runs = sum(n for n in (min(n_split, -(-k // run_keys)) for k in keys) if n > 1)
    assert runs * Hkv <= 148
    assert got <= max(64 * MB, 148 * rows * (D + 2) * 4 + 4096)
    assert got >= 4 * len(keys) * Hkv + runs * Hkv * rows * (D + 2) * 4


def test_even_batches_keep_a_place_for_every_run():
    keys = [9000, 12000, 8000, 16000]
    run_keys, n_split = _plan(keys, 8)
    assert nat.fp4_extend_workspace(np.array(keys), 4, run_keys, n_split, 8, 128, 1) == \
        nat.LIB.b2a_fp4_extend_workspace_bytes(4, n_split, 8, 128)
    assert nat.fp4_extend_workspace(np.array(keys), 4, 0, 1, 8, 128, 1) == 0


def test_packed_bytes():
    f = nat.LIB.b2a_fp4_extend_packed_bytes
    assert f(8, 1, 8, 128, 1) == 0 and f(0, 4, 8, 128, 1) == 0
    assert f(8, 4, 8, 128, 1) == 256 + 4 * 8 * 256 * 130 * 4
    assert f(80, 4, 1, 256, 1) == 512 + 4 * 128 * 258 * 4
    assert f(8, 4, 8, 128, 0) == 256 + 4 * 8 * 128 * 130 * 4
