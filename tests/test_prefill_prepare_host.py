"""CPU tests of the scheduler's prefill preparation: which builder a batch goes to, and what it gets.

The engine, the backend and the uploads are stand-ins; only Scheduler's own code runs.
"""

from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest

from minisgl_b200.engine import scheduler as S


class _Backend:
    MAX_DEVICE_EXTEND = 8192
    device_extend = True

    def __init__(self):
        self.calls = []

    def prepare_metadata(self, batch):
        self.calls.append(("host", batch.size))


def _req(row, n, cached=0):
    return SimpleNamespace(table_idx=row, cached_len=cached, device_len=n, extend_len=n - cached,
                           input_ids=np.arange(n, dtype=np.int32))


def _batch(reqs):
    return SimpleNamespace(reqs=reqs, size=len(reqs), is_prefill=True, is_decode=False)


def _scheduler(table, page_size=4):
    be = _Backend()
    engine = SimpleNamespace(attn_backend=be, page_table=table, page_table_dev=object(), device="cpu")
    return SimpleNamespace(engine=engine, cfg=SimpleNamespace(page_size=page_size), graphs=None,
                           _stager=SimpleNamespace(upload=lambda arrays, device: list(arrays)),
                           _prepare_prefill_device=lambda batch: be.calls.append(("device", batch.size)))


@pytest.mark.parametrize("n,where", [(1, "device"), (8192, "device"), (8193, "host")])
def test_batches_past_the_device_tables_go_to_the_host_builder(n, where, monkeypatch):
    monkeypatch.setattr(S, "page_table_scatter", lambda *a: None)
    s = _scheduler(np.arange(n * 4, dtype=np.int32).reshape(n, 4))
    S.Scheduler._prepare(s, _batch([_req(b, 1) for b in range(n)]))
    assert s.engine.attn_backend.calls == [(where, n)]
