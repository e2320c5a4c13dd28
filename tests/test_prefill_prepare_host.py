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

    def extend_tiles(self, cached, lens):
        return int(sum(-(-(n - c) // 3) for c, n in zip(cached, lens)))

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


class _Tables:
    """Stands in for the metadata that the device fills."""

    positions = out_loc = "device"


def _device_scheduler(table, monkeypatch, page_size=4):
    s = _scheduler(table, page_size)
    monkeypatch.setattr(S, "page_table_scatter", lambda *a: None)
    be = s.engine.attn_backend
    be.alloc_extend_metadata = lambda *a, **kw: be.calls.append((a, kw)) or _Tables()
    be.build_extend_metadata_device = lambda *a: None
    return s


@pytest.mark.parametrize("bad", [None, "broken run", "slot of another page"])
def test_the_metadata_check_covers_device_built_tables(bad, monkeypatch):
    """Every page has to be an aligned run of slots, also where its first slot, all the kernel sees, is right."""
    table = np.concatenate([np.arange(8, 16), np.arange(32, 40)]).astype(np.int32).reshape(2, 8)
    if bad == "broken run":
        table[1, 5:7] = table[1, [6, 5]]
    elif bad:
        table[0, 5] = 60
    s = _device_scheduler(table, monkeypatch)
    monkeypatch.setattr(S, "CHECK_METADATA", True, raising=False)
    batch = _batch([_req(0, 6, 2), _req(1, 8)])
    if bad is None:
        S.Scheduler._prepare_prefill_device(s, batch)
    else:
        with pytest.raises(ValueError, match="aligned runs"):
            S.Scheduler._prepare_prefill_device(s, batch)


def test_device_built_tables_keep_the_host_offsets(monkeypatch):
    """q_offsets, a field of the prefill metadata that a model may read, as the host builder gives it."""
    s = _device_scheduler(np.arange(24, dtype=np.int32).reshape(3, 8), monkeypatch)
    batch = _batch([_req(0, 6, 2), _req(1, 8), _req(2, 7, 6)])
    S.Scheduler._prepare_prefill_device(s, batch)
    assert batch.attn_metadata.q_offsets == [0, 4, 12, 13]


def test_device_built_tables_hold_the_batch_s_own_tiles(monkeypatch):
    """No empty tiles behind the work list of a batch whose lengths are known here: ceil(4/3) + ceil(8/3) + 1."""
    s = _device_scheduler(np.arange(24, dtype=np.int32).reshape(3, 8), monkeypatch)
    S.Scheduler._prepare_prefill_device(s, _batch([_req(0, 6, 2), _req(1, 8), _req(2, 7, 6)]))
    (args, kw), = s.engine.attn_backend.calls
    assert args == (3, 13, 6) and kw["n_work"] == 6
