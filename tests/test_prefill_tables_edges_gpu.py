"""Device-built prefill tables (b2a_extend_metadata) where a batch is smaller than its buffers, does
not fit them or names rows that do not exist: what a store and an attention call behind them do.
"""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from helpers import HeadConfig, rand, to_dev, torch_dtype
from minisgl_b200 import workloads as W

pytestmark = pytest.mark.gpu

HQ, HKV, D, P = 16, 8, 128, 16


def _device_error() -> int:
    import torch

    from minisgl_b200 import _native as nat

    code = ctypes.c_int(-1)
    nat.call("b2a_device_error", torch.cuda.current_stream().cuda_stream, ctypes.byref(code))
    return code.value


def _i32(a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def _cache(pool, n, dtype="bfloat16"):
    from minisgl_b200 import FP4KVCache, MHAKVCache

    return (FP4KVCache if pool == "fp4" else MHAKVCache)(1, n, HKV, D, torch_dtype(dtype), "cuda")


def _backend(lens, pool="fp4", dtype="bfloat16"):
    from minisgl_b200 import B200AttnBackend

    lens = np.asarray(lens)
    rng = np.random.default_rng(int(lens.sum()))
    pb = W.allocate_pages(lens, (int(((lens + P - 1) // P).sum()) + 4) * P, P, rng)
    cache = _cache(pool, pb.num_slots, dtype)
    return B200AttnBackend(HeadConfig(HQ, HKV, D), cache, pb.page_table, P), pb, rng


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("pool", ["fp4", "dense"])
def test_a_captured_step_stores_its_own_batch_only(pool, dtype):
    """Tables, store and extend captured once at full capacity: a replay with fewer tokens leaves
    every other slot of the pool as it was, byte for byte, and attends as the eager call does."""
    import torch

    cap = np.array([200, 96, 40, 130])
    be, pb, rng = _backend(cap, pool, dtype)
    cache, T = be.kv_cache, int(cap.sum())
    meta = be.alloc_extend_metadata(4, T, int(((cap + P - 1) // P).sum()))
    table, rows = _i32(pb.page_table), _i32(pb.rows)
    cached, lens = _i32(np.zeros(4)), _i32(cap)
    q = torch.zeros(T, HQ, D, dtype=torch_dtype(dtype), device="cuda")
    k = torch.zeros(T, HKV, D, dtype=torch_dtype(dtype), device="cuda")
    v = torch.zeros_like(k)

    def step():
        be.build_extend_metadata_device(meta, table, rows, cached, lens)
        cache.store_kv(k, v, meta.out_loc, 0)
        return be._forward_prefill(q, None, None, 0, meta)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    done = np.zeros(4, np.int64)
    for upto in ([200, 96, 3, 130], [200, 96, 40, 130], [200, 96, 40, 130]):
        upto = np.array(upto)
        ext = upto - done
        if not ext.any():  # a second pass over the last request's last tokens
            done = upto - np.array([0, 0, 0, 7])
            ext = upto - done
        n = int(ext.sum())
        for t, h in ((q, HQ), (k, HKV), (v, HKV)):
            t.copy_(to_dev(rand(rng, (T, h, D), dtype), dtype))
        cached.copy_(_i32(done))
        lens.copy_(_i32(upto))
        before = cache.buffer.clone()
        loc = pb.page_table[np.repeat(pb.rows, ext), np.concatenate([np.arange(a, b) for a, b in zip(done, upto)])]
        g.replay()
        torch.cuda.synchronize()
        got = out[:n].clone()
        np.testing.assert_array_equal(meta.out_loc[:n].cpu().numpy(), loc)
        assert (meta.out_loc[n:] == -1).all()
        changed = cache.buffer[0] != before[0]
        changed = changed.any(-1) if pool == "fp4" else changed.any(0).flatten(1).any(-1)
        others = np.setdiff1d(np.arange(pb.num_slots), loc)
        assert not changed[torch.from_numpy(others).cuda()].any(), "a slot of another batch was written"
        host = be.extend_metadata_from_lens(pb.rows, upto, ext)
        cache.store_kv(k[:n], v[:n], _i32(loc), 0)
        assert bool((be._forward_prefill(q[:n], None, None, 0, host) == got).all())
        done = upto
    assert _device_error() == 0


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_stores_skip_rows_without_a_slot(dtype):
    """Slot -1 is padding: not stored, not an error; any other slot outside the pool is one."""
    import torch

    from minisgl_b200.config import RotaryConfig
    from minisgl_b200.layers import RotaryEmbedding

    rng = np.random.default_rng(3)
    k, v = (to_dev(rand(rng, (4, HKV, D), dtype), dtype) for _ in range(2))
    q = to_dev(rand(rng, (4, HQ, D), dtype), dtype)
    rope = RotaryEmbedding(RotaryConfig(D, D, 1e6, 4096))
    pos = _i32(np.arange(4))
    for pool in ("fp4", "dense"):
        for call in ("store", "rope"):
            for loc, code in (([5, -1, 2, -1], 0), ([5, -2, 2, -1], 32), ([5, 16, 2, -1], 32)):
                cache = _cache(pool, 16, dtype)
                if call == "store":
                    cache.store_kv(k, v, _i32(loc), 0)
                else:
                    rope.rope_store_(q.clone(), k.clone(), v, pos, _i32(loc), cache, 0)
                assert _device_error() == code, (pool, call, loc)
                used = cache.rows(0).any(-1) if pool == "fp4" else cache.v_cache(0).flatten(1).any(-1)
                assert torch.nonzero(used).flatten().tolist() == [2, 5]


def test_no_slot_is_left_from_an_earlier_batch():
    """Rows outside the table and batches that do not fit: their slots are -1, whatever the buffers held."""
    lens, cached = np.array([40, 33, 64]), np.array([8, 0, 60])
    be, pb, _ = _backend(lens)
    T, NP = int((lens - cached).sum()), int(((lens + P - 1) // P).sum())
    table = _i32(pb.page_table)
    pos = np.concatenate([np.arange(c, n) for c, n in zip(cached, lens)])
    req = np.repeat(np.arange(3), lens - cached)
    loc = pb.page_table[pb.rows[req], pos]
    for bad in (-1, 99):  # a request whose row does not exist
        meta = be.alloc_extend_metadata(3, T + 9, NP + 3)
        meta.out_loc.fill_(7)
        meta.kv_indices.fill_(1)
        rows = pb.rows.copy()
        rows[1] = bad
        be.build_extend_metadata_device(meta, table, _i32(rows), _i32(cached), _i32(lens))
        assert _device_error() == 34
        np.testing.assert_array_equal(meta.out_loc.cpu().numpy(), np.concatenate([np.where(req == 1, -1, loc), [-1] * 9]))
        pages = meta.kv_indices.cpu().numpy()
        assert (pages[3:6] == -1).all() and (pages[[0, 1, 2, 6, 7, 8, 9]] >= 0).all() and (pages[10:] == 1).all()
    for t, p in ((T - 1, NP), (T, NP - 1)):  # a capacity one short
        meta = be.alloc_extend_metadata(3, t, p)
        meta.out_loc.fill_(7)
        be.build_extend_metadata_device(meta, table, _i32(pb.rows), _i32(cached), _i32(lens))
        assert _device_error() == 34
        assert (meta.out_loc == -1).all() and (meta.work == 0).all()


def test_negative_slots_of_the_table_are_reported():
    """An entry of the page table that was never filled is an error, not padding."""
    be, pb, _ = _backend([40])
    table = pb.page_table.copy()
    table[0, 21] = -1
    meta = be.alloc_extend_metadata(1, 40, 3)
    be.build_extend_metadata_device(meta, _i32(table), _i32([0]), _i32([0]), _i32([40]))
    assert _device_error() == 32


def test_a_batch_past_the_counters_leaves_no_table():
    """8,192 requests of 300,000 new tokens: their sum passes 2^31, and nothing is left of the batch before."""
    import torch

    B, L = 8192, 300_000
    be, pb, _ = _backend([40])
    table = torch.zeros(1, L, dtype=torch.int32, device="cuda")  # all requests share a row: no entry is read
    meta = be.alloc_extend_metadata(B, 64, 64)
    rows, cached, lens = (torch.zeros(B, dtype=torch.int32, device="cuda") for _ in range(3))
    lens[5] = 9
    be.build_extend_metadata_device(meta, table, rows, cached, lens)
    assert _device_error() == 0 and meta.counts.tolist() == [9, 1]
    lens.fill_(L)
    be.build_extend_metadata_device(meta, table, rows, cached, lens)
    assert _device_error() == 34
    assert meta.counts.tolist() == [0, 0]
    for t in (meta.work, meta.qo_indptr, meta.kv_indptr, meta.kv_last_page_len):
        assert (t == 0).all()
    assert (meta.out_loc == -1).all() and (meta.last_indices == -1).all()


def test_last_indices_stay_inside_a_buffer_that_is_too_small():
    """A gather of the last tokens behind a batch that does not fit reads rows that exist."""
    be, pb, _ = _backend([40, 33])
    meta = be.alloc_extend_metadata(2, 50, 6)
    be.build_extend_metadata_device(meta, _i32(pb.page_table), _i32(pb.rows), _i32([0, 0]), _i32([40, 33]))
    assert _device_error() == 34
    assert meta.last_indices.tolist() == [39, 49]


@pytest.mark.parametrize("pool", ["fp4", "dense"])
def test_tables_of_too_large_tiles_are_refused(pool):
    """The kernel would leave the rows past its own tile unwritten; smaller tiles give the same rows."""
    lens = np.array([300, 90])
    be, pb, rng = _backend(lens, pool)
    x = to_dev(rand(rng, (pb.num_slots, HKV, D), "bfloat16"), "bfloat16")
    be.kv_cache.store_kv(x, x, _i32(np.arange(pb.num_slots)), 0)
    q = to_dev(rand(rng, (390, HQ, D), "bfloat16"), "bfloat16")
    tile = be._tile_q(P)
    got = {}
    for t in (None, tile // 2, 16, tile + 1, 256):
        meta = be.alloc_extend_metadata(2, 390, 25, tile_q=t)
        be.build_extend_metadata_device(meta, _i32(pb.page_table), _i32(pb.rows), _i32([0, 0]), _i32(lens))
        if t is not None and t > tile:
            with pytest.raises(ValueError, match="tile"):
                be._forward_prefill(q, None, None, 0, meta)
        else:
            got[t] = be._forward_prefill(q, None, None, 0, meta).float()
    # either output: weights rounded to bf16 at worst (2^-8 of the values they weigh), one bf16 rounding (2^-8)
    for t in (tile // 2, 16):
        assert (got[t] - got[None]).abs().max() <= 2 * 2.0 ** -7 * x.float().abs().max()
    assert _device_error() == 0


@pytest.mark.parametrize("pool", ["fp4", "dense"])
def test_work_lists_of_known_batches_are_exact(pool):
    """With its number of tiles given, a device-built work list is the host's, without empty tiles; the
    default list has some, which the attention call skips."""
    lens, cached = np.array([256, 90, 17, 40]), np.array([0, 80, 16, 0])
    be, pb, rng = _backend(lens, pool)
    x = to_dev(rand(rng, (pb.num_slots, HKV, D), "bfloat16"), "bfloat16")
    be.kv_cache.store_kv(x, x, _i32(np.arange(pb.num_slots)), 0)
    T, NP = int((lens - cached).sum()), int(((lens + P - 1) // P).sum())
    q = to_dev(rand(rng, (T, HQ, D), "bfloat16"), "bfloat16")
    host = be.extend_metadata_from_lens(pb.rows, lens, lens - cached)
    assert be.extend_tiles(cached, lens) == host.n_work
    want = be._forward_prefill(q, None, None, 0, host)
    for n_work in (host.n_work, None):
        meta = be.alloc_extend_metadata(4, T, NP, cached=cached, lens=lens, n_work=n_work)
        assert (meta.n_work == host.n_work) == (n_work is not None)
        be.build_extend_metadata_device(meta, _i32(pb.page_table), _i32(pb.rows), _i32(cached), _i32(lens))
        assert bool((be._forward_prefill(q, None, None, 0, meta) == want).all())
    assert _device_error() == 0
    for bad in (-1, T + 5):
        with pytest.raises(ValueError, match="tiles"):
            be.alloc_extend_metadata(4, T, NP, n_work=bad)


@pytest.mark.parametrize("short", ["tokens", "pages", "tiles", "nothing"])
def test_nothing_is_written_past_a_buffer(short):
    """Buffers that lie between guard words, at and one below the size the batch needs."""
    import torch

    lens, cached = np.array([300, 90, 17, 4000]), np.array([0, 80, 16, 3990])
    be, pb, _ = _backend(lens)
    T, NP = int((lens - cached).sum()), int(((lens + P - 1) // P).sum())
    tiles = be.extend_tiles(cached, lens)
    n = dict(positions=T - (short == "tokens"), out_loc=T - (short == "tokens"), kv_indices=NP - (short == "pages"),
             work=4 * (tiles - (short == "tiles")), qo_indptr=5, kv_indptr=5, last_indices=4, kv_last_page_len=4, counts=2)
    meta = be.alloc_extend_metadata(4, T, NP, n_work=tiles)
    bufs = {}
    for name, size in n.items():
        b = torch.full((64 + size + 64,), 0x5A5A, dtype=torch.int32, device="cuda")  # 256 bytes of guard: work stays aligned
        bufs[name] = b
        t = b[64: 64 + size]
        setattr(meta, name, t.view(-1, 4) if name == "work" else t)
    meta.n_work = n["work"] // 4
    be.build_extend_metadata_device(meta, _i32(pb.page_table), _i32(pb.rows), _i32(cached), _i32(lens))
    assert _device_error() == (0 if short == "nothing" else 34)
    for name, b in bufs.items():
        assert (b[:64] == 0x5A5A).all() and (b[64 + n[name]:] == 0x5A5A).all(), name
    if short == "nothing":
        host = be.extend_metadata_from_lens(pb.rows, lens, lens - cached)
        for name in ("qo_indptr", "kv_indptr", "kv_indices", "kv_last_page_len", "work", "last_indices"):
            assert bool((getattr(meta, name) == getattr(host, name)).all()), name


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("lengths", ["known", "unknown"])
def test_long_prefixes_in_runs_behind_device_tables(lengths, dtype):
    """Keys cut into runs from host copies of the lengths or from a guess of equal ones, with empty tiles
    in the list: the float64 attention, again on a second call, and after other lengths used the buffers."""
    import torch

    from oracle import fp4 as F

    lens, cached = np.array([6000, 3100]), np.array([5990, 3099])
    be, pb, rng = _backend(lens, "fp4", dtype)
    cache = be.kv_cache
    k, v = (rand(rng, (pb.num_slots, HKV, D), dtype) for _ in range(2))
    cache.store_kv(to_dev(k, dtype), to_dev(v, dtype), _i32(np.arange(pb.num_slots)), 0)
    kr, vr = F.roundtrip(k), F.roundtrip(v)
    T, NP = 40, int(((lens + P - 1) // P).sum())
    kw = dict(cached=cached, lens=lens) if lengths == "known" else {}
    meta = be.alloc_extend_metadata(2, T, NP, **kw)
    assert meta.n_split > 1
    table, rows = _i32(pb.page_table), _i32(pb.rows)
    q = rand(rng, (T, HQ, D), dtype)
    for c2, n2 in ((cached, lens), (np.array([4980, 100]), np.array([5000, 120])), (cached, lens)):
        be.build_extend_metadata_device(meta, table, rows, _i32(c2), _i32(n2))
        out = be._forward_prefill(to_dev(q, dtype), None, None, 0, meta)
        again = be._forward_prefill(to_dev(q, dtype), None, None, 0, meta)
        o = 0
        for b in range(2):
            m = int(n2[b] - c2[b])
            s = pb.page_table[b, : int(n2[b])]
            ref, A, X, S = F.attend(q[o:o + m].astype(np.float64), kr[s], vr[s], be.scale, int(c2[b]))
            got = out[o:o + m].double().cpu().numpy()
            assert (np.abs(got - ref) <= F.tolerance(ref, A, X, S, dtype, D, int(n2[b]))).all()
            o += m
        assert bool((out[:o] == again[:o]).all()), "extend is not repeatable"
    assert _device_error() == 0
