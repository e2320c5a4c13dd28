"""Prefill tables built on the device (b2a_extend_metadata) against the host builders, integer for integer."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from helpers import HeadConfig, rand, to_dev
from minisgl_b200 import workloads as W

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


def _backend(table, P, num_tokens=4096):
    import torch

    from minisgl_b200 import B200AttnBackend, FP4KVCache

    return B200AttnBackend(HeadConfig(16, 8, 128), FP4KVCache(1, num_tokens, 8, 128, torch.bfloat16, "cuda"), table, P)


def _batch(B, P, hi, ext_hi, seed, zero=False):
    rng = np.random.default_rng(seed)
    lens = rng.integers(1, hi + 1, B)
    ext = np.minimum(rng.integers(1, ext_hi + 1, B), lens)
    if zero and B > 3:  # requests without tokens and without new tokens, first, last and in a row
        lens[[0, 2]] = 0
        ext[[0, 1, 2, B - 1]] = 0
    pb = W.allocate_pages(lens, int(((lens + P - 1) // P).sum() + 4) * P, P, rng, max_seq_len=hi + P)
    R = B + 5
    table = rng.integers(0, 1 << 20, (R, pb.page_table.shape[1])).astype(np.int32)
    rows = rng.permutation(R)[:B]
    table[rows] = pb.page_table
    return table, rows.astype(np.int64), lens.astype(np.int64), ext.astype(np.int64)


def _expect(table, rows, lens, ext, P, tile):
    from minisgl_b200 import _native as nat
    from minisgl_b200.attention.base import paged_kv_indices

    qo = np.zeros(len(ext) + 1, np.int32)
    np.cumsum(ext, out=qo[1:])
    kv, idx, lpl = paged_kv_indices(table, rows, lens, P)
    pos = np.concatenate([np.arange(L - n, L) for L, n in zip(lens, ext)])
    loc = table[np.repeat(rows, ext), pos]
    work = nat.extend_plan(qo, kv, lpl, P, tile)
    return dict(qo_indptr=qo, kv_indptr=kv, kv_indices=idx, kv_last_page_len=lpl, positions=pos, out_loc=loc,
                last_indices=qo[1:] - 1, work=work)


def _compare(meta, want):
    n = want["work"].shape[0]
    work = meta.work.cpu().numpy()
    np.testing.assert_array_equal(work[:n], want["work"])
    assert (work[n:] == 0).all()
    assert meta.counts.tolist() == [int(want["qo_indptr"][-1]), n]
    for name in ("qo_indptr", "kv_indptr", "kv_last_page_len", "last_indices"):
        np.testing.assert_array_equal(getattr(meta, name).cpu().numpy(), want[name], err_msg=name)
    for name in ("positions", "out_loc", "kv_indices"):
        np.testing.assert_array_equal(getattr(meta, name).cpu().numpy()[: len(want[name])], want[name], err_msg=name)


@pytest.mark.parametrize("P", [1, 16, 64])
@pytest.mark.parametrize("B,hi,ext_hi,tile", [(1, 1, 1, 128), (1, 9000, 8000, 32), (7, 40, 40, 1), (33, 900, 300, 64),
                                              (300, 500, 7, 256), (2500, 60, 60, 16), (8192, 3, 3, 128)])
def test_tables_equal_the_host_builders(B, hi, ext_hi, tile, P):
    table, rows, lens, ext = _batch(B, P, hi, ext_hi, seed=B + P)
    be = _backend(table, P)
    want = _expect(table, rows, lens, ext, P, tile)
    meta = be.alloc_extend_metadata(B, int(ext.sum()), len(want["kv_indices"]), tile_q=tile)
    be.build_extend_metadata_device(meta, _i32(table), _i32(rows), _i32(lens - ext), _i32(lens))
    _compare(meta, want)
    assert _device_error() == 0


@pytest.mark.parametrize("B", [4, 700])
def test_requests_without_tokens(B):
    table, rows, lens, ext = _batch(B, 16, 200, 90, seed=3, zero=True)
    be = _backend(table, 16)
    want = _expect(table, rows, lens, ext, 16, 64)
    meta = be.alloc_extend_metadata(B, int(ext.sum()), len(want["kv_indices"]), tile_q=64)
    be.build_extend_metadata_device(meta, _i32(table), _i32(rows), _i32(lens - ext), _i32(lens))
    _compare(meta, want)


def test_equal_costs_keep_request_order():
    """Hundreds of equal tiles: the sort is stable."""
    B, P = 900, 16
    rng = np.random.default_rng(0)
    lens, ext = np.full(B, 96), np.full(B, 32)
    pb = W.allocate_pages(lens, B * 96, P, rng)
    be = _backend(pb.page_table, P)
    want = _expect(pb.page_table, pb.rows, lens, ext, P, 16)
    meta = be.alloc_extend_metadata(B, int(ext.sum()), len(want["kv_indices"]), tile_q=16)
    be.build_extend_metadata_device(meta, _i32(pb.page_table), _i32(pb.rows), _i32(lens - ext), _i32(lens))
    _compare(meta, want)


def test_a_smaller_batch_leaves_the_tails():
    """One captured call serves batches of other lengths: tails stay, unused tiles are empty."""
    import torch

    B, P, tile = 20, 16, 64
    table, rows, lens, ext = _batch(B, P, 800, 300, seed=5)
    be = _backend(table, P)
    meta = be.alloc_extend_metadata(B, 20 * 300, 20 * 50, tile_q=tile)
    t, r, c, n = _i32(table), _i32(rows), _i32(lens - ext), _i32(lens)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        be.build_extend_metadata_device(meta, t, r, c, n)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        be.build_extend_metadata_device(meta, t, r, c, n)
    for seed in (1, 2):
        rng = np.random.default_rng(seed)
        l2 = np.array([rng.integers(1, L + 1) for L in lens])
        e2 = np.array([rng.integers(0, min(300, L) + 1) for L in l2])
        c.copy_(_i32(l2 - e2))
        n.copy_(_i32(l2))
        meta.positions.fill_(-5)
        meta.kv_indices.fill_(-5)
        g.replay()
        want = _expect(table, rows, l2, e2, P, tile)
        _compare(meta, want)
        assert (meta.positions[int(e2.sum()):] == -5).all()
        assert (meta.kv_indices[len(want["kv_indices"]):] == -5).all()
    assert _device_error() == 0


def test_bad_lengths_are_flagged():
    B, P = 6, 16
    table, rows, lens, ext = _batch(B, P, 300, 100, seed=8)
    be = _backend(table, P)
    good = dict(r=rows, c=lens - ext, n=lens)
    for bad in (dict(n=np.where(np.arange(B) == 2, -4, lens)), dict(n=np.where(np.arange(B) == 1, 10 ** 6, lens)),
                dict(c=np.where(np.arange(B) == 3, -1, lens - ext)), dict(c=np.where(np.arange(B) == 0, lens + 1, lens - ext)),
                dict(r=np.where(np.arange(B) == 4, 99, rows)), dict(r=np.where(np.arange(B) == 5, -1, rows))):
        a = {**good, **bad}
        meta = be.alloc_extend_metadata(B, 2000, 200, tile_q=64)
        assert _device_error() == 0
        be.build_extend_metadata_device(meta, _i32(table), _i32(a["r"]), _i32(a["c"]), _i32(a["n"]))
        assert _device_error() == 34
    # capacities one short: flagged, nothing past them written
    T, NP = int(ext.sum()), int(((lens + P - 1) // P).sum())
    for t, p in ((T - 1, NP), (T, NP - 1)):
        meta = be.alloc_extend_metadata(B, t, p, tile_q=64)
        be.build_extend_metadata_device(meta, _i32(table), _i32(rows), _i32(lens - ext), _i32(lens))
        assert _device_error() == 34
        assert (meta.work == 0).all() and int(meta.counts[1]) == 0  # nothing is attended


def test_refusals():
    import torch

    table, rows, lens, ext = _batch(4, 16, 100, 50, seed=2)
    be = _backend(table, 16)
    meta = be.alloc_extend_metadata(4, 200, 40)
    t, r, c, n = _i32(table), _i32(rows), _i32(lens - ext), _i32(lens)
    for a in ((t.long(), r, c, n), (t, r[:3], c, n), (t, r, c.long(), n), (t, r, c, n.cpu()), (t[:, ::2], r, c, n),
              (t.cpu(), r, c, n), (t[0], r, c, n)):
        with pytest.raises(ValueError):
            be.build_extend_metadata_device(meta, *a)
    with pytest.raises(ValueError):
        be.build_extend_metadata_device(be.extend_metadata_from_lens(rows, lens, ext), t, r, c, n)
    for kw in ((0, 10, 10), (4, -1, 10), (4, 10, -1), (4, 10, 10, 0)):
        with pytest.raises(ValueError):
            be.alloc_extend_metadata(*kw)
    # a 16-bit pool with small pages extends over host-built key groups
    from minisgl_b200 import B200AttnBackend, MHAKVCache

    dense = B200AttnBackend(HeadConfig(16, 8, 128), MHAKVCache(1, 64, 8, 128, torch.bfloat16), table, 1)
    with pytest.raises(ValueError):
        dense.alloc_extend_metadata(4, 200, 40)


@pytest.mark.parametrize("pool", ["fp4", "dense"])
def test_extend_through_device_tables(pool):
    """Extend attention gives the same bytes whether its tables were built here or on the host."""
    import torch

    from minisgl_b200 import B200AttnBackend, FP4KVCache, MHAKVCache

    P, Hq, Hkv, D = 16, 16, 8, 128
    table, rows, lens, ext = _batch(9, P, 500, 200, seed=11)
    n = (int(table[rows].max()) // P + 1) * P
    cls = FP4KVCache if pool == "fp4" else MHAKVCache
    cache = cls(1, n, Hkv, D, torch.bfloat16, "cuda")
    rng = np.random.default_rng(0)
    x = to_dev(rand(rng, (n, Hkv, D), "bfloat16"), "bfloat16")
    cache.store_kv(x, x.flip(0).contiguous(), _i32(np.arange(n)), 0)
    be = B200AttnBackend(HeadConfig(Hq, Hkv, D), cache, table, P)
    q = to_dev(rand(rng, (int(ext.sum()), Hq, D), "bfloat16"), "bfloat16")
    host = be.extend_metadata_from_lens(rows, lens, ext)
    want = be._forward_prefill(q, None, None, 0, host)
    meta = be.alloc_extend_metadata(9, int(ext.sum()), int(((lens + P - 1) // P).sum()))
    assert meta.n_work >= host.n_work
    be.build_extend_metadata_device(meta, _i32(table), _i32(rows), _i32(lens - ext), _i32(lens))
    got = be._forward_prefill(q, None, None, 0, meta)
    assert bool((got == want).all())
    assert _device_error() == 0
