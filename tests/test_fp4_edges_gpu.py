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


class Pool:
    """A filled pool, its page table and its rows' exact values."""

    def __init__(self, lens, Hkv, D, dtype, P, seed, gk=1.0, gv=1.0, k=None, v=None):
        from minisgl_b200 import FP4KVCache

        self.rng = rng = np.random.default_rng(seed)
        lens = np.asarray(lens, dtype=np.int64)
        n = int(((lens + P - 1) // P).sum() + 3) * P
        self.pb = W.allocate_pages(lens, n, P, rng)
        k = rand(rng, (n, Hkv, D), dtype) if k is None else np.broadcast_to(k, (n, Hkv, D)).astype(np.float32)
        v = rand(rng, (n, Hkv, D), dtype) if v is None else np.broadcast_to(v, (n, Hkv, D)).astype(np.float32)
        kd, vd = to_dev(k * np.float32(gk), dtype), to_dev(v * np.float32(gv), dtype)
        self.cache = FP4KVCache(1, n, Hkv, D, torch_dtype(dtype), "cuda", k_scale=gk, v_scale=gv)
        self.cache.store_kv(kd, vd, _i32(np.arange(n)), 0)
        self.k = F.roundtrip(kd.double().cpu().numpy(), gk)
        self.v = F.roundtrip(vd.double().cpu().numpy(), gv)

    def of(self, b):
        s = self.pb.page_table[b, : int(self.pb.lens[b])]
        return self.k[s], self.v[s]


def _check(got, refs, dtype, D, L, rows=slice(None)):
    got = got.double().cpu().numpy()
    ref, A, X, S = (np.concatenate(x) for x in zip(*refs))
    err, tol = np.abs(got - ref)[rows], F.tolerance(ref, A, X, S, dtype, D, L)[rows]
    assert np.isfinite(got[rows]).all()
    assert (err <= tol).all(), (err - tol).max()


def _refs(p, q, lens, ext, scale):
    refs, o = [], 0
    with np.errstate(invalid="ignore"):
        for b, (L, n) in enumerate(zip(lens, ext)):
            refs.append(F.attend(q[o:o + n], *p.of(b), scale, L - n))
            o += n
    return refs


# what a query row holds -> nothing but NaN may come out of its heads, and nothing else changes
BAD_QUERIES = {"nan": np.nan, "inf": np.inf, "-inf": -np.inf}


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("what", BAD_QUERIES)
@pytest.mark.parametrize("keys", ["ones", "random"])
def test_infinite_and_nan_queries_show_in_decode(what, keys, dtype):
    """Over keys that are all ones, -inf makes every score -inf and +inf every score +inf: softmax has no
    value either way. Requests of one token, of part of a step, of whole steps, and split over CTAs."""
    from minisgl_b200 import B200AttnBackend

    Hq, Hkv, D = 4, 2, 128
    lens = [1, 15, 64, 130, 2500, 40]
    p = Pool(lens, Hkv, D, dtype, 16, seed=3, k=1.0 if keys == "ones" else None)
    q = rand(p.rng, (len(lens), Hq, D), dtype)
    bad = np.zeros((len(lens), Hq), bool)
    bad[:5, 1] = bad[3] = True  # the last request, and most heads, stay as they are
    q[bad, 17] = BAD_QUERIES[what]
    be = B200AttnBackend(HeadConfig(Hq, Hkv, D), p.cache, p.pb.page_table, 16)
    good = np.where(bad[..., None], 0, q)
    refs = _refs(p, good.astype(np.float64), lens, [1] * len(lens), be.scale)
    for nc in (None, 1, 31):
        out = be.forward_decode(to_dev(q, dtype), 0, be.decode_metadata_from_lens(p.pb.rows, p.pb.lens, num_ctas=nc))
        assert np.isnan(out.double().cpu().numpy()[bad]).all(), (what, nc)
        _check(out, refs, dtype, D, max(lens), rows=~bad)
    assert _device_error() == 0


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("what", BAD_QUERIES)
@pytest.mark.parametrize("keys", ["ones", "random"])
@pytest.mark.parametrize("D", [128, 256])
def test_infinite_and_nan_queries_show_in_extend(D, keys, what, dtype):
    """The same for extend: tiles of one and of two streams, a row with one visible key, a prompt in runs."""
    from minisgl_b200 import B200AttnBackend

    Hq, Hkv = 4, 2
    lens, ext = np.array([1, 200, 90, 700]), np.array([1, 200, 3, 9])
    p = Pool(lens, Hkv, D, dtype, 16, seed=5, k=1.0 if keys == "ones" else None)
    q = rand(p.rng, (int(ext.sum()), Hq, D), dtype)
    bad = np.zeros(q.shape[:2], bool)
    bad[[0, 1, 2, 130, 200, 202, 212], 1] = bad[77] = True
    q[bad, 17] = BAD_QUERIES[what]
    be = B200AttnBackend(HeadConfig(Hq, Hkv, D), p.cache, p.pb.page_table, 16)
    refs = _refs(p, np.where(bad[..., None], 0, q).astype(np.float64), lens, ext, be.scale)
    for runs in (None, 128):
        meta = be.extend_metadata_from_lens(p.pb.rows, lens, ext)
        _force_runs(be, meta, runs, 6)
        out = be._forward_prefill(to_dev(q, dtype), None, None, 0, meta)
        assert np.isnan(out.double().cpu().numpy()[bad]).all(), (what, runs)
        _check(out, refs, dtype, D, int(lens.max()), rows=~bad)
    assert _device_error() == 0


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_scores_past_the_softmax_s_range_are_never_a_silent_zero(dtype):
    """Scores of about 2^40: fp32 rounds them by 2^16, so a row has no weights that mean anything. Values
    are at least 1, so an output of 0 would be a row whose weights vanished unseen."""
    from minisgl_b200 import B200AttnBackend

    Hq, Hkv, D = 16, 8, 128
    lens, ext = np.array([40, 300, 2500, 130]), np.array([40, 9, 64, 130])
    p = Pool(lens, Hkv, D, dtype, 16, seed=6, v=2.0)
    q = rand(p.rng, (int(ext.sum()), Hq, D), dtype) * np.float32(2.0 ** 37)
    be = B200AttnBackend(HeadConfig(Hq, Hkv, D), p.cache, p.pb.page_table, 16)
    last = np.cumsum(ext) - 1
    for nc in (None, 1, 31):
        out = be.forward_decode(to_dev(q[last], dtype), 0, be.decode_metadata_from_lens(p.pb.rows, p.pb.lens, num_ctas=nc))
        assert not (out == 0).any()
    for runs in (None, 256):
        meta = be.extend_metadata_from_lens(p.pb.rows, lens, ext)
        _force_runs(be, meta, runs, 10)
        assert not (be._forward_prefill(to_dev(q, dtype), None, None, 0, meta) == 0).any()
    assert _device_error() == 0


def _force_runs(be, meta, run_keys, n_split):
    """The same work items with their keys in runs of run_keys (None: whole)."""
    import torch

    from minisgl_b200 import _native as nat

    meta.run_keys, meta.n_split = (0, 1) if run_keys is None else (run_keys, n_split)
    n = int(nat.LIB.b2a_fp4_extend_workspace_bytes(meta.n_work, meta.n_split, be.Hkv, be.D))
    meta.workspace = torch.zeros(n, dtype=torch.uint8, device="cuda") if n else None


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("amp,gk", [(2.0 ** -80, 2.0 ** -100), (2.0 ** -100, 2.0 ** -30), (2.0 ** 60, 2.0 ** -100)])
def test_scores_below_fp32_weigh_all_keys_alike(amp, gk, dtype):
    from minisgl_b200 import B200AttnBackend

    Hq, Hkv, D = 4, 2, 128
    lens, ext = np.array([140, 9, 300, 700]), np.array([60, 1, 64, 2])  # rows that see a part of the blocks
    p = Pool(lens, Hkv, D, dtype, 16, seed=8, gk=gk)
    q = rand(p.rng, (int(ext.sum()), Hq, D), dtype) * np.float32(amp)
    be = B200AttnBackend(HeadConfig(Hq, Hkv, D), p.cache, p.pb.page_table, 16)
    last = np.cumsum(ext) - 1
    refs = _refs(p, q[last].astype(np.float64), lens, [1] * 4, be.scale)
    out = be.forward_decode(to_dev(q[last], dtype), 0, be.decode_metadata_from_lens(p.pb.rows, p.pb.lens))
    _check(out, refs, dtype, D, 700)
    refs = _refs(p, q.astype(np.float64), lens, ext, be.scale)
    for runs in (None, 128):
        meta = be.extend_metadata_from_lens(p.pb.rows, lens, ext)
        _force_runs(be, meta, runs, 6)
        _check(be._forward_prefill(to_dev(q, dtype), None, None, 0, meta), refs, dtype, D, 700)
    assert _device_error() == 0


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("gv", [2.0 ** 100, 2.0 ** -100, 2.0 ** 65])
def test_value_scales_at_the_ends_of_their_range(gv, dtype):
    """Values of 2,000 * v_scale over many keys: sums of them pass fp32's end, their means do not."""
    from minisgl_b200 import B200AttnBackend

    Hq, Hkv, D = 4, 2, 128
    lens, ext = np.array([5000, 60, 1]), np.array([3, 60, 1])
    big = 2000 * np.sign(np.random.default_rng(0).standard_normal((1, Hkv, D)) + 1.0)
    p = Pool(lens, Hkv, D, dtype, 16, seed=8, gv=gv, k=1.0, v=big)  # every key weighs 2^7
    q = rand(p.rng, (int(ext.sum()), Hq, D), dtype)
    be = B200AttnBackend(HeadConfig(Hq, Hkv, D), p.cache, p.pb.page_table, 16)
    last = np.cumsum(ext) - 1
    refs = _refs(p, q[last].astype(np.float64), lens, [1] * 3, be.scale)
    for nc in (None, 1, 2):
        out = be.forward_decode(to_dev(q[last], dtype), 0, be.decode_metadata_from_lens(p.pb.rows, p.pb.lens, num_ctas=nc))
        _check(out, refs, dtype, D, 5000)
    refs = _refs(p, q.astype(np.float64), lens, ext, be.scale)
    for runs in (None, 640):
        meta = be.extend_metadata_from_lens(p.pb.rows, lens, ext)
        _force_runs(be, meta, runs, 8)
        _check(be._forward_prefill(to_dev(q, dtype), None, None, 0, meta), refs, dtype, D, 5000)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("gk,gv,amp", [(2.0 ** -10, 64.0, 2.0 ** 10), (4.0, 2.0 ** -20, 1.0)])
def test_extend_over_scaled_pools(gk, gv, amp, dtype):
    from minisgl_b200 import B200AttnBackend

    Hq, Hkv, D = 16, 8, 128
    lens, ext = np.array([700, 90, 200]), np.array([130, 3, 200])
    p = Pool(lens, Hkv, D, dtype, 16, seed=2, gk=gk, gv=gv)
    q = rand(p.rng, (int(ext.sum()), Hq, D), dtype) * np.float32(amp)
    be = B200AttnBackend(HeadConfig(Hq, Hkv, D), p.cache, p.pb.page_table, 16)
    refs = _refs(p, q.astype(np.float64), lens, ext, be.scale)
    for runs in (None, 256):
        meta = be.extend_metadata_from_lens(p.pb.rows, lens, ext)
        _force_runs(be, meta, runs, 3)
        _check(be._forward_prefill(to_dev(q, dtype), None, None, 0, meta), refs, dtype, D, 700)
    assert _device_error() == 0


@pytest.mark.parametrize("dtype,D", [("bfloat16", 128), ("float32", 128), ("bfloat16", 256), ("float32", 64)])
def test_extend_in_a_packed_workspace(dtype, D):
    """Workspaces of any size between two runs and all of them: items are cut as far as it goes, the
    rows agree with float64, a second call on the same workspace repeats them, and nothing is written behind it."""
    import torch

    from minisgl_b200 import B200AttnBackend
    from minisgl_b200 import _native as nat

    Hq, Hkv = 4, 2
    lens = np.array([40, 700, 33, 1100, 300, 64, 513])
    ext = np.array([40, 5, 1, 200, 2, 64, 90])
    p = Pool(lens, Hkv, D, dtype, 16, seed=9)
    q = rand(p.rng, (int(ext.sum()), Hq, D), dtype)
    qd = to_dev(q, dtype)
    be = B200AttnBackend(HeadConfig(Hq, Hkv, D), p.cache, p.pb.page_table, 16)
    refs = _refs(p, q.astype(np.float64), lens, ext, be.scale)
    meta = be.extend_metadata_from_lens(p.pb.rows, lens, ext)
    w = meta.work.cpu().numpy()
    keys = (lens - ext)[w[:, 0]] + w[:, 1] + w[:, 2]
    meta.run_keys, meta.n_split = 128, 9
    runs = np.minimum(-(-keys // 128), 9)
    total = int(runs[runs > 1].sum())
    code = be.dtype_code
    n_all = int(nat.LIB.b2a_fp4_extend_workspace_bytes(meta.n_work, 9, Hkv, D))
    sizes = [int(nat.LIB.b2a_fp4_extend_packed_bytes(meta.n_work, r, Hkv, D, code)) for r in (2, 3, 7, total - 1, total)]
    outs = []
    for n in [*sizes, sizes[-1] + 64, n_all - 4, n_all]:
        buf = torch.zeros(n + 4096, dtype=torch.uint8, device="cuda")
        buf[n:] = 0x5A
        meta.workspace = buf[:n]
        first = be._forward_prefill(qd, None, None, 0, meta)
        assert bool((be._forward_prefill(qd, None, None, 0, meta) == first).all()), "extend is not repeatable"
        _check(first, refs, dtype, D, int(lens.max()))
        assert (buf[n:] == 0x5A).all(), "written behind the workspace"
        assert (buf[: 4 * meta.n_work * Hkv] == 0).all(), "merge counters are not re-armed"
        outs.append(first)
    assert all(bool((o == outs[-1]).all()) for o in outs[4:])  # the same runs, wherever their rows lie
    meta.workspace = torch.zeros(sizes[0] - 4, dtype=torch.uint8, device="cuda")
    with pytest.raises(nat.B200AttnError):
        be._forward_prefill(qd, None, None, 0, meta)
    assert _device_error() == 0


def test_one_long_request_among_short_ones_through_the_backend():
    """Tables of both builders ask for the batch's own runs only, and attend alike."""
    import torch

    from minisgl_b200 import B200AttnBackend

    Hq, Hkv, D, P = 2, 1, 128, 16
    lens = np.array([300] * 40 + [20000] + [300] * 43)
    ext = np.where(lens > 300, 3, 128)
    p = Pool(lens, Hkv, D, "bfloat16", P, seed=1)
    be = B200AttnBackend(HeadConfig(Hq, Hkv, D), p.cache, p.pb.page_table, P)
    q = to_dev(rand(p.rng, (int(ext.sum()), Hq, D), "bfloat16"), "bfloat16")
    host = be.extend_metadata_from_lens(p.pb.rows, lens, ext)
    assert host.n_split > 8 and host.workspace.numel() <= 64 << 20
    want = be._forward_prefill(q, None, None, 0, host)
    o = int(ext[:40].sum())
    ref = F.attend(q[o:o + 3].double().cpu().numpy(), *p.of(40), be.scale, 20000 - 3)
    _check(want[o:o + 3], [ref], "bfloat16", D, 20000)
    meta = be.alloc_extend_metadata(84, int(ext.sum()), int(((lens + P - 1) // P).sum()), cached=lens - ext, lens=lens)
    assert meta.workspace.numel() <= 64 << 20
    be.build_extend_metadata_device(meta, _i32(p.pb.page_table), _i32(p.pb.rows), _i32(lens - ext), _i32(lens))
    for _ in range(2):
        assert bool((be._forward_prefill(q, None, None, 0, meta) == want).all())
    assert _device_error() == 0
    torch.cuda.empty_cache()


@pytest.mark.parametrize("Hkv,D", [(4, 128), (8, 64), (16, 128), (8, 256)])
def test_a_pool_of_another_shape_is_refused(Hkv, D):
    import torch

    from minisgl_b200 import B200AttnBackend, FP4KVCache

    cache = FP4KVCache(1, 64, Hkv, D, torch.bfloat16, "cuda")
    with pytest.raises(ValueError, match="kv heads"):
        B200AttnBackend(HeadConfig(16, 8, 128), cache, np.zeros((1, 64), np.int32), 16)


def test_a_captured_decode_keeps_its_workspace():
    """A decode captured with host-built metadata goes on after a larger batch has replaced the workspace."""
    import weakref

    import torch

    from minisgl_b200 import B200AttnBackend

    lens = [900, 70]
    p = Pool(lens, 8, 128, "bfloat16", 16, seed=4)
    be = B200AttnBackend(HeadConfig(16, 8, 128), p.cache, p.pb.page_table, 16)
    q = to_dev(rand(p.rng, (2, 16, 128), "bfloat16"), "bfloat16")
    meta = be.decode_metadata_from_lens(p.pb.rows, p.pb.lens, num_ctas=8)
    want = be.forward_decode(q, 0, meta)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = be.forward_decode(q, 0, meta)
    used = weakref.ref(be._workspace)
    big = be.decode_metadata_from_lens(p.pb.rows, p.pb.lens, num_ctas=31)
    be.forward_decode(q, 0, big)
    assert be._workspace is not used() and used() is not None, "the captured workspace was given back"
    g.replay()
    torch.cuda.synchronize()
    assert bool((out == want).all())
