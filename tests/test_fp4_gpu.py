"""The 4-bit KV pool on the GPU: store, load, decode and extend against the float64 oracle.

Store and load are compared bit for bit (the format's codes are those of the exact quotient).
Attention is compared within oracle.fp4.tolerance, a bound counted from the roundings.
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


def _cache(n, Hkv, D, dtype, **kw):
    from minisgl_b200 import FP4KVCache

    return FP4KVCache(1, n, Hkv, D, torch_dtype(dtype), "cuda", **kw)


def _i32(a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


# ------------------------------------------------------------------ store and load
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("T,Hkv,D", [(1, 8, 128), (3, 1, 64), (70, 8, 128), (257, 3, 256), (33, 16, 64)])
def test_store_and_load_are_exact(T, Hkv, D, dtype):
    rng = np.random.default_rng(T + D)
    k = rand(rng, (T, Hkv, D), dtype) * 2.0 ** rng.integers(-6, 4, (T, Hkv, 1))
    v = rand(rng, (T, Hkv, D), dtype)
    v[:, :, :16] = 0
    n = T + 5
    loc = rng.permutation(n)[:T]
    c = _cache(n, Hkv, D, dtype)
    c.store_kv(to_dev(k, dtype), to_dev(v, dtype), _i32(loc), 0)
    rows = c.rows(0).cpu().numpy()
    np.testing.assert_array_equal(rows[loc], F.pack_rows(k, v))
    free = np.setdiff1d(np.arange(n), loc)
    assert (rows[free] == 0).all()  # other slots stay as they were
    gk, gv = c.load_kv(_i32(loc[::-1].copy()), 0)
    np.testing.assert_array_equal(gk.float().cpu().numpy()[::-1], F.roundtrip(k))
    np.testing.assert_array_equal(gv.float().cpu().numpy()[::-1], F.roundtrip(v))
    assert _device_error() == 0


def test_store_on_the_borders():
    """Elements on and next to every border between codes, maxima on borders between scales."""
    s = F.e4m3_values()
    rows = []
    for sc in s[1:]:
        m = np.float32(6 * sc)
        ties = np.float32([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]) * np.float32(sc)
        x = np.concatenate([[m], ties, np.nextafter(ties, np.float32(0))[:4], np.nextafter(ties, np.float32(1e9))[:4]])
        rows.append(x[:16])
        up = np.float32(6 * (sc + s[min(np.searchsorted(s, sc) + 1, len(s) - 1)]) / 2)
        for a in (up, np.nextafter(up, np.float32(0)), np.nextafter(up, np.float32(1e9))):
            rows.append(np.concatenate([[-a], x[1:16]]).astype(np.float32))
    x = np.zeros((-(-len(rows) // 4), 1, 64), np.float32)
    x.reshape(-1, 16)[: len(rows)] = rows
    T = len(x)
    c = _cache(T, 1, 64, "float32")
    c.store_kv(to_dev(x, "float32"), to_dev(-x, "float32"), _i32(np.arange(T)), 0)
    np.testing.assert_array_equal(c.rows(0).cpu().numpy(), F.pack_rows(x, -x))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_store_keeps_the_pool_finite(dtype):
    x = np.ones((2, 1, 64), np.float32)
    x[0, 0, 3], x[0, 0, 20], x[0, 0, 33] = np.nan, np.inf, -np.inf
    x[1, 0, :16] = np.nan
    x[1, 0, 16:32] = 3e38 if dtype == "float32" else 1e30
    x[1, 0, 32:48] = 1e-30
    c = _cache(2, 1, 64, dtype)
    c.store_kv(to_dev(x, dtype), to_dev(x, dtype), _i32([0, 1]), 0)
    k, _ = c.load_kv(_i32([0, 1]), 0)
    got = k.float().cpu().numpy()
    assert np.isfinite(got).all()
    np.testing.assert_array_equal(got, F.roundtrip(x))


@pytest.mark.parametrize("gk,gv", [(2.0 ** -8, 4.0), (1024.0, 2.0 ** -12)])
def test_pool_scales(gk, gv):
    rng = np.random.default_rng(5)
    k, v = rand(rng, (9, 2, 128), "bfloat16") * 0.01, rand(rng, (9, 2, 128), "bfloat16") * 100
    c = _cache(9, 2, 128, "bfloat16", k_scale=gk, v_scale=gv)
    kd, vd = to_dev(k, "bfloat16"), to_dev(v, "bfloat16")
    c.store_kv(kd, vd, _i32(np.arange(9)), 0)
    a, b = c.load_kv(_i32(np.arange(9)), 0)
    np.testing.assert_array_equal(a.float().cpu().numpy(), F.roundtrip(kd.float().cpu().numpy(), gk))
    np.testing.assert_array_equal(b.float().cpu().numpy(), F.roundtrip(vd.float().cpu().numpy(), gv))


@pytest.mark.parametrize("off", [0, 1, 3])
def test_store_of_strided_and_unaligned_rows(off):
    """k, v as views of a fused projection, at any element offset."""
    T, Hq, Hkv, D = 21, 4, 2, 64
    rng = np.random.default_rng(off)
    w = (Hq + 2 * Hkv) * D + off
    buf = to_dev(rand(rng, (T, w), "bfloat16"), "bfloat16")
    k = buf[:, off + Hq * D: off + (Hq + Hkv) * D].view(T, Hkv, D)
    v = buf[:, off + (Hq + Hkv) * D:].view(T, Hkv, D)
    c = _cache(64, Hkv, D, "bfloat16")
    loc = rng.permutation(64)[:T]
    c.store_kv(k, v, _i32(loc), 0)
    np.testing.assert_array_equal(c.rows(0).cpu().numpy()[loc],
                                  F.pack_rows(k.float().cpu().numpy(), v.float().cpu().numpy()))


def test_slots_outside_the_pool_are_skipped():
    rng = np.random.default_rng(1)
    x = rand(rng, (3, 2, 64), "bfloat16")
    c = _cache(8, 2, 64, "bfloat16")
    assert _device_error() == 0
    c.store_kv(to_dev(x, "bfloat16"), to_dev(x, "bfloat16"), _i32([2, 8, -1]), 0)
    assert _device_error() == 32
    rows = c.rows(0).cpu().numpy()
    np.testing.assert_array_equal(rows[2], F.pack_rows(x, x)[0])
    assert (np.delete(rows, 2, 0) == 0).all()
    k, v = c.load_kv(_i32([2, 99]), 0)
    assert _device_error() == 32
    np.testing.assert_array_equal(k[0].float().cpu().numpy(), F.roundtrip(x)[0])
    assert (k[1] == 0).all() and (v[1] == 0).all()


def test_offsets_past_32_bits():
    """A pool of more than 2^32 bytes: the last slot's row is at a 33-bit offset."""
    import torch

    n = (1 << 32) // 1168 + 1000
    c = _cache(n, 8, 128, "bfloat16")
    rng = np.random.default_rng(2)
    k, v = rand(rng, (2, 8, 128), "bfloat16"), rand(rng, (2, 8, 128), "bfloat16")
    loc = _i32([n - 1, 0])
    c.store_kv(to_dev(k, "bfloat16"), to_dev(v, "bfloat16"), loc, 0)
    gk, gv = c.load_kv(loc, 0)
    np.testing.assert_array_equal(gk.float().cpu().numpy(), F.roundtrip(k))
    np.testing.assert_array_equal(gv.float().cpu().numpy(), F.roundtrip(v))
    # decode over one 64-slot page at the end of the pool
    q = to_dev(rand(rng, (1, 16, 128), "bfloat16"), "bfloat16")
    from minisgl_b200 import B200AttnBackend

    m = (n // 64 - 1) * 64
    fill = _i32(np.arange(m, m + 64))
    kk, vv = rand(rng, (64, 8, 128), "bfloat16"), rand(rng, (64, 8, 128), "bfloat16")
    c.store_kv(to_dev(kk, "bfloat16"), to_dev(vv, "bfloat16"), fill, 0)
    table = np.arange(m, m + 64, dtype=np.int32)[None]
    be = B200AttnBackend(HeadConfig(16, 8, 128), c, table, 64)
    out = be.forward_decode(q, 0, be.decode_metadata_from_lens(np.array([0]), np.array([61])))
    ref, A, X, S = F.attend(q.float().cpu().numpy().astype(np.float64), F.roundtrip(kk)[:61], F.roundtrip(vv)[:61],
                         be.scale, 60)
    assert (np.abs(out.float().cpu().numpy() - ref) <= F.tolerance(ref, A, X, S, "bfloat16", 128, 61)).all()
    del c, be
    torch.cuda.empty_cache()


# ------------------------------------------------------------------ attention
class Pool:
    """A filled 4-bit pool with a fragmented page table, and its rows' exact values."""

    def __init__(self, lens, Hkv, D, dtype, P, seed, spike=0.0, gk=1.0, gv=1.0):
        import torch

        rng = np.random.default_rng(seed)
        self.rng = rng
        lens = np.asarray(lens, dtype=np.int64)
        n = int(((lens + P - 1) // P).sum() + 7) * P
        self.pb = W.allocate_pages(lens, n, P, rng)
        k = rand(rng, (n, Hkv, D), dtype) * np.exp(0.4 * rng.standard_normal((Hkv, D)))
        k = k * (1 + spike * (rng.random((n, Hkv, 1)) < 0.01))
        v = rand(rng, (n, Hkv, D), dtype)
        kd, vd = to_dev(k * gk, dtype), to_dev(v * gv, dtype)
        self.cache = _cache(n, Hkv, D, dtype, k_scale=gk, v_scale=gv)
        # garbage in every slot first (a slot's last user), then the rows
        self.cache.buffer.copy_(torch.randint(0, 255, self.cache.buffer.shape, dtype=torch.uint8, device="cuda"))
        self.cache.store_kv(kd, vd, _i32(np.arange(n)), 0)
        self.k = F.roundtrip(kd.double().cpu().numpy(), gk)
        self.v = F.roundtrip(vd.double().cpu().numpy(), gv)

    def of(self, b):
        s = self.pb.page_table[b, : int(self.pb.lens[b])]
        return self.k[s], self.v[s]


def _check(got, refs, dtype, D, L):
    got = got.double().cpu().numpy()
    ref, A, X, S = (np.concatenate(x) for x in zip(*refs))
    err, tol = np.abs(got - ref), F.tolerance(ref, A, X, S, dtype, D, L)
    assert np.isfinite(got).all()
    worst = np.unravel_index(np.argmax(err - tol), err.shape)
    assert (err <= tol).all(), (worst, err[worst], tol[worst], got[worst], ref[worst])


DECODE_SHAPES = [(16, 8, 128), (8, 8, 128), (32, 8, 128), (64, 8, 128), (3, 1, 128), (4, 1, 128), (16, 2, 128),
                 (12, 4, 128), (32, 16, 128), (4, 2, 64), (16, 16, 64), (64, 8, 64), (16, 8, 256), (8, 1, 256),
                 (16, 16, 256), (14, 2, 256)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("Hq,Hkv,D", DECODE_SHAPES)
def test_decode_shapes(Hq, Hkv, D, dtype):
    from minisgl_b200 import B200AttnBackend

    lens = [1, 0, 15, 16, 17, 33, 300, 129]
    p = Pool(lens, Hkv, D, dtype, 16, seed=Hq + Hkv + D)
    q = rand(p.rng, (len(lens), Hq, D), dtype)
    be = B200AttnBackend(HeadConfig(Hq, Hkv, D), p.cache, p.pb.page_table, 16)
    meta = be.decode_metadata_from_lens(p.pb.rows, p.pb.lens)
    out = be.forward_decode(to_dev(q, dtype), 0, meta)
    refs = [F.attend(q[b:b + 1].astype(np.float64), *p.of(b), be.scale, L - 1) for b, L in enumerate(lens)]
    _check(out, refs, dtype, D, max(lens))
    assert (out[1] == 0).all()  # no tokens: a row of zeros
    assert _device_error() == 0


@pytest.mark.parametrize("P", [1, 2, 16, 64, 512])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_decode_page_sizes_and_splits(P, dtype):
    """Long requests split over CTAs (few CTAs and many), pages that end inside a stage."""
    from minisgl_b200 import B200AttnBackend

    Hq, Hkv, D = 16, 8, 128
    lens = [2500, 7, 1024, 63, 641]
    p = Pool(lens, Hkv, D, dtype, P, seed=P)
    q = rand(p.rng, (len(lens), Hq, D), dtype)
    be = B200AttnBackend(HeadConfig(Hq, Hkv, D), p.cache, p.pb.page_table, P)
    refs = [F.attend(q[b:b + 1].astype(np.float64), *p.of(b), be.scale, L - 1) for b, L in enumerate(lens)]
    for nc in (None, 3, 1, 31):
        meta = be.decode_metadata_from_lens(p.pb.rows, p.pb.lens, num_ctas=nc)
        out = be.forward_decode(to_dev(q, dtype), 0, meta)
        again = be.forward_decode(to_dev(q, dtype), 0, meta)
        _check(out, refs, dtype, D, max(lens))
        assert bool((out == again).all()), "decode is not repeatable"
    assert _device_error() == 0


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_decode_magnitudes(dtype):
    """Spiky keys (the maximum moves late), tiny and huge queries, pool scales away from one."""
    from minisgl_b200 import B200AttnBackend

    Hq, Hkv, D = 8, 4, 128
    lens = [700, 90, 33, 200]
    for gk, gv, amp in ((1.0, 1.0, 1.0), (2.0 ** -10, 64.0, 2.0 ** 10), (4.0, 2.0 ** -20, 2.0 ** -40)):
        p = Pool(lens, Hkv, D, dtype, 16, seed=3, spike=12.0, gk=gk, gv=gv)
        q = rand(p.rng, (len(lens), Hq, D), dtype) * np.float32(amp)
        q[0, 0] = 0
        q[1, :, 5] *= 2.0 ** 12
        be = B200AttnBackend(HeadConfig(Hq, Hkv, D), p.cache, p.pb.page_table, 16)
        out = be.forward_decode(to_dev(q, dtype), 0, be.decode_metadata_from_lens(p.pb.rows, p.pb.lens))
        qd = to_dev(q, dtype).double().cpu().numpy()
        refs = [F.attend(qd[b:b + 1], *p.of(b), be.scale, L - 1) for b, L in enumerate(lens)]
        _check(out, refs, dtype, D, max(lens))


EXTEND_SHAPES = [(16, 8, 128), (8, 8, 128), (32, 8, 128), (8, 1, 128), (4, 2, 64), (8, 8, 64),
                 (16, 2, 64), (4, 2, 256), (16, 2, 256)]


def _extend_case(Hq, Hkv, D, dtype, P, lens, ext, seed, **kw):
    from minisgl_b200 import B200AttnBackend

    p = Pool(lens, Hkv, D, dtype, P, seed=seed, **kw)
    lens, ext = np.asarray(lens), np.asarray(ext)
    q = rand(p.rng, (int(ext.sum()), Hq, D), dtype)
    return p, lens, ext, q, B200AttnBackend(HeadConfig(Hq, Hkv, D), p.cache, p.pb.page_table, P)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("Hq,Hkv,D", EXTEND_SHAPES)
def test_extend_shapes(Hq, Hkv, D, dtype):
    lens, ext = [1, 40, 130, 17, 300, 129], [1, 40, 2, 16, 77, 1]
    p, lens, ext, q, be = _extend_case(Hq, Hkv, D, dtype, 16, lens, ext, seed=Hq + D)
    meta = be.extend_metadata_from_lens(p.pb.rows, lens, ext)
    out = be._forward_prefill(to_dev(q, dtype), None, None, 0, meta)
    refs, o = [], 0
    for b, (L, n) in enumerate(zip(lens, ext)):
        refs.append(F.attend(q[o:o + n].astype(np.float64), *p.of(b), be.scale, L - n))
        o += n
    _check(out, refs, dtype, D, int(lens.max()))
    assert _device_error() == 0


@pytest.mark.parametrize("P", [1, 4, 16, 64])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_extend_page_sizes(P, dtype):
    """Tiles and key blocks that end anywhere, few new tokens on long prefixes, a long first prompt."""
    Hq, Hkv, D = 16, 8, 128
    lens, ext = [900, 5, 270, 1500, 128], [3, 5, 270, 1, 128]
    p, lens, ext, q, be = _extend_case(Hq, Hkv, D, dtype, P, lens, ext, seed=P, spike=6.0)
    meta = be.extend_metadata_from_lens(p.pb.rows, lens, ext)
    out = be._forward_prefill(to_dev(q, dtype), None, None, 0, meta)
    again = be._forward_prefill(to_dev(q, dtype), None, None, 0, meta)
    assert bool((out == again).all()), "extend is not repeatable"
    refs, o = [], 0
    for b, (L, n) in enumerate(zip(lens, ext)):
        refs.append(F.attend(q[o:o + n].astype(np.float64), *p.of(b), be.scale, L - n))
        o += n
    _check(out, refs, dtype, D, int(lens.max()))
    assert _device_error() == 0


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("Hq,Hkv,D", [(2, 1, 128), (4, 1, 64), (2, 2, 256), (8, 1, 128)])
def test_extend_long_prompts_in_runs(Hq, Hkv, D, dtype):
    """One long prompt: tiles whose keys are cut into runs, the first tile of a pair needing fewer
    blocks than the second, and a last run shorter than the others."""
    for L, n, run_keys in ((1500, 250, None), (1500, 250, 128), (900, 900, 640), (2049, 65, 256)):
        p, lens, ext, q, be = _extend_case(Hq, Hkv, D, dtype, 16, [L], [n], seed=L + D, spike=4.0)
        meta = be.extend_metadata_from_lens(p.pb.rows, lens, ext)
        if run_keys is None:
            assert meta.n_split > 1
        else:
            _force_runs(be, meta, run_keys, -(-L // run_keys))
        out = be._forward_prefill(to_dev(q, dtype), None, None, 0, meta)
        again = be._forward_prefill(to_dev(q, dtype), None, None, 0, meta)
        assert bool((out == again).all()), "extend is not repeatable"
        _check(out, [F.attend(q.astype(np.float64), *p.of(0), be.scale, L - n)], dtype, D, L)
    assert _device_error() == 0


def _force_runs(be, meta, run_keys, n_split):
    """Another cut of the same work items, with a workspace for it."""
    import torch

    from minisgl_b200 import _native as nat

    meta.run_keys, meta.n_split = run_keys, n_split
    n = int(nat.LIB.b2a_fp4_extend_workspace_bytes(meta.n_work, n_split, be.Hkv, be.D))
    meta.workspace = torch.zeros(n, dtype=torch.uint8, device="cuda")


def test_a_bad_page_is_reported():
    from minisgl_b200 import B200AttnBackend

    p = Pool([64, 32], 8, 128, "bfloat16", 16, seed=9)
    table = p.pb.page_table.copy()
    table[0, 16:32] = np.arange(16) + (p.cache.num_tokens // 16 + 3) * 16
    be = B200AttnBackend(HeadConfig(16, 8, 128), p.cache, table, 16)
    assert _device_error() == 0
    q = to_dev(rand(p.rng, (2, 16, 128), "bfloat16"), "bfloat16")
    out = be.forward_decode(q, 0, be.decode_metadata_from_lens(p.pb.rows, p.pb.lens))
    assert _device_error() == 32
    ref, A, X, S = F.attend(q[1:].double().cpu().numpy(), *p.of(1), be.scale, 31)
    assert (np.abs(out[1:].double().cpu().numpy() - ref) <= F.tolerance(ref, A, X, S, "bfloat16", 128, 32)).all()
    be._forward_prefill(q, None, None, 0, be.extend_metadata_from_lens(p.pb.rows, p.pb.lens, np.array([1, 1])))
    assert _device_error() == 32


def test_bad_tiles_are_skipped():
    """A work list with a request out of range, or with more tokens than q has rows, stays in bounds."""
    from minisgl_b200 import B200AttnBackend

    p = Pool([64, 32], 8, 128, "bfloat16", 16, seed=9)
    be = B200AttnBackend(HeadConfig(16, 8, 128), p.cache, p.pb.page_table, 16)
    q = to_dev(rand(p.rng, (2, 16, 128), "bfloat16"), "bfloat16")
    want = be._forward_prefill(q, None, None, 0, be.extend_metadata_from_lens(p.pb.rows, p.pb.lens, np.array([1, 1])))
    for i, bad, code in ((0, 7, 35), (0, -1, 35), (2, 9, 33)):
        meta = be.extend_metadata_from_lens(p.pb.rows, p.pb.lens, np.array([1, 1]))
        last = int((meta.work[:, 0] == 1).nonzero()[0])  # request 1's tile
        meta.work[last, i] = bad
        assert _device_error() == 0
        out = be._forward_prefill(q, None, None, 0, meta)
        assert _device_error() == code
        assert bool((out[0] == want[0]).all())


def test_python_refusals():
    import torch

    from minisgl_b200 import B200AttnBackend

    p = Pool([20, 20], 8, 128, "bfloat16", 16, seed=1)
    c = p.cache
    be = B200AttnBackend(HeadConfig(16, 8, 128), c, p.pb.page_table, 16)
    x = torch.zeros(2, 8, 128, dtype=torch.bfloat16, device="cuda")
    loc = _i32([0, 1])
    for k, v, l in ((x.float(), x, loc), (x, x[:1], loc), (x.cpu(), x, loc), (x, x, loc.long()), (x, x, loc[:1]),
                    (x, x, loc.cpu()), (x, x, _i32([0, 1, 2, 3])[::2]), (x.transpose(0, 1)[:2], x, loc)):
        with pytest.raises(ValueError):
            c.store_kv(k, v, l, 0)
    with pytest.raises(ValueError):
        c.load_kv(loc.long(), 0)
    meta = be.decode_metadata_from_lens(p.pb.rows, p.pb.lens)
    with pytest.raises(ValueError):
        be.forward_decode(torch.zeros(2, 16, 128, device="cuda"), 0, meta)
    with pytest.raises(ValueError):
        be.forward_decode(torch.zeros(2, 16, 128, dtype=torch.bfloat16), 0, meta)


def test_side_stream_and_graph():
    """Store and decode captured on a side stream and replayed with new inputs give the eager bytes."""
    import torch

    from minisgl_b200 import B200AttnBackend

    p = Pool([500, 20, 1, 64], 8, 128, "bfloat16", 16, seed=21)
    be = B200AttnBackend(HeadConfig(16, 8, 128), p.cache, p.pb.page_table, 16)
    meta = be.decode_metadata_from_lens(p.pb.rows, p.pb.lens)
    loc = _i32([p.pb.page_table[b, int(L) - 1] for b, L in enumerate(p.pb.lens)])
    q = torch.zeros(4, 16, 128, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(4, 8, 128, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)

    def step():
        p.cache.store_kv(k, v, loc, 0)
        return be.forward_decode(q, 0, meta)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for seed in (1, 2, 3):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=gen, device="cuda"))
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert bool((step() == got).all())


# ------------------------------------------------------------------ together, as a serving step uses them
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_attention_layer_over_the_pool(dtype):
    """Norm, rotation, store and attention through AttentionLayer: prefill of two chunks, then a decode step,
    against attention over what the pool then holds."""
    import torch

    from minisgl_b200 import AttentionLayer, B200AttnBackend, Batch, Context, Req, RotaryConfig, set_global_ctx
    from minisgl_b200.core import batch_positions_out_loc

    Hq, Hkv, D, P = 16, 8, 128, 16
    rng = np.random.default_rng(4)
    total = [75, 40]
    pb = W.allocate_pages(np.array(total) + 1, 1024, P, rng)
    cache = _cache(1024, Hkv, D, dtype)
    ctx = Context(page_size=P)
    ctx.page_table, ctx.kv_cache = pb.page_table, cache
    be = B200AttnBackend(HeadConfig(Hq, Hkv, D), cache, pb.page_table, P)
    ctx.attn_backend = be
    set_global_ctx(ctx)
    layer = AttentionLayer(0, Hq, Hkv, D, RotaryConfig(D, D, 1e6, 40960))
    plain = AttentionLayer(0, Hq, Hkv, D, RotaryConfig(D, D, 1e6, 40960))
    nw = to_dev(1 + 0.1 * rng.standard_normal(D), dtype)
    done = [0, 0]
    for phase, upto in (("prefill", [50, 7]), ("prefill", [75, 40]), ("decode", [76, 41])):
        reqs = []
        for b in range(2):
            r = Req(np.zeros(upto[b], np.int32), table_idx=b, cached_len=done[b], output_len=4)
            reqs.append(r)
        batch = Batch(reqs, phase)
        pos, loc = batch_positions_out_loc(batch, pb.page_table)
        batch.positions, batch.out_loc = _i32(pos), _i32(loc)
        be.prepare_metadata(batch)
        T = len(pos)
        qkv = to_dev(rand(rng, (T, (Hq + 2 * Hkv) * D), dtype), dtype)
        q = qkv[:, : Hq * D].view(T, Hq, D)
        k = qkv[:, Hq * D: (Hq + Hkv) * D].view(T, Hkv, D)
        v = qkv[:, (Hq + Hkv) * D:].view(T, Hkv, D)
        q2, k2, v2 = q.clone(), k.clone(), v.clone()
        with ctx.forward_batch(batch):
            out = layer(q, k, v, nw, nw).view(T, Hq, D)
        # the same norm and rotation with a 16/32-bit pool give the rows that were quantised
        from minisgl_b200 import MHAKVCache

        dense = MHAKVCache(1, 1024, Hkv, D, torch_dtype(dtype))
        qo = torch.empty_like(q2)
        plain.rotary.rope_store_(q2, k2, v2, batch.positions, batch.out_loc, dense, 0, nw, nw, q_out=qo)
        gk, gv = cache.load_kv(batch.out_loc, 0)
        np.testing.assert_array_equal(gk.float().cpu().numpy(), F.roundtrip(k2.float().cpu().numpy()))
        np.testing.assert_array_equal(gv.float().cpu().numpy(), F.roundtrip(v2.float().cpu().numpy()))
        refs, o = [], 0
        for b in range(2):
            n = upto[b] - done[b]
            kk, vv = cache.load_kv(_i32(pb.page_table[b, : upto[b]]), 0)
            refs.append(F.attend(qo[o:o + n].double().cpu().numpy(), kk.double().cpu().numpy(), vv.double().cpu().numpy(),
                                 be.scale, done[b]))
            o += n
            done[b] = upto[b]
        _check(out, refs, dtype, D, 76)
    assert _device_error() == 0
