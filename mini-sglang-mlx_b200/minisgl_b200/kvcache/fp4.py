"""KV pool held in 4 bits (``FP4KVCache``).

Takes the place of ``MHAKVCache`` (python/minisgl_mlx/kvcache/pool.py:24-54) where the cache,
not the arithmetic, limits how many tokens fit: 4.5 bits per cached value instead of 16 or
32, so a pool of the same bytes holds 3.5 (bf16) or 7 (fp32) times the tokens, and a decode
step reads that much less.

Format. A head row is cut into blocks of 16 features. A block keeps one e4m3 scale
``s = e4m3(min(max|x| / 6, 448))`` and sixteen e2m1 codes of ``x / s`` (0, .5, 1, 1.5, 2, 3, 4,
6 with a sign), both rounded to nearest, ties to even; a stored value stands for
``code * s``. ``k_scale`` / ``v_scale`` (powers of two, default 1) move the range for a model
whose keys or values are far from one: the pool then holds ``x / k_scale``. With the default a
block keeps its accuracy for maxima from about 0.1 to 2688; smaller ones lose bits and vanish
below 0.006. The pool holds finite values only: a NaN is stored as 0 and an infinity as the
largest value of its block (the query of such a token is NaN too, and shows it).

Attention over the pool (``B200AttnBackend`` built on this cache) reads exactly the values
that ``load_kv`` returns. Activations stay in ``dtype``.
"""

from __future__ import annotations

from contextlib import nullcontext

import torch

from .. import _native as nat
from .pool import dtype_code, raw_stream


def on_device(device: torch.device):
    """Make ``device`` current for a launch when it is not (a kernel runs on the current device)."""
    return nullcontext() if torch.cuda.current_device() == device.index else torch.cuda.device(device)


class FP4KVCache:
    def __init__(
        self,
        num_layers: int,
        num_tokens: int,
        num_kv_heads: int,
        head_dim: int,
        dtype: torch.dtype,
        device: torch.device | str | None = None,
        k_scale: float = 1.0,
        v_scale: float = 1.0,
    ) -> None:
        row = int(nat.LIB.b2a_fp4_row_bytes(num_kv_heads, head_dim))
        if row == 0:
            raise ValueError(f"FP4KVCache: {num_kv_heads} kv heads of {head_dim} features (64, 128 or 256) not supported")
        dtype_code(dtype)  # refuses a type the kernels do not take
        for name, s in (("k_scale", k_scale), ("v_scale", v_scale)):
            if not (s > 0 and 2.0 ** -100 <= s <= 2.0 ** 100 and float(s).hex().split("p")[0] == "0x1.0000000000000"):
                raise ValueError(f"FP4KVCache: {name} must be a power of two in [2^-100, 2^100], got {s}")
        if num_layers <= 0 or num_tokens <= 0:
            raise ValueError("FP4KVCache: num_layers and num_tokens must be > 0")
        if not torch.cuda.is_available():
            raise RuntimeError("FP4KVCache needs a CUDA device (no CPU fallback)")
        device = torch.device("cuda") if device is None else torch.device(device)
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        # [layers, slots, row]: a token's K and V of all heads are one run of bytes, a page one run of rows
        self.buffer = torch.zeros((num_layers, num_tokens, row), dtype=torch.uint8, device=device)
        self.num_layers = num_layers
        self.num_tokens = num_tokens
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.dtype = dtype
        self.device = device
        self.row_bytes = row
        self.k_scale = float(k_scale)
        self.v_scale = float(v_scale)
        self._code = dtype_code(dtype)
        self._base = [self.buffer[l].data_ptr() for l in range(num_layers)]

    def rows(self, layer_id: int) -> torch.Tensor:
        """uint8 ``[num_tokens, row_bytes]`` of a layer: the bytes the kernels read."""
        return self.buffer[layer_id]

    def _slots(self, slots: torch.Tensor) -> int:
        if slots.dtype != torch.int32 or slots.dim() != 1 or not slots.is_contiguous() or slots.device != self.device:
            raise ValueError(f"FP4KVCache: slots must be contiguous int32 [n] on {self.device}, got "
                             f"{slots.dtype} {tuple(slots.shape)} on {slots.device}")
        return slots.shape[0]

    def _rows(self, name: str, t: torch.Tensor, T: int) -> int:
        """Element stride between the token rows of k or v ``[T, Hkv, D]``, checked."""
        H, D = self.num_kv_heads, self.head_dim
        if t.shape != (T, H, D) or t.dtype != self.dtype or t.device != self.device:
            raise ValueError(f"FP4KVCache.store_kv: {name} must be {self.dtype} {(T, H, D)} on {self.device}, got "
                             f"{t.dtype} {tuple(t.shape)} on {t.device}")
        row, head, elem = t.stride()
        if T > 0 and (elem != 1 or (H > 1 and head != D)):
            raise ValueError(f"FP4KVCache.store_kv: {name} rows must be [Hkv, D] contiguous")
        return row if T > 1 else H * D

    def store_kv(self, k: torch.Tensor, v: torch.Tensor, out_loc: torch.Tensor, layer_id: int) -> None:
        """Quantise k/v ``[T, Hkv, D]`` into slots ``out_loc`` ``[T]`` (unique, or -1: the row is skipped;
        token rows may be strided)."""
        T = self._slots(out_loc)
        ks, vs = self._rows("k", k, T), self._rows("v", v, T)
        index = self.device.index
        args = (k.data_ptr(), ks, v.data_ptr(), vs, out_loc.data_ptr(), self._base[layer_id], self.num_tokens, T,
                self.num_kv_heads, self.head_dim, self.k_scale, self.v_scale, self._code, raw_stream(index))
        if torch.cuda.current_device() == index:
            rc = nat.LIB.b2a_fp4_store_kv(*args)
        else:
            with torch.cuda.device(index):
                rc = nat.LIB.b2a_fp4_store_kv(*args)
        if rc:
            nat.fail("b2a_fp4_store_kv", rc)

    def load_kv(self, slots: torch.Tensor, layer_id: int) -> tuple[torch.Tensor, torch.Tensor]:
        """The k and v ``[n, Hkv, D]`` that slots ``slots`` ``[n]`` of a layer stand for, in ``dtype``.

        Exact in fp32 and bf16. Rows of slots outside the pool are zero (and device error 32 is set).
        """
        n = self._slots(slots)
        shape = (n, self.num_kv_heads, self.head_dim)
        k = torch.empty(shape, dtype=self.dtype, device=self.device)
        v = torch.empty(shape, dtype=self.dtype, device=self.device)
        index = self.device.index
        args = (self._base[layer_id], self.num_tokens, slots.data_ptr(), n, self.num_kv_heads, self.head_dim,
                self.k_scale, self.v_scale, k.data_ptr(), v.data_ptr(), self._code, raw_stream(index))
        if torch.cuda.current_device() == index:
            rc = nat.LIB.b2a_fp4_load_kv(*args)
        else:
            with torch.cuda.device(index):
                rc = nat.LIB.b2a_fp4_load_kv(*args)
        if rc:
            nat.fail("b2a_fp4_load_kv", rc)
        return k, v

    @property
    def nbytes(self) -> int:
        return self.buffer.numel()
