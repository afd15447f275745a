"""A paged K/V cache held in 4 bits, in the microscaling format of 4-bit floats.

An element is a sign, two bits of exponent and one of mantissa (0, 0.5, 1, 1.5, 2, 3, 4, 6), 32 elements share a power of
two. Every value is a bf16, so attention over the cache equals, to the bit, attention over the bf16 cache of its values
(hip.DeviceProblem's "kv4", serving.PagedKVCache(bits=4)). Rotary.append writes it. No reference counterpart: the reference's
caches are bf16 (scripts/spec_decode_demo.py:116-125).
"""

from __future__ import annotations

import ctypes

from . import hip

GROUP = 32  # elements to a scale


class KV4Pool:
    """Pages of `page_size` slots, a head's slots one after another; w is head_dim in whole groups of 32:

      k          (pages, Hkv, page_size, w / 2) uint8, element 2 i of a key in the low half of byte i
      k_scales   (pages, Hkv, page_size, w / 32) uint8, 2^(byte - 127), 255 NaN
      v          (pages, Hkv, page_size / 16, w / 2, 16) uint8: for 16 slots, channels 2 i and 2 i + 1 (its low half the first)
                 of each slot, as the matrix instructions sum over keys
      v_scales   (pages, Hkv, page_size / 16, w / 32, 16) uint8

    zero in a new pool (all values 0). `of` takes arrays that are there already."""

    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, device="cuda"):
        import torch
        if num_pages < 0 or num_kv_heads <= 0 or head_dim <= 0:
            raise ValueError("num_pages must not be negative, num_kv_heads and head_dim positive")
        w = -(-head_dim // GROUP)
        new = [torch.zeros((num_pages, num_kv_heads, page_size, n), dtype=torch.uint8, device=device) for n in (16 * w, w)]
        new += [torch.zeros((num_pages, num_kv_heads, page_size // 16, n, 16), dtype=torch.uint8, device=device) for n in (16 * w, w)]
        self._take(*new, head_dim)

    @classmethod
    def of(cls, k, k_scales, v, v_scales, head_dim: int) -> "KV4Pool":
        """A pool on these four tensors (contiguous), v and v_scales in tiles as above, or, copied then, in rows as k and k_scales
        are."""
        self = cls.__new__(cls)
        tiles = [t.unflatten(2, (-1, 16)).transpose(3, 4).contiguous() if t.dim() == 4 and t.shape[2] % 16 == 0 else t for t in (v, v_scales)]
        self._take(k, k_scales, *tiles, head_dim)
        return self

    def rows(self):
        """k, k_scales, v and v_scales, all in rows: what `of` takes (copies of v's)."""
        return (self.k, self.k_scales, *(t.transpose(3, 4).flatten(2, 3).contiguous() for t in (self.v, self.v_scales)))

    def _take(self, k, ks, v, vs, d):
        import torch
        w = -(-d // GROUP)
        if k.dim() != 4 or k.shape[3] != 16 * w:
            raise ValueError(f"k must be (pages, heads, page_size, {16 * w})")
        pages, heads, P, _ = k.shape
        if P <= 0 or P & (P - 1) or P < 16:
            raise ValueError("page_size must be a power of two of 16 slots or more")
        for name, t, shape in (("k", k, (P, 16 * w)), ("k_scales", ks, (P, w)), ("v", v, (P // 16, 16 * w, 16)),
                               ("v_scales", vs, (P // 16, w, 16))):
            shape = (pages, heads, *shape)
            if t.dtype != torch.uint8 or tuple(t.shape) != shape or not t.is_contiguous() or t.device != k.device:
                raise ValueError(f"{name} must be a contiguous uint8 tensor {shape} on {k.device}")
        if d <= 0 or d % 8:
            raise ValueError("head_dim must be a multiple of 8")
        if k.data_ptr() % 16 or v.data_ptr() % 16 or vs.data_ptr() % 4:
            raise ValueError("k and v must start on 16 bytes, v_scales on 4")
        at = [(t.data_ptr(), t.data_ptr() + t.numel()) for t in (k, ks, v, vs)]
        if any(a[0] < b[1] and b[0] < a[1] for i, a in enumerate(at) for b in at[i + 1:]):
            raise ValueError("the pool's tensors share memory")
        self.k, self.k_scales, self.v, self.v_scales, self.head_dim, self.width = k, ks, v, vs, d, GROUP * w
        self.num_pages, self.Hkv, self.page_size, self.dev = pages, heads, P, k.device

    def geometry(self) -> dict:
        """The cache's part of an ea_geometry."""
        slot = self.width
        head, page = self.page_size * slot, self.Hkv * self.page_size * slot
        return dict(num_kv_heads=self.Hkv, head_dim=self.head_dim, head_dim_v=self.head_dim, page_size=self.page_size,
                    k_page_stride=page, k_slot_stride=slot, k_head_stride=head, v_page_stride=page, v_slot_stride=slot,
                    v_head_stride=head)

    def args(self) -> hip.KV4Args:
        return hip.KV4Args(self.k_scales.data_ptr(), self.v_scales.data_ptr())

    def values(self):
        """The cache's values: k, v (pages, Hkv, page_size, head_dim) bf16, new tensors."""
        import torch
        C = torch._C
        x = self.k.new_empty((2, self.num_pages, self.Hkv, self.page_size, self.head_dim), dtype=torch.bfloat16)
        index, rows = self.dev.index, self.num_pages * self.Hkv * self.page_size
        fn, at = hip.load().ea_hip_kv4_values, x.data_ptr()

        def launch():
            st = C._cuda_getCurrentRawStream(index)
            hip._check(fn(rows, self.head_dim, 0, self.k.data_ptr(), self.k_scales.data_ptr(), at, st), "ea_hip_kv4_values")
            hip._check(fn(rows, self.head_dim, 1, self.v.data_ptr(), self.v_scales.data_ptr(), at + 2 * rows * self.head_dim, st),
                       "ea_hip_kv4_values")

        if C._cuda_getDevice() == index:
            launch()
        else:
            with torch.cuda.device(index):
                launch()
        return x.unbind(0)

    def append(self, k, v, dst_rows) -> None:
        """k and v (tokens, Hkv, head_dim), bf16 (or int16) or fp32 with any strides over tokens and heads, to rows
        dst_rows (int64, page * page_size + slot; rows outside the pool, such as -1, are skipped; a row may be named once).
        Rotary.append turns and norms k on the way."""
        from .step import append_kv4
        append_kv4(self, k, v, dst_rows)
