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
    """Pages of `page_size` slots, a head's slots one after another:

      k, v                 (pages, Hkv, page_size, width / 2) uint8, element 2 i in the low half of byte i; width:
                           head_dim in whole groups of 32
      k_scales, v_scales   (pages, Hkv, page_size, width / 32) uint8, 2^(byte - 127), 255 NaN

    zero in a new pool (all values 0). `of` takes arrays that are there already."""

    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, device="cuda"):
        import torch
        if num_pages < 0 or num_kv_heads <= 0 or head_dim <= 0:
            raise ValueError("num_pages must not be negative, num_kv_heads and head_dim positive")
        w = -(-head_dim // GROUP)
        new = [torch.zeros((num_pages, num_kv_heads, page_size, n), dtype=torch.uint8, device=device)
               for n in (16 * w, w, 16 * w, w)]
        self._take(*new, head_dim)

    @classmethod
    def of(cls, k, k_scales, v, v_scales, head_dim: int) -> "KV4Pool":
        """A pool on these four tensors (in the layout above, contiguous)."""
        self = cls.__new__(cls)
        self._take(k, k_scales, v, v_scales, head_dim)
        return self

    def _take(self, k, ks, v, vs, d):
        import torch
        w = -(-d // GROUP)
        if k.dim() != 4 or k.shape[3] != 16 * w:
            raise ValueError(f"k must be (pages, heads, page_size, {16 * w})")
        pages, heads, P, _ = k.shape
        for name, t, n in (("k", k, 16 * w), ("k_scales", ks, w), ("v", v, 16 * w), ("v_scales", vs, w)):
            if t.dtype != torch.uint8 or tuple(t.shape) != (pages, heads, P, n) or not t.is_contiguous() or t.device != k.device:
                raise ValueError(f"{name} must be a contiguous uint8 tensor ({pages}, {heads}, {P}, {n}) on {k.device}")
        if d <= 0 or d % 8:
            raise ValueError("head_dim must be a multiple of 8")
        if P <= 0 or P & (P - 1) or P < 16:
            raise ValueError("page_size must be a power of two of 16 slots or more")
        if k.data_ptr() % 16 or v.data_ptr() % 16:
            raise ValueError("k and v must start on 16 bytes")
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
        shape = (self.num_pages, self.Hkv, self.page_size, self.head_dim)
        out = []
        with torch.cuda.device(self.dev):
            for codes, scales in ((self.k, self.k_scales), (self.v, self.v_scales)):
                x = torch.empty(shape, dtype=torch.bfloat16, device=self.dev)
                hip._check(hip.load().ea_hip_kv4_values(x.numel() // self.head_dim, self.head_dim, codes.data_ptr(), scales.data_ptr(),
                                                        x.data_ptr(), hip._stream_ptr(torch)), "ea_hip_kv4_values")
                out.append(x)
        return tuple(out)

    def append(self, k, v, dst_rows) -> None:
        """k and v (tokens, Hkv, head_dim), bf16 (or int16) or fp32 with any strides over tokens and heads, to rows
        dst_rows (int64, page * page_size + slot; rows outside the pool, such as -1, are skipped; a row may be named once).
        Rotary.append turns and norms k on the way."""
        from .step import append_kv4
        append_kv4(self, k, v, dst_rows)
