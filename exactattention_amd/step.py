"""What a serving step does before its attention call: the step plan and the rotary positions.

  StepPlan  where the new tokens go, from lengths that are on the device: block-table growth from a
            stack of free pages, each token's slot in the pool, its position and its visible length
            (ea_hip_step_plan). Lengths and the stack's height go in and come out as device tensors,
            so a loop that keeps them there, or a captured graph, needs no host between its steps.
  Rotary    q and k turned by positions of one or several axes, k and v written into a paged cache in
            the same launch, or the rotation and its inverse alone (ea_hip_rotary).

Both enqueue on torch's current stream of the tensors' device and do not wait. No reference
counterpart: the reference's demo leaves its cache and positions to transformers
(scripts/spec_decode_demo.py:116-125).
"""

from __future__ import annotations

import contextlib
import ctypes
import math

import numpy as np

from . import hip

PLAN_STATUS = {1: "out of pages", 2: "a sequence longer than its table row or max_seq_len",
               4: "more tokens than max_tokens or than pad_tokens of a sequence",
               8: "a negative length or count, or a table row outside the table or used twice"}


def _on(dev):
    """The device made current for a launch, when it is not already."""
    import torch
    if torch.cuda.current_device() == dev.index:
        return contextlib.nullcontext()
    return torch.cuda.device(dev)


def _stream(dev):
    import torch
    return ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)


def _vec(t, name, dev, dtype, n=None):
    if t.dtype != dtype or t.device != dev or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor on {dev}")
    if n is not None and t.numel() != n:
        raise ValueError(f"{name} must have {n} entries, got {t.numel()}")
    return t.data_ptr()


class StepPlan:
    """The plan of a step of num_seqs sequences and up to max_tokens new tokens, pad_tokens of a sequence
    at most. build() writes these tensors, made once here (a captured graph can hold them):

      dst_rows (max_tokens,) int64   pool row of each token, the tokens of sequence 0 first; -1 past the last
      positions, seq_of (max_tokens,) int32   its position and its sequence; -1 past the last
      q_rows (max_tokens,) int64     its row among num_seqs x pad_tokens; -1 past the last
      kv_len (num_seqs, pad_tokens) int32   visible keys of those rows, 0 for rows without a token
      seq_len (num_seqs,) int32, num_free (1,) int32   lengths and free pages after the step
      status (1,) int32              0, or PLAN_STATUS bits: then nothing is appended and no entry of the
                                     block table is written
    """

    def __init__(self, num_seqs: int, max_tokens: int, pad_tokens: int, device="cuda"):
        import torch
        if num_seqs < 0 or max_tokens < 0 or pad_tokens <= 0:
            raise ValueError("num_seqs and max_tokens must not be negative, pad_tokens positive")
        if num_seqs > 8192:
            raise ValueError("at most 8192 sequences")
        dev = torch.empty(0, device=device).device
        if dev.type != "cuda":
            raise ValueError("the step plan runs on the GPU")
        self.dev, self.num_seqs, self.max_tokens, self.pad_tokens = dev, num_seqs, max_tokens, pad_tokens
        i32, i64 = torch.int32, torch.int64
        self.dst_rows = torch.empty(max_tokens, dtype=i64, device=dev)
        self.positions = torch.empty(max_tokens, dtype=i32, device=dev)
        self.seq_of = torch.empty(max_tokens, dtype=i32, device=dev)
        self.q_rows = torch.empty(max_tokens, dtype=i64, device=dev)
        self.kv_len = torch.empty((num_seqs, pad_tokens), dtype=i32, device=dev)
        self.seq_len = torch.empty(num_seqs, dtype=i32, device=dev)
        self.num_free = torch.empty(1, dtype=i32, device=dev)
        self.status = torch.empty(1, dtype=i32, device=dev)

    def build(self, seq_len, counts, block_table, free_pages, num_free, page_size: int, *, slots=None,
              max_seq_len: int | None = None) -> None:
        """seq_len, counts: (num_seqs,) int32; block_table: (rows, width) int32, its rows those of `slots`
        (int32; None: row b) grown in place; free_pages: the stack's int32 array, num_free its height (a
        one-entry int32 tensor). max_seq_len: bound of the lengths (None: what a table row holds). The
        outputs must not be passed in as the inputs of the same build: copy them (or use two plans in
        turn)."""
        import torch
        i32, dev = torch.int32, self.dev
        if block_table.dim() != 2:
            raise ValueError("block_table must be (rows, width)")
        rows, width = block_table.shape
        if page_size <= 0 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two")
        if rows > 65536:
            raise ValueError("at most 65536 block table rows")
        B = self.num_seqs
        a = hip.StepPlanArgs(
            num_seqs=B, page_size=page_size, table_rows=rows, table_width=width, max_tokens=self.max_tokens,
            pad_tokens=self.pad_tokens, max_seq_len=(1 << 31) - 1 if max_seq_len is None else int(max_seq_len),
            free_capacity=free_pages.numel(), seq_len=_vec(seq_len, "seq_len", dev, i32, B),
            counts=_vec(counts, "counts", dev, i32, B), slots=None if slots is None else _vec(slots, "slots", dev, i32, B),
            free_pages=_vec(free_pages, "free_pages", dev, i32), num_free=_vec(num_free, "num_free", dev, i32, 1),
            block_table=_vec(block_table, "block_table", dev, i32), dst_rows=self.dst_rows.data_ptr(),
            positions=self.positions.data_ptr(), seq_of=self.seq_of.data_ptr(), q_rows=self.q_rows.data_ptr(),
            kv_len=self.kv_len.data_ptr(), new_seq_len=self.seq_len.data_ptr(), new_num_free=self.num_free.data_ptr(),
            status=self.status.data_ptr())
        with _on(dev):
            hip._check(hip.load().ea_hip_step_plan(ctypes.byref(a), _stream(dev)), "ea_hip_step_plan")

    def check(self) -> None:
        """Waits for the plan and raises when the step did not fit."""
        st = int(self.status.item())
        if st:
            raise RuntimeError("step plan: " + "; ".join(m for b, m in PLAN_STATUS.items() if st & b))


class Rotary:
    """Rotary positions of heads of head_dim elements, the first rot_dim of them in pairs: (i, i +
    rot_dim / 2), or (2i, 2i + 1) with `adjacent`. Pair i turns by position * inv_freq[i] (default
    base^(-2i / rot_dim)); `scale` multiplies the rotated pairs. With several position axes (time,
    height, width), `sections` gives the pairs of each axis, one axis after another or, `interleaved`,
    dealt in turn; axis_of_pair gives them one by one instead."""

    def __init__(self, head_dim: int, *, base: float = 10000.0, rot_dim: int | None = None, inv_freq=None, sections=None,
                 interleaved: bool = False, axis_of_pair=None, adjacent: bool = False, scale: float = 1.0, device="cuda"):
        import torch
        rot = head_dim if rot_dim is None else rot_dim
        if not 0 < head_dim <= 256 or rot <= 0 or rot > head_dim or rot % 2:
            raise ValueError("head_dim must be at most 256 and rot_dim an even number up to it")
        half = rot // 2
        f = base ** (-np.arange(half, dtype=np.float64) / half) if inv_freq is None else np.asarray(inv_freq, dtype=np.float64)
        if f.shape != (half,) or not np.all(np.isfinite(f)):
            raise ValueError(f"inv_freq must hold {half} finite frequencies")
        if not math.isfinite(scale):
            raise ValueError("scale must be finite")
        if axis_of_pair is not None and sections is not None:
            raise ValueError("give sections or axis_of_pair, not both")
        if sections is not None:
            axis_of_pair = _deal(list(sections), half, interleaved)
        ax = np.zeros(half, np.uint8) if axis_of_pair is None else np.asarray(axis_of_pair)
        if ax.shape != (half,) or ax.min() < 0 or ax.max() > 255:
            raise ValueError(f"axis_of_pair must hold the axis of each of the {half} pairs")
        self.dev = torch.empty(0, device=device).device
        if self.dev.type != "cuda":
            raise ValueError("the rotation runs on the GPU")
        self.head_dim, self.rot_dim, self.adjacent, self.scale = head_dim, rot, bool(adjacent), float(scale)
        self.axes = len(sections) if sections is not None else int(ax.max()) + 1
        self.half_turns = torch.from_numpy(f / math.pi).to(self.dev)
        self.axis_of_pair = torch.from_numpy(ax.astype(np.uint8)).to(self.dev)

    def _tokens(self, x, name, n=None):
        """Checks a (tokens, heads, head_dim) input and returns it, int16 standing for bf16 bits."""
        import torch
        if x.dim() != 3 or x.shape[2] != self.head_dim or (n is not None and x.shape[0] != n):
            raise ValueError(f"{name} must be (tokens, heads, {self.head_dim}), one row per token")
        if x.dtype not in (torch.bfloat16, torch.int16, torch.float32) or x.device != self.dev:
            raise ValueError(f"{name} must be bf16 (or int16 bit patterns) or fp32 on {self.dev}")
        if x.numel() and x.stride(2) != 1:
            raise ValueError(f"{name} needs a contiguous last dimension")
        return x

    def _args(self, q, k, v, positions, inverse, pos_offset):
        import torch
        n = q.shape[0]
        q, k = self._tokens(q, "q"), self._tokens(k, "k", n)
        wide = q.dtype == torch.float32
        if (k.dtype == torch.float32) != wide or (v is not None and (self._tokens(v, "v", n).dtype == torch.float32) != wide):
            raise ValueError("q, k and v must have one type")
        if v is not None and v.shape[1] != k.shape[1]:
            raise ValueError("k and v must have the same heads")
        if positions.dtype != torch.int32 or positions.device != self.dev:
            raise ValueError(f"positions must be int32 on {self.dev}")
        p = positions.unsqueeze(0) if positions.dim() == 1 else positions
        if p.dim() != 2 or p.shape[1] != n or p.shape[0] < self.axes or (n > 1 and p.stride(1) != 1):
            raise ValueError(f"positions must be ({self.axes}, {n}) or, for one axis, ({n},), each axis contiguous")
        a = hip.RotaryArgs(
            num_tokens=n, num_q_heads=q.shape[1], num_kv_heads=k.shape[1], head_dim=self.head_dim, rot_dim=self.rot_dim,
            num_axes=self.axes, adjacent=self.adjacent, inverse=int(bool(inverse)), in_fp32=int(wide), pos_offset=int(pos_offset),
            scale=self.scale, q_tok_stride=q.stride(0), q_head_stride=q.stride(1), k_tok_stride=k.stride(0),
            k_head_stride=k.stride(1), pos_axis_stride=p.stride(0), q=q.data_ptr(), k=k.data_ptr(), positions=p.data_ptr(),
            half_turns=self.half_turns.data_ptr(), axis_of_pair=self.axis_of_pair.data_ptr())
        if v is not None:
            a.v, a.v_tok_stride, a.v_head_stride = v.data_ptr(), v.stride(0), v.stride(1)
        return a

    def _launch(self, a) -> None:
        with _on(self.dev):
            hip._check(hip.load().ea_hip_rotary(ctypes.byref(a), _stream(self.dev)), "ea_hip_rotary")

    def rotate(self, q, k, positions, *, inverse: bool = False, q_out=None, k_out=None):
        """q (tokens, Hq, head_dim) and k (tokens, Hkv, head_dim) turned by positions ((tokens,) or (axes,
        tokens) int32), into new tensors of their type or into q_out and k_out (which may be q and k
        themselves). inverse turns back: the gradient of the rotation. Returns (q_out, k_out)."""
        import torch
        a = self._args(q, k, None, positions, inverse, 0)
        outs = []
        for x, o, name in ((q, q_out, "q_out"), (k, k_out, "k_out")):
            if o is None:
                o = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            elif o.shape != x.shape or self._tokens(o, name).dtype != x.dtype:
                raise ValueError(f"{name} must have the input's shape and type")
            outs.append(o)
        qo, ko = outs
        a.out_fp32 = a.in_fp32
        a.q_out, a.qo_tok_stride, a.qo_head_stride, a.q_out_rows = qo.data_ptr(), qo.stride(0), qo.stride(1), qo.shape[0]
        a.k_out, a.ko_tok_stride, a.ko_head_stride, a.pool_rows = ko.data_ptr(), ko.stride(0), ko.stride(1), ko.shape[0]
        self._launch(a)
        return qo, ko

    def append(self, q, k, v, positions, dst_rows, k_pool, v_pool, *, q_rows=None, q_out=None, pos_offset: int = 0):
        """A step's tokens into the cache: q and k turned by positions (+ pos_offset), k and v (tokens, Hkv,
        head_dim) to rows dst_rows (int64, page * page_size + slot; rows outside the pool, such as -1, are
        skipped) of the pools [pages, page_size, Hkv, head_dim], bf16. The rotated q goes to a new bf16
        tensor of q's shape, or to rows q_rows (int64; rows outside are skipped) of q_out (rows, Hq,
        head_dim). Returns it. Rows that no token names are not written; a row may be named once."""
        import torch
        a = self._args(q, k, v, positions, False, pos_offset)
        n, i64 = a.num_tokens, torch.int64
        for pool, name in ((k_pool, "k_pool"), (v_pool, "v_pool")):
            if pool.dtype not in (torch.bfloat16, torch.int16) or pool.device != self.dev or not pool.is_contiguous():
                raise ValueError(f"{name} must be a contiguous bf16 (or int16) tensor on {self.dev}")
            if pool.dim() != 4 or pool.shape[2:] != k.shape[1:] or pool.shape != k_pool.shape:
                raise ValueError(f"{name} must be (pages, page_size, {k.shape[1]}, {self.head_dim})")
        if q_out is None:
            if q_rows is not None:
                raise ValueError("q_rows needs q_out")
            q_out = torch.empty(q.shape, dtype=torch.bfloat16, device=self.dev)
        elif q_out.dtype not in (torch.bfloat16, torch.int16) or self._tokens(q_out, "q_out").shape[1] != q.shape[1]:
            raise ValueError("q_out must be (rows, Hq, head_dim) bf16 (or int16)")
        elif q_rows is None and q_out.shape[0] < n:
            raise ValueError("q_out has fewer rows than there are tokens")
        a.dst_rows = _vec(dst_rows, "dst_rows", self.dev, i64, n)
        if q_rows is not None:
            a.q_rows = _vec(q_rows, "q_rows", self.dev, i64, n)
        row = k.shape[1] * self.head_dim
        a.q_out, a.qo_tok_stride, a.qo_head_stride, a.q_out_rows = q_out.data_ptr(), q_out.stride(0), q_out.stride(1), q_out.shape[0]
        a.k_out, a.ko_tok_stride, a.ko_head_stride = k_pool.data_ptr(), row, self.head_dim
        a.v_out, a.vo_tok_stride, a.vo_head_stride = v_pool.data_ptr(), row, self.head_dim
        a.pool_rows = k_pool.shape[0] * k_pool.shape[1]
        self._launch(a)
        return q_out


def _deal(sections, half: int, interleaved: bool):
    """The axis of each pair for `sections` pairs per axis: one axis after another, or dealt in turn to
    the axes that still have pairs left."""
    if any(n < 0 for n in sections) or sum(sections) != half:
        raise ValueError(f"sections must be pair counts that add up to {half}")
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    out, a = [], 0
    while len(out) < half:
        if sections[a]:
            out.append(a)
            sections[a] -= 1
        a = (a + 1) % len(sections)
    return out
