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

import ctypes
import math

import numpy as np

from . import hip

PLAN_SEQS, PLAN_ROWS = 8192, 65536  # sequences of a plan, rows of its block table

PLAN_STATUS = {1: "out of pages", 2: "a sequence longer than its table row or max_seq_len",
               4: "more tokens than max_tokens or than pad_tokens of a sequence",
               8: "a negative length or count, or a table row outside the table or used twice"}


def _call(fn, args, index: int, what: str) -> None:
    """One launch on torch's current stream of device `index`, made current when it is not."""
    import torch
    C = torch._C
    if C._cuda_getDevice() == index:
        rc = fn(ctypes.byref(args), C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(ctypes.byref(args), C._cuda_getCurrentRawStream(index))
    if rc:
        raise ValueError(f"{what}: error code {rc}")


def _vec(t, name, index, dtype, n=None):
    """The address of a contiguous tensor of this type on this device (of n entries)."""
    if t.dtype is not dtype or not t.is_cuda or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor on cuda:{index}")
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
        if num_seqs > PLAN_SEQS or num_seqs * pad_tokens >= 1 << 31 or max_tokens >= 1 << 31:
            raise ValueError(f"at most {PLAN_SEQS} sequences, and fewer than 2^31 tokens and padded rows")
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
        self._lib, self._i32 = hip.load().ea_hip_step_plan, i32
        self._fixed = bytes(hip.StepPlanArgs(
            num_seqs=num_seqs, max_tokens=max_tokens, pad_tokens=pad_tokens, dst_rows=self.dst_rows.data_ptr(),
            positions=self.positions.data_ptr(), seq_of=self.seq_of.data_ptr(), q_rows=self.q_rows.data_ptr(),
            kv_len=self.kv_len.data_ptr(), new_seq_len=self.seq_len.data_ptr(), new_num_free=self.num_free.data_ptr(),
            status=self.status.data_ptr()))

    def build(self, seq_len, counts, block_table, free_pages, num_free, page_size: int, *, slots=None,
              max_seq_len: int | None = None) -> None:
        """seq_len, counts: (num_seqs,) int32; block_table: (rows, width) int32, its rows those of `slots`
        (int32; None: row b) grown in place; free_pages: the stack's int32 array, num_free its height (a
        one-entry int32 tensor). max_seq_len: bound of the lengths (None: what a table row holds). The
        outputs must not be passed in as the inputs of the same build: copy them (or use two plans in
        turn)."""
        if block_table.dim() != 2:
            raise ValueError("block_table must be (rows, width)")
        rows, width = block_table.shape
        if page_size <= 0 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two")
        if rows > PLAN_ROWS:
            raise ValueError(f"at most {PLAN_ROWS} block table rows")
        B, i32, at = self.num_seqs, self._i32, self.dev.index
        a = hip.StepPlanArgs.from_buffer_copy(self._fixed)
        a.page_size, a.table_rows, a.table_width = page_size, rows, width
        a.max_seq_len = 0x7FFFFFFF if max_seq_len is None else int(max_seq_len)
        a.free_capacity = free_pages.numel()
        a.seq_len = _vec(seq_len, "seq_len", at, i32, B)
        a.counts = _vec(counts, "counts", at, i32, B)
        if slots is not None:
            a.slots = _vec(slots, "slots", at, i32, B)
        a.free_pages = _vec(free_pages, "free_pages", at, i32)
        a.num_free = _vec(num_free, "num_free", at, i32, 1)
        a.block_table = _vec(block_table, "block_table", at, i32)
        _call(self._lib, a, at, "ea_hip_step_plan")

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
        self._lib = hip.load().ea_hip_rotary
        self._bits, self._f32 = (torch.bfloat16, torch.int16), torch.float32
        self._fixed = bytes(hip.RotaryArgs(head_dim=head_dim, rot_dim=rot, num_axes=self.axes, adjacent=self.adjacent,
                                           scale=self.scale, half_turns=self.half_turns.data_ptr(),
                                           axis_of_pair=self.axis_of_pair.data_ptr()))

    def _tokens(self, x, name, n=None, dtypes=None):
        """Checks a (tokens, heads, head_dim) tensor, int16 standing for bf16 bits: (tokens, heads, fp32, strides)."""
        if x.dim() != 3:
            raise ValueError(f"{name} must be (tokens, heads, {self.head_dim})")
        m, h, d = x.shape
        st = x.stride()
        if d != self.head_dim or (n is not None and m != n):
            raise ValueError(f"{name} must be (tokens, heads, {self.head_dim}), one row per token")
        wide = x.dtype is self._f32
        if not (wide or x.dtype in self._bits) or not x.is_cuda or x.get_device() != self.dev.index:
            raise ValueError(f"{name} must be bf16 (or int16 bit patterns) or fp32 on {self.dev}")
        if st[2] != 1 and m * h:
            raise ValueError(f"{name} needs a contiguous last dimension")
        return m, h, wide, st

    def _target(self, x, name):
        """_tokens of a tensor to be written, whose rows must not share memory."""
        m, h, wide, st = self._tokens(x, name)
        end = self.head_dim
        for stride, size in sorted(((st[0], m), (st[1], h))):
            if size > 1:
                if stride < end:
                    raise ValueError(f"{name} has rows that share memory")
                end += stride * (size - 1)
        return m, h, wide, st

    def _args(self, q, k, v, positions):
        """The arguments that the inputs give, checked; (arguments, fp32, tokens, Hq, Hkv)."""
        import torch
        n, hq, wide, sq = self._tokens(q, "q")
        _, hk, wk, sk = self._tokens(k, "k", n)
        a = hip.RotaryArgs.from_buffer_copy(self._fixed)
        if v is not None:
            _, hv, wv, sv = self._tokens(v, "v", n)
            if hv != hk:
                raise ValueError("k and v must have the same heads")
            wk = wk if wv == wk else None
            a.v, a.v_tok_stride, a.v_head_stride = v.data_ptr(), sv[0], sv[1]
        if wk is not wide:
            raise ValueError("q, k and v must have one type")
        if positions.dtype is not torch.int32 or not positions.is_cuda or positions.get_device() != self.dev.index:
            raise ValueError(f"positions must be int32 on {self.dev}")
        shape, sp = tuple(positions.shape), positions.stride()
        if shape != (n,) if len(shape) == 1 else (len(shape) != 2 or shape[1] != n or shape[0] < self.axes):
            raise ValueError(f"positions must be ({self.axes}, {n}) or, for one axis, ({n},)")
        if (len(shape) == 1 and self.axes > 1) or (n > 1 and sp[-1] != 1):
            raise ValueError(f"positions must be ({self.axes}, {n}), each axis contiguous")
        a.num_tokens, a.num_q_heads, a.num_kv_heads, a.in_fp32 = n, hq, hk, wide
        a.q_tok_stride, a.q_head_stride, a.k_tok_stride, a.k_head_stride = sq[0], sq[1], sk[0], sk[1]
        a.pos_axis_stride = sp[0] if len(shape) == 2 else 0
        a.q, a.k, a.positions = q.data_ptr(), k.data_ptr(), positions.data_ptr()
        return a, wide, n, hq, hk

    def rotate(self, q, k, positions, *, inverse: bool = False, q_out=None, k_out=None):
        """q (tokens, Hq, head_dim) and k (tokens, Hkv, head_dim) turned by positions ((tokens,) or (axes,
        tokens) int32), into new tensors of their type or into q_out and k_out (which may be q and k
        themselves). inverse turns back: the gradient of the rotation. Returns (q_out, k_out)."""
        import torch
        a, wide, n, hq, hk = self._args(q, k, None, positions)
        if q_out is None:
            q_out = torch.empty((n, hq, self.head_dim), dtype=q.dtype, device=self.dev)
        elif q_out.shape != q.shape or q_out.dtype != q.dtype:
            raise ValueError("q_out must have q's shape and type")
        if k_out is None:
            k_out = torch.empty((n, hk, self.head_dim), dtype=k.dtype, device=self.dev)
        elif k_out.shape != k.shape or k_out.dtype != k.dtype:
            raise ValueError("k_out must have k's shape and type")
        so, ko = self._target(q_out, "q_out")[3], self._target(k_out, "k_out")[3]
        a.inverse, a.out_fp32, a.q_out_rows, a.pool_rows = bool(inverse), wide, n, n
        a.q_out, a.qo_tok_stride, a.qo_head_stride = q_out.data_ptr(), so[0], so[1]
        a.k_out, a.ko_tok_stride, a.ko_head_stride = k_out.data_ptr(), ko[0], ko[1]
        _call(self._lib, a, self.dev.index, "ea_hip_rotary")
        return q_out, k_out

    def append(self, q, k, v, positions, dst_rows, k_pool, v_pool, *, q_rows=None, q_out=None, pos_offset: int = 0):
        """A step's tokens into the cache: q and k turned by positions (+ pos_offset), k and v (tokens, Hkv,
        head_dim) to rows dst_rows (int64, page * page_size + slot; rows outside the pool, such as -1, are
        skipped) of the pools [pages, page_size, Hkv, head_dim], bf16. The rotated q goes to a new bf16
        tensor of q's shape, or to rows q_rows (int64; rows outside are skipped) of q_out (rows, Hq,
        head_dim). Returns it. Rows that no token names are not written; a row may be named once."""
        import torch
        a, _, n, hq, hk = self._args(q, k, v, positions)
        if not -1 << 31 <= pos_offset < 1 << 31:
            raise ValueError("pos_offset must fit 32 bits")
        at, d, i64 = self.dev.index, self.head_dim, torch.int64
        shape = k_pool.shape
        for pool, name in ((k_pool, "k_pool"), (v_pool, "v_pool")):
            if pool.dtype not in self._bits or not pool.is_cuda or pool.get_device() != at or not pool.is_contiguous():
                raise ValueError(f"{name} must be a contiguous bf16 (or int16) tensor on {self.dev}")
            if pool.shape != shape:
                raise ValueError("k_pool and v_pool must have one shape")
        if len(shape) != 4 or shape[2] != hk or shape[3] != d:
            raise ValueError(f"the pools must be (pages, page_size, {hk}, {d})")
        if q_out is None:
            if q_rows is not None:
                raise ValueError("q_rows needs q_out")
            q_out = torch.empty((n, hq, d), dtype=torch.bfloat16, device=self.dev)
            rows, so = n, (hq * d, d)
        else:
            rows, ho, wide, so = self._target(q_out, "q_out")
            if q_rows is not None and q_out.data_ptr() == q.data_ptr():
                raise ValueError("q_out must not be q when q_rows moves its rows")
            if wide or ho != hq or (q_rows is None and rows < n):
                raise ValueError("q_out must be (rows, Hq, head_dim) bf16 (or int16), a row per token without q_rows")
        a.dst_rows = _vec(dst_rows, "dst_rows", at, i64, n)
        if q_rows is not None:
            a.q_rows = _vec(q_rows, "q_rows", at, i64, n)
        row = hk * d
        a.pos_offset, a.q_out_rows, a.pool_rows = pos_offset, rows, shape[0] * shape[1]
        a.q_out, a.qo_tok_stride, a.qo_head_stride = q_out.data_ptr(), so[0], so[1]
        a.k_out, a.ko_tok_stride, a.ko_head_stride = k_pool.data_ptr(), row, d
        a.v_out, a.vo_tok_stride, a.vo_head_stride = v_pool.data_ptr(), row, d
        _call(self._lib, a, at, "ea_hip_rotary")
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
