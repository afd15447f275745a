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
import struct

import numpy as np

from . import hip

PLAN_SEQS, PLAN_ROWS = 8192, 65536  # sequences of a plan, rows of its block table

PLAN_STATUS = {1: "out of pages", 2: "a sequence longer than its table row or max_seq_len",
               4: "more tokens than max_tokens or than pad_tokens of a sequence",
               8: "a negative length or count, or a table row outside the table or used twice"}


# ea_step_plan and ea_rotary as struct formats: a call packs its arguments in one go, where setting the fields of a
# ctypes structure one by one costs about 70 ns each
_PLAN, _ROTARY = struct.Struct("8i14Q"), struct.Struct("11if15q11Q")
assert _PLAN.size == ctypes.sizeof(hip.StepPlanArgs) and _ROTARY.size == ctypes.sizeof(hip.RotaryArgs)


_C = None  # torch's, once a plan or a rotation exists


def _entry(name: str):
    """The C entry point, taking its arguments packed."""
    global _C
    import torch
    _C = torch._C
    fn = hip.load()[name]  # a function object of its own
    fn.argtypes, fn.restype = [ctypes.c_char_p, ctypes.c_void_p], ctypes.c_int
    return fn


def _call(fn, args: bytes, index: int, what: str) -> None:
    """One launch on torch's current stream of device `index`, made current when it is not."""
    if _C._cuda_getDevice() == index:
        rc = fn(args, _C._cuda_getCurrentRawStream(index))
    else:
        import torch
        with torch.cuda.device(index):
            rc = fn(args, _C._cuda_getCurrentRawStream(index))
    if rc:
        raise ValueError(f"{what}: error code {rc}")


_TURN = None


def _turn():
    """The rotation as a differentiable function: its gradient is the rotation back (one launch)."""
    global _TURN
    if _TURN is None:
        import torch

        class Turn(torch.autograd.Function):
            @staticmethod
            def forward(ctx, q, k, positions, rotary, inverse):
                ctx.save_for_backward(positions)
                ctx.rotary, ctx.inverse = rotary, inverse
                ctx.set_materialize_grads(False)
                out = rotary.rotate(q, k, positions, inverse=inverse)
                ctx.mark_non_differentiable(*(o for o, need in zip(out, ctx.needs_input_grad) if not need))
                return out

            @staticmethod
            def backward(ctx, *grads):
                have = [g is not None and need for g, need in zip(grads, ctx.needs_input_grad)]
                if not any(have):
                    return (None,) * 5
                none = grads[have.index(True)][:, :0]  # no heads
                gs = [(g if g.stride(2) == 1 else g.contiguous()) if h else none for g, h in zip(grads, have)]
                out = ctx.rotary.rotate(*gs, *ctx.saved_tensors, inverse=not ctx.inverse)
                return tuple(g if h else None for g, h in zip(out, have)) + (None,) * 3

        _TURN = Turn.apply
    return _TURN


class _At:
    """Rows of memory as numpy sees an array, for its test of shared memory alone: nothing is read."""

    def __init__(self, x, d):
        ptr, n, h, st, sh, e = x
        self.__array_interface__ = dict(data=(ptr, True), shape=(n, h, d * e), strides=(st * e, sh * e, 1), typestr="|u1", version=3)


def _apart(x, y, d: int) -> bool:
    """Whether two sets of rows of d elements, each (address, tokens, heads, their strides in elements, bytes an
    element), have no byte in common."""
    px, n, h, sx, hx, ex = x
    py, m, g, sy, hy, ey = y
    sx, sy, wx, wy = sx * ex, sy * ey, ((h - 1) * hx + d) * ex, ((g - 1) * hy + d) * ey
    if px + (n - 1) * sx + wx <= py or py + (m - 1) * sy + wy <= px:
        return True
    if not (n and h and m and g):
        return True
    # views of one tensor, such as a fused projection: side by side within a token, or within a head's row
    if sx == sy > 0 and wx <= (py - px) % sx <= sx - wy:
        return True
    hx, hy = hx * ex, hy * ey
    if hx == hy > 0 and sx % hx == 0 == sy % hx and d * ex <= (py - px) % hx <= hx - d * ey:
        return True
    try:
        return not np.shares_memory(np.asarray(_At(x, d)), np.asarray(_At(y, d)), max_work=1 << 20)
    except np.exceptions.TooHardError:
        return False


def _same(x, y) -> bool:
    """Whether they are the same rows: the rotation may then be done in place."""
    return x[0] == y[0] and x[5] == y[5] and (x[1] == 1 or x[3] == y[3]) and (x[2] == 1 or x[4] == y[4])


def _vec(t, name, index, dtype, n=None):
    """The address of a contiguous tensor of this type on this device (of n entries)."""
    if t.dtype is not dtype or t.get_device() != index or not t.is_contiguous():  # -1 on the host
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
        self._fn, self._i32, self._at = _entry("ea_hip_step_plan"), i32, dev.index
        self._out = tuple(t.data_ptr() for t in (self.dst_rows, self.positions, self.seq_of, self.q_rows, self.kv_len,
                                                 self.seq_len, self.num_free, self.status))

    def build(self, seq_len, counts, block_table, free_pages, num_free, page_size: int, *, slots=None,
              max_seq_len: int | None = None) -> None:
        """seq_len, counts: (num_seqs,) int32; block_table: (rows, width) int32, its rows those of `slots`
        (int32; None: row b) grown in place; free_pages: the stack's int32 array, num_free its height (a
        one-entry int32 tensor). max_seq_len: bound of the lengths (None: what a table row holds). The
        outputs must not be passed in as the inputs of the same build (it is refused, as any array written that
        shares memory with another one): copy them, or use two plans in turn."""
        if block_table.dim() != 2:
            raise ValueError("block_table must be (rows, width)")
        rows, width = block_table.shape
        if page_size <= 0 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two")
        if rows > PLAN_ROWS:
            raise ValueError(f"at most {PLAN_ROWS} block table rows")
        B, i32, at = self.num_seqs, self._i32, self._at
        longest = 0x7FFFFFFF if max_seq_len is None else int(max_seq_len)
        if not 0 <= longest < 1 << 31:
            raise ValueError("max_seq_len must fit 31 bits")
        _call(self._fn, _PLAN.pack(
            B, page_size, rows, width, self.max_tokens, self.pad_tokens, longest, free_pages.numel(),
            _vec(seq_len, "seq_len", at, i32, B), _vec(counts, "counts", at, i32, B),
            0 if slots is None else _vec(slots, "slots", at, i32, B), _vec(free_pages, "free_pages", at, i32),
            _vec(num_free, "num_free", at, i32, 1), _vec(block_table, "block_table", at, i32), *self._out),
            at, "ea_hip_step_plan")

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
        self._fn, self._at = _entry("ea_hip_rotary"), self.dev.index
        self._bits, self._f32, self._i32, self._i64 = (torch.bfloat16, torch.int16), torch.float32, torch.int32, torch.int64
        self._half, self._axis = self.half_turns.data_ptr(), self.axis_of_pair.data_ptr()

    def _tokens(self, x, name, n=None):
        """Checks a (tokens, heads, head_dim) tensor, int16 standing for bf16 bits: (tokens, heads, fp32, strides)."""
        shape, st = x.shape, x.stride()
        if len(shape) != 3:
            raise ValueError(f"{name} must be (tokens, heads, {self.head_dim})")
        m, h, d = shape
        if d != self.head_dim or (n is not None and m != n):
            raise ValueError(f"{name} must be (tokens, heads, {self.head_dim}), one row per token")
        wide = x.dtype is self._f32
        if not (wide or x.dtype in self._bits) or x.get_device() != self._at:  # -1 on the host
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
        """The inputs, checked: (tokens, Hq, Hkv, fp32, strides of q, k and v in order, the positions' axis stride)."""
        n, hq, wide, sq = self._tokens(q, "q")
        _, hk, wk, sk = self._tokens(k, "k", n)
        sv = (0, 0)
        if v is not None:
            _, hv, wv, sv = self._tokens(v, "v", n)
            if hv != hk:
                raise ValueError("k and v must have the same heads")
            wk = wk if wv == wk else None
        if wk is not wide:
            raise ValueError("q, k and v must have one type")
        if positions.dtype is not self._i32 or positions.get_device() != self._at:
            raise ValueError(f"positions must be int32 on {self.dev}")
        shape, sp = positions.shape, positions.stride()
        if shape != (n,) if len(shape) == 1 else (len(shape) != 2 or shape[1] != n or shape[0] < self.axes):
            raise ValueError(f"positions must be ({self.axes}, {n}) or, for one axis, ({n},)")
        if (len(shape) == 1 and self.axes > 1) or (n > 1 and sp[-1] != 1):
            raise ValueError(f"positions must be ({self.axes}, {n}), each axis contiguous")
        return n, hq, hk, wide, (sq[0], sq[1], sk[0], sk[1], sv[0], sv[1]), sp[0] if len(shape) == 2 else 0

    def _launch(self, n, hq, hk, wide, strides, axis_stride, inverse, offset, so, sk, sv, rows, pool, inputs, outputs):
        """strides: the inputs'; so, sk, sv: of q's, k's and v's output; rows, pool: theirs; inputs: addresses of q, k,
        v and positions, outputs: of q_rows, dst_rows and the outputs."""
        _call(self._fn, _ROTARY.pack(n, hq, hk, self.head_dim, self.rot_dim, self.axes, self.adjacent, inverse, wide,
                                     wide and not sv, offset, self.scale, *strides, so[0], so[1], sk[0], sk[1],
                                     *(sv or (0, 0)), axis_stride, rows, pool, *inputs, self._half, self._axis, *outputs),
              self._at, "ea_hip_rotary")

    def _check_memory(self, q, k, q_out, k_out):
        """rotate's outputs (None: a new one) are their own input, or share no memory with the inputs and each other."""
        d = self.head_dim
        q_in, k_in = q_out is not None and _same(q_out, q), k_out is not None and _same(k_out, k)
        if q_out and not ((q_in or _apart(q_out, q, d)) and _apart(q_out, k, d)):
            raise ValueError("q_out shares memory with k, or with q without being q")
        if k_out and not ((k_in or _apart(k_out, k, d)) and (q_in or _apart(k_out, q, d)) and
                          (k_in or not q_out or _apart(q_out, k_out, d))):
            raise ValueError("k_out shares memory with q or q_out, or with k without being k")

    def rotate(self, q, k, positions, *, inverse: bool = False, q_out=None, k_out=None):
        """q (tokens, Hq, head_dim) and k (tokens, Hkv, head_dim) turned by positions ((tokens,) or (axes,
        tokens) int32), into new tensors of their type or into q_out and k_out (which may be q and k
        themselves). inverse turns back: the gradient of the rotation. Returns (q_out, k_out). Gradients of q
        and k pass through, with q_out and k_out not given."""
        if (q.requires_grad or k.requires_grad) and _C.is_grad_enabled():
            if q_out is not None or k_out is not None:
                raise ValueError("q_out and k_out take no part in gradients: leave them out, or call under no_grad")
            return _turn()(q, k, positions, self, bool(inverse))
        n, hq, hk, wide, strides, axis_stride = self._args(q, k, None, positions)
        d = self.head_dim
        given = q_out is not None, k_out is not None
        if not given[0]:
            q_out, so = q.new_empty((n, hq, d)), (hq * d, d)
        elif q_out.shape != q.shape or q_out.dtype != q.dtype:
            raise ValueError("q_out must have q's shape and type")
        else:
            so = self._target(q_out, "q_out")[3]
        if not given[1]:
            k_out, sk = k.new_empty((n, hk, d)), (hk * d, d)
        elif k_out.shape != k.shape or k_out.dtype != k.dtype:
            raise ValueError("k_out must have k's shape and type")
        else:
            sk = self._target(k_out, "k_out")[3]
        qp, kp, to_q, to_k = q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr()
        if True in given:
            e = 4 if wide else 2
            self._check_memory((qp, n, hq, strides[0], strides[1], e), (kp, n, hk, strides[2], strides[3], e),
                               (to_q, n, hq, so[0], so[1], e) if given[0] else None,
                               (to_k, n, hk, sk[0], sk[1], e) if given[1] else None)
        self._launch(n, hq, hk, wide, strides, axis_stride, bool(inverse), 0, so, sk, None, n, n,
                     (qp, kp, 0, positions.data_ptr()), (0, 0, to_q, to_k, 0))
        return q_out, k_out

    def _check_target(self, out, at, n, hk, e, st, in_place, pools, size):
        """append's q_out is q (in_place: rows in q's order), or shares no memory with the inputs (at addresses `at`,
        their strides one after another) and the pools of `size` bytes."""
        d, lo, h = self.head_dim, out[0], out[2]
        hi = lo + 2 * ((out[1] - 1) * out[3] + (h - 1) * out[4] + d)
        for p in pools:
            if p < hi and lo < p + size and out[1] and h:
                raise ValueError("q_out shares memory with a pool")
        for i, p in enumerate(at):
            if p < hi:  # else past its end
                x = (p, n, hk if i else h, st[2 * i], st[2 * i + 1], e)
                if not _apart(out, x, d) and not (i == 0 and in_place and _same(out, x)):
                    raise ValueError("q_out shares memory with k or v, or with q without being q in its own rows")

    def append(self, q, k, v, positions, dst_rows, k_pool, v_pool, *, q_rows=None, q_out=None, pos_offset: int = 0):
        """A step's tokens into the cache: q and k turned by positions (+ pos_offset), k and v (tokens, Hkv,
        head_dim) to rows dst_rows (int64, page * page_size + slot; rows outside the pool, such as -1, are
        skipped) of the pools [pages, page_size, Hkv, head_dim], bf16. The rotated q goes to a new bf16
        tensor of q's shape, or to rows q_rows (int64; rows outside are skipped) of q_out (rows, Hq,
        head_dim). Returns it, without a gradient. Rows that no token names are not written; a row may be named
        once."""
        n, hq, hk, wide, strides, axis_stride = self._args(q, k, v, positions)
        if not -1 << 31 <= pos_offset < 1 << 31:
            raise ValueError("pos_offset must fit 32 bits")
        at, d, i64 = self._at, self.head_dim, self._i64
        shape = k_pool.shape
        for pool, name in ((k_pool, "k_pool"), (v_pool, "v_pool")):
            if pool.dtype not in self._bits or pool.get_device() != at or not pool.is_contiguous():
                raise ValueError(f"{name} must be a contiguous bf16 (or int16) tensor on {self.dev}")
        if v_pool.shape != shape:
            raise ValueError("k_pool and v_pool must have one shape")
        if len(shape) != 4 or shape[2] != hk or shape[3] != d:
            raise ValueError(f"the pools must be (pages, page_size, {hk}, {d})")
        slots = shape[0] * shape[1]
        qp, kp, vp, to_k, to_v = q.data_ptr(), k.data_ptr(), v.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr()
        if abs(to_k - to_v) < 2 * slots * hk * d:
            raise ValueError("k_pool and v_pool share memory")
        if q_out is None:
            if q_rows is not None:
                raise ValueError("q_rows needs q_out")
            q_out = q.new_empty((n, hq, d), dtype=self._bits[0])
            rows, so = n, (hq * d, d)
        else:
            rows, ho, w, so = self._target(q_out, "q_out")
            if w or ho != hq or (q_rows is None and rows < n):
                raise ValueError("q_out must be (rows, Hq, head_dim) bf16 (or int16), a row per token without q_rows")
            self._check_target((q_out.data_ptr(), n if q_rows is None else rows, hq, so[0], so[1], 2), (qp, kp, vp), n, hk,
                               4 if wide else 2, strides, q_rows is None, (to_k, to_v), 2 * slots * hk * d)
        to = _vec(dst_rows, "dst_rows", at, i64, n)
        self._launch(n, hq, hk, wide, strides, axis_stride, False, pos_offset, so, (hk * d, d), (hk * d, d), rows, slots,
                     (qp, kp, vp, positions.data_ptr()),
                     (0 if q_rows is None else _vec(q_rows, "q_rows", at, i64, n), to, q_out.data_ptr(), to_k, to_v))
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
