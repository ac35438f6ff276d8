"""``KVCache4``: keys and values of one decoder layer in 4 bits, and the attention over them.

The reference keeps its KV cache in bf16 (src/cobaltkernel/ref_llama.py:117-137); next to 2- to 4-bit weights the cache is what
fills the memory, and the time, of many or long sequences.  Here 64 neighbouring channels of a slot share a bf16 scale and an
fp16 zero point: 4.5 bits per value.  The format and the kernels' contract are in ``include/cobalt_b200.h``.

There is no backward pass (codes have no gradient) and no torch fallback: on a non-CUDA tensor every method raises.
"""
from __future__ import annotations

import ctypes
import functools
from typing import Optional

import torch

from . import _lib
from .linear import _raw_stream

GROUP = 64
TILE = 32
HEAD_DIMS = (64, 128, 192, 256)


@functools.lru_cache(maxsize=4096)
def _attend_scratch(device: int, *sizes: int) -> int:
    with torch.cuda.device(device):
        return _lib.load().cobalt_kv4_attend_scratch_bytes(*sizes)


class KVCache4:
    """Keys and values of ``n_seq`` sequences, ``slots`` positions each, ``n_kv_heads`` heads of ``head_dim`` (64, 128, 192 or 256).
    ``tiles [n_seq, n_kv_heads, ceil(slots / 32), 36 * head_dim]`` (uint8) is the whole state.  ``status`` (int32 ``[1]``, zero): where
    ``device_status()`` finds waits that gave up; caches may share one, each has its own by default.

    Every method takes ``n`` sequences of ``T`` tokens each, the first of them being sequence ``seq`` of the cache, and int64
    ``positions`` - ``[n, T]``, or ``[T]`` for the same in every sequence - read on the device: a captured graph follows them.  Calls run on
    the current stream of the cache's device."""

    def __init__(self, n_seq: int, n_kv_heads: int, slots: int, head_dim: int, device="cuda", status: Optional[torch.Tensor] = None):
        if min(n_seq, n_kv_heads, slots) < 1:
            raise ValueError("a cache needs at least one sequence, one KV head and one slot")
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        tiles = torch.zeros(n_seq, n_kv_heads, -(-slots // TILE), 36 * head_dim, dtype=torch.uint8, device=device)
        self._install(tiles, head_dim, slots, torch.zeros(1, dtype=torch.int32, device=device) if status is None else status)

    @classmethod
    def wrap(cls, tiles: torch.Tensor, head_dim: int, slots: Optional[int] = None, status: Optional[torch.Tensor] = None) -> "KVCache4":
        """A cache over existing tiles ``[n_seq, n_kv_heads, n_tiles, 36 * head_dim]`` (shared, not copied); the sequences may lie apart.  Without
        a ``status`` word it reports to the one of its device, which all such caches share."""
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        row, shape = 36 * head_dim, tiles.shape
        if tiles.dtype is not torch.uint8 or len(shape) != 4 or shape[3] != row or 0 in shape:
            raise ValueError(f"tiles must be uint8 [n_seq, n_kv_heads, n_tiles, {row}], got {tiles.dtype} {list(shape)}")
        _, heads, n, _ = shape
        apart, *inner = tiles.stride()
        if inner != [n * row, row, 1] or apart % 16 or tiles.data_ptr() % 16 or (shape[0] > 1 and apart < heads * n * row):
            raise ValueError("the tiles of a sequence must be contiguous, and sequences must begin on 16-byte boundaries without overlap")
        if slots is None:
            slots = n * TILE
        elif not (n - 1) * TILE < slots <= n * TILE:
            raise ValueError(f"{n} tiles hold {n * TILE} slots, not {slots}")
        obj = cls.__new__(cls)
        obj._install(tiles, head_dim, slots, status)
        return obj

    def _install(self, tiles, head_dim, slots, status):
        self.tiles, self.head_dim, self.slots = tiles, int(head_dim), int(slots)
        self.n_seq, self.n_kv_heads = tiles.shape[0], tiles.shape[1]
        self._index = tiles.get_device()                     # -1: not on a GPU
        self._apart = tiles.stride(0) if self.n_seq > 1 else 0
        if status is not None and (status.dtype is not torch.int32 or status.shape != (1,) or status.device != tiles.device):
            raise ValueError(f"status must be int32 [1] on {tiles.device}, got {status.dtype} {list(status.shape)} on {status.device}")
        self._status = status
        self._word = None if status is None else status.data_ptr()
        self._lib = _lib.load()

    @property
    def device(self) -> torch.device:
        return self.tiles.device

    # ------------------------------------------------------------------ arguments
    def _rows(self, name: str, t: torch.Tensor, width: int, lead):
        """(address, row stride, owner of the memory) of ``t [n, T, width]`` (or ``[T, width]``: one sequence) as rows the kernels take."""
        if self._index < 0 or not t.is_cuda:
            raise RuntimeError("KVCache4 needs CUDA tensors; there is no CPU path")
        if t.get_device() != self._index:
            raise ValueError(f"{name} is on {t.device}, the cache on {self.device}")
        if t.dtype is not torch.bfloat16:
            raise TypeError(f"{name} must be bfloat16, got {t.dtype}")
        shape = t.shape
        if not 2 <= len(shape) <= 3 or shape[-1] != width or (lead is not None and shape[:-1] != lead):
            raise ValueError(f"{name} must be [n, T, {width}]{'' if lead is None else ' with [n, T] = ' + str(list(lead))}, got {list(shape)}")
        self._no_grad(name, t)
        p = t.data_ptr()
        if p % 16 == 0 and t.is_contiguous():
            return p, width, t
        rows = t if len(shape) == 2 else t.reshape(-1, width)
        if rows.stride(1) != 1 or rows.stride(0) % 8 or rows.stride(0) < width or rows.data_ptr() % 16:
            rows = rows.clone(memory_format=torch.contiguous_format)
        return rows.data_ptr(), rows.stride(0), rows

    def _place(self, positions: torch.Tensor, n: int, T: int, seq: int):
        """(address of the positions, their stride from sequence to sequence, address of the first sequence's tiles, owner of the positions)"""
        if positions.dtype is not torch.int64 or positions.get_device() != self._index:
            raise TypeError(f"positions must be int64 on {self.device}, got {positions.dtype} on {positions.device}")
        shape = positions.shape
        if shape != (n, T) and shape != (T,):
            raise ValueError(f"positions must be [{n}, {T}] or [{T}], got {list(shape)}")
        if seq < 0 or seq + n > self.n_seq:
            raise ValueError(f"sequences {seq} .. {seq + n - 1} of a cache of {self.n_seq}")
        stride = positions.stride()
        if stride[-1] != 1 and T > 1:
            positions = positions.contiguous()
            stride = positions.stride()
        return positions.data_ptr(), stride[0] if n > 1 and len(shape) == 2 else 0, self.tiles.data_ptr() + seq * self._apart, positions

    def _call(self, name: str, *args):
        index = self._index
        if index == torch._C._cuda_getDevice():
            rc = getattr(self._lib, name)(*args, _raw_stream(index))
        else:
            with torch.cuda.device(index):
                rc = getattr(self._lib, name)(*args, _raw_stream(index))
        if rc:
            _lib.check(name, rc)

    # ------------------------------------------------------------------ the operators
    def append(self, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, q: Optional[torch.Tensor] = None,
               inv_freq: Optional[torch.Tensor] = None, q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None,
               eps: float = 1e-6, seq: int = 0, q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """Quantise ``k, v [n, T, n_kv_heads * head_dim]`` into the slots at ``positions`` (outside ``[0, slots)``: not stored; the
        positions of one sequence must differ).  With ``inv_freq`` (fp32 ``[head_dim / 2]``) ``k`` is rotated by its position first, as
        ``cobalt_rope_kv`` does, and with ``k_norm`` (bf16 ``[head_dim]``) normalised per head before that; the same is done to
        ``q [n, T, n_heads * head_dim]`` (``q_norm``), which is returned - in ``q_out`` if given (may be ``q`` itself)."""
        D, width = self.head_dim, self.n_kv_heads * self.head_dim
        kp, ld_k, k_own = self._rows("k", k, width, None)
        lead = k.shape[:-1]
        vp, ld_v, v_own = self._rows("v", v, width, lead)
        n, T = lead if len(lead) == 2 else (1, lead[0])
        if inv_freq is not None:
            self._weight("inv_freq", inv_freq, torch.float32, D // 2)
        if k_norm is not None:
            self._weight("k_norm", k_norm, torch.bfloat16, D)
        qp, ld_q, op, heads = None, 0, None, 0
        if q is None:
            if q_norm is not None or q_out is not None:
                raise ValueError("q_norm and q_out belong to a q")
        else:
            heads = q.shape[-1] // D
            if heads < 1:
                raise ValueError(f"q must be [n, T, n_heads * {D}], got {list(q.shape)}")
            qp, ld_q, q_own = self._rows("q", q, heads * D, lead)
            if q_norm is not None:
                self._weight("q_norm", q_norm, torch.bfloat16, D)
            if q_out is None:
                q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
            else:
                self._result("q_out", q_out, q)
            op = q_out.data_ptr()
        pos, stride, tiles, p_own = self._place(positions, n, T, seq)
        if n * T:
            self._call("cobalt_kv4_append", kp, ld_k, vp, ld_v, qp, ld_q, op, heads * D, pos, stride, tiles, self._apart, n, T, heads, self.n_kv_heads, D,
                       self.slots, None if inv_freq is None else inv_freq.data_ptr(), None if q_norm is None else q_norm.data_ptr(),
                       None if k_norm is None else k_norm.data_ptr(), eps)
        return q_out

    @staticmethod
    def _no_grad(name: str, t: torch.Tensor):
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{name} requires a gradient: KVCache4 has no backward pass (use torch.no_grad())")

    def _result(self, name: str, t: torch.Tensor, like: torch.Tensor):
        if t.shape != like.shape or t.dtype is not like.dtype or t.device != like.device or not t.is_contiguous() or t.data_ptr() % 16:
            raise ValueError(f"{name} must be a contiguous tensor like q on a 16-byte boundary")
        self._no_grad(name, t)

    def _weight(self, name: str, w: torch.Tensor, dtype, size: int):
        self._no_grad(name, w)
        if w.dtype is not dtype or w.shape != (size,) or w.get_device() != self._index or not w.is_contiguous() or w.data_ptr() % 4:
            raise ValueError(f"{name} must be a contiguous {dtype} [{size}] on {self.device}")

    def read(self, positions: torch.Tensor, seq: int = 0, n: Optional[int] = None):
        """``(k, v)`` bf16 ``[n, T, n_kv_heads, head_dim]`` of the slots at ``positions`` (outside ``[0, slots)``: zeros).  ``n`` says how many
        sequences a ``positions [T]`` is for (all from ``seq`` on by default)."""
        if self._index < 0:
            raise RuntimeError("KVCache4 needs CUDA tensors; there is no CPU path")
        shape = positions.shape
        if not 1 <= len(shape) <= 2:
            raise ValueError(f"positions must be [n, T] or [T], got {list(shape)}")
        if n is None:
            n = shape[0] if len(shape) == 2 else self.n_seq - seq
        T = shape[-1]
        pos, stride, tiles, p_own = self._place(positions, n, T, seq)
        k = self.tiles.new_empty((n, T, self.n_kv_heads, self.head_dim), dtype=torch.bfloat16)
        v = torch.empty_like(k)
        if n * T:
            self._call("cobalt_kv4_read", tiles, self._apart, pos, stride, k.data_ptr(), v.data_ptr(), n, T, self.n_kv_heads, self.head_dim, self.slots)
        return k, v

    def attend(self, q: torch.Tensor, positions: torch.Tensor, window: int = 0, sinks: int = 0, scale: Optional[float] = None, seq: int = 0,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of ``q [n, T, n_heads * head_dim]`` (rotated) over the cache; query head ``h`` reads KV head ``h * n_kv_heads // n_heads``.
        A token at position ``p`` sees the slots ``j <= p`` - with ``window > 0`` only the last ``window`` of them and the first ``sinks``
        slots.  One that sees none (``p < 0``: padding) gets zeros.  ``scale``: of the scores, ``head_dim ** -0.5`` by default."""
        D, n_kv = self.head_dim, self.n_kv_heads
        shape = q.shape
        heads = shape[-1] // D
        if heads < 1 or heads % n_kv:
            raise ValueError(f"q must hold a multiple of {n_kv} heads of {D}, got {list(shape)}")
        qp, ld_q, q_own = self._rows("q", q, heads * D, None)
        n, T = shape[:2] if len(shape) == 3 else (1, shape[0])
        if not 0 <= window < 1 << 31 or not 0 <= sinks < 1 << 31:
            raise ValueError("window and sinks must be between 0 and 2^31 - 1")
        pos, stride, tiles, p_own = self._place(positions, n, T, seq)
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        else:
            self._result("out", out, q)
        if n * T:
            need = _attend_scratch(self._index, n, T, heads, n_kv, D, self.slots, window, sinks)
            # a buffer per call, from the stream's own pool: calls on other streams and captured graphs never share one
            scratch = q.new_empty(need, dtype=torch.uint8) if need else None
            self._call("cobalt_kv4_attend_watched", qp, ld_q, tiles, self._apart, pos, stride, out.data_ptr(), n, T, heads, n_kv, D, self.slots, window, sinks,
                       D ** -0.5 if scale is None else scale, None if scratch is None else scratch.data_ptr(), need, self._word)
        return out

    def device_status(self) -> int:
        """0, or the code of the first bounded wait of an attention over this cache (and those that share its word) that gave up since the
        last question; rows that it concerns are NaN.  Waits for the current stream."""
        if self._status is not None:
            code = int(self._status.item())
            if code:                                         # (never cleared unread: kernels write it while it is 0 alone)
                self._status.zero_()
            return code
        word = ctypes.c_uint32(0)
        with torch.cuda.device(self.device):
            rc = self._lib.cobalt_kv4_status(_raw_stream(self._index), ctypes.byref(word))
        if rc not in (0, _lib.ETIMEOUT):
            _lib.check("cobalt_kv4_status", rc)
        return int(word.value)

    # ------------------------------------------------------------------ size
    def nbytes(self) -> int:
        return self.tiles.numel()

    def __repr__(self) -> str:
        return f"KVCache4(n_seq={self.n_seq}, n_kv_heads={self.n_kv_heads}, slots={self.slots}, head_dim={self.head_dim}, device={self.device})"
