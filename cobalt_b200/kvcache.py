"""``KVCache4``: keys and values of one decoder layer in 4 bits, and the attention over them.

The reference keeps its KV cache in bf16 (src/cobaltkernel/ref_llama.py:117-137); next to 2- to 4-bit weights the cache is what
fills the memory, and the time, of many or long sequences.  Here 64 neighbouring channels of a slot share a bf16 scale and an
fp16 zero point: 4.5 bits per value.  The format and the kernels' contract are in ``include/cobalt_b200.h``.

There is no backward pass (codes have no gradient) and no torch fallback: on a non-CUDA tensor every method raises.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib
from .linear import _raw_stream

GROUP = 64
TILE = 32
HEAD_DIMS = (64, 128, 192, 256)


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


class KVCache4:
    """Keys and values of ``n_seq`` sequences, ``slots`` positions each, ``n_kv_heads`` heads of ``head_dim`` (64, 128, 192 or 256).
    ``tiles [n_seq, n_kv_heads, ceil(slots / 32), 36 * head_dim]`` (uint8) is the whole state.

    Every method takes ``n`` sequences of ``T`` tokens each, the first of them being sequence ``seq`` of the cache, and int64
    ``positions`` - ``[n, T]``, or ``[T]`` for the same in every sequence - read on the device: a captured graph follows them.  Calls run on
    the current stream of the cache's device."""

    def __init__(self, n_seq: int, n_kv_heads: int, slots: int, head_dim: int, device="cuda"):
        if min(n_seq, n_kv_heads, slots) < 1:
            raise ValueError("a cache needs at least one sequence, one KV head and one slot")
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        self._install(torch.zeros(n_seq, n_kv_heads, -(-slots // TILE), 36 * head_dim, dtype=torch.uint8, device=device), head_dim, slots)

    @classmethod
    def wrap(cls, tiles: torch.Tensor, head_dim: int, slots: Optional[int] = None) -> "KVCache4":
        """A cache over existing tiles ``[n_seq, n_kv_heads, n_tiles, 36 * head_dim]`` (shared, not copied); the sequences may lie apart."""
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        if tiles.dtype is not torch.uint8 or tiles.dim() != 4 or tiles.shape[3] != 36 * head_dim or 0 in tiles.shape:
            raise ValueError(f"tiles must be uint8 [n_seq, n_kv_heads, n_tiles, {36 * head_dim}], got {tiles.dtype} {list(tiles.shape)}")
        if not tiles[0].is_contiguous() or tiles.stride(0) % 16 or tiles.data_ptr() % 16 or (
                tiles.shape[0] > 1 and tiles.stride(0) < tiles[0].numel()):
            raise ValueError("the tiles of a sequence must be contiguous, and sequences must begin on 16-byte boundaries without overlap")
        n = tiles.shape[2]
        if slots is not None and not (n - 1) * TILE < slots <= n * TILE:
            raise ValueError(f"{n} tiles hold {n * TILE} slots, not {slots}")
        obj = cls.__new__(cls)
        obj._install(tiles, head_dim, n * TILE if slots is None else slots)
        return obj

    def _install(self, tiles, head_dim, slots):
        self.tiles, self.head_dim, self.slots = tiles, int(head_dim), int(slots)
        self.n_seq, self.n_kv_heads = tiles.shape[0], tiles.shape[1]
        self.device = tiles.device
        self._lib = _lib.load()

    # ------------------------------------------------------------------ arguments
    def _check(self, name: str, t: torch.Tensor, width: int, lead=None, align: int = 4) -> torch.Tensor:
        """``t [n, T, width]`` (or ``[T, width]``: one sequence) as rows the kernels take."""
        if not t.is_cuda or not self.tiles.is_cuda:
            raise RuntimeError("KVCache4 needs CUDA tensors; there is no CPU path")
        if t.device != self.device:
            raise ValueError(f"{name} is on {t.device}, the cache on {self.device}")
        if t.dtype is not torch.bfloat16:
            raise TypeError(f"{name} must be bfloat16, got {t.dtype}")
        if t.dim() not in (2, 3) or t.shape[-1] != width or (lead is not None and t.shape[:-1] != lead):
            raise ValueError(f"{name} must be [n, T, {width}]{'' if lead is None else ' with [n, T] = ' + str(list(lead))}, got {list(t.shape)}")
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{name} requires a gradient: KVCache4 has no backward pass (use torch.no_grad())")
        rows = t if t.dim() == 2 else t.reshape(-1, width)
        if rows.stride(1) != 1 or rows.stride(0) * 2 % align or rows.stride(0) < width or rows.data_ptr() % align:
            rows = rows.clone(memory_format=torch.contiguous_format)
        return rows

    def _place(self, positions: torch.Tensor, n: int, T: int, seq: int):
        """(positions, their stride from sequence to sequence, address of the first sequence's tiles)"""
        if positions.dtype is not torch.int64 or positions.device != self.device:
            raise TypeError(f"positions must be int64 on {self.device}, got {positions.dtype} on {positions.device}")
        if positions.shape != (n, T) and positions.shape != (T,):
            raise ValueError(f"positions must be [{n}, {T}] or [{T}], got {list(positions.shape)}")
        if seq < 0 or seq + n > self.n_seq:
            raise ValueError(f"sequences {seq} .. {seq + n - 1} of a cache of {self.n_seq}")
        if positions.stride(-1) != 1 and T > 1:
            positions = positions.contiguous()
        stride = positions.stride(0) if positions.dim() == 2 and n > 1 else 0
        return positions, stride, self.tiles.data_ptr() + seq * self.tiles.stride(0)

    @staticmethod
    def _lead(t: torch.Tensor):
        return (1, t.shape[0]) if t.dim() == 2 else tuple(t.shape[:2])

    def _call(self, name: str, *args):
        index = self.device.index
        if index != torch._C._cuda_getDevice():
            with torch.cuda.device(index):
                rc = getattr(self._lib, name)(*args, _raw_stream(index))
        else:
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
        kr, vr = self._check("k", k, width), self._check("v", v, width, k.shape[:-1])
        n, T = self._lead(k)
        for name, w, dtype, size in (("inv_freq", inv_freq, torch.float32, D // 2), ("q_norm", q_norm, torch.bfloat16, D),
                                     ("k_norm", k_norm, torch.bfloat16, D)):
            if w is not None and (w.dtype is not dtype or w.shape != (size,) or w.device != self.device or not w.is_contiguous()
                                  or w.data_ptr() % 4):
                raise ValueError(f"{name} must be a contiguous {dtype} [{size}] on {self.device}")
        qr, heads = None, 0
        if q is None:
            if q_norm is not None or q_out is not None:
                raise ValueError("q_norm and q_out belong to a q")
        else:
            heads = q.shape[-1] // D
            if heads < 1:
                raise ValueError(f"q must be [n, T, n_heads * {D}], got {list(q.shape)}")
            qr = self._check("q", q, heads * D, k.shape[:-1])
            if q_out is None:
                q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            elif q_out.shape != q.shape or q_out.dtype is not q.dtype or q_out.device != q.device or not q_out.is_contiguous() or q_out.data_ptr() % 4:
                raise ValueError("q_out must be a contiguous tensor like q")
        pos, stride, tiles = self._place(positions, n, T, seq)
        if n * T:
            self._call("cobalt_kv4_append", kr.data_ptr(), kr.stride(0), vr.data_ptr(), vr.stride(0), _ptr(qr), 0 if qr is None else qr.stride(0),
                       _ptr(q_out), heads * D, pos.data_ptr(), stride, tiles, self.tiles.stride(0), n, T, heads, self.n_kv_heads, D, self.slots,
                       _ptr(inv_freq), _ptr(q_norm), _ptr(k_norm), float(eps))
        return q_out

    def read(self, positions: torch.Tensor, seq: int = 0, n: Optional[int] = None):
        """``(k, v)`` bf16 ``[n, T, n_kv_heads, head_dim]`` of the slots at ``positions`` (outside ``[0, slots)``: zeros).  ``n`` says how many
        sequences a ``positions [T]`` is for (all from ``seq`` on by default)."""
        if not self.tiles.is_cuda:
            raise RuntimeError("KVCache4 needs CUDA tensors; there is no CPU path")
        if positions.dim() not in (1, 2):
            raise ValueError(f"positions must be [n, T] or [T], got {list(positions.shape)}")
        if n is None:
            n = positions.shape[0] if positions.dim() == 2 else self.n_seq - seq
        T = positions.shape[-1]
        pos, stride, tiles = self._place(positions, n, T, seq)
        k = torch.empty(n, T, self.n_kv_heads, self.head_dim, dtype=torch.bfloat16, device=self.device)
        v = torch.empty_like(k)
        if n * T:
            self._call("cobalt_kv4_read", tiles, self.tiles.stride(0), pos.data_ptr(), stride, k.data_ptr(), v.data_ptr(), n, T, self.n_kv_heads,
                       self.head_dim, self.slots)
        return k, v

    def attend(self, q: torch.Tensor, positions: torch.Tensor, window: int = 0, sinks: int = 0, scale: Optional[float] = None, seq: int = 0,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of ``q [n, T, n_heads * head_dim]`` (rotated) over the cache; query head ``h`` reads KV head ``h * n_kv_heads // n_heads``.
        A token at position ``p`` sees the slots ``j <= p`` - with ``window > 0`` only the last ``window`` of them and the first ``sinks``
        slots.  One that sees none (``p < 0``: padding) gets zeros.  ``scale``: of the scores, ``head_dim ** -0.5`` by default."""
        D = self.head_dim
        heads = q.shape[-1] // D
        if heads < 1 or heads % self.n_kv_heads:
            raise ValueError(f"q must hold a multiple of {self.n_kv_heads} heads of {D}, got {list(q.shape)}")
        qr = self._check("q", q, heads * D, align=16)
        n, T = self._lead(q)
        window, sinks = int(window), int(sinks)
        if window < 0 or sinks < 0 or window >= 1 << 31 or sinks >= 1 << 31:
            raise ValueError("window and sinks must be between 0 and 2^31 - 1")
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        elif out.shape != q.shape or out.dtype is not q.dtype or out.device != q.device or not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError("out must be a contiguous tensor like q on a 16-byte boundary")
        pos, stride, tiles = self._place(positions, n, T, seq)
        if n * T:
            need = self._lib.cobalt_kv4_attend_scratch_bytes(n, T, heads, self.n_kv_heads, D, self.slots, window, sinks)
            # a buffer per call, from the stream's own pool: calls on other streams and captured graphs never share one
            scratch = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
            self._call("cobalt_kv4_attend", qr.data_ptr(), qr.stride(0), tiles, self.tiles.stride(0), pos.data_ptr(), stride, out.data_ptr(), n, T,
                       heads, self.n_kv_heads, D, self.slots, window, sinks, D ** -0.5 if scale is None else float(scale), _ptr(scratch), need)
        return out

    def device_status(self) -> int:
        """0, or the code of the first bounded wait of an attention over such caches on this device that gave up since the last
        question (its rows are then not written).  Waits for the current stream."""
        word = ctypes.c_uint32(0)
        with torch.cuda.device(self.device):
            rc = self._lib.cobalt_kv4_status(_raw_stream(self.device.index), ctypes.byref(word))
        if rc not in (0, _lib.ETIMEOUT):
            _lib.check("cobalt_kv4_status", rc)
        return int(word.value)

    # ------------------------------------------------------------------ size
    def nbytes(self) -> int:
        return self.tiles.numel()

    def __repr__(self) -> str:
        return f"KVCache4(n_seq={self.n_seq}, n_kv_heads={self.n_kv_heads}, slots={self.slots}, head_dim={self.head_dim}, device={self.device})"
