"""Key and value caches: packed NVFP4 rows on top of the quantise-and-pack kernel, and E4M3 with block scales (Fp8Cache).

The reference quantises keys after RoPE: Hadamard over the head dimension, then its activation quantiser on
per-head rows `k.view(-1, head_dim)` with the last `high_bits_length` channels of every head in the
high-precision format (promix/quantize/kv_quant.py:244-279, `k_groupsize != -1` branch; the FP configs
`promix/configs/*-kv4.yaml` name the formats).  With head_dim = 128 that is exactly one row of the pack kernel
per (token, head): block-Hadamard(128), NVFP4 codes + E4M3 scales for the first 128 - k_hi channels, MXFP8 codes +
E8M0 scales for the last k_hi.  The packed cache holds 0.5625 byte per NVFP4 element instead of 2; `dequantize`
returns what the reference's fake quantiser would have put in the cache.  Queries must be rotated by the same
Hadamard (`rotate_heads`), which leaves q . k unchanged up to quantisation error.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import ops
from .rotation import get_hadamard_matrix


_H = {}


def quantize_heads(x: torch.Tensor, k_hi: int = 0, hadamard: bool = True) -> ops.PackedMatrix:
    """x: bf16 [..., heads, head_dim] (keys after RoPE, or values) -> packed rows, one per (token, head).
    head_dim must be 128 for the rotation; k_hi is the MXFP8 channel count per head (the reference's
    high_bits_length).  The packed formats need (head_dim - k_hi) % 64 == 0 and k_hi % 32 == 0, so with
    head_dim = 128 the choices are 0 (all NVFP4, the default) and 64; the reference's 0.125 * head_dim = 16
    does not fill a 32-element MXFP8 block."""
    d = x.shape[-1]
    if hadamard and d != 128:
        raise ValueError("the block-Hadamard rotation of the cache needs head_dim = 128")
    return ops.pack(x.reshape(-1, d), k_hi, hadamard=hadamard, sf_layout="rowmajor")


def dequantize_heads(p: ops.PackedMatrix, shape) -> torch.Tensor:
    """Packed rows -> bf16 tensor of `shape` ([..., heads, head_dim]); still in the rotated basis."""
    return ops.unpack(p).view(*shape)


def rotate_heads(q: torch.Tensor) -> torch.Tensor:
    """The same normalised Hadamard(128) on the head dimension of the queries (float32 product, one rounding:
    inference/quantize.py:447-448 in the reference)."""
    return (q.float() @ head_rotation(q.device, q.shape[-1])).to(q.dtype)


def head_rotation(device, size: int = 128) -> torch.Tensor:
    """The normalised Hadamard matrix, float32, built once per device: no host-to-device copy inside a CUDA-graph capture."""
    key = (size, torch.device(device))
    h = _H.get(key)
    if h is None:
        h = _H[key] = get_hadamard_matrix(size).to(device=device, dtype=torch.float32)
    return h


HEAD_DIM = 128
ROW_BYTES = HEAD_DIM // 2 + HEAD_DIM // 16      # 64 bytes of E2M1 codes + 8 E4M3 scale bytes per (token, head)


def pack_head_rows(x: torch.Tensor, hadamard: bool) -> torch.Tensor:
    """x: bf16 [..., heads, 128] -> uint8 [..., heads, 72]: the cache's storage form, per (token, head) the 64
    code bytes of the NVFP4 row followed by its 8 scale bytes (keys: `hadamard=True`, the rotation over the head
    dimension; values: False).  0.5625 byte per element instead of 2."""
    if x.shape[-1] != HEAD_DIM:
        raise ValueError("the packed key/value cache needs head_dim = 128")
    p = quantize_heads(x.contiguous(), 0, hadamard=hadamard)
    return torch.cat([p.lo_codes, p.lo_sf], 1).view(*x.shape[:-1], ROW_BYTES)


def unpack_head_rows(rows: torch.Tensor) -> torch.Tensor:
    """uint8 [..., heads, 72] -> bf16 [..., heads, 128]: the values the reference's fake quantiser leaves in its
    cache (keys still in the rotated basis).  All-zero rows (positions not written yet) give zeros."""
    flat = rows.reshape(-1, ROW_BYTES)
    n = flat.shape[0]
    empty = torch.zeros(n, 0, dtype=torch.uint8, device=rows.device)
    p = ops.PackedMatrix(n, HEAD_DIM, 0, flat[:, : HEAD_DIM // 2].contiguous(), flat[:, HEAD_DIM // 2:].contiguous(),
                         empty, empty, ops.SF_ROWMAJOR)
    return ops.unpack(p).view(*rows.shape[:-1], HEAD_DIM)


CACHE_BLOCK = 64        # positions that share a scale of an Fp8Cache


@dataclass
class Fp8Cache:
    """Keys and values of one layer in E4M3, `room` positions for each sequence of a batch, heads of 128.  One scale per
    64 positions and head, a power of two: value = code * scale.  Positions nobody has written may hold anything.
    ops.rope_kv_append_fp8 fills it in place, ops.fp8_cache_attention reads it; 1.0005 bytes per element, a bf16 cache has 2.

    `length`: how many leading positions are written, where the host keeps count (the decoder does for its caches), else None.
    An append at a host position within them moves it, one at positions in device memory makes it None.  The decoder refuses to
    begin behind it; without one the room is the limit, and what lies there is the caller's to answer for."""
    k: torch.Tensor           # u8 [B, room, kv_heads, 128]
    k_scale: torch.Tensor     # float32 [B, kv_heads, ceil(room / 64)]
    v: torch.Tensor
    v_scale: torch.Tensor
    length: Optional[int] = None

    @classmethod
    def empty(cls, batch: int, room: int, kv_heads: int, device, length: Optional[int] = None) -> "Fp8Cache":
        """Nothing written yet: `length` is 0 for a cache whose positions are to be counted."""
        def side():
            return (torch.empty(batch, room, kv_heads, HEAD_DIM, dtype=torch.uint8, device=device),
                    torch.empty(batch, kv_heads, -(-room // CACHE_BLOCK), dtype=torch.float32, device=device))
        return cls(*side(), *side(), length)

    @property
    def batch(self) -> int:
        return self.k.shape[0]

    @property
    def room(self) -> int:
        return self.k.shape[1]

    @property
    def kv_heads(self) -> int:
        return self.k.shape[2]

    def check(self, batch: int, kv_heads: int, device) -> None:
        """Raises unless this is a well-formed cache of `batch` sequences on `device`."""
        if self.k.dim() != 4 or self.room < 1 or kv_heads < 1:
            raise TypeError(f"cache.k must be uint8 [B, room, kv_heads, {HEAD_DIM}], it is {list(self.k.shape)}")
        room = self.room
        for name, c, s in (("k", self.k, self.k_scale), ("v", self.v, self.v_scale)):
            if c.dtype != torch.uint8 or tuple(c.shape) != (batch, room, kv_heads, HEAD_DIM) or not c.is_contiguous():
                raise TypeError(f"cache.{name} must be contiguous uint8 {[batch, room, kv_heads, HEAD_DIM]}, it is {c.dtype} {list(c.shape)}")
            if s.dtype != torch.float32 or tuple(s.shape) != (batch, kv_heads, -(-room // CACHE_BLOCK)) or not s.is_contiguous():
                raise TypeError(f"cache.{name}_scale must be contiguous float32 {[batch, kv_heads, -(-room // CACHE_BLOCK)]}")
            if c.device != device or s.device != device:
                raise RuntimeError(f"cache.{name} is on {c.device}, the call on {device}")

    def clone(self) -> "Fp8Cache":
        return Fp8Cache(self.k.clone(), self.k_scale.clone(), self.v.clone(), self.v_scale.clone(), self.length)

    def grown(self, room: int) -> "Fp8Cache":
        """A cache with room for `room` positions (at least this one's) that holds what this one does."""
        new = Fp8Cache.empty(self.batch, room, self.kv_heads, self.k.device)
        new.copy_from(self, self.room)
        return new

    def appended(self, pos, t: int) -> None:
        """Notes that `t` positions from `pos` on (an int, or a tensor of positions) have been written."""
        if isinstance(pos, torch.Tensor):
            self.length = None
        elif self.length is not None and 0 <= pos <= self.length:
            self.length = max(self.length, pos + t)

    def copy_from(self, other: "Fp8Cache", t: int) -> None:
        """Takes over the first `t` positions of another cache; what this one held behind them is no longer part of it."""
        blocks = -(-t // CACHE_BLOCK)
        for dst, src in ((self.k, other.k), (self.v, other.v)):
            dst[:, :t].copy_(src[:, :t])
        for dst, src in ((self.k_scale, other.k_scale), (self.v_scale, other.v_scale)):
            dst[..., :blocks].copy_(src[..., :blocks])
        self.length = None if other.length is None else min(t, other.length)

    def values(self, t: int):
        """bf16 keys and values [B, t, kv_heads, 128] of the first `t` positions."""
        def side(codes, scale):
            s = scale[..., : -(-t // CACHE_BLOCK)].repeat_interleave(CACHE_BLOCK, -1)[..., :t]
            return (codes[:, :t].view(torch.float8_e4m3fn).float() * s.transpose(1, 2)[..., None]).to(torch.bfloat16)
        return side(self.k, self.k_scale), side(self.v, self.v_scale)
