"""Attention over a paged key/value cache: the half of a decoder layer next to the routed experts.

`PagedAttention` wraps one moe_attn handle (include/moe_b200.h): `append` writes a pass of new tokens into the
cache's pages (per-head RMS norm and rotary positions applied on the way), `decode` attends with one new token
per sequence, `prefill` with a ragged batch of prompt chunks. The reference has no counterpart (its attention
belongs to the model it links against); the operators follow the manner of RoutedExperts: torch CUDA tensors are
the containers, errors raise MoeError, calls run on the current stream unless one is given (the caller orders it
behind what made the inputs) and do not synchronise. A handle's calls must not overlap on the GPU: they share its workspace.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

from . import _lib
from ._lib import AttnDesc, MoeError, check, lib
from .layer import _torch, run_on

_PAIRS = {"halves": _lib.ROPE_HALVES, "adjacent": _lib.ROPE_ADJACENT}


@dataclass
class AttentionConfig:
    """One layer's attention. rope_pairs: "halves" (value i turns with i + rope_dim / 2) or "adjacent" (2i with
    2i + 1); rope_sections: () for one position axis, or the pairs that follow the time, height and width
    axes. scale 0: 1 / sqrt(head_dim); softcap 0: scores are not capped; window 0: every position is seen."""

    num_heads: int
    num_kv_heads: int
    head_dim: int
    scale: float = 0.0
    softcap: float = 0.0
    window: int = 0
    rope_dim: int = 0
    rope_pairs: str = "halves"
    rope_sections: tuple = ()
    norm_eps: float = 1e-6


def rope_table(rope_dim: int, positions: int, base: float = 10000.0, inv_freq=None, device="cuda"):
    """[positions, rope_dim / 2, 2] f32 {cos, sin}, angles in f64. inv_freq (rope_dim / 2 values) replaces
    base ** (-2 i / rope_dim), for scaled variants."""
    torch = _torch()
    if inv_freq is None:
        inv_freq = base ** (-torch.arange(0, rope_dim, 2, dtype=torch.float64) / rope_dim)
    inv = torch.as_tensor(inv_freq, dtype=torch.float64).cpu()
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * inv[None]
    return torch.stack([angle.cos(), angle.sin()], -1).float().to(device)


def kv_pools(num_pages: int, num_kv_heads: int, page_size: int, head_dim: int, dtype=None, device="cuda"):
    """A layer's (k_pool, v_pool), [num_pages, num_kv_heads, page_size, head_dim] each, uninitialised."""
    torch = _torch()
    shape = (num_pages, num_kv_heads, page_size, head_dim)
    dtype = dtype or torch.bfloat16
    return torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device)


def page_slots(page_table, seqs, positions, page_size: int):
    """The cache slots ([T] int64) of tokens at `positions` of sequences `seqs` (CUDA int tensors), for append. A token
    without a page (an entry below 0, a position or sequence outside the table) gets -2, which append reports; -1 would
    pass for padding."""
    torch = _torch()
    pos, seq = positions.long(), seqs.long()
    rows, width = page_table.shape
    if not rows or not width:
        return torch.full_like(pos, -2)
    col = pos.div(page_size, rounding_mode="floor")
    page = page_table[seq.clamp(0, rows - 1), col.clamp(0, width - 1)].long()
    here = (page >= 0) & (pos >= 0) & (col < width) & (seq >= 0) & (seq < rows)
    return torch.where(here, page * page_size + pos % page_size, -2)


def _invalid(msg: str):
    return MoeError(_lib.MOE_ERR_INVALID, msg)


class PagedAttention:
    """The attention of one decoder layer over its pools. k_pool, v_pool: [pages, num_kv_heads, page_size,
    head_dim] bf16 or f16 CUDA tensors, of which only the first dimension may be strided (so both may be views of
    one [pages, 2, ...] tensor); rope_table [positions, rope_dim / 2, 2] f32; q_norm, k_norm [head_dim] or None."""

    def __init__(self, cfg: AttentionConfig, k_pool, v_pool, rope_table=None, q_norm=None, k_norm=None,
                 max_seqs: int = 256):
        torch = _torch()
        self.config = cfg
        self._dtype = k_pool.dtype
        kinds = {torch.bfloat16: _lib.ATTN_BF16, torch.float16: _lib.ATTN_F16}
        if self._dtype not in kinds or v_pool.dtype != self._dtype:
            raise _invalid("PagedAttention: the pools must both be bf16 or both f16")
        if k_pool.dim() != 4 or k_pool.shape != v_pool.shape or not k_pool.is_cuda or k_pool.device != v_pool.device:
            raise _invalid("PagedAttention: the pools must be CUDA tensors of one shape [pages, heads, page, head_dim]")
        pages, heads, page, dim = k_pool.shape
        if heads != cfg.num_kv_heads or dim != cfg.head_dim:
            raise _invalid("PagedAttention: the pools do not have the configuration's heads and head_dim")
        for pool in (k_pool, v_pool):
            if pages and (pool.stride()[1:] != (page * dim, dim, 1) or pool.stride(0) != k_pool.stride(0)):
                raise _invalid("PagedAttention: pages must be contiguous and both pools' page strides equal")
        if cfg.rope_pairs not in _PAIRS:
            raise _invalid("PagedAttention: rope_pairs is 'halves' or 'adjacent'")
        sections = tuple(cfg.rope_sections)
        if len(sections) not in (0, 1, 3):
            raise _invalid("PagedAttention: rope_sections holds no, one or three numbers")
        if cfg.rope_dim:
            if (rope_table is None or rope_table.dtype != torch.float32 or rope_table.device != k_pool.device or
                    rope_table.shape[1:] != (cfg.rope_dim // 2, 2)):
                raise _invalid("PagedAttention: rope_table must be [positions, rope_dim / 2, 2] f32 on the pools' device")
            rope_table = rope_table.contiguous()
        for w in (q_norm, k_norm):
            if w is not None and (w.dtype != self._dtype or w.shape != (dim,) or w.device != k_pool.device):
                raise _invalid("PagedAttention: norm weights must be [head_dim] in the pools' type, on their device")
        q_norm = None if q_norm is None else q_norm.contiguous()
        k_norm = None if k_norm is None else k_norm.contiguous()
        self._keep = (k_pool, v_pool, rope_table, q_norm, k_norm)  # the handle holds their addresses
        self.axes = 3 if len(sections) == 3 else 1
        self.max_seqs = int(max_seqs)
        self.device = k_pool.device
        self._torch, self._int32, self._dim, self._index = torch, torch.int32, dim, k_pool.get_device()
        self._raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        d = AttnDesc()
        d.dtype = kinds[self._dtype]
        d.num_heads, d.num_kv_heads, d.head_dim = cfg.num_heads, cfg.num_kv_heads, cfg.head_dim
        d.scale, d.softcap, d.window = cfg.scale, cfg.softcap, cfg.window
        d.k_pool, d.v_pool = k_pool.data_ptr(), v_pool.data_ptr()
        d.num_pages, d.page_size, d.page_stride = pages, page, k_pool.stride(0)
        d.rope_dim = cfg.rope_dim
        if cfg.rope_dim:
            d.rope_table, d.rope_positions = rope_table.data_ptr(), rope_table.shape[0]
            d.rope_pairs, d.rope_axes = _PAIRS[cfg.rope_pairs], self.axes
            if self.axes == 3:
                d.rope_sections = (ctypes.c_int * 3)(*sections)
        d.q_norm = None if q_norm is None else q_norm.data_ptr()
        d.k_norm = None if k_norm is None else k_norm.data_ptr()
        d.norm_eps = cfg.norm_eps
        d.device = self._index
        d.max_seqs = self.max_seqs
        handle = ctypes.c_void_p()
        check(lib().moe_attn_create(ctypes.byref(d), ctypes.byref(handle)))
        self._h = handle
        self._append, self._decode, self._prefill = lib().moe_attn_append, lib().moe_attn_decode, lib().moe_attn_prefill

    def close(self):
        if getattr(self, "_h", None) is not None and self._h.value:
            lib().moe_attn_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def device_bytes(self) -> int:
        return int(lib().moe_attn_device_bytes(self._h))

    def check(self, stream=None):
        """Raise MoeError when a previous call latched a device-side error (a slot, page, position or length out of
        range)."""
        check(lib().moe_attn_check(self._h, self._stream(stream)))

    def set_wait_limit(self, sm_clocks: int):
        """How long prefill's device-side waits last, in SM clocks (default 400 million, about 200 ms). One that runs out is
        reported by check() as MOE_ERR_TIMEOUT; until then further prefill calls do nothing."""
        check(lib().moe_attn_set_wait_limit(self._h, int(sm_clocks)))

    # -- argument checks (a small call is a few microseconds on the device: each of these counts) --------------
    def _rows(self, x, heads: int, what: str):
        """(x, token stride, head stride) as rows the kernels take: one head's values consecutive, 16-byte aligned
        (else a copy)."""
        shape = x.shape
        if len(shape) != 3 or shape[1] != heads or shape[2] != self._dim:
            raise _invalid(f"{what}: expected [tokens, {heads}, {self._dim}]")
        if x.dtype is not self._dtype or x.get_device() != self._index:
            raise _invalid(f"{what}: must be a CUDA tensor of the pools' type on their device")
        ts, hs, one = x.stride()
        if one != 1 or (ts | hs) & 7 or x.data_ptr() & 15:
            x = x.clone(memory_format=self._torch.contiguous_format)
            ts, hs, one = x.stride()
        return x, ts, hs

    def _ints(self, t, shape, dtype, what: str):
        if t.dtype is not dtype or t.shape != shape or t.get_device() != self._index:
            raise _invalid(f"{what}: must be a {tuple(shape)} {dtype} tensor on the pools' device")
        return t if t.is_contiguous() else t.contiguous()

    def _table(self, table, B: int, what: str):
        shape = table.shape
        if len(shape) != 2 or shape[0] != B:
            raise _invalid(f"{what}: page_table must be [sequences, pages]")
        return self._ints(table, shape, self._int32, what + ": page_table"), shape[1]

    def _stream(self, stream):
        """The raw handle of `stream`, or of the device's current stream (by torch's direct lookup where it has one)."""
        if stream is not None:
            return stream.cuda_stream
        if self._raw_stream is not None:
            return self._raw_stream(self._index)
        return self._torch.cuda.current_stream(self.device).cuda_stream

    def _outputs(self, q, out, lse, return_lse, what: str):
        if out is None:
            out = self._torch.empty_like(q, memory_format=self._torch.contiguous_format)
        elif (out.shape != q.shape or out.dtype is not self._dtype or out.get_device() != self._index or
              not out.is_contiguous() or out.data_ptr() & 15):
            raise _invalid(f"{what}: out must be a contiguous, 16-byte aligned tensor of q's shape and type")
        if lse is not None:
            if (lse.shape != q.shape[:2] or lse.dtype is not self._torch.float32 or
                    lse.get_device() != self._index or not lse.is_contiguous()):
                raise _invalid(f"{what}: lse must be a contiguous [tokens, num_heads] f32 tensor")
        elif return_lse:
            lse = q.new_empty(q.shape[:2], dtype=self._torch.float32)
        return out, lse

    # -- the operators -------------------------------------------------------------------------------------
    def append(self, q, k, v, positions, slots, out=None, stream=None):
        """New tokens into the cache. q [T, num_heads, head_dim], k and v [T, num_kv_heads, head_dim] (any token and
        head strides), positions [T] or [axes, T] int32 (None without rotation), slots [T] int64 (page *
        page_size + offset; -1: a padding token). Returns norm(q) rotated ([T, num_heads, head_dim], or `out`,
        which may be q)."""
        if stream is not None:
            return run_on(stream, self._index, self.append, q, k, v, positions, slots, out=out)
        cfg = self.config
        T = q.shape[0]
        q, qt, qh = self._rows(q, cfg.num_heads, "append: q")
        k, kt, kh = self._rows(k, cfg.num_kv_heads, "append: k")
        v, vt, vh = self._rows(v, cfg.num_kv_heads, "append: v")
        if k.shape[0] != T or v.shape[0] != T:
            raise _invalid("append: q, k and v hold different numbers of tokens")
        where = None
        if cfg.rope_dim:
            if positions is None:
                raise _invalid("append: positions are needed with rotation")
            shape = (T,) if self.axes == 1 and positions.dim() == 1 else (self.axes, T)
            positions = self._ints(positions, shape, self._int32, "append: positions")
            where = positions.data_ptr()
        slots = self._ints(slots, (T,), self._torch.int64, "append: slots")
        if out is None:
            out = self._torch.empty_like(q, memory_format=self._torch.contiguous_format)
            ot, oh = cfg.num_heads * self._dim, self._dim
        else:
            given = out
            out, ot, oh = self._rows(out, cfg.num_heads, "append: out")
            if out is not given or out.shape[0] != T:
                raise _invalid("append: out must be [T, num_heads, head_dim] with consecutive, 16-byte aligned heads")
        check(self._append(self._h, q.data_ptr(), qt, qh, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, T, where,
                           slots.data_ptr(), out.data_ptr(), ot, oh, self._stream(None)))
        return out

    def decode(self, q, seq_lens, page_table, out=None, lse=None, return_lse=False, stream=None):
        """One new token per sequence: q [B, num_heads, head_dim] against the seq_lens[b] cached tokens (the new one
        included, int32) in the pages of page_table[b] ([B, pages] int32). Returns y [B, num_heads, head_dim],
        or (y, lse) with return_lse or an lse tensor. A sequence of length 0 gives zeros and lse = -inf."""
        if stream is not None:
            return run_on(stream, self._index, self.decode, q, seq_lens, page_table, out=out, lse=lse, return_lse=return_lse)
        q, qt, qh = self._rows(q, self.config.num_heads, "decode: q")
        B = q.shape[0]
        if B > self.max_seqs:
            raise _invalid("decode: more sequences than max_seqs")
        seq_lens = self._ints(seq_lens, (B,), self._int32, "decode: seq_lens")
        page_table, pages = self._table(page_table, B, "decode")
        out, lse = self._outputs(q, out, lse, return_lse, "decode")
        check(self._decode(self._h, q.data_ptr(), qt, qh, seq_lens.data_ptr(), page_table.data_ptr(), pages, B,
                           out.data_ptr(), None if lse is None else lse.data_ptr(), self._stream(None)))
        return out if lse is None else (out, lse)

    def prefill(self, q, cu_q, seq_lens, page_table, out=None, lse=None, return_lse=False, stream=None):
        """Causal attention of prompt chunks that append has written: q [T, num_heads, head_dim], sequence b's rows
        cu_q[b] .. cu_q[b + 1] - 1 (cu_q [B + 1] int32), the last of its seq_lens[b] cached tokens. Returns y
        [T, num_heads, head_dim], or (y, lse). Rows from cu_q[B] on are padding: zeros and lse = -inf."""
        if stream is not None:
            return run_on(stream, self._index, self.prefill, q, cu_q, seq_lens, page_table, out=out, lse=lse,
                          return_lse=return_lse)
        q, qt, qh = self._rows(q, self.config.num_heads, "prefill: q")
        if not (qt and qh):  # an expanded tensor: the tile loads take positive strides only
            q = q.clone(memory_format=self._torch.contiguous_format)
            qt, qh, _ = q.stride()
        B = seq_lens.shape[0]
        cu_q = self._ints(cu_q, (B + 1,), self._int32, "prefill: cu_q")
        seq_lens = self._ints(seq_lens, (B,), self._int32, "prefill: seq_lens")
        page_table, pages = self._table(page_table, B, "prefill")
        out, lse = self._outputs(q, out, lse, return_lse, "prefill")
        check(self._prefill(self._h, q.data_ptr(), qt, qh, cu_q.data_ptr(), seq_lens.data_ptr(), page_table.data_ptr(),
                            pages, B, q.shape[0], out.data_ptr(), None if lse is None else lse.data_ptr(),
                            self._stream(None)))
        return out if lse is None else (out, lse)
