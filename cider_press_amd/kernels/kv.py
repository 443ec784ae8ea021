"""Key/value cache in 4 bits: block tables and slots from request lengths, the
quantizing append (with the position rotation on the way), the dequantizing
gather, and attention over the cache (with capped or biased scores).

No reference counterpart: its KV cache (crates/cider-press-runtime/src/
kv_cache.rs) holds dense T.  Layouts and semantics are stated in
include/cpq.h (cpq_kv_cache and the functions after it).
"""
from __future__ import annotations

import ctypes
import struct

from .. import _lib
from . import Buffer, Commands, Device, _ptr

NO_SLOT = 0xFFFFFFFF  # the slot of a padding token


class _CacheArgs(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int), ("head_dim", ctypes.c_uint32), ("n_kv_heads", ctypes.c_uint32),
                ("group_size", ctypes.c_uint32), ("block_size", ctypes.c_uint32), ("n_blocks", ctypes.c_size_t),
                ("k_q", ctypes.c_void_p), ("k_q_len", ctypes.c_size_t), ("k_sb", ctypes.c_void_p),
                ("k_sb_len", ctypes.c_size_t), ("v_q", ctypes.c_void_p), ("v_q_len", ctypes.c_size_t),
                ("v_sb", ctypes.c_void_p), ("v_sb_len", ctypes.c_size_t)]


# cpq_kv_attention_args, packed: a ctypes structure of its fields takes longer to fill than the launch.
_ATTENTION_ARGS = struct.Struct("@PNNPNNNNPNPPNNNfiN")


def _attention_args(*fields) -> bytes:
    """q, its token and head strides, out, its strides, tokens, heads, block
    table, max_blocks, query starts, key lengths, sequences, max_q, max_kv,
    scale, causal, window."""
    try:
        return _ATTENTION_ARGS.pack(*fields)
    except struct.error as e:  # a negative or too large count
        raise _lib.InvalidArgument(f"kv_attention: {e}") from None


# cpq_kv_scores and cpq_kv_append_rotary_args, likewise.
_SCORES = struct.Struct("@fPP")
_ROTARY_ARGS = struct.Struct("@PNNPNNNPNNPNNPPNPIif0P")


def _pack(op: str, fields: struct.Struct, *values) -> bytes:
    try:
        return fields.pack(*values)
    except (struct.error, OverflowError) as e:
        raise _lib.InvalidArgument(f"{op}: {e}") from None


class KvCache:
    """One layer's cache: four u32 buffers, allocated here (not cleared: slots
    are written before they are read) or the caller's own in `buffers`
    (k_q, k_sb, v_q, v_sb)."""

    def __init__(self, device: Device, dtype: str, n_blocks: int, block_size: int, n_kv_heads: int, head_dim: int,
                 group_size: int, buffers=None):
        self.device, self.dtype = device, dtype
        self.n_blocks, self.block_size = n_blocks, block_size
        self.n_kv_heads, self.head_dim, self.group_size = n_kv_heads, head_dim, group_size
        self._args = _CacheArgs(_lib.DTYPES[dtype], head_dim, n_kv_heads, group_size, block_size, n_blocks)
        self._ref = ctypes.byref(self._args)
        q, sb = ctypes.c_size_t(), ctypes.c_size_t()
        _lib.check(_lib.lib().cpq_kv_cache_words(self._ref, ctypes.byref(q), ctypes.byref(sb)))
        if buffers is None:
            buffers = [device.alloc_buffer(n.value, "u32") for n in (q, sb, q, sb)]
        self.k_q, self.k_sb, self.v_q, self.v_sb = buffers
        for name, b in zip(("k_q", "k_sb", "v_q", "v_sb"), buffers):
            _need("KvCache", "u32", (b, 0))
            setattr(self._args, name, b.ptr)
            setattr(self._args, name + "_len", len(b))
        _lib.check(_lib.lib().cpq_check_kv_cache(self._ref))


def _need(op: str, dtype: str, *pairs) -> None:
    """Each (buffer, elements): TypeError when it is of another type,
    InvalidArgument when it is shorter."""
    for b, n in pairs:
        if b.dtype != dtype:
            raise TypeError(f"{op}: expected a {dtype} buffer, got {b.dtype}")
        if b._len < n:
            raise _lib.InvalidArgument(f"{op}: a buffer of {b._len} elements where {n} are needed")


def _strides(op: str, dtype: str, strides, b: Buffer, tokens: int, heads: int, dim: int):
    """(token, head) strides in elements, dense by default, checked against the buffer."""
    token, head = strides if strides is not None else (heads * dim, dim)
    if token < 0 or head < 0:
        raise _lib.InvalidArgument(f"{op}: negative strides")
    n = (tokens - 1) * token + (heads - 1) * head + dim if tokens > 0 and heads > 0 else 0
    if b.dtype != dtype or b._len < n:
        _need(op, dtype, (b, n))
    return token, head


def kv_release(commands: Commands, finished: Buffer, lens: Buffer, block_table: Buffer, max_blocks: int,
               block_size: int, free_list: Buffer, free_count: Buffer, lens_out: Buffer,
               free_count_out: Buffer) -> None:
    """Blocks of sequences with finished != 0 go on top of the free list, their
    lens_out is 0.  Encodes only."""
    n = lens._len
    _need("kv_release", "u32", (finished, n), (lens, n), (block_table, n * max_blocks), (free_list, 0),
          (free_count, 1), (lens_out, n), (free_count_out, 1))
    _lib.check(_lib.lib().cpq_kv_release(
        commands.handle, finished.ptr, lens.ptr, block_table.ptr, n, max_blocks, block_size, free_list.ptr,
        len(free_list), free_count.ptr, lens_out.ptr, free_count_out.ptr))


def kv_plan(commands: Commands, lens: Buffer, new_lens: Buffer, block_table: Buffer, max_blocks: int, block_size: int,
            free_list: Buffer, free_count: Buffer, query_starts: Buffer, kv_lens: Buffer, slots: Buffer,
            positions: Buffer, free_count_out: Buffer) -> None:
    """Query starts, key lengths, slots and positions of a step's new tokens,
    and the blocks they open entered in the block table; len(slots) is the
    step's capacity, unused entries are NO_SLOT.  Encodes only."""
    n, cap = lens._len, slots._len
    _need("kv_plan", "u32", (lens, n), (new_lens, n), (block_table, n * max_blocks), (free_list, 0), (free_count, 1),
          (query_starts, n + 1), (kv_lens, n), (slots, cap), (positions, cap), (free_count_out, 1))
    _lib.check(_lib.lib().cpq_kv_plan(
        commands.handle, lens.ptr, new_lens.ptr, block_table.ptr, n, max_blocks, block_size, free_list.ptr,
        len(free_list), free_count.ptr, query_starts.ptr, kv_lens.ptr, slots.ptr, positions.ptr, cap,
        free_count_out.ptr))


def kv_append(commands: Commands, cache: KvCache, k: Buffer, v: Buffer, slots: Buffer, tokens: int, k_strides=None,
              v_strides=None) -> None:
    """Quantizes the keys and values of `tokens` tokens into their slots;
    strides are (token, head) in elements.  Encodes only."""
    _need("kv_append", "u32", (slots, tokens))
    kt, kh = _strides("kv_append", cache.dtype, k_strides, k, tokens, cache.n_kv_heads, cache.head_dim)
    vt, vh = _strides("kv_append", cache.dtype, v_strides, v, tokens, cache.n_kv_heads, cache.head_dim)
    _lib.check(_lib.lib().cpq_kv_append(commands.handle, cache._ref, k.ptr, kt, kh, v.ptr, vt, vh, slots.ptr,
                                        tokens))


def kv_append_rotary(commands: Commands, cache: KvCache, q, k: Buffer, v: Buffer, slots: Buffer, positions: Buffer,
                     frequencies: Buffer, q_out, tokens: int, n_heads: int, interleaved: bool = False,
                     magnitude: float = 1.0, q_strides=None, k_strides=None, v_strides=None,
                     q_out_strides=None) -> None:
    """kv_append with the position rotation of keys on the way, queries rotated
    into q_out; the first 2 * len(frequencies) dimensions rotate, as pairs
    (i, i + len(frequencies)) or, interleaved, (2 i, 2 i + 1), by positions[t] *
    frequencies[i], cosines and sines times magnitude.  n_heads = 0 with q and
    q_out None: keys and values only.  Encodes only."""
    op, dtype, heads, dim = "kv_append_rotary", cache.dtype, cache.n_kv_heads, cache.head_dim
    _need(op, "u32", (slots, tokens), (positions, tokens))
    _need(op, "f32", (frequencies, 0))
    kt, kh = _strides(op, dtype, k_strides, k, tokens, heads, dim)
    vt, vh = _strides(op, dtype, v_strides, v, tokens, heads, dim)
    q_ptr = out_ptr = qt = qh = ot = oh = 0
    if n_heads:
        qt, qh = _strides(op, dtype, q_strides, q, tokens, n_heads, dim)
        ot, oh = _strides(op, dtype, q_out_strides, q_out, tokens, n_heads, dim)
        q_ptr, out_ptr = q.ptr, q_out.ptr
    args = _pack(op, _ROTARY_ARGS, q_ptr, qt, qh, out_ptr, ot, oh, n_heads, k.ptr, kt, kh, v.ptr, vt, vh, slots.ptr,
                 positions.ptr, tokens, frequencies.ptr, 2 * frequencies._len, bool(interleaved), magnitude)
    _lib.check(_lib.lib().cpq_kv_append_rotary(commands.handle, cache._ref, args))


def kv_gather(commands: Commands, cache: KvCache, slots: Buffer, rows: int, k_out=None, v_out=None) -> None:
    """Cached keys and values of `rows` slots as dense T [rows, n_kv_heads,
    head_dim]; either output may be None.  Encodes only."""
    _need("kv_gather", "u32", (slots, rows))
    for b in (k_out, v_out):
        if b is not None:
            _need("kv_gather", cache.dtype, (b, rows * cache.n_kv_heads * cache.head_dim))
    _lib.check(_lib.lib().cpq_kv_gather(commands.handle, cache._ref, slots.ptr, rows, _ptr(k_out), _ptr(v_out)))


def kv_attention(commands: Commands, cache: KvCache, q: Buffer, block_table: Buffer, max_blocks: int,
                 query_starts: Buffer, kv_lens: Buffer, out: Buffer, tokens: int, n_heads: int, n_seqs: int,
                 max_q: int, max_kv: int, scale: float, causal: bool = True, window: int = 0, q_strides=None,
                 out_strides=None) -> None:
    """Softmax attention of q [tokens, n_heads, head_dim] over each sequence's
    cached keys and values; strides are (token, head) in elements.  max_q and
    max_kv bound the sequences' queries and keys.  Encodes only."""
    _need("kv_attention", "u32", (block_table, n_seqs * max_blocks), (query_starts, n_seqs + 1), (kv_lens, n_seqs))
    qt, qh = _strides("kv_attention", cache.dtype, q_strides, q, tokens, n_heads, cache.head_dim)
    ot, oh = _strides("kv_attention", cache.dtype, out_strides, out, tokens, n_heads, cache.head_dim)
    args = _attention_args(q.ptr, qt, qh, out.ptr, ot, oh, tokens, n_heads, block_table.ptr, max_blocks,
                           query_starts.ptr, kv_lens.ptr, n_seqs, max_q, max_kv, scale, bool(causal), window)
    _lib.check(_lib.lib().cpq_kv_attention(commands.handle, cache._ref, args))


def kv_attention_scored(commands: Commands, cache: KvCache, q: Buffer, block_table: Buffer, max_blocks: int,
                        query_starts: Buffer, kv_lens: Buffer, out: Buffer, tokens: int, n_heads: int, n_seqs: int,
                        max_q: int, max_kv: int, scale: float, causal: bool = True, window: int = 0,
                        softcap: float = 0.0, slopes=None, prefix_lens=None, q_strides=None, out_strides=None) -> None:
    """kv_attention whose scores t become softcap * tanh(t / softcap) (softcap >
    0), plus slopes[h] * (key's position - query's), and whose first
    prefix_lens[s] keys every query of sequence s sees.  Encodes only."""
    op = "kv_attention_scored"
    _need(op, "u32", (block_table, n_seqs * max_blocks), (query_starts, n_seqs + 1), (kv_lens, n_seqs))
    if slopes is not None:
        _need(op, "f32", (slopes, n_heads))
    if prefix_lens is not None:
        _need(op, "u32", (prefix_lens, n_seqs))
    qt, qh = _strides(op, cache.dtype, q_strides, q, tokens, n_heads, cache.head_dim)
    ot, oh = _strides(op, cache.dtype, out_strides, out, tokens, n_heads, cache.head_dim)
    args = _pack(op, _ATTENTION_ARGS, q.ptr, qt, qh, out.ptr, ot, oh, tokens, n_heads, block_table.ptr, max_blocks,
                 query_starts.ptr, kv_lens.ptr, n_seqs, max_q, max_kv, scale, bool(causal), window)
    scores = _pack(op, _SCORES, softcap, _ptr(slopes) or 0, _ptr(prefix_lens) or 0)
    _lib.check(_lib.lib().cpq_kv_attention_scored(commands.handle, cache._ref, args, scores))
