"""A cache of keys and values in 8 bits, and attention over it: beside the attention blocks of the UNets (which see a whole image at
once), what a sequence model over codebook indices is served with.

    cache = KVCache(blocks, kv_heads, head_dim, block=64, format="e4m3", device="cuda")
    cache.append(k, v, table, start)                    # a decoding step: one row for each sequence
    out = cache.attend(q, table, start + 1)
    cache.append(k, v, table, start, offsets, most)     # prompts of unequal length, packed
    out = cache.attend(q, table, lengths, offsets, most, window=1024, sinks=4)
    k, v = cache.read(table, start, rows)

The cache is one pool of `blocks` blocks of `block` tokens for all heads; `table` [sequences, width] (int32) names the blocks of
each sequence in order, entries outside 0 .. blocks-1 are holes.  Each (block, head) has one power-of-two scale for its keys and one
for its values; a block's scale starts with the write of its first token and never shrinks after that.
Rows k, v [rows, kv_heads, head_dim], q and out [rows, heads, head_dim] (heads a multiple of kv_heads; head h reads key head
h // (heads // kv_heads)) are float32 or bfloat16 with any strides and adjacent features; packed one sequence after the other:
sequence b owns rows offsets[b] .. offsets[b+1]-1 (`offsets` int32, [sequences + 1]), or without `offsets` rows / sequences each.
`most` bounds the rows of a sequence where the caller knows it (default: all rows); rows of a sequence beyond it are left out.  Launches
are sized by it and by the rows there are: without it, finding whose rows a workgroup takes costs many short sequences some time.  `start`, `lengths`: int32, [sequences], on the GPU; nothing
is copied to the host, so all of it can be captured into a graph.  Rows behind the last sequence are neither read nor written (in a
result that the call allocates they hold nothing in particular).

The layout is the kernels' own (csrc/kv_layout.h); there is no CPU path and no gradient, backward or forward: tensors that require one or
carry a tangent are refused.  A call cannot be recorded by torch.jit.trace or make_fx; `out` counts as modified in place.
"""
import torch

from . import _lib
from ._lib import call_on, has_tangent, lib, overlapping, overwritten, self_overlapping

_TYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}
_INT_MAX = 2 ** 31 - 1
_FORMATS = {"e4m3": _lib.KV_E4M3, "int8": _lib.KV_INT8}


class KVCache:
    def __init__(self, blocks, kv_heads, head_dim, block=64, format="e4m3", device="cuda"):
        if format not in _FORMATS:
            raise ValueError(f"format {format!r} (e4m3 or int8)")
        if block not in (64, 128, 256):
            raise ValueError(f"block {block}: 64, 128 or 256 tokens")
        if head_dim % 16 or not 16 <= head_dim <= 256:
            raise ValueError(f"head_dim {head_dim}: a multiple of 16, 16 to 256")
        if blocks < 1 or kv_heads < 1:
            raise ValueError(f"{blocks} blocks of {kv_heads} heads")
        self.blocks, self.kv_heads, self.head_dim, self.block, self.format = blocks, kv_heads, head_dim, block, format
        shape = (blocks, kv_heads, block * head_dim)
        self.codes_k = torch.zeros(shape, dtype=torch.uint8, device=device)
        self.codes_v = torch.zeros(shape, dtype=torch.uint8, device=device)
        self.scales_k = torch.zeros(shape[:2], dtype=torch.float32, device=device)
        self.scales_v = torch.zeros(shape[:2], dtype=torch.float32, device=device)
        self.device = self.codes_k.device
        self._index = self.codes_k.get_device()                  # -1 on the CPU
        self._format = _FORMATS[format]

    # ---- checks

    def _pool(self):
        return self.codes_k.data_ptr(), self.codes_v.data_ptr(), self.scales_k.data_ptr(), self.scales_v.data_ptr()

    def _rows(self, name, t, heads):
        if t.dtype not in _TYPES:
            raise TypeError(f"{name} is {t.dtype}: float32 or bfloat16")
        shape = t.shape
        if len(shape) != 3 or shape[1] != heads or shape[2] != self.head_dim:
            raise ValueError(f"{name} has shape {tuple(shape)}, not [rows, {heads}, {self.head_dim}]")
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{name} requires a gradient: the cache passes none (use torch.no_grad())")
        if has_tangent(t):
            raise RuntimeError(f"{name} carries a tangent: the cache passes none")
        if t.get_device() != self._index:
            raise ValueError(f"{name} is on {t.device}, the cache on {self.device}")
        if t.is_neg():
            t = t.resolve_neg()                          # a view whose sign torch keeps apart from the memory (tensor.conj().imag)
        return t if t.stride(2) == 1 else t.contiguous()

    def _numbers(self, name, t, size):
        """An int32 [size] on the cache's device."""
        if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != size or not t.is_contiguous():
            raise ValueError(f"{name}: {t.dtype} {tuple(t.shape)}, not contiguous int32 [{size}]")
        if t.get_device() != self._index:
            raise ValueError(f"{name} is on {t.device}, the cache on {self.device}")
        return t.data_ptr()

    def _batch(self, table, what, positions, offsets, rows, most):
        """Checks the batch's description; returns the entry points' arguments (table, its stride, positions, offsets), then
        (sequences, width, rows of a sequence at most)."""
        shape = table.shape
        if table.dtype != torch.int32 or len(shape) != 2 or shape[0] < 1 or shape[1] < 1 or (table.stride(1) != 1 and shape[1] > 1):
            raise ValueError(f"table: {table.dtype} {tuple(shape)}, not int32 [sequences, blocks] with adjacent blocks")
        n, width = shape
        at = self._numbers(what, positions, n)
        if offsets is None:
            if rows % n:
                raise ValueError(f"{rows} rows for {n} sequences, and no offsets")
            each = rows // n
            if most is not None and most != each:
                raise ValueError(f"most {most}, but {each} rows each without offsets")
            most, first = each, None
        else:
            first = self._numbers("offsets", offsets, n + 1)
            most = rows if most is None else min(int(most), rows)
            if most < 0:
                raise ValueError(f"most {most}")
        if table.get_device() != self._index:
            raise ValueError(f"table is on {table.device}, the cache on {self.device}")
        if self._index < 0:
            raise RuntimeError("KVCache runs on the GPU only (libvision_amd.so has no CPU path)")
        return (table.data_ptr(), table.stride(0), at, first), n, width, most

    # ---- the operators

    def append(self, k, v, table, start, offsets=None, most=None):
        """Writes rows k, v at positions start[b], start[b]+1, ... of their sequences.  A block whose first token is written starts
        anew (whatever it held behind that is gone); otherwise its scale grows if the rows need it, and its codes move along.  A block
        that gets an infinity or a NaN reads as NaN until it starts anew.  Rows in holes, behind the table's end or of a sequence
        with start < 0 are dropped.  A block that is written must belong to one sequence of the call, and once to that."""
        k, v = self._rows("k", k, self.kv_heads), self._rows("v", v, self.kv_heads)
        if k.dtype != v.dtype or k.shape != v.shape:
            raise ValueError(f"k and v differ: {k.dtype} {tuple(k.shape)}, {v.dtype} {tuple(v.shape)}")
        rows = k.shape[0]
        batch, n, width, most = self._batch(table, "start", start, offsets, rows, most)
        ks, vs = k.stride(), v.stride()
        call_on(self.device, "vamd_kv_append", k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], *self._pool(), *batch, rows, n, most,
                self.kv_heads, self.head_dim, self.block, width, self.blocks, self._format, _TYPES[k.dtype])

    def read(self, table, start, rows, offsets=None, most=None, dtype=torch.bfloat16, out=None):
        """(k, v): the values at positions start[b], start[b]+1, ... of each sequence, `rows` rows in all, exact in either dtype; zeros
        in holes and behind the table's end.  `out`: two tensors [rows, kv_heads, head_dim] to write into; rows of no sequence, beyond `most`
        or of a sequence with start < 0 keep what they held (in a result that the call allocates they hold nothing in particular)."""
        if out is None:
            if dtype not in _TYPES:
                raise TypeError(f"dtype {dtype}: float32 or bfloat16")
            if rows < 0:
                raise ValueError(f"{rows} rows")
            shape = (rows, self.kv_heads, self.head_dim)
            k, v = torch.empty(shape, dtype=dtype, device=self.device), torch.empty(shape, dtype=dtype, device=self.device)
        else:
            k, v = out
            for name, t in (("out[0]", k), ("out[1]", v)):
                self._written(name, t, (rows, self.kv_heads, self.head_dim))
            if k.dtype != v.dtype:
                raise ValueError(f"out: {k.dtype} and {v.dtype}")
            if overlapping(k, v):
                raise ValueError("out's two tensors share memory")
        batch, n, width, most = self._batch(table, "start", start, offsets, rows, most)
        if out is not None:
            overwritten(k, v)
        ks, vs = k.stride(), v.stride()
        call_on(self.device, "vamd_kv_read", *self._pool(), *batch, rows, n, most, self.kv_heads, self.head_dim, self.block, width,
                self.blocks, self._format, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], _TYPES[k.dtype])
        return k, v

    def attend(self, q, table, lengths, offsets=None, most=None, longest=None, scale=None, causal=True, window=0, sinks=0, out=None):
        """softmax(scale * q k^T) v over the first lengths[b] tokens of each sequence, whose queries are its last tokens: query i of n
        has position lengths[b] - n + i.  causal: it sees the tokens up to its position, with `window` > 0 only the last `window` of
        them (its own among them) and the first `sinks`.  A query that sees nothing gives zeros.  Lengths are cut to the table's room.  scale: head_dim ** -0.5 if None.
        longest: a bound of the lengths that the caller knows (default: the table's width); it steers how the work is cut, never
        what is computed.  out: the result's memory, which may be q's own; rows of no sequence keep what it held."""
        if q.dim() != 3 or q.shape[1] < 1 or q.shape[1] % self.kv_heads:
            raise ValueError(f"q has shape {tuple(q.shape)}, not [rows, a multiple of {self.kv_heads}, {self.head_dim}]")
        heads = q.shape[1]
        q = self._rows("q", q, heads)
        if window < 0 or sinks < 0 or (window and not causal):
            raise ValueError(f"window {window}, sinks {sinks}: not negative, and a window needs causal queries")
        window, sinks = min(int(window), _INT_MAX), min(int(sinks), _INT_MAX)
        if out is not None:
            self._written("out", out, q.shape)
            if out.dtype != q.dtype:
                raise ValueError(f"out is {out.dtype}, q {q.dtype}")
            # every row's queries are read before its result is written: the two may be the same memory
            if (q.data_ptr() != out.data_ptr() or q.stride() != out.stride()) and overlapping(q, out):
                raise ValueError("q and out share memory")
        rows = q.shape[0]
        batch, n, width, most = self._batch(table, "lengths", lengths, offsets, rows, most)
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=self.device)
        else:
            overwritten(out)
        room = width * self.block
        longest = room if longest is None else min(max(int(longest), 0), room)
        group = heads // self.kv_heads
        size = lib.vamd_kv_attend_workspace(rows, n, most, longest, self.kv_heads, group, self.head_dim, window, sinks, _TYPES[q.dtype])
        work = torch.empty(size, dtype=torch.uint8, device=self.device) if size else None
        qs, os = q.stride(), out.stride()
        call_on(self.device, "vamd_kv_attend", q.data_ptr(), qs[0], qs[1], *self._pool(), *batch, rows, n, most, longest, self.kv_heads,
                group, self.head_dim, self.block, width, self.blocks, self._format, self.head_dim ** -0.5 if scale is None else float(scale),
                bool(causal), window, sinks, out.data_ptr(), os[0], os[1], None if work is None else work.data_ptr(), size, _TYPES[q.dtype])
        return out

    def _written(self, name, t, shape):
        if t.dtype not in _TYPES or t.shape != shape or t.device != self.device:
            raise ValueError(f"{name} is {t.dtype} {tuple(t.shape)} on {t.device}, not float32 or bfloat16 {tuple(shape)} on {self.device}")
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{name} requires a gradient: the cache passes none (use torch.no_grad())")
        if has_tangent(t):
            raise RuntimeError(f"{name} carries a tangent: the cache passes none")
        if t.numel() and (t.stride(2) != 1 or self_overlapping(t) or t.is_neg()):
            raise ValueError(f"{name} with strides {t.stride()}{' and a lazy sign' if t.is_neg() else ''} cannot be written: adjacent features, no "
                             "element twice")
