"""A decoder's keys and values held in 4 bits, and attention over them.

``KVCache4`` takes the place of the growing ``self_keys / self_values`` (and of the standing ``memory_keys /
memory_values``) of a decoder layer's cache (onmt/decoders/transformer.py:268-287, onmt/modules/multi_headed_attn.py:
131-160): every 32 features of a token and head are 4-bit codes with an fp16 scale and zero, 5 bits a feature where the
reference keeps 32.  Tokens are quantised once, when they are written; ``attention`` multiplies the codes as they lie.

These are decoding operators: they build no graph and refuse inputs that would need one.
"""
import ctypes
import math

import torch

from . import _lib as L

MAX_DIM = 128


def _no_graph(who, *tensors):
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError("%s builds no graph: call it under torch.no_grad()" % who)


def _rows(who, name, x, B, H, dh):
    """A [B, H, T, dh] operand with contiguous features, in any order of the other three."""
    if x.dim() != 4 or x.shape[0] != B or x.shape[1] != H or x.shape[3] != dh:
        raise ValueError("%s: %s [%d, %d, T, %d] expected (got %s)" % (who, name, B, H, dh, tuple(x.shape)))
    return x if x.stride(3) == 1 else x.contiguous()


def _index(who, name, t, B, device):
    """-> (tensor or None, scalar, is int64) of an int or of an integer tensor [B] on the device."""
    if not torch.is_tensor(t):
        return None, int(t), 0
    if t.shape != (B,) or t.dtype not in (torch.int32, torch.int64) or t.device != device:
        raise ValueError("%s: %s must be an int or an int32 / int64 tensor [%d] on %s (got %s %s on %s)" % (
            who, name, B, device, t.dtype, tuple(t.shape), t.device))
    t = t.contiguous()
    return t, 0, int(t.dtype == torch.int64)


class KVCache4:
    """Keys and values of up to ``capacity`` tokens of ``batch`` sentences, ``heads`` heads of ``dim`` features (a
    multiple of 8 up to 128).  It keeps no count of what was written: a caller says where tokens go and how many there are.

    ``nbytes`` is what it holds on the device.  Tokens nothing was written to read as zeros."""

    def __init__(self, batch, heads, dim, capacity, device="cuda"):
        n = L.load().mssr_kv4_bytes(int(batch), int(heads), int(capacity), int(dim))
        if n < 0:
            raise ValueError("KVCache4: %s sentences x %s heads x %s tokens x %s features (a multiple of 8 up to %d)" % (
                batch, heads, capacity, dim, MAX_DIM))
        self.heads, self.dim, self.capacity = int(heads), int(dim), int(capacity)
        # [sentence, bytes]: map() reorders whole sentences
        self.data = torch.zeros(int(batch), n // int(batch), dtype=torch.uint8, device=device)
        L.require_cuda(self.data)

    @property
    def batch(self):
        return self.data.shape[0]

    @property
    def device(self):
        return self.data.device

    @property
    def nbytes(self):
        return self.data.numel()

    def _desc(self):
        return L.Kv4Cache(self.data.data_ptr(), self.batch, self.capacity, self.heads, self.dim)

    def _span(self, who, start, T, counts):
        start, start0, wide = _index(who, "start", start, self.batch, self.device)
        if start is None and not 0 <= start0 <= self.capacity - T:
            raise ValueError("%s: tokens %d .. %d of a cache of %d" % (who, start0, start0 + T, self.capacity))
        if T > self.capacity:
            raise ValueError("%s: %d tokens, the cache holds %d" % (who, T, self.capacity))
        if counts is not None and not torch.is_tensor(counts):
            raise ValueError("%s: counts must be an integer tensor [%d] or None" % (who, self.batch))
        counts, _, wide_c = (None, 0, 0) if counts is None else _index(who, "counts", counts, self.batch, self.device)
        return start, start0, counts, wide | (wide_c << 1)

    def write(self, k, v, start=0, counts=None):
        """Quantises k, v [B, heads, T, dim] (float32 or bfloat16, any strides) to positions ``start`` + 0 .. T - 1.

        ``start``: an int, or an integer tensor [B] (every sentence at its own position); ``counts``: integer tensor [B],
        sentence b writes its first counts[b] tokens only (a padded batch).  Positions outside the cache are dropped where
        ``start`` is a tensor and refused where it is an int.  A group of 32 features that holds a NaN or an infinity reads
        back as NaN; values beyond +-65504 are clamped to that."""
        who = "KVCache4.write"
        _no_graph(who, k, v)
        L.require_cuda(k, v)
        k, v = (_rows(who, n, x, self.batch, self.heads, self.dim) for n, x in (("k", k), ("v", v)))
        T = k.shape[2]
        if v.shape[2] != T or k.dtype != v.dtype or k.device != self.device or v.device != self.device:
            raise ValueError("%s: k and v differ in length, type or device (%s %s %s, %s %s %s; the cache is on %s)" % (
                who, tuple(k.shape), k.dtype, k.device, tuple(v.shape), v.dtype, v.device, self.device))
        start, start0, counts, bits = self._span(who, start, T, counts)
        if self.batch == 0:
            return
        with torch.cuda.device(self.device):
            d = self._desc()
            L.check(L.load().mssr_kv4_write(ctypes.byref(d), k.data_ptr(), k.stride(0), k.stride(1), k.stride(2),
                                            v.data_ptr(), v.stride(0), v.stride(1), v.stride(2), T, L.ptr(start), start0,
                                            L.ptr(counts), bits, L.dt(k), L.stream()), "kv4_write")

    def read(self, start, length, counts=None, dtype=torch.float32):
        """(k, v), each [B, heads, length, dim] (a view of [B, length, heads, dim] memory), of positions ``start`` + 0 ..
        length - 1 in ``dtype``; zeros past counts[b] and outside the cache.  Arguments as in ``write``."""
        who, T = "KVCache4.read", int(length)
        if T < 0:
            raise ValueError("%s: length %d" % (who, T))
        start, start0, counts, bits = self._span(who, start, T, counts)
        k, v = (torch.empty(self.batch, T, self.heads, self.dim, dtype=dtype, device=self.device).transpose(1, 2)
                for _ in "kv")
        if self.batch == 0:
            return k, v
        with torch.cuda.device(self.device):
            d = self._desc()
            L.check(L.load().mssr_kv4_read(ctypes.byref(d), k.data_ptr(), k.stride(0), k.stride(1), k.stride(2),
                                           v.data_ptr(), v.stride(0), v.stride(1), v.stride(2), T, L.ptr(start), start0,
                                           L.ptr(counts), bits, L.dt(k), L.stream()), "kv4_read")
        return k, v

    def map(self, fn):
        """Reorders the sentences: ``fn(tensor, batch_dim)`` as in TransformerDecoder.map_state."""
        self.data = fn(self.data, 0).contiguous()


def attention(q, cache, lengths, scale=None, causal=False, longest=0):
    """softmax(scale * q k^T) v over the first ``lengths`` tokens of every sentence in ``cache``.

    q [B, H, T, dim] (float32 or bfloat16, any strides), H a multiple of the cache's heads: query head h reads head
    h // (H / heads).  ``lengths``: an int or an integer tensor [B].  ``scale``: 1 / sqrt(dim) if not given.  ``causal``: the
    rows are the sentence's last T tokens (their keys written already), row i sees the first lengths - T + 1 + i.  A row
    that sees no token gives zeros.  ``longest``: an upper bound of the lengths, if the caller knows one below the cache's
    capacity (it shapes the launch, nothing else).  Returns [B, H, T, dim], a view of [B, T, H, dim] memory, in q's type;
    probabilities are not returned."""
    who = "kv_cache.attention"
    _no_graph(who, q)
    L.require_cuda(q)
    if q.dim() != 4 or q.shape[1] % cache.heads or q.shape[1] == 0:
        raise ValueError("%s: q [%d, n * %d, T, %d] expected (got %s)" % (who, cache.batch, cache.heads, cache.dim,
                                                                        tuple(q.shape)))
    if q.device != cache.device:
        raise ValueError("%s: q is on %s, the cache on %s" % (who, q.device, cache.device))
    B, H, T, dh = q.shape
    q = _rows(who, "q", q, cache.batch, H, cache.dim)
    lengths, n, wide = _index(who, "lengths", lengths, B, q.device)
    if lengths is None and not 0 <= n <= cache.capacity:
        raise ValueError("%s: %d tokens of a cache of %d" % (who, n, cache.capacity))
    scale = 1.0 / math.sqrt(dh) if scale is None else float(scale)
    out = torch.empty(B, T, H, dh, dtype=q.dtype, device=q.device).transpose(1, 2)
    code = L.dt(q)
    lib, d = L.load(), cache._desc()
    longest = int(longest) if lengths is not None else n
    if T == 0 or B == 0:
        return out
    with torch.cuda.device(q.device):
        need = lib.mssr_kv4_attention_scratch(ctypes.byref(d), T, H, longest, code)
        # from the allocator, per call: a call's scratch is its own on every stream and in every captured graph
        ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need > 0 else None
        L.check(lib.mssr_kv4_attention(ctypes.byref(d), q.data_ptr(), q.stride(0), q.stride(1), q.stride(2), out.data_ptr(),
                                       out.stride(0), out.stride(1), out.stride(2), H, T, L.ptr(lengths), n, wide, longest,
                                       scale, int(bool(causal)), L.ptr(ws), max(need, 0), code, L.stream()), "kv4_attention")
    return out
