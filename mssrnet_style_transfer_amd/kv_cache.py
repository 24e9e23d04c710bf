"""A decoder's keys and values held in 4 bits, and attention over them.

``KVCache4`` takes the place of the growing ``self_keys / self_values`` (and of the standing ``memory_keys /
memory_values``) of a decoder layer's cache (onmt/decoders/transformer.py:268-287, onmt/modules/multi_headed_attn.py:
131-160): every 32 features of a token and head are 4-bit codes with an fp16 scale and zero, 5 bits a feature where the
reference keeps 32.  Tokens are quantised once, when they are written; ``attention`` multiplies the codes as they lie.

These are decoding operators: they build no graph and refuse inputs that would need one, or that carry a forward-mode tangent.
"""
import ctypes
from functools import lru_cache

import torch

from . import _lib as L

MAX_DIM = 128


_INTS = (torch.int32, torch.int64)
_pack_rows, _pack_attention = L.packer(L.Kv4Rows), L.packer(L.Kv4AttentionDesc)


def _index(who, name, t, B, device):
    """-> (tensor or None, scalar, is int64) of an int or of an integer tensor [B] on the device."""
    if not isinstance(t, torch.Tensor):
        return None, int(t), 0
    dtype = t.dtype
    if t.shape != (B,) or dtype not in _INTS or t.device != device:
        raise ValueError("%s: %s must be an int or an int32 / int64 tensor [%d] on %s (got %s %s on %s)" % (
            who, name, B, device, dtype, tuple(t.shape), t.device))
    return (t if t.is_contiguous() else t.contiguous()), 0, int(dtype is torch.int64)


def _address(t):
    return 0 if t is None else t.data_ptr()


@lru_cache(maxsize=1024)
def _scratch_bytes(B, Hkv, capacity, dh, T, H, longest, code):
    """How much scratch a shape takes: a number of the shape alone."""
    return L.load().mssr_kv4_attention_scratch(ctypes.byref(L.Kv4Cache(None, B, capacity, Hkv, dh)), T, H, longest, code)


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
        self._held = None
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

    def __getstate__(self):
        return dict(self.__dict__, _held=None)      # checkpoints and copies hold the data, not its address

    def _desc(self):
        """(what it describes, the C descriptor of the present data, its address), built again where the data has moved or
        changed its batch.  A caller keeps the tuple until its C call is over: another thread may have replaced it here by
        then, and the address alone keeps nothing alive."""
        at, held = (self.data.data_ptr(), self.data.shape[0]), self._held
        if held is None or held[0] != at:
            d = L.Kv4Cache(*at, self.capacity, self.heads, self.dim)
            self._held = held = (at, d, ctypes.addressof(d))
        return held

    def _span(self, who, start, T, counts):
        B, device = self.batch, self.device
        start, start0, wide = _index(who, "start", start, B, device)
        if T > self.capacity or (start is None and not 0 <= start0 <= self.capacity - T):
            raise ValueError("%s: tokens %d .. %d of a cache of %d" % (who, start0, start0 + T, self.capacity))
        if counts is None:
            return start, start0, None, wide
        if not isinstance(counts, torch.Tensor):
            raise ValueError("%s: counts must be an integer tensor [%d] or None" % (who, B))
        counts, _, wide_c = _index(who, "counts", counts, B, device)
        return start, start0, counts, wide | (wide_c << 1)

    def _rows(self, who, name, x):
        shape = x.shape
        if len(shape) != 4 or shape[0] != self.batch or shape[1] != self.heads or shape[3] != self.dim:
            raise ValueError("%s: %s [%d, %d, T, %d] expected (got %s)" % (who, name, self.batch, self.heads, self.dim,
                                                                         tuple(shape)))
        return x if x.stride(3) == 1 else x.contiguous()

    def write(self, k, v, start=0, counts=None):
        """Quantises k, v [B, heads, T, dim] (float32 or bfloat16, any strides) to positions ``start`` + 0 .. T - 1.

        ``start``: an int, or an integer tensor [B] (every sentence at its own position); ``counts``: integer tensor [B],
        sentence b writes its first counts[b] tokens only (a padded batch).  Positions outside the cache are dropped where
        ``start`` is a tensor and refused where it is an int.  A group of 32 features that holds a NaN or an infinity reads
        back as NaN; values beyond +-65504 are clamped to that."""
        who = "KVCache4.write"
        L.refuse_graph(who, k, v)
        if not (k.is_cuda and v.is_cuda):
            L.require_cuda(k, v)
        k, v = self._rows(who, "k", k), self._rows(who, "v", v)
        device, T = self.device, k.shape[2]
        if v.shape[2] != T or k.dtype != v.dtype or k.device != device or v.device != device:
            raise ValueError("%s: k and v differ in length, type or device (%s %s %s, %s %s %s; the cache is on %s)" % (
                who, tuple(k.shape), k.dtype, k.device, tuple(v.shape), v.dtype, v.device, device))
        start, start0, counts, bits = self._span(who, start, T, counts)
        if self.batch == 0:
            return
        kb, kh, kt, _ = k.stride()
        vb, vh, vt, _ = v.stride()
        held = self._desc()
        L.call("mssr_kv4_write", device, _pack_rows(
            held[2], k.data_ptr(), kb, kh, kt, v.data_ptr(), vb, vh, vt, T, _address(start), start0, _address(counts),
            bits, L.dt(k)))

    def read(self, start, length, counts=None, dtype=torch.float32):
        """(k, v), each [B, heads, length, dim] (a view of [B, length, heads, dim] memory), of positions ``start`` + 0 ..
        length - 1 in ``dtype``; zeros past counts[b] and outside the cache.  Arguments as in ``write``."""
        who, T = "KVCache4.read", int(length)
        if T < 0:
            raise ValueError("%s: length %d" % (who, T))
        start, start0, counts, bits = self._span(who, start, T, counts)
        B, H, dh = self.batch, self.heads, self.dim
        # one allocation for both: [2, B, T, H, dh]
        both = torch.empty_strided((2, B, H, T, dh), (B * T * H * dh, T * H * dh, dh, H * dh, 1), dtype=dtype,
                                   device=self.device)
        k, v = both.unbind(0)
        if B == 0:
            return k, v
        held = self._desc()
        L.call("mssr_kv4_read", self.device, _pack_rows(
            held[2], k.data_ptr(), T * H * dh, dh, H * dh, v.data_ptr(), T * H * dh, dh, H * dh, T, _address(start),
            start0, _address(counts), bits, L.dt(k)))
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
    capacity (it shapes the launch, nothing else).  Sums are fp32 ones of operands of 22 bits.  Returns [B, H, T, dim], a view of [B, T, H, dim] memory, in q's type;
    probabilities are not returned."""
    who = "kv_cache.attention"
    L.refuse_graph(who, q)
    if not q.is_cuda:
        L.require_cuda(q)
    device, shape, dh = cache.device, q.shape, cache.dim
    if len(shape) != 4 or shape[0] != cache.batch or shape[3] != dh or shape[1] % cache.heads or shape[1] == 0:
        raise ValueError("%s: q [%d, n * %d, T, %d] expected (got %s)" % (who, cache.batch, cache.heads, dh, tuple(shape)))
    if q.device != device:
        raise ValueError("%s: q is on %s, the cache on %s" % (who, q.device, device))
    B, H, T, _ = shape
    if q.stride(3) != 1:
        q = q.contiguous()
    lengths, n, wide = _index(who, "lengths", lengths, B, device)
    if lengths is None:
        longest = n
        if not 0 <= n <= cache.capacity:
            raise ValueError("%s: %d tokens of a cache of %d" % (who, n, cache.capacity))
    code = L.dt(q)
    out = torch.empty_strided((B, H, T, dh), (T * H * dh, dh, H * dh, 1), dtype=q.dtype, device=device)
    if T == 0 or B == 0:
        return out
    need = _scratch_bytes(B, cache.heads, cache.capacity, dh, T, H, longest, code)
    # from the allocator, per call: a call's scratch is its own on every stream and in every captured graph
    ws = torch.empty(need, dtype=torch.uint8, device=device) if need > 0 else None
    qb, qh, qt, _ = q.stride()
    held = cache._desc()
    L.call("mssr_kv4_attention", device, _pack_attention(
        held[2], q.data_ptr(), qb, qh, qt, out.data_ptr(), T * H * dh, dh, H * dh, T, _address(lengths), n, longest,
        _address(ws), need, H, wide, dh ** -0.5 if scale is None else scale, 1 if causal else 0, code))
    return out
