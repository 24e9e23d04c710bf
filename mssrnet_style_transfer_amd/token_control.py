"""Control of the next token's logits: penalties for tokens that were used, biases, grammar masks, no repeated n-grams.

What stands between a decoder's generator and its pick (the reference's search takes the largest logit,
onmt/translate/greedy_search.py:135-165, with its n-gram rule in onmt/translate/decode_strategy.py): one pass over the
logits, which leaves either new logits (for a sampler) or only the picked ids.  Decoding operators: they build no graph and
refuse logits, biases and rates that would need one, or that carry a forward-mode tangent.
"""
from dataclasses import dataclass
from functools import lru_cache
from typing import Optional, Union

import torch

from . import _lib as L


@dataclass
class TokenControl:
    """The rules of a batch.  In fp32, each step rounded, for every word v of the vocabulary:

    1. a word of the history: ``x = x / repetition`` where x > 0, ``x * repetition`` elsewhere;
    2. where the history holds it ``count > 0`` times from prompt_lengths on: ``x - (frequency * count + presence)``;
    3. ``x + bias[v]``;
    4. minus infinity where ``allowed`` has no bit for it, or where it would complete an ``ngram``-gram of the history
       (1: no word twice).

    ``repetition, frequency, presence``: numbers, or float32 tensors [B].  ``bias``: float32 [V] or [B, V].  ``allowed``:
    int32 [S, (V + 31) // 32], bit v % 32 of word v // 32 (``pack_allowed``); ``state``: integer tensor [B], the row of
    ``allowed`` for each sentence (below 0: no rule for it; a number that is not a row allows nothing); without ``state``
    S is 1 (one row for all) or B."""
    repetition: Union[float, torch.Tensor] = 1.0
    frequency: Union[float, torch.Tensor] = 0.0
    presence: Union[float, torch.Tensor] = 0.0
    ngram: int = 0
    bias: Optional[torch.Tensor] = None
    allowed: Optional[torch.Tensor] = None
    state: Optional[torch.Tensor] = None

    def rows(self, index, batch):
        """The rules of the sentences ``index`` (int64 tensor) of a batch of ``batch``."""
        def pick(t, per_row):
            return t.index_select(0, index) if torch.is_tensor(t) and per_row(t) else t
        vec = lambda t: True                                                                   # noqa: E731
        shared = self.state is not None or (self.allowed is not None and self.allowed.shape[0] == 1 and batch != 1)
        return TokenControl(pick(self.repetition, vec), pick(self.frequency, vec), pick(self.presence, vec), self.ngram,
                            pick(self.bias, lambda t: t.dim() == 2), pick(self.allowed, lambda t: not shared),
                            pick(self.state, vec))


_NO_RULES = TokenControl()


def pack_allowed(allowed):
    """Bool [S, V] -> the int32 words [S, (V + 31) // 32] that ``TokenControl.allowed`` takes."""
    if allowed.dim() != 2 or allowed.dtype != torch.bool:
        raise ValueError("pack_allowed: a Bool [S, V] tensor expected (got %s %s)" % (allowed.dtype, tuple(allowed.shape)))
    S, V = allowed.shape
    bits = torch.nn.functional.pad(allowed, (0, -V % 32)).view(S, -1, 32).long()
    words = (bits << torch.arange(32, device=allowed.device)).sum(2)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).int()


_INTS = (torch.int32, torch.int64)
_pack = L.packer(L.TokenControlDesc)


@lru_cache(maxsize=1024)
def _scratch_bytes(B, V, T):
    """How much scratch a pick of this shape takes: a number of the shape alone."""
    return L.load().mssr_token_control_scratch(B, V, T)


def _int_error(who, name, shape, device):
    raise ValueError("%s: %s must be an int32 / int64 tensor %s on %s" % (who, name, shape, device))


def _vector(who, name, t, B, device):
    """-> (contiguous integer tensor [B], its element is 64 bits wide)."""
    if not isinstance(t, torch.Tensor) or t.shape != (B,) or t.dtype not in _INTS or t.device != device:
        _int_error(who, name, "[%d]" % B, device)
    return (t if t.is_contiguous() else t.contiguous()), t.dtype is torch.int64


def _rate(who, name, x, B, device):
    """-> (tensor or None, number) of a penalty."""
    if not isinstance(x, torch.Tensor):
        return None, float(x)
    if x.shape != (B,) or x.dtype != torch.float32 or x.device != device:
        raise ValueError("%s: %s must be a number or a float32 tensor [%d] on %s (got %s %s on %s)" % (
            who, name, B, device, x.dtype, tuple(x.shape), x.device))
    return (x if x.is_contiguous() else x.contiguous()), 0.0


def _address(t):
    return 0 if t is None else t.data_ptr()


def _call(who, logits, control, history, lengths, prompt_lengths, out, ids, empty):
    """Checks, then one call; every tensor made on the way is a local and lives until it is launched."""
    c = _NO_RULES if control is None else control
    L.refuse_graph(who, logits, c.bias, c.repetition, c.frequency, c.presence, out)
    if not logits.is_cuda:
        L.require_cuda(logits)
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError("%s: logits [B, V] expected (got %s)" % (who, tuple(logits.shape)))
    B, V = logits.shape
    dev = logits.device
    if not logits.is_contiguous() and (V > 1 and logits.stride(1) != 1 or B > 1 and logits.stride(0) < V):
        logits = logits.contiguous()
    bits = h_bs = h_ts = T = bias_bs = states = mode = 0
    if history is not None:
        if not isinstance(history, torch.Tensor) or history.dim() != 2 or history.shape[0] != B or \
                history.dtype not in _INTS or history.device != dev:
            _int_error(who, "history", "[%d, T]" % B, dev)
        bits = int(history.dtype is torch.int64)
        h_bs, h_ts = history.stride()
        T = history.shape[1]
        if lengths is not None:
            lengths, wide = _vector(who, "lengths", lengths, B, dev)
            bits |= 2 * wide
        if prompt_lengths is not None:
            prompt_lengths, wide = _vector(who, "prompt_lengths", prompt_lengths, B, dev)
            bits |= 4 * wide
    elif lengths is not None or prompt_lengths is not None:
        raise ValueError("%s: lengths without a history" % who)
    rep, rep0 = _rate(who, "repetition", c.repetition, B, dev)
    freq, freq0 = _rate(who, "frequency", c.frequency, B, dev)
    pres, pres0 = _rate(who, "presence", c.presence, B, dev)
    if not 0 <= c.ngram <= 64:
        raise ValueError("%s: ngram %d (0 = none, up to 64)" % (who, c.ngram))
    bias, allowed, state = c.bias, c.allowed, c.state
    if bias is not None:
        if bias.dtype != torch.float32 or bias.device != dev or tuple(bias.shape) not in ((V,), (B, V)):
            raise ValueError("%s: bias must be a float32 tensor [%d] or [%d, %d] on %s (got %s %s on %s)" % (
                who, V, B, V, dev, bias.dtype, tuple(bias.shape), bias.device))
        if bias.stride(-1) != 1:
            bias = bias.contiguous()
        if bias.dim() == 2:
            bias_bs = bias.stride(0)
    if allowed is not None:
        states = allowed.shape[0]
        if allowed.dim() != 2 or allowed.shape[1] != (V + 31) // 32 or states < (B > 0) or allowed.dtype != torch.int32 or \
                allowed.device != dev:
            raise ValueError("%s: allowed must be an int32 tensor [S, %d] on %s" % (who, (V + 31) // 32, dev))
        if not allowed.is_contiguous():
            allowed = allowed.contiguous()
        if state is not None:
            state, wide = _vector(who, "state", state, B, dev)
            mode = 2
            bits |= 8 * wide
        elif states == B:
            mode = 1
        elif states != 1:
            raise ValueError("%s: %d rows of allowed words for %d sentences need a state" % (who, states, B))
    elif state is not None:
        raise ValueError("%s: a state without a table of allowed words" % who)
    code = L.dt(logits)
    if B == 0:
        return
    ws, need = None, 0
    if ids is not None:
        bits |= 16 * int(ids.dtype is torch.int64)
        need = _scratch_bytes(B, V, T)
        if need > 0:                             # a call's own: streams and captured graphs share none
            ws = torch.empty(need, dtype=torch.uint8, device=dev)
    ptr = _address
    L.call("mssr_token_control", dev, _pack(
        logits.data_ptr(), ptr(out), B, V, logits.stride(0) if B > 1 else V,
        0 if out is None else (out.stride(0) if B > 1 else V), ptr(history), h_bs, h_ts, T, ptr(lengths),
        ptr(prompt_lengths), ptr(rep), ptr(freq), ptr(pres), rep0, freq0, pres0, int(c.ngram), ptr(bias), bias_bs, ptr(allowed),
        states, ptr(state), mode, ptr(ids), int(empty), bits, code, ptr(ws), need))


def control_logits(logits, control=None, history=None, lengths=None, prompt_lengths=None, out=None):
    """The logits [B, V] (float32 or bfloat16, contiguous rows) under the rules of ``control``, in the same type.

    ``history``: int32 / int64 tensor [B, T] of tokens so far, any strides (a [T, B] buffer's transpose is read in place);
    entries outside the vocabulary are passed over.  ``lengths``: integer tensor [B], how many of them count (default: all).
    ``prompt_lengths``: integer tensor [B], frequency and presence count from there on.  ``out``: where to write; ``logits``
    itself changes them in place (memory that overlaps theirs in another way, or the bias, is refused)."""
    who = "control_logits"
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    elif out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device or logits.dim() != 2 or \
            (out.shape[1] > 1 and out.stride(1) != 1) or (out.shape[0] > 1 and out.stride(0) < out.shape[1]):
        raise ValueError("%s: out must be like logits with contiguous rows" % who)
    _call(who, logits, control, history, lengths, prompt_lengths, out, None, 0)
    return out


def pick_token(logits, control=None, history=None, lengths=None, prompt_lengths=None, empty=-1, out=None):
    """The word with the largest controlled logit of every row, int64 [B] (or written to ``out``, an int32 / int64 tensor
    [B]): the lowest one on ties, NaN above everything as in torch.argmax, ``empty`` where every word is at minus infinity.
    Other arguments as for ``control_logits``; the new logits are not written.  ``out`` may lie in the history past ``lengths``."""
    who = "pick_token"
    if logits.dim() != 2:
        raise ValueError("%s: logits [B, V] expected (got %s)" % (who, tuple(logits.shape)))
    if out is None:
        out = torch.empty(logits.shape[0], dtype=torch.int64, device=logits.device)
    elif out.shape != logits.shape[:1] or out.dtype not in (torch.int32, torch.int64) or out.device != logits.device or \
            not out.is_contiguous():
        raise ValueError("%s: out must be a contiguous int32 / int64 tensor [%d]" % (who, logits.shape[0]))
    _call(who, logits, control, history, lengths, prompt_lengths, None, out, empty)
    return out
