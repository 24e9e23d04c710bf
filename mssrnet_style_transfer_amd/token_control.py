"""Control of the next token's logits: penalties for tokens that were used, biases, grammar masks, no repeated n-grams.

What stands between a decoder's generator and its pick (the reference's search takes the largest logit,
onmt/translate/greedy_search.py:135-165, with its n-gram rule in onmt/translate/decode_strategy.py): one pass over the
logits, which leaves either new logits (for a sampler) or only the picked ids.  Decoding operators: they build no graph.
"""
import ctypes
from dataclasses import dataclass
from typing import Optional, Union

import torch

from . import _lib as L


@dataclass
class TokenControl:
    """The rules of a batch.  In fp32, each step rounded, for every word v of the vocabulary:

    1. a word of the history: ``x = x / repetition`` where x > 0, ``x * repetition`` elsewhere;
    2. ``x - (frequency * count + presence * (count > 0))``, count = how often the history holds it from prompt_lengths on;
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


def pack_allowed(allowed):
    """Bool [S, V] -> the int32 words [S, (V + 31) // 32] that ``TokenControl.allowed`` takes."""
    if allowed.dim() != 2 or allowed.dtype != torch.bool:
        raise ValueError("pack_allowed: a Bool [S, V] tensor expected (got %s %s)" % (allowed.dtype, tuple(allowed.shape)))
    S, V = allowed.shape
    bits = torch.nn.functional.pad(allowed, (0, -V % 32)).view(S, -1, 32).long()
    words = (bits << torch.arange(32, device=allowed.device)).sum(2)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).int()


def _ids(who, name, t, shape, device):
    if t is None:
        return None, 0
    if not torch.is_tensor(t) or t.dim() != len(shape) or any(s not in (None, n) for s, n in zip(shape, t.shape)) \
            or t.dtype not in (torch.int32, torch.int64) or t.device != device:
        raise ValueError("%s: %s must be an int32 / int64 tensor %s on %s" % (
            who, name, [s if s is not None else "T" for s in shape], device))
    return t, int(t.dtype == torch.int64)


def _f32(who, name, t, shapes, device):
    if t.dtype != torch.float32 or t.device != device or tuple(t.shape) not in shapes:
        raise ValueError("%s: %s must be a float32 tensor %s on %s (got %s %s on %s)" % (
            who, name, " or ".join(map(str, map(list, shapes))), device, t.dtype, tuple(t.shape), t.device))
    return t


def _call(who, logits, control, history, lengths, prompt_lengths, out, ids, empty):
    if torch.is_grad_enabled() and logits.requires_grad:
        raise RuntimeError("%s builds no graph: call it under torch.no_grad()" % who)
    L.require_cuda(logits)
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError("%s: logits [B, V] expected (got %s)" % (who, tuple(logits.shape)))
    B, V = logits.shape
    dev = logits.device
    if V > 1 and logits.stride(1) != 1 or B > 1 and logits.stride(0) < V:
        logits = logits.contiguous()
    c = TokenControl() if control is None else control
    d = L.TokenControlDesc()
    keep = []                                    # operands made here live until the launch

    def hold(t):
        keep.append(t)
        return t.data_ptr()

    d.logits, d.B, d.V, d.ld, d.dtype = logits.data_ptr(), B, V, (logits.stride(0) if B > 1 else V), L.dt(logits)
    bits = 0
    if history is not None:
        history, wide = _ids(who, "history", history, (B, None), dev)
        bits |= wide
        d.history, d.h_bs, d.h_ts, d.T = history.data_ptr(), history.stride(0), history.stride(1), history.shape[1]
    for name, t, bit in (("lengths", lengths, 2), ("prompt_lengths", prompt_lengths, 4)):
        t, wide = _ids(who, name, t, (B,), dev)
        if t is not None:
            if history is None:
                raise ValueError("%s: %s without a history" % (who, name))
            setattr(d, name, hold(t.contiguous()))
            bits |= bit * wide
    for name in ("repetition", "frequency", "presence"):
        t = getattr(c, name)
        if torch.is_tensor(t):
            setattr(d, name, hold(_f32(who, name, t, ((B,),), dev).contiguous()))
        else:
            setattr(d, name + "0", float(t))
    if c.ngram < 0 or c.ngram > 64:
        raise ValueError("%s: ngram %d (0 = none, up to 64)" % (who, c.ngram))
    d.ngram = int(c.ngram)
    if c.bias is not None:
        t = _f32(who, "bias", c.bias, ((V,), (B, V)), dev)
        if t.stride(-1) != 1 and V > 1:
            t = t.contiguous()
        d.bias, d.bias_bs = hold(t), (t.stride(0) if t.dim() == 2 and B > 1 else 0)
    if c.state is not None and c.allowed is None:
        raise ValueError("%s: a state without a table of allowed words" % who)
    if c.allowed is not None:
        W = (V + 31) // 32
        t, _ = _ids(who, "allowed", c.allowed, (None, W), dev)
        if t.dtype != torch.int32 or t.shape[0] < 1:
            raise ValueError("%s: allowed must be int32 [S, %d]" % (who, W))
        S = t.shape[0]
        d.allowed, d.states = hold(t.contiguous()), S
        if c.state is not None:
            t, wide = _ids(who, "state", c.state, (B,), dev)
            d.state, d.state_mode = hold(t.contiguous()), 2
            bits |= 8 * wide
        elif S in (1, B):
            d.state_mode = 0 if S == 1 else 1
        else:
            raise ValueError("%s: %d rows of allowed words for %d sentences need a state" % (who, S, B))
    if out is not None:
        d.out, d.ldo = out.data_ptr(), (out.stride(0) if B > 1 else V)
    with torch.cuda.device(dev):
        lib = L.load()
        if ids is not None:
            d.ids, d.empty = ids.data_ptr(), int(empty)
            bits |= 16 * int(ids.dtype == torch.int64)
            need = lib.mssr_token_control_scratch(max(B, 1), V)
            if need > 0:                         # a call's own: streams and captured graphs share none
                d.scratch, d.scratch_bytes = hold(torch.empty(need, dtype=torch.uint8, device=dev)), need
        d.index_bits = bits
        L.check(lib.mssr_token_control(ctypes.byref(d), L.stream()), "token_control")


def control_logits(logits, control=None, history=None, lengths=None, prompt_lengths=None, out=None):
    """The logits [B, V] (float32 or bfloat16, contiguous rows) under the rules of ``control``, in the same type.

    ``history``: int32 / int64 tensor [B, T] of tokens so far, any strides (a [T, B] buffer's transpose is read in place);
    entries outside the vocabulary are passed over.  ``lengths``: integer tensor [B], how many of them count (default: all).
    ``prompt_lengths``: integer tensor [B], frequency and presence count from there on.  ``out``: where to write; ``logits``
    itself changes them in place."""
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
    Other arguments as for ``control_logits``; the new logits are not written."""
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
