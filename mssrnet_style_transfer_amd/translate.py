"""Greedy style-transfer decoding (trans_beam_size 1).

Counterpart of onmt/translate/translator_wh.py: ``_run_encoder`` (:576-605: StyleGenerator2 +
TransformerEncoder + BondLayer) and the step loop of ``_translate_batch_with_strategy`` (:665-756)
with ``GreedySearch`` (onmt/translate/greedy_search.py:59-190).  Text I/O (fields, TranslationBuilder,
post_handle_sent) is outside the path: the result is token ids per sentence.
"""
import torch

from . import ops
from .decode_engine import greedy_decode_ids
from .token_control import pick_token


def greedy_decode_cached(model, cfg, memory_bank, src_lengths, max_length, kv_bits=4, control=None, check_every=4):
    """decode_engine.greedy_decode_ids with the decoder's keys and values in a 4-bit cache (TransformerDecoder.init_state):
    for memory banks and decodes too long, or batches too large, for full-precision ones.  The step loop runs over
    TransformerDecoder.forward(step=s); finished sentences leave the batch at the check points.  Token ids int32 [steps, B],
    past a sentence's first </s> unspecified."""
    dev, B = memory_bank.device, memory_bank.size(1)
    src_lengths = src_lengths.to(dev)
    if max_length == 0:
        return torch.empty(0, B, dtype=torch.int32, device=dev)
    with torch.no_grad():
        src = torch.zeros(memory_bank.size(0), B, 1, dtype=torch.long, device=dev)
        model.decoder.init_state(src, memory_bank, None, kv_bits=kv_bits, max_steps=max_length)
        try:
            return _cached_steps(model, cfg, memory_bank, src_lengths, max_length, control, check_every)
        finally:                                            # the cache goes with the search, not into the next checkpoint
            model.decoder.init_state(None, None, None)


def _cached_steps(model, cfg, memory_bank, src_lengths, max_length, control, check_every):
    """The steps of greedy_decode_cached over the decoder's state."""
    dev, B, lin = memory_bank.device, memory_bank.size(1), model.generator[0]
    out = torch.full((max_length, B), cfg.eos_idx, dtype=torch.int32, device=dev)
    ids = torch.full((max_length, B), cfg.eos_idx, dtype=torch.int32, device=dev)     # columns of the running sentences
    rows = torch.arange(B, device=dev)
    tok = torch.full((1, B, 1), cfg.bos_idx, dtype=torch.long, device=dev)
    done = torch.zeros(B, dtype=torch.bool, device=dev)
    flushed = steps = 0
    for step in range(max_length):
        dec_out, _ = model.decoder(tok, memory_bank, memory_lengths=src_lengths, step=step)
        logits = ops.linear(dec_out[-1], lin.weight, lin.bias)
        pick_token(logits, control, ids[:step].t() if step else None, empty=cfg.eos_idx, out=ids[step])
        tok = ids[step].long().view(1, -1, 1)
        steps = step + 1
        if steps % check_every and steps != max_length:
            continue
        out[flushed:steps, rows] = ids[flushed:steps]
        done[rows] |= (ids[flushed:steps] == cfg.eos_idx).any(0)
        flushed = steps
        keep = (~done[rows]).nonzero().squeeze(1)       # the one host sync of this check point
        if keep.numel() == 0 or steps == max_length:
            break
        if keep.numel() < rows.numel():
            model.decoder.map_state(lambda t, dim: t.index_select(dim, keep))
            memory_bank, src_lengths = memory_bank.index_select(1, keep), src_lengths.index_select(0, keep)
            if control is not None:
                control = control.rows(keep, rows.numel())
            tok, ids, rows = tok.index_select(1, keep), ids.index_select(1, keep), rows.index_select(0, keep)
    return out[:steps]


def greedy_translate(model, style_generator, cfg, src, src_lengths, desired_styles, max_length=100, control=None,
                     kv_bits=None):
    """src Long [L, B, 1], src_lengths Long [B], desired_styles Long [B] -> list of B token-id lists, each
    ending at its first </s> (inclusive) or cut at ``max_length`` (GreedySearch.update_finished semantics).

    ``control``: token_control.TokenControl, rules for every step's logits over the sentence so far (penalties for repeated
    words, biases, words allowed per sentence, no repeated n-grams).  ``kv_bits=4``: keys and values in a 4-bit cache
    (greedy_decode_cached)."""
    model.eval()
    style_generator.eval()
    with torch.no_grad():
        rep = style_generator(desired_styles, src, src_lengths)
        enc_state, memory_bank, lengths = model.encoder(src, src_lengths)
        memory_bank = model.bond_layer(memory_bank, rep)
        if kv_bits is None:
            model.decoder.init_state(src, memory_bank, enc_state)
            ids = greedy_decode_ids(model, cfg, memory_bank, src_lengths, max_length, control=control)
        else:
            ids = greedy_decode_cached(model, cfg, memory_bank, src_lengths, max_length, kv_bits, control)
    rows = ids.t().tolist()
    out = []
    for sent in rows:
        cut = sent.index(cfg.eos_idx) + 1 if cfg.eos_idx in sent else len(sent)
        out.append(sent[:cut])
    return out
