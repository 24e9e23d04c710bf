"""Measured cases of the decoding operators: the 4-bit key/value cache (write, read back), attention over it, and the
control of the next token's logits.

Each case runs either in plain torch (``own = False``: products, comparisons, indexing in 32 bits, rounded once) or
through this package's operators (``own = True``) on the same inputs."""
import math

import torch

own = False

DEV = "cuda"
F15 = torch.tensor(1.0 / 15.0, dtype=torch.float32).item()      # the fp32 number nearest 1/15
TOP = 65504.0                                                    # largest finite fp16 value
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of the batch-512 greedy search: one token a sentence, each at its own position
        dict(name="cache_step", op="cache", B=512, H=8, dh=64, T=1, cap=256, dtype="bf16", ragged=True),
        # the memory bank's keys and values of a padded batch of 64-128 word sentences (label + words)
        dict(name="cache_memory", op="cache", B=256, H=8, dh=64, T=130, cap=130, dtype="fp32", ragged=True),
        # long prompts with wide heads
        dict(name="cache_prompt", op="cache", B=8, H=8, dh=128, T=8191, cap=8192, dtype="bf16", ragged=False),
        # a single sentence's decode step: latency
        dict(name="attend_one", op="attend", B=1, H=8, Hkv=8, dh=64, Tq=1, L=20, low=20, dtype="bf16", causal=True),
        # the batch-512 greedy search at the long workload's lengths
        dict(name="attend_batch", op="attend", B=512, H=8, Hkv=8, dh=64, Tq=1, L=140, low=65, dtype="bf16", causal=True),
        # a document-length cache of a few sentences
        dict(name="attend_long", op="attend", B=16, H=8, Hkv=8, dh=64, Tq=1, L=32768, low=20000, dtype="bf16", causal=True),
        # shared key/value heads in full precision
        dict(name="attend_shared_fp32", op="attend", B=8, H=32, Hkv=8, dh=128, Tq=1, L=8190, low=4001, dtype="fp32",
             causal=True),
        # several new tokens at once (forced words, drafted words), odd head size
        dict(name="attend_chunk", op="attend", B=24, H=16, Hkv=4, dh=96, Tq=5, L=2050, low=700, dtype="bf16", causal=True),
        # the pick of one sentence's next word at this framework's vocabulary
        dict(name="pick_one", op="pick", B=1, V=9606, hist=12, dtype="fp32", ngram=3, states=2, bias=True, per_row=False),
        # the pick of the batch-512 greedy search
        dict(name="pick_batch", op="pick", B=512, V=9606, hist=20, dtype="bf16", ngram=2, states=4, bias=True, per_row=False),
        # a sampler's logits over a wide vocabulary, per-request penalties, long histories
        dict(name="control_wide", op="control", B=64, V=131071, hist=2000, dtype="bf16", ngram=4, states=9, bias=False,
             per_row=True),
        dict(name="control_fp32", op="control", B=128, V=50001, hist=300, dtype="fp32", ngram=0, states=0, bias=True,
             per_row=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["cache", "attend", "attend", "pick", "control"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    while True:
        if op == "cache":
            T = rng.choice([1, _log(rng, 1, 8192), _log(rng, 2, 300)])
            c = dict(op=op, B=_log(rng, 1, 512), H=rng.choice([1, 2, 4, 8, 12, 16]), dh=8 * rng.randint(2, 16), T=T,
                     cap=T + _log(rng, 1, 300), dtype=dtype, ragged=rng.random() < 0.6)
        elif op == "attend":
            Hkv, g = rng.choice([1, 2, 4, 8, 8]), rng.choice([1, 1, 1, 2, 3, 4, 8])
            L = _log(rng, 1, 32768)
            c = dict(op=op, B=_log(rng, 1, 512), H=Hkv * g, Hkv=Hkv, dh=8 * rng.randint(2, 16),
                     Tq=rng.choice([1, 1, 1, rng.randint(2, 9)]), L=L, low=rng.randint(0, L), dtype=dtype,
                     causal=rng.random() < 0.8)
        else:
            c = dict(op=op, B=_log(rng, 1, 512), V=_log(rng, 200, 131071), hist=rng.choice([0, _log(rng, 1, 4000)]),
                     dtype=dtype, ngram=rng.choice([0, 0, 1, 2, 3, 5]), states=rng.choice([0, 1, 3, 17]),
                     bias=rng.random() < 0.5, per_row=rng.random() < 0.5)
        w = work(c)
        if w["bytes"] <= 2.2e8 and w["flops"] <= 4e9 and c["B"] * c.get("V", 0) <= 9e6:
            return c


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "cache":
        n = case["B"] * case["H"] * case["T"]
        groups = (case["dh"] + 31) // 32
        # keys and values once in, once out; the 4-bit form written and read
        return {"bytes": n * 2 * (2 * case["dh"] * e + 2 * (case["dh"] // 2 + 4 * groups)), "flops": n * 2 * case["dh"] * 8}
    if case["op"] == "attend":
        tokens = case["B"] * (case["L"] + case["low"]) // 2
        groups = (case["dh"] + 31) // 32
        return {"bytes": tokens * case["Hkv"] * 2 * (case["dh"] // 2 + 4 * groups)
                + 2 * case["B"] * case["H"] * case["Tq"] * case["dh"] * e,
                "flops": 4 * tokens * case["H"] * case["Tq"] * case["dh"]}
    n = case["B"] * case["V"]
    out = n * e if case["op"] == "control" else 8 * case["B"]
    return {"bytes": n * e + out + 8 * case["B"] * case["hist"] + (4 * case["V"] if case["bias"] else 0)
            + case["states"] * ((case["V"] + 31) // 32) * 4, "flops": 4 * n}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed * 7919 + 17)


def _heads(g, B, T, H, dh, dtype, offset):
    """[B, H, T, dh] view of [B, T, H, dh] memory (a projection's output), some channels far from zero as keys have."""
    x = torch.randn(B, T, H, dh, device=DEV, generator=g)
    if offset:
        far = torch.randn(1, 1, H, dh, device=DEV, generator=g)
        x = x + 3.0 * far * (far.abs() > 1.3)
    return x.to(dtype).transpose(1, 2)


def _ints(g, lo, hi, shape):
    return torch.randint(lo, hi, shape, device=DEV, generator=g)


def prepare(case, seed):
    g, dtype = _gen(seed), DT[case["dtype"]]
    st = dict(case=case)
    if case["op"] == "cache":
        B, H, dh, T, cap = (case[n] for n in ("B", "H", "dh", "T", "cap"))
        st["k"], st["v"] = _heads(g, B, T, H, dh, dtype, True), _heads(g, B, T, H, dh, dtype, False)
        st["start"] = _ints(g, 0, cap - T + 1, (B,)).int()
        st["counts"] = _ints(g, (T + 1) // 2, T + 1, (B,)).int() if case["ragged"] else None
        st["cache"] = _new_cache(B, H, dh, cap)
    elif case["op"] == "attend":
        B, H, Hkv, dh, L, Tq = (case[n] for n in ("B", "H", "Hkv", "dh", "L", "Tq"))
        st["q"] = _heads(g, B, Tq, H, dh, dtype, False)
        lengths = _ints(g, case["low"], L + 1, (B,)).int()
        lengths[B // 2] = L
        st["lengths"] = lengths
        st["cache"] = _new_cache(B, Hkv, dh, L)
        k, v = _heads(g, B, L, Hkv, dh, dtype, True), _heads(g, B, L, Hkv, dh, dtype, False)
        _write(st["cache"], k, v, 0, None)
        if exact_inputs:
            st["k"], st["v"] = k, v
    else:
        B, V, T = case["B"], case["V"], case["hist"]
        st["logits"] = (3.0 * torch.randn(B, V, device=DEV, generator=g)).to(dtype)
        # token ids of the steps so far, time-major as a decode loop collects them; frequent words recur
        ids = (torch.rand(T, B, device=DEV, generator=g) ** 4 * min(V, 4 * T + 20)).long()
        st["history"] = ids.int().t() if T else None
        st["lengths"] = _ints(g, (T + 1) // 2, T + 1, (B,)).int() if T and case["per_row"] else None
        st["prompt"] = _ints(g, 0, T // 4 + 1, (B,)).int() if T and case["per_row"] else None
        if case["per_row"]:
            st["rep"] = 1.0 + 0.5 * torch.rand(B, device=DEV, generator=g)
            st["freq"] = 0.3 * torch.rand(B, device=DEV, generator=g)
            st["pres"] = 0.5 * torch.rand(B, device=DEV, generator=g)
        else:
            st["rep"], st["freq"], st["pres"] = 1.25, 0.125, 0.5
        st["bias"] = torch.randn(V, device=DEV, generator=g) if case["bias"] else None
        S, W = case["states"], (V + 31) // 32
        st["allowed"] = st["state"] = None
        if S:
            words = _ints(g, -2 ** 31, 2 ** 31, (3, S, W)).int()
            words = torch.where(_ints(g, 0, 2, (S, 1)) == 0, words[0] | words[1], words[0] & words[1] & words[2])
            if S > 2:
                words[S - 1] = 0                    # a state that allows nothing
            st["allowed"] = words
            st["state"] = _ints(g, -1, S, (B,)).int()       # -1: this sentence is not under a grammar
        if own:
            from mssrnet_style_transfer_amd.token_control import TokenControl
            st["control"] = TokenControl(repetition=st["rep"], frequency=st["freq"], presence=st["pres"],
                                         ngram=case["ngram"], bias=st["bias"], allowed=st["allowed"], state=st["state"])
    return st


exact_inputs = False        # exact() keeps the unquantised keys and values; a pass has no use for them


def _new_cache(B, H, dh, cap):
    if own:
        from mssrnet_style_transfer_amd.kv_cache import KVCache4
        return KVCache4(B, H, dh, cap, device=DEV)
    groups = (dh + 31) // 32
    return {n: (torch.zeros(B, H, cap, groups * 16, dtype=torch.uint8, device=DEV),
                torch.zeros(B, H, cap, groups, 2, dtype=torch.float16, device=DEV)) for n in "kv"}


def _write(cache, k, v, start, counts):
    if own:
        cache.write(k, v, start, counts)
    else:
        for n, x in (("k", k), ("v", v)):
            _plain_write(cache[n], x, start, counts)


def run(state):
    case = state["case"]
    if case["op"] == "cache":
        _write(state["cache"], state["k"], state["v"], state["start"], state["counts"])
        if own:
            return state["cache"].read(state["start"], case["T"], state["counts"], dtype=state["k"].dtype)
        return tuple(_plain_read(state["cache"][n], state["start"], case["T"], state["counts"], case["dh"]).to(state["k"].dtype)
                     for n in "kv")
    if case["op"] == "attend":
        if own:
            from mssrnet_style_transfer_amd import kv_cache
            return kv_cache.attention(state["q"], state["cache"], state["lengths"], causal=case["causal"])
        return _plain_attention(state["q"], state["cache"], state["lengths"], case)
    if own:
        from mssrnet_style_transfer_amd import token_control
        fn = token_control.pick_token if case["op"] == "pick" else token_control.control_logits
        return fn(state["logits"], state["control"], state["history"], state["lengths"], state["prompt"])
    x = _plain_control(state)
    if case["op"] == "control":
        return x.to(state["logits"].dtype)
    return torch.where(x.amax(1) == float("-inf"), -1, x.argmax(1))


# ------------------------------------------------------------------------------------------------ plain forms
def _groups(x):
    return [x[..., c:c + 32] for c in range(0, x.shape[-1], 32)]


def _plain_codes(x):
    """-> codes [..., dh padded to 32] in 0..15 and (scale, zero) [..., groups, 2] in fp16."""
    codes, meta = [], []
    for xg in _groups(x.float()):
        bad = ~torch.isfinite(xg).all(-1)
        xg = xg.clamp(-TOP, TOP)
        lo, hi = xg.amin(-1), xg.amax(-1)
        s = torch.where(bad, float("nan"), (hi - lo) * F15).half()
        z = torch.where(bad, float("nan"), lo).half()
        inv = torch.where(s > 0, torch.ones_like(lo) / s.float(), torch.zeros_like(lo))
        c = ((xg - z.float().unsqueeze(-1)) * inv.unsqueeze(-1)).round().clamp(0, 15).nan_to_num(0.0)
        codes.append(torch.nn.functional.pad(c.to(torch.uint8), (0, 32 - xg.shape[-1])))
        meta.append(torch.stack([s, z], -1))
    return torch.cat(codes, -1), torch.stack(meta, -2)


def _positions(start, T, cap, like):
    pos = torch.arange(T, device=DEV)
    return ((start.long().view(-1, 1) if torch.is_tensor(start) else torch.full((like.shape[0], 1), start, device=DEV)) + pos)


def _plain_write(held, x, start, counts):
    codes, meta = _plain_codes(x)
    packed = codes[..., 0::2] | (codes[..., 1::2] << 4)
    B, H, T = x.shape[:3]
    if not torch.is_tensor(start) and counts is None:
        held[0][:, :, start:start + T], held[1][:, :, start:start + T] = packed, meta
        return
    pos = _positions(start, T, held[0].shape[2], x)
    for dst, src in ((held[0], packed), (held[1].flatten(3), meta.flatten(3))):
        at = pos.view(B, 1, T, 1).expand(B, H, T, src.shape[-1])
        if counts is not None:
            keep = (torch.arange(T, device=DEV) < counts.view(-1, 1)).view(B, 1, T, 1)
            src = torch.where(keep, src, dst.gather(2, at))
        dst.scatter_(2, at, src)


def _plain_values(packed, meta, dh):
    c = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).float()
    m = meta.float()
    c = c.view(c.shape[:-1] + (-1, 32)) * m[..., :1] + m[..., 1:]
    return c.flatten(-2)[..., :dh]


def _plain_read(held, start, T, counts, dh):
    B, H = held[0].shape[:2]
    pos = _positions(start, T, held[0].shape[2], held[0])
    packed = held[0].gather(2, pos.view(B, 1, T, 1).expand(B, H, T, held[0].shape[3]))
    flat = held[1].flatten(3)
    meta = flat.gather(2, pos.view(B, 1, T, 1).expand(B, H, T, flat.shape[3])).view(B, H, T, -1, 2)
    out = _plain_values(packed, meta, dh)
    if counts is not None:
        out = torch.where((torch.arange(T, device=DEV) < counts.view(-1, 1)).view(B, 1, T, 1), out, 0.0)
    return out


def _visible(lengths, L, Tq, causal):
    """[B, Tq, L]: which cached tokens a query row sees."""
    lim = lengths.view(-1, 1).long()
    rows = torch.arange(Tq, device=DEV)
    lim = lim - Tq + 1 + rows if causal else lim.expand(-1, Tq)
    return torch.arange(L, device=DEV) < lim.unsqueeze(-1)


def _plain_attention(q, cache, lengths, case):
    B, H, Hkv, dh, Tq, L = (case[n] for n in ("B", "H", "Hkv", "dh", "Tq", "L"))
    k, v = (_plain_values(cache[n][0], cache[n][1], dh) for n in "kv")
    qs = q.float().reshape(B, Hkv, H // Hkv * Tq, dh) * (1.0 / math.sqrt(dh))
    see = _visible(lengths, L, Tq, case["causal"]).unsqueeze(1).unsqueeze(1)
    s = torch.matmul(qs, k.transpose(2, 3)).view(B, Hkv, H // Hkv, Tq, L)
    s = torch.where(see, s, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.where(see, torch.exp(s - torch.where(top == float("-inf"), 0.0, top)), 0.0)
    o = torch.matmul(p.view(B, Hkv, -1, L), v).view(B, H, Tq, dh)
    total = p.sum(-1).view(B, H, Tq, 1)
    return torch.where(total > 0, o / total, 0.0).to(q.dtype)


def _column(x, B):
    return x.view(B, 1) if torch.is_tensor(x) else torch.full((B, 1), x, device=DEV)


def _repeats(state, V):
    """-> (seen [B, V] bool, counts [B, V], banned [B, V] bool) of a history."""
    case, h = state["case"], state["history"]
    B = case["B"]
    zeros = torch.zeros(B, V, dtype=torch.int32, device=DEV)
    if h is None:
        return zeros.bool(), zeros, zeros.bool()
    h = h.long()
    T, at = h.shape[1], torch.arange(h.shape[1], device=DEV)
    n_h = state["lengths"].long().view(B, 1) if state["lengths"] is not None else torch.full((B, 1), T, device=DEV)
    prompt = state["prompt"].long().view(B, 1) if state["prompt"] is not None else torch.zeros(B, 1, dtype=torch.long, device=DEV)
    live = at < n_h
    seen = zeros.scatter_add(1, h, live.int()) > 0
    counts = zeros.scatter_add(1, h, (live & (at >= prompt)).int())
    n, banned = case["ngram"], zeros
    if n == 1:
        banned = seen.int()
    elif n > 1 and T >= n:
        tail = h.gather(1, (n_h - n + 1 + torch.arange(n - 1, device=DEV)).clamp(min=0))      # the last n - 1 tokens
        same = (h.unfold(1, n, 1)[..., :n - 1] == tail.unsqueeze(1)).all(-1)                  # [B, T - n + 1]
        same &= at[n - 1:] < n_h
        banned = zeros.scatter_add(1, h[:, n - 1:], same.int())
    return seen, counts, banned > 0


def _plain_control(state):
    case = state["case"]
    B, V = case["B"], case["V"]
    x = state["logits"].float()
    seen, counts, banned = _repeats(state, V)
    rep, freq, pres = (_column(state[n], B) for n in ("rep", "freq", "pres"))
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - (freq * counts + pres * (counts > 0))
    if state["bias"] is not None:
        x = x + state["bias"]
    if state["allowed"] is not None:
        bits = (state["allowed"].unsqueeze(-1) >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
        bits = bits.flatten(1)[:, :V].bool()
        banned = banned | ((state["state"] >= 0).view(B, 1) & ~bits[state["state"].long().clamp(min=0)])
    return x.masked_fill(banned, float("-inf"))


# ------------------------------------------------------------------------------------------------ in 64 bits
def _to(x, dtype):
    """A 64-bit value rounded as the definition rounds it there."""
    return x.to(dtype).double()


def _exact_values(x):
    """What the 4-bit form of x [..., dh] stands for: scale and zero are fp16 numbers by definition, and the quotient
    whose nearest integer is the code is an fp32 number (difference, reciprocal and product, each rounded)."""
    out = []
    for c in range(0, x.shape[-1], 32):
        v = x[..., c:c + 32].double()
        v = v.clamp(-TOP, TOP)
        low, span = v.min(-1, keepdim=True).values, None
        span = _to(v.max(-1, keepdim=True).values - low, torch.float32)
        s = _to(_to(span * F15, torch.float32), torch.float16)
        z = _to(low, torch.float16)
        r = _to(1.0 / s.masked_fill(s == 0, 1.0), torch.float32).masked_fill(s == 0, 0.0)
        n = torch.round(_to(_to(v - z, torch.float32) * r, torch.float32))
        out.append(z + s * n.clamp(0, 15))
    return torch.cat(out, -1)


def exact(case, seed):
    global exact_inputs
    exact_inputs = True
    try:
        st = prepare(case, seed)
    finally:
        exact_inputs = False
    if case["op"] == "cache":
        out = []
        for x in (st["k"], st["v"]):
            y = _exact_values(x)
            if st["counts"] is not None:
                for b, n in enumerate(st["counts"].tolist()):
                    y[b, :, n:] = 0
            out.append(y)
        return tuple(out)
    if case["op"] == "attend":
        H, Hkv, Tq, dh = case["H"], case["Hkv"], case["Tq"], case["dh"]
        out = torch.zeros(case["B"], H, Tq, dh, dtype=torch.float64, device=DEV)
        for b, n in enumerate(st["lengths"].tolist()):
            for hk in range(Hkv):
                k, v = _exact_values(st["k"][b, hk, :n]), _exact_values(st["v"][b, hk, :n])
                heads = slice(hk * (H // Hkv), (hk + 1) * (H // Hkv))
                for i in range(Tq):
                    m = n - Tq + 1 + i if case["causal"] else n
                    if m > 0:
                        w = torch.softmax(st["q"][b, heads, i].double() @ k[:m].t() / math.sqrt(dh), -1)
                        out[b, heads, i] = w @ v[:m]
        return out
    return _exact_control(case, st)


def _exact_control(case, st):
    """Row by row in 64 bits.  A pick is the largest of fp32 numbers: there each of the definition's steps is rounded."""
    B, V = case["B"], case["V"]
    step = (lambda t: _to(t, torch.float32)) if case["op"] == "pick" else (lambda t: t)
    x = st["logits"].double()
    rows = st["history"].tolist() if st["history"] is not None else [[]] * B
    per_row = lambda t: t.double().tolist() if torch.is_tensor(t) else [float(torch.tensor(t))] * B  # noqa: E731
    rep, freq, pres = per_row(st["rep"]), per_row(st["freq"]), per_row(st["pres"])
    lens = st["lengths"].tolist() if st["lengths"] is not None else [case["hist"]] * B
    prompt = st["prompt"].tolist() if st["prompt"] is not None else [0] * B
    state = st["state"].tolist() if st["state"] is not None else None
    n = case["ngram"]
    for b in range(B):
        h = rows[b][:lens[b]]
        if h:
            ids = torch.tensor(sorted(set(h)), device=DEV)
            y = x[b, ids]
            x[b, ids] = torch.where(y > 0, step(y / rep[b]), step(y * rep[b]))
            tail = h[prompt[b]:]
            if tail:
                ids, cnt = torch.unique(torch.tensor(tail, device=DEV), return_counts=True)
                x[b, ids] = step(x[b, ids] - step(step(freq[b] * cnt.double()) + pres[b]))
        if st["bias"] is not None:
            x[b] = step(x[b] + st["bias"].double())
        if n and len(h) >= n:
            end = h[len(h) - n + 1:]
            for i in range(len(h) - n + 1):
                if h[i:i + n - 1] == end:
                    x[b, h[i + n - 1]] = float("-inf")
        if state is not None and state[b] >= 0:
            at = torch.arange(V, device=DEV)
            word = st["allowed"][state[b]][at // 32].long()
            x[b, ((word >> (at % 32)) & 1) == 0] = float("-inf")
    if case["op"] == "control":
        return x
    top = x.max(1, keepdim=True).values
    first = torch.where(x == top, torch.arange(V, device=DEV), V).min(1).values
    return torch.where(top.view(-1) == float("-inf"), torch.full_like(first, -1), first)
