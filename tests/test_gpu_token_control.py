"""Control of the next token's logits (mssrnet_style_transfer_amd/token_control.py) against the definition, row by row in
64 bits and written here from its statement, shared with nothing else."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tc():
    from mssrnet_style_transfer_amd import token_control
    with torch.no_grad():
        yield token_control


def make(B, V, T, dtype, seed, states=0, per_row=True, bias=None, ngram=0, wide=torch.int64, spread=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.rand(*s, device="cuda", generator=g)                                    # noqa: E731
    c = dict(logits=(4 * torch.randn(B, V, device="cuda", generator=g)).to(dtype), ngram=ngram)
    c["history"] = (rnd(B, T) * (spread or V)).to(wide) if T else None
    c["lengths"] = (rnd(B) * (T + 1)).to(wide) if T and per_row else None
    c["prompt"] = (rnd(B) * (T // 2 + 1)).to(wide) if T and per_row else None
    c["rep"], c["freq"], c["pres"] = (1 + rnd(B), rnd(B), rnd(B) - 0.3) if per_row else (1.3, 0.25, -0.5)
    c["bias"] = None if bias is None else torch.randn(*((V,) if bias == 1 else (B, V)), device="cuda", generator=g)
    c["bits"] = rnd(states, V) < rnd(states, 1) if states else None
    if states > 1:
        c["bits"][-1] = False
    c["state"] = ((rnd(B) * (states + 2)).to(wide) - 1) if states else None      # from -1 to one past the table
    return c


def rules(tc, c):
    return tc.TokenControl(c["rep"], c["freq"], c["pres"], c["ngram"], c["bias"],
                           None if c["bits"] is None else tc.pack_allowed(c["bits"]), c["state"])


def expect(c, rounding):
    """The controlled logits [B, V] in 64 bits; ``rounding``: every step is an fp32 number, as the pick compares them."""
    step = (lambda t: t.float().double()) if rounding else (lambda t: t)
    x = c["logits"].double().cpu()
    B, V = x.shape
    num = lambda t, b: float(t[b]) if torch.is_tensor(t) else float(torch.tensor(t, dtype=torch.float32))   # noqa: E731
    for b in range(B):
        h = [] if c["history"] is None else c["history"][b].tolist()
        n = len(h) if c["lengths"] is None else max(0, min(len(h), int(c["lengths"][b])))
        h = h[:n]
        first = 0 if c["prompt"] is None else int(c["prompt"][b])
        for v in sorted(set(t for t in h if 0 <= t < V)):
            y = x[b, v]
            y = step(y / num(c["rep"], b)) if y > 0 else step(y * num(c["rep"], b))
            k = sum(1 for i, t in enumerate(h) if t == v and i >= first)
            if k:
                y = step(y - step(step(torch.tensor(num(c["freq"], b) * k, dtype=torch.float64)) + num(c["pres"], b)))
            x[b, v] = y
        if c["bias"] is not None:
            x[b] = step(x[b] + (c["bias"] if c["bias"].dim() == 1 else c["bias"][b]).double().cpu())
        m = c["ngram"]
        if m:
            for i in range(m - 1, n):
                if h[i - m + 1:i] == h[n - m + 1:] if m > 1 else True:
                    if 0 <= h[i] < V:
                        x[b, h[i]] = float("-inf")
        if c["bits"] is not None:
            s = int(c["state"][b])
            if s >= c["bits"].shape[0]:
                x[b] = float("-inf")
            elif s >= 0:
                x[b][~c["bits"][s].cpu()] = float("-inf")
    return x


def same_logits(got, want):
    """Four fp32 roundings at most on the way (quotient or product, penalty, difference, sum), the penalty's own ones
    counted with the penalty's size (below 40 here): 4 * 2^-24 of the largest number met, then the type's half step."""
    half = torch.finfo(got.dtype).eps / 2
    got = got.double().cpu()
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and not torch.isnan(got).any()
    ok = ~torch.isinf(want)
    err = (got - want)[ok].abs()
    assert (err <= half * want[ok].abs() + 6 * 2.0 ** -24 * (want[ok].abs() + 80)).all(), float(err.max())


def picks(want, empty=-1):
    top = want.max(1, keepdim=True).values
    return [empty if top[b] == float("-inf") else int((want[b] == top[b]).nonzero()[0]) for b in range(want.shape[0])]


CASES = [  # B, V, T, states, per_row, bias, ngram, spread
    (1, 1, 0, 0, False, None, 0, None),
    (1, 33, 3, 0, True, 1, 1, None),
    (3, 9606, 20, 3, False, 1, 2, 12),
    (5, 200, 40, 2, True, 2, 3, 4),
    (2, 2048, 1, 0, True, None, 1, None),
    (2, 2049, 700, 5, True, 1, 4, 3),
    (70, 517, 9, 1, True, None, 5, 2),
    (1, 70001, 300, 4, True, 2, 2, 40),
    (4, 131071, 1500, 2, False, None, 3, None),
    (600, 4100, 30, 7, True, 1, 2, 20),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,V,T,states,per_row,bias,ngram,spread", CASES)
def test_logits_and_picks(tc, B, V, T, states, per_row, bias, ngram, spread, dtype):
    c = make(B, V, T, dtype, 5, states, per_row, bias, ngram, spread=spread)
    args = (rules(tc, c), c["history"], c["lengths"], c["prompt"])
    new = tc.control_logits(c["logits"], *args)
    assert new.dtype == dtype
    same_logits(new, expect(c, False))
    want = picks(expect(c, True))
    got = tc.pick_token(c["logits"], *args)
    assert got.dtype == torch.int64 and got.tolist() == want
    ids = torch.full((B,), 7, dtype=torch.int32, device="cuda")
    assert tc.pick_token(c["logits"], *args, empty=3, out=ids) is ids
    assert ids.tolist() == [3 if w == -1 else w for w in want]
    # in place
    x = c["logits"].clone()
    assert tc.control_logits(x, *args, out=x) is x
    assert torch.equal(x, new)


@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
def test_strides_types_and_padded_rows(tc, wide):
    B, V, T = 6, 1001, 25
    c = make(B, V, T, torch.bfloat16, 6, 2, True, 2, 2, wide=wide, spread=10)
    plain = tc.control_logits(c["logits"], rules(tc, c), c["history"], c["lengths"], c["prompt"])
    rows = torch.zeros(B, V + 39, dtype=torch.bfloat16, device="cuda")          # odd row starts, a padded slab
    rows[:, 1:V + 1] = c["logits"]
    major = torch.full((T + 5, B), -7, dtype=wide, device="cuda")
    major[2:T + 2] = c["history"].t()                                           # time-major, as a decode loop keeps it
    bias = torch.zeros(B, V + 3, device="cuda")
    bias[:, :V] = c["bias"]
    c["bias"] = bias[:, :V]
    view = rows[:, 1:V + 1]
    got = tc.control_logits(view, rules(tc, c), major[2:T + 2].t(), c["lengths"], c["prompt"])
    assert torch.equal(got, plain)
    assert torch.equal(tc.pick_token(view, rules(tc, c), major[2:T + 2].t(), c["lengths"], c["prompt"]),
                       tc.pick_token(plain))
    tc.control_logits(view, rules(tc, c), major[2:T + 2].t(), c["lengths"], c["prompt"], out=view)
    assert torch.equal(rows[:, 1:V + 1], plain) and (rows[:, 0] == 0).all() and (rows[:, V + 1:] == 0).all()
    columns = c["logits"].t().contiguous().t()                                  # words far apart: copied first
    assert torch.equal(tc.control_logits(columns, rules(tc, c), c["history"], c["lengths"], c["prompt"]), plain)


def test_history_entries_outside_the_vocabulary_and_odd_lengths(tc):
    V = 50
    c = make(4, V, 6, torch.float32, 8)
    c["history"] = torch.tensor([[-1, 3, 50, 3, 1 << 40, -(1 << 40)], [5, 5, 5, 5, 5, 5], [1, 2, 1, 2, 1, 2], [9] * 6],
                                device="cuda")
    c["lengths"] = torch.tensor([6, 0, -4, 99], device="cuda")
    c["prompt"] = torch.tensor([2, 0, 0, 77], device="cuda")
    for n in (0, 1, 2, 6, 7):
        c["ngram"] = n
        same_logits(tc.control_logits(c["logits"], rules(tc, c), c["history"], c["lengths"], c["prompt"]), expect(c, False))


def test_counts_of_a_long_history(tc):
    """One word 100 000 times, and a penalty that counts them exactly."""
    x = torch.zeros(2, 40, device="cuda")
    h = torch.full((2, 100000), 7, device="cuda")
    y = tc.control_logits(x, tc.TokenControl(frequency=1.0), h, torch.tensor([100000, 99999], device="cuda"))
    assert y[:, 7].tolist() == [-100000.0, -99999.0] and (y[:, :7] == 0).all() and (y[:, 8:] == 0).all()


@pytest.mark.parametrize("V", [40, 9606, 40000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ties_infinities_and_nan(tc, V, dtype):
    x = torch.full((8, V), -1.0, device="cuda", dtype=dtype)
    x[0] = 0.0
    x[0, 5], x[0, 9] = -0.0, 0.0                        # -0 equals +0: the lowest index
    x[1, V - 1], x[1, 17] = 2.0, 2.0
    x[2] = float("-inf")
    x[3, 30], x[3, 11] = float("inf"), float("inf")
    x[4, 33], x[4, 21], x[4, 2] = float("nan"), float("nan"), float("inf")
    x[5] = float("nan")
    x[6] = torch.finfo(dtype).min
    x[7, V - 1] = 3.0
    want = [0, 17, -1, 11, 21, 0, 0, V - 1]
    assert tc.pick_token(x).tolist() == want
    # a mask takes NaN and infinities out
    bits = torch.ones(8, V, dtype=torch.bool, device="cuda")
    bits[3, [30, 11]] = bits[4, [33, 21, 2]] = False
    bits[5, 1:] = False
    bits[5, 0] = False
    c = tc.TokenControl(allowed=tc.pack_allowed(bits))
    assert tc.pick_token(x, c).tolist() == [0, 17, -1, 0, 0, -1, 0, V - 1]
    y = tc.control_logits(x, c)
    assert torch.equal(y[~bits], torch.full_like(y[~bits], float("-inf")))
    assert torch.equal(y[bits].nan_to_num(9.0), x[bits].nan_to_num(9.0))


def test_one_mask_row_for_all_and_one_each(tc):
    B, V = 3, 77
    x = torch.randn(B, V, device="cuda")
    bits = torch.rand(B, V, device="cuda") < 0.5
    each = tc.control_logits(x, tc.TokenControl(allowed=tc.pack_allowed(bits)))
    assert torch.equal(each == float("-inf"), ~bits)
    one = tc.control_logits(x, tc.TokenControl(allowed=tc.pack_allowed(bits[:1])))
    assert torch.equal(one == float("-inf"), ~bits[:1].expand(B, V))
    # the bits past the vocabulary's end say nothing
    words = tc.pack_allowed(bits)
    words[:, -1] |= -1 << (V % 32)
    assert torch.equal(tc.control_logits(x, tc.TokenControl(allowed=words)), each)


def test_rules_of_some_rows(tc):
    c = make(6, 300, 12, torch.float32, 9, 3, True, 2, 2, spread=8)
    r = rules(tc, c)
    keep = torch.tensor([4, 0, 3], device="cuda")
    part = tc.control_logits(c["logits"][keep], r.rows(keep, 6), c["history"][keep], c["lengths"][keep], c["prompt"][keep])
    full = tc.control_logits(c["logits"], r, c["history"], c["lengths"], c["prompt"])
    assert torch.equal(part, full[keep])
    bits = torch.rand(6, 300, device="cuda") < 0.5
    each = tc.TokenControl(allowed=tc.pack_allowed(bits))
    assert torch.equal(tc.control_logits(c["logits"][keep], each.rows(keep, 6)), tc.control_logits(c["logits"], each)[keep])
    one = tc.TokenControl(allowed=tc.pack_allowed(bits[:1]))
    assert torch.equal(tc.control_logits(c["logits"][keep], one.rows(keep, 6)), tc.control_logits(c["logits"], one)[keep])


def test_other_stream_and_captured_replays(tc):
    B, V, T = 3, 30000, 16                              # several chunks a row: scratch and a second launch
    c = make(B, V, T, torch.bfloat16, 10, 3, True, 1, 2, spread=6)
    r = rules(tc, c)
    args = (r, c["history"], c["lengths"], c["prompt"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ids = tc.pick_token(c["logits"], *args)
    torch.cuda.current_stream().wait_stream(side)
    assert ids.tolist() == picks(expect(c, True))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, new = tc.pick_token(c["logits"], *args), tc.control_logits(c["logits"], *args)
    for i in range(4):
        c["logits"].normal_()
        c["history"].random_(0, 6)
        g.replay()
        assert out.tolist() == picks(expect(c, True)), i
        assert torch.equal(new, tc.control_logits(c["logits"], *args))


def test_refusals(tc):
    x = torch.zeros(2, 50, device="cuda")
    h = torch.zeros(2, 4, dtype=torch.int64, device="cuda")
    n = torch.zeros(2, dtype=torch.int64, device="cuda")
    words = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    K = tc.TokenControl
    for logits, kw in ((x[0], {}), (x[:, :0], {}), (x, dict(history=h[:1])), (x, dict(history=h.float())),
                       (x, dict(history=h.cpu())), (x, dict(history=h, lengths=n[:1])), (x, dict(lengths=n)),
                       (x, dict(history=h, prompt_lengths=n.float())), (x, dict(control=K(ngram=-1))),
                       (x, dict(control=K(ngram=65))), (x, dict(control=K(repetition=n.float()[:1]))),
                       (x, dict(control=K(frequency=n))), (x, dict(control=K(bias=x[:, :49]))),
                       (x, dict(control=K(bias=x.bfloat16()))), (x, dict(control=K(allowed=words))),
                       (x, dict(control=K(allowed=words[:, :1], state=n))), (x, dict(control=K(allowed=words.long(), state=n))),
                       (x, dict(control=K(state=n))), (x, dict(control=K(allowed=words, state=n[:1])))):
        for fn in (tc.control_logits, tc.pick_token):
            with pytest.raises(ValueError):
                fn(logits, **kw)
    for fn in (tc.control_logits, tc.pick_token):
        with pytest.raises(TypeError):
            fn(x.half())
        with pytest.raises(RuntimeError, match="no CPU path"):
            fn(x.cpu())
        with torch.enable_grad(), pytest.raises(RuntimeError, match="no graph"):
            fn(x.clone().requires_grad_())
        assert fn(x[:0]).shape[0] == 0
    for out in (x[:1], x.bfloat16(), x.t().contiguous().t()):
        with pytest.raises(ValueError):
            tc.control_logits(x, out=out)
    for out in (n[:1], n.float(), torch.zeros(4, dtype=torch.int64, device="cuda")[::2]):
        with pytest.raises(ValueError):
            tc.pick_token(x, out=out)
    with pytest.raises(ValueError):
        tc.pack_allowed(words)


def test_infinite_rates_leave_what_they_do_not_count(tc):
    inf = float("inf")
    x = torch.zeros(2, 40, device="cuda")
    h = torch.tensor([[3, 5, 5, 7], [1, 1, 2, 3]], device="cuda")
    first = torch.tensor([1, 2], device="cuda")
    for c in (tc.TokenControl(frequency=inf), tc.TokenControl(presence=inf)):
        got = tc.control_logits(x, c, h, prompt_lengths=first)
        want = x.clone()
        want[0, [5, 7]] = -inf                          # word 3 stands in the prompt only
        want[1, [2, 3]] = -inf
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_where_the_new_logits_may_lie(tc, dtype):
    g = torch.Generator(device="cuda").manual_seed(21)
    both = torch.randn(5, 2 * 130 + 7, device="cuda", generator=g).to(dtype)
    x, beside = both[:, :130], both[:, 137:]
    c = tc.TokenControl(bias=torch.randn(130, device="cuda", generator=g))
    want = tc.control_logits(x, c)
    assert torch.equal(tc.control_logits(x, c, out=beside), want) and torch.equal(beside, want)
    before = both.clone()
    with pytest.raises(RuntimeError, match="overlap"):
        tc.control_logits(x, c, out=both[:, 1:131])
    with pytest.raises(RuntimeError, match="overlap"):
        tc.control_logits(x[:4], c, out=both[1:, 3:133])
    assert torch.equal(both, before)
    assert torch.equal(tc.control_logits(x[:4], c, out=both[1:, 137:]), want[:4])       # other columns, a row further on
    assert torch.equal(tc.control_logits(x, c, out=x), want) and torch.equal(x, want)


def test_a_batch_without_rows(tc):
    x = torch.zeros(0, 40, device="cuda")
    each = tc.TokenControl(allowed=torch.zeros(0, 2, dtype=torch.int32, device="cuda"))
    assert tc.control_logits(x, each).shape == (0, 40) and tc.pick_token(x, each).shape == (0,)


def test_two_picks_at_once(tc):
    g = torch.Generator(device="cuda").manual_seed(8)
    x = [torch.randn(3, 50000, device="cuda", generator=g) for _ in range(2)]           # several chunks a row: scratch
    h = torch.randint(0, 50000, (3, 40), device="cuda", generator=g)
    c = tc.TokenControl(repetition=1.3, ngram=1)
    want = [tc.pick_token(t, c, h) for t in x]
    streams = [torch.cuda.Stream() for _ in x]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(tc.pick_token(x[i], c, h))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(t, want[i]) for t in got[i])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,V,T,spread", [(260, 131071, 40, 50),        # the largest chunk of a row that a block takes, 16-bit marks
                                          (130, 20000, 17000, 3)])      # and 32-bit ones
def test_the_largest_chunks(tc, dtype, B, V, T, spread):
    c = make(B, V, T, dtype, 31, spread=spread)
    c["history"][:, ::9] = V - 1 - c["history"][:, ::9]                 # both ends of the row
    args = (rules(tc, c), c["history"], c["lengths"], c["prompt"])
    same_logits_of(tc.control_logits(c["logits"], *args), expect(c, False), T)
    assert tc.pick_token(c["logits"], *args).tolist() == picks(expect(c, True))


def same_logits_of(got, want, T):
    """same_logits for penalties up to 2 T + 1: their roundings counted with that size."""
    half = torch.finfo(got.dtype).eps / 2
    got = got.double().cpu()
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and not torch.isnan(got).any()
    assert ((got - want).abs() <= half * want.abs() + 6 * 2.0 ** -24 * (want.abs() + 4 * T + 80)).all()
