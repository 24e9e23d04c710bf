"""The 4-bit key/value cache and attention over it (mssrnet_style_transfer_amd/kv_cache.py) against the definition in 64
bits, written here from the formulas of csrc/kv4.hpp and shared with nothing else."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv():
    from mssrnet_style_transfer_amd import kv_cache
    with torch.no_grad():
        yield kv_cache


def f(x, dtype):
    """Rounded to dtype, held in 64 bits."""
    return x.to(dtype).double()


def values(x):
    """What the 4-bit form of x [..., dh] stands for, in 64 bits; the definition's own roundings are kept."""
    out = []
    third = f(torch.tensor(1.0 / 15.0, dtype=torch.float64), torch.float32)
    for part in x.double().split(32, -1):
        bad = ~torch.isfinite(part).all(-1, keepdim=True)
        y = part.nan_to_num(0.0, 65504.0, -65504.0).clamp(-65504, 65504)
        lo, hi = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
        s = f(f(f(hi - lo, torch.float32) * third, torch.float32), torch.float16)
        z = f(lo, torch.float16)
        inv = torch.where(s > 0, f(1.0 / s.clamp(min=1e-30), torch.float32), 0.0)
        code = torch.round(f(f(y - z, torch.float32) * inv, torch.float32)).clamp(0, 15)
        out.append(torch.where(bad, float("nan"), z + s * code))
    return torch.cat(out, -1)


def attend(q, k, v, lengths, scale, causal):
    """-> (context, bound): the formula in 64 bits over the values k, v stand for, and how far the kernels' arithmetic on
    the codes may be from it before the result is rounded.  Per row, with u = 2^-24 the fp32 half step:
      a score: q is one fp16 part (bf16: exact but for 2^-39 of the row's largest element) or two (fp32: 2^-22 = 4 u each);
        its products add up in fp32 (at most 34 roundings a group, a few for scales and zeros, one of scale * log2 e):
        |ds| <= 48 u sum_c |q_c| (|z| + 15 s + |k|)  (bounded by 3 max|k| for the bracket's terms), exp2 adds 2 u;
      so p is off by a factor 1 +- (|ds| + 4 u), and the quotient by twice that of max |v|;
      p s is one fp16 part (bf16: 2^-11) or two (fp32: 2^-22), and where it is below 2^-21 of the largest scale at most
        2^-32 of that scale: m tokens * 15 codes of it, 15 * scale <= 2 max |v|;
      sums over m tokens: m / 8 + 40 roundings (a matrix product adds 32 terms at a time, then blocks, waves and splits
        are joined)."""
    B, H, T, dh = q.shape
    G = H // k.shape[1]
    bf16 = q.dtype == torch.bfloat16
    out = torch.zeros(B, H, T, dh, dtype=torch.float64, device=q.device)
    bound = torch.zeros(B, H, T, 1, dtype=torch.float64, device=q.device)
    u = 2.0 ** -24
    for b in range(B):
        n = int(lengths[b])
        for h in range(H):
            kk, vv = k[b, h // G], v[b, h // G]
            for i in range(T):
                m = max(0, n - T + 1 + i) if causal else n
                if m == 0:
                    continue
                qq = q[b, h, i].double()
                out[b, h, i] = torch.softmax(scale * (kk[:m] @ qq), 0) @ vv[:m]
                ds = 48 * u * abs(scale) * float(qq.abs().sum()) * 3 * float(kk[:m].abs().max())
                rel = 2 * (ds + 4 * u) + (2.0 ** -11 if bf16 else 4 * u) + m * 2.0 ** -32 + (m / 8 + 40) * u
                # zeros and codes are summed apart: up to |z| + 15 s <= 3 max |v| a term
                bound[b, h, i] = rel * 3 * float(vv[:m].abs().max())
    return out, bound


def close(got, want, bound, name=""):
    half = torch.finfo(torch.bfloat16).eps / 2 if got.dtype == torch.bfloat16 else 0     # one rounding of the result
    got = got.double()
    err = (got - want).abs()
    tol = bound + half * want.abs()
    assert torch.isfinite(got).all(), name
    assert (err <= tol).all(), "%s: %.3g beyond a bound of %.3g" % (name, float((err - tol).max()), float(tol.max()))


def heads(B, H, T, dh, dtype, seed, far=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(B, T, H, dh, device="cuda", generator=g)
    if far:
        x = x + far * torch.randn(1, 1, H, dh, device="cuda", generator=g)
    return x.to(dtype).transpose(1, 2)


def rounded(x, dtype):
    return x.to(dtype) if dtype == torch.float32 else x.float().to(dtype)       # z + s * code is first an fp32 number


# ------------------------------------------------------------------------------------------------ write, read back
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dh", [8, 16, 32, 40, 64, 96, 120, 128])
@pytest.mark.parametrize("T,start", [(1, 0), (1, 63), (3, 62), (15, 57), (16, 0), (17, 50), (64, 64), (130, 5), (200, 0)])
def test_write_then_read(kv, dtype, dh, T, start):
    B, H, cap = 3, 2, 210
    c = kv.KVCache4(B, H, dh, cap)
    c.data.fill_(0xA5)                                  # whatever the memory held before
    before = c.data.clone()
    k, v = heads(B, H, T, dh, dtype, 1, 2.0), heads(B, H, T, dh, dtype, 2)
    c.write(k, v, start)
    for out, x in zip(c.read(start, T, dtype=torch.float32), (k, v)):
        assert torch.equal(out, values(x).float())
    for out, x in zip(c.read(start, T, dtype=torch.bfloat16), (k, v)):
        assert torch.equal(out, values(x).float().bfloat16())
    # the tokens around it still hold what they held
    d = kv.KVCache4(B, H, dh, cap)
    d.data.copy_(before)
    for lo, n in ((0, start), (start + T, cap - start - T)):
        for x, y in zip(c.read(lo, n), d.read(lo, n)):
            assert torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0))


@pytest.mark.parametrize("T", [1, 5, 40])
@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
def test_ragged_starts_and_counts(kv, T, wide):
    B, H, dh, cap = 7, 3, 48, 100
    c = kv.KVCache4(B, H, dh, cap)
    k, v = heads(B, H, T, dh, torch.float32, 3), heads(B, H, T, dh, torch.float32, 4)
    base = heads(B, H, cap, dh, torch.float32, 5)
    c.write(base, base, 0)
    start = torch.tensor([0, 99, 60, -2, 100, 1 << 30, 64 - T], device="cuda", dtype=wide)
    counts = torch.tensor([T, T, 0, T, T, T, max(T - 1, 0)], device="cuda", dtype=wide)
    c.write(k, v, start, counts)
    want = [values(base), values(base)]
    for b in range(B):
        for t in range(min(T, int(counts[b]))):
            p = int(start[b]) + t
            if 0 <= p < cap:
                want[0][b, :, p], want[1][b, :, p] = values(k[b, :, t]), values(v[b, :, t])
    for got, w in zip(c.read(0, cap), want):
        assert torch.equal(got, w.float())
    for got, w in zip(c.read(start, T, counts), want):
        for b in range(B):
            for t in range(T):
                p = int(start[b]) + t
                inside = t < int(counts[b]) and 0 <= p < cap
                assert torch.equal(got[b, :, t], w[b, :, p].float() if inside else torch.zeros_like(got[b, :, t]))


def test_strides_and_alignment(kv):
    B, H, T, dh = 2, 3, 21, 40
    c, d = kv.KVCache4(B, H, dh, 64), kv.KVCache4(B, H, dh, 64)
    for dtype in (torch.float32, torch.bfloat16):
        packed = torch.randn(T, B, H * dh * 3 + 1, device="cuda").to(dtype)[..., 1:]         # odd base, odd row stride
        k = packed[..., :H * dh].view(T, B, H, dh).permute(1, 2, 0, 3)
        v = packed[..., H * dh:2 * H * dh].unflatten(-1, (H, dh)).permute(1, 2, 0, 3)
        c.write(k, v, 3)
        d.write(k.contiguous(), v.contiguous(), 3)
        assert torch.equal(c.data, d.data)
        feat = torch.randn(B, H, dh, T, device="cuda").to(dtype).transpose(2, 3)             # features not contiguous
        c.write(feat, feat, 3)
        d.write(feat.contiguous(), feat.contiguous(), 3)
        assert torch.equal(c.data, d.data)
        q = packed[:5, :, 2 * H * dh:].view(5, B, H, dh).permute(1, 2, 0, 3)
        assert torch.equal(kv.attention(q, c, 24), kv.attention(q.contiguous(), c, 24))


def test_extreme_values(kv):
    dh, T = 64, 20
    k = torch.randn(1, 1, T, dh, device="cuda")
    k[0, 0, 0] = 0.0                                    # no range: every code 0
    k[0, 0, 1] = 3.25
    k[0, 0, 2, :32] = 1e-9                              # a range below fp16's smallest step
    k[0, 0, 3, 5], k[0, 0, 3, 6] = 3e38, -3e38          # clamped
    k[0, 0, 4, 3] = float("nan")
    k[0, 0, 5, 40] = float("inf")
    k[0, 0, 6, 63] = float("-inf")
    k[0, 0, 7] *= 1e4
    k[0, 0, 8] *= 1e-4
    for n in (T, 9):                                    # both kernels
        c = kv.KVCache4(1, 1, dh, 32)
        c.write(k[:, :, :n], k[:, :, :n], 1)
        for got in c.read(1, n):
            assert torch.equal(got.nan_to_num(1e30), values(k[:, :, :n]).float().nan_to_num(1e30))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_every_rounding_of_many_groups(kv, dtype):
    """Half a million groups: a scale rounded once instead of twice shows in one of some 8000."""
    k, v = heads(8, 8, 2048, 64, dtype, 17, 2.0), heads(8, 8, 2048, 64, dtype, 18)
    c = kv.KVCache4(8, 8, 64, 2048)
    c.write(k, v)
    for got, x in zip(c.read(0, 2048), (k, v)):
        assert torch.equal(got, values(x).float())
    few = kv.KVCache4(8 * 2048, 8, 64, 1)                           # the same tokens, one a sentence
    one = lambda x: x.transpose(1, 2).reshape(8 * 2048, 1, 8, 64).transpose(1, 2)              # noqa: E731
    few.write(one(k), one(v))
    for got, x in zip(few.read(0, 1), (one(k), one(v))):
        assert torch.equal(got, values(x).float())


def test_rounding_is_within_half_a_step(kv):
    x = heads(2, 2, 70, 64, torch.float32, 9, 3.0)
    c = kv.KVCache4(2, 2, 64, 70)
    c.write(x, x, 0)
    got = c.read(0, 70)[0]
    for a, y in zip(x.split(32, -1), got.split(32, -1)):
        step = (a.amax(-1) - a.amin(-1)) / 15
        # half a step, and what the fp16 scale (15 codes of it) and zero add: 2^-11 relative each
        tol = 0.5 * step + 2.0 ** -11 * (15 * step + a.abs().amax(-1)) + 1e-6
        assert ((a - y).abs().amax(-1) <= tol).all()


# ------------------------------------------------------------------------------------------------ attention
SHAPES = [  # B, H, Hkv, dh, Tq, capacity, lengths
    (1, 1, 1, 64, 1, 1, [1]),
    (4, 8, 8, 64, 1, 200, [1, 64, 65, 200]),
    (3, 4, 4, 16, 1, 70, [0, 7, 70]),
    (2, 2, 2, 8, 1, 130, [129, 63]),
    (2, 3, 1, 40, 1, 300, [300, 11]),
    (2, 8, 2, 96, 5, 400, [400, 3]),
    (2, 4, 4, 128, 1, 900, [900, 513]),
    (1, 16, 2, 128, 3, 150, [150]),
    (2, 6, 2, 80, 9, 140, [140, 6]),
    (1, 2, 1, 32, 70, 200, [190]),
    (2, 5, 5, 120, 2, 64, [64, 1]),
    (1, 1, 1, 64, 1, 20000, [19990]),
    (1, 9, 3, 64, 1, 9000, [8999]),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("B,H,Hkv,dh,Tq,cap,lengths", SHAPES)
def test_attention_matches_the_formula(kv, B, H, Hkv, dh, Tq, cap, lengths, causal, dtype):
    c = kv.KVCache4(B, Hkv, dh, cap)
    c.data.fill_(0xFF)                                  # past the lengths: NaN scales, codes of 15
    n = torch.tensor(lengths, device="cuda", dtype=torch.int32)
    k, v = heads(B, Hkv, cap, dh, dtype, 11, 1.5), heads(B, Hkv, cap, dh, dtype, 12)
    c.write(k, v, 0, n)
    q = heads(B, H, Tq, dh, dtype, 13)
    want, bound = attend(q, values(k), values(v), n, 1.0 / math.sqrt(dh), causal)
    got = kv.attention(q, c, n, causal=causal)
    assert got.dtype == dtype and got.shape == q.shape
    close(got, want, bound, "attention")
    close(kv.attention(q, c, n.long(), causal=causal, longest=max(lengths)), want, bound, "longest given")
    if len(set(lengths)) == 1:
        close(kv.attention(q, c, lengths[0], causal=causal), want, bound, "length as a number")


@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
def test_attention_scales(kv, scale):
    B, H, dh, n = 2, 2, 64, 150
    k, v, q = (heads(B, H, t, dh, torch.float32, s) for t, s in ((n, 1), (n, 2), (1, 3)))
    c = kv.KVCache4(B, H, dh, n)
    c.write(k, v)
    want, bound = attend(q, values(k), values(v), [n, n], scale, False)
    close(kv.attention(q, c, n, scale=scale), want, bound, "scale %g" % scale)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_scores_far_apart(kv, dtype):
    """Scores that grow by hundreds along the sequence (the running maximum moves in every block) and values over many
    orders of magnitude."""
    B, H, dh, n = 1, 2, 64, 700
    k = heads(B, H, n, dh, dtype, 21) * torch.linspace(0.1, 30, n, device="cuda").view(1, 1, n, 1).to(dtype)
    v = heads(B, H, n, dh, dtype, 22) * torch.logspace(-4, 3, n, device="cuda").view(1, 1, n, 1).to(dtype)
    q = heads(B, H, 2, dh, dtype, 23)
    c = kv.KVCache4(B, H, dh, n)
    c.write(k, v)
    want, bound = attend(q, values(k), values(v), [n], 1.0, True)
    close(kv.attention(q, c, n, scale=1.0, causal=True), want, bound, "far apart")
    small = (heads(B, H, n, dh, dtype, 24) * 1e-5).to(dtype)         # scales are subnormal fp16 numbers
    c.write(k, small)
    want, bound = attend(q, values(k), values(small), [n], 0.01, False)
    close(kv.attention(q, c, n, scale=0.01), want, bound, "small values")


def test_what_is_masked_does_not_count(kv):
    """NaN and infinities in tokens that a row does not see; rows that see none."""
    B, H, dh, n = 3, 2, 64, 90
    k, v = heads(B, H, n, dh, torch.float32, 31), heads(B, H, n, dh, torch.float32, 32)
    q = heads(B, H, 4, dh, torch.float32, 33)
    lengths = torch.tensor([88, 2, 0], device="cuda")
    clean = kv.KVCache4(B, H, dh, n)
    clean.write(k, v)
    want = kv.attention(q, clean, lengths, causal=True)
    k[0, :, 88:], v[0, :, 88:] = float("nan"), float("inf")
    k[1, :, 2:], v[1, :, 2:] = float("inf"), float("nan")
    dirty = kv.KVCache4(B, H, dh, n)
    dirty.write(k, v)
    got = kv.attention(q, dirty, lengths, causal=True)
    assert torch.equal(got, want)
    assert (got[1, :, :2] == 0).all() and (got[2] == 0).all() and (got[1, :, 2:] != 0).any()
    # the last token is NaN: earlier rows do not see it, the last row is NaN where the formula makes it so
    k2, v2 = k.clone(), v.clone()
    v2[0, :, 87, :32] = float("nan")
    dirty.write(k2, v2)
    last = kv.attention(q, dirty, lengths, causal=True)
    assert torch.equal(last[0, :, :3], want[0, :, :3])
    assert torch.isnan(last[0, :, 3, :32]).all() and torch.equal(last[0, :, 3, 32:], want[0, :, 3, 32:])


def test_lengths_outside_the_cache_are_clamped(kv):
    B, H, dh, n = 3, 2, 64, 70
    k, v, q = heads(B, H, n, dh, torch.float32, 41), heads(B, H, n, dh, torch.float32, 42), heads(B, H, 1, dh, torch.float32, 43)
    c = kv.KVCache4(B, H, dh, n)
    c.write(k, v)
    far = torch.tensor([1 << 40, -5, 70], device="cuda")
    got = kv.attention(q, c, far)
    assert torch.equal(got, kv.attention(q, c, torch.tensor([70, 0, 70], device="cuda")))


def test_offsets_past_32_bits(kv):
    """The second sentence, and late tokens of the first, lie more than 4 GB into the cache."""
    dh, cap = 128, 27 << 20
    c = kv.KVCache4(2, 1, dh, cap)
    assert c.nbytes // 2 > 1 << 32
    k, v, q = heads(2, 1, 70, dh, torch.float32, 51), heads(2, 1, 70, dh, torch.float32, 52), heads(2, 1, 1, dh, torch.float32, 53)
    start = torch.tensor([cap - 70, 3], device="cuda")
    c.write(k, v, start)
    for got, x in zip(c.read(start, 70), (k, v)):
        assert torch.equal(got, values(x).float())
    d = kv.KVCache4(2, 1, dh, 128)
    d.write(k, v, torch.tensor([0, 3], device="cuda"))
    # sentence 0: 27 M tokens of zero score (keys 0) against 70 whose scores are made large: the 70 decide
    big = q * 40
    n = torch.tensor([cap, 73], device="cuda")
    got, near = kv.attention(big, c, n, scale=1.0), kv.attention(big, d, torch.tensor([70, 73], device="cuda"), scale=1.0)
    assert (got - near).abs().max() <= 1e-5 * near.abs().max()


def test_other_stream_and_captured_replays(kv):
    B, H, dh, cap = 4, 2, 64, 300
    step = torch.zeros(B, device="cuda", dtype=torch.int32)
    k, v, q = (heads(B, H, 1, dh, torch.bfloat16, s) for s in (61, 62, 63))
    c, ref = kv.KVCache4(B, H, dh, cap), kv.KVCache4(B, H, dh, cap)
    pre = heads(B, H, 200, dh, torch.bfloat16, 64)
    c.write(pre, pre, 0)
    ref.write(pre, pre, 0)
    step += 200
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.write(k, v, step)
        first = kv.attention(q, c, step + 1, causal=True)
    torch.cuda.current_stream().wait_stream(side)
    ref.write(k, v, 200)
    assert torch.equal(first, kv.attention(q, ref, 201, causal=True))
    g = torch.cuda.CUDAGraph()
    n = step + 1
    with torch.cuda.graph(g):
        c.write(k, v, step)
        out = kv.attention(q, c, n, causal=True)
    for t in range(201, 206):
        k.normal_()
        v.normal_()
        q.normal_()
        step.fill_(t)
        n.fill_(t + 1)
        g.replay()
        ref.write(k, v, t)
        assert torch.equal(out, kv.attention(q, ref, torch.full((B,), t + 1, device="cuda"), causal=True)), t
        assert torch.equal(c.data, ref.data)


def test_same_answer_every_time(kv):
    k, v, q = (heads(2, 2, t, 64, torch.float32, s) for t, s in ((5000, 71), (5000, 72), (1, 73)))
    c = kv.KVCache4(2, 2, 64, 5000)
    c.write(k, v)
    a = kv.attention(q, c, 5000)
    for _ in range(5):
        assert torch.equal(a, kv.attention(q, c, 5000))


def test_map_reorders_sentences(kv):
    k, v, q = (heads(4, 2, t, 64, torch.bfloat16, s) for t, s in ((30, 81), (30, 82), (1, 83)))
    c = kv.KVCache4(4, 2, 64, 32)
    c.write(k, v)
    want = kv.attention(q, c, 30)
    order = torch.tensor([3, 1, 1], device="cuda")
    c.map(lambda t, dim: t.index_select(dim, order))
    assert c.batch == 3 and torch.equal(kv.attention(q[order], c, 30), want[order])
    c.map(lambda t, dim: t.index_select(dim, order[:0]))
    assert kv.attention(q[:0], c, 30).shape == (0, 2, 1, 64)


def test_copies_and_checkpoints(kv):
    import copy
    import pickle
    c = kv.KVCache4(2, 1, 32, 20)
    k, q = heads(2, 1, 20, 32, torch.float32, 91), heads(2, 1, 1, 32, torch.float32, 92)
    c.write(k, k)
    want = kv.attention(q, c, 20)
    twin, back = copy.deepcopy(c), pickle.loads(pickle.dumps(c))
    c.write(k * 2, k * 2)
    for other in (twin, back):
        assert other.data.data_ptr() != c.data.data_ptr() and torch.equal(kv.attention(q, other, 20), want)


def test_refusals(kv):
    c = kv.KVCache4(2, 2, 64, 40)
    x = torch.zeros(2, 2, 3, 64, device="cuda")
    for bad in (dict(dim=4), dict(dim=136), dict(dim=60), dict(capacity=0), dict(batch=0), dict(heads=0)):
        with pytest.raises(ValueError):
            kv.KVCache4(**{**dict(batch=1, heads=1, dim=64, capacity=8), **bad})
    for k, v, kw in ((x, x[:, :, :2], {}), (x[:1], x[:1], {}), (x[..., :32], x[..., :32], {}), (x, x.bfloat16(), {}),
                     (x, x, dict(start=38)), (x, x, dict(start=-1)), (x, x, dict(counts=3)),
                     (x, x, dict(start=torch.zeros(3, device="cuda", dtype=torch.int32))),
                     (x, x, dict(start=torch.zeros(2, device="cuda"))),
                     (x, x, dict(counts=torch.zeros(2, dtype=torch.int32)))):
        with pytest.raises(ValueError):
            c.write(k, v, **kw)
    with pytest.raises(TypeError):
        c.write(x.half(), x.half())
    with pytest.raises(TypeError):
        c.read(0, 3, dtype=torch.float16)
    with pytest.raises(ValueError):
        c.read(0, 41)
    for q, n in ((x[:, :1], 3), (x[:1], 3), (x[..., :32], 3), (x, 41), (x, -1), (x[0], 3)):
        with pytest.raises(ValueError):
            kv.attention(q, c, n)
    with pytest.raises(RuntimeError, match="no CPU path"):
        c.write(x.cpu(), x.cpu())
    with torch.enable_grad(), pytest.raises(RuntimeError, match="no graph"):
        kv.attention(x.clone().requires_grad_(), c, 3)


def test_data_that_moves_or_shrinks_in_place(kv):
    k, q = heads(3, 2, 20, 64, torch.float32, 95), heads(3, 2, 1, 64, torch.float32, 96)
    c = kv.KVCache4(3, 2, 64, 20)
    c.write(k, k)
    want = kv.attention(q, c, 20)
    c.map(lambda t, dim: t[:2])                         # the same address, fewer sentences
    assert c.batch == 2 and torch.equal(kv.attention(q[:2], c, 20), want[:2])
    held = c.data
    c.data = torch.cat([held, held])[2:]                # moved
    held.zero_()
    assert torch.equal(kv.attention(q[:2], c, 20), want[:2])
    moved = c.data.clone()
    c.data.set_(moved)                                  # the same tensor object, another address
    c.write(k[:2] * 0, k[:2] * 0)
    assert int(c.data.data_ptr()) == moved.data_ptr() and torch.equal(kv.attention(q[:2], c, 20), torch.zeros_like(want[:2]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,H,Hkv,dh,Tq,cap", [(2, 8, 2, 32, 1, 1100), (1, 12, 3, 96, 1, 1500), (3, 2, 2, 64, 1, 700),
                                              (1, 4, 1, 128, 5, 1300)])
def test_scales_that_grow_along_the_sentence(kv, dtype, B, H, Hkv, dh, Tq, cap):
    # the V scales rise by 2^(1/5) a block, then jump up and down: within a power of two, past it, far past it
    t = torch.arange(cap, device="cuda")
    ramp = torch.exp2((t // 64) / 5.0) * torch.where(t % 300 == 299, 40.0, 1.0)
    k, v = heads(B, Hkv, cap, dh, dtype, 61), (heads(B, Hkv, cap, dh, torch.float32, 62) * ramp[:, None]).to(dtype)
    q = heads(B, H, Tq, dh, dtype, 63)
    c = kv.KVCache4(B, Hkv, dh, cap)
    c.write(k, v)
    n = [cap - 3 * b for b in range(B)]
    want, bound = attend(q, values(k), values(v), n, 1.0 / math.sqrt(dh), True)
    close(kv.attention(q, c, torch.tensor(n, device="cuda"), causal=True), want, bound, "growing scales")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dh", [24, 64, 88, 128])
@pytest.mark.parametrize("T", [64, 70, 127, 200])
def test_many_heads_at_once_write_the_same_bytes(kv, dtype, dh, T):
    # 1120 heads go through whole blocks; the same tokens 40 at a time do not: every byte of the cache must agree
    B, H, cap = 140, 8, 210
    k, v = heads(B, H, T, dh, dtype, 71, 2.0), heads(B, H, T, dh, dtype, 72)
    k[3, 1, 5, 0], k[4, 2, T - 1, dh - 1], v[5, 3, 9, 3], v[6, 0, 0, 1] = float("nan"), float("inf"), 1e30, -float("inf")
    g = torch.Generator().manual_seed(T)
    start = torch.randint(-5, cap - T // 2, (B,), generator=g)
    start[:4] = torch.tensor([0, 64, -200, cap])
    counts = torch.randint(0, T + 2, (B,), generator=g)
    for st, n in ((0, None), (min(5, cap - T), None), (start.cuda(), None), (start.cuda(), counts.cuda())):
        c, d = kv.KVCache4(B, H, dh, cap), kv.KVCache4(B, H, dh, cap)
        for x in (c, d):
            x.data.fill_(0xA5)
        c.write(k, v, st, n)
        for lo in range(0, T, 40):
            hi = min(lo + 40, T)
            d.write(k[:, :, lo:hi], v[:, :, lo:hi], st + lo, None if n is None else n - lo)
        assert torch.equal(c.data, d.data)
    got = c.read(start.cuda(), T, counts.cuda(), dtype=torch.float32)
    for out, x in zip(got, (k, v)):
        b = 10
        lo, hi = max(0, -int(start[b])), min(T, int(counts[b]), cap - int(start[b]))
        assert torch.equal(out[b, :, lo:hi], values(x[b, :, lo:hi]).float())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,H,Hkv,dh,Tq,cap", [
    (256, 8, 8, 64, 1, 140),        # a wave each: one row
    (256, 32, 8, 32, 1, 200),       # four rows
    (256, 8, 8, 40, 5, 150),        # sixteen
    (128, 8, 4, 96, 1, 60),         # 512 heads of one block, two rows
    (40, 8, 8, 64, 9, 60),          # 320 of sixteen rows
    (8, 8, 8, 64, 1, 1700),         # eight waves, unsplit
    (64, 8, 8, 64, 1, 1100),
    (32, 8, 8, 128, 1, 400),
    (6, 8, 8, 64, 1, 6000),         # split: one row,
    (3, 16, 4, 128, 1, 2600),       # four,
    (2, 8, 4, 64, 6, 2500),         # sixteen
    (2, 8, 2, 128, 5, 700),         # the largest block: eight waves of sixteen rows and 128 features
    (1, 8, 2, 128, 5, 2000),
])
def test_every_way_a_call_is_cut(kv, dtype, B, H, Hkv, dh, Tq, cap):
    g = torch.Generator().manual_seed(B + cap)
    n = torch.randint(0, cap + 1, (B,), generator=g)
    n[0], n[-1] = cap, cap - 1
    k, v, q = heads(B, Hkv, cap, dh, dtype, 41, 0.7), heads(B, Hkv, cap, dh, dtype, 42), heads(B, H, Tq, dh, dtype, 43)
    c = kv.KVCache4(B, Hkv, dh, cap)
    c.data.fill_(0xFF)                                  # past the lengths: NaN scales
    c.write(k, v, 0, n.cuda())
    got = kv.attention(q, c, n.cuda(), causal=True)
    assert torch.isfinite(got).all()
    for b in sorted({0, min(1, B - 1), B // 2, B - 1}):
        at = slice(b, b + 1)
        want, bound = attend(q[at], values(k[at]), values(v[at]), n[at].tolist(), 1.0 / math.sqrt(dh), True)
        close(got[at], want, bound, "sentence %d of %d tokens" % (b, int(n[b])))


def test_two_calls_at_once(kv):
    # both are split, so both use scratch; each has its own
    k, v = heads(2, 4, 9000, 64, torch.float32, 31), heads(2, 4, 9000, 64, torch.float32, 32)
    c = kv.KVCache4(2, 4, 64, 9000)
    c.write(k, v)
    q = [heads(2, 4, 1, 64, torch.float32, 33 + i) for i in range(2)]
    want = [kv.attention(x, c, 9000 - 100 * i) for i, x in enumerate(q)]
    streams = [torch.cuda.Stream() for _ in q]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(kv.attention(q[i], c, 9000 - 100 * i))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


@pytest.mark.parametrize("longest", [1, 64, 700, 1 << 40])
def test_longest_shapes_the_launch_and_nothing_else(kv, longest):
    for H, Tq in ((2, 1), (8, 1), (4, 7)):
        k, v, q = (heads(2, h, t, 64, torch.float32, s) for h, t, s in ((2, 3000, 51), (2, 3000, 52), (H, Tq, 53)))
        c = kv.KVCache4(2, 2, 64, 3000)
        c.write(k, v)
        n = torch.tensor([3000, 1234], device="cuda")
        want, bound = attend(q, values(k), values(v), n, 1 / 8, False)
        close(kv.attention(q, c, n, longest=longest), want, bound, "longest %d" % longest)


@pytest.mark.parametrize("T,B", [(6, 1), (64, 140)])                # token by token, and whole blocks
def test_values_beyond_the_clamp_in_a_group_that_reaches_it(kv, T, B):
    # the group's range ends at the clamp and is narrow: codes of 65504 and of what lies beyond it would differ
    x = torch.zeros(B, 8, T, 64, device="cuda")
    for t, base in enumerate((65490.0, 65500.0, 65400.0, 60000.0, 65504.0, 65488.0)):
        x[:, :, t] = base
        x[:, :, t, 7], x[:, :, t, 40:44] = 1e6, 3e38
        x[:, :, t, 50] = base - 30.0
    x[:, 4:] *= -1
    c = kv.KVCache4(B, 8, 64, T)
    c.write(x, x)
    for got in c.read(0, T):
        assert torch.equal(got, values(x).float())
