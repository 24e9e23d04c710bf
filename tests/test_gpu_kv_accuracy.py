"""How near attention over the 4-bit cache comes to the formula in 64 bits over the values that the cache stands for, judged
by what typical roundings add up to (tests/test_gpu_kv_cache.py bounds the worst case, which is far wider)."""
import math

import pytest
import torch

from test_gpu_kv_cache import SHAPES, heads, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv():
    from mssrnet_style_transfer_amd import kv_cache
    with torch.no_grad():
        yield kv_cache


def exact(q, k, v, scale, visible=None):
    """softmax(scale q k^T) v in 64 bits; k, v [B, Hkv, n, dh] in 64 bits already; visible: Bool [B, Tq, n], rows that see
    something."""
    B, H, T, dh = q.shape
    G = H // k.shape[1]
    s = torch.matmul(q.double(), k.repeat_interleave(G, 1).transpose(2, 3).contiguous()) * scale
    if visible is not None:
        s = s.masked_fill(~visible.unsqueeze(1), float("-inf"))
    return torch.matmul(torch.softmax(s, -1), v.repeat_interleave(G, 1))


def judge(got, want, share):
    """``share``: how large the error before the result's rounding may be, as a part of the result's norm.

    fp32: that, and the rounding itself (2^-24).  bf16: an error e moves a number over the border between two roundings with
    probability |e| / ulp, ulp >= 2^-8 |x|.  With E|e| = 0.8 rms(e) and E min(ulp, .) / |x| about 5 / rms(x) for normally
    distributed x, a share of 2^8 * 5 * 0.8 * share ~ 1024 share of the numbers; twice that is allowed."""
    assert torch.isfinite(got).all()
    if got.dtype == torch.float32:
        err = float((got.double() - want).norm() / want.norm())
        assert err <= share + 2.0 ** -24, "%.3g of the result, %.3g allowed" % (err, share)
    else:
        # Stored values lie on a grid, so that means of a few of equal weight often lie halfway between two bf16 numbers, both
        # of them nearest then: 9 % of single values, 4 % of means of three, 0.5 % of means of a hundred (counted in 64 bits).
        least = (want.float().bfloat16().double() - want).abs()             # (rounded twice: moves one in 2^16)
        off = float(((got.double() - want).abs() > least * (1 + 1e-9)).double().mean())
        assert off <= 2048 * share + 2 / got.numel(), "%.3g of the numbers are not the nearest, %.3g allowed" % (off, 2048 * share)


ROWS = [(2, 2, 1), (8, 2, 1)]           # query heads, key/value heads, new tokens: one query row a head, four


def check_one_token(kv, dtype, dh, H, Hkv, Tq):
    B = 64
    k, v, q = heads(B, Hkv, 1, dh, dtype, 1), heads(B, Hkv, 1, dh, dtype, 2), heads(B, H, Tq, dh, dtype, 3)
    c = kv.KVCache4(B, Hkv, dh, 1)
    c.write(k, v)
    want = values(v).repeat_interleave(H // Hkv, 1).expand(B, H, Tq, dh)
    # p cancels in the quotient; codes and zeros meet as |z| + 15 s <= 3 max |v| of the group, each held to 2^-22 and summed in
    # half a dozen roundings: 2^-19 of the group's largest value, then the result's own rounding
    top = torch.cat([g.abs().amax(-1, keepdim=True).expand_as(g) for g in want.split(32, -1)], -1)
    half = torch.finfo(dtype).eps / 2
    err = (kv.attention(q, c, 1).double() - want).abs()
    assert (err <= 2.0 ** -19 * top + half * want.abs()).all(), float((err / (2.0 ** -19 * top + half * want.abs())).max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dh", [8, 40, 64, 96, 128])
@pytest.mark.parametrize("H,Hkv,Tq", ROWS)
def test_a_sentence_of_one_token_is_that_token(kv, dtype, dh, H, Hkv, Tq):
    check_one_token(kv, dtype, dh, H, Hkv, Tq)


def check_mean_zero(kv, dtype, n, H, Hkv, Tq, same):
    """Values about zero: the codes' and the zeros' share of the context cancel to 1 / sqrt(n) of either, and what is
    cut off each time 64 tokens are added up does not average out: 2.4e-7 sqrt(n) (7.5 s = 2 deviations, 2^-24 each), over 1e-5 of
    the parts' 2^-21 times 4 deviations and the scores' roundings."""
    B, dh = 2 if n > 1000 else 16, 64
    k, v, q = heads(B, Hkv, n, dh, dtype, 11), heads(B, Hkv, n, dh, dtype, 12), heads(B, H, Tq, dh, dtype, 13)
    if same:
        k = k[:, :, :1].expand(B, Hkv, n, dh)           # every token has the same score
    c = kv.KVCache4(B, Hkv, dh, n)
    c.write(k, v)
    want = exact(q, values(k), values(v), 1 / math.sqrt(dh))
    judge(kv.attention(q, c, n), want, 1e-5 + 2.4e-7 * math.sqrt(n))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("same", [False, True])
@pytest.mark.parametrize("n", [3, 100, 2000, 16000])
@pytest.mark.parametrize("H,Hkv,Tq", ROWS)
def test_values_about_zero(kv, dtype, n, H, Hkv, Tq, same):
    check_mean_zero(kv, dtype, n, H, Hkv, Tq, same)


MORE_ROWS = [(4, 2, 5), (8, 2, 5), (2, 2, 16)]         # ten, twenty and sixteen query rows a key/value head


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dh", [8, 40, 64, 96, 128])
@pytest.mark.parametrize("H,Hkv,Tq", MORE_ROWS)
def test_a_sentence_of_one_token_is_that_token_in_every_row(kv, dtype, dh, H, Hkv, Tq):
    check_one_token(kv, dtype, dh, H, Hkv, Tq)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("same", [False, True])
@pytest.mark.parametrize("n", [3, 100, 2000, 16000])
@pytest.mark.parametrize("H,Hkv,Tq", MORE_ROWS)
def test_values_about_zero_in_many_rows(kv, dtype, n, H, Hkv, Tq, same):
    check_mean_zero(kv, dtype, n, H, Hkv, Tq, same)


# ------------------------------------------------------------------------------------------------ values of other sizes beside
ALL_ROWS = ROWS + MORE_ROWS
# p s is held to 2^-22 of itself, its products and sums in fp32: 4 deviations * 2^-21 = 2e-6 as in check_mean_zero; the largest of
# some 50 rows' errors is twice the typical one.  The scores' part is small: keys of deviation 1 and queries of 1.
BESIDE = 5e-6


def judge_rows(got, want, share):
    """judge() of every query row and group of 32 features for itself."""
    for a, b in zip(got.split(32, -1), want.split(32, -1)):
        if got.dtype == torch.float32:
            err = ((a.double() - b).norm(dim=-1) / b.norm(dim=-1)).max()
            assert float(err) <= share + 2.0 ** -24, "%.3g of a row, %.3g allowed" % (float(err), share)
        else:
            judge(a, b, 2 * share)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ratio", [1e3, 1e6])
@pytest.mark.parametrize("where", [2, 150, 299])
@pytest.mark.parametrize("H,Hkv,Tq", ALL_ROWS)
def test_a_large_value_that_nobody_attends_to(kv, dtype, ratio, where, H, Hkv, Tq):
    B, n, dh = 3, 300, 64
    k, v, q = heads(B, Hkv, n, dh, dtype, 21), heads(B, Hkv, n, dh, dtype, 22), heads(B, H, Tq, dh, dtype, 23)
    q[..., 0] = 8.0                                     # the token's key is far off along this feature for every row
    k[..., 0] *= 0.01
    k[:, :, where, 0] = -100.0
    v *= 1e-3
    v[:, :, where] *= ratio
    c = kv.KVCache4(B, Hkv, dh, n)
    c.write(k, v)
    want = exact(q, values(k), values(v), 1 / math.sqrt(dh))
    judge_rows(kv.attention(q, c, n), want, BESIDE)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,Hkv,Tq", [r for r in ALL_ROWS if r[0] * r[2] > r[1]])
def test_a_large_value_that_one_row_attends_to(kv, dtype, H, Hkv, Tq):
    B, n, dh = 2, 200, 64
    k, v, q = heads(B, Hkv, n, dh, dtype, 31), heads(B, Hkv, n, dh, dtype, 32), heads(B, H, Tq, dh, dtype, 33)
    q[..., 0] = 8.0
    q[:, ::H // Hkv, 0, 0] = -8.0                       # the first row of every key/value head
    k[..., 0] *= 0.01
    k[:, :, 70, 0] = -100.0
    v *= 1e-3
    v[:, :, 70] *= 1e6
    c = kv.KVCache4(B, Hkv, dh, n)
    c.write(k, v)
    want = exact(q, values(k), values(v), 1 / math.sqrt(dh))
    assert (want[:, 0, 0].abs().amax(-1) > 100).all() and (want[:, 0, 1:] if Tq > 1 else want[:, 1]).abs().max() < 1e-2
    judge_rows(kv.attention(q, c, n), want, BESIDE)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,Hkv,Tq", ALL_ROWS)
def test_groups_of_other_sizes(kv, dtype, H, Hkv, Tq):
    B, n, dh = 3, 500, 96
    k, v, q = heads(B, Hkv, n, dh, dtype, 41), heads(B, Hkv, n, dh, dtype, 42), heads(B, H, Tq, dh, dtype, 43)
    v[..., :32] *= 1e3
    v[..., 64:] *= 1e-3
    c = kv.KVCache4(B, Hkv, dh, n)
    c.write(k, v)
    judge_rows(kv.attention(q, c, n), exact(q, values(k), values(v), 1 / math.sqrt(dh)), BESIDE)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,Hkv,Tq", [(4, 2, 2), (4, 2, 5), (2, 2, 16)])
def test_a_large_value_that_later_rows_see(kv, dtype, H, Hkv, Tq):
    B, n, dh = 2, 130, 64
    k, v, q = heads(B, Hkv, n, dh, dtype, 51), heads(B, Hkv, n, dh, dtype, 52), heads(B, H, Tq, dh, dtype, 53)
    v *= 1e-3
    v[:, :, n - 1] *= 1e6
    c = kv.KVCache4(B, Hkv, dh, n)
    c.write(k, v)
    see = torch.arange(n, device="cuda") < (n - Tq + 1 + torch.arange(Tq, device="cuda")).view(1, Tq, 1)
    want = exact(q, values(k), values(v), 1 / math.sqrt(dh), see.expand(B, Tq, n))
    judge_rows(kv.attention(q, c, n, causal=True), want, BESIDE)


# ------------------------------------------------------------------------------------------------ ordinary inputs
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("B,H,Hkv,dh,Tq,cap,lengths", SHAPES)
def test_ordinary_inputs_in_norm(kv, B, H, Hkv, dh, Tq, cap, lengths, causal, dtype):
    """A score is a sum over dh features of |q| (|z| + 15 s) ~ 5, codes' and zeros' parts apart, times scale: 5 sqrt(dh) ~ 50 at
    most, with the parts' 2^-22 (bf16: the low codes' 2^-21) and some roundings, of which a random half cancels: rms 1e-6 of a
    probability, and 2e-6 of the codes (check_mean_zero) at most: 3e-6 together in fp32, 1e-5 in bf16, whose scores take one part
    and low codes.  (Probabilities of one part would be 2^-12 / sqrt(3) = 1.4e-4 off, a dropped last token of 20000 7e-3.)"""
    c = kv.KVCache4(B, Hkv, dh, cap)
    c.data.fill_(0xFF)
    n = torch.tensor(lengths, device="cuda", dtype=torch.int32)
    k, v = heads(B, Hkv, cap, dh, dtype, 11, 1.5), heads(B, Hkv, cap, dh, dtype, 12)
    c.write(k, v, 0, n)
    q = heads(B, H, Tq, dh, dtype, 13)
    got = kv.attention(q, c, n, causal=causal)
    kk, vv = values(k), values(v)
    got_rows, want_rows = [], []
    for b, m in enumerate(lengths):
        for i in range(Tq):
            see = max(0, m - Tq + 1 + i) if causal else m
            if see == 0:
                assert (got[b, :, i] == 0).all()
                continue
            at = slice(b, b + 1)
            got_rows.append(got[at, :, i])
            want_rows.append(exact(q[at, :, i:i + 1], kk[at, :, :see], vv[at, :, :see], 1 / math.sqrt(dh))[:, :, 0])
    judge(torch.cat(got_rows), torch.cat(want_rows), 3e-6 if dtype == torch.float32 else 1e-5)
