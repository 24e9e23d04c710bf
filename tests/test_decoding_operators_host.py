"""Refusals of the decoding operators' C entry points (include/mssr_hip.h): every bad shape is an error code before
anything is launched, so these run without a GPU; and the host-side helpers."""
import ctypes

import pytest
import torch

from mssrnet_style_transfer_amd import _lib as L
from mssrnet_style_transfer_amd.token_control import TokenControl, pack_allowed

FAKE = 1 << 20          # an address that no call here may reach


def cache(B=2, H=2, capacity=100, dh=64, data=FAKE):
    return L.Kv4Cache(data, B, capacity, H, dh)


def test_cache_sizes():
    lib = L.load()
    assert lib.mssr_kv4_bytes(1, 1, 1, 8) == 2560
    assert lib.mssr_kv4_bytes(3, 2, 65, 64) == 3 * 2 * 2 * 2 * 2560
    assert lib.mssr_kv4_bytes(2, 8, 1 << 24, 128) == 2 * 8 * (1 << 18) * 4 * 2560
    for B, H, cap, dh in ((0, 1, 1, 64), (1, 0, 1, 64), (1, 1, 0, 64), (1, 1, 1, 0), (1, 1, 1, 60), (1, 1, 1, 136),
                          (-1, 1, 1, 64), (1, 1, -1, 64), (1 << 40, 8, 1 << 40, 128), (1, 1, 1 << 62, 64)):
        assert lib.mssr_kv4_bytes(B, H, cap, dh) == -1, (B, H, cap, dh)


@pytest.mark.parametrize("fn", ["mssr_kv4_write", "mssr_kv4_read"])
def test_cache_refusals(fn):
    lib = L.load()

    def call(c, k=FAKE, v=FAKE, T=3, start=None, start0=0, counts=None, bits=0, dtype=L.F32):
        r = L.Kv4Rows(ctypes.addressof(c), k, 0, 0, 64, v, 0, 0, 64, T, start, start0, counts, bits, dtype)
        return getattr(lib, fn)(ctypes.byref(r), None)

    for c in (cache(data=None), cache(dh=60), cache(dh=0), cache(dh=256), cache(B=0), cache(H=0), cache(capacity=0),
              cache(data=FAKE + 8)):
        assert call(c) == 1
    for kw in (dict(k=None), dict(v=None), dict(T=-1), dict(dtype=2), dict(dtype=-1), dict(T=101), dict(start0=98),
               dict(start0=-1), dict(bits=4), dict(start0=1 << 62), dict(T=1 << 62)):
        assert call(cache(), **kw) == 1, kw
    # more heads x blocks than one grid has room for
    assert call(cache(B=1 << 24, H=8, capacity=1 << 20), T=1 << 19) == 1
    assert lib.mssr_last_error()
    assert call(cache(), k=None, v=None, T=0) == 0                          # no tokens: nothing to do


def test_attention_refusals():
    lib = L.load()

    def call(c, q=FAKE, out=FAKE, H=2, Tq=1, lengths=None, n=10, longest=0, scratch=None, nbytes=0, dtype=L.F32):
        d = L.Kv4AttentionDesc(ctypes.addressof(c), q, 0, 0, 64, out, 0, 0, 64, Tq, lengths, n, longest, scratch, nbytes, H, 0,
                               1.0, 0, dtype)
        return lib.mssr_kv4_attention(ctypes.byref(d), None)

    for c in (cache(data=None), cache(dh=60), cache(dh=160), cache(B=0), cache(H=0), cache(capacity=0), cache(data=FAKE + 4)):
        assert call(c) == 1
    for kw in (dict(q=None), dict(out=None), dict(H=3), dict(H=1), dict(H=0), dict(Tq=-1), dict(dtype=2), dict(n=101),
               dict(n=-1), dict(Tq=1 << 40), dict(Tq=(1 << 31) - 1)):
        assert call(cache(), **kw) == 1, kw
    # a long cache of few heads is split, which takes scratch
    c = cache(B=1, capacity=100000)
    need = lib.mssr_kv4_attention_scratch(ctypes.byref(c), 1, 2, 0, L.F32)
    assert need > 0 and call(c, n=100000) == 1 and call(c, n=100000, scratch=FAKE, nbytes=need - 1) == 1
    assert lib.mssr_kv4_attention_scratch(ctypes.byref(cache(capacity=64)), 1, 2, 0, L.F32) == 0
    for kw in (dict(Tq=0), dict(H=3), dict(dtype=5), dict(Tq=1 << 40)):
        a = {**dict(Tq=1, H=2, dtype=0), **kw}
        assert lib.mssr_kv4_attention_scratch(ctypes.byref(c), a["Tq"], a["H"], 0, a["dtype"]) == -1
    assert call(cache(), q=None, out=None, Tq=0) == 0


def control(**kw):
    d = L.TokenControlDesc()
    d.logits, d.out, d.B, d.V, d.ld, d.ldo, d.repetition0 = FAKE, FAKE, 2, 50, 50, 50, 1.0
    for k, v in kw.items():
        setattr(d, k, v)
    return L.load().mssr_token_control(ctypes.byref(d), None)


def test_token_control_refusals():
    for kw in (dict(logits=None), dict(out=None), dict(V=0), dict(V=1 << 31), dict(ld=49), dict(ldo=49), dict(B=-1),
               dict(dtype=2), dict(T=-1), dict(T=1 << 30), dict(ngram=-1), dict(ngram=65),
               dict(allowed=FAKE, states=0), dict(allowed=FAKE, states=1, state_mode=1),
               dict(allowed=FAKE, states=9, state_mode=2), dict(allowed=FAKE, states=9, state_mode=3),
               dict(B=1 << 40), dict(ids=FAKE, V=100000, ld=100000, ldo=100000)):
        assert control(**kw) == 1, kw
    assert L.load().mssr_token_control(None, None) == 1
    assert control(B=0, logits=None) == 0
    lib = L.load()
    for B, V, T in ((0, 5, 0), (1, 0, 0), (1, 5, -1), (1, 5, 1 << 30), (1, 1 << 31, 0)):
        assert lib.mssr_token_control_scratch(B, V, T) == -1
    assert lib.mssr_token_control_scratch(1, 20, 0) == 0 and lib.mssr_token_control_scratch(1, 100000, 0) > 0


def test_new_logits_overlap_the_old_ones_in_place_or_not_at_all():
    # rows of 50 fp32 words, 120 apart: their own place and other columns of the same rows hold nothing of another row.  A call
    # without columns to spare that is let through would launch, so only refusals are made here.
    for kw in (dict(out=FAKE + 4), dict(out=FAKE - 4), dict(out=FAKE + 4 * 49), dict(out=FAKE + 4 * 71, ld=120, ldo=120),
               dict(out=FAKE + 4 * 49, ld=120, ldo=120), dict(out=FAKE - 4 * 71, ld=120, ldo=120),
               dict(ld=120, ldo=110), dict(out=FAKE + 4 * 60, ld=120, ldo=110), dict(out=FAKE + 4 * 99)):
        assert control(**kw) == 1, kw
        assert b"overlap" in L.load().mssr_last_error(), kw
    for kw in (dict(ids=FAKE, empty=1 << 31), dict(ids=FAKE, empty=-(1 << 31) - 1)):
        assert control(**kw) == 1, kw
        assert b"32-bit picks" in L.load().mssr_last_error(), kw
    for kw in (dict(ld=1 << 40), dict(ldo=1 << 40)):
        assert control(**kw) == 1, kw


def test_packed_descriptors_lie_as_the_structures_do():
    for desc in (L.Kv4Rows, L.Kv4AttentionDesc, L.TokenControlDesc):
        fields = [1.25 * i if t is ctypes.c_float else 3 * i + 1 for i, (_, t) in enumerate(desc._fields_)]
        packed = L.packer(desc)(*fields)
        assert len(packed) == ctypes.sizeof(desc)
        back = desc.from_buffer_copy(packed)
        assert [getattr(back, name) for name, _ in desc._fields_] == fields
    assert L.load().mssr_kv4_write(None, None) == 1 and L.load().mssr_kv4_read(None, None) == 1
    assert L.load().mssr_kv4_attention(None, None) == 1
    assert L.load().mssr_kv4_attention(bytes(ctypes.sizeof(L.Kv4AttentionDesc)), None) == 1


def test_pack_allowed():
    g = torch.Generator().manual_seed(3)
    for S, V in ((1, 1), (2, 32), (3, 33), (2, 95)):
        a = torch.rand(S, V, generator=g) < 0.5
        w = pack_allowed(a)
        assert w.dtype == torch.int32 and w.shape == (S, (V + 31) // 32)
        bits = torch.tensor([[(int(w[s, v // 32]) >> (v % 32)) & 1 for v in range(V)] for s in range(S)], dtype=torch.bool)
        assert torch.equal(bits, a)
        assert V % 32 == 0 or all((int(x) & 0xffffffff) >> (V % 32) == 0 for x in w[:, -1])
    with pytest.raises(ValueError):
        pack_allowed(torch.ones(3, 4))


def test_rows_of_a_control():
    index = torch.tensor([2, 0])
    c = TokenControl(repetition=torch.arange(3.0), frequency=0.5, bias=torch.arange(6.0).view(3, 2),
                     allowed=torch.arange(4).view(4, 1).int(), state=torch.tensor([5, 6, 7]))
    r = c.rows(index, 3)
    assert r.repetition.tolist() == [2, 0] and r.frequency == 0.5 and r.bias.tolist() == [[4, 5], [0, 1]]
    assert r.state.tolist() == [7, 5] and r.allowed is c.allowed
    each = TokenControl(bias=torch.zeros(2), allowed=torch.arange(3).view(3, 1).int()).rows(index, 3)
    assert each.allowed.view(-1).tolist() == [2, 0] and each.bias.shape == (2,)
    one = TokenControl(allowed=torch.arange(1).view(1, 1).int()).rows(index, 3)
    assert one.allowed.shape == (1, 1)


def test_cpu_tensors_are_refused():
    from mssrnet_style_transfer_amd import kv_cache, token_control
    with pytest.raises(RuntimeError, match="no CPU path"):
        kv_cache.KVCache4(1, 1, 64, 4, device="cpu")
    with pytest.raises(RuntimeError, match="no CPU path"):
        token_control.pick_token(torch.zeros(2, 5))
    with pytest.raises(ValueError):
        kv_cache.KVCache4(1, 1, 60, 4, device="cpu")


def without_gpu(fn, *args, **kw):
    """What a call says on CPU tensors: graphs are refused before devices."""
    with pytest.raises(RuntimeError) as e:
        fn(*args, **kw)
    return str(e.value)


def test_graphs_and_tangents_are_refused():
    import torch.autograd.forward_ad as fwd

    from mssrnet_style_transfer_amd import kv_cache, token_control
    x, h, n = torch.ones(2, 5), torch.zeros(2, 2, 1, 64), torch.ones(2)
    cache = kv_cache.KVCache4.__new__(kv_cache.KVCache4)

    def calls(mark):
        yield kv_cache.attention, (mark(h), cache, 1), {}
        yield cache.write, (mark(h), h), {}
        yield cache.write, (h, mark(h)), {}
        for fn in (token_control.pick_token, token_control.control_logits):
            yield fn, (mark(x),), {}
            for name, t in (("bias", x), ("repetition", n), ("frequency", n), ("presence", n)):
                yield fn, (x, TokenControl(**{name: mark(t)})), {}
        yield token_control.control_logits, (x,), dict(out=mark(x.clone()))

    for fn, args, kw in calls(lambda t: t.clone().requires_grad_()):
        assert "no graph" in without_gpu(fn, *args, **kw)
        with torch.no_grad():                       # then they are the data that they are
            assert "no CPU path" in without_gpu(fn, *args, **kw)
    with fwd.dual_level():
        for fn, args, kw in calls(lambda t: fwd.make_dual(t.clone(), t.clone())):
            with torch.no_grad():
                assert "without tangents" in without_gpu(fn, *args, **kw)
        assert "no CPU path" in without_gpu(token_control.pick_token, x, TokenControl(bias=x))


def test_a_descriptor_lives_until_its_call_is_over(monkeypatch):
    """Two threads' first calls on one cache both build its descriptor, and the second replaces the first while that one's C
    call may read it.  Here the other thread's turn comes inside the call, by hand."""
    import struct
    import weakref

    from mssrnet_style_transfer_amd import kv_cache
    made = []

    class Watched(L.Kv4Cache):
        def __init__(self, *args):
            super().__init__(*args)
            made.append((ctypes.addressof(self), weakref.ref(self)))

    class OnDevice(torch.Tensor):               # CPU data that passes for a device's
        is_cuda = True

    calls = []

    def call(name, device, desc):
        address = struct.unpack_from("P", desc)[0]
        other = L.Kv4Cache(0, 2, 64, 2, 64)         # the other thread found none either, built its own
        cache._held = (None, other, 0)              # and stores it
        assert any(a == address and ref() is not None for a, ref in made), name
        calls.append(name)

    monkeypatch.setattr(L, "Kv4Cache", Watched)
    monkeypatch.setattr(L, "call", call)
    monkeypatch.setattr(kv_cache, "_scratch_bytes", lambda *a: 0)
    cache = kv_cache.KVCache4.__new__(kv_cache.KVCache4)
    cache.heads, cache.dim, cache.capacity, cache._held = 2, 64, 64, None
    cache.data = torch.zeros(2, L.load().mssr_kv4_bytes(2, 2, 64, 64) // 2, dtype=torch.uint8)
    x = torch.zeros(2, 2, 1, 64).as_subclass(OnDevice)
    for fn in (lambda: cache.write(x, x), lambda: cache.read(0, 1), lambda: kv_cache.attention(x, cache, 1)):
        cache._held = None
        fn()
    assert calls == ["mssr_kv4_write", "mssr_kv4_read", "mssr_kv4_attention"]


def test_a_cached_search_that_fails_leaves_no_state():
    from types import SimpleNamespace

    from mssrnet_style_transfer_amd.config import MSSRConfig
    from mssrnet_style_transfer_amd.style_generator_builder import build_all
    from mssrnet_style_transfer_amd.translate import greedy_decode_cached
    cfg = MSSRConfig.small()
    model = build_all(cfg, device="cpu", seed=1)["model"].eval()
    mem, lens = torch.zeros(5, 3, cfg.d_model), torch.tensor([5, 2, 3])
    with pytest.raises(RuntimeError, match="no CPU path"):              # the first step's cache has no place on the CPU
        greedy_decode_cached(model, cfg, mem, lens, 4)
    assert all(model.decoder.state[name] is None for name in ("src", "cache", "kv4_steps"))
    nothing = SimpleNamespace()                                         # a search of no steps asks nothing of the model
    assert greedy_decode_cached(nothing, cfg, mem, lens, 0).shape == (0, 3)


def test_new_logits_over_the_bias_are_refused():
    far = FAKE + (1 << 16)
    for kw in (dict(out=far, bias=far), dict(out=far, bias=far + 4 * 99), dict(out=far, bias=far - 4 * 49),
               dict(out=far, bias=far - 4 * 60, bias_bs=50), dict(out=far, bias=far, dtype=L.BF16, logits=FAKE)):
        assert control(**kw) == 1, kw
        assert b"overlap the bias" in L.load().mssr_last_error(), kw
    for kw in (dict(out=far, bias=FAKE + 4096, bias_bs=-1), dict(out=far, bias=FAKE + 4096, bias_bs=1 << 40)):
        assert control(**kw) == 1, kw
