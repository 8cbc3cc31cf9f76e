"""Host side of the paged KV-cache operators: rotary frequencies under every
scaling against their formulas, and the refusals of the C entry points, which
come before anything touches a device."""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def P():
    from jetsonfabric_b200 import build_cuda
    build_cuda.build()
    from jetsonfabric_b200 import paged
    paged._bind()
    return paged


@pytest.mark.parametrize("dims,base", [(128, 1e6), (64, 1e4), (2, 1e6), (96, 5e5)])
def test_frequencies_by_formula(P, dims, base):
    i = np.arange(dims // 2)
    plain = base ** (-2.0 * i / dims)
    freq, factor = P.rope_frequencies(dims, base)
    assert factor == 1.0 and np.allclose(freq, plain, rtol=1e-14)
    freq, factor = P.rope_frequencies(dims, base, "linear", factor=8.0)
    assert factor == 1.0 and np.allclose(freq, plain / 8, rtol=1e-14)
    if dims > 2:
        freq, factor = P.rope_frequencies(dims, base, "ntk", factor=4.0)
        assert factor == 1.0 and np.allclose(freq, (base * 4 ** (dims / (dims - 2))) ** (-2.0 * i / dims), rtol=1e-13)


def test_yarn_keeps_fast_pairs_and_divides_slow_ones(P):
    dims, base, trained, s = 128, 1e6, 32768, 4.0
    freq, factor = P.rope_frequencies(dims, base, "yarn", factor=s, trained=trained)
    plain = base ** (-2.0 * np.arange(64) / dims)
    turns = trained * plain / (2 * math.pi)
    assert math.isclose(factor, 0.1 * math.log(4) + 1, rel_tol=1e-15)
    assert np.allclose(freq[turns > 40], plain[turns > 40], rtol=1e-14)
    assert np.allclose(freq[turns < 0.8], plain[turns < 0.8] / s, rtol=1e-14)
    ratio = freq / plain
    assert np.all(np.diff(ratio) <= 1e-15) and ratio.min() >= 1 / s - 1e-15
    low = max(math.floor(dims * math.log(trained / (32 * 2 * math.pi)) / (2 * math.log(base))), 0)
    high = min(math.ceil(dims * math.log(trained / (2 * math.pi)) / (2 * math.log(base))), dims - 1)
    for i in range(64):
        kept = 1 - min(max((i - low) / (high - low), 0), 1)
        assert math.isclose(freq[i], plain[i] * kept + plain[i] / s * (1 - kept), rel_tol=1e-13)


@pytest.mark.parametrize("dims,base,trained", [(16, 100.0, 1e7), (64, 1e4, 1e12), (128, 1e6, 1e16), (64, 1e4, 5.0), (128, 1e6, 0.5),
                                               (64, 1e4, 1e-3), (16, 0.5, 1e7), (16, 0.5, 1.0), (2, 1e4, 1e8), (2, 1e4, 1.0)])
def test_yarn_beyond_its_ramp(P, dims, base, trained):
    """A trained context over which every pair makes more turns than `high` keeps all frequencies; one over which
    none makes as many as `low` divides all."""
    plain = base ** (-2.0 * np.arange(dims // 2) / dims)
    turns = trained * plain / (2 * math.pi)
    assert turns.min() > 32 or turns.max() < 1
    freq, _ = P.rope_frequencies(dims, base, "yarn", factor=4.0, trained=trained)
    assert np.allclose(freq, plain if turns.min() > 32 else plain / 4, rtol=1e-14)


def test_bands_blend_by_wavelength(P):
    dims, base, trained, s, lo, hi = 128, 5e5, 8192, 8.0, 1.0, 4.0
    freq, factor = P.rope_frequencies(dims, base, "bands", factor=s, trained=trained, low=lo, high=hi)
    assert factor == 1.0
    for i, f in enumerate(base ** (-2.0 * np.arange(64) / dims)):
        wave = 2 * math.pi / f
        if wave < trained / hi:
            want = f
        elif wave > trained / lo:
            want = f / s
        else:
            kept = (trained / wave - lo) / (hi - lo)
            want = (1 - kept) * f / s + kept * f
        assert math.isclose(freq[i], want, rel_tol=1e-13)


@pytest.mark.parametrize("kw", [
    dict(rope_dims=63, base=1e6), dict(rope_dims=0, base=1e6), dict(rope_dims=64, base=0.0), dict(rope_dims=64, base=math.nan),
    dict(rope_dims=64, base=1e6, scaling="linear", factor=0.5), dict(rope_dims=64, base=1e6, scaling="ntk", factor=math.nan),
    dict(rope_dims=2, base=1e6, scaling="ntk", factor=2.0), dict(rope_dims=64, base=1e6, scaling="yarn", factor=2.0),
    dict(rope_dims=64, base=1e6, scaling="yarn", factor=2.0, trained=4096, low=4.0, high=4.0),
    dict(rope_dims=64, base=1.0, scaling="yarn", factor=2.0, trained=4096),
    dict(rope_dims=64, base=1e6, scaling="bands", factor=2.0, trained=-1.0), dict(rope_dims=64, base=1e6, scaling="cubic"),
])
def test_frequency_refusals(P, kw):
    with pytest.raises(P.InvalidArgument):
        P.rope_frequencies(**kw)


# Addresses that are never followed: a refused call reads no device memory.
A = 1 << 20


def cache(P, **kw):
    d = dict(k=A, v=A, page_stride=16 * 2 * 128, token_stride=2 * 128, head_stride=128, dtype=1, pages=10, page_size=16,
             kv_heads=2, head_dim=128, reserved=0)
    d.update(kw)
    return P.CacheC(**d)


def batch(P, **kw):
    d = dict(q_start=A, kv_len=A, page_table=A, table_stride=4, sequences=2, table_width=4)
    d.update(kw)
    return P.BatchC(**d)


BAD_CACHES = [dict(k=None), dict(v=None), dict(dtype=0), dict(dtype=3), dict(page_size=12), dict(page_size=4), dict(page_size=2048),
              dict(page_size=0), dict(head_dim=0), dict(head_dim=132), dict(head_dim=136), dict(head_dim=4), dict(pages=0),
              dict(kv_heads=0), dict(page_stride=0), dict(token_stride=250), dict(head_stride=4), dict(head_stride=64),
              dict(token_stride=1 << 40), dict(k=A + 2), dict(v=A + 8)]
BAD_BATCHES = [dict(kv_len=None), dict(page_table=None), dict(table_width=0), dict(table_stride=3), dict(sequences=4097)]


def refused(st):
    assert st.code == 1 and st.message, (st.code, st.message)


def rope_call(P, c, b, **kw):
    d = dict(q=A, k=A, v=A, dtype=0, qs=4 * 128, ks=256, vs=256, rows=3, heads=4, pos=A, freq=A, dims=128, q_out=2 * A, os=4 * 128)
    d.update(kw)
    rope = P.RopeC(d["freq"], d["dims"], 0, 1.0, 0)
    return P._bind().jfb_rope_paged_append(d["q"], d["k"], d["v"], d["dtype"], d["qs"], d["ks"], d["vs"], d["rows"], d["heads"],
                                           d["pos"], C.byref(rope), C.byref(c), C.byref(b), d["q_out"], d["os"], None, None)


def attention_call(P, c, b, **kw):
    d = dict(q=A, qs=4 * 128, rows=3, heads=4, scale=0.1, window=0, out=A, os=4 * 128)
    d.update(kw)
    return P._bind().jfb_paged_attention(d["q"], d["qs"], d["rows"], d["heads"], d["scale"], d["window"], C.byref(c), C.byref(b),
                                         d["out"], d["os"], None, None, 0, None, None)


def mass_call(P, c, b, **kw):
    d = dict(q=A, qs=4 * 128, rows=3, heads=4, scale=0.1, window=0, lse=A, out=A, slots=64)
    d.update(kw)
    return P._bind().jfb_paged_attention_mass(d["q"], d["qs"], d["rows"], d["heads"], d["scale"], d["window"], d["lse"],
                                              C.byref(c), C.byref(b), None, d["out"], d["slots"], None, None)


def evict_call(P, c, b, **kw):
    d = dict(mass=A, slots=64, budget=32, recent=8, keep=A, kv_out=A, mass_out=2 * A, out_slots=64, table=2 * A, stride=4, width=4)
    d.update(kw)
    return P._bind().jfb_paged_evict(d["mass"], d["slots"], C.byref(c), C.byref(b), d["budget"], d["recent"], d["keep"],
                                     d["kv_out"], d["mass_out"], d["out_slots"], d["table"], d["stride"], d["width"], None, None)


CALLS = [rope_call, attention_call, mass_call, evict_call]


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("bad", BAD_CACHES)
def test_bad_caches_are_refused(P, call, bad):
    refused(call(P, cache(P, **bad), batch(P)))


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("bad", BAD_BATCHES)
def test_bad_batches_are_refused(P, call, bad):
    refused(call(P, cache(P), batch(P, **bad)))


@pytest.mark.parametrize("bad", [dict(q=None), dict(k=None), dict(v=None), dict(pos=None), dict(freq=None), dict(q_out=None),
                                 dict(dtype=3), dict(heads=0), dict(dims=0), dict(dims=63), dict(dims=130), dict(qs=511),
                                 dict(ks=255), dict(vs=255), dict(os=256), dict(q=A + 2), dict(q_out=A + 1, dtype=1),
                                 dict(q=A, q_out=A), dict(q=A, q_out=A, dtype=1, os=1024), dict(rows=1 << 31)])
def test_rope_refusals(P, bad):
    refused(rope_call(P, cache(P), batch(P), **bad))


@pytest.mark.parametrize("call", [attention_call, mass_call])
@pytest.mark.parametrize("bad", [dict(q=None), dict(q=A + 2), dict(qs=511), dict(qs=256), dict(heads=3), dict(heads=0), dict(scale=0.0),
                                 dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(scale=2e38), dict(window=1 << 31), dict(out=None),
                                 dict(rows=1 << 31)])
def test_attention_refusals(P, call, bad):
    refused(call(P, cache(P), batch(P), **bad))


@pytest.mark.parametrize("q,qs,out,os,rows,overlap", [
    (A, 512, A, 512, 3, True), (A, 512, A + 16, 512, 1, True), (A, 512, A + 1024, 512, 3, True), (A, 512, A + 5120, 512, 5, False),
    (A + 5120, 512, A, 512, 5, False), (A + 5104, 512, A, 512, 5, True), (A, 512, A + 1024, 512, 1, False),
    (A, 1024, A + 1024, 1024, 3, False), (A + 1024, 1024, A, 1024, 3, False), (A, 1024, A + 1008, 1024, 3, True),  # slices of one buffer
    (A, 1024, A + 1040, 1024, 3, True), (A, 1024, A + 1040, 1024, 1, False), (A, 1032, A + 1024, 1024, 3, True)])
def test_attention_refuses_out_over_q(P, q, qs, out, os, rows, overlap):
    st = attention_call(P, cache(P), batch(P), q=q, qs=qs, out=out, os=os, rows=rows)
    # what passes is refused for its missing workspace, or for the missing device
    assert st.code != 0 and (b"overlap" in st.message if isinstance(st.message, bytes) else "overlap" in st.message) == overlap


@pytest.mark.parametrize("bad", [dict(lse=None), dict(slots=0)])
def test_mass_refusals(P, bad):
    refused(mass_call(P, cache(P), batch(P), **bad))


@pytest.mark.parametrize("bad", [dict(mass=None), dict(keep=None), dict(kv_out=None), dict(mass_out=None), dict(table=None),
                                 dict(budget=0), dict(recent=33), dict(slots=0), dict(out_slots=31), dict(width=1), dict(stride=3),
                                 dict(mass_out=A, out_slots=32), dict(table=A, stride=8)])
def test_evict_refusals(P, bad):
    refused(evict_call(P, cache(P), batch(P), **bad))


def test_empty_calls_need_no_device(P):
    """No sequences: nothing to do, nothing launched."""
    for call in (rope_call, evict_call):
        assert call(P, cache(P), batch(P, sequences=0)).code == 0
    assert rope_call(P, cache(P), batch(P), rows=0).code == 0


def test_empty_arrays_may_be_absent(P):
    """Tensors without elements have no address: no sequences, or no rows."""
    none = batch(P, q_start=None, kv_len=None, page_table=None, sequences=0)
    assert rope_call(P, cache(P), none).code == 0
    assert attention_call(P, cache(P), none).code == 0
    assert mass_call(P, cache(P), none, out=None).code == 0
    assert evict_call(P, cache(P), none, mass=None, mass_out=None, keep=None, kv_out=None, table=None).code == 0
    assert rope_call(P, cache(P), batch(P), rows=0, q=None, k=None, v=None, pos=None, q_out=None).code == 0
    assert attention_call(P, cache(P), batch(P), rows=0, q=None, out=None).code == 0
    refused(attention_call(P, cache(P), batch(P), rows=0, heads=3))


def test_python_refuses_host_tensors(P):
    pool = torch.zeros(4, 16, 2, 128, dtype=torch.float16)
    with pytest.raises(P.InvalidArgument):
        P.PagedCache(pool, pool)
    with pytest.raises(P.InvalidArgument):
        P.PagedBatch(torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(2, 4, dtype=torch.int32))
    with pytest.raises(P.InvalidArgument):
        P.Rope(torch.zeros(64, dtype=torch.float64))
