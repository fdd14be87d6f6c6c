"""Frequencies of multi-axis rotary embeddings (iian_pa_mrope_frequencies, host
code) against their formulas in 64 bits, and what the entry points of prompts
with images refuse before any launch."""
import ctypes as C
import math

import numpy as np
import pytest

import iian_amd as pa
from iian_amd import _lib


def freqs(n_dims=128, base=1e6, sections=(16, 24, 24), layout=pa.MROPE_SECTIONS, **kw):
    f, a, ms = pa.mrope_frequencies(pa.RopeParams(n_dims=n_dims, freq_base=base, **kw), sections, layout, device="cpu")
    return f.numpy(), a.numpy(), ms


def test_sections():
    f, a, ms = freqs()
    j = np.arange(64)
    assert np.allclose(f, 1e6 ** (-j / 64.0), rtol=1e-14, atol=0) and ms == 1.0
    assert a.tolist() == [0] * 16 + [1] * 24 + [2] * 24


def test_sections_of_nothing_are_skipped():
    assert freqs(8, sections=(0, 2, 0, 2))[1].tolist() == [1, 1, 3, 3]


def test_interleaved():
    f, a, _ = freqs(sections=(24, 20, 20), layout=pa.MROPE_INTERLEAVED)
    want = [j % 3 if j % 3 and j < 3 * 20 else 0 for j in range(64)]
    assert a.tolist() == want
    assert np.allclose(f, 1e6 ** (-np.arange(64) / 64.0), rtol=1e-14, atol=0)


def test_restart():
    f, a, _ = freqs(80, base=1e4, sections=(20, 20), layout=pa.MROPE_RESTART)
    one = 1e4 ** (-np.arange(20) / 20.0)
    assert np.allclose(f, np.concatenate([one, one]), rtol=1e-14, atol=0)
    assert a.tolist() == [0] * 20 + [1] * 20


def test_scale_factors_and_ramp():
    import torch
    ff = torch.linspace(1, 4, 32)
    f, _, ms = freqs(64, base=1e4, sections=(32,), freq_scale=0.25, ext_factor=1.0, n_ctx_orig=4096, attn_factor=0.5,
                     freq_factors=ff)
    j = np.arange(32)
    end = lambda beta, r: r(64 * math.log(4096 / (beta * 2 * math.pi)) / (2 * math.log(1e4)))
    low, high = max(0, end(32.0, math.floor)), min(63, end(1.0, math.ceil))
    mix = 1 - np.clip((j - low) / max(0.001, high - low), 0, 1)
    want = 1e4 ** (-j / 32.0) / ff.numpy() * (0.25 * (1 - mix) + mix)
    assert np.allclose(f, want, rtol=1e-13, atol=0)
    assert abs(ms - 0.5 * (1 + 0.1 * math.log(4))) < 1e-7
    assert np.allclose(freqs(64, base=1e4, sections=(32,), freq_scale=0.25)[0], 0.25 * 1e4 ** (-j / 32.0), rtol=1e-14)


@pytest.mark.parametrize("kw,code", [
    (dict(n_dims=127), -2), (dict(n_dims=0), -2), (dict(n_dims=2048), -2), (dict(sections=(16, 24, 23)), -2),
    (dict(sections=(80, -16)), -2), (dict(layout=3), -2), (dict(base=0.0), -2), (dict(freq_scale=0.0), -2),
    (dict(ext_factor=1.0), -2),                                                    # a ramp without n_ctx_orig
    (dict(ext_factor=1.0, n_ctx_orig=4096, sections=(32, 32), layout=pa.MROPE_RESTART), -3),
])
def test_frequencies_refused(kw, code):
    with pytest.raises(pa.PagedAttnError) as e:
        freqs(**kw)
    assert e.value.status == code


def test_frequencies_null():
    lib = _lib.load()
    assert lib.iian_pa_mrope_frequencies(None, None, None, None, None) == -1


def positions(**over):
    a = dict(spans=0x1000, off=0x2000, n_spans=4, nc=0x3000, qsl=0x4000, S=2, T=8, full=0, pos=0x5000, end=0x6000, err=None)
    a.update(over)
    return _lib.load().iian_pa_mrope_positions(None, a["spans"], a["off"], a["n_spans"], a["nc"], a["qsl"], a["S"],
                                               a["T"], a["full"], a["pos"], a["end"], a["err"])


@pytest.mark.parametrize("over,code", [
    ({"spans": None}, -1), ({"off": None}, -1), ({"nc": None}, -1), ({"qsl": None}, -1), ({"pos": None}, -1),
    ({"S": -1}, -2), ({"T": -1}, -2), ({"n_spans": -1}, -2), ({"n_spans": 2 ** 31 - 1}, -2), ({"spans": 0x1008}, -2), ({"S": 0}, 0), ({"T": 0}, 0),
])
def test_positions_refused(over, code):
    assert positions(**over) == code


def kv_write(**over):
    a = dict(q=0x10000, k=0x20000, v=0x30000, qo=0x40000, ko=None, qs=1024, ks=256, vs=256, qos=1024, kos=256, qn=None,
             kn=None, eps=1e-6, type=30, pos=0x50000, slots=0x60000, n=4, H=8, Hkv=2, D=128, Dv=128, freqs=0x70000,
             axis=0x80000, n_axes=3, n_dims=128, mode=2, ms=1.0, kp=0x90000, vp=0xa0000, cells=64, tk=1, tv=1)
    a.update(over)
    r = _lib.MRopeRows(a["q"], a["k"], a["v"], a["qo"], a["ko"], a["qs"], a["ks"], a["vs"], a["qos"], a["kos"],
                       a["qn"], a["kn"], a["eps"], a["type"])
    return _lib.load().iian_pa_mrope_kv_write(None, C.byref(r), a["pos"], a["slots"], a["n"], a["H"], a["Hkv"], a["D"],
                                              a["Dv"], a["freqs"], a["axis"], a["n_axes"], a["n_dims"], a["mode"],
                                              a["ms"], a["kp"], a["vp"], a["cells"], a["tk"], a["tv"], None)


@pytest.mark.parametrize("over,code", [
    ({"k": None}, -1), ({"v": None}, -1), ({"pos": None}, -1), ({"slots": None}, -1), ({"freqs": None}, -1),
    ({"axis": None}, -1), ({"kp": None}, -1), ({"vp": None}, -1), ({"kp": None, "vp": None, "slots": None}, -1),
    ({"q": None}, -2), ({"qo": None}, -2), ({"H": 0}, -2), ({"Hkv": 0}, -2), ({"D": 0}, -2), ({"n": -1}, -2),
    ({"n_axes": 0}, -2), ({"n_axes": 5}, -2), ({"n_dims": 0}, -2), ({"n_dims": 127}, -2), ({"n_dims": 130}, -2),
    ({"mode": 1}, -3), ({"mode": 8}, -3), ({"type": 8}, -3), ({"type": 2}, -3), ({"tk": 30}, -3), ({"tv": 2}, -3),
    ({"D": 1025, "n_dims": 128, "qs": 8200, "qos": 8200, "ks": 2050}, -3), ({"ms": math.inf}, -2), ({"eps": -1.0}, -2),
    ({"eps": math.nan}, -2), ({"qs": 1023}, -2), ({"qos": 1023}, -2), ({"ks": 255}, -2), ({"vs": 255}, -2),
    ({"ko": 0xb0000, "kos": 255}, -2), ({"q": 0x10001}, -2), ({"k": 0x20001}, -2), ({"v": 0x30001}, -2),
    ({"qo": 0x40001}, -2), ({"qn": 0xc0002}, -2), ({"kn": 0xc0001}, -2), ({"pos": 0x50002}, -2), ({"freqs": 0x70004}, -2),
    ({"slots": 0x60004}, -2), ({"kp": 0x90001}, -2), ({"tk": 0, "kp": 0x90002}, -2),
    ({"qo": 0x10000, "qos": 2048}, -2), ({"ko": 0x20000, "kos": 512}, -2),             # in place only row for row
    ({"tk": 8, "D": 80, "n_dims": 80, "Hkv": 2}, -3), ({"n": 0}, 0),
])
def test_kv_write_refused(over, code):
    assert kv_write(**over) == code


def prompt(**over):
    a = dict(q=0x10000, k=0x20000, v=0x30000, type=30, qs=1024, ks=256, vs=256, qsl=0x40000, end=None, T=8, S=2, maxq=6,
             H=8, Hkv=2, D=128, Dv=128, scale=0.1, cap=0.0, causal=1, swa=0, out=0x50000, os=1024)
    a.update(over)
    return _lib.load().iian_pa_prompt_attention(None, a["q"], a["k"], a["v"], a["type"], a["qs"], a["ks"], a["vs"],
                                                a["qsl"], a["end"], a["T"], a["S"], a["maxq"], a["H"], a["Hkv"], a["D"],
                                                a["Dv"], a["scale"], a["cap"], a["causal"], a["swa"], a["out"], a["os"],
                                                None)


@pytest.mark.parametrize("over,code", [
    ({"q": None}, -1), ({"k": None}, -1), ({"v": None}, -1), ({"qsl": None}, -1), ({"out": None}, -1),
    ({"T": -1}, -2), ({"S": -1}, -2), ({"maxq": -1}, -2), ({"maxq": 0}, -2), ({"maxq": 9}, -2), ({"H": 0}, -2),
    ({"H": 7}, -2), ({"Hkv": 0}, -2), ({"D": 0}, -2), ({"Dv": 0}, -2), ({"swa": -1}, -2), ({"cap": -1.0}, -2),
    ({"scale": math.nan}, -2), ({"cap": math.inf}, -2), ({"type": 8}, -3), ({"type": 2}, -3),
    ({"D": 1025, "qs": 9000, "ks": 9000}, -3), ({"qs": 1023}, -2), ({"ks": 255}, -2), ({"vs": 255}, -2),
    ({"os": 1023}, -2), ({"q": 0x10001}, -2), ({"out": 0x50001}, -2), ({"type": 0, "v": 0x30002}, -2),
    ({"end": 0x60002}, -2), ({"T": 1 << 30, "maxq": 1}, -2), ({"T": (1 << 31) - 1, "H": 1, "Hkv": 1, "maxq": 1}, -2),
    ({"T": (1 << 30) - 1, "H": 2, "Hkv": 1, "maxq": 1}, -2), ({"T": 0}, 0), ({"S": 0}, 0),
])
def test_prompt_refused(over, code):
    assert prompt(**over) == code
