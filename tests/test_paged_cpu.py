"""The paged serving entry points without a GPU: every refusal of shapes, types and options (made before a context is
looked at, so a null context answers last), and the device-side index arithmetic on hostile values
(tests/cpp/test_paged_math.cpp, a host program over the header the kernels use)."""
import ctypes as C
import shutil
import subprocess
from pathlib import Path

import pytest

import soc_amd as S
from soc_amd.capi import PagedCacheC, RopeSpecC, SOC_ERR_INVALID, lib

ROOT = Path(__file__).resolve().parents[1]
SOME = 4096  # an aligned address that is never read


def refused(rc, text):
    msg = lib().soc_last_error().decode()
    assert rc == SOC_ERR_INVALID and text in msg, (rc, msg)


def test_paged_math_program(tmp_path):
    exe = ROOT / "tests" / "cpp" / "test_paged_math"
    if not exe.exists():
        if shutil.which("g++") is None:
            pytest.skip("g++ not available")
        exe = tmp_path / "test_paged_math"
        subprocess.run(["g++", "-O1", "-std=c++17", str(ROOT / "tests/cpp/test_paged_math.cpp"), "-o", str(exe)],
                       check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "paged math ok" in r.stdout, r.stdout + r.stderr


# ---- rope ------------------------------------------------------------------------------------------------------------
def spec(**kw):
    d = dict(head_dim=128, rotary_dim=128, layout=0, scaling=0, theta=1e6, factor=1.0, original_max_position=0,
             beta_fast=0.0, beta_slow=0.0, attention_factor=0.0)
    d.update(kw)
    return RopeSpecC(*d.values())


@pytest.mark.parametrize("kw,text", [
    ({"head_dim": 0}, "head_dim"), ({"head_dim": 127}, "head_dim"), ({"head_dim": 2048}, "head_dim"),
    ({"rotary_dim": 0}, "rotary_dim"), ({"rotary_dim": 63}, "rotary_dim"), ({"rotary_dim": 130}, "rotary_dim"),
    ({"layout": 2}, "layout"), ({"layout": -1}, "layout"), ({"scaling": 4}, "scaling"), ({"scaling": -1}, "scaling"),
    ({"theta": 1.0}, "theta"), ({"theta": float("nan")}, "theta"), ({"theta": float("inf")}, "theta"),
    ({"scaling": 1, "factor": 0.5}, "factor"), ({"scaling": 2, "factor": float("nan")}, "factor"),
    ({"scaling": 2, "factor": 2.0, "rotary_dim": 2}, "NTK"), ({"scaling": 3, "factor": 2.0}, "original max position"),
    ({"scaling": 3, "factor": 2.0, "original_max_position": 9, "beta_fast": 1.0, "beta_slow": 2.0}, "beta_fast"),
    ({"scaling": 3, "factor": 2.0, "original_max_position": 9, "beta_fast": 1.0}, "beta_fast"),
    ({"scaling": 3, "factor": 2.0, "original_max_position": 9, "attention_factor": -1.0}, "attention_factor"),
    ({}, "null context"), ({"scaling": 3, "factor": 2.0, "original_max_position": 4096}, "null context"),
])
def test_rope_create_refusals(kw, text):
    h = C.c_void_p(77)
    refused(lib().soc_rope_create(None, C.byref(spec(**kw)), C.byref(h)), text)
    assert h.value is None


def test_rope_null_arguments():
    refused(lib().soc_rope_create(None, None, C.byref(C.c_void_p())), "null argument")
    refused(lib().soc_rope_create(None, C.byref(spec()), None), "null argument")
    assert lib().soc_rope_destroy(None) == 0


@pytest.mark.parametrize("dtype,rows,heads,strides,text", [
    (2, 1, 1, (128, 128), "dtype"), (-1, 1, 1, (128, 128), "dtype"), (0, 0, 1, (128, 128), "rows"),
    (0, -3, 1, (128, 128), "rows"), (0, 1, 0, (128, 128), "heads"), (0, 1, 1, (128, 256), "equal strides"),
    (0, 1, 1, (128, 128), "null rope"),
])
def test_rope_apply_refusals(dtype, rows, heads, strides, text):
    refused(lib().soc_rope_apply(None, SOME, strides[0], SOME, strides[1], dtype, rows, heads, None, 0), text)


# ---- plan ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kw,text", [
    ({"n": 0}, "4096 requests"), ({"n": 4097}, "4096 requests"), ({"n": -1}, "4096 requests"),
    ({"page": 8}, "page_size"), ({"page": 48}, "page_size"), ({"page": 0}, "page_size"), ({"page": 512}, "page_size"),
    ({"max_pages": 0}, "max_pages"), ({"max_pages": (1 << 18) + 1}, "max_pages"), ({"max_rows": 0}, "max_rows"),
    ({"max_rows": (1 << 22) + 1}, "max_rows"), ({"num_pages": 0}, "num_pages"), ({"num_pages": 1 << 27}, "num_pages"),
    ({}, "null context"), ({"n": 4096, "max_rows": 1 << 22, "max_pages": 1 << 18}, "null context"),
])
def test_plan_refusals(kw, text):
    a = dict(n=4, page=16, max_pages=8, num_pages=100, max_rows=64)
    a.update(kw)
    refused(lib().soc_paged_plan(None, a["n"], SOME, SOME, a["page"], SOME, a["max_pages"], a["max_pages"], SOME,
                                 a["num_pages"], SOME, SOME, SOME, SOME, SOME, a["max_rows"], SOME), text)


# ---- append and attention ----------------------------------------------------------------------------------------------
def cache(**kw):
    d = dict(keys=SOME, values=2 * SOME, page_stride=0, num_pages=10, page_size=16, kv_heads=2, head_dim=128)
    d.update(kw)
    return C.byref(PagedCacheC(*d.values()))


BAD_CACHES = [
    ({"page_size": 8}, "page_size"), ({"page_size": 24}, "page_size"), ({"head_dim": 32}, "head_dim"),
    ({"head_dim": 256}, "head_dim"), ({"kv_heads": 0}, "kv_heads"), ({"num_pages": 0}, "num_pages"),
    ({"num_pages": -5}, "num_pages"), ({"num_pages": 1 << 27}, "2^31"), ({"page_stride": 4095}, "page_stride"),
    ({"page_stride": 4100}, "page_stride"), ({"page_stride": -8}, "page_stride"), ({"keys": SOME + 8}, "aligned"),
    ({"values": SOME + 2}, "aligned"),
]


def append(c, dtype=0, rows=3, q_heads=0, q=None, q_out=None, strides=(0, 0)):
    return lib().soc_paged_append(None, c, None, q, strides[0], SOME, 256, SOME, 256, dtype, q_out, strides[1], rows,
                                  q_heads, SOME, SOME)


def attend(c, dtype=0, n=3, max_pages=4, q_heads=4, scale=0.0, out=2 * SOME, out_stride=512):
    return lib().soc_paged_attention_decode(None, c, SOME, 512, dtype, SOME, max_pages, max_pages, SOME, n, q_heads,
                                            scale, out, out_stride, None)


@pytest.mark.parametrize("kw,text", BAD_CACHES)
def test_cache_refusals(kw, text):
    refused(append(cache(**kw)), text)
    refused(attend(cache(**kw)), text)


def test_append_refusals():
    refused(append(None), "null paged cache")
    refused(append(cache(), dtype=3), "dtype")
    refused(append(cache(), rows=0), "rows")
    refused(append(cache(), q_heads=-1), "q_heads")
    refused(append(cache(), q_heads=1 << 17), "q_heads")
    refused(append(cache(), q_heads=4, q=SOME, q_out=2 * SOME), "need a rope")
    refused(append(cache()), "null context")


def test_attention_refusals():
    refused(attend(None), "null paged cache")
    refused(attend(cache(), dtype=2), "dtype")
    refused(attend(cache(), n=0), "sequences")
    refused(attend(cache(), n=65536), "sequences")
    refused(attend(cache(), max_pages=0), "max_pages")
    refused(attend(cache(), max_pages=1 << 27), "max_pages")
    refused(attend(cache(), max_pages=(1 << 26) + 1), "max_pages")
    refused(attend(cache(), max_pages=1 << 26), "null context")
    refused(attend(cache(), q_heads=0), "query heads")
    refused(attend(cache(), q_heads=3), "query heads")
    refused(attend(cache(), q_heads=34), "query heads")
    refused(attend(cache(), scale=float("nan")), "scale")
    refused(attend(cache(), scale=float("inf")), "scale")
    refused(attend(cache(), out=SOME, out_stride=1024), "equal strides")
    refused(attend(cache()), "null context")


# ---- log probabilities -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kw,text", [
    ({"dtype": 2}, "dtype"), ({"rows": 0}, "rows"), ({"vocab": 0}, "vocabulary"), ({"vocab": (1 << 20) + 1}, "vocabulary"),
    ({"top": -1}, "top_n"), ({"top": 65}, "top_n"), ({"vocab": 5, "top": 6}, "top_n"),
    ({"t": float("nan")}, "temperature"), ({"t": float("inf")}, "temperature"), ({"t": 1e-40}, "temperature"),
    ({"tokens": None}, "need tokens"), ({"tokens": None, "logprobs": None}, "nothing"),
    ({}, "null context"), ({"t": -1.0}, "null context"), ({"t": 0.0}, "null context"),
    ({"tokens": None, "logprobs": None, "entropy": SOME}, "null context"),
])
def test_logprobs_refusals(kw, text):
    a = dict(dtype=0, rows=2, vocab=100, t=1.0, tokens=SOME, logprobs=SOME, entropy=None, top=0)
    a.update(kw)
    refused(lib().soc_logprobs(None, SOME, a["dtype"], 100, a["rows"], a["vocab"], a["t"], a["tokens"], a["logprobs"],
                               None, a["entropy"], a["top"], None, None), text)


def test_python_names_are_checked():
    with pytest.raises(KeyError):
        S.Rope(None, 128, layout="quarter")
    with pytest.raises(S.SocError):
        S.Rope(None, 127)
