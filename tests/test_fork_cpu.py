"""The entry points for rows that go on from other rows without a GPU: every refusal of shapes and options (made before a
context is looked at, so a null context answers last), and the device-side index arithmetic on hostile values
(tests/cpp/test_fork_math.cpp, a host program over the header the kernels use)."""
import ctypes as C
import shutil
import subprocess
from pathlib import Path

import pytest

from soc_amd.capi import PagedCacheC, SOC_ERR_INVALID, lib

ROOT = Path(__file__).resolve().parents[1]
SOME = 4096  # an aligned address that is never read


def refused(rc, text):
    msg = lib().soc_last_error().decode()
    assert rc == SOC_ERR_INVALID and text in msg, (rc, msg)


def test_fork_math_program(tmp_path):
    exe = ROOT / "tests" / "cpp" / "test_fork_math"
    if not exe.exists():
        if shutil.which("g++") is None:
            pytest.skip("g++ not available")
        exe = tmp_path / "test_fork_math"
        subprocess.run(["g++", "-O1", "-std=c++17", str(ROOT / "tests/cpp/test_fork_math.cpp"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "fork math ok" in r.stdout, r.stdout + r.stderr


POOL = [({"n": 0}, "4096 rows"), ({"n": -1}, "4096 rows"), ({"n": 4097}, "4096 rows"), ({"page": 24}, "page_size"),
        ({"page": 0}, "page_size"), ({"page": 512}, "page_size"), ({"max_pages": 0}, "max_pages"),
        ({"max_pages": (1 << 18) + 1}, "max_pages"), ({"num_pages": 0}, "num_pages"), ({"num_pages": -5}, "num_pages"),
        ({"num_pages": 1 << 27}, "num_pages"), ({}, "null context")]


@pytest.mark.parametrize("kw,text", POOL)
def test_fork_refusals(kw, text):
    a = dict(n=4, page=16, max_pages=8, num_pages=100)
    a.update(kw)
    refused(lib().soc_paged_fork(None, a["n"], SOME, SOME, SOME, a["page"], SOME, SOME, a["max_pages"], a["max_pages"], SOME,
                                 a["num_pages"], SOME, SOME, SOME, SOME, SOME, SOME, SOME), text)


@pytest.mark.parametrize("kw,text", POOL + [({"num_pages": (1 << 20) + 1}, "2^20 pages"), ({"max_moves": 0}, "2^22 moves"),
                                            ({"max_moves": (1 << 22) + 1}, "2^22 moves")])
def test_compact_refusals(kw, text):
    a = dict(n=4, page=16, max_pages=8, num_pages=100, max_moves=9)
    a.update(kw)
    refused(lib().soc_paged_compact(None, a["n"], SOME, a["page"], SOME, SOME, a["max_pages"], a["max_pages"], SOME, SOME,
                                    a["num_pages"], SOME, SOME, a["max_moves"], SOME, SOME), text)


def cache(**kw):
    d = dict(keys=SOME, values=SOME, page_stride=0, num_pages=10, page_size=16, kv_heads=2, head_dim=128)
    d.update(kw)
    return PagedCacheC(*d.values())


@pytest.mark.parametrize("second,layers,moves,text", [
    ({}, 0, 4, "layers"), ({}, 4097, 4, "layers"), ({}, 2, 0, "moves"), ({}, 2, (1 << 22) + 1, "moves"),
    ({"num_pages": 11}, 2, 4, "one shape"), ({"page_size": 32}, 2, 4, "one shape"), ({"kv_heads": 3}, 2, 4, "one shape"),
    ({"head_dim": 64}, 2, 4, "one shape"), ({"page_size": 48}, 2, 4, "page_size"), ({"head_dim": 96}, 2, 4, "head_dim"),
    ({"kv_heads": 0}, 2, 4, "kv_heads"), ({"page_stride": 8}, 2, 4, "page_stride"), ({"keys": SOME + 8}, 2, 4, "aligned"),
    ({"page_stride": 8192}, 2, 4, "null context"), ({}, 2, 4, "null context"),
])
def test_copy_refusals(second, layers, moves, text):
    c = (PagedCacheC * 2)(cache(), cache(**second))
    refused(lib().soc_paged_copy(None, c, layers, SOME, SOME, moves), text)


def test_copy_needs_caches():
    refused(lib().soc_paged_copy(None, None, 2, SOME, SOME, 4), "null paged cache")


@pytest.mark.parametrize("kw,text", [
    ({"dtype": 2}, "dtype"), ({"groups": 0}, "groups"), ({"beams": 0}, "64 beams"), ({"beams": 65}, "64 beams"),
    ({"groups": 1 << 19}, "2^20 rows"), ({"vocab": 0}, "vocabulary"), ({"vocab": (1 << 20) + 1}, "vocabulary"),
    ({"temperature": float("nan")}, "temperature"), ({"temperature": float("inf")}, "temperature"),
    ({"temperature": 2e30}, "temperature"), ({"temperature": 1e-39}, "temperature"), ({"stops": -1}, "stop tokens"),
    ({"stops": 9}, "stop tokens"), ({"stop_p": None}, "stop tokens"), ({"top": -1}, "top_n"), ({"top": 65}, "top_n"),
    ({"beams": 22, "stops": 2}, "at most 64"), ({"next": None, "top": 0}, "nothing"), ({}, "null context"),
    ({"beams": 22, "stops": 2, "next": None}, "null context"), ({"top": 0}, "null context"),
])
def test_beam_refusals(kw, text):
    a = dict(dtype=0, groups=2, beams=4, vocab=100, temperature=1.0, stops=1, stop_p=(C.c_int32 * 9)(), top=8, next=SOME)
    a.update(kw)
    refused(lib().soc_beam_select(None, SOME, a["dtype"], a["vocab"], a["groups"], a["beams"], a["vocab"], a["temperature"],
                                  SOME, a["stop_p"], a["stops"], a["top"], SOME, SOME, SOME, a["next"], a["next"],
                                  a["next"]), text)


@pytest.mark.parametrize("kw,text", [
    ({"dtype": 2}, "dtype"), ({"n": 0}, "65535 sequences"), ({"n": 65536, "groups": 1}, "65535 sequences"),
    ({"max_pages": 0}, "max_pages"), ({"max_pages": 1 << 27}, "max_pages"), ({"groups": 0}, "groups"),
    ({"groups": 5}, "groups"), ({"n": 5000, "groups": 4097}, "groups"), ({"max_group": 0}, "max_group"),
    ({"max_group": -2}, "max_group"), ({"max_prefix": -1}, "max_prefix"), ({"max_prefix": 129, "max_group": 5}, "null context"),
    ({"q_heads": 0}, "query heads"), ({"q_heads": 5}, "query heads"), ({"q_heads": 34}, "query heads"),
    ({"scale": float("inf")}, "scale"), ({"out": SOME, "out_stride": 513}, "in place"),
    ({"cache": cache(page_size=8)}, "page_size"), ({"cache": None}, "null paged cache"),
    ({"cache": cache(kv_heads=1024), "q_heads": 1024, "n": 1025}, "2^20"), ({}, "null context"),
])
def test_shared_attention_refusals(kw, text):
    a = dict(cache=cache(), dtype=0, max_pages=8, n=4, groups=2, max_group=4, max_prefix=128, q_heads=4, scale=0.0,
             out=2 * SOME, out_stride=512)
    a.update(kw)
    refused(lib().soc_paged_attention_shared(None, C.byref(a["cache"]) if a["cache"] else None, SOME, 512, a["dtype"], SOME,
                                             a["max_pages"], a["max_pages"], SOME, a["n"], SOME, SOME, a["groups"],
                                             a["max_group"], a["max_prefix"], a["q_heads"], a["scale"], a["out"],
                                             a["out_stride"], SOME), text)
