"""Refusals of the paged serving entry points that need no GPU, beside those of test_paged_cpu.py."""
from types import SimpleNamespace

import pytest

import soc_amd as S
from soc_amd.capi import SOC_ERR_INVALID, lib

SOME = 4096  # an aligned address that is never read


def refused(rc, text):
    msg = lib().soc_last_error().decode()
    assert rc == SOC_ERR_INVALID and text in msg, (rc, msg)


@pytest.mark.parametrize("kw,text", [
    ({"n": 0}, "4096 requests"), ({"page": 24}, "page_size"), ({"max_pages": 0}, "max_pages"), ({"max_rows": 0}, "max_rows"),
    ({"num_pages": 0}, "num_pages"), ({"step_lens": SOME}, "overlap"), ({"step_lens": SOME + 12}, "overlap"),
    ({"step_lens": 2 * SOME - 12}, "overlap"), ({"step_lens": 2 * SOME}, "overlap"), ({"step_lens": SOME + 16}, "null context"),
    ({"step_lens": 2 * SOME - 16}, "null context"), ({"step_lens": None}, "null context"), ({}, "null context"),
])
def test_plan_step_refusals(kw, text):
    a = dict(n=4, page=16, max_pages=8, num_pages=100, max_rows=64, step_lens=3 * SOME)
    a.update(kw)
    refused(lib().soc_paged_plan_step(None, a["n"], SOME, 2 * SOME, a["page"], SOME, a["max_pages"], a["max_pages"], SOME,
                                      a["num_pages"], SOME, SOME, SOME, SOME, SOME, a["max_rows"], SOME, a["step_lens"]), text)


def test_append_with_a_closed_rope():
    """A closed Rope's handle is null, which the library takes as keys stored without rotation."""
    rope = S.Rope.__new__(S.Rope)
    rope.h = None
    with pytest.raises(S.SocError, match="rope is closed") as e:
        S.paged_append(SimpleNamespace(h=None), S.PagedCache(SOME, SOME, 10, 16, 2, 128), rope, None, 0, SOME, 256, SOME, 256,
                       "f32", None, 0, 3, 0, SOME, SOME)
    assert e.value.code == SOC_ERR_INVALID
