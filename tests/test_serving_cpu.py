"""Refusals of the paged serving entry points that need no GPU, beside those of test_paged_cpu.py."""
import pytest

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
