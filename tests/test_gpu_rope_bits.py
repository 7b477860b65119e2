"""Rotated values have the same bits whatever width they are worked in: 16-bit results are the 32-bit result rounded once
more, in soc_rope_apply and in soc_paged_append, for queries and for cached keys, at every alignment and pair layout.

Exact: rotation in 32 bits is the same operations at every width, and its rounding to 16 bits is the nearest-even one. Half a
million values a case hold some hundred whose 32-bit result lies on a border of the 16-bit rounding."""
import numpy as np
import pytest

import soc_amd as S
from tests.device import NP, Arrays

pytestmark = pytest.mark.gpu

# pairs of head_dim 128 that are worked eight (fp16) or four wide; fp16 four wide; one by one
PARTS = [128, 72, 6]


def rotated(ctx, x, positions, d, layout, dtype, pad=0, shift=0):
    """soc_rope_apply of x [rows][heads][128], rows `pad` elements apart, the first `shift` elements in."""
    rows, heads, hd = x.shape
    row = heads * hd + pad
    flat = np.zeros(shift + rows * row, NP[dtype])
    flat[shift:].reshape(rows, row)[:, : heads * hd] = x.reshape(rows, -1)
    with Arrays(ctx) as mem:
        p, pp = mem.up(flat), mem.up(positions)
        rope = S.Rope(ctx, hd, d, layout=layout)
        rope.apply(p + shift * flat.itemsize, p + shift * flat.itemsize, dtype, rows, heads, positions=pp, x_stride=row,
                   y_stride=row)
        out = mem.down(p)
        rope.close()
    return out[shift:].reshape(rows, row)[:, : heads * hd].reshape(rows, heads, hd)


def differing(a, b):
    return int((a.view(np.uint16) != b.view(np.uint16)).sum())


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d", PARTS)
def test_fp16_rows_are_the_fp32_rows_rounded(gpu_ctx, layout, d):
    rng = np.random.default_rng(d)
    x = rng.standard_normal((2000, 2, 128)).astype(np.float16)
    positions = rng.integers(0, 40960, 2000).astype(np.int32)
    want = rotated(gpu_ctx, x.astype(np.float32), positions, d, layout, "f32").astype(np.float16)
    for pad, shift in ((0, 0), (4, 4), (1, 0), (0, 3)):
        got = rotated(gpu_ctx, x, positions, d, layout, "f16", pad, shift)
        assert differing(got, want) == 0, (pad, shift)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d", PARTS)
def test_cached_keys_are_the_fp32_rows_rounded(gpu_ctx, dtype, layout, d):
    """A position's cached key does not depend on where the projection it came from lies, nor on its type's unit width."""
    rng = np.random.default_rng(d + 1)
    rows, heads, page = 2000, 2, 16
    x = rng.standard_normal((rows, 2 * heads, 128)).astype(np.float16)  # query heads, then key heads
    positions = rng.integers(0, 40960, rows).astype(np.int32)
    full = rotated(gpu_ctx, x.astype(np.float32), positions, d, layout, "f32")
    want = full[:, heads:].astype(np.float16)
    for pad, shift in ((0, 0), (4, 4), (1, 0), (0, 3)):
        row = 2 * heads * 128 + pad
        flat = np.zeros(shift + rows * row, NP[dtype])
        flat[shift:].reshape(rows, row)[:, : row - pad] = x.reshape(rows, -1)
        with Arrays(gpu_ctx) as mem:
            p, pp, ps = mem.up(flat), mem.up(positions), mem.up(np.arange(rows, dtype=np.int32))
            pk, pv = (mem.up(np.zeros((rows // page, heads, page, 128), np.float16)) for _ in range(2))
            pq = mem.up(np.zeros((rows, heads * 128), NP[dtype]))
            rope = S.Rope(gpu_ctx, 128, d, layout=layout)
            at = p + shift * flat.itemsize
            k = at + heads * 128 * flat.itemsize
            S.paged_append(gpu_ctx, S.PagedCache(pk, pv, rows // page, page, heads, 128), rope, at, row, k, row, k, row,
                           dtype, pq, heads * 128, rows, heads, pp, ps)
            keys = mem.down(pk).transpose(0, 2, 1, 3).reshape(rows, heads, 128)
            q = mem.down(pq).reshape(rows, heads, 128)
            rope.close()
        assert differing(np.ascontiguousarray(keys), want) == 0, (pad, shift)
        assert np.array_equal(q, full[:, :heads].astype(NP[dtype])), (pad, shift)
