"""Rotary positions of given rows (soc_rope_apply) against the formula in 64 bits: both pair layouts, parts of the head,
every scaling, far and negative positions, fp32 and fp16, strided, unaligned and in-place rows, odd sizes.

Tolerance of a rotated value m (a c - b s): the fraction of a turn is rounded to 2^-26 turns and read to about one more
bit (in radians 2 pi 2^-26 + 2^-24), cosine and sine are rounded (2^-24 each, their function good to two steps), the gain,
two products and a sum add four roundings: below 8 * 2^-24 (|a| + |b|) m. The 64-bit angle itself is off by at most four
steps of 2^-53 relative: 2^-50 |position| radians. fp16 results add half a step, 2^-11 relative (or 2^-25)."""
import math

import numpy as np
import pytest

import soc_amd as S
from soc_amd.capi import SOC_ERR_INVALID
from tests.device import NP, Arrays

pytestmark = pytest.mark.gpu


def frequencies(d, theta, scaling, factor, original, fast=32.0, slow=1.0):
    if scaling == "ntk":
        theta *= factor ** (d / (d - 2))
    f = np.array([theta ** (-2.0 * i / d) for i in range(d // 2)])
    if scaling == "linear":
        f = f / factor
    if scaling == "yarn":
        pair = [d * math.log(original / (t * 2 * math.pi)) / (2 * math.log(theta)) for t in (fast, slow)]
        low, high = max(0, math.floor(pair[0])), min(d - 1, math.ceil(pair[1]))
        ramp = np.clip((np.arange(d // 2) - low) / max(high - low, 0.001), 0, 1)
        f = f / factor * ramp + f * (1 - ramp)
    return f


def rotate(x, positions, d, layout, f, gain):
    """x [rows][heads][head_dim] -> (rotated in 64 bits, tolerance of an fp32 result)."""
    x = x.astype(np.float64)
    a = positions.astype(np.float64)[:, None, None] * f
    c, s = np.cos(a) * gain, np.sin(a) * gain
    y, tol = x.copy(), np.zeros_like(x)
    i, j = (slice(0, d // 2), slice(d // 2, d)) if layout == "half" else (slice(0, d, 2), slice(1, d, 2))
    u, v = x[..., i], x[..., j]
    y[..., i], y[..., j] = u * c - v * s, v * c + u * s
    off = (8 * 2.0 ** -24 + np.abs(positions.astype(np.float64))[:, None, None] * 2.0 ** -50) * gain
    tol[..., i] = tol[..., j] = (np.abs(u) + np.abs(v)) * off
    return y, tol


def check(got, want, tol, dtype):
    if dtype == "f16":
        tol = tol + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
    worst = np.max(np.abs(got.astype(np.float64) - want) - tol, initial=-1.0)
    assert worst <= 0, worst


def run(ctx, dtype, rows, heads, hd, d, layout="half", scaling="none", factor=1.0, theta=1e6, original=4096,
        longest=40960, pad=(0, 0), shift=0, in_place=False, use_positions=True, offset=0, gain=0.0, seed=1):
    rng = np.random.default_rng(seed)
    width = heads * hd
    xs, ys = width + pad[0], width + (pad[0] if in_place else pad[1])
    flat = (rng.standard_normal(shift + rows * xs) * 2).astype(NP[dtype])
    x = flat[shift:].reshape(rows, xs)[:, :width].reshape(rows, heads, hd)
    positions = rng.integers(0, longest, rows).astype(np.int32)
    before = np.full(shift + rows * ys, 7.0, NP[dtype])
    with Arrays(ctx) as mem:
        px, pp = mem.up(flat), mem.up(positions)
        py = px if in_place else mem.up(before)
        size = flat.itemsize
        rope = S.Rope(ctx, hd, d, layout=layout, theta=theta, scaling=scaling, factor=factor,
                      original_max_position=original, attention_factor=gain)
        try:
            rope.apply(px + shift * size, py + shift * size, dtype, rows, heads,
                       positions=pp if use_positions else None, offset=offset, x_stride=xs, y_stride=ys)
            out = mem.down(py)
        finally:
            rope.close()
    if not use_positions:
        positions = offset + np.arange(rows)
    m = 1.0 if scaling != "yarn" else gain if gain > 0 else 0.1 * math.log(factor) + 1
    want, tol = rotate(x, positions, d, layout, frequencies(d, theta, scaling, factor, original), m)
    got = out[shift:].reshape(rows, ys)
    check(got[:, :width].reshape(rows, heads, hd), want, tol, dtype)
    # behind each row and before the first one, nothing is written
    rest = flat if in_place else before
    assert np.array_equal(out[:shift], rest[:shift])
    assert np.array_equal(got[:, width:], rest[shift:].reshape(rows, ys)[:, width:])
    if d < hd:
        assert np.array_equal(got[:, :width].reshape(rows, heads, hd)[..., d:], x[..., d:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd,d", [(128, 128), (128, 64), (64, 64), (80, 20), (80, 40), (96, 96), (2, 2), (10, 6), (256, 64),
                                  (1024, 1024)])
def test_layouts_and_parts(gpu_ctx, layout, dtype, hd, d):
    run(gpu_ctx, dtype, 7, 3, hd, d, layout)


@pytest.mark.parametrize("scaling,factor,longest", [("none", 1.0, 100), ("linear", 4.0, 131072), ("ntk", 8.0, 300000),
                                                    ("yarn", 4.0, 131072), ("yarn", 1.0, 4096), ("yarn", 32.0, 1000000)])
def test_scalings(gpu_ctx, scaling, factor, longest):
    run(gpu_ctx, "f32", 33, 5, 128, 128, "half", scaling, factor, longest=longest)
    run(gpu_ctx, "f32", 9, 2, 128, 32, "interleaved", scaling, factor, longest=longest, theta=10000.0, gain=1.3)


@pytest.mark.parametrize("rows,heads", [(1, 1), (1, 40), (2, 17), (257, 8), (1000, 2)])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_sizes(gpu_ctx, rows, heads, dtype):
    run(gpu_ctx, dtype, rows, heads, 128, 128)


@pytest.mark.parametrize("pad,shift", [((0, 4), 0), ((12, 0), 4), ((3, 0), 0), ((0, 5), 0), ((8, 8), 1), ((1, 1), 3)])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_strides_and_alignment(gpu_ctx, pad, shift, dtype, layout):
    run(gpu_ctx, dtype, 11, 3, 128, 96, layout, pad=pad, shift=shift)
    run(gpu_ctx, dtype, 11, 3, 128, 96, layout, pad=pad, shift=shift, in_place=True)


def test_consecutive_positions(gpu_ctx):
    run(gpu_ctx, "f32", 50, 4, 128, 128, use_positions=False, offset=1000)


def test_extreme_positions(gpu_ctx):
    """Negative positions turn backwards; the largest of 32 bits keep their angle."""
    ctx, hd = gpu_ctx, 64
    positions = np.array([-1, -2 ** 31, 2 ** 31 - 1, 0, -40961], np.int32)
    x = np.random.default_rng(3).standard_normal((5, 2, hd)).astype(np.float32)
    with Arrays(ctx) as mem:
        px, py, pp = mem.up(x), mem.up(np.zeros_like(x)), mem.up(positions)
        rope = S.Rope(ctx, hd, theta=10000.0)
        rope.apply(px, py, "f32", 5, 2, positions=pp)
        got = mem.down(py)
        rope.close()
    want, tol = rotate(x, positions, hd, "half", frequencies(hd, 10000.0, "none", 1.0, 0), 1.0)
    check(got, want, tol, "f32")
    assert np.array_equal(got[3], x[3])


def test_agrees_with_the_reference_op(gpu_ctx):
    """Unscaled half pairs at consecutive positions are soc_op_rope, up to its 32-bit tables' rounding."""
    from soc_amd.capi import check as ok, lib
    x = np.random.default_rng(9).standard_normal((21, 6 * 128)).astype(np.float32)
    with Arrays(gpu_ctx) as mem:
        px, pa, pb = mem.up(x), mem.up(np.zeros_like(x)), mem.up(np.zeros_like(x))
        ok(lib().soc_op_rope(gpu_ctx.h, px, pa, 21, 6, 128, 128, 500, 1e6))
        rope = S.Rope(gpu_ctx, 128)
        rope.apply(px, pb, "f32", 21, 6, offset=500)
        a, b = mem.down(pa), mem.down(pb)
        rope.close()
    # each of the two is within 8 * 2^-24 of the pair's two magnitudes
    size = np.abs(x.reshape(21, 6, 2, 64)).sum(2, keepdims=True).repeat(2, 2).reshape(21, -1)
    assert np.max(np.abs(a - b) - size * 16 * 2.0 ** -24) <= 0


def test_bits_do_not_depend_on_the_neighbours(gpu_ctx):
    """A row's result is the same alone, among others, four wide or one wide."""
    x = np.random.default_rng(4).standard_normal((9, 5 * 128)).astype(np.float32)
    pos = np.arange(9, dtype=np.int32) * 1234
    with Arrays(gpu_ctx) as mem:
        px, py, pp = mem.up(x), mem.up(np.zeros_like(x)), mem.up(pos)
        odd = np.zeros(9 * 641 + 1, np.float32)
        odd[1:].reshape(9, 641)[:, :640] = x
        po = mem.up(odd)
        rope = S.Rope(gpu_ctx, 128)
        rope.apply(px, py, "f32", 9, 5, positions=pp)
        whole = mem.down(py)
        rope.apply(po + 4, po + 4, "f32", 9, 5, positions=pp, x_stride=641, y_stride=641)
        narrow = mem.down(po)[1:].reshape(9, 641)[:, :640]
        rope.apply(px + 4 * 640 * 6, py, "f32", 1, 5, positions=pp + 4 * 6)
        alone = mem.down(py)[0]
        rope.close()
    assert np.array_equal(whole.view(np.uint32), narrow.copy().view(np.uint32))
    assert np.array_equal(alone.view(np.uint32), whole[6].view(np.uint32))


def test_operands_are_checked(gpu_ctx):
    x = np.zeros((4, 256), np.float32)
    with Arrays(gpu_ctx) as mem:
        px, py, pp = mem.up(x), mem.up(x), mem.up(np.zeros(3, np.int32))
        rope = S.Rope(gpu_ctx, 128)

        def refused(text, *args, **kw):
            with pytest.raises(S.SocError, match=text) as e:
                rope.apply(*args, **kw)
            assert e.value.code == SOC_ERR_INVALID

        refused("past the end", px, py, "f32", 5, 2)
        refused("past the end", px, py, "f32", 4, 2, x_stride=300)
        refused("past the end", px, py, "f32", 4, 2, y_stride=1 << 39)
        refused("stride", px, py, "f32", 4, 2, x_stride=255)
        refused("stride", px, py, "f32", 4, 2, y_stride=(1 << 40) + 1)
        refused("past the end", px, py, "f32", 4, 2, positions=pp)
        refused("null", 0, py, "f32", 4, 2)
        refused("not in device memory", x.ctypes.data, py, "f32", 4, 2)
        refused("aligned", px + 2, py, "f32", 3, 2)
        refused("aligned", px, py, "f32", 2, 2, positions=pp + 1)
        rope.apply(px, py, "f32", 3, 2, positions=pp)
        gpu_ctx.synchronize()
        rope.close()
