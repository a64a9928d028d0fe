"""Every angle of the scaled rotation tables (kv_append.rope_cos_sin) against
the scalings' formulas, one angle at a time in Python's 64-bit floats; the fp32
entries are within half a step of values up to 2 in size (2^-24), the angles of
up to 4000 within 2^-40."""

import math

import pytest


def _angle(kind, j, dim, base, factor, original, low=1.0, high=4.0, slow=1.0, fast=32.0):
    """The j-th angle per position."""
    if kind == "base":
        base *= factor ** (dim / (dim - 2))
    f = base ** (-2 * j / dim)
    if kind == "linear":
        return f / factor
    if kind == "bands":
        wave = 2 * math.pi / f
        if wave < original / high:
            return f
        if wave > original / low:
            return f / factor
        part = (original / wave - low) / (high - low)
        return (1 - part) * f / factor + part * f
    if kind == "yarn":
        # index of the angle that makes n turns in `original` positions:
        # original base^(-2 i / dim) = 2 pi n
        index = [dim / 2 * math.log(original / (2 * math.pi * n), base) for n in (fast, slow)]
        first, last = max(0, math.floor(index[0])), min(dim - 1, math.ceil(index[1]))
        part = min(1.0, max(0.0, (j - first) / max(last - first, 0.001)))
        return f * (1 - part) + f / factor * part
    return f


@pytest.mark.parametrize("dim,base,factor,original,extra", [
    (64, 10000.0, 8.0, 2048, {}), (128, 10000.0, 4.0, 4096, {}), (128, 500000.0, 8.0, 8192, {}),
    (64, 10000.0, 40.0, 4096, {}), (96, 1000000.0, 1.5, 32768, {}), (16, 10000.0, 16.0, 256, {}),
    (64, 10000.0, 8.0, 64, {}), (128, 50000.0, 32.0, 4096, dict(low=2.0, high=9.0, slow=3.0, fast=17.0))])
@pytest.mark.parametrize("kind", [None, "linear", "base", "bands", "yarn"])
def test_every_scaled_angle(kind, dim, base, factor, original, extra):
    import kv_append

    own = dict(bands=("low", "high"), yarn=("slow", "fast")).get(kind, ())
    extra = {k: v for k, v in extra.items() if k in own}
    scaling = kind and dict(type=kind, factor=factor, original=original, **extra)
    t = kv_append.rope_cos_sin(4001, dim, base=base, scaling=scaling, device="cpu").double()
    gain = 0.1 * math.log(factor) + 1 if kind == "yarn" else 1.0
    angles = [_angle(kind, j, dim, base, factor, original, **extra) for j in range(dim // 2)]
    for p in (0, 1, 7, 300, 4000):
        for j, f in enumerate(angles):
            tol = 2.0 ** -24 * gain + p * f * 2.0 ** -48
            assert abs(t[p, j].item() - gain * math.cos(p * f)) <= tol, (p, j)
            assert abs(t[p, dim // 2 + j].item() - gain * math.sin(p * f)) <= tol, (p, j)
    if kind in ("bands", "yarn"):  # some angles lie between the two ends
        plain = [base ** (-2 * j / dim) for j in range(dim // 2)]
        between = [f for f, g in zip(angles, plain) if g / factor * (1 + 1e-9) < f < g * (1 - 1e-9)]
        assert between or dim == 16 or original == 64
