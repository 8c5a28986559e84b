"""Rotary positions in 64 bits, from the formulas, for the tests."""
import math

import numpy as np


def freqs(head_dim, freq_base=10000.0, rot_dim=0, freq_dim=0, scaling="none", factor=1.0, original_ctx=0, low=1.0, high=32.0,
          divisors=None, **_):
    """Radians a position of each pair, pair by pair."""
    rot = rot_dim or head_dim
    fd = freq_dim or rot
    out = []
    for p in range(rot // 2):
        g = freq_base ** (-2.0 * p / fd) / (float(divisors[p]) if divisors is not None else 1.0)
        if scaling == "linear":
            g /= factor
        elif scaling == "bands":
            t = original_ctx * g / (2 * math.pi)
            w = min(1.0, max(0.0, (t - low) / (high - low)))
            g = (1 - w) * g / factor + w * g
        elif scaling == "yarn":
            def e(t):
                return fd * math.log(original_ctx / (2 * math.pi * t)) / (2 * math.log(freq_base))
            a, b = max(math.floor(e(high)), 0), min(math.ceil(e(low)), fd - 1)
            w = 1 - min(1.0, max(0.0, (p - a) / max(b - a, 0.001)))
            g = (1 - w) * g / factor + w * g
        out.append(g)
    return np.array(out)


def amplitude(scaling="none", factor=1.0, amplitude=0.0, **_):
    if amplitude:
        return amplitude
    return 0.1 * math.log(factor) + 1 if scaling == "yarn" and factor > 1 else 1.0


def rotate(x, pos, layout="interleaved", **spec):
    """x [rows][heads][d] at positions [rows]: (f64 result, how far a kernel may be off). A value is rounded once (half a
    step); the angle carries the relative error of the frequency, of the product and of the reduction, a few steps of 64
    bits, and the products one each."""
    x = np.asarray(x, np.float64)
    f = freqs(x.shape[-1], **spec)
    amp = amplitude(**spec)
    n = len(f)
    ang = np.asarray(pos, np.float64)[:, None] * f
    c, s = np.cos(ang)[:, None, :] * amp, np.sin(ang)[:, None, :] * amp
    ia, ib = (np.arange(n), n + np.arange(n)) if layout == "half" else (2 * np.arange(n), 2 * np.arange(n) + 1)
    a, b = x[..., ia], x[..., ib]
    out, tol = x.copy(), np.zeros_like(x)
    out[..., ia], out[..., ib] = a * c - b * s, a * s + b * c
    slack = (np.abs(a) + np.abs(b)) * amp * (np.abs(ang)[:, None, :] + 1) * 2.0 ** -48
    tol[..., ia] = tol[..., ib] = slack
    return out, tol + np.abs(out) * 2.0 ** -24 + 2.0 ** -149
