"""gla_rope_rows against the formulas in 64 bits."""
import numpy as np
import pytest

import rope_ref
from glint_amd import _lib

pytestmark = pytest.mark.gpu

BANDS = dict(freq_base=500000.0, scaling="bands", factor=8.0, original_ctx=8192, low=1.0, high=4.0)
YARN = dict(scaling="yarn", factor=16.0, original_ctx=4096)


def run(be, x, pos, in_place=False, x_pad=0, out_pad=0, shift=0, **spec):
    """x [rows][heads][d] rotated on the device, through rows x_pad and out_pad floats wider than needed, `shift` floats
    off the allocation's start; what lies between the rows has to stay."""
    n, heads, d = x.shape
    plan = be.create_rope_plan(d, **spec)
    xs, os = heads * d + x_pad, heads * d + (x_pad if in_place else out_pad)
    src = np.full((n, xs), 7.5, np.float32)
    src[:, :heads * d] = x.reshape(n, -1)
    bx = be.buffer(np.concatenate([np.zeros(shift, np.float32), src.reshape(-1)]))
    bo = bx if in_place else be.buffer(np.full(shift + n * os, 7.5, np.float32))

    class At:
        def __init__(self, b):
            self.ptr = type(b.ptr)(b.ptr.value + 4 * shift)

    be.rope_rows(plan, At(bx), n, heads, be.buffer(np.asarray(pos, np.int32)), out=None if in_place else At(bo),
                 x_stride=xs if x_pad else 0, out_stride=os if out_pad else 0)
    be.sync()
    got = bo.download(shift + n * os)[shift:].reshape(n, os)
    assert np.all(got[:, heads * d:] == 7.5)
    return got[:, :heads * d].reshape(x.shape)


def check(got, x, pos, **spec):
    want, tol = rope_ref.rotate(x, pos, **spec)
    err = np.abs(got.astype(np.float64) - want)
    assert np.all(err <= tol), (err / tol).max()
    rot = spec.get("rot_dim") or x.shape[-1]
    assert np.array_equal(got[..., rot:], x[..., rot:])


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("n, heads, d, more", [
    (1, 1, 2, {}), (1, 32, 128, BANDS), (3, 9, 64, {}), (5, 16, 256, dict(rot_dim=96, scaling="linear", factor=4.0)),
    (2, 3, 7, dict(rot_dim=6)), (4, 5, 66, dict(rot_dim=34)), (130, 8, 128, YARN), (2, 2, 256, dict(freq_dim=64, rot_dim=250)),
    (7, 4, 80, dict(rot_dim=20, amplitude=0.5)), (3, 1, 250, {}), (1000, 3, 64, dict(rot_dim=2)), (3, 5, 136, {}), (2, 4, 200, dict(rot_dim=198)), (2, 1, 166, {}),
])
def test_rows_match_the_formula(backend, layout, n, heads, d, more):
    rng = np.random.default_rng(n * 1000 + heads * 10 + d)
    x = rng.standard_normal((n, heads, d)).astype(np.float32)
    pos = rng.integers(-20, 70000, n)
    pos[0] = 0
    spec = dict(layout=layout, **more)
    for kw in ({}, dict(in_place=True), dict(x_pad=8, out_pad=16), dict(x_pad=3, out_pad=1), dict(in_place=True, x_pad=5),
               dict(shift=1)):
        check(run(backend, x, pos, **kw, **spec), x, pos, **spec)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_far_and_extreme_positions(backend, layout):
    pos = np.array([0, 1, -1, 131071, 1 << 20, (1 << 31) - 1, -(1 << 31), 12345678])
    x = np.random.default_rng(3).standard_normal((len(pos), 4, 128)).astype(np.float32)
    check(run(backend, x, pos, layout=layout), x, pos, layout=layout)
    turned = run(backend, x, pos, layout=layout)
    assert np.array_equal(turned[0], x[0])  # position 0 is the identity, bit for bit


def test_quarter_turns_and_octant_borders(backend):
    """Angles at and next to multiples of an eighth turn: divisors that make pair 0 turn by them."""
    turns = np.array([0.125, 0.25, 0.375, 0.5, 0.625, 0.75, 0.875, 1.0, 0.124999, 0.250001])
    x = np.random.default_rng(4).standard_normal((3, 2, 20)).astype(np.float32)
    spec = dict(layout="half", divisors=(1.0 / (turns * 2 * np.pi) * 10000.0 ** (-2 * np.arange(10) / 20)).astype(np.float32))
    check(run(backend, x, [1, 2, 1001], **spec), x, [1, 2, 1001], **spec)


def test_back_and_forth_is_the_identity_to_two_roundings(backend):
    x = np.random.default_rng(5).standard_normal((9, 4, 128)).astype(np.float32)
    pos = np.arange(9) * 997
    there = run(backend, x, pos, layout="half")
    back = run(backend, there, -pos, layout="half")
    # each turn rounds both of a pair's values by half a step at most: 2^-24 of |a| + |b| each
    pair = np.abs(x[..., :64]) + np.abs(x[..., 64:])
    assert np.all(np.abs(back - x) <= 4 * 2.0 ** -24 * np.concatenate([pair, pair], -1))


def test_non_finite_values_stay_in_their_pair(backend):
    x = np.random.default_rng(6).standard_normal((2, 3, 64)).astype(np.float32)
    y = x.copy()
    y[0, 1, 5], y[1, 2, 40], y[1, 0, 63] = np.inf, np.nan, -np.inf  # the last beyond rot_dim
    spec = dict(layout="half", rot_dim=48)
    got, clean = run(backend, y, [3, 4], **spec), run(backend, x, [3, 4], **spec)
    hit = np.zeros(x.shape, bool)
    hit[0, 1, [5, 29]] = hit[1, 2, [40, 16]] = True
    assert not np.isfinite(got[hit]).any()
    assert got[1, 0, 63] == -np.inf
    hit[1, 0, 63] = True
    assert np.array_equal(got[~hit], clean[~hit])


def test_refusals(backend):
    be = backend
    plan = be.create_rope_plan(64)
    b = be.empty(4 * 64 * 2)
    pos = be.buffer(np.zeros(2, np.int32))
    lib, ctx = _lib.lib(), be.ctx

    def call(x=b.ptr, xs=0, out=b.ptr, os=0, n=2, heads=1, p=pos.ptr, plan=plan.handle):
        return lib.gla_rope_rows(ctx, plan, x, xs, out, os, n, heads, p)

    assert call(n=0, x=None) == _lib.GLA_OK
    for kw in (dict(n=-1), dict(heads=0), dict(x=None), dict(out=None), dict(p=None), dict(xs=63), dict(os=63), dict(os=128),
               dict(xs=-64), dict(plan=None), dict(heads=1 << 26)):
        assert call(**kw) == _lib.GLA_ERR_INVALID, kw
    from glint_amd.attn import GpuBackend
    other = GpuBackend(0)
    assert lib.gla_rope_rows(other.ctx, plan.handle, b.ptr, 0, b.ptr, 0, 2, 1, pos.ptr) == _lib.GLA_ERR_INVALID
    theirs = other.create_rope_plan(64)
    other.close()
    assert "destroyed" in (call(plan=theirs.handle) and _lib.last_error())
    theirs.destroy()
    assert call() == _lib.GLA_OK
    be.sync()
