"""Rotary specifications, the append's and the 4-bit weights' refusals, and the structures' layout: no device needed."""
import ctypes as C
import re
from pathlib import Path

import numpy as np
import pytest

import rope_ref
from glint_amd import _lib
from glint_amd.attn import rope_freqs

HEADER = (Path(__file__).resolve().parents[1] / "include" / "glint_attn.h").read_text()

SPECS = [
    dict(head_dim=128),
    dict(head_dim=64, freq_base=500000.0, rot_dim=32),
    dict(head_dim=96, rot_dim=50, freq_dim=96),
    dict(head_dim=128, scaling="linear", factor=4.0),
    dict(head_dim=128, freq_base=500000.0, scaling="bands", factor=8.0, original_ctx=8192, low=1.0, high=4.0),
    dict(head_dim=128, scaling="yarn", factor=16.0, original_ctx=4096, low=1.0, high=32.0),
    dict(head_dim=64, scaling="yarn", factor=0.5, original_ctx=1, low=1.0, high=2.0),  # no pair turns even once
    dict(head_dim=2, scaling="yarn", factor=2.0, original_ctx=100, low=1.0, high=2.0),
    dict(head_dim=256, rot_dim=64, divisors=np.linspace(1, 8, 32, dtype=np.float32)),
    dict(head_dim=128, amplitude=1.25),
]


@pytest.mark.parametrize("spec", SPECS, ids=lambda s: "-".join(f"{v}" for k, v in s.items() if k != "divisors"))
def test_frequencies_are_the_formulas(hip_lib, spec):
    f, amp = rope_freqs(**spec)
    want = rope_ref.freqs(**spec)
    assert f.shape == want.shape
    # pow, the divisions and the blend: a few roundings of 64 bits (the exponent of pow adds its own)
    assert np.abs(f - want).max() <= 1e-13 * want.max()
    assert np.all(np.abs(f - want) <= 1e-12 * want)
    assert amp == pytest.approx(rope_ref.amplitude(**spec), rel=1e-15)


def test_bands_and_yarn_end_at_both_frequencies(hip_lib):
    base, _ = rope_freqs(head_dim=128)
    for rule in ("bands", "yarn"):
        f, _ = rope_freqs(head_dim=128, scaling=rule, factor=8.0, original_ctx=4096, low=1.0, high=32.0)
        assert f[0] == base[0] and f[-1] == pytest.approx(base[-1] / 8, rel=1e-14)
        assert np.all(f <= base * (1 + 1e-14)) and np.all(f >= base / 8 * (1 - 1e-14))


@pytest.mark.parametrize("bad", [
    dict(head_dim=0), dict(head_dim=-2), dict(head_dim=257), dict(head_dim=7), dict(head_dim=64, rot_dim=66),
    dict(head_dim=64, rot_dim=31), dict(head_dim=64, rot_dim=-2), dict(head_dim=64, freq_dim=-1),
    dict(head_dim=64, freq_base=0.0), dict(head_dim=64, freq_base=-1.0), dict(head_dim=64, freq_base=float("nan")),
    dict(head_dim=64, freq_base=float("inf")), dict(head_dim=64, scaling="linear", factor=0.0),
    dict(head_dim=64, scaling="linear", factor=float("nan")), dict(head_dim=64, scaling="bands", factor=2.0),
    dict(head_dim=64, scaling="bands", factor=2.0, original_ctx=100, low=4.0, high=4.0),
    dict(head_dim=64, scaling="bands", factor=2.0, original_ctx=100, low=float("nan"), high=4.0),
    dict(head_dim=64, scaling="yarn", factor=2.0, original_ctx=100, low=0.0, high=4.0),
    dict(head_dim=64, scaling="yarn", factor=2.0, original_ctx=100, freq_base=1.0),
    dict(head_dim=64, amplitude=-1.0), dict(head_dim=64, amplitude=float("inf")),
    dict(head_dim=8, divisors=np.array([1, 0, 1, 1], np.float32)),
    dict(head_dim=8, divisors=np.array([1, np.nan, 1, 1], np.float32)),
    dict(head_dim=64, freq_base=1e-300, freq_dim=2),
], ids=str)
def test_bad_specifications_are_refused(hip_lib, bad):
    with pytest.raises(_lib.GlaError) as e:
        rope_freqs(**bad)
    assert e.value.code == _lib.GLA_ERR_INVALID


def test_an_odd_head_rotated_in_part_is_a_specification(hip_lib):
    f, _ = rope_freqs(head_dim=7, rot_dim=6)
    assert len(f) == 3


def test_null_arguments_are_refused(hip_lib):
    out = C.c_void_p()
    bad = _lib.GLA_ERR_INVALID
    assert hip_lib.gla_rope_freqs(None, None, None) == bad
    assert hip_lib.gla_rope_plan_create(None, None, C.byref(out)) == bad
    assert hip_lib.gla_rope_rows(None, None, None, 0, None, 0, 1, 1, None) == bad
    assert hip_lib.gla_kv_append(None, None) == bad
    assert hip_lib.gla_kv_append(None, C.byref(_lib.AppendArgs())) == bad
    assert hip_lib.gla_kv_read_rows(None, None, None, None, None, 1) == bad
    assert hip_lib.gla_q4w_create(None, 0, None, 1, 32, C.byref(out)) == bad
    assert hip_lib.gla_matvec_q4(None, None, None, 1, None) == bad
    assert hip_lib.gla_q4w_rows(None) == -1 and hip_lib.gla_q4w_cols(None) == -1
    assert hip_lib.gla_rope_plan_destroy(None) == _lib.GLA_OK and hip_lib.gla_q4w_destroy(None) == _lib.GLA_OK


@pytest.mark.parametrize("name, mirror", [("gla_rope_spec", _lib.RopeSpec), ("gla_append_args", _lib.AppendArgs)])
def test_structures_have_the_headers_fields(name, mirror):
    body = HEADER[HEADER.index(f"typedef struct {name}"):HEADER.index(f"}} {name};")]
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = [n for decl in re.findall(r"([\w\s*,]+);", body) for n in re.findall(r"(\w+)\s*(?:,|$)", decl.strip())]
    assert names == [f for f, _ in mirror._fields_]
