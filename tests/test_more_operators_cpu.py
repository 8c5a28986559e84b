"""Windows with sinks, shared prefixes and block norms where no device is needed: refusals, the structures' layout, and
which pages a window with sinks touches."""
import ctypes as C
import re
import subprocess
from pathlib import Path

import pytest

from glint_amd import _lib, build

HEADER = (Path(__file__).resolve().parents[1] / "include" / "glint_attn.h").read_text()


def test_null_arguments_are_refused(hip_lib):
    bad = _lib.GLA_ERR_INVALID
    assert hip_lib.gla_decode_sinks(None, None, 1) == bad
    assert hip_lib.gla_decode_sinks(None, C.byref(_lib.DecodeArgs()), 1) == bad
    assert hip_lib.gla_prefill_sinks(None, None, 1) == bad
    assert hip_lib.gla_prefill_sinks(None, C.byref(_lib.PrefillArgs()), 1) == bad
    assert hip_lib.gla_decode_shared(None, None) == bad
    assert hip_lib.gla_decode_shared(None, C.byref(_lib.DecodeSharedArgs())) == bad
    assert hip_lib.gla_block_norm(None, None) == bad
    assert hip_lib.gla_block_norm(None, C.byref(_lib.BlockNormArgs())) == bad


def test_a_negative_number_of_sinks_is_refused(hip_lib):
    for fn, args in ((hip_lib.gla_decode_sinks, _lib.DecodeArgs()), (hip_lib.gla_prefill_sinks, _lib.PrefillArgs())):
        assert fn(None, C.byref(args), -1) == _lib.GLA_ERR_INVALID
        assert "n_sinks" in _lib.last_error()


@pytest.mark.parametrize("name, mirror", [("gla_decode_shared_args", _lib.DecodeSharedArgs),
                                          ("gla_block_norm_args", _lib.BlockNormArgs)])
def test_structures_have_the_headers_fields(name, mirror):
    body = HEADER[HEADER.index(f"typedef struct {name}"):HEADER.index(f"}} {name};")]
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = [n for decl in re.findall(r"([\w\s*,]+);", body) for n in re.findall(r"(\w+)\s*(?:,|$)", decl.strip())]
    assert names == [f for f, _ in mirror._fields_]


def test_pages_of_a_window_with_sinks():
    """Every page that holds a seen position, once and in order, and no other: the C++ rule against every position."""
    if not build.PAGES_TEST.exists():
        build.build_pages_test()
    out = subprocess.run([str(build.PAGES_TEST)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and "pages ok" in out.stdout, out.stdout + out.stderr
