"""test_gpu_shared_prefix.py's cases with every prefix read apart, the short ones too that gla_decode_shared reads row by row."""
import pytest

from test_gpu_shared_prefix import *  # noqa: F401,F403

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def apart(monkeypatch):
    monkeypatch.setenv("GLA_DECODE_PREFIX", "1")
