"""The plan of a batch's shared prefixes, on the host (tests/cpp/test_prefix_plan.hip)."""
import subprocess

from glint_amd import build


def test_plan_of_shared_prefixes():
    if not build.PLAN_TEST.exists():
        build.build_plan_test()
    out = subprocess.run([str(build.PLAN_TEST)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and "plan ok" in out.stdout, out.stdout + out.stderr
