"""The plan of a batch's shared prefixes (tests/cpp/test_prefix_plan.hip) and the groups of sequences that the host layer
reads together (tests/cpp/test_prefix_groups.cpp), on the host."""
import subprocess

from glint_amd import build


def test_plan_of_shared_prefixes():
    if not build.PLAN_TEST.exists():
        build.build_plan_test()
    out = subprocess.run([str(build.PLAN_TEST)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and "plan ok" in out.stdout, out.stdout + out.stderr


def test_groups_of_sequences():
    if not build.GROUPS_TEST.exists():
        build.build_groups_test()
    out = subprocess.run([str(build.GROUPS_TEST)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and "groups ok" in out.stdout, out.stdout + out.stderr
