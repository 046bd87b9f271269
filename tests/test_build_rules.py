"""The Makefile's own rules: what a change of the compile flags rebuilds, and what `clean` takes away."""
import os
import re
import shutil
import subprocess

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "opensearch-jvector_amd", "csrc")

pytestmark = pytest.mark.skipif(shutil.which("make") is None, reason="needs make")


def make(*args):
    return subprocess.run(["make", "-C", CSRC, *args], capture_output=True, text=True, check=False).stdout


def test_every_object_follows_the_flags():
    """All objects and libraries that are compiled with flags from the Makefile depend on it, so that a change of the flags reaches a tree that was built before."""
    database = make("-np", "all", "stamps")
    needs = {}
    for target, deps in re.findall(r"^(\.\./lib/[\w/]+\.(?:o|so)):(?!=) *(.*)$", database, re.M):
        needs.setdefault(target, set()).update(deps.split())
    objects = {t for t in needs if t.endswith(".o")}
    assert {"../lib/obj/jv_kernels.o", "../lib/obj/jv_kernels_sx.o", "../lib/obj/jv_abi.o", "../lib/obj_stamps/jv_kernels_xb.o"} <= objects and len(objects) >= 30
    for target in sorted(objects | {"../lib/libjvbuild.so", "../lib/libjvbuildgpu.so"}):
        assert "Makefile" in needs[target], target
    for lib in ("libjvgpu.so", "libjvgpu_stamps.so"):
        assert len([d for d in needs["../lib/" + lib] if d in objects]) >= 15


def test_clean_takes_the_objects_too():
    removed = set(make("-n", "clean").split())
    database = make("-np", "all", "stamps")
    for target in re.findall(r"^(\.\./lib/[\w/]+\.(?:o|so)):(?!=)", database, re.M):
        assert target in removed, target
