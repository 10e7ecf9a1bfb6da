"""Waits inside the experts' kernels that run out, with the kernels' own text compiled by g++: no GPU has to wait for anything."""
import os
import re
import subprocess

import pytest

from tests.test_warp_order_cpu import CHECKS, constant, function, source


def without_asm(text):
    return re.sub(r"asm volatile\((?:[^;\"]|\"[^\"]*\")*\);", "", text)


def run(tmp_path, check, code, *args):
    with open(str(tmp_path / "kernels.inc"), "w") as f:
        f.write(code)
    exe = str(tmp_path / "check")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-g", "-pthread", "-Wno-unknown-pragmas", "-I" + str(tmp_path), "-I" + CHECKS, os.path.join(CHECKS, check), "-o", exe])
    out = subprocess.run([exe] + [str(a) for a in args], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=60)
    assert out.returncode == 0 and out.stdout == "ok\n", out.stdout[:3000]


# the last thread of a team, a warp of it, some of a warp, all of it; a team's first step, or a later one
@pytest.mark.parametrize("thread,step,both", [(127, 0, 0), (96, 1, 0), (77, 2, 1), (0, 1, 0), (127, 3, 1)])
def test_a_team_leaves_together(tmp_path, thread, step, both):
    """Threads that go on alone would wait for ever for those that have left."""
    text = source("experts.cu")
    run(tmp_path, "few_steps_check.cpp", constant("FEW_STAGES", text) + without_asm(function("few_steps", text)), thread, step, both)


@pytest.mark.parametrize("name", ["tensor.cuh", "experts.cu", "logits.cuh", "rows.cuh", "groups.cu"])
def test_arrivals_at_another_cta_order_what_it_reads(name):
    """An mbarrier's arrival is a release for the CTA alone unless it says more: what another CTA of the cluster reads after it is not ordered by that."""
    for arrival in re.findall(r"mbarrier\.arrive[a-z_.:0-9]*", source(name)):
        assert "shared::cluster" not in arrival or ".release.cluster" in arrival, arrival
