"""Waits inside the experts' kernels that run out, and what host threads share, with the sources' own text compiled by g++: no GPU has to wait for anything."""
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


# the most steps that a tile has: of the longest operand, of the most entries that the entry points take, all of one expert; a step takes 0.35 to 0.5 us
@pytest.mark.parametrize("steps", [1, 2 ** 15, 4000000, 0x70000000 // 64])
@pytest.mark.parametrize("ns", [350, 500, 2000])
def test_a_tile_of_many_steps_is_waited_for(tmp_path, steps, ns):
    came, broken, seconds = limit_check(tmp_path, steps, ns)
    assert came == 1 and broken == 0 and abs(seconds - steps * ns * 1e-9) < 0.01


@pytest.mark.parametrize("steps", [0, 1, 2 ** 15, 0x70000000 // 64])
def test_a_wait_ends(tmp_path, steps):
    """Two seconds where there is little to wait for, and never more than some minutes."""
    came, broken, seconds = limit_check(tmp_path, steps, -1)
    assert came == 0 and broken == 1 and 1.9 < seconds < 2.2 + steps * 1e-5


def limit_check(tmp_path, steps, ns):
    code = function("bar_wait", source("tensor.cuh").replace("// Waits for a phase", "\n// Waits for a phase"))
    code = re.sub(r"asm volatile\(\"mov.u64 %0, %%globaltimer;\" : \"=l\"\((\w+)\)\);", r"\1 = global_timer();", code)
    with open(str(tmp_path / "kernels.inc"), "w") as f:
        f.write(code)
    exe = str(tmp_path / "check")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-pthread", "-Wno-unknown-pragmas", "-I" + str(tmp_path), "-I" + CHECKS,
                           os.path.join(CHECKS, "wait_limit_check.cpp"), "-o", exe])
    out = subprocess.run([exe, str(steps), str(ns)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=60)
    assert out.returncode == 0, out.stdout
    return tuple(float(v) if "." in v else int(v) for v in out.stdout.split())


def test_takers_wait_for_all_of_a_tiles_steps():
    """The sums of a tile are waited for once: with the limit of its steps."""
    assert re.findall(r"bar_wait\(done [^;]*?broken, ([^)]*)\)", source("experts.cu")) == ["t.steps"]


def test_first_tensor_maps_by_several_threads(tmp_path):
    text = source("experts.cu")
    code = text[text.index("typedef CUresult (*EncodeTiled)"):text.index("enum Form")]
    with open(str(tmp_path / "kernels.inc"), "w") as f:
        f.write(code)
    exe = str(tmp_path / "check")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=thread", "-pthread", "-I" + str(tmp_path), "-I/usr/local/cuda/include",
                           os.path.join(CHECKS, "tensor_map_check.cpp"), "-o", exe])
    out = subprocess.run([exe], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=60)
    assert out.returncode == 0 and out.stdout == "ok\n", out.stdout[:3000]
