"""The waits of the 8-bit tiles (csrc/fp8_waits.h) on the CPU: the loads of each variant in the order in which the kernel issues
them, and of every barrier that the set read behind it has arrived; and the same of the compiled kernels."""

from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "plm-anon_amd" / "csrc"
SOURCE = """
#include <cstdio>
#include <cstdlib>
#include "fp8_waits.h"
int main(int, char** v) {
  const plm::Fp8TileLoads z{std::atoi(v[1]), std::atoi(v[2]), std::atoi(v[3]), std::atoi(v[4])};
  std::printf("%d", plm::fp8_first_wait(z));
  for (int j = 0; j < 4; ++j) std::printf(" %d", plm::fp8_step_wait(z, j));
}
"""


def _variants():
    """(wavefronts of D and of S, fragments of D and of S, blocks ahead) of every tile that a call can launch."""
    text = (CSRC / "fp8_tile.hip").read_text()
    found = {tuple(map(int, m)) for m in re.findall(r"launch<(\d), (\d), (\d), (\d), (\d), (?:true|false), ", text)}
    assert len(found) >= 5
    return sorted(found)


@pytest.fixture(scope="module")
def waits(tmp_path_factory):
    compiler = shutil.which("g++") or shutil.which("clang++") or shutil.which("amdclang++")
    if compiler is None:
        pytest.skip("no host C++ compiler")
    folder = tmp_path_factory.mktemp("waits")
    (folder / "waits.cpp").write_text(SOURCE)
    subprocess.run([compiler, "-std=c++17", f"-I{CSRC}", str(folder / "waits.cpp"), "-o", str(folder / "waits")], check=True,
                   capture_output=True)

    def call(*sizes):
        first, *steps = map(int, subprocess.run([str(folder / "waits"), *map(str, sizes)], check=True, capture_output=True,
                                                text=True).stdout.split())
        return first, steps

    return call


def _uncovered(fd, fs, staged, ahead, first, steps, groups=4):
    """Barriers (0 the first of all, then one a step) behind which a set is read that may not have arrived."""
    sent = ["scale"] * (fd + fs) + ["d"] * (2 * fd * ahead) + [block for block in range(3) for _ in range(staged)]
    missing, barrier, arrived = [], 0, 0

    def wait(allowed):
        nonlocal barrier, arrived
        arrived = max(arrived, len(sent) - allowed)
        if barrier in sent[arrived:]:          # the set of block `barrier` is read behind barrier `barrier`
            missing.append(barrier)
        barrier += 1

    wait(first)
    for step in range(4 * groups):
        j = step % 4
        if j == 3:
            sent += ["scale"] * fd
        for t in range(fs):
            if t == fs // 2:
                wait(steps[j])
            if j == 3:
                sent.append("scale")
            half = t % (fs // 2)
            pieces = 2 * fd if t < fs // 2 else staged
            of_t = (half + 1) * 2 * pieces // fs - half * 2 * pieces // fs
            sent += ["d" if t < fs // 2 else step + 3] * of_t
    return missing


@pytest.mark.parametrize("wd,ws,fd,fs,ahead", _variants())
def test_every_set_has_arrived(waits, wd, ws, fd, fs, ahead):
    staged = 2 * ws * fs // (wd * ws)
    first, steps = waits(fd, fs, staged, ahead)
    assert _uncovered(fd, fs, staged, ahead, first, steps) == []
    assert all(0 <= n <= 63 for n in (first, *steps))   # what the instruction holds
    # The replay sees what is wrong: a wait for the first set alone before steps that count two steps' operands, and steps that wait
    # for nothing.
    if ahead == 3:
        assert _uncovered(fd, fs, staged, ahead, 2 * staged, steps) == [1]
    assert _uncovered(fd, fs, staged, ahead, first, [1 << 10] * 4) == list(range(1 if first == 2 * staged else 2, 17))


def _flow(lines):
    """A kernel's loads, waits and barriers from its beginning through its first loop over K, which is gone round twice: the
    instructions between the first barrier and the last backward branch to a label behind it whose body has four barriers."""
    first = next(i for i, line in enumerate(lines) if line.startswith("s_barrier"))
    labels = {line[:-1]: i for i, line in enumerate(lines) if line.endswith(":")}
    for i in range(first, len(lines)):
        m = re.match(r"s_c?branch\w*\s+(\S+)", lines[i])
        if m and labels.get(m.group(1), i) < i:
            body = lines[labels[m.group(1)]:i]
            if sum(line.startswith("s_barrier") for line in body) == 4:
                return lines[:first + 1] + body + body
    raise AssertionError("no loop of four barriers")


def test_the_compiled_kernels_wait(tmp_path):
    from plm_amd import _build

    text = tmp_path / "tile.s"
    subprocess.run([_build.hipcc(), *_build.HIPCC_FLAGS, f"-I{_build.INCLUDE}", f"-I{_build.CSRC}", "-S", "--cuda-device-only",
                    str(CSRC / "fp8_tile.hip"), "-o", str(text)], check=True, capture_output=True)
    kernels = re.findall(r"^(\S*tile_kernel\S*):.*?\n(.*?)s_endpgm", text.read_text(), re.S | re.M)
    assert len({name for name, _ in kernels}) >= len(_variants())
    for name, body in kernels:
        wd, ws, _, fs = map(int, re.search(r"tile_kernelILi(\d)ELi(\d)ELi(\d)ELi(\d)E", name).groups())
        staged = 2 * ws * fs // (wd * ws)
        lines = [line.split(";")[0].strip() for line in body.splitlines()]
        flying, sent, arrived, barrier = [], 0, 0, 0
        for line in _flow([line for line in lines if line]):
            if re.match(r"(buffer|global|scratch|flat)_(load|store)", line):
                to_lds = line.endswith(" lds")
                flying.append(to_lds)
                sent += to_lds
            elif (m := re.match(r"s_waitcnt.*vmcnt\((\d+)\)", line)) and int(m.group(1)) < len(flying):
                keep = len(flying) - int(m.group(1))
                arrived += sum(flying[:keep])
                del flying[:keep]
            elif line.startswith("s_barrier"):
                assert sent == staged * (3 + max(barrier - 1, 0)), (name, barrier)
                assert arrived >= staged * (barrier + 1), (name, barrier, arrived)
                barrier += 1
        assert barrier == 9, name
