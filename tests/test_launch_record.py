"""The record of what each stream's last launch wrote (tessera_b200/csrc/launch_record.h), compiled by the host compiler."""
import os
import subprocess

from test_attention_plan import ROOT

PROGRAM = """
#include <cstdio>
#include "launch_record.h"
static tsr::LaunchRecord record;
static char memory[1 << 12], streams[32];
// a launch that writes [w, w + wn) and reads [r, r + rn) ahead of its wait (rn 0: nothing)
static void launch(int device, int stream, int w, size_t wn, int r, size_t rn) {
  const void *read = memory + r, *write = memory + w;
  std::printf("%%d", record.next(device, streams + stream, &read, &rn, rn != 0, &write, &wn, 1));
}
int main() { %s }
"""


def allowed(tmp_path, *launches):
    (tmp_path / "p.cpp").write_text(PROGRAM % " ".join("launch(%d, %d, %d, %d, %d, %d);" % x for x in launches))
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", os.path.join(ROOT, "tessera_b200", "csrc"),
                    str(tmp_path / "p.cpp"), "-o", str(tmp_path / "p")], check=True)
    return [c == "1" for c in subprocess.run([str(tmp_path / "p")], check=True, capture_output=True, text=True).stdout]


def test_what_the_last_launch_wrote(tmp_path):
    assert allowed(tmp_path, (0, 1, 100, 50, 0, 0), (0, 1, 500, 10, 149, 1), (0, 1, 500, 10, 100, 50), (0, 1, 700, 10, 509, 8), (0, 1, 0, 10, 510, 8)) == [
        True, False, True, False, True]


def test_streams_are_told_apart_by_device_too(tmp_path):
    assert allowed(tmp_path, (0, 1, 100, 50, 0, 0), (1, 1, 300, 50, 0, 0), (0, 1, 500, 10, 120, 1)) == [True, True, False]


def test_a_stream_that_is_not_on_record(tmp_path):
    """New, or pushed out by others: nothing is read ahead; a launch that reads nothing ahead may start."""
    others = [(0, 2 + i, 1000 + i, 1, 0, 0) for i in range(16)]
    found = allowed(tmp_path, (0, 0, 600, 10, 700, 10), (0, 1, 100, 50, 0, 0), *others, (0, 1, 500, 10, 120, 1), (0, 1, 500, 10, 120, 1))
    assert found == [False, True] + [True] * 16 + [False, True]
