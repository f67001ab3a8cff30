"""A kernel whose bounded wait runs out leaves the wait's number in the device's status word: the numbers of every kernel are its own, and the message
of SB200_ERR_TIMEOUT names the kernel."""
import glob
import os
import re
import subprocess

from spoc_b200.build import CSRC, _nvcc

HARNESS = """#include <stdio.h>
#include <stdlib.h>
#include "internal.hpp"
int main(int argc, char** argv) {
  for (int i = 1; i < argc; ++i) printf("%s\\n", sb200::waiting_kernel(static_cast<int>(strtol(argv[i], nullptr, 16))));
}
"""


def sites():
    """(file, number) of every wait that reports."""
    found = []
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu*"))):
        with open(path) as f:
            found += [(os.path.basename(path), n) for n in re.findall(r"atomicCAS\(\s*(?:\w+(?:\.|->))*status,\s*0,\s*(0x[0-9a-fA-F]+)", f.read())]
    return found


def test_no_two_files_share_a_range():
    ranges = {}
    for name, n in sites():
        ranges.setdefault(int(n, 16) >> 12, set()).add(name)
    assert len(ranges) >= 5 and all(len(files) == 1 for files in ranges.values()), ranges


def test_the_message_names_the_kernel(tmp_path):
    src, exe = tmp_path / "sites.cu", str(tmp_path / "sites")
    src.write_text(HARNESS)
    res = subprocess.run([_nvcc(), "-std=c++17", "-I", CSRC, "-o", exe, str(src)], capture_output=True, text=True, timeout=600)
    assert res.returncode == 0, res.stderr
    found = sites()
    names = subprocess.run([exe] + [n for _, n in found], capture_output=True, text=True, timeout=60, check=True).stdout.splitlines()
    assert len(names) == len(found)
    for (file, n), name in zip(found, names):
        with open(os.path.join(CSRC, file)) as f:
            assert re.search(rf"\b{re.escape(name)}\s*\(", f.read()), f"{file}: {n} is reported as {name}"
