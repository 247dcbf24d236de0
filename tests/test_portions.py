"""Calls too long for one launch (csrc/portions.h): every piece once and in order, up to totals of 2^32 - 1, and no further piece after one that fails."""
import os
import re
import subprocess

from conftest import ROOT

CSRC = os.path.join(ROOT, "nano_b200", "csrc")


def test_portions(tmp_path):
    exe = str(tmp_path / "probe")
    subprocess.run(["g++", "-O1", "-I" + CSRC, os.path.join(ROOT, "tests", "portions_probe.cpp"), "-o", exe], check=True)
    cases = [(0, 5, 0), (1, 5, 0), (5, 5, 0), (6, 5, 0), (3 * 2 ** 30 + 1, 2 ** 30, 0), (2 ** 32 - 1, 2 ** 30, 0), (2 ** 32 - 1, 2 ** 30 // 3, 0), (2 ** 32 - 1, 2 ** 32 - 1, 0), (2 ** 32 - 2, 2 ** 32 - 3, 0), (100, 7, 3)]
    out = subprocess.run([exe], input="\n".join("%d %d %d" % c for c in cases), capture_output=True, text=True, check=True, timeout=20).stdout.split()
    got = [tuple(map(int, out[i:i + 3])) for i in range(0, len(out), 3)]
    assert got == [(7, stop, stop * most) if stop else (0, -(-total // most), total) for total, most, stop in cases]


def test_launches_of_long_calls_are_counted_in_64_bits():
    """The launchers of ops.cu and kv4.cu cut their calls by in_portions and in no other way."""
    for name, calls in (("ops.cu", 3), ("kv4.cu", 1)):
        text = re.sub(r"//.*", "", open(os.path.join(CSRC, name)).read())
        assert len(re.findall(r"\bin_portions\(", text)) == calls, name
        assert not re.search(r"for \(uint32_t (\w+) = 0; \1 < [^;]*(?:rows|\bn|n_pools|\.T); \1 \+= ", text), name
