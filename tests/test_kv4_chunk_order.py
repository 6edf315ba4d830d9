"""The barriers of the chunk kernel over the 4-bit cache: every order in which its parts can meet them, walked through on the host with
the phases that the kernel waits for."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_no_order_of_the_chunk_kernels_parts_reads_or_ends_early(tmp_path):
    exe = tmp_path / "kv4_chunk_order_test"
    r = subprocess.run(["/usr/bin/g++", "-std=c++17", "-Wall", "-O1", "-I", os.path.join(ROOT, "litert-lm_b200", "csrc"),
                        os.path.join(ROOT, "tests", "cpp", "kv4_chunk_order_test.cc"), "-o", str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout
