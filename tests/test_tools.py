"""The static check of prefetches (tools/isa_scan.py): it compiles with the product's flags, and says what the compiler says."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _scan(*args):
    return subprocess.run([sys.executable, os.path.join(ROOT, "tools", "isa_scan.py"), *args], cwd=ROOT, capture_output=True, text=True)


def test_isa_scan_reads_a_kernel_file():
    r = _scan("ttts_amd/csrc/peq.hip")
    assert r.returncode == 0, r.stderr[-2000:]
    r = _scan("ttts_amd/csrc/paged.hip", "--trace", "attn_paged_decode_kernelIDF16bLi64ELi8E")
    assert r.returncode == 0 and "M" in r.stdout and "attn_paged_decode_kernel" in r.stdout, (r.stdout[-500:], r.stderr[-2000:])


def test_isa_scan_shows_the_compilers_message():
    r = _scan("ttts_amd/csrc/no_such_file.hip")
    assert r.returncode != 0 and "no such file" in r.stderr
