"""The build script stops where a source does not compile, also when objects of an earlier build are there."""
import os
import re
import shutil
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_a_source_that_does_not_compile_stops_the_build(tmp_path):
    csrc = tmp_path / "pkg" / "csrc"
    csrc.mkdir(parents=True)
    script = os.path.join(ROOT, "cutile_rs_b200", "csrc", "build.sh")
    shutil.copy(script, csrc)
    names = re.search(r"for src in ([\w ]+);", open(script).read()).group(1).split()
    for n in names:
        (csrc / f"{n}.cu").write_text("")
        (csrc / f"_{n}.o").write_text("old")
    os.utime(csrc / f"{names[0]}.cu", (2e9, 2e9))          # newer than its object
    nvcc = tmp_path / "nvcc"
    for fails, code in (("1", 1), ("0", 0)):
        nvcc.write_text(f'#!/bin/sh\nfor a in "$@"; do [ "$a" = -c ] && exit {fails}; done\nexit 0\n')
        nvcc.chmod(0o755)
        r = subprocess.run(["bash", str(csrc / "build.sh")], env=dict(os.environ, NVCC=str(nvcc)), capture_output=True, text=True)
        assert (r.returncode != 0) == bool(code) and ("built" in r.stdout) == (not code), (r.returncode, r.stdout, r.stderr)
