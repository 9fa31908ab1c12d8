"""Every way to compile the library's sources uses the flags of mockingbird_amd/build.py: objects of variant and diagnostics builds are linked
beside the library's own and compared with it (no GPU, and no compiler: hipcc is a stub that records its arguments)."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent

STUB = """#!/usr/bin/env python3
import pathlib, sys
with open({log!r}, "a") as f:
    f.write("\\x1f".join(sys.argv[1:]) + "\\n")
pathlib.Path(sys.argv[sys.argv.index("-o") + 1]).write_bytes(b"")
"""


@pytest.mark.parametrize("script,args", [("build_variant.sh", ["flagtest", "-DSOME_KNOB=1"]), ("build_diag.sh", [])])
def test_scripts_compile_with_the_library_flags(tmp_path, script, args):
    from mockingbird_amd import build
    # the script works in its own copy of the tree: sources and scripts are links, what it builds stays there
    (tmp_path / "mockingbird_amd/csrc").mkdir(parents=True)
    (tmp_path / "tools").mkdir()
    (tmp_path / "tools" / script).write_bytes((ROOT / "tools" / script).read_bytes())
    for f in [*(ROOT / "mockingbird_amd/csrc").glob("*.h*"), ROOT / "mockingbird_amd/build.py"]:
        os.symlink(f, tmp_path / f.relative_to(ROOT))
    for name in build.SOURCES:
        (tmp_path / "mockingbird_amd/csrc" / name).with_suffix(".o").write_bytes(b"")
    log, stub = tmp_path / "calls", tmp_path / "hipcc"
    stub.write_text(STUB.format(log=str(log)))
    stub.chmod(0o755)
    log.write_text("")
    env = dict(os.environ, HIPCC=str(stub), MODULE="maximum_path", PATH=f"{Path(sys.executable).parent}:{os.environ['PATH']}")
    subprocess.run(["bash", str(tmp_path / "tools" / script), *args], check=True, env=env, timeout=100, stdout=subprocess.DEVNULL)
    calls = [line.split("\x1f") for line in log.read_text().splitlines()]
    compiled = [c for c in calls if "-c" in c]
    assert compiled and any("-shared" in c for c in calls)
    for c in compiled:
        at = [i for i in range(len(c)) if c[i:i + len(build.FLAGS)] == build.FLAGS]
        assert at, (script, c)
    for a in args[1:]:
        assert all(a in c for c in compiled)
    if script == "build_diag.sh":  # a library of all modules, not of those that some earlier library had
        assert sorted(Path(c[c.index("-c") + 1]).name for c in compiled) == sorted(build.SOURCES)


def test_recipes_of_the_micro_programs_switch_packed_fp32_off():
    for src in sorted((ROOT / "tools").rglob("*.hip")):
        lines = [line for line in src.read_text().splitlines()[:12] if "hipcc" in line]
        assert all("-packed-fp32-ops" in line for line in lines), (src.name, lines)
