"""CPU test of the library's build: several processes that find it stale at once (ranks of one job importing a fresh tree)."""
import os
import subprocess
import sys
import textwrap

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# stands in for the compiler: writes what it is asked for after a while, and wants the files it links to be there
NVCC = """\
#!/bin/sh
echo "$@" >> "{log}"
out=""; src=""; prev=""
for a in "$@"; do
  if [ "$prev" = "-o" ]; then out="$a"; fi
  case "$a" in *.cu) src="$a";; esac
  prev="$a"
done
if [ -n "$src" ]; then
  case "$src" in *fbev_kernels.cu) sleep {slow};; *) sleep {fast};; esac
else
  for a in "$@"; do case "$a" in *.o) [ -f "$a" ] || {{ echo "missing $a" >&2; exit 1; }};; esac; done
fi
echo made > "$out"
"""

# the build module with its products in another folder; listing a folder takes `pause` seconds, as on a slow file system
CHILD = """\
import os, sys, time
sys.path.insert(0, {root!r})
import importlib
b = importlib.import_module("flashbev_b200.build")
tmp, nvcc, pause = sys.argv[1], sys.argv[2], float(sys.argv[3])
b.PKG_DIR, b.OBJ_DIR, b.LIB_PATH = tmp, os.path.join(tmp, "build"), os.path.join(tmp, "libfbev.so")
b.HASH_PATH = b.LIB_PATH + ".srchash"
b.find_nvcc = lambda: nvcc
listdir = os.listdir
def slow(path):
    time.sleep(pause)
    return listdir(path)
b.os.listdir = slow
print("ready", flush=True)
sys.stdin.readline()
assert b.build() == b.LIB_PATH and not b.is_stale()
"""


def test_processes_that_build_at_once(tmp_path):
    out = tmp_path / "out"
    (out / "build").mkdir(parents=True)
    for stem in ("fbev_kernels", "fbev_query", "fbev_hash"):  # objects of earlier sources, which a build removes
        (out / "build" / f"{stem}.0123456789abcdef.o").write_text("old")
    log, child = tmp_path / "calls", tmp_path / "child.py"
    child.write_text(textwrap.dedent(CHILD.format(root=ROOT)))
    procs = []
    # the second lists the objects after the first has made its quick ones and before that one links; its own take longer
    for name, slow, fast, pause in (("a", 1.5, 0.1, 0.0), ("b", 3, 3, 0.6)):
        nvcc = tmp_path / f"nvcc_{name}"
        nvcc.write_text(NVCC.format(log=log, slow=slow, fast=fast))
        nvcc.chmod(0o755)
        procs.append(subprocess.Popen([sys.executable, str(child), str(out), str(nvcc), str(pause)], stdin=subprocess.PIPE,
                                      stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True))
    for p in procs:
        assert p.stdout.readline() == "ready\n"
    for p in procs:
        p.stdin.write("go\n")
        p.stdin.flush()
    ends = [p.communicate(timeout=120) for p in procs]
    assert [p.returncode for p in procs] == [0, 0], ends
    # each source once and one link: who came second found the library made
    assert len(log.read_text().splitlines()) == 4
    left = sorted(f for f in os.listdir(out / "build") if f.endswith(".o"))
    assert len(left) == 3 and not any("0123456789abcdef" in f for f in left)
