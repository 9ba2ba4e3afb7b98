"""CPU: csrc/build.sh compiles again what its own flags or any header changed, and the library's stamp tells other flags."""
import os
import shutil
import subprocess

from wide_deep_amd import capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_objects_and_stamp_follow_the_flags(tmp_path):
    csrc, tools = tmp_path / "wide_deep_amd" / "csrc", tmp_path / "bin"
    shutil.copytree(os.path.join(ROOT, "wide_deep_amd", "csrc"), csrc, ignore=shutil.ignore_patterns("_obj"))
    shutil.copytree(os.path.join(ROOT, "include"), tmp_path / "include")
    tools.mkdir()
    for name in ("hipcc", "g++", "gcc"):              # writes its output file and a line of what it was asked for
        (tools / name).write_text("#!/bin/sh\necho \"%s $*\" >> %s/log\nwhile [ $# -gt 0 ]; do if [ \"$1\" = -o ]; then : > \"$2\"; fi; shift; done\n" % (name, tmp_path))
        (tools / name).chmod(0o755)

    def build(**env):
        log = tmp_path / "log"
        log.write_text("")
        subprocess.check_call(["sh", str(csrc / "build.sh")], stdout=subprocess.DEVNULL, env=dict(os.environ, PATH="%s:%s" % (tools, os.environ["PATH"]), **env))
        lines = log.read_text().splitlines()
        stamp = (csrc / "_obj" / "build_stamp.cpp").read_text().split('"')[3]
        return [x.split(" -c ")[1].split()[0].rsplit("/", 1)[1] for x in lines if x.startswith("hipcc") and " -c " in x], stamp

    def later(path, was):                              # newer than the objects, whatever the file system's resolution
        at = max(os.stat(f).st_mtime for f in (csrc / "_obj").iterdir()) + 2
        os.utime(path, (at, at))

    every = sorted(f.name for f in csrc.glob("*.hip"))
    first, stamp = build()
    assert sorted(first) == every
    again, same = build()
    assert again == [] and same == stamp
    sh = csrc / "build.sh"
    sh.write_text(sh.read_text().replace("-O3 -std=c++17", "-O2 -std=c++17", 1))
    later(sh, stamp)
    flags, other = build()
    assert sorted(flags) == every and other != stamp
    for f in (csrc / "_obj").iterdir():                # objects as new as what they were made from
        later(f, None)
    later(csrc / "mlp_chain.h", None)
    assert sorted(build()[0]) == every
    assert build(WD_REBUILD="1")[0] != []


def test_the_tree_and_the_script_stamp_alike():
    with open(os.path.join(ROOT, "wide_deep_amd", "csrc", "build.sh")) as f:
        line = [x for x in f if x.startswith("STAMP=")][0]
    got = subprocess.check_output(["sh", "-c", 'HERE="%s"; %s; echo "$STAMP"' % (os.path.join(ROOT, "wide_deep_amd", "csrc"), line.strip())], text=True).strip()
    assert got == capi.source_stamp()
