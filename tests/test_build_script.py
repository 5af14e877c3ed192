"""What build.sh compiles again."""
import os
import re
import shutil
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_objects_follow_the_build_script(tmp_path):
    """The flags of every object stand in build.sh: an object that is older than the script is compiled again, like one that is older than its source or a
    header.  (Checked on a copy of the tree, by what the script says that it would compile.)"""
    csrc = tmp_path / "horizonnet_amd" / "csrc"
    (tmp_path / "include").mkdir()
    shutil.copytree(os.path.join(ROOT, "horizonnet_amd", "csrc"), csrc)
    shutil.copy(os.path.join(ROOT, "include", "horizonnet_hip.h"), tmp_path / "include")
    sources = sorted(re.search(r'^SRCS="([^"]*)"', (csrc / "build.sh").read_text(), re.M).group(1).split())
    objects = tmp_path / "objects"
    objects.mkdir()
    for f in list(csrc.iterdir()) + [tmp_path / "include" / "horizonnet_hip.h"]:
        os.utime(f, (1000, 1000))
    for f in sources:
        (objects / (f[:-4] + ".o")).touch()
        os.utime(objects / (f[:-4] + ".o"), (2000, 2000))

    def listed():
        env = dict(os.environ, HN_BUILD_LIST="1", HN_BUILD_OBJ=str(objects), HN_BUILD_OUT=str(tmp_path / "lib.so"))
        done = subprocess.run(["bash", str(csrc / "build.sh")], env=env, capture_output=True, text=True, timeout=60)
        assert done.returncode == 0, done.stderr
        return sorted(done.stdout.split())

    assert listed() == []
    for f, want in (("build.sh", sources), ("seq_common.h", sources), ("dropout.hip", ["dropout.hip"])):
        os.utime(csrc / f, (3000, 3000))
        assert listed() == want
        os.utime(csrc / f, (1000, 1000))
    os.utime(tmp_path / "include" / "horizonnet_hip.h", (3000, 3000))
    assert listed() == sources
    os.utime(tmp_path / "include" / "horizonnet_hip.h", (1000, 1000))
    (objects / "peaks.o").unlink()
    assert listed() == ["peaks.hip"]
