"""What makes an object stale: its source, and every header that a source may include."""
import glob
import os
import re

from triton_ssm_b200 import build


def test_every_included_file_counts_as_a_header():
    known = {os.path.realpath(h) for h in build._headers()}
    seen = set()
    for f in glob.glob(os.path.join(build.CSRC, "*")):
        with open(f) as src:
            for name in re.findall(r'^\s*#include "([^"]+)"', src.read(), re.M):
                at = os.path.realpath(os.path.join(build.CSRC, name))
                assert at in known, "%s includes %s, whose edits rebuild nothing" % (os.path.basename(f), name)
                seen.add(at)
    assert len(seen) >= 5


def test_a_newer_header_makes_an_object_stale(tmp_path):
    src, obj = tmp_path / "a.cu", tmp_path / "a.o"
    src.write_text("")
    obj.write_text("")
    os.utime(src, (100, 100))
    os.utime(obj, (200, 200))
    assert not build._stale(str(src), str(obj), 150.0)
    assert build._stale(str(src), str(obj), 250.0)
