"""The status word's code names the wait that gave up: no two waits share one."""
import glob
import os
import re
from collections import defaultdict

from triton_ssm_b200 import build

CODE = re.compile(r"\b(?:fail|atomicExch|wait\w*)\((?:[^()]|\([^()]*\))*?\b([1-9]\d{3})\)")


def test_codes_are_unique():
    found = defaultdict(list)
    for f in sorted(glob.glob(os.path.join(build.CSRC, "*.cu"))):
        with open(f) as src:
            for code in CODE.findall(src.read()):
                found[code].append(os.path.basename(f))
    assert not {c: where for c, where in found.items() if len(where) > 1}
    assert len(found) > 30
