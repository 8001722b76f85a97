"""The library's sources by themselves."""
import collections
import glob
import os
import re

import mcw_cppamp_torch_b200 as gt

CSRC = os.path.join(os.path.dirname(gt.__file__), "csrc")


def test_a_type_has_one_definition():
    """Types of two files share a namespace, so that two of one name would break the rule of one definition."""
    where = collections.defaultdict(set)
    for path in glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h")):
        with open(path) as f:
            for name in re.findall(r"^(?:template <[^{};]*> ?)?(?:struct|class|union|enum) (\w+)[^;(]*\{", f.read(), re.M):
                where[name].add(os.path.basename(path))
    assert len(where) > 50
    assert not {n: sorted(f) for n, f in where.items() if len(f) > 1}
