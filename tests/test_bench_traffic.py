"""CPU: the measured traffic that bench.py reports is that of the sources in this tree, and only the measured layer's sources
can put it out of date."""
import glob
import os
import re
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "ppl.pmx_amd", "csrc")


def bench():
    sys.path.insert(0, ROOT)
    try:
        import bench
    finally:
        sys.path.remove(ROOT)
    return bench


def test_every_recorded_counter_run_is_reported():
    b, n = bench(), 0
    for path in sorted(glob.glob(os.path.join(ROOT, "profiles", "*.txt"))):
        for workload, forms, value in re.findall(r"bench-traffic: workload=(\S+) forms=(\w+) bytes_per_launch=(\d+) ",
                                                 open(path).read()):
            assert b.measured_traffic(workload, forms) == (int(value), os.path.relpath(path, ROOT))
            n += 1
    assert n >= 9 and b.measured_traffic("decode-T32", "none")[0] == 1887085343
    assert b.measured_traffic("decode-T3", "none")[0] is None


def test_the_layer_is_built_from_the_hashed_sources_alone():
    """What its files include is among them, and the other sources are of the operators for training or the device probe."""
    b = bench()
    for name in b.LAYER_SOURCES:
        text = open(os.path.join(CSRC, name)).read()
        assert set(re.findall(r'#include "([^"]+)"', text)) <= set(b.LAYER_SOURCES) | {"opmx_moe.h"}, name
    others = {os.path.basename(p) for p in glob.glob(os.path.join(CSRC, "*.hip")) + glob.glob(os.path.join(CSRC, "*.h"))}
    others -= set(b.LAYER_SOURCES) | {"device_ceilings.hip", "train.h", "linear_step.h"}
    for name in others:
        assert re.search(r'#include "(train|checkpoint8|linear_epilogue)\.h"', open(os.path.join(CSRC, name)).read()), name
