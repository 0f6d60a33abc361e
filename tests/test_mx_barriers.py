"""What no run can show: the scope of the arrivals by which one CTA of a pair hands work to the other. The memory model
orders nothing between two CTAs behind a release that covers one."""
import pathlib
import re

import custom_matmul_kernels_b200

CSRC = pathlib.Path(custom_matmul_kernels_b200.__file__).parent / "csrc"


def arrivals(pattern):
    """(file, instruction, whether it releases at cluster scope: itself, or relaxed right behind a fence that does)."""
    for path in sorted(CSRC.glob("*.cuh")):
        text = path.read_text()
        for found in re.finditer(pattern, text):
            op = found.group()
            before = re.findall(r'"([\w.:]+);\\n"\s*"$', text[:found.start()])
            fenced = ".relaxed." in op and before and re.fullmatch(r"fence\.release\.[\w.:]*cluster|fence\.acq_rel\.cluster", before[0])
            yield path.name, op, bool(fenced)


def test_arrivals_at_another_cta_release_at_cluster_scope():
    """mbarrier.arrive defaults to CTA scope; at a cluster-window address it has to name the cluster's, and either
    releases itself or stands right behind a fence that does."""
    found = [a for a in arrivals(r"mbarrier\.arrive[\w.:]*") if "shared::cluster" in a[1]]
    assert found
    for name, op, fenced in found:
        assert ".release.cluster." in op or (".relaxed.cluster." in op and fenced), f"{name}: {op}"


def test_cluster_barriers_release():
    """Behind a cluster's barrier its CTAs write, read or give up shared memory that others have read or written."""
    found = list(arrivals(r"barrier\.cluster\.arrive[\w.:]*"))
    assert found
    for name, op, fenced in found:
        assert ".relaxed" not in op or fenced, f"{name}: {op}"
