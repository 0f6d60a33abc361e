"""What no run can show: the scope of the arrivals by which one CTA of a pair hands work to the other. The memory model
orders nothing between two CTAs behind a release that covers one."""
import pathlib
import re

import custom_matmul_kernels_b200

CSRC = pathlib.Path(custom_matmul_kernels_b200.__file__).parent / "csrc"


def test_arrivals_at_another_cta_release_at_cluster_scope():
    """mbarrier.arrive defaults to CTA scope; at a cluster-window address it has to name the cluster's, and either
    releases itself or stands right behind a fence that does."""
    seen = 0
    for path in sorted(CSRC.glob("*.cuh")):
        text = path.read_text()
        for found in re.finditer(r"mbarrier\.arrive[\w.:]*", text):
            op = found.group()
            if "shared::cluster" not in op:
                continue
            seen += 1
            before = re.findall(r'"([\w.:]+);\\n"\s*"$', text[:found.start()])
            fenced = ".relaxed.cluster." in op and before and re.fullmatch(r"fence\.release\.[\w.:]*cluster|fence\.acq_rel\.cluster", before[0])
            assert ".release.cluster." in op or fenced, f"{path.name}: {op}"
    assert seen > 0
