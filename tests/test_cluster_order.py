"""A CTA touches another CTA's shared memory only behind a barrier of the cluster: until then the other need not have started. No run
can be relied on to show it, so it is read from the kernels' sources."""

import re
from pathlib import Path

import pytest

from tests.test_source_order import _body

CSRC = Path(__file__).resolve().parent.parent / "flashrnn_b200" / "csrc"
REMOTE = r"\bmap_to_cta\(|shared::cluster\.f32"      # an address in another CTA, or a store to it
BARRIER = r"\bcluster_(sync_all|wait)\(\)"


def kernels():
    for path in sorted(CSRC.glob("*.cu*")):
        text = path.read_text()
        for m in re.finditer(r"__global__[^;{]*?\b(\w+_kernel)\(", text):
            body = _body(text[m.start():], m.group(1) + "(")
            if re.search(REMOTE, body):
                yield pytest.param(body, id=f"{path.name}:{m.group(1)}")


@pytest.mark.parametrize("body", list(kernels()))
def test_a_cluster_barrier_stands_before_the_first_access_to_another_cta(body):
    barrier = re.search(BARRIER, body)
    assert barrier and barrier.start() < re.search(REMOTE, body).start()


def test_the_sum_over_rows_has_both_halves_of_its_first_barrier():
    """Arrive at the start, wait in front of the store: the loads of the rows lie between."""
    body = _body((CSRC / "column_sum.cuh").read_text(), "column_sum_kernel(")
    arrive, loads, wait, store, last = (body.index(s) for s in ("cluster_arrive();", "part + r * cols", "cluster_wait();", "st.shared::cluster", "cluster_sync_all();"))
    assert arrive < loads < wait < store < last
