"""CTAs that read one another's shared memory leave their cluster by a barrier that orders those reads (CPU: the sources)."""

from __future__ import annotations

import re

from .conftest import ROOT


def test_no_cluster_is_left_without_order():
    """A relaxed arrive orders no memory: a CTA could exit, and its shared memory go to another block, while a read of it
    whose value nobody waits for is still on its way. Every cluster barrier in the sources releases and acquires."""
    sources = [p for ext in ("*.cu", "*.cuh") for p in (ROOT / "selas_b200" / "csrc").glob(ext)]
    assert any("ld.shared::cluster" in p.read_text() for p in sources)
    for p in sources:
        for op in re.findall(r"barrier\.cluster\.[a-z.]+", p.read_text()):
            assert op in ("barrier.cluster.arrive.release.aligned", "barrier.cluster.wait.acquire.aligned"), (p.name, op)
