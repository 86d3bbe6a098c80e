"""What the kernels' sources must hold to, read from the files (no GPU)."""

import os
import re

from lorafusion_b200.csrc import build


def sources():
    names = [s for s in build.SOURCES if s.endswith(".cu")] + [h for h in build.HEADERS if h.endswith(".cuh")]
    return {n: open(os.path.join(build.HERE, n)).read() for n in names}


def test_arrivals_at_another_cta_are_released_at_cluster_scope():
    """A release at CTA scope orders nothing for a thread of another CTA that waits on the barrier.  A relaxed arrival comes
    right behind its release fence."""
    found = 0
    for name, text in sources().items():
        for m in re.finditer(r'((?:"[^"\n]*"\s*)*)"([^"\n]*mbarrier\.arrive[\w.:]*shared::cluster[^"\n]*)"', text):
            found += 1
            fenced = ".relaxed.cluster." in m[2] and "fence.release.sync_restrict::shared::cta.cluster;" in m[1]
            assert ".release.cluster." in m[2] or fenced, f"{name}: {m.group()}"
    assert found >= 2


def test_barriers_that_another_cta_arrives_at_are_acquired_at_cluster_scope():
    """In the CTA-pair kernel: `full` where the odd CTA's decoded tiles are reported, `tempty` of both CTAs' epilogues."""
    text = sources()["lf_tc.cu"]
    text = text[text.index("tc_gemm_pair_kernel(const __grid_constant__"):]
    text = text[:text.index("\n}\n")]
    waits = re.findall(r"mbar_wait\w*(<\w+>)?\(&(full|tempty)\[", text)
    assert sorted(waits) == [("<kMx4>", "full"), ("<kMx4>", "full"), ("<true>", "tempty")]
