"""What the tcgen05 kernels do when a bounded wait of theirs expires, read from their sources: no wait of the real
kernels runs out in a test."""
from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "parakeet.wgsl_b200" / "csrc"


def _without_comments(text: str) -> str:
    return re.sub(r"//[^\n]*", "", text)


@pytest.mark.parametrize("name", ["gemm_tc.cu", "int4_umma.cu", "joint_logits.cu"])
def test_mmas_are_waited_for_before_tmem_is_given_back(name):
    """Any role may give up, the one that issues the MMAs may be the one that does not: it commits and waits for them
    last of all, under no condition but that it is the issuing thread, in every kernel of the file."""
    text = _without_comments((CSRC / name).read_text())
    kernels = len(re.findall(r"\btmem_dealloc(?:_pair)?\(tmem", text))
    drained = re.findall(r"[;}]\s*tc_commit(?:_pair)?\((?:smem_addr\()?&?drain(?:\[\w+\])?\)?\);\s*"
                         r"mbar_wait_drain\(&?drain(?:\[\w+\])?, 0, p\.status\);", text)
    guarded = re.findall(r"if \(!?(?:good|ok)[^;{]*mbar_wait_drain\(", text)
    if name == "int4_umma.cu":  # the elected lane of each MMA warp
        drained += re.findall(r"if \(leader\) \{\s*tc_commit\(&drain\[pair\]\);\s*mbar_wait_drain\(&drain\[pair\], 0, p\.status\);", text)
    assert kernels >= 1 and len(drained) == kernels and not guarded
