"""The kernels of layer norm, dropout and dot-product attention keep their registers out of scratch memory: a reload goes through
the counter of the direct loads and would wait for all of them.  Needs the built library and the ROCm LLVM tools, no GPU."""
import os
import re
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tools"))
import scan_code_objects as sco  # noqa: E402

pytestmark = pytest.mark.skipif(not (os.path.exists(sco.LIB) and os.path.exists(os.path.join(sco.LLVM, "llvm-objdump"))),
                                reason="needs the built library and the ROCm LLVM tools")
OURS = re.compile(r"\d(attention_(kernel|dq_kernel|dkv_kernel|join_kernel|dq_join_kernel|dkv_join_kernel)|layer_norm\w*_kernel|dropout_kernel)I?")
# fp32's gradients of more than 96 elements: accumulators, two sets of operands in three parts and a tile on its way do not fit
SPILLED = re.compile(r"attention_d(q|kv)_kernelIfLi128E")


def test_no_scratch_memory_but_in_the_largest_fp32_gradients():
    scratch, _, _ = sco.count_per_kernel(r"\bscratch_(load|store)_")
    ours = {k for k in sco.count_per_kernel(r"\bs_endpgm\b")[0] if OURS.search(k)}
    assert len([k for k in ours if "attention" in k]) >= 50 and len([k for k in ours if "layer_norm" in k]) >= 30, len(ours)
    spilled = {k: scratch[k] for k in ours if k in scratch}
    assert not {k: v for k, v in spilled.items() if not SPILLED.search(k)}, spilled
    assert all(v <= 64 for v in spilled.values()), spilled
