"""Code generation of the rotation, the append and the paged attention (CPU only):
no kernel spills registers to scratch memory."""
import os
import re
from concurrent.futures import ThreadPoolExecutor

import pytest

import test_codegen as cg

pytestmark = pytest.mark.skipif(not os.path.exists(cg.HIPCC), reason="hipcc not found")

# kernels of each unit: rope and append by type pair, width and layout; the join by
# batch; attention by head size and page form (5 of two, and two general sizes), rows,
# and parts of the weights (fp16 2, bf16 3)
UNITS = {"rope.hip": 60, "attn.hip": 2, "attn_f16.hip": 48, "attn_bf16.hip": 72}


def test_no_kernel_uses_scratch(tmp_path):
    with ThreadPoolExecutor(4) as ex:
        asm = dict(zip(UNITS, ex.map(lambda u: cg._asm(u, str(tmp_path / (u + ".s"))), UNITS)))
    for unit, lines in asm.items():
        name, sizes = None, {}
        for line in lines:
            m = re.match(r"^(_Z\w+):", line)
            name = m.group(1) if m else name
            m = re.match(r"^; ScratchSize: (\d+)", line)
            if m:
                sizes[name] = int(m.group(1))
        assert len(sizes) == UNITS[unit], (unit, len(sizes))
        assert not any(sizes.values()), {k: v for k, v in sizes.items() if v}
        # (a stack object that is not a spill would show as a scratch access)
        assert not any(re.search(r"\bscratch_(load|store)", l) for l in lines), unit
