"""Code generation of the 8-bit products, the beam selection and the page kernels (CPU
only): no kernel spills registers to scratch memory, and the products' counted waits."""
import os
import re
from concurrent.futures import ThreadPoolExecutor

import pytest

import test_codegen as cg

pytestmark = pytest.mark.skipif(not os.path.exists(cg.HIPCC), reason="hipcc not found")

UNITS = ("rows_i8.hip", "beam.hip", "pages.hip")


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("asm")
    with ThreadPoolExecutor(3) as ex:
        return dict(zip(UNITS, ex.map(lambda u: cg._asm(u, str(tmp / (u + ".s"))), UNITS)))


def test_no_kernel_uses_scratch(asm):
    for unit, lines in asm.items():
        name, sizes = None, {}
        for line in lines:
            m = re.match(r"^(_Z\w+):", line)
            name = m.group(1) if m else name
            m = re.match(r"^; ScratchSize: (\d+)", line)
            if m:
                sizes[name] = int(m.group(1))
        assert sizes and not any(sizes.values()), {k: v for k, v in sizes.items() if v}
        assert not any(re.search(r"\bscratch_(load|store)", l) for l in lines), unit


def test_no_packed_fp32(asm):
    for unit, lines in asm.items():
        assert not any(re.search(r"\bv_pk_(add|mul|fma)_f32", l) for l in lines), unit
