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


def _body(lines, name):
    at = next(i for i, l in enumerate(lines) if re.match(r"^" + re.escape(name) + r":", l))
    end = next(i for i in range(at, len(lines)) if ".Lfunc_end" in lines[i])
    return lines[at:end]


def test_counted_waits_of_the_products(asm):
    """The products' waits count the DMAs that may stay in flight (the memory counter is in
    order): the compiler must leave each DMA in its half of its step and add no other vector
    memory access before the loop's end."""
    lines = asm["rows_i8.hip"]
    names = [m.group(1) for l in lines
             if (m := re.match(r"^(_ZN12_GLOBAL__N_111gemm_kernelI\w+):", l))]
    assert len(names) == 15  # 5 tiles, 3 output types
    for name in names:
        wm, wn, nwm, nwn = (int(x) for x in re.findall(r"Li(\d+)E", name)[-4:])
        tm, tn, waves = 32 * wm * nwm, 32 * wn * nwn, nwm * nwn
        pairs = min(6, (160 * 1024 // ((tm + tn) * 64) - 1) // 2)
        dma = (tm + tn) // (16 * waves)
        first = (dma + 1) // 2
        body = _body(lines, name)
        waits = [i for i, l in enumerate(body) if re.search(r"s_waitcnt vmcnt\(\d+\)", l)]
        # the fill: `pairs` pairs of steps, of which all but the first may be on their way
        count = lambda a, b: sum(l.rstrip().endswith(" lds") for l in body[a:b])
        n = lambda i: int(re.search(r"vmcnt\((\d+)\)", body[i]).group(1))
        assert count(0, waits[0]) == 2 * pairs * dma, name
        assert n(waits[0]) == 2 * (pairs - 1) * dma, name
        # an odd step: half of a pair before its wait, half behind it
        assert count(waits[0], waits[1]) == 2 * first, name
        assert n(waits[1]) == 2 * (pairs - 2) * dma + 2 * first, name
        assert "lgkmcnt(0)" in body[waits[1]], name
        loop_end = next(i for i in range(waits[1], len(body)) if "s_cbranch" in body[i])
        assert count(waits[1], loop_end) == 2 * (dma - first), name
        start = next(i for i, l in enumerate(body) if l.rstrip().endswith(" lds"))
        other = [l for l in body[start:loop_end]
                 if re.search(r"\b(global|flat|scratch)_|\bbuffer_(load|store|atomic)", l)
                 and not l.rstrip().endswith(" lds")]
        assert not other, (name, other[:3])
        # nothing more is fetched, and every wave waits for what is on its way
        assert count(loop_end, len(body)) == 0, name
        assert any("vmcnt(0) lgkmcnt(0)" in l for l in body[loop_end:]), name
