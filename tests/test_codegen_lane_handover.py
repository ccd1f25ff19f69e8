"""The 8-bit products' results go from a wave's lanes to its other lanes through LDS (CPU
only: generated code).  LDS keeps the order of a wave's accesses, so what is needed, and
enough, is that the compiler keeps it too: on every path through the code a barrier of the wave
(which is no instruction) or of the workgroup stands between writes and the reads behind them,
and between reads and the next writes."""
import os
import re

import pytest

import test_codegen as cg
from test_codegen_many_rows import _body

pytestmark = pytest.mark.skipif(not os.path.exists(cg.HIPCC), reason="hipcc not found")


def bare_handovers(body):
    """Lines that write what was read last, or read what was written last, on some path
    without a barrier between."""
    label = {m.group(1): i for i, l in enumerate(body) if (m := re.match(r"^(\.?\w+):", l))}
    seen, found, work = set(), set(), [(0, None)]
    while work:
        i, last = work.pop()
        if i >= len(body) or (i, last) in seen:
            continue
        seen.add((i, last))
        line = body[i].strip()
        if re.match(r"; wave barrier|s_barrier", line) or re.match(r"s_waitcnt.*s_barrier", line):
            last = None
        elif m := re.match(r"ds_(read|write)", line):
            if last not in (None, m.group(1)):
                found.add(i)
            last = m.group(1)
        elif m := re.match(r"s_(c?)branch\w*\s+(\S+)", line):
            work.append((label[m.group(2)], last))
            if not m.group(1):
                continue
        elif line.startswith("s_endpgm"):
            continue
        work.append((i + 1, last))
    return [body[i].strip() for i in sorted(found)]


def test_the_search_itself():
    w, r, b = "\tds_write_b32 v0, v1", "\tds_read_b128 v[0:3], v1", "\t; wave barrier"
    assert not bare_handovers([w, b, r, b, w, "\ts_barrier", r])
    assert len(bare_handovers([w, r])) == 1 and len(bare_handovers([w, b, r, w, r])) == 2
    # two paths, of which one has no barrier; a loop whose end meets its start
    assert not bare_handovers([w, "\ts_branch .L1", r, ".L1:", b, r])
    assert len(bare_handovers([w, "\ts_cbranch_vccz .L1", b, ".L1:", r])) == 1
    assert len(bare_handovers([".L0:", w, b, r, "\ts_cbranch_vccz .L0"])) == 1
    assert not bare_handovers([".L0:", w, b, r, b, "\ts_cbranch_vccz .L0"])


def test_lanes_of_the_products(tmp_path):
    lines = cg._asm("rows_i8.hip", str(tmp_path / "rows_i8.s"))
    names = [m.group(1) for l in lines
             if (m := re.match(r"^(_ZN12_GLOBAL__N_111gemm_kernelI\w+):", l))]
    assert len(names) == 15
    for name in names:
        body = _body(lines, name)
        assert sum(bool(re.match(r"\s+ds_write", l)) for l in body) >= 32, name
        found = bare_handovers(body)
        assert not found, (name, len(found), found[:3])
