# SPDX-License-Identifier: Apache-2.0
"""The built kernels keep the distance that a matrix instruction's result needs.

Its registers may be read (or written) by another kind of instruction only some wait states
after it: 7 for the products of 16 x 16, of four passes, 11 for those of 32 x 32, of eight
(CDNA3 and CDNA4 instruction set guides, manually inserted wait states).  The compiler sees
to it, but has been seen to keep 3 where the reader stands behind a branch whose other side
is long; what it read then was wrong now and then, which tests of results see only by luck.
So every path from every matrix instruction of the library is searched here, without a GPU.
"""

from __future__ import annotations

import re
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

import pytest

from vllm_ascend_quantized_kv_cache.ops import _native

OBJDUMP = Path("/opt/rocm/llvm/bin/llvm-objdump")
_REGISTER = re.compile(r"\b([av])(?:(\d+)\b|\[(\d+):(\d+)\])")
_NEED = {"16x16": 7, "32x32": 11}


def _registers(text):
    out = set()
    for file, one, low, high in _REGISTER.findall(text):
        out.update((file, i) for i in (
            (int(one),) if one else range(int(low), int(high) + 1)))
    return out


def _operands(text):
    """The operands of an instruction: commas inside brackets do not part them."""
    return re.split(r",\s*(?![^\[]*\])", text)


def _functions(listing):
    """(name, start, [(operation, operands, address, target's offset or None)]) of a listing."""
    name = None
    for line in listing.splitlines():
        head = re.match(r"([0-9a-f]+) <(\S+)>:", line)
        if head:
            if name:
                yield name, start, code
            name, start, code = head[2], int(head[1], 16), []
        elif line.startswith("\t") and "// " in line:
            text, _, note = line.partition("//")
            operation, _, operands = text.strip().partition(" ")
            target = re.search(r"<[^>]*?(?:\+0x([0-9a-f]+))?>", note) if "branch" in operation else None
            code.append((operation, operands.strip(), int(note.split(":")[0], 16),
                         int(target[1] or "0", 16) if target else None))
    if name:
        yield name, start, code


def short_distances(listing):
    """[(kernel, address of the product, of the reader, states between, states needed)] of the
    results that are touched too early on some path, and the number of products."""
    found, products = [], 0
    for name, start, code in _functions(listing):
        if not any(c[0].startswith("v_mfma") for c in code):
            continue
        index = {c[2] - start: i for i, c in enumerate(code)}
        touched = [set() if c[0].startswith("s_") else _registers(c[1]) for c in code]
        for i, (operation, operands, address, _) in enumerate(code):
            if not operation.startswith("v_mfma"):
                continue
            products += 1
            need = next(n for size, n in _NEED.items() if size in operation)
            result = _registers(_operands(operands)[0])
            best: dict[int, int] = {}
            paths = [(i + 1, 0)]
            while paths:
                p, states = paths.pop()
                while p < len(code) and states < need and best.get(p, need) > states:
                    best[p] = states
                    op, args, at, target = code[p]
                    if op.startswith("v_mfma"):
                        # (sums go on from sums without a wait: the hardware's own)
                        a = _operands(args)
                        if result & (_registers(a[1]) | _registers(a[2])):
                            found.append((name, address, at, states, need))
                        if result & _registers(a[0]):
                            break
                    elif result & touched[p]:
                        found.append((name, address, at, states, need))
                        break
                    if op in ("s_endpgm", "s_setpc_b64"):
                        break
                    states += int(args, 0) + 1 if op == "s_nop" else 1
                    if op == "s_branch":
                        p = index[target]
                        continue
                    if op.startswith("s_cbranch"):
                        paths.append((index[target], states))
                    p += 1
    return found, products


def _listing(gap, nop):
    """A product, a branch over `gap` instructions, and a reader on its far side."""
    lines = ["0000000000001000 <k>:", "\tv_mfma_f32_32x32x16_f16 a[0:15], v[0:3], v[4:7], a[0:15]// 000000001000: 0",
             f"\ts_nop {nop}// 000000001008: 0",
             f"\ts_cbranch_scc1 9// 00000000100C: 0 <k+0x{0x10 + 4 * gap:x}>"]
    lines += [f"\ts_add_u32 s0, s0, s1// {0x1010 + 4 * j:012X}: 0" for j in range(gap)]
    end = 0x1010 + 4 * gap
    return "\n".join([*lines, f"\tv_accvgpr_read_b32 v9, a15// {end:012X}: 0",
                      f"\ts_endpgm// {end + 4:012X}: 0"])


def test_the_search_finds_a_reader_behind_a_branch():
    found, products = short_distances(_listing(20, 1))
    assert products == 1 and [x[3:] for x in found] == [(3, 11)]
    assert short_distances(_listing(20, 9)) == ([], 1)
    assert short_distances(_listing(0, 8))[0][0][3:] == (10, 11)


def test_no_result_is_touched_early(tmp_path):
    library = _native.library_path()
    if not library.exists():
        pytest.skip("libkvq_hip.so not built (run __graft_entry__.build())")
    if not OBJDUMP.exists():
        pytest.skip("no llvm-objdump")
    copy = tmp_path / library.name  # its parts land beside it
    shutil.copy(library, copy)
    subprocess.run([OBJDUMP, "--offloading", copy], check=True, capture_output=True)
    parts = sorted(tmp_path.glob("*gfx950"))
    assert parts
    with ThreadPoolExecutor(8) as pool:
        listings = list(pool.map(lambda f: subprocess.run(
            [OBJDUMP, "-d", f], check=True, capture_output=True, text=True).stdout, parts))
    total = 0
    for listing in listings:
        found, products = short_distances(listing)
        assert not found, found[:5]
        total += products
    assert total > 1000  # the products were there to be searched
