"""Lanes of a wave that exchange chunks through LDS: what keeps the compiler from moving a read across the stores it depends on,
or a store across the reads of what was there before."""
import os
import re
import subprocess

import pytest

VECTOR = r"<\d+ x \w+>"
EVENT = re.compile(rf"(?P<store>store {VECTOR} .*ptr addrspace\(3\))|(?P<load>load {VECTOR}, ptr addrspace\(3\))|(?P<fence>\bfence |\.s\.barrier|asm sideeffect .*~\{{memory\}})")


def kernels(ir):
    """(name, {block: (its stores, loads and fences of LDS vectors in order, the blocks behind it)}, first block)."""
    for m in re.finditer(r"^define [^\n]*amdgpu_kernel[^\n]*@([^\s(]+)\(.*?^}", ir, re.M | re.S):
        blocks, at = {"entry": ([], [])}, "entry"
        for line in m.group(0).split("\n")[1:]:
            label = re.match(r"([\w.]+):", line)
            if label:
                at = label.group(1)
                blocks[at] = ([], [])
                continue
            event = EVENT.search(line)
            if event:
                blocks[at][0].append(event.lastgroup)
            if re.match(r"\s+(br|switch) |\s+i\d+ -?\d+, label", line):
                blocks[at][1].extend(re.findall(r"label %([\w.]+)", line))
        yield m.group(1), blocks


def unordered(blocks):
    """Whether some way through the kernel leads from a store to a load, or from a load to a store, with no fence in between."""
    reach, todo = {"entry": set()}, ["entry"]
    while todo:
        at = todo.pop()
        before = set(reach[at])
        for event in blocks[at][0]:
            if event == "fence":
                before = set()
            elif before - {event}:
                return True
            else:
                before = {event}
        for to in blocks[at][1]:
            if to not in reach or not before <= reach[to]:
                reach[to] = reach.get(to, set()) | before
                todo.append(to)
    return False


@pytest.mark.parametrize("source", ["quantize_int4.hip", "grouped_int4.hip", "moe_layer.hip", "grouped_mm.hip"])
def test_a_fence_between_stores_and_reads_of_other_lanes_chunks(source, tmp_path):
    """In the optimised code of every kernel: a fence (the workgroup's barrier, assembly that
    touches memory) stands between vectors stored to LDS and vectors
    read from it, in both orders, on every way through the kernel."""
    from prime_moe import build
    out = tmp_path / "kernels.ll"
    res = subprocess.run([build.hipcc(), f"--offload-arch={build.ARCH}", "-O3", "-std=c++17", "-munsafe-fp-atomics", *build.DEVICE_FLAGS,
                          "--cuda-device-only", "-S", "-emit-llvm", os.path.join(build.CSRC, source), "-o", str(out)], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-3000:]
    found = dict(kernels(out.read_text()))
    events = [{e for b in blocks.values() for e in b[0]} for blocks in found.values()]
    assert sum(e >= {"store", "load"} for e in events) >= 12  # (the compiler's text is understood)
    assert [name for name, blocks in found.items() if unordered(blocks)] == []
