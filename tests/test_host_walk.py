"""The walks over the tiles of the ragged products, cut out of the kernels' source and run on the CPU: every tile once, and
the same walk whichever wave of a workgroup is ahead of the others."""
import os
import re
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


def cut(text, *starts):
    """The declarations that begin with `starts` at the start of a line, each to its closing brace or semicolon."""
    out = []
    for start in starts:
        m = re.search(r"^(?:template <[^\n]*>\n)?" + re.escape(start) + r"(?:[^\n]*[;}](?:[ ]*//[^\n]*)?\n|.*?^\};?\n)", text, re.M | re.S)
        assert m, start
        out.append(m.group(0))
    return "".join(out)


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    from prime_moe import build
    tile = open(os.path.join(build.CSRC, "grouped_tile.h")).read()
    kernel = open(os.path.join(build.CSRC, "grouped_kernel.h")).read()
    folder = tmp_path_factory.mktemp("walk")
    (folder / "walk.inc").write_text(
        cut(tile, "constexpr int kThreads", "constexpr int kWaves", "constexpr int kCols")
        + cut(kernel, "constexpr int kMaxGroups", "constexpr int kWalkCols", "struct RowsArgs", "struct WgradArgs",
              "__device__ __forceinline__ int uniform", "__device__ __forceinline__ int group_end", "struct Tile", "struct Walk {",
              "struct Place", "struct WgradWalk"))
    exe = folder / "walk"
    cmd = ["g++", "-std=c++17", "-O1", "-fwrapv", "-I", str(folder), os.path.join(HERE, "host", "walk.cpp"), "-o", str(exe)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-3000:]
    return str(exe)


def test_walks_do_not_depend_on_the_order_of_the_waves(walk):
    res = subprocess.run([walk], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr


def test_walk_over_the_longest_groups(walk):
    """Groups of nearly 2^31 rows: no sum of rows and tiles passes 32 bits."""
    res = subprocess.run([walk, "huge"], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr


def test_slabs_of_the_longest_contractions(tmp_path):
    from prime_moe import build
    tile = open(os.path.join(build.CSRC, "grouped_tile.h")).read()
    (tmp_path / "slabs.inc").write_text(cut(tile, "constexpr int kSlab"))
    member = re.search(r"^    __device__ __forceinline__ void set_length\(.*?^    \}\n", tile, re.M | re.S)
    (tmp_path / "set_length.inc").write_text(member.group(0))
    exe = str(tmp_path / "slabs")
    res = subprocess.run(["g++", "-std=c++17", "-O1", "-fwrapv", "-I", str(tmp_path), os.path.join(HERE, "host", "slabs.cpp"), "-o", exe],
                         capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-3000:]
    res = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0, res.stderr
