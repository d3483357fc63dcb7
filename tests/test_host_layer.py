"""The whole layer for a few tokens, its kernels included, from the source, on the CPU: no access leaves a buffer or an array, whoever
runs first and however few workgroups run at a time, every wait ends, and the outputs are the layer's."""
import os
import platform
import re
import subprocess

import pytest

from test_host_walk import cut

HERE = os.path.dirname(os.path.abspath(__file__))
pytestmark = pytest.mark.skipif(platform.machine() != "x86_64", reason="its threads change stacks in x86 assembly")


def read(csrc, name):
    text = open(os.path.join(csrc, name)).read()
    return re.sub(r"^#(include|pragma once)[^\n]*\n", "", text, flags=re.M)


def sources(csrc):
    tile, kernel, ring = (read(csrc, n) for n in ("moe_tile.h", "grouped_kernel.h", "moe_ring.h"))
    text = "namespace pmoe {\n"
    text += cut(tile, "__device__ __forceinline__ void wave_lds_order", "__device__ __forceinline__ uint32_t pack2_bf16")
    text += "namespace ring {\n" + cut(ring, "__device__ __forceinline__ const char *uniform_ptr") + "}\n"
    text += "namespace gmm {\n" + cut(kernel, "__device__ __forceinline__ int uniform") + "}\n}\n"
    text += "".join(read(csrc, n) for n in ("int4_tile.h", "route_topk.h", "moe_layer.h", "moe_layer.hip"))
    text, n = re.subn(r"__ballot\(most == kAbsent\)", "divergent_ballot(most == kAbsent)", text)
    assert n == 1
    text = text.replace("__amdgpu_buffer_rsrc_t", "emu_rsrc").replace("__builtin_amdgcn_", "emu_").replace("__hip_atomic_", "emu_hip_")
    text = re.sub(r"\basm(?: volatile)?\(\"[^;]*;", ";", text)
    places = iter(range(3))
    text, n = re.subn(r"__shared__ (?:__attribute__\(\([^;]*?\)\)\) )?(\w+) (\w+)((?:\[\w+\])*);",
                      lambda m: f"typedef {m[1]} Lds{m[2]}{m[3]}; Lds{m[2]} &{m[2]} = emu::shared<Lds{m[2]}>({next(places)});", text)
    assert n == 3 and "__shared__" not in text
    return text


@pytest.fixture(scope="module")
def layer(tmp_path_factory):
    from prime_moe import build
    folder = tmp_path_factory.mktemp("layer")
    (folder / "layer.inc").write_text(sources(build.CSRC))
    clang = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(build.hipcc()))), "llvm", "bin", "clang++")
    exe = str(folder / "layer")
    res = subprocess.run([clang, "-std=c++17", "-O2", "-fwrapv", "-fno-strict-aliasing", "-w", "-fsanitize=bounds", "-fsanitize-trap=bounds", "-I", str(folder),
                          "-I", os.path.join(os.path.dirname(os.path.dirname(build.CSRC)), "include"), os.path.join(HERE, "host", "layer.cpp"), "-o", exe],
                         capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-4000:]
    return exe


BF16, F16 = 1, 2
CASES = [  # group, dtype, T, K, H, E, top_k, experts that everybody takes, compute units, resident workgroups
    (0, BF16, 1, 136, 72, 5, 3, 0, 8, 16),
    (0, BF16, 6, 264, 72, 6, 3, 0, 8, 16),
    (0, BF16, 6, 264, 72, 6, 3, 0, 1, 1),       # one workgroup at a time
    (0, F16, 5, 264, 72, 6, 3, 0, 7, 2),
    (0, F16, 16, 136, 40, 4, 2, 0, 3, 6),
    (0, BF16, 16, 136, 40, 4, 1, 1, 3, 3),      # everybody on one expert
    (0, BF16, 9, 72, 16, 300, 2, 0, 4, 5),
    (0, BF16, 3, 64, 8, 512, 32, 0, 8, 16),
    (0, F16, 16, 40, 8, 160, 10, 0, 16, 3),     # strips of out that workgroups share, wherever a step ends
    (0, BF16, 3, 24, 136, 70, 32, 0, 24, 5),
    (0, BF16, 1, 24, 520, 32, 32, 0, 24, 22),
    (32, BF16, 1, 160, 96, 6, 3, 0, 7, 3),
    (32, BF16, 6, 160, 96, 6, 3, 0, 3, 6),
    (64, F16, 16, 192, 64, 4, 2, 0, 1, 1),
    (128, BF16, 13, 128, 128, 2, 1, 1, 4, 2),
    (32, F16, 5, 64, 3808, 3, 3, 0, 16, 3),
    (64, BF16, 1, 128, 4032, 5, 5, 0, 13, 2),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_layer_on_the_cpu(layer, case):
    for seed in (1, 2):
        res = subprocess.run([layer, *map(str, case), str(seed)], capture_output=True, text=True, timeout=300)
        assert res.returncode == 0, (seed, res.returncode, res.stderr[-500:])


def test_one_token_and_every_number_of_experts(layer):
    """The choice of one token's experts has four forms, by their number."""
    for E, top_k in ((1, 1), (2, 2), (4, 3), (63, 5), (64, 8), (65, 7), (128, 32), (129, 1), (200, 8), (256, 31), (257, 6), (511, 32)):
        res = subprocess.run([layer, "0", str(BF16), "1", "16", "8", str(E), str(top_k), "0", "4", "3", "5"], capture_output=True, text=True, timeout=300)
        assert res.returncode == 0, (E, top_k, res.returncode, res.stderr[-500:])


def test_five_tokens_on_experts_of_4096_by_256(layer):
    """Sizes at which an instrumented copy of the kernel, not this one, has faulted on a GPU."""
    res = subprocess.run([layer, "0", str(F16), "5", "4096", "256", "8", "4", "0", "256", "24", "3"], capture_output=True, text=True, timeout=600)
    assert res.returncode == 0, (res.returncode, res.stderr[-500:])
