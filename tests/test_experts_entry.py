"""CPU suite: entry points of the operators around a router whose host side can be seen without a GPU."""
import os
import re
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def call(body):
    """Runs `body` in a process of its own that sees no GPU, so that nothing is ever launched on the made-up addresses; what it printed."""
    script = "import ctypes as C\nfrom nacho_b200 import _capi\nfrom nacho_b200._capi import DenseStruct, Fp8Struct, lib\n" + body
    r = subprocess.run([sys.executable, "-c", script], cwd=ROOT, env={**os.environ, "CUDA_VISIBLE_DEVICES": ""}, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.returncode, r.stderr)
    return r.stdout.strip()


def test_a_product_without_experts_returns():
    """Rows of no expert are zeros, also where there are no experts at all: without a GPU the call fails, it does not end the process."""
    assert call("""
a, w, y = Fp8Struct(1, 5, 256, 0, 4096, 8192), Fp8Struct(0, 16, 256, 1, 12288, 16384), DenseStruct(5, 16, 16, 0, 20480)
print(lib.nb200_fp8_product(C.byref(a), C.byref(w), C.c_void_p(24576), C.byref(y), None) == _capi.E_CUDA)
print(lib.nb200_fp8_product(C.byref(a), C.byref(w), None, C.byref(y), None) == _capi.E_BADARG)
""").split() == ["True", "True"]


def rule(name, source="expert_sort.cu"):
    """The definition of a host-side rule, as its source has it."""
    text = open(os.path.join(ROOT, "nacho_b200", "csrc", source)).read()
    text = text[text.index(f"struct {name} {{"):]
    return text[:text.index("\n};") + 4]


def compiled(tmp_path, definitions, body):
    (tmp_path / "rule.cpp").write_text("#include <algorithm>\n#include <cstdint>\n#include <cstdio>\n" + definitions + "\nint main() {" + body + "}")
    subprocess.run(["g++", "-std=c++17", "-o", str(tmp_path / "rule"), str(tmp_path / "rule.cpp")], check=True)
    return subprocess.run([str(tmp_path / "rule")], check=True, capture_output=True, text=True).stdout


@pytest.mark.skipif(not shutil.which("g++"), reason="no host compiler")
def test_tiles_of_an_order_hold_all_entries(tmp_path):
    """All entries have a tile, no tile is one too many, and the tiles' counts fit in where the order's rows go, for any number of experts."""
    entries = [2561, 4096, 4097, 6145, 8193, 2048 * 256, 2048 * 256 + 1, 1 << 23, (1 << 23) + 1, (1 << 24) - 1, (1 << 24) + 1, 1 << 30, (1 << 31) - (1 << 23),
               (1 << 31) - (1 << 23) + 1, (1 << 31) - 1025, (1 << 31) - 1]
    out = compiled(tmp_path, "constexpr int MAX_TILES = 256;\n" + rule("OrderTiles"),
                   "for (long long n : {" + ", ".join(f"{n}ll" for n in entries) + """}) for (int experts : {0, 1, 64, 1280, 2559, 2560, 2561, 4095, 4096}) {
                        OrderTiles c((int32_t)n, experts);
                        printf("%lld %d %d %d %d\\n", n, experts, c.tile, c.tiles, (int)c.narrow());
                    }""")
    lines = out.splitlines()
    assert len(lines) == 9 * len(entries)
    for line in lines:
        n, experts, tile, tiles, narrow = map(int, line.split())
        assert tile % 256 == 0 and 1 <= tiles <= 256 and (tiles - 1) * tile < n <= tiles * tile, line
        assert tiles * experts * (2 if narrow else 4) <= 4 * n and (not narrow or tile < 1 << 16), line
        assert tile == 2048 or tiles > 64 or experts > 2560, line  # no larger than it has to be


def test_an_order_keeps_nothing_between_calls():
    """What a captured graph writes into has to be the graph's own: a pool that grows frees what it had, and two graphs would share it."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(ROOT, "nacho_b200", "csrc", "expert_sort.cu")).read())
    assert not re.search(r"acquire_workspace|acquire_tagged|cudaMalloc", text)


def test_extents_whose_codes_64_bits_do_not_count():
    from nacho_b200._capi import Fp8Struct, lib
    import ctypes as C
    values, scales = (lambda *m: lib.nb200_fp8_value_count(C.byref(Fp8Struct(*m, None, None)))), (lambda *m: lib.nb200_fp8_scale_count(C.byref(Fp8Struct(*m, None, None))))
    most = (1 << 31) - 1
    assert values(1, 9, 129, 0) == 2 * 16 * 128 and scales(1, 9, 129, 0) == 2 * 16
    assert values(3, 130, 129, 1) == 3 * 2 * 136 * 128 and scales(3, 130, 129, 1) == 3 * 2 * 2
    assert values(1, most, most, 0) == (1 << 24) * (1 << 31) * 128 and scales(1, most, most, 0) == (1 << 24) * (1 << 31)
    for m in ((2, most, most, 1), (4096, most, most, 1), (most, most, most, 1), (-1, 1, 1, 1), (2, 1, 1, 0)):
        assert values(*m) == -1 and scales(*m) == -1
    assert values(most, 0, most, 1) == 0 and values(most, most, 0, 1) == 0
