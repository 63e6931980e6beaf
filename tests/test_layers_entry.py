"""CPU suite: entry points of gated layers, integer products and clipped gradients whose host side can be seen without a GPU: what they refuse, and rules of theirs."""
import os
import re
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def call(body):
    """Runs `body` in a process of its own that sees no GPU, so that nothing is ever launched on the made-up addresses; what it printed."""
    script = """import ctypes as C
from nacho_b200._capi import DenseStruct as D, Int8Struct as I, SpanStruct as S, lib
from nacho_b200._capi import OK, E_BADARG as BAD, E_UNSUPPORTED as UN, E_CAPACITY as CAP, E_CUDA as CUDA
r = C.byref
""" + body
    r = subprocess.run([sys.executable, "-c", script], cwd=ROOT, env={**os.environ, "CUDA_VISIBLE_DEVICES": ""}, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.returncode, r.stderr)
    return r.stdout.split()


def test_gated_refusals():
    """Dense: rows, columns, stride, type (1: float16, 2: bfloat16), address."""
    assert set(call("""
A = 1 << 20
def go(x=(40, 64, 64, 2, A), w=(32, 64, 64, 2, A), groups=1, offsets=None, act=0, h=(40, 16, 16, 2, A), both=None, scratch=None, bytes=0):
    return lib.nb200_gated_product(r(D(*x)), r(D(*w)), groups, offsets, act, r(D(*h)), r(D(*both)) if both else None, scratch, bytes, None)
print(go() == CUDA)                                     # only the missing GPU stops it
print(go(x=(40, 64, 64, 0, A), w=(32, 64, 64, 0, A), h=(40, 16, 16, 0, A)) == BAD)
print(go(w=(32, 64, 64, 1, A)) == BAD)
print(go(w=(33, 64, 64, 2, A)) == BAD)                  # as many gates as values
print(go(w=(34, 64, 64, 2, A), groups=2) == BAD)        # not in two groups
print(go(w=(64, 64, 64, 2, A), groups=2, h=(40, 16, 16, 2, A)) == BAD)  # groups without offsets
print(go(x=(40, 65, 65, 2, A)) == BAD)
print(go(h=(40, 17, 17, 2, A)) == BAD, go(h=(39, 16, 16, 2, A)) == BAD, go(h=(40, 16, 16, 1, A)) == BAD)
print(go(act=2) == BAD, go(act=-1) == BAD, go(groups=-1) == BAD)
print(go(x=(40, 64, 64, 2, A + 1)) == BAD, go(x=(40, 64, 64, 2, None)) == BAD)
print(go(both=(40, 31, 31, 2, A)) == BAD, go(both=(40, 32, 33, 2, A)) == BAD, go(both=(40, 32, 32, 1, A)) == BAD)
print(go(w=(2 * 4097, 64, 64, 2, A), groups=4097, offsets=C.c_void_p(A), h=(40, 1, 1, 2, A)) == UN)
# rows that the copy engine cannot read are copied, for which there has to be room
odd, need = dict(x=(400, 63, 63, 2, A), w=(32, 63, 63, 2, A), h=(400, 16, 16, 2, A)), 400 * 64 * 2 + 32 * 64 * 2
print(lib.nb200_gated_product_scratch(r(D(*odd["x"])), r(D(*odd["w"])), 1) == need)
print(go(**odd) == BAD, go(**odd, scratch=C.c_void_p(A + 8), bytes=need) == BAD, go(**odd, scratch=C.c_void_p(A), bytes=need - 1) == CAP, go(**odd, scratch=C.c_void_p(A), bytes=need) == CUDA)
print(lib.nb200_gated_product_scratch(r(D(400, 64, 64, 2, A)), r(D(32, 64, 64, 2, A)), 1) == 0, lib.nb200_gated_product_scratch(r(D(4, 63, 63, 2, A)), r(D(32, 63, 63, 2, A)), 1) == 0)
print(lib.nb200_gated_product_scratch(r(D(-1, 64, 64, 2, A)), r(D(32, 64, 64, 2, A)), 1) == -1, lib.nb200_gated_product_scratch(None, None, 1) == -1)
""")) == {"True"}


def test_gated_gradient_refusals():
    assert set(call("""
A = 1 << 20
need = lib.nb200_gated_product_grad_scratch(r(D(40, 64, 64, 2, A)), r(D(32, 64, 64, 2, A)), 1)
print(need == 40 * 32 * 2)
def go(dh=(40, 16, 16, 2, A), both=(40, 32, 32, 2, A), x=(40, 64, 64, 2, A), w=(32, 64, 64, 2, A), groups=1, offsets=None, act=0, dx=(40, 64, 64, 2, A), dw=(32, 64, 64, 2, A), scratch=A, bytes=need):
    return lib.nb200_gated_product_grad(r(D(*dh)), r(D(*both)), r(D(*x)), r(D(*w)), groups, offsets, act, r(D(*dx)), r(D(*dw)), scratch, bytes, None)
print(go() == CUDA)
print(go(dh=(40, 15, 15, 2, A)) == BAD, go(dh=(39, 16, 16, 2, A)) == BAD, go(dh=(40, 16, 16, 1, A)) == BAD, go(both=(40, 31, 31, 2, A)) == BAD, go(both=(41, 32, 32, 2, A)) == BAD)
print(go(dx=(40, 63, 63, 2, A)) == BAD, go(dw=(31, 64, 64, 2, A)) == BAD, go(dw=(32, 64, 64, 0, A)) == BAD, go(act=5) == BAD, go(groups=0) == BAD)
print(go(scratch=None) == BAD, go(scratch=A + 128) == BAD, go(bytes=need - 1) == CAP)
print(go(dh=(0, 16, 16, 2, None), both=(0, 32, 32, 2, None), x=(0, 64, 64, 2, None), dx=(0, 64, 64, 2, None), dw=(0, 64, 64, 2, None), w=(0, 64, 64, 2, None), groups=0, offsets=C.c_void_p(A)) == OK)
""")) == {"True"}


def test_int8_refusals():
    assert set(call("""
A = 1 << 20
count, pitch = lib.nb200_int8_value_count, lib.nb200_int8_pitch
print(pitch(r(I(1, 5, 33, None, None))) == 64, count(r(I(3, 5, 33, None, None))) == 15 * 64, count(r(I(1, 0, 33, None, None))) == 0)
most = (1 << 31) - 1
print(count(r(I(most, most, 2, None, None))) == -1, count(r(I(-1, 1, 1, None, None))) == -1, count(None) == -1, count(r(I(1, most, most, None, None))) == most * ((most + 31) // 32 * 32))
def go(a=(1, 40, 64, A, A), w=(1, 32, 64, A, A), offsets=None, y=(40, 32, 32, 0, A)):
    return lib.nb200_int8_product(r(I(*a)), r(I(*w)), offsets, r(D(*y)), None)
print(go() == CUDA, go(a=(1, 3, 64, A, A), y=(3, 32, 32, 0, A)) == CUDA)
print(go(a=(2, 20, 64, A, A)) == BAD, go(w=(2, 32, 64, A, A)) == BAD, go(a=(1, 40, 65, A, A)) == BAD, go(y=(40, 31, 31, 0, A)) == BAD, go(y=(39, 32, 32, 0, A)) == BAD, go(y=(40, 32, 32, 3, A)) == BAD)
print(go(a=(1, 40, 64, A + 8, A)) == BAD, go(a=(1, 40, 64, None, A)) == BAD, go(a=(1, 40, 64, A, None)) == BAD, go(a=(1, 40, 64, A, A + 2)) == BAD)
print(go(a=(1, 40, 131072, A, A), w=(1, 32, 131072, A, A)) == UN, go(a=(1, 40, 131071, A, A), w=(1, 32, 131071, A, A)) == CUDA, go(w=(4097, 32, 64, A, A), offsets=C.c_void_p(A)) == UN)
print(go(a=(1, 0, 64, None, None), y=(0, 32, 32, 0, None)) == OK, go(w=(1, 0, 64, None, None), y=(40, 0, 0, 0, None)) == OK)
q = lambda x, z: lib.nb200_int8_quantise(r(D(*x)), r(I(*z)), None)
print(q((40, 64, 64, 0, A), (1, 40, 64, A, A)) == CUDA, q((40, 64, 64, 0, A), (1, 39, 64, A, A)) == BAD, q((40, 64, 64, 0, A), (2, 20, 64, A, A)) == CUDA, q((40, 63, 64, 0, A), (1, 40, 64, A, A)) == BAD, q((0, 64, 64, 0, None), (1, 0, 64, None, None)) == OK)
p = lambda codes, scales, z: lib.nb200_int8_pack(codes, scales, r(I(*z)), None)
print(p(None, A, (1, 4, 4, A, A)) == BAD, p(A, None, (1, 4, 4, A, A)) == BAD, p(None, None, (1, 0, 4, None, None)) == OK, p(A, A, (1, 4, 4, A, A)) == CUDA)
print(lib.nb200_int8_unpack(r(I(1, 4, 4, A, A)), None, None) == BAD, lib.nb200_int8_unpack(r(I(1, 4, 0, None, A)), None, None) == OK)
""")) == {"True"}


def test_clip_refusals():
    assert set(call("""
A = 1 << 20
def go(spans=((A, A, 10, 0, 0),), limit=1.0, norm=A, scratch=A, bytes=None):
    n = len(spans)
    all = (S * max(n, 1))(*[S(*s) for s in spans])
    need = lib.nb200_clip_scratch(all, n)
    return lib.nb200_clip(all, n, limit, norm, scratch, need if bytes is None else bytes, None)
print(go() == CUDA, go(spans=()) == CUDA, go(spans=((None, None, 0, 0, 0),)) == CUDA)
print(go(spans=((A, A, -1, 0, 0),)) == BAD, go(spans=((A, A, 1, 3, 0),)) == BAD, go(spans=((A, A, 1, 0, -1),)) == BAD, go(spans=((A, A, 1, 0, 1),)) == BAD, go(spans=((None, A, 1, 0, 0),)) == BAD)
print(go(spans=((A + 2, A, 1, 0, 0),)) == BAD, go(spans=((A + 2, A, 1, 1, 0),)) == CUDA, go(spans=((A, A + 1, 1, 0, 1),)) == BAD)
print(go(limit=-1.0) == BAD, go(limit=float("nan")) == BAD, go(limit=float("inf")) == CUDA, go(norm=None) == BAD, go(scratch=None) == BAD, go(scratch=A + 64) == BAD, go(bytes=8) == CAP)
print(lib.nb200_clip_scratch(None, 1) == -1, lib.nb200_clip_scratch(None, -1) == -1)
""")) == {"True"}


def test_nothing_is_kept_between_calls():
    """What a captured graph writes into has to be the graph's own: a pool that grows frees what it had, and two graphs would share it."""
    for name in ("gated_product.cu", "int8_product.cu", "clip.cu", "tile_product.cuh", "few_rows.cuh"):
        text = re.sub(r"//[^\n]*", "", open(os.path.join(ROOT, "nacho_b200", "csrc", name)).read())
        assert not re.search(r"acquire_workspace|acquire_tagged|cudaMalloc|__device__\s+\w+\s+\w+\[", text), name


def test_shares_of_a_launch_that_starts_beside_another():
    """A kernel that starts beside the one in front and reads what that one does not write has to come behind one that has waited before it let others start, and has
    to end after it: else "this kernel is complete" says nothing about the ones before."""
    text = open(os.path.join(ROOT, "nacho_b200", "csrc", "tile_product.cuh")).read()
    kernel = text[text.index("k_tiles(const TileArgs args"):]
    assert kernel.index("if (!args.beside) wait_for_previous();") < kernel.index("trigger_dependents();") < kernel.index("if (args.beside) finish_after_previous();")
    gated = open(os.path.join(ROOT, "nacho_b200", "csrc", "gated_product.cu")).read()
    for name in ("k_align_rows(", "k_gate_grad("):
        body = gated[gated.index(name):]
        assert body.index("wait_for_previous();") < body.index("trigger_dependents();")
    align = gated[gated.index("k_align_rows("):gated.index("k_gate_grad(")]
    assert "if (beside) finish_after_previous();" in align
    grad = gated[gated.index("int nb200_gated_product_grad(const"):]
    order = [grad.index(w) for w in ('LaunchScope scope("gate_grad"', "aligned(*x, s.x, *w, s.w, &ax, &aw, true", '"gated_grad_x"', "args.beside = true", '"gated_grad_w"')]
    assert order == sorted(order)


@pytest.mark.skipif(not shutil.which("g++"), reason="no host compiler")
def test_the_way_of_a_product(tmp_path):
    """The choice of tiles by itself: narrow sides that the kernels take, parts only where all of them find room at once and have blocks enough, and never a dearer way than
    the plain one."""
    text = open(os.path.join(ROOT, "nacho_b200", "csrc", "tile_product.cuh")).read()
    rule = text[text.index("struct TileWork {"):]
    rule = rule[:rule.index("\n};") + 4]
    (tmp_path / "rule.cpp").write_text("""
#include <algorithm>
#include <cstdint>
#include <cstdio>
constexpr int TILE_M = 256, TILE_N = 256;
""" + rule + """
int main() {
    const int clusters[2] = {33, 14};
    long long seen[3] = {};
    for (long long rows : {1ll, 33ll, 64ll, 65ll, 500ll, 1003ll, 8192ll, 2147482623ll}) for (long long groups : {1ll, 3ll, 64ll, 4096ll}) for (long long wide : {1ll, 6ll, 32ll, 4000000ll})
        for (long long blocks : {1ll, 15ll, 16ll, 40ll, 128ll, 33554432ll}) for (long long pairs : {1ll, 9ll, 74ll}) {
            const TileWork work{rows, groups, wide, blocks};
            const TileWork::Way way = work.best(pairs, clusters);
            const long long mean = (rows + groups - 1) / groups, tiles = groups * ((mean + way.n - 1) / way.n) * wide;
            const bool fits = way.parts == 1 || (tiles * way.parts <= pairs && tiles <= clusters[way.parts / 4] && blocks >= 8 * way.parts);
            if (way.n < 64 || way.n > 256 || way.n % 64 || !(way.parts == 1 || way.parts == 2 || way.parts == 4) || !fits || way.cost <= 0) printf("bad %lld %lld %lld %lld %lld\\n", rows, groups, wide, blocks, pairs);
            ++seen[way.parts / 2];
        }
    printf("%d\\n", seen[0] > 0 && seen[1] > 0 && seen[2] > 0);
}""")
    subprocess.run(["g++", "-std=c++17", "-o", str(tmp_path / "rule"), str(tmp_path / "rule.cpp")], check=True)
    assert subprocess.run([str(tmp_path / "rule")], check=True, capture_output=True, text=True).stdout.split() == ["1"]


@pytest.mark.skipif(not shutil.which("g++"), reason="no host compiler")
def test_the_tiles_that_a_product_is_launched_for(tmp_path):
    """One count of tiles for the choice and for the launch: what groups that share the rows in any way have at most, for one group what it has, and with parts no more
    than find room. 256 rows of 4096 hidden units and a width of 8192, a multiple of every narrow side, are shared by two."""
    text = open(os.path.join(ROOT, "nacho_b200", "csrc", "tile_product.cuh")).read()
    rule = text[text.index("struct TileWork {"):]
    launch = text[text.index("int launch_tiles("):]
    # the launch takes over what was chosen, for as many tiles as were counted then
    assert "work.most(args.tile_n)" in launch and re.search(r"parts = args\.parts;", launch)
    (tmp_path / "count.cpp").write_text("""
#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <random>
constexpr int TILE_M = 256, TILE_N = 256;
""" + rule[:rule.index("\n};") + 4] + """
int main() {
    const int clusters[2] = {33, 14};
    int shared = 0, bad = 0;
    for (long long rows = 1; rows <= 1100; ++rows)
        for (long long wide : {1ll, 6ll, 8ll, 32ll, 64ll}) for (long long blocks : {1ll, 16ll, 128ll, 256ll}) for (long long pairs : {9ll, 37ll, 74ll}) {
            const TileWork work{rows, 1, wide, blocks};
            const TileWork::Way way = work.best(pairs, clusters);
            const long long tiles = (rows + way.n - 1) / way.n * wide;
            bad += work.most(way.n) != tiles || (way.parts > 1 && (tiles * way.parts > pairs || tiles > clusters[way.parts / 4]));
            shared += way.parts > 1 && rows % way.n == 0;
        }
    std::mt19937 draw(1);
    for (int i = 0; i < 20000; ++i) {
        const int groups = 1 + draw() % 40, n = 64 * (1 + draw() % 4);
        long long rows = draw() % 30, tiles = 0;  // some rows of nobody
        for (int g = 0; g < groups; ++g) {
            const long long mine = draw() % 3 ? draw() % 300 : draw() % 2;
            rows += mine, tiles += (mine + n - 1) / n;
        }
        if (rows == 0) continue;
        const TileWork work{rows, groups, 3, 128};
        bad += work.most(n) < 3 * tiles;
        const TileWork::Way way = work.best(74, clusters);
        bad += way.parts > 1 && (work.most(way.n) * way.parts > 74 || work.most(way.n) > clusters[way.parts / 4]);
    }
    const TileWork::Way way = TileWork{256, 1, 32, 128}.best(74, clusters);
    printf("%d %d %d\\n", bad, shared > 0, (int)(way.parts == 2 && TileWork{256, 1, 32, 128}.most(way.n) == 32));
}""")
    subprocess.run(["g++", "-std=c++17", "-o", str(tmp_path / "count"), str(tmp_path / "count.cpp")], check=True)
    assert subprocess.run([str(tmp_path / "count")], check=True, capture_output=True, text=True).stdout.split() == ["0", "1", "1"]


@pytest.mark.skipif(not shutil.which("g++"), reason="no host compiler")
def test_narrow_sides_no_wider_than_the_rows(tmp_path):
    """Few rows of one group take the narrow side that holds them, with which more stages fit."""
    text = open(os.path.join(ROOT, "nacho_b200", "csrc", "tile_product.cuh")).read()
    rule = text[text.index("struct TileWork {"):]
    (tmp_path / "side.cpp").write_text("""
#include <algorithm>
#include <cstdint>
#include <cstdio>
constexpr int TILE_M = 256, TILE_N = 256;
""" + rule[:rule.index("\n};") + 4] + """
int main() {
    const int clusters[2] = {33, 14};
    for (long long rows = 1; rows <= 256; ++rows) for (long long wide : {1ll, 8ll, 16ll, 32ll, 74ll, 300ll}) for (long long blocks : {1ll, 18ll, 64ll, 128ll}) {
        const TileWork::Way way = TileWork{rows, 1, wide, blocks}.best(74, clusters);
        if (way.n - 64 >= rows) printf("%lld %lld %lld: %d\\n", rows, wide, blocks, way.n);
    }
}""")
    subprocess.run(["g++", "-std=c++17", "-o", str(tmp_path / "side"), str(tmp_path / "side.cpp")], check=True)
    assert subprocess.run([str(tmp_path / "side")], check=True, capture_output=True, text=True).stdout == ""
