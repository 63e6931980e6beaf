"""CPU suite: what the barriers of the 8-bit products' pipelines order, followed from the source. A copy may overwrite a place of scales only when all
warps have read what lay there, and that has to follow from the barriers, however slow a warp is."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nacho_b200", "csrc")


def source():
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, "fp8_product.cu")).read())


def constants(shape, **known):
    """STAGES, SUMS and SCALES of a shape, from its definition."""
    text = source()
    body = text[text.index(f"struct {shape} {{"):]
    body = body[:body.index("struct Shared")]
    names = dict(known)
    for name, value in re.findall(r"\b([A-Z_]+) = ([^,;]+)", body):
        value = re.sub(r"(\w+) \? (\d+) : (\d+)", r"(\2 if \1 else \3)", value).replace("/", "//")
        names[name] = eval(value, {}, names)
    return names["STAGES"], names["SUMS"], names["SCALES"]


def summing_loop(function, first):
    """The loop over blocks in which warps add sums times scales, from the wait for the sums on."""
    text = source()
    text = text[text.index(function):]
    text = text[text.index(first):]
    return text[:text.index("__fmaf_rn")]


def read_before_arrival(loop, scale):
    """Whether a warp has read a block's scales when it says that the block's sums have been read."""
    return loop.rindex(scale) < loop.index("sum_empty[sums.at]")


def ordered(stages, sums, scales, before, blocks=64):
    """Whether the last read of every block's scales comes before the copy into the same place, by the barriers alone."""
    after = {}

    def edge(a, b):
        after.setdefault(a, []).append(b)

    for b in range(blocks):
        edge(("copy", b), ("product", b))                   # full
        edge(("product", b), ("copy", b + stages))          # empty
        edge(("product", b), ("arrive", b))                 # sum_full
        edge(("arrive", b), ("product", b + sums))          # sum_empty
        edge(("copy", b), ("copy", b + 1))                  # each warp one block after the other
        edge(("product", b), ("product", b + 1))
        edge(("read", b), ("arrive", b if before else b + 1))
        edge(("arrive", b), ("read", b + 1 if before else b))

    def reaches(start, goal):
        seen, todo = set(), [start]
        while todo:
            at = todo.pop()
            if at == goal:
                return True
            if at not in seen and at[1] <= goal[1] + 1:
                seen.add(at)
                todo += after.get(at, [])
        return False

    return all(reaches(("read", b), ("copy", b + scales)) for b in range(blocks // 2))


def test_the_model_finds_a_missing_order():
    assert ordered(4, 2, 6, before=True) and not ordered(4, 2, 5, before=True)
    assert ordered(4, 2, 7, before=False) and not ordered(4, 2, 6, before=False)


@pytest.mark.parametrize("pair", [False, True])
def test_scales_of_tiles_are_read_before_they_are_overwritten(pair):
    loop = summing_loop("void product(", "sh.sum_full[sums.at]")
    sizes = constants("Shape", PAIR=pair)
    assert sizes[:2] == ((4, 2) if pair else (4, 4))
    assert read_before_arrival(loop, "sh.scale[place.at]")
    assert ordered(*sizes, before=read_before_arrival(loop, "sh.col_scale[place.at]"))


@pytest.mark.parametrize("rows", [16, 32, 64, 128])
def test_scales_of_few_rows_are_read_before_they_are_overwritten(rows):
    loop = summing_loop("k_product_few(", "sh.sum_full[sums.at]")
    assert ordered(*constants("FewShape", NB=rows), before=read_before_arrival(loop, "sh.scale[place.at]"))
