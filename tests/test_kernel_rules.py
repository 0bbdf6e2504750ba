"""Rules of PTX and of the CUDA memory model that a kernel can break and still pass its tests, read off the sources."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "picoforge_b200" / "csrc"
SOURCES = sorted(p for p in CSRC.iterdir() if p.suffix in (".cu", ".cuh"))


def without_comments(text):
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


def functions(text, mark):
    """(head, body) of every function whose head begins with `mark`."""
    for m in re.finditer(mark, text):
        start = text.find("{", m.end())
        if ";" in text[m.end():start]:
            continue                                         # a declaration
        depth, at = 0, start
        while True:
            depth += {"{": 1, "}": -1}.get(text[at], 0)
            at += 1
            if not depth:
                break
        yield text[m.start():start], text[start:at]


def with_helpers(text):
    """The kernels of a source, calls of its own barrier helpers replaced by what these do."""
    helpers = {}
    for head, body in functions(text, r"__device__ __forceinline__ void \w*bar_init\("):
        helpers[re.search(r"(\w+)\(", head).group(1)] = body
    for head, body in functions(text, r"__global__"):
        for name, does in helpers.items():
            body = re.sub(rf"\b{name}\([^;]*;", lambda _: does, body)
        yield head, body


@pytest.mark.parametrize("source", SOURCES, ids=lambda p: p.name)
def test_barriers_are_fenced_before_copies_and_products_use_them(source):
    """mbarrier.init is a store of the generic proxy; asynchronous copies and commits complete on the barrier in another one.
    A barrier's initialisation is therefore fenced before the threads of the CTA meet."""
    for _, body in with_helpers(without_comments(source.read_text())):
        inits = [m.start() for m in re.finditer(r"mbarrier\.init", body)]
        if inits:
            meet = body.find("__syncthreads()", inits[-1])
            assert meet > 0 and re.search(r"fence\.(mbarrier_init|proxy\.async)", body[inits[-1]:meet]), body[inits[-1]:inits[-1] + 300]


@pytest.mark.parametrize("source", SOURCES, ids=lambda p: p.name)
def test_collectives_stay_where_they_are_written(source):
    """An asm statement that is not volatile may move to where its result is used, which only some of the lanes may reach; one in
    which all lanes of a warp have to take part then never ends."""
    for m in re.finditer(r"\basm\s*\(\s*\"[^\"]*\b(redux|elect|vote|shfl|match|bar|barrier|activemask)\.", without_comments(source.read_text())):
        pytest.fail(f"{source.name}: collective in an asm that is not volatile: {m.group(0)}")


@pytest.mark.parametrize("source", SOURCES, ids=lambda p: p.name)
def test_kernels_launched_early_read_nothing_as_constant(source):
    """A kernel that may begin before the launch ahead of it has ended runs while its inputs are written.  A load that is told otherwise (__ldg, or a
    pointer to const that is __restrict__) may come before the wait, and may find a line that the SM kept from the launch ahead."""
    weights = r"\(m \? a\.row_scale1 : a\.row_scale0\)"     # scales of the weights' rows, written when the layer was made
    for head, body in functions(without_comments(source.read_text()), r"__global__"):
        if "griddepcontrol.wait" in body or "grid_wait()" in body:
            assert not re.search(r"\bconst\s[^,()]*__restrict__", head), head
            assert not re.search(rf"__ldg\((?!{weights})", body), head
