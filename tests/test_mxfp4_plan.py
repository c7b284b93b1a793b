"""Which kernels products and linears of 4-bit operands take, from the library's own
rules (csrc/mxfp4_plan.h, host arithmetic, compiled here by the host's compiler): every
kernel that some size takes is run by a GPU test, and tests that rely on a size's kernel
have it."""
import os
import random
import shutil
import subprocess

import pytest

import test_gpu_mxfp4 as base
import test_gpu_mxfp4_kinds as kinds

SOURCE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "native", "mxfp4_plan.cpp")
TILES = ("256", "128", "128x64", "64", "64 ring")


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """The kernel of each product (linear False) or linear of (m, n, k)."""
    compiler = shutil.which("g++") or shutil.which("c++")
    if compiler is None:
        pytest.skip("no host compiler")
    exe = str(tmp_path_factory.mktemp("plan") / "mxfp4_plan")
    subprocess.run([compiler, "-std=c++17", "-Wall", "-Werror", "-O1", "-o", exe, SOURCE], check=True)

    def ask(sizes, linear):
        text = "\n".join("%d %d %d" % s for s in sizes)
        out = subprocess.run([exe], input=text, capture_output=True, text=True, check=True).stdout.splitlines()
        assert len(out) == len(sizes)
        return [_name(s[0], [int(v) for v in line.split()], linear) for s, line in zip(sizes, out)]
    return ask


def _name(m, plan, linear):
    kind, splits, takes_rows, codes = plan[:4]
    few = plan[8:] if linear and codes else plan[4:8]
    if m <= 64:
        scales = "coding" if linear and codes else "slabs" if linear else "rows"
        return "few %s %d %d %d" % (scales, *few[:3]) + (" split" if few[3] > 1 else "")
    rows = takes_rows and not linear
    tile = "64 ring" if rows else TILES[kind]  # (the kind with room for scales as rows)
    return f"tile {tile} {'rows' if rows else 'slabs'}" + (" split" if splits > 1 else "")


def _marked(test, names):
    """The first three values of the parameters that begin with `names`."""
    return [a[:3] for mark in test.pytestmark if mark.name == "parametrize" and mark.args[0].startswith(names)
            for a in mark.args[1]]


def test_sizes_have_the_kernels_they_are_listed_for(kernels):
    for cases, linear in ((kinds.PRODUCTS, False), (kinds.LINEARS, True)):
        assert kernels([c[1:] for c in cases], linear) == [c[0] for c in cases]


def test_every_kernel_is_run(kernels):
    """Those of 40000 sizes are among the tests'."""
    tested = {False: set(kernels([c[1:] for c in kinds.PRODUCTS] + base.SIZES + base.LONG, False)),
              True: set(kernels([c[1:] for c in kinds.LINEARS] + _marked(base.test_linear, "m,n,k") + base.LONG, True))}
    r = random.Random(7)
    sizes = [(r.randint(1, 64) if r.random() < 0.5 else round(2 ** r.uniform(6, 15)), round(2 ** r.uniform(0, 16.5)),
              round(2 ** r.uniform(0, 17))) for _ in range(40000)]
    sizes = [(m, n, min(k, (1 << 17) - 1)) for m, n, k in sizes]
    for linear in (False, True):
        missing = set(kernels(sizes, linear)) - tested[linear]
        assert not missing, sorted(missing)


def test_sizes_that_have_to_take_slabs(kernels):
    """A workspace that cannot be had is asked for before anything is launched, and
    slabs of more rows than a dimension of the grid holds are laid out."""
    assert kernels([((1 << 31) - 1, 70, 131040), ((1 << 29) + 77, 65, 288)], False) == ["tile 128 slabs"] * 2


def test_scales_as_rows_where_the_launch_saved_pays(kernels):
    """Many small tiles lay out their own scales more slowly than a launch before them
    does."""
    many = [(4096, 4100, 512), (12000, 1000, 64), (400, 6000, 4000), (16000, 300, 128), (5000, 611, 1542)]
    few = [(333, 8192, 256), (1000, 2304, 256), (333, 1000, 2000), (65, 130, 511)]
    assert kernels(many, False) == ["tile 64 slabs"] * len(many)
    assert kernels(few, False) == ["tile 64 ring rows"] * len(few)
