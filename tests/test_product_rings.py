"""The rings of the tcgen05 products (csrc/qs_matmul_tc.cuh): no scale is overwritten before it is read.

The kernel's roles are ordered by barriers alone, so the test follows what those guarantee, in the
configurations that the header defines (compiled for the host; nothing runs on a GPU):

* stage j is unpacked, and its scales written to slot j % DR, once the products of stage j - NS are done;
* the products that begin accumulator g start once the sums have read accumulator g - NB;
* the sums read accumulator g together with the scales of the stage that ends it, in rising order.
"""

import os
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "quant-studio_b200" / "csrc"
NVCC = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"

PROGRAM = r"""
#include <stdio.h>
#include "qs_matmul_tc.cuh"
using namespace qs;
template <int T, int BN, bool LO> void show() {
    using C = TcCfg<T, BN, LO>;
    printf("%d %d %d %d %d %d %d %d\n", T, BN, (int)LO, C::NS, C::NB, C::GROUP, C::DR, C::BYTES + BN * 8 + 512);
}
int main() {
#define X(T) show<T, 128, true>(); show<T, 128, false>(); show<T, 256, false>();
    QS_FOR_TYPES(X)
    return 0;
}
"""


@pytest.fixture(scope="module")
def configurations(tmp_path_factory):
    if not os.path.exists(NVCC):
        pytest.skip("no nvcc")
    d = tmp_path_factory.mktemp("rings")
    (d / "rings.cu").write_text(PROGRAM)
    subprocess.run([NVCC, "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", f"-I{CSRC}", "-o", d / "rings", d / "rings.cu"],
                   check=True, capture_output=True)
    out = subprocess.run([d / "rings"], check=True, capture_output=True, text=True).stdout
    return [tuple(map(int, line.split())) for line in out.splitlines()]


def accumulators(main, extra, group):
    """(first stage, last stage) of every accumulator: one per `group` of the `main` stages of levels (0: one per
    unit of 32 values, two a stage), one per stage of the `extra` ones with minima."""
    r = [(i, min(i + group, main) - 1) for i in range(0, main, group)] if group else [(i, i) for i in range(main) for _ in range(2)]
    return r + [(i, i) for i in range(main, main + extra)]


def lapped(main, extra, ns, nb, group, dr):
    """(stage written, stage not yet read) where the barriers leave the order open."""
    acc = accumulators(main, extra, group)
    bad = []
    for j in range(dr, main + extra):
        done = j - ns                                                  # products of this stage are over
        begun = max(g for g, (first, _) in enumerate(acc) if first <= done)
        read = begun - nb                                              # the sums are through with this accumulator
        bad += [(j, last) for g, (_, last) in enumerate(acc) if last == j - dr and g > read]
    return bad


def test_scales_are_read_before_they_are_overwritten(configurations):
    assert len(configurations) == 16 * 3
    for typ, bn, lo, ns, nb, group, dr, smem in configurations:
        for main in (1, 3, 4, 5, 15, 16, 17, 20, 40, 64, 128):
            for extra in (0, 1, 2, 6, 12):
                assert not lapped(main, extra, ns, nb, group, dr), (typ, bn, lo)


def test_the_model_sees_a_short_ring():
    """Four accumulators of four stages with four stages of operands reach 16 back."""
    assert lapped(40, 0, 4, 4, 4, 16) and not lapped(40, 0, 4, 4, 4, 17)


def test_shared_memory_fits(configurations):
    """The dynamic part, the slots' tables and the barriers, within 227 KB."""
    for typ, bn, lo, ns, nb, group, dr, smem in configurations:
        assert smem <= 227 * 1024 and ns >= 2, (typ, bn, lo, ns, smem)
