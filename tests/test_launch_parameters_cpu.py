"""The products' parameter block has a value in every field that a launch reads, whatever the caller's stack held: an entry point
that names only its own fields must not have a tile, an accumulate flag or loss operands chosen for it by old stack contents."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include "gemm.h"
#include <cstdio>
#include <cstring>
#include <new>
int main() {
    alignas(GemmParams) static unsigned char memory[sizeof(GemmParams)];
    memset(memory, 0x80, sizeof(memory));                 // (a tile of 0x80808080, pointers that are not null)
    asm volatile("" ::: "memory");
    GemmParams* p = new (memory) GemmParams;
    asm volatile("" : "+r"(p) :: "memory");
    printf("%d %d %d\n", p->tile, p->accumulate, p->drop.thresh);
    printf("%d\n", p->A || p->B || p->C || p->aux || p->tk_cand || p->tk_cnt || p->tk_thr || p->ce_labels || p->ce_lse || p->ce_g || p->ce_err || p->ce_lo || p->ce_part || p->ce_target);
    printf("%d\n", p->M || p->N || p->K || p->lda || p->ldb || p->ldc || p->ldaux || p->k_per_split || p->tk_cap || p->tk_row_base || p->ce_vocab || p->ce_first || p->ce_rows || p->drop_narrow);
    printf("%d\n", p->a_heads || p->b_heads || p->c_heads || p->strideA || p->strideB || p->strideC || p->ce_ignore);
    printf("%d %g %g\n", p->batch, p->alpha, p->mask_scale);
    return 0;
}
"""


def test_no_field_keeps_what_the_memory_held(tmp_path):
    sys.path.insert(0, ROOT)
    import __graft_entry__ as g
    if not os.path.exists(g.HIPCC):
        pytest.skip("no hipcc here")
    src, exe = tmp_path / "fields.cpp", tmp_path / "fields"
    src.write_text(PROGRAM)
    subprocess.check_call([g.HIPCC, "-x", "hip", "--offload-arch=gfx950", "--cuda-host-only", "-std=c++17", "-O2", "-I" + g.CSRC, str(src), "-o", str(exe)],
                          stderr=subprocess.DEVNULL)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n")
    assert out[:5] == ["0 0 0", "0", "0", "0", "1 1 1"], out
