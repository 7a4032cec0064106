"""How rows are cut among blocks when the teacher's entries are counted: the parts hold a row, and where a row is given to one block, or to four, two such blocks fit a multiprocessor."""
import os
import subprocess
import tempfile

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SRC = r'''
#include <cstdio>
#include "goneuron_b200/csrc/op_rules.cuh"
using namespace gn;
int main() {
  int bad = 0;
  for (int top : {0, 1, 64, 256, 1024}) for (int size : {2, 4}) for (long rows : {1L, 75L, 4096L}) for (long vocab = 1; vocab < 800000; vocab += 1 + vocab / 200) {
    const DistillPlan p = distill_plan(rows, vocab, size, 148, top); const int V = 16 / size;
    if (p.cluster == 0) { if (vocab * size <= 8L * DISTILL_PART_MOST - 200) { bad++; std::printf("%ld fits\n", vocab); } continue; }
    for (int lead = 0; lead < V; lead++) if (ceil_div(lead + vocab, V) > (long)p.cluster * p.per) { bad++; std::printf("vocab %ld top %d\n", vocab, top); }
    const long block = p.per * 16 + teacher_smem(top) + DISTILL_FIXED;
    if (block > 227 * 1024 + 1024) { bad++; std::printf("vocab %ld top %d: %ld bytes\n", vocab, top, block); }
    if ((p.cluster == 1 || p.cluster == 4) && 2 * block > DISTILL_SM_SMEM) { bad++; std::printf("vocab %ld top %d: %ld bytes twice\n", vocab, top, block); }
  }
  // the sizes at which one block of a row used to have a multiprocessor to itself
  struct { long vocab; int size, top; } alone[] = {{50257, 2, 256}, {53000, 2, 64}, {25600, 4, 256}};
  for (auto& a : alone) { const DistillPlan p = distill_plan(4096, a.vocab, a.size, 148, a.top); if (p.cluster == 1 && 2 * (p.per * 16 + teacher_smem(a.top) + DISTILL_FIXED) > DISTILL_SM_SMEM) bad++; }
  return bad != 0;
}
'''


def test_plans():
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "t.cpp"), os.path.join(d, "t")
        open(src, "w").write(SRC)
        subprocess.check_call(["g++", "-std=c++17", "-O1", "-I", ROOT, "-x", "c++", src, "-o", exe])
        r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
        assert r.returncode == 0, r.stdout
