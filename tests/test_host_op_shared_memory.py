"""The most shared memory that a call of the operators on device memory asks for, as op_rules.cuh states it: no plan needs more, and a block may have it."""
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
  const int block = 227 * 1024, fixed = 3 * 1024;                     // what a block may have, and more than the kernels' own arrays take of it
  if (DISTILL_SMEM_MOST + fixed > block || QK_ROWS_SMEM_MOST + fixed > block) { bad++; std::printf("%d, %d: more than a block may have\n", DISTILL_SMEM_MOST, QK_ROWS_SMEM_MOST); }
  for (long rows : {1L, 75L, 100000L}) for (long vocab = 1; vocab < 1000000; vocab += 1 + vocab / 50) for (int size : {2, 4}) for (int top : {0, 1, 64, 256, 1023, 1024}) {
    const DistillPlan p = distill_plan(rows, vocab, size, 148);
    if (p.per * 16 + teacher_smem(top) > DISTILL_SMEM_MOST) { bad++; std::printf("distill: vocab %ld, top %d\n", vocab, top); }
  }
  for (long tokens : {1L, 500L, 100000L}) for (int heads : {1, 3, 40}) for (int head = 1; head <= 1024; head++) for (int rotated = 0; rotated <= head; rotated += 2) {
    const int n = qk_tokens(tokens, 148, 0, heads, 1, rotated);
    if (((long)n * rotated + ((rotated + 3) & ~3) + QK_ROW_WARPS * head) * 4 > QK_ROWS_SMEM_MOST) { bad++; std::printf("norm of queries and keys: head %d, rotated %d\n", head, rotated); }
  }
  return bad != 0;
}
'''


def test_no_plan_needs_more_than_the_most():
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "t.cpp"), os.path.join(d, "t")
        open(src, "w").write(SRC)
        subprocess.check_call(["g++", "-std=c++17", "-O1", "-I", ROOT, "-x", "c++", src, "-o", exe])
        r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
        assert r.returncode == 0, r.stdout
