"""Outputs that lie on tensors which other blocks still read are refused; in place, side by side and between each other's rows they are not."""
import os
import subprocess
import tempfile

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SRC = r'''
#include <cstdio>
#include "goneuron_b200/csrc/op_rules.cuh"
using namespace gn;
static int bad = 0;
#define OK(x) do { if (const char* e_ = (x)) { bad++; std::printf("line %d: refused: %s\n", __LINE__, e_); } } while (0)
#define NO(x) do { if (!(x)) { bad++; std::printf("line %d: not refused\n", __LINE__); } } while (0)
static void* at(uintptr_t a) { return reinterpret_cast<void*>(a); }
int main() {
  gn_heads q{at(4096), 512, 64, 8, 0}, k{at(8192), 512, 64, 8, 0}, none{at(4096), 512, 64, 0, 0}, empty{nullptr, 0, 0, 8, 0};
  NO(check_apart(&q, &q)); OK(check_apart(&q, &k)); OK(check_apart(&q, &none)); OK(check_apart(&q, nullptr)); OK(check_apart(nullptr, &q)); OK(check_apart(&empty, &empty));
  auto distill = [](int64_t rows, int64_t vocab, int64_t stride, int64_t dstride, int64_t out) {      // out: elements of 2 bytes from the logits
    return check_distill(GN_F16, rows, vocab, 0, 1.f, at(1 << 20), stride, nullptr, GN_I64, nullptr, nullptr, (const float*)at(256), at((1 << 20) + 2 * out), dstride);
  };
  OK(distill(5, 100, 100, 100, 0)); OK(distill(5, 100, 100, 100, 500)); OK(distill(5, 100, 100, 100, -500));
  for (int64_t d : {1, 99, 100, 300, 499, -1, -100, -250, -499}) NO(distill(5, 100, 100, 100, d));
  OK(distill(5, 100, 200, 200, 100)); OK(distill(5, 100, 200, 200, -100)); OK(distill(5, 100, 200, 200, 300)); OK(distill(5, 100, 200, 200, 900)); OK(distill(5, 100, 200, 200, 1000)); OK(distill(5, 100, 200, 200, -900));
  for (int64_t d : {99, 101, 200, -99, -101, 301, 899}) NO(distill(5, 100, 200, 200, d));
  OK(distill(1, 100, 100, 100, 100)); OK(distill(1, 100, 7, 0, 100)); OK(distill(1, 100, 100, 100, -100)); NO(distill(1, 100, 100, 100, 99)); NO(distill(1, 100, 0, 5, -3));
  return bad != 0;
}
'''


def test_what_lies_on_what():
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "t.cpp"), os.path.join(d, "t")
        open(src, "w").write(SRC)
        subprocess.check_call(["g++", "-std=c++17", "-O1", "-I", ROOT, "-x", "c++", src, "-o", exe])
        r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
        assert r.returncode == 0, r.stdout
