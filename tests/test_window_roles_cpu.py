"""Window attention's copying and multiplying threads leave nothing in flight: the kernel's own steps
(mc_window_roles.h) compiled for the host, run with every wait giving up in turn, and with none."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mignon_ai_b200", "csrc")

PROGRAM = r"""
#include <cstdio>
#include "mc_window_roles.h"

// The `at`-th wait (from 0) gives up, and so do all after it; -1: none does.
struct Waits {
  int at, n = 0;
  bool wait() { return at < 0 || n++ < at; }
};

// A buffer: copies asked for, and whether the last one is known to have landed.
struct Buffer {
  int copies = 0;
  bool landed = true;
  void copy() { ++copies, landed = false; }
  void drain(int phase) { if (copies > 0 && phase == (copies - 1) % 2) landed = true; }
};

struct Copier {
  Waits w;
  Buffer q, k, v;
  bool early = false;  // a copy over one that may still be in flight
  void copy_queries() { q.copy(); }
  void copy_keys(int i) { early |= !k.landed || i != k.copies; k.copy(); }
  void copy_values(int i) { early |= !v.landed || i != v.copies; v.copy(); }
  // the products of a tile have read its keys (its values)
  bool wait_scores(int phase) { const bool ok = w.wait(); if (ok) k.drain(phase); return ok; }
  bool wait_values_free(int phase) { const bool ok = w.wait(); if (ok) v.drain(phase); return ok; }
  void drain_queries(int phase) { q.drain(phase); }
  void drain_keys(int phase) { k.drain(phase); }
  void drain_values(int phase) { v.drain(phase); }
};

struct Multiplier {
  Waits w;
  int issued = 0, covered = 0, outputs = 0, scores = 0, values = 0;  // covered: products before the last commit to the outputs
  bool drained = false;
  void multiply_scores() { ++issued, ++scores; }
  void multiply_values(int) { ++issued, ++values; }
  void commit_values_free() {}
  void commit_outputs() { ++outputs, covered = issued; }
  bool wait_queries(int) { return w.wait(); }
  bool wait_keys(int) { return w.wait(); }
  bool wait_values(int) { return w.wait(); }
  bool wait_weights(int) { return w.wait(); }
  void drain_outputs(int phase) { drained = outputs == 1 && phase == 0 && covered == issued; }
};

int main() {
  int runs = 0;
  for (int n = 1; n <= 6; ++n)
    for (int at = -1; at < 4 * n + 2; ++at, ++runs) {
      Copier c{{at}};
      mc::win::copy_tiles(c, n);
      if (c.early || !c.q.landed || !c.k.landed || !c.v.landed) return printf("copies in flight: n %d, wait %d\n", n, at), 1;
      if (at < 0 && (c.k.copies != n || c.v.copies != n)) return printf("copies missing: n %d\n", n), 1;
      Multiplier m{{at}};
      mc::win::multiply_tiles(m, n);
      if (!m.drained) return printf("products in flight: n %d, wait %d\n", n, at), 1;
      if (at < 0 && (m.scores != n || m.values != n)) return printf("products missing: n %d\n", n), 1;
    }
  return printf("%d runs\n", runs), 0;
}
"""


def test_no_role_leaves_with_work_in_flight(tmp_path):
    source, program = tmp_path / "roles.cpp", tmp_path / "roles"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-I", CSRC, "-o", str(program), str(source)], check=True)
    done = subprocess.run([str(program)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout
    assert done.stdout == "102 runs\n"
