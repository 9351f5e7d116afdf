// kq4_mx_run for a host program, through a C entry (test_mx_runs.py).
#include "../../kestrel-llm_amd/csrc/kq4_mx.h"

extern "C" void t_run(int rows, int cols, int type, int scales, int t0, int off, long *o) {
  const KQ4MxRun r = kq4_mx_run(kq4_mx_dims(rows, cols), type, scales != 0, t0, off);
  o[0] = r.at;
  o[1] = r.bytes;
  o[2] = r.step;
}
