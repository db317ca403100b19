// Window attention on tcgen05: what its copying and its multiplying thread do, in order. Written over
// an F that does the copies, products and waits, so that a host program can run the same steps with any wait
// giving up. A wait returns false once it gave up; waits have a limit, so every role ends.
//
// Whoever gives up, here or in another warp, both roles leave only after their own work has ended: copies into
// the CTA's shared memory have landed, products that read it and write TMEM are done. After a whole run
// these phases are complete, and the last waits cost nothing.
#pragma once

#ifdef __CUDACC__
#define MC_ROLE_FN __device__ __forceinline__
#else
#define MC_ROLE_FN inline
#endif

namespace mc {
namespace win {

// The queries once, then the keys and the values of n tiles, into one buffer each.
template <class F>
MC_ROLE_FN void copy_tiles(F& f, int n) {
  int keys = 0, values = 0;  // copies asked for
  f.copy_queries();
  for (int i = 0; i < n; ++i) {
    // the key buffer is free once the score product of tile i - 1 is done
    if (i > 0 && !f.wait_scores((i - 1) & 1)) break;
    f.copy_keys(i);
    ++keys;
    if (i > 0 && !f.wait_values_free((i - 1) & 1)) break;
    f.copy_values(i);
    ++values;
  }
  f.drain_queries(0);
  if (keys > 0) f.drain_keys((keys - 1) & 1);
  if (values > 0) f.drain_values((values - 1) & 1);
}

// Per tile the score product, and once the weights are there the value product. The scores of tile i + 1
// go over the columns of the weights of tile i: products run in order.
template <class F>
MC_ROLE_FN void multiply_tiles(F& f, int n) {
  bool ok = f.wait_queries(0) && f.wait_keys(0);
  if (ok) f.multiply_scores();
  for (int i = 0; ok && i < n; ++i) {
    ok = f.wait_weights(i & 1) && f.wait_values(i & 1);
    if (!ok) break;
    f.multiply_values(i);
    if (i + 1 < n) {
      f.commit_values_free();
      ok = f.wait_keys((i + 1) & 1);
      if (ok) f.multiply_scores();
    } else {
      f.commit_outputs();
    }
  }
  if (!ok) f.commit_outputs();
  f.drain_outputs(0);
}

}  // namespace win
}  // namespace mc
