// Which drafted tokens are accepted (gfx950): the walk from a tree's first node along the model's picks.
//
// A wave takes a sequence, a lane a node: each step is one comparison in every lane and the lowest set bit of the
// ballot, so that a path of n nodes costs n steps of a few instructions, and no memory after the first loads.  A
// launch's own time and one memory round trip bound it.
#include "../../include/dsqg.h"
#include "dsqg_common.hpp"

namespace dsqg {
namespace {

struct TreeAccept {
  const long long* tokens; long long ts;
  const int* parents; long long ps;
  const long long* picks; long long ks;
  const long long* counts;
  long long* path;
  long long* n;
  long long* next;
  int B, T;
};

__global__ __launch_bounds__(64) void tree_accept_kernel(TreeAccept p) {
  const long long b = blockIdx.x;
  const int i = threadIdx.x;
  const long long have = p.counts ? p.counts[b] : p.T;
  const bool live = i < p.T && i < have;
  const long long token = live ? p.tokens[b * p.ts + i] : 0, pick = live ? p.picks[b * p.ks + i] : 0;
  const int parent = live ? p.parents[b * p.ps + i] : -1;
  if (have <= 0) {
    if (i < p.T) p.path[b * p.T + i] = -1;
    if (i == 0) {
      p.n[b] = 0;
      p.next[b] = -1;
    }
    return;
  }
  int at = 0, n = 1;
  long long mine = i == 0 ? 0 : -1, want = __shfl(pick, 0, 64);
  while (true) {  // (`at` grows with every step)
    const unsigned long long fits = __ballot(live && i > at && parent == at && token == want);
    if (fits == 0) break;
    at = __builtin_ctzll(fits);
    if (i == n) mine = at;
    ++n;
    want = __shfl(pick, at, 64);
  }
  if (i < p.T) p.path[b * p.T + i] = mine;
  if (i == 0) {
    p.n[b] = n;
    p.next[b] = want;
  }
}

}  // namespace
}  // namespace dsqg

using namespace dsqg;

extern "C" int dsqg_tree_accept(const dsqg_tree_accept_args* a, dsqg_stream_t stream) {
  if (!a || a->B < 0 || a->T < 1) return DSQG_EINVAL;
  if (a->T > DSQG_MAX_TREE || a->B >= 1 << 26) return DSQG_EUNSUPPORTED;  // (a grid has less than 2^32 lanes)
  if (a->B == 0) return DSQG_OK;
  if (!a->tokens || !a->parents || !a->picks || !a->path || !a->n || !a->next) return DSQG_EINVAL;
  for (long long s : {a->tokens_stride, a->parents_stride, a->picks_stride})
    if (s < 0 || s > (1ll << 50)) return DSQG_EINVAL;
  TreeAccept p = {};
  p.B = a->B; p.T = a->T;
  p.tokens = reinterpret_cast<const long long*>(a->tokens); p.ts = a->tokens_stride;
  p.parents = a->parents; p.ps = a->parents_stride;
  p.picks = reinterpret_cast<const long long*>(a->picks); p.ks = a->picks_stride;
  p.counts = reinterpret_cast<const long long*>(a->counts);
  p.path = reinterpret_cast<long long*>(a->path);
  p.n = reinterpret_cast<long long*>(a->n);
  p.next = reinterpret_cast<long long*>(a->next);
  hipLaunchKernelGGL(tree_accept_kernel, dim3((unsigned)a->B), dim3(64), 0, reinterpret_cast<hipStream_t>(stream), p);
  return hipGetLastError() == hipSuccess ? DSQG_OK : DSQG_EHIP;
}
