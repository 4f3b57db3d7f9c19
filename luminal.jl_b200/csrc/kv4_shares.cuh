// How the pieces of work of an attention call are dealt out, and on which words the shares that cut a (sequence, row tile, kv head) triple are counted.  Plain arithmetic, for the
// kernel and for whoever checks it on the host.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define LMB_HD __host__ __device__ __forceinline__
#else
#define LMB_HD inline
#endif

namespace lmb {
namespace kv4 {

constexpr int kMostShares = 1024, kJoin = 16;
// Words that count arrivals, zero between calls: for every share one of the triple that it is the first to have a part of, and two for a group of shares that begins with it.
constexpr int kCounters = 3 * kMostShares;

// Share s has the pieces [pieces s / shares, pieces (s + 1) / shares).
LMB_HD int64_t share_begin(int share, int64_t pieces, int shares) { return pieces * share / shares; }
LMB_HD int share_of(int64_t piece, int64_t pieces, int shares) { return (int)(((piece + 1) * shares - 1) / pieces); }

// What share `share` counts for the triple of the pieces item0 .. item0 + n_pieces - 1, which it has a part of: that one of `count` shares from `first` on is done.  Behind
// kJoin + kJoin / 2 shares the last of every kJoin neighbours joins theirs, and then counts one of `groups` groups.
struct Part {
  int first, count, groups, sa;              // sa: the triple's first share
};
LMB_HD Part part_of(int64_t item0, int n_pieces, int share, int64_t pieces, int shares) {
  Part q;
  q.sa = share_of(item0, pieces, shares);
  const int n = share_of(item0 + n_pieces - 1, pieces, shares) - q.sa + 1;
  const bool grouped = n > kJoin + kJoin / 2;
  const int group = grouped ? (share - q.sa) / kJoin : 0;
  q.groups = grouped ? (n + kJoin - 1) / kJoin : 1;
  q.first = q.sa + group * kJoin;
  q.count = grouped ? (n - group * kJoin < kJoin ? n - group * kJoin : kJoin) : n;
  return q;
}
// The words.  A share is the first of one cut triple at most (one that begins behind another's end in the same share; those between lie in it whole), so the triple's word is its own.  A share may end a
// triple, alone in that one's last group, and begin the next, whose first group then has the same first share: the groups that begin with their triple have words of their own, and all
// other first shares of a triple's groups lie behind its first share and up to its last, where no other triple has them.
LMB_HD int triple_counter(const Part& q) { return q.sa; }
LMB_HD int part_counter(const Part& q) { return q.groups > 1 ? kMostShares + 2 * q.first + (q.first == q.sa ? 1 : 0) : triple_counter(q); }

}  // namespace kv4
}  // namespace lmb
