// attend_walk.cpp -- goes over the walk that divides attention over many rows, on the
// host: every step of every unit has to be done once, by parts that their workgroups count
// alike.  Batches come from standard input, one a line:
//   rep heads few_rows grid num  n_0 past_0  n_1 past_1 ...
// The first fault ends the program with a line that says which.
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>

#include <algorithm>
#include <map>
#include <tuple>
#include <vector>

#include "dm_attend_walk.h"

using namespace dm;

namespace {

struct Seq {
  int n, past;
};
struct Batch {
  int rep, heads, few, grid;
  std::vector<Seq> seqs;
};
struct Did {
  int group, slot, from, to, parts;
  bool starts, whole;
};

long line_no;
void need(bool ok, const char* what, long a = 0, long b = 0, long c = 0) {
  if (ok) return;
  printf("batch %ld: %s (%ld %ld %ld)\n", line_no, what, a, b, c);
  exit(1);
}

template <int N>
void check(const Batch& b) {
  const int num = (int)b.seqs.size();
  const ManyCost cost(b.rep, b.few);
  // the line's length without a bound on its numbers
  __int128 wide = 0;
  std::vector<int64_t> ends(N);
  int counted = 0;
  // (added in the order of the kernel's lanes and waves)
  const auto count = [&](int i0) {
    counted = i0;
    std::vector<int64_t> sum(N, 0), before(N);
    for (int i = 0; i < N && i0 + i < num; ++i)
      sum[i] = b.heads * ManyLine(cost, b.seqs[i0 + i].n, b.seqs[i0 + i].past).head();
    for (int o = 1; o < 64; o *= 2) {
      before = sum;
      for (int i = 0; i < N; ++i)
        if (i % 64 >= o) sum[i] += before[i - o];
    }
    for (int i = 0; i < N; ++i) {
      ends[i] = sum[i];
      for (int w = 0; w < i / 64; ++w) ends[i] += sum[64 * w + 63];
    }
    return ends[N - 1];
  };
  for (const Seq& q : b.seqs) {
    const ManyLine l(cost, q.n, q.past);
    const __int128 blocks = l.blocks;
    wide += b.heads * (blocks * l.one + l.per * blocks * (blocks + 1) / 2);
  }
  int64_t total = count(0);
  for (int i0 = N; i0 < num; i0 += N) total += count(i0);
  need(total >= 0 && wide == total, "the line is too long");
  const ManyShares shares(cost, total, b.grid);
  need(shares.groups <= b.grid && (shares.groups > 0) == (total > 0), "groups", shares.groups);
  if (!shares.groups) return;
  need(shares.at(0) == 0 && shares.at(shares.groups) == total, "the shares' ends");

  std::map<std::tuple<int, int, int>, std::vector<Did>> units;
  long walked = 0, most = b.grid;
  for (const Seq& q : b.seqs) most += (long)b.heads * ManyLine(cost, q.n, q.past).blocks;
  for (int g = 0; g < shares.groups; ++g) {
    need(shares.at(g) < shares.at(g + 1), "an empty share", g);
    int unfinished = 0, i0_last = -1;
    // (a workgroup has the line's first sequences when it begins)
    if (counted) count(0);
    many_walk<N>(
        cost, shares, g, num, ends.data(), count, [&](int i) {
          need(i >= 0 && i < N && counted + i < num, "a sequence that is not there", g, counted, i);
          return b.seqs[counted + i];
        },
        [&](int i0, int i, const Seq& q, const ManyPart& p, int slot) {
          need(++walked <= most, "the walk does not end", g);
          need(i0 >= i0_last && i0 == counted, "sequences of another turn", g, i0, i);
          i0_last = i0;
          const Seq& s = b.seqs[i0 + i];
          need(q.n == s.n && q.past == s.past, "another sequence");
          const ManyLine l(cost, s.n, s.past);
          need((int64_t)s.n * b.rep > b.few, "a sequence of few rows", g, i0 + i);
          need(p.head >= 0 && p.head < b.heads && p.block >= 0 && p.block < l.blocks, "a unit that is not there",
               g, p.head, p.block);
          // a block's steps are those of 64 tokens up to its last row's
          const int64_t last = std::min<int64_t>((int64_t)(p.block + 1) * 128, (int64_t)s.n * b.rep) - 1;
          need(l.steps(p.block) == (s.past + last / b.rep) / 64 + 1, "steps", l.steps(p.block));
          need(0 <= p.from && p.from <= p.to && p.to <= l.steps(p.block), "steps of a part", p.from, p.to);
          need(slot == unfinished && slot <= 1, "more than two unfinished units", g, slot);
          unfinished += !p.whole;
          units[{i0 + i, p.head, p.block}].push_back(
              {g, slot, p.from, p.to, p.starts && !p.whole ? shares.parts(g, p.end) : 1, p.starts, p.whole});
        });
  }
  size_t want = 0;
  for (int i = 0; i < num; ++i) {
    const ManyLine l(cost, b.seqs[i].n, b.seqs[i].past);
    want += (size_t)b.heads * l.blocks;
    for (int h = 0; h < b.heads; ++h)
      for (int k = 0; k < l.blocks; ++k) {
        const auto it = units.find({i, h, k});
        need(it != units.end(), "a unit that no one does", i, h, k);
        const std::vector<Did>& d = it->second;
        int at = 0;
        for (size_t x = 0; x < d.size(); ++x) {
          need(d[x].from == at, "a part that does not begin where the one before it ends", i, h, k);
          at = d[x].to;
          need(d[x].starts == (x == 0), "the part that begins a unit", i, h, k);
          need(d[x].whole == (d.size() == 1), "a whole unit", i, h, k);
          // (the join looks for later parts in the first place of the workgroups behind)
          need(d[x].group == d[0].group + (int)x && (x == 0 || d[x].slot == 0), "a part's place", i, h, k);
        }
        need(at == l.steps(k), "steps that no one does", i, h, k);
        need(d[0].parts == (int)d.size(), "the number of parts", i, h, k);
      }
  }
  need(units.size() == want, "units");
}

}  // namespace

int main() {
  Batch b;
  int num;
  while (scanf("%d %d %d %d %d", &b.rep, &b.heads, &b.few, &b.grid, &num) == 5) {
    ++line_no;
    b.seqs.resize(num);
    for (Seq& q : b.seqs)
      if (scanf("%d %d", &q.n, &q.past) != 2) return 2;
    check<256>(b);
    check<512>(b);
  }
  printf("%ld batches\n", line_no);
  return 0;
}
