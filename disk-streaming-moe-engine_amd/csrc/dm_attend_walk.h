// dm_attend_walk.h -- how attention over many rows is divided over workgroups: each
// walks its share of a line on which all units lie.  Plain integers, without anything of
// the device, so that a host program can go over the same walk.
//
// A unit is a block of 128 rows of a key head (a row is one token and one of the `rep`
// query heads that share the key head).  It has a length, about the tokens that it attends
// over; a sequence's units lie on the line head by head, block by block, the sequences
// one behind the other, and workgroups take equal shares.  Nobody talks to anybody: a
// unit that lies in several shares is done in parts, whose steps, places and number every
// workgroup has to compute alike.  All places are therefore sums of whole numbers, the same
// in whatever order they are added (sums of fractions, rounded differently from lane to
// lane, would make units that end behind the line's end or where no one else takes
// them up).  A sequence without units has no length: it ends exactly where it begins.
#pragma once
#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#endif
#include <stdint.h>

#include "dm_layout.h"

namespace dm {

constexpr int kManyRows = 128;       // rows of a block
constexpr int kManyStep = 64;        // tokens of a step
// What beginning and ending a unit costs, in tokens of its context, and the least that is given a
// workgroup.  In us, 16 heads on 2 of 256 in bf16:
//   unit  0, 160, 320, 640:        prefill of 2048 rows 247, 141, 124, 126; 4096 rows 596, 377, 301,
//                                  312; 512 behind 16000 tokens 276, 273, 274, 271; 8 prompts of
//                                  128 rows 169, 84, 74, 62
//   share 128, 256, 512, 2048:     124, 126, 124, 154; 300, 300, 301, 300; 274, 274, 274, 275; 61, 63,
//                                  74, 133; one prompt of 200 rows 39, 41, 58, 109
// So few short prompts would take smaller shares, which change nothing for long ones.
constexpr int64_t kUnitCost = 320;
constexpr int64_t kShareCost = 512;

// What a token costs, and by how much each block sees further than the one before it:
// `rep` and 128, halved together while both can be (the tokens' cost is cut to a whole number
// where rep cannot).
//
// Lengths stay below 2^62.  A call has fewer than 2^30 rows, and its sequences here have more
// than 64 of them each: at most 3/128 blocks a row.  Their queries and outputs, 2 * 64 bytes
// or more for a row and key head, lie in 2^39 bytes of device memory: fewer than 2^32 * 3/128
// units, each with up to 2^30 + 320 tokens of cost 32 (rep 4096), and a head's blocks, up to
// 2^23, of 128 or less for each block before them.
struct ManyCost {
  int rep, few_rows, shift;
  int64_t per;
  // few_rows: sequences of up to so many rows have no units
  DM_HD ManyCost(int rep, int few_rows) : rep(rep), few_rows(few_rows) {
    shift = 31 - __builtin_clz((unsigned)rep);
    if (shift > 7) shift = 7;
    per = kManyRows >> shift;
  }
  DM_HD int64_t tokens(int64_t n) const { return n * rep >> shift; }
};

// A sequence's n rows behind `past` tokens on the line.  Block b of a head is
// one + per * (b + 1) long.
struct ManyLine {
  int64_t rows, one, per;
  int blocks, past, rep;
  DM_HD ManyLine(const ManyCost& c, int n, int past)
      : rows((int64_t)n * c.rep), one(c.tokens(kUnitCost + past)), per(c.per), past(past), rep(c.rep) {
    blocks = rows > c.few_rows ? (int)((rows + kManyRows - 1) / kManyRows) : 0;
  }
  DM_HD int64_t to(int64_t b) const { return b * one + per * (b * (b + 1) / 2); }  // the blocks before b
  DM_HD int64_t head() const { return to(blocks); }
  // The steps of block b: up to its last row's token.
  DM_HD int steps(int b) const {
    const int64_t end = (int64_t)(b + 1) * kManyRows;
    const int tokens = past + (int)(((end < rows ? end : rows) - 1) / rep) + 1;
    return (tokens + kManyStep - 1) / kManyStep;
  }
};

// Equal shares of a line of `total`, for at most `most` workgroups (2^15 or fewer).
struct ManyShares {
  int64_t total, each;
  int groups, rest;
  DM_HD ManyShares(const ManyCost& c, int64_t total, int most) : total(total) {
    const int64_t least = c.tokens(kShareCost), n = (total + least - 1) / least;
    groups = n < most ? (int)n : most;
    each = groups ? total / groups : 0;
    rest = groups ? (int)(total - each * groups) : 0;
  }
  DM_HD int64_t at(int group) const { return each * group + rest * group / groups; }
  // How many workgroups from `group` on, in whose share a unit begins, have a part of it.
  DM_HD int parts(int group, int64_t end) const {
    int g = (int)(end / (each + 1));  // (a share is each or each + 1: no later one begins at end)
    g = g > group + 1 ? g : group + 1;
    while (g < groups && at(g) < end) ++g;
    return g - group;
  }
};

// What a workgroup does of a unit: steps from .. to - 1.
struct ManyPart {
  int head, block, from, to;
  bool starts, whole;  // whether the unit begins here, and whether it ends here as well
  int64_t end;         // of the unit
  // The unit at `at` of a sequence that begins at `first`, for a share that ends at hi.
  DM_HD ManyPart(const ManyLine& l, int64_t first, int64_t at, int64_t hi) {
    const int64_t length = l.head();
    head = (int)((at - first) / length);
    first += head * length;
    block = 0;
    for (int step = 1 << (31 - __builtin_clz((unsigned)l.blocks)); step; step /= 2)
      if (block + step < l.blocks && first + l.to(block + step) <= at) block += step;
    const int64_t begin = first + l.to(block);
    end = first + l.to(block + 1);
    starts = at == begin;
    whole = starts && hi >= end;
    const int steps = l.steps(block);
    // (the same for the share that ends at x and for the one that begins there)
    from = starts ? 0 : (int)((at - begin) * steps / (end - begin));
    to = hi >= end ? steps : (int)((hi - begin) * steps / (end - begin));
  }
};

// A workgroup's walk.  The line is known N sequences (a power of two) at a time:
//   count(i0)  puts the places where sequences i0, i0 + 1, ... end, from the first one's
//              beginning on, into ends; the last of them.  It has been called for 0.
//   seq(i)     the i-th of them
//   work(i0, i, seq, part, slot)   slot: how many unfinished units came before
template <int N, typename Count, typename Seq, typename Work>
DM_HD void many_walk(const ManyCost& cost, const ManyShares& shares, int group, int num, const int64_t* ends,
                     Count count, Seq seq, Work work) {
  const int64_t hi = shares.at(group + 1);
  int64_t at = shares.at(group), base = 0;
  int slot = 0;
  for (int i0 = 0; i0 < num && at < hi; i0 += N) {
    const int64_t sum = num > N ? count(i0) : shares.total;
    while (at < hi && at < base + sum) {
      int i = 0;  // the first that ends behind `at`, so one with units
      for (int step = N / 2; step; step /= 2)
        if (base + ends[i + step - 1] <= at) i += step;
      const auto q = seq(i);
      const ManyPart part(ManyLine(cost, q.n, q.past), base + (i ? ends[i - 1] : 0), at, hi);
      work(i0, i, q, part, slot);
      slot += !part.whole;
      at = part.end;
    }
    base += sum;
  }
}

}  // namespace dm
