// Parameters of the kernels on the paged 8-bit key/value cache, and the arithmetic
// that turns lengths, starts and page tables from device memory into addresses.  It
// is plain C++ so that the host can compile and test it: whatever these arrays hold,
// what comes out lies inside the buffers or is marked as not there.
#pragma once

#include <math.h>
#include <stdint.h>

#ifdef __CUDACC__
#define HC_KV_FN __host__ __device__ __forceinline__
#else
#define HC_KV_FN inline
#endif

struct HcKvCacheDev {
  void *k, *v;            // 8-bit elements, dim contiguous
  float *kScale, *vScale; // [pages, heads]
  long long pageStride, headStride, tokenStride; // elements
  long long scalePitch;                          // elements
  int pages, block, heads, dim, dtype;
};

// Where the new tokens of a call belong.
struct HcKvPlaceDev {
  const int *table;   // [seqs, width]: page of each block of a sequence
  const int *lengths; // [seqs]: tokens, the new ones included
  const int *starts;  // [seqs + 1]: rows of the new tokens; null: one row per sequence
  long long tablePitch;
  int seqs, width;
  int tokens; // rows of the new arrays
  int maxNew; // most new tokens of a sequence
};

// One sequence: rows [row, row + count) are its newest tokens, at positions
// [first, first + count).  Its rows are [allRow, allRow + allCount); those outside the
// former have no place in the cache (before position 0, behind the table's last block,
// behind maxNew).
struct HcKvSpan {
  int row, count, first, allRow, allCount;
};

HC_KV_FN HcKvSpan hcKvSpanOf(const HcKvPlaceDev &p, int block, int length, int begin, int end) {
  HcKvSpan s;
  const long long most = (long long)p.width * block;
  begin = begin < 0 ? 0 : (begin > p.tokens ? p.tokens : begin);
  end = end < begin ? begin : (end > p.tokens ? p.tokens : end);
  s.allRow = begin;
  s.allCount = end - begin;
  int count = end - begin;
  long long first = (long long)(length < 0 ? 0 : length) - count;
  if (first < 0) { // more new tokens than the sequence is long: its newest
    begin += int(-first);
    count -= int(-first);
    first = 0;
  }
  if (count > p.maxNew)
    count = p.maxNew;
  if (first + count > most)
    count = first >= most ? 0 : int(most - first);
  s.row = begin;
  s.count = count;
  s.first = int(first > most ? most : first);
  return s;
}

#ifdef __CUDACC__
__device__ __forceinline__ HcKvSpan hcKvLoadSpan(const HcKvPlaceDev &p, int block, int seq) {
  const int begin = p.starts ? p.starts[seq] : seq;
  const int end = p.starts ? p.starts[seq + 1] : seq + 1;
  return hcKvSpanOf(p, block, p.lengths[seq], begin, end);
}
#endif

// The page of a sequence's block, or -1 where the table names none that exists.
HC_KV_FN int hcKvPageOf(int entry, int pages) {
  return entry >= 0 && entry < pages ? entry : -1;
}

// Blocks that a sequence's new tokens can touch.
HC_KV_FN int hcKvTouchedBlocks(int maxNew, int block) {
  return maxNew <= 0 ? 0 : (maxNew - 1 + block - 1) / block + 1;
}

// ---- equal shares of a ragged batch ---------------------------------------------------
// The tiles of all units (sequence, head, rows) stand in one line of `total` tiles, cut
// into `shares` (at most total) of total / shares, the first ones one tile longer.  No
// share is empty.
struct HcKvShares {
  unsigned each, longer; // tiles of a share; how many have one more
  // Or, where every unit is alike: its tiles, and the shares that it is cut into (0: as
  // above).  No share then holds pieces of two units.
  unsigned unitTiles, perUnit;
};
HC_KV_FN HcKvShares hcKvSharesOf(unsigned total, unsigned shares) {
  HcKvShares s;
  s.each = total / shares;
  s.longer = total - s.each * shares;
  s.unitTiles = s.perUnit = 0;
  return s;
}
// perUnit: at most unitTiles.
HC_KV_FN HcKvShares hcKvSharesOfUnits(unsigned unitTiles, unsigned perUnit) {
  HcKvShares s;
  s.each = s.longer = 0;
  s.unitTiles = unitTiles;
  s.perUnit = perUnit;
  return s;
}
HC_KV_FN unsigned hcKvShareBegin(const HcKvShares &s, unsigned c) {
  if (s.perUnit) {
    const unsigned unit = c / s.perUnit, part = c - unit * s.perUnit;
    return unit * s.unitTiles +
           unsigned((unsigned long long)s.unitTiles * part / s.perUnit);
  }
  return c * s.each + (c < s.longer ? c : s.longer);
}
// The share that holds tile x.
HC_KV_FN unsigned hcKvShareOf(const HcKvShares &s, unsigned x) {
  if (s.perUnit) { // the last part that begins at x or before it
    const unsigned unit = x / s.unitTiles, r = x - unit * s.unitTiles;
    return unit * s.perUnit +
           unsigned(((unsigned long long)(r + 1) * s.perUnit - 1) / s.unitTiles);
  }
  const unsigned head = s.longer * (s.each + 1);
  return x < head ? x / (s.each + 1) : s.longer + (x - head) / s.each;
}

// ---- joining the parts of a unit -----------------------------------------------------
// What a part of a unit's tokens leaves for a row: the sum of its exponentials and the
// reference that they were taken against (-infinity: it saw nothing, or only NaN).
struct HcKvPart {
  float top, sum;
};
// A part whose CTA gave up a wait: nothing of its outputs is read, and the row's sum -
// so its outputs and logarithm too - becomes NaN.
HC_KV_FN HcKvPart hcKvLostPart() {
  HcKvPart p;
  p.top = -INFINITY;
  p.sum = NAN;
  return p;
}
// Its outputs' weight and its share of the sum; `power` is 2^(its top - the largest).
HC_KV_FN float hcKvPartWeight(const HcKvPart &p, float power) {
  return p.top == -INFINITY ? 0.0f : power;
}
HC_KV_FN float hcKvPartSum(const HcKvPart &p, float power) {
  return p.top == -INFINITY ? p.sum : p.sum * power;
}
