// nkv_packed.h — the host schedule of packed attention: which (sequence,
// key/value head, rows, key tiles) each CTA takes.  Pure host code.
#pragma once

#include <algorithm>
#include <cstdint>
#include <queue>
#include <vector>

#include "nkv_kernels.h"

namespace nkv {

struct PackedSchedule {
  std::vector<PackedItem> items;
  std::vector<PackedUnit> units;  // split units only
  int64_t part_rows = 0;
  int32_t max_unit_rows = 0;
};

// Keys visible to token i of a sequence.
inline int64_t packed_key_limit(int64_t q_len, int64_t k_len, bool causal, int64_t block, int64_t i) {
  if (!causal) return k_len;
  const int64_t p = i + k_len - q_len;
  if (p < 0) return 0;
  return std::min(k_len, (p / block + 1) * block);
}

namespace packed_detail {

struct Unit {
  PackedItem it;  // t_hi = tiles of the unit
  double weight;  // cost of one tile
};

// Relative costs, in tiles of 256 rows: a tile of a half-filled item takes
// about 0.7 of a full one (the two halves hide each other's softmax), an item
// about 3 for its start and end, a partial row block 2 more to write and
// merge, the merge launch 4.
constexpr double kHalfTile = 0.7, kItem = 3.0, kPart = 2.0, kMerge = 4.0;

inline std::vector<Unit> make_units(const std::vector<int64_t>& q_lens, const std::vector<int64_t>& k_lens, int H,
                                    int kv_heads, bool causal, int64_t block, int64_t rows_per_item) {
  const int64_t G = H / kv_heads;
  std::vector<Unit> units;
  int64_t q0 = 0, k0 = 0;
  for (size_t s = 0; s < q_lens.size(); ++s) {
    const int64_t ql = q_lens[s], kl = k_lens[s], rows = ql * G;
    for (int64_t r0 = 0; r0 < rows; r0 += rows_per_item) {
      const int64_t n = std::min(rows_per_item, rows - r0);
      const int64_t lim = packed_key_limit(ql, kl, causal, block, (r0 + n - 1) / G);
      PackedItem it{};
      it.q_start = int32_t(q0), it.q_len = int32_t(ql), it.k_start = int32_t(k0), it.k_len = int32_t(kl);
      it.row0 = int32_t(r0), it.rows = int32_t(n);
      it.t_lo = 0, it.t_hi = int32_t((lim + kPackedTileKeys - 1) / kPackedTileKeys);
      it.part_row = -1;
      for (int g = 0; g < kv_heads; ++g) {
        it.kvh = g;
        units.push_back({it, n > kPackedItemRows / 2 ? 1.0 : kHalfTile});
      }
    }
    q0 += ql;
    k0 += kl;
  }
  return units;
}

inline int64_t parts_of(int64_t tiles, int64_t chunk) {
  return chunk <= 0 || tiles <= chunk ? 1 : (tiles + chunk - 1) / chunk;
}

// The finishing time of the items dealt longest first to `sms` SMs.
inline double finish(const std::vector<Unit>& units, int64_t chunk, int sms) {
  std::vector<double> cost;
  bool split = false;
  for (const Unit& u : units) {
    const int64_t p = parts_of(u.it.t_hi, chunk);
    split |= p > 1;
    for (int64_t i = 0; i < p; ++i)
      cost.push_back(kItem + (p > 1 ? kPart : 0.0) + u.weight * double((u.it.t_hi + p - 1) / p));
  }
  std::sort(cost.begin(), cost.end(), [](double a, double b) { return a > b; });
  std::priority_queue<double, std::vector<double>, std::greater<double>> sm;
  double last = 0.0;
  for (double c : cost) {
    double t = c;
    if (int(sm.size()) >= sms) {
      t += sm.top();
      sm.pop();
    }
    sm.push(t);
    last = std::max(last, t);
  }
  return last + (split ? kMerge : 0.0);
}

// The steps of an item whose tile range is set.
inline void set_steps(PackedItem* it, int64_t G, bool causal, int64_t block) {
  auto limit = [&](int64_t row) { return packed_key_limit(it->q_len, it->k_len, causal, block, row / G); };
  auto steps = [&](int64_t first, int64_t rows) -> int32_t {
    if (rows <= 0) return 0;
    const int64_t lim = std::min<int64_t>(limit(it->row0 + first + rows - 1), int64_t(it->t_hi) * kPackedTileKeys) -
                        int64_t(it->t_lo) * kPackedTileKeys;
    return int32_t(std::max<int64_t>(0, (lim + kPackedStepKeys - 1) / kPackedStepKeys));
  };
  constexpr int kHalf = kPackedItemRows / 2;
  it->steps0 = steps(0, std::min(kHalf, it->rows));
  it->steps1 = steps(kHalf, it->rows - kHalf);
  it->first_partial = int32_t(std::max<int64_t>(0, limit(it->row0) / kPackedTileKeys - it->t_lo));
}

}  // namespace packed_detail

// The schedule for `sms` SMs.  Items of 256 rows share each K / V tile between
// two halves; with fewer of them than SMs, items of 128 rows are weighed
// against them.  Key ranges are split (into ranges of at least four tiles)
// when the estimate with one to three rounds of items beats no split.
inline PackedSchedule packed_schedule(const std::vector<int64_t>& q_lens, const std::vector<int64_t>& k_lens, int H,
                                      int kv_heads, bool causal, int64_t block, int sms) {
  using namespace packed_detail;
  sms = std::max(sms, 1);
  std::vector<Unit> best_units;
  int64_t best_chunk = 0;
  double best = -1.0;
  for (int64_t rows : {int64_t(kPackedItemRows), int64_t(kPackedItemRows / 2)}) {
    std::vector<Unit> units = make_units(q_lens, k_lens, H, kv_heads, causal, block, rows);
    if (best >= 0.0 && int64_t(best_units.size()) >= sms) break;
    std::vector<int64_t> chunks{0};
    int64_t tiles = 0, longest = 0;
    for (const Unit& u : units) tiles += u.it.t_hi, longest = std::max<int64_t>(longest, u.it.t_hi);
    if (int64_t(units.size()) < 4 * int64_t(sms))
      for (int64_t w = 1; w <= 3; ++w) {
        int64_t lo = 4, hi = std::max<int64_t>(longest, 4);  // the smallest chunk with at most w * sms items
        while (lo < hi) {
          const int64_t mid = (lo + hi) / 2;
          int64_t n = 0;
          for (const Unit& u : units) n += parts_of(u.it.t_hi, mid);
          if (n <= w * sms) hi = mid;
          else lo = mid + 1;
        }
        chunks.push_back(lo);
      }
    for (int64_t c : chunks) {
      const double f = finish(units, c, sms);
      if (best < 0.0 || f < best) best = f, best_chunk = c, best_units = units;
    }
  }
  // longest first; equal ones keep sequence and head order
  PackedSchedule out;
  for (const Unit& u : best_units) {
    const int64_t p = parts_of(u.it.t_hi, best_chunk), n = u.it.t_hi;
    if (p == 1) {
      out.items.push_back(u.it);
      continue;
    }
    PackedUnit pu{u.it.q_start, u.it.row0, u.it.rows, u.it.kvh, int32_t(out.part_rows), int32_t(p)};
    out.units.push_back(pu);
    out.max_unit_rows = std::max(out.max_unit_rows, u.it.rows);
    for (int64_t i = 0; i < p; ++i) {
      PackedItem it = u.it;
      it.t_lo = int32_t(n * i / p), it.t_hi = int32_t(n * (i + 1) / p);
      it.part_row = int32_t(out.part_rows);
      out.part_rows += u.it.rows;
      out.items.push_back(it);
    }
  }
  for (PackedItem& it : out.items) set_steps(&it, H / kv_heads, causal, block);
  std::stable_sort(out.items.begin(), out.items.end(),
                   [](const PackedItem& a, const PackedItem& b) { return a.t_hi - a.t_lo > b.t_hi - b.t_lo; });
  return out;
}

}  // namespace nkv
