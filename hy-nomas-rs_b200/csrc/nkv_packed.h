// nkv_packed.h — the host schedule of packed attention: which (sequence,
// key/value head, rows, key tiles) each CTA takes.  Pure host code.
#pragma once

#include <algorithm>
#include <cstdint>
#include <functional>
#include <numeric>
#include <queue>
#include <utility>
#include <vector>

#include "nkv_kernels.h"

namespace nkv {

struct PackedSchedule {
  std::vector<PackedItem> items;   // by CTA
  std::vector<int32_t> cta_begin;  // [CTAs + 1]
  std::vector<PackedUnit> units;   // split units only
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

// Relative costs, in key tiles of an item with two halves (about 1.5 us): a
// tile of an item with one half takes 0.85 (two halves hide each other's
// latencies), an item 1.5 for what its start and end do not hide, a block of
// partial rows 1 more to write and merge, the merge's launch 3.
constexpr double kHalfTile = 0.85, kItem = 1.5, kPart = 1.0, kMerge = 3.0;

struct Unit {
  PackedItem it;  // t_hi = tiles of the unit
  double weight;  // cost of one tile
};

inline std::vector<Unit> make_units(const std::vector<int64_t>& q_lens, const std::vector<int64_t>& k_lens, int H,
                                    int kv_heads, bool causal, int64_t block, int halves) {
  const int64_t G = H / kv_heads, half = G * (kPackedHalfRows / G);
  std::vector<Unit> units;
  int64_t q0 = 0, k0 = 0;
  for (size_t s = 0; s < q_lens.size(); ++s) {
    const int64_t ql = q_lens[s], kl = k_lens[s], rows = ql * G;
    for (int64_t r0 = 0; r0 < rows; r0 += half * halves) {
      const int64_t n = std::min(half * halves, rows - r0);
      const int64_t lim = packed_key_limit(ql, kl, causal, block, (r0 + n - 1) / G);
      PackedItem it{};
      it.q_start = int32_t(q0), it.q_len = int32_t(ql), it.k_start = int32_t(k0), it.k_len = int32_t(kl);
      it.row0 = int32_t(r0), it.rows = int32_t(n);
      it.t_lo = 0, it.t_hi = int32_t((lim + kPackedTileKeys - 1) / kPackedTileKeys);
      it.part_row = -1;
      for (int g = 0; g < kv_heads; ++g) {
        it.kvh = g;
        units.push_back({it, n > half ? 1.0 : kHalfTile});
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

inline double item_cost(double weight, int64_t tiles, bool part) {
  return kItem + (part ? kPart : 0.0) + weight * double(tiles);
}

// Deals costs, longest first, to the CTA that is free first; returns each
// one's CTA and the time the last is done.
inline std::pair<std::vector<int32_t>, double> deal(const std::vector<double>& cost, int ctas) {
  std::vector<int32_t> order(cost.size()), cta(cost.size());
  std::iota(order.begin(), order.end(), 0);
  std::stable_sort(order.begin(), order.end(), [&](int32_t a, int32_t b) { return cost[a] > cost[b]; });
  using Free = std::pair<double, int32_t>;  // time, CTA
  std::priority_queue<Free, std::vector<Free>, std::greater<Free>> free;
  for (int32_t c = 0; c < ctas; ++c) free.push({0.0, c});
  double last = 0.0;
  for (int32_t i : order) {
    Free f = free.top();
    free.pop();
    cta[i] = f.second;
    f.first += cost[i];
    last = std::max(last, f.first);
    free.push(f);
  }
  return {cta, last};
}

// The steps and visibility bounds of an item whose tile range is set.
inline void set_steps(PackedItem* it, int64_t G, bool causal, int64_t block) {
  const int64_t half = G * (kPackedHalfRows / G), k0 = int64_t(it->t_lo) * kPackedTileKeys;
  auto limit = [&](int64_t row) { return packed_key_limit(it->q_len, it->k_len, causal, block, row / G); };
  auto steps = [&](int64_t first, int64_t rows) -> int32_t {
    if (rows <= 0) return 0;
    const int64_t lim =
        std::min<int64_t>(limit(it->row0 + first + rows - 1), int64_t(it->t_hi) * kPackedTileKeys) - k0;
    return int32_t(std::max<int64_t>(0, (lim + kPackedStepKeys - 1) / kPackedStepKeys));
  };
  it->steps0 = steps(0, std::min<int64_t>(half, it->rows));
  it->steps1 = steps(half, it->rows - half);
  it->lo_vis = int32_t(std::max<int64_t>(0, limit(it->row0) - k0));
  it->hi_vis = int32_t(std::max<int64_t>(0, limit(it->row0 + it->rows - 1) - k0));
}

}  // namespace packed_detail

// The schedule for `sms` SMs.  Items of two halves share each K / V tile
// between them; with fewer of them than SMs, items of one half are weighed
// against them (256 queries over 512 keys, 24 heads: 14.5 us against 16.5; 640
// over 20,000 stay in two halves: 155 against 221).  Key ranges are split (into
// ranges of at least four tiles) when the estimate with one to three rounds of
// items beats no split (one token over 29,056 keys, 24 heads: 65 us against
// 305; 6,496 over 6,496 stay whole).  One length of range is sought for all
// units, such that all items, those of units too short to be split among them,
// are at most one to three per SM; from four units per SM on none is sought.  So
// one long cache among many short ones (from some 440 units on 148 SMs) stays
// whole and is what the call then waits for: with 55 single tokens, 8 key/value
// heads, one cache of 60,000 keys and the others of 1,000, the longest CTA has
// 400 tiles where the mean has 46.
inline PackedSchedule packed_schedule(const std::vector<int64_t>& q_lens, const std::vector<int64_t>& k_lens, int H,
                                      int kv_heads, bool causal, int64_t block, int sms) {
  using namespace packed_detail;
  sms = std::max(sms, 1);
  std::vector<Unit> best_units;
  int64_t best_chunk = 0;
  double best = -1.0;
  for (int halves : {2, 1}) {
    if (best >= 0.0 && int64_t(best_units.size()) >= sms) break;
    std::vector<Unit> units = make_units(q_lens, k_lens, H, kv_heads, causal, block, halves);
    std::vector<int64_t> chunks{0};
    int64_t longest = 0;
    for (const Unit& u : units) longest = std::max<int64_t>(longest, u.it.t_hi);
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
      std::vector<double> cost;
      bool split = false;
      for (const Unit& u : units) {
        const int64_t p = parts_of(u.it.t_hi, c);
        split |= p > 1;
        cost.insert(cost.end(), size_t(p), item_cost(u.weight, (u.it.t_hi + p - 1) / p, p > 1));
      }
      const double f = deal(cost, sms).second + (split ? kMerge : 0.0);
      if (best < 0.0 || f < best) best = f, best_chunk = c, best_units = units;
    }
  }
  PackedSchedule out;
  std::vector<PackedItem> items;
  std::vector<double> cost;
  for (const Unit& u : best_units) {
    const int64_t p = parts_of(u.it.t_hi, best_chunk), n = u.it.t_hi;
    if (p > 1) {
      out.units.push_back({u.it.q_start, u.it.row0, u.it.rows, u.it.kvh, int32_t(out.part_rows), int32_t(p)});
      out.max_unit_rows = std::max(out.max_unit_rows, u.it.rows);
    }
    for (int64_t i = 0; i < p; ++i) {
      PackedItem it = u.it;
      it.t_lo = int32_t(n * i / p), it.t_hi = int32_t(n * (i + 1) / p);
      if (p > 1) {
        it.part_row = int32_t(out.part_rows);
        out.part_rows += u.it.rows;
      }
      set_steps(&it, H / kv_heads, causal, block);
      items.push_back(it);
      cost.push_back(item_cost(u.weight, it.t_hi - it.t_lo, p > 1));
    }
  }
  // each CTA's items together, longest first
  const int ctas = int(std::min<size_t>(items.size(), size_t(sms)));
  const std::vector<int32_t> cta = ctas ? deal(cost, ctas).first : std::vector<int32_t>();
  std::vector<int32_t> order(items.size());
  std::iota(order.begin(), order.end(), 0);
  std::stable_sort(order.begin(), order.end(), [&](int32_t a, int32_t b) {
    return cta[a] != cta[b] ? cta[a] < cta[b] : cost[a] > cost[b];
  });
  out.cta_begin.assign(size_t(ctas) + 1, 0);
  for (int32_t i : order) {
    out.items.push_back(items[i]);
    ++out.cta_begin[cta[i] + 1];
  }
  for (int c = 0; c < ctas; ++c) out.cta_begin[c + 1] += out.cta_begin[c];
  return out;
}

}  // namespace nkv
