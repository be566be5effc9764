// Host planner of windowed and 8-bit paged attention: cascade levels -> items.
//
// An item is "some consecutive queries of one group x a range of the tokens that
// they see".  What a query at position p sees of its sequence is t <= p (causal)
// and, under a window, t >= p - window or t < sinks: two runs of tokens at most
// for a tile of queries, [0, sinks) and [lowest p - window, highest p].  The two
// runs are put next to each other in a virtual index v (t = v, plus a shift from
// v = n0 on), so items, their splits and the kernels' token steps know one range
// and a window costs no partly filled steps and no second item.
//
// Narrow tiles hold up to 16 query-head rows (one query's heads, or a few), wide
// tiles up to 256.  Long ranges are split so that the items fill
// the GPU; rows in several items are partial and merged by log-sum-exp.
#include <algorithm>
#include <climits>
#include <cstring>
#include <exception>
#include <vector>

#include "beam_b200.h"

namespace be {
void set_error(const char* fmt, ...);

namespace {

struct Run {            // consecutive queries of one group, positions known
  int q_begin, q_len, kv_off, kv_len;
  int64_t pos0;         // position of query 0 in the group's tokens
  int step;             // 1: positions ascend with the queries, 0: all at pos0
  bool causal;
  int sink_end;         // first tokens of the group that stay visible
};

struct Tile {           // a run's queries [q0, q0 + ql) and the tokens they see
  int run, q0, ql;
  int n0, shift;        // virtual index: t = v + (v >= n0 ? shift : 0)
  int n;                // tokens seen by some query
  bool wide;
  bool alone;           // no other tile of its queries
};

// Steps of 128 tokens per wide item.  One CTA (item x KV head) occupies an SM, so what counts is
// when the last SM is done if CTAs go longest first to whichever SM is free: that is tried for
// whole tiles and for cuts at fractions of the average load, with 3 steps' time for a CTA's start
// and end (7.7 us against 2.8 us a step), and where the cut is what makes rows partial one more
// for writing them and 3 for their merge.  (8 prefixes of 1024 tokens under 16 beams each, 8 KV heads:
// whole tiles leave 84 of 148 SMs idle.)
int wide_chunk(const std::vector<Tile>& tiles, int64_t total_steps, int sms, int hkv) {
  int longest = 0;
  int64_t n = 0;
  for (const Tile& t : tiles)
    if (t.wide) {
      longest = std::max(longest, (t.n + 127) / 128);
      ++n;
    }
  if (n == 0 || n * hkv > 8 * (int64_t)sms) return 1 << 20;   // many CTAs: even as they are
  const double load = std::max(1.0, (double)total_steps * hkv / sms);
  int best_chunk = 1 << 20;
  int64_t best = INT64_MAX;
  std::vector<int> cost;
  std::vector<int64_t> busy;
  for (const double f : {0.0, 1.0, 0.5, 0.34, 0.25, 0.125}) {
    const int chunk = f == 0.0 ? 1 << 20 : std::max(1, (int)(load * f + 0.999));
    if (f != 0.0 && chunk >= longest) continue;
    cost.clear();
    bool split = false;
    for (const Tile& t : tiles) {
      if (!t.wide) continue;
      const int steps = (t.n + 127) / 128, ns = (steps + chunk - 1) / chunk;
      const int len = (steps + ns - 1) / ns;
      const bool partial = ns > 1 && t.alone;
      split = split || partial;
      for (int s = 0; s < steps; s += len)
        for (int h = 0; h < hkv; ++h) cost.push_back(std::min(len, steps - s) + 3 + partial);
    }
    if (cost.size() > 65536) continue;
    std::sort(cost.begin(), cost.end(), [](int a, int b) { return a > b; });
    busy.assign(sms, 0);
    auto later = [](int64_t a, int64_t b) { return a > b; };      // min-heap
    int64_t end = 0;
    for (const int c : cost) {
      std::pop_heap(busy.begin(), busy.end(), later);
      busy.back() += c;
      end = std::max(end, busy.back());
      std::push_heap(busy.begin(), busy.end(), later);
    }
    end += split ? 3 : 0;
    if (end < best) {
      best = end;
      best_chunk = chunk;
    }
  }
  return best_chunk;
}

// Tokens per narrow item.  Items are cut as if 4 CTAs, (item, KV head) pairs, ran per SM at a time.  That is the
// most that any variant of the kernel has: 8-bit rows of up to 8 query rows do, 16-bit rows of 128 dims have 2 and
// up to 16 query rows 3, for which the cuts come out finer than one wave.  (Measured on the latter kind, window
// 4096 over 64 requests, bf16, when this came: 172 us planned for 4 per SM, 185 for 3 or 6.)
// whole tiles and cuts at fractions of the average share are tried longest first, with 192 tokens'
// time for a CTA's start and end and 512 for the merge launch that a cut brings.
int narrow_chunk(const std::vector<Tile>& tiles, int64_t total, int sms, int hkv) {
  int longest = 0;
  for (const Tile& t : tiles)
    if (!t.wide) longest = std::max(longest, t.n);
  if (longest == 0) return 1 << 28;
  const int slots = std::max(1, sms * 4 / hkv);
  const int64_t share = std::max<int64_t>(1, total / slots);
  int best_chunk = 1 << 28;
  int64_t best = INT64_MAX;
  std::vector<int> cost;
  std::vector<int64_t> busy;
  for (const double f : {0.0, 1.0, 0.5, 0.34, 0.25, 0.17}) {
    const int chunk = f == 0.0 ? 1 << 28 : (int)std::max<int64_t>(128, ((int64_t)(share * f) + 63) / 64 * 64);
    if (f != 0.0 && chunk >= longest) continue;
    cost.clear();
    for (const Tile& t : tiles) {
      if (t.wide) continue;
      const int ns = (t.n + chunk - 1) / chunk, len = ((t.n + ns - 1) / ns + 63) / 64 * 64;
      for (int v = 0; v < t.n; v += len) cost.push_back(std::min(len, t.n - v) + 192);
    }
    if (cost.size() > 32768) continue;
    std::sort(cost.begin(), cost.end(), [](int a, int b) { return a > b; });
    busy.assign(slots, 0);
    auto later = [](int64_t a, int64_t b) { return a > b; };      // min-heap
    int64_t end = 0;
    for (const int c : cost) {
      std::pop_heap(busy.begin(), busy.end(), later);
      busy.back() += c;
      end = std::max(end, busy.back());
      std::push_heap(busy.begin(), busy.end(), later);
    }
    end += f != 0.0 ? 512 : 0;
    if (end < best) {
      best = end;
      best_chunk = chunk;
    }
  }
  return best_chunk;
}

int make_plan(int num_levels, const int32_t* const* qo_indptr, const int32_t* const* kv_indptr,
              const int32_t* const* kv_indices, const int32_t* const* last_page_len,
              const int32_t* num_groups, int num_queries, int page_size, int num_qo_heads,
              int num_kv_heads, int causal_last, int window_left, int num_sinks, int num_sms,
              int32_t* plan, int64_t plan_capacity, be_paged_plan_info* info) {
  if (num_levels < 1 || num_queries < 0 || page_size < 1 || num_kv_heads < 1 || num_qo_heads < 1 ||
      num_qo_heads % num_kv_heads || num_sinks < 0 || !info) {
    set_error("be_paged_plan: invalid arguments");
    return BE_EINVAL;
  }
  const int g = num_qo_heads / num_kv_heads;
  if (g > 128) {
    set_error("be_paged_plan: %d query heads per KV head (at most 128)", g);
    return BE_EINVAL;
  }
  // every extent before anything is indexed by one
  for (int l = 0; l < num_levels; ++l) {
    const int G = num_groups[l];
    if (G < 0 || (G > 0 && (qo_indptr[l][0] != 0 || kv_indptr[l][0] != 0 ||
                            qo_indptr[l][G] > num_queries))) {
      set_error("be_paged_plan: level %d indptr does not start at 0 or exceeds %d queries", l,
                num_queries);
      return BE_EINVAL;
    }
    for (int i = 0; i < G; ++i)
      if (qo_indptr[l][i + 1] < qo_indptr[l][i] || kv_indptr[l][i + 1] < kv_indptr[l][i]) {
        set_error("be_paged_plan: level %d group %d has negative extent", l, i);
        return BE_EINVAL;
      }
  }
  // tokens of every query over all levels, and the start of each level's part
  std::vector<int64_t> total(num_queries, 0);
  std::vector<int32_t> kvlist;
  std::vector<int> base(num_levels);
  std::vector<std::vector<int>> lens(num_levels);
  for (int l = 0; l < num_levels; ++l) {
    const int G = num_groups[l];
    base[l] = (int)kvlist.size();
    lens[l].resize(G);
    for (int i = 0; i < G; ++i) {
      const int np = kv_indptr[l][i + 1] - kv_indptr[l][i];
      const int last = last_page_len[l][i];
      if (np > 0 && (last < 0 || last > page_size)) {
        set_error("be_paged_plan: level %d group %d last_page_len %d outside [0, %d]", l, i, last,
                  page_size);
        return BE_EINVAL;
      }
      const int64_t len = np > 0 ? (int64_t)(np - 1) * page_size + last : 0;
      if (len > INT32_MAX / 2) {
        set_error("be_paged_plan: level %d group %d has %lld tokens", l, i, (long long)len);
        return BE_EINVAL;
      }
      lens[l][i] = (int)len;
      for (int q = qo_indptr[l][i]; q < qo_indptr[l][i + 1]; ++q) total[q] += len;
    }
    if (G > 0) kvlist.insert(kvlist.end(), kv_indices[l], kv_indices[l] + kv_indptr[l][G]);
  }
  for (int q = 0; q < num_queries; ++q)
    if (total[q] > INT32_MAX / 2) {
      set_error("be_paged_plan: query %d has %lld tokens", q, (long long)total[q]);
      return BE_EINVAL;
    }
  // positions: the last level's queries are the last tokens of their sequences
  std::vector<int64_t> pos(num_queries), off(num_queries, 0);
  for (int q = 0; q < num_queries; ++q) pos[q] = total[q] - 1;
  {
    const int l = num_levels - 1;
    for (int i = 0; i < num_groups[l]; ++i) {
      const int a = qo_indptr[l][i], b = qo_indptr[l][i + 1];
      for (int q = a; q < b; ++q) pos[q] = total[q] - (b - a) + (q - a);
    }
  }
  // runs: queries of a group whose positions in the group ascend by one, or agree
  std::vector<Run> runs;
  const bool window = window_left >= 0;
  for (int l = 0; l < num_levels; ++l) {
    const bool causal = causal_last != 0 && l == num_levels - 1;
    for (int i = 0; i < num_groups[l]; ++i) {
      const int a = qo_indptr[l][i], b = qo_indptr[l][i + 1], len = lens[l][i];
      for (int q = a; q < b;) {
        const int64_t p0 = pos[q] - off[q];
        int e = q + 1, step = 0;
        if (!causal && !window) {
          e = b;                                    // positions do not matter
        } else if (e < b) {
          const int64_t d = pos[e] - off[e] - p0;
          step = d == 1 ? 1 : 0;
          if (d == 0 || d == 1) {
            // the sinks' end must agree too: they lie at the start of the sequence
            while (e < b && pos[e] - off[e] - p0 == (int64_t)step * (e - q) && off[e] == off[q]) ++e;
          }
        }
        const int64_t sink = window ? std::max<int64_t>(0, (int64_t)num_sinks - off[q]) : 0;
        if (len > 0)
          runs.push_back({q, e - q, base[l] + kv_indptr[l][i], len, p0, step, causal,
                          (int)std::min<int64_t>(sink, len)});
        q = e;
      }
    }
    for (int i = 0; i < num_groups[l]; ++i)
      for (int q = qo_indptr[l][i]; q < qo_indptr[l][i + 1]; ++q) off[q] += lens[l][i];
  }
  // tiles
  std::vector<Tile> tiles;
  int64_t narrow_tokens = 0, wide_steps = 0;
  for (size_t r = 0; r < runs.size(); ++r) {
    const Run& R = runs[r];
    // up to 16 rows the narrow kernel reads each token once for all of them; more rows are
    // the tensor cores' (256 per tile, the tiles of a run of even size)
    const bool wide = R.q_len * g > 16;
    const int most = wide ? 256 / g : 16 / g;
    const int nt = (R.q_len + most - 1) / most, tq = (R.q_len + nt - 1) / nt;
    for (int q0 = 0; q0 < R.q_len; q0 += tq) {
      Tile t;
      t.run = (int)r;
      t.q0 = q0;
      t.ql = std::min(tq, R.q_len - q0);
      t.wide = wide;
      const int64_t pmin = R.pos0 + (int64_t)R.step * q0;
      const int64_t pmax = R.pos0 + (int64_t)R.step * (q0 + t.ql - 1);
      const int64_t hi = R.causal ? std::min<int64_t>(R.kv_len, pmax + 1) : R.kv_len;
      if (hi <= 0) continue;                        // sees nothing
      // where pages are multiples of 16 (8) tokens, so are the ends of the two runs: groups of 16 (8) tokens
      // then share a page (the kernels mask by position, so the few tokens more are not seen)
      const int64_t round = page_size % 16 == 0 ? 15 : page_size % 8 == 0 ? 7 : 0;
      const int64_t lo = window ? std::max<int64_t>(0, pmin - window_left) & ~round : 0;
      const int64_t s = window ? std::min<int64_t>((R.sink_end + round) & ~round, hi) : 0;
      if (lo <= s) {
        t.n0 = (int)hi;
        t.shift = 0;
        t.n = (int)hi;
      } else {
        t.n0 = (int)s;
        t.shift = (int)(lo - s);
        t.n = (int)(s + std::max<int64_t>(0, hi - lo));
      }
      if (t.n <= 0) continue;
      if (wide) wide_steps += (t.n + 127) / 128;
      else narrow_tokens += t.n;
      tiles.push_back(t);
    }
  }
  std::vector<int32_t> cover(num_queries, 0);
  for (const Tile& t : tiles)
    for (int q = 0; q < t.ql; ++q) cover[runs[t.run].q_begin + t.q0 + q]++;
  for (Tile& t : tiles) {
    t.alone = true;
    for (int q = 0; q < t.ql; ++q) t.alone = t.alone && cover[runs[t.run].q_begin + t.q0 + q] == 1;
  }
  const int sms = num_sms > 0 ? num_sms : 148;
  const int chunk_n = narrow_chunk(tiles, narrow_tokens, sms, num_kv_heads);
  const int chunk_w = wide_chunk(tiles, wide_steps, sms, num_kv_heads) * 128;
  struct Item {
    int tile, v0, v1, part;
  };
  std::vector<Item> items;
  cover.assign(num_queries, 0);
  for (size_t i = 0; i < tiles.size(); ++i) {
    const Tile& t = tiles[i];
    const int chunk = t.wide ? chunk_w : chunk_n, unit = t.wide ? 128 : 64;
    const int nsplit = (t.n + chunk - 1) / chunk;
    const int len = ((t.n + nsplit - 1) / nsplit + unit - 1) / unit * unit;
    for (int v = 0; v < t.n; v += len) {
      items.push_back({(int)i, v, std::min(t.n, v + len), -1});
      for (int q = 0; q < t.ql; ++q) cover[runs[t.run].q_begin + t.q0 + q]++;
    }
  }
  // partial rows and the merge lists (queries in no item merge nothing: out 0, lse -inf)
  int64_t n_parts = 0;
  std::vector<int64_t> pcount(num_queries + 1, 0);
  for (Item& it : items) {
    const Tile& t = tiles[it.tile];
    const int q = runs[t.run].q_begin + t.q0;
    bool direct = true;
    for (int i = 0; i < t.ql; ++i) direct = direct && cover[q + i] == 1;
    if (direct) {
      for (int i = 0; i < t.ql; ++i) cover[q + i] = -1;
      continue;
    }
    it.part = (int)n_parts;
    n_parts += t.ql;
    for (int i = 0; i < t.ql; ++i) pcount[q + i + 1]++;
  }
  for (int q = 0; q < num_queries; ++q) pcount[q + 1] += pcount[q];
  std::vector<int32_t> flat(pcount[num_queries]);
  {
    std::vector<int64_t> fill(pcount.begin(), pcount.end() - 1);
    for (const Item& it : items)
      if (it.part >= 0) {
        const Tile& t = tiles[it.tile];
        const int q = runs[t.run].q_begin + t.q0;
        for (int i = 0; i < t.ql; ++i) flat[fill[q + i]++] = it.part + i;
      }
  }
  std::vector<int32_t> mq, mptr{0}, mparts;
  for (int q = 0; q < num_queries; ++q) {
    if (cover[q] < 0) continue;
    mq.push_back(q);
    mparts.insert(mparts.end(), flat.begin() + pcount[q], flat.begin() + pcount[q + 1]);
    mptr.push_back((int32_t)mparts.size());
  }
  // longest first, wide tiles before narrow ones
  std::vector<int> order(items.size());
  for (size_t i = 0; i < items.size(); ++i) order[i] = (int)i;
  std::stable_sort(order.begin(), order.end(), [&](int a, int b) {
    const bool wa = tiles[items[a].tile].wide, wb = tiles[items[b].tile].wide;
    if (wa != wb) return wa;
    return items[a].v1 - items[a].v0 > items[b].v1 - items[b].v0;
  });
  be_paged_plan_info in{};
  in.n_work = (int32_t)items.size();
  for (const Item& it : items) in.n_work_wide += tiles[it.tile].wide ? 1 : 0;
  in.n_queries = num_queries;
  in.n_parts = (int32_t)n_parts;
  in.n_merge = (int32_t)mq.size();
  in.page_size = page_size;
  in.group_size = g;
  for (const Tile& t : tiles)
    if (!t.wide) in.narrow_rows = std::max(in.narrow_rows, t.ql * g);
  for (const Item& it : items) {
    const int len = it.v1 - it.v0;
    in.max_item_tokens = std::max(in.max_item_tokens, len);
    in.total_tokens = (int32_t)std::min<int64_t>(INT32_MAX, (int64_t)in.total_tokens + len);
    if (tiles[it.tile].wide) in.max_wide_tokens = std::max(in.max_wide_tokens, len);
  }
  int64_t at = BE_PLAN_HEADER_INTS;
  in.off_work = (int32_t)at;
  at += (int64_t)items.size() * (sizeof(be_paged_item) / 4);
  in.off_qlist = (int32_t)std::min<int64_t>(at, INT32_MAX);
  in.off_kvlist = in.off_qlist;
  at += (int64_t)kvlist.size();
  in.off_merge_q = (int32_t)std::min<int64_t>(at, INT32_MAX);
  at += (int64_t)mq.size();
  in.off_merge_ptr = (int32_t)std::min<int64_t>(at, INT32_MAX);
  at += (int64_t)mptr.size();
  in.off_merge_parts = (int32_t)std::min<int64_t>(at, INT32_MAX);
  at += (int64_t)mparts.size();
  if (at > INT32_MAX || n_parts > INT32_MAX) {
    set_error("be_paged_plan: plan too large (%lld ints)", (long long)at);
    return BE_EINVAL;
  }
  in.total_ints = (int32_t)at;
  *info = in;
  if (at > plan_capacity || !plan) {
    set_error("plan buffer too small: need %lld ints, have %lld", (long long)at,
              (long long)plan_capacity);
    return BE_ECAPACITY;
  }
  std::memset(plan, 0, BE_PLAN_HEADER_INTS * sizeof(int32_t));
  std::memcpy(plan, &in, sizeof(in));
  auto* out = reinterpret_cast<be_paged_item*>(plan + in.off_work);
  for (int k : order) {
    const Item& it = items[k];
    const Tile& t = tiles[it.tile];
    const Run& R = runs[t.run];
    be_paged_item w{};
    w.q_begin = R.q_begin + t.q0;
    w.q_len = t.ql;
    w.kv_off = R.kv_off;
    w.v_begin = it.v0;
    w.v_end = it.v1;
    w.n0 = t.n0;
    w.shift = t.shift;
    // positions fit 32 bits: a run's tokens do, and positions before its first token see none
    w.pos0 = (int32_t)std::max<int64_t>(R.pos0 + (int64_t)R.step * t.q0, -(1 << 30));
    w.pos_step = R.step;
    w.sink_end = R.sink_end;
    w.window = window ? std::min(window_left, 1 << 30) : -1;
    w.flags = (R.causal ? BE_ITEM_CAUSAL : 0);
    w.part_base = it.part;
    *out++ = w;
  }
  int32_t* p = plan + in.off_kvlist;
  auto put = [&](const std::vector<int32_t>& v) {
    if (!v.empty()) std::memcpy(p, v.data(), v.size() * sizeof(int32_t));
    p += v.size();
  };
  put(kvlist);
  put(mq);
  put(mptr);
  put(mparts);
  return BE_OK;
}

}  // namespace
}  // namespace be

extern "C" int be_paged_plan(int num_levels, const int32_t* const* qo_indptr,
                             const int32_t* const* kv_indptr, const int32_t* const* kv_indices,
                             const int32_t* const* last_page_len, const int32_t* num_groups,
                             int num_queries, int page_size, int num_qo_heads, int num_kv_heads,
                             int causal_last, int window_left, int num_sinks, int num_sms,
                             int32_t* plan, int64_t plan_capacity, be_paged_plan_info* info) {
  try {
    return be::make_plan(num_levels, qo_indptr, kv_indptr, kv_indices, last_page_len, num_groups,
                         num_queries, page_size, num_qo_heads, num_kv_heads, causal_last,
                         window_left, num_sinks, num_sms, plan, plan_capacity, info);
  } catch (const std::exception& e) {       // no memory for the lists
    be::set_error("be_paged_plan: %s", e.what());
    return BE_ENOMEM;
  }
}
