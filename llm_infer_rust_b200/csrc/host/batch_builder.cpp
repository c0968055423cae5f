#include "batch_builder.h"

#include <algorithm>
#include <cstring>
#include <iterator>
#include <stdexcept>
#include <string>

namespace b200 {

static int align4(int n) { return (n + 3) & ~3; }

namespace {
struct Shared {
  std::vector<int> rows;      // of the batch
  int keys = 0;               // that all of them hold in whole pages (of a division: those pages)
};
struct Held { int row, pages; const std::vector<int>* table; };      // a decode row, its whole pages

// Rows divided into sets that share pages, and those left over.
struct Division {
  std::vector<Shared> sets;
  std::vector<int> loose;
  int64_t saved = 0;          // pages that the sets' rows need not read again
};
// Rows [begin, end), which hold the same first `depth` pages.  Where they part, those of a branch form sets by themselves if that saves more
// than sharing what all have in common, which the others do; so no row takes from the others what they share, and what is saved is
// no less than in one set.
Division divide(std::vector<Held>::iterator begin, std::vector<Held>::iterator end, int depth) {
  Division d;
  if (end - begin < 2) {
    for (auto i = begin; i != end; ++i) d.loose.push_back(i->row);
    return d;
  }
  const int* lead = begin->table->data();
  int common = begin->pages;
  for (auto i = begin + 1; i != end; ++i) {
    const int* pages = i->table->data();
    common = std::min(common, i->pages);
    if (std::memcmp(lead + depth, pages + depth, sizeof(int) * (common - depth)) != 0)      // (as a rule they are the same, and this is quicker)
      common = static_cast<int>(std::mismatch(lead + depth, lead + common, pages + depth).first - lead);
  }
  depth = common;
  // the branches: rows that end here are one each
  const auto page_of = [&](const Held& h) { return h.pages > depth ? (*h.table)[depth] : 0; };
  std::stable_sort(begin, end, [&](const Held& a, const Held& b) { return page_of(a) < page_of(b); });
  std::vector<Division> branches;
  std::vector<char> apart;                       // whether a branch forms sets by itself
  std::vector<int> staying;
  int64_t saved = 0, saved_apart = 0;
  for (auto i = begin, j = i; i != end; i = j) {
    for (j = i + 1; j != end && page_of(*i) != 0 && page_of(*j) == page_of(*i); ++j) {}
    branches.push_back(divide(i, j, std::min(depth + 1, i->pages)));
    const Division& b = branches.back();
    apart.push_back(b.saved + static_cast<int64_t>(b.loose.size()) * depth > static_cast<int64_t>(j - i) * depth);
    saved_apart += b.saved;
    if (apart.back()) {
      saved += b.saved;
      staying.insert(staying.end(), b.loose.begin(), b.loose.end());
    } else {
      for (auto x = i; x != j; ++x) staying.push_back(x->row);
    }
  }
  saved += (static_cast<int64_t>(staying.size()) - 1) * depth;
  const bool set_here = staying.size() > 1 && saved >= saved_apart;
  for (size_t x = 0; x < branches.size(); ++x) {
    Division& b = branches[x];
    if (set_here && !apart[x]) continue;
    std::move(b.sets.begin(), b.sets.end(), std::back_inserter(d.sets));
    if (!set_here) d.loose.insert(d.loose.end(), b.loose.begin(), b.loose.end());
  }
  if (set_here) {
    std::sort(staying.begin(), staying.end());
    d.sets.push_back({std::move(staying), depth});
  }
  d.saved = set_here ? saved : saved_apart;
  return d;
}

// Sets of decode rows that hold the same first pages, at least two rows each.
std::vector<Shared> shared_rows(const CacheManager& cache, const BatchRequest& req) {
  std::vector<Shared> found;
  const int g = req.prefix_group;
  if (g < 0) return found;
  if (g >= cache.num_groups() || cache.group(g).window != 0) throw std::invalid_argument("rows share pages of a group that keeps all keys");
  if (cache.shared_pages(g) == 0) return found;
  const int P = cache.group(g).page_size;
  std::vector<Held> held;
  for (int r = 0; r < static_cast<int>(req.ids.size()); ++r) {
    if (req.counts[r] != 1) continue;
    const std::vector<int>& table = cache.block_table(req.ids[r], g);
    const int pages = std::min(cache.length(req.ids[r]) / P, static_cast<int>(table.size()));
    if (pages > 0) held.push_back({r, pages, &table});
  }
  const auto first = [](const Held& h) { return h.table->front(); };
  std::stable_sort(held.begin(), held.end(), [&](const Held& a, const Held& b) { return first(a) < first(b); });
  for (auto i = held.begin(), j = i; i != held.end(); i = j) {
    for (j = i + 1; j != held.end() && first(*j) == first(*i); ++j) {}
    std::vector<Shared> sets = divide(i, j, 1).sets;
    std::move(sets.begin(), sets.end(), std::back_inserter(found));
  }
  for (Shared& s : found) s.keys *= P;
  return found;
}
}  // namespace

PrefixCount count_prefix_groups(const CacheManager& cache, const BatchRequest& req) {
  PrefixCount found;
  std::vector<int> of(req.ids.size(), 0);
  for (const Shared& s : shared_rows(cache, req)) {
    found.groups += 1;
    found.saved_keys += static_cast<int64_t>(s.rows.size() - 1) * s.keys;
    found.most_shared = std::max(found.most_shared, s.keys);
    for (int r : s.rows) of[r] = s.keys;
  }
  for (size_t r = 0; r < req.ids.size(); ++r)
    if (req.counts[r] == 1) found.most_own = std::max(found.most_own, cache.length(req.ids[r]) + 1 - of[r]);
  return found;
}

BatchLayout plan_batch(const CacheManager& cache, const BatchRequest& req) {
  const int real = static_cast<int>(req.ids.size());
  if (static_cast<int>(req.counts.size()) != real || static_cast<int>(req.want_counts.size()) != real)
    throw std::invalid_argument("ids, counts and want_counts must have one entry per row");
  BatchLayout L;
  L.num_real_rows = real;
  L.num_rows = std::max(real, req.pad_rows_to);
  const int pad = L.num_rows - real;
  int tokens = 0, wants = 0;
  for (int r = 0; r < real; ++r) {
    if (req.counts[r] <= 0) throw std::invalid_argument("a row must bring at least one token");
    if (!cache.has(req.ids[r])) throw std::invalid_argument("a row names a request that holds no cache");
    for (int q = 0; q < r; ++q)
      if (req.ids[q] == req.ids[r]) throw std::invalid_argument("a request may appear once in a step");
    int prefix = cache.length(req.ids[r]);
    tokens += req.counts[r];
    wants += req.want_counts[r];
    (req.counts[r] == 1 ? L.num_decode : L.num_prefill) += 1;
    L.max_q_len = std::max(L.max_q_len, req.counts[r]);
    L.max_kv_len = std::max(L.max_kv_len, prefix + req.counts[r]);
  }
  if (static_cast<int>(req.tokens.size()) != tokens) throw std::invalid_argument("tokens do not add up to the rows' counts");
  if (static_cast<int>(req.want_index.size()) != wants) throw std::invalid_argument("want_index does not add up to want_counts");
  if (pad > 0) { L.max_q_len = std::max(L.max_q_len, 1); L.max_kv_len = std::max(L.max_kv_len, 1); }
  L.num_decode += pad;
  L.num_tokens = tokens + pad;
  L.num_logits = wants + pad;

  const int G = cache.num_groups();
  if (!req.fixed_table_width.empty() && static_cast<int>(req.fixed_table_width.size()) != G)
    throw std::invalid_argument("fixed_table_width needs one entry per cache group");
  int off = 0;
  auto take = [&off](int n) { int at = off; off += align4(std::max(n, 1)); return at; };
  L.off_tokens = take(L.num_tokens);
  L.off_positions = take(L.num_tokens);
  L.off_row_of_token = take(L.num_tokens);
  L.off_cu_q = take(L.num_rows + 1);
  L.off_kv_len = take(L.num_rows);
  L.off_prefix_len = take(L.num_rows);
  L.off_state_slot = take(L.num_rows);
  L.off_decode_rows = take(L.num_decode);
  L.off_decode_order = take(L.num_decode);
  L.off_prefill_rows = take(L.num_prefill);
  L.off_logit_rows = take(L.num_logits);
  for (int g = 0; g < G; ++g) {
    int width = 1;
    if (!req.fixed_table_width.empty()) {
      width = req.fixed_table_width[g];
    } else {
      int P = cache.group(g).page_size;
      width = std::max(1, (L.max_kv_len + P - 1) / P);
    }
    L.table_width.push_back(width);
    L.off_slots.push_back(take(L.num_tokens));
    L.off_table.push_back(take(L.num_rows * width));
  }
  const int found = req.prefix_group < 0 || L.num_decode == 0 ? 0 : req.prefix_groups > 0 ? req.prefix_groups : count_prefix_groups(cache, req).groups;
  if (found > 0) {
    L.num_prefix_groups = req.prefix_groups > 0 ? found : found + 1;
    L.off_prefix_rows = take(L.num_decode);
    L.off_prefix_groups = take(2 * L.num_prefix_groups);
  }
  L.total_ints = off;
  return L;
}

BatchLayout build_batch(const CacheManager& cache, const BatchRequest& req, int32_t* out, int64_t capacity) {
  BatchLayout L = plan_batch(cache, req);
  if (L.total_ints > capacity) throw std::length_error("the batch buffer is too small for this step");
  std::fill(out, out + L.total_ints, 0);
  const int G = cache.num_groups();
  int t = 0, w = 0, n_dec = 0, n_pf = 0, n_logit = 0;
  out[L.off_cu_q] = 0;
  for (int r = 0; r < L.num_rows; ++r) {
    const bool real = r < L.num_real_rows;
    const int count = real ? req.counts[r] : 1;
    const int prefix = real ? cache.length(req.ids[r]) : 0;
    out[L.off_kv_len + r] = prefix + count;
    out[L.off_prefix_len + r] = prefix;
    out[L.off_state_slot + r] = real ? cache.state_slot(req.ids[r]) : 0;
    out[L.off_cu_q + r + 1] = t + count;
    if (count == 1) out[L.off_decode_rows + n_dec++] = r; else out[L.off_prefill_rows + n_pf++] = r;
    if (real) {
      for (int i = 0; i < req.want_counts[r]; ++i) {
        int idx = req.want_index[w++];
        if (idx < 0 || idx >= count) throw std::out_of_range("a wanted position lies outside its row");
        out[L.off_logit_rows + n_logit++] = t + idx;
      }
    } else {
      out[L.off_logit_rows + n_logit++] = t;
    }
    for (int g = 0; g < G; ++g) {
      const int width = L.table_width[g];
      int32_t* row = out + L.off_table[g] + static_cast<int64_t>(r) * width;
      if (real) {
        const std::vector<int>& table = cache.block_table(req.ids[r], g);
        const int P = cache.group(g).page_size;
        const int used = (prefix + count + P - 1) / P;
        if (used > width) throw std::length_error("a block table is wider than the batch allows");
        for (int lp = 0; lp < used && lp < static_cast<int>(table.size()); ++lp) row[lp] = table[lp];
      }
    }
    for (int i = 0; i < count; ++i, ++t) {
      out[L.off_tokens + t] = real ? req.tokens[t] : 0;
      out[L.off_positions + t] = prefix + i;
      out[L.off_row_of_token + t] = r;
      for (int g = 0; g < G; ++g) {
        int slot = 0;
        if (real) {
          slot = cache.slot_of(req.ids[r], g, prefix + i);
          if (slot < 0)
            throw std::runtime_error("token at position " + std::to_string(prefix + i) +
                                     " has no page to be written to in cache group " + std::to_string(g));
        }
        out[L.off_slots[g] + t] = slot;
      }
    }
  }
  // Decode attention starts its CTAs in the order of this list: in a grid of several waves the long rows then begin first and
  // the short ones fill the gaps behind them.
  int32_t* order = out + L.off_decode_order;
  std::copy(out + L.off_decode_rows, out + L.off_decode_rows + n_dec, order);
  const int32_t* kv_len = out + L.off_kv_len;
  std::sort(order, order + n_dec, [kv_len](int32_t a, int32_t b) { return kv_len[a] != kv_len[b] ? kv_len[a] > kv_len[b] : a < b; });
  if (L.num_prefix_groups > 0) {
    const std::vector<Shared> shared = shared_rows(cache, req);
    if (static_cast<int>(shared.size()) >= L.num_prefix_groups) throw std::length_error("more groups of rows share pages than the batch has places for");
    std::vector<char> taken(L.num_rows, 0);
    int32_t* rows = out + L.off_prefix_rows;
    int32_t* groups = out + L.off_prefix_groups;
    int at = 0, group = 0;
    for (const Shared& s : shared) {
      groups[2 * group] = at;
      groups[2 * group++ + 1] = s.keys;
      for (int r : s.rows) {
        rows[at++] = r;
        taken[r] = 1;
        L.most_own_keys = std::max(L.most_own_keys, kv_len[r] - s.keys);
      }
      L.most_prefix_rows = std::max(L.most_prefix_rows, static_cast<int>(s.rows.size()));
      L.most_prefix_keys = std::max(L.most_prefix_keys, s.keys);
    }
    for (int g = group; g < L.num_prefix_groups; ++g) {      // the other rows share nothing; places that are left hold no rows
      groups[2 * g] = at;
      groups[2 * g + 1] = 0;
    }
    for (int d = 0; d < n_dec; ++d) {
      const int r = out[L.off_decode_rows + d];
      if (taken[r]) continue;
      rows[at++] = r;
      L.most_own_keys = std::max(L.most_own_keys, kv_len[r]);
    }
  }
  return L;
}

}  // namespace b200
