// Walks the lines of csrc/kvquant_line.h as the kernels' CTAs do: every unit of every item is one CTA's, every slot of the workspace one piece's, every
// count of arrivals one sum's, and as many arrive as are waited for.  Prints what does not hold; 0 findings: exit 0.
#include <math.h>
#include <stdio.h>

#include <map>
#include <random>
#include <set>
#include <utility>
#include <vector>

#include "kvquant_line.h"

static int findings = 0;
static long long neighbours = 0;  // groups of one piece whose CTA is the first one of another item with groups
static const char* where = "";
static void found(const char* what, long long a, long long b) {
  if (findings++ < 20) printf("%s: %s (%lld, %lld)\n", where, what, a, b);
}

struct Piece {
  int cta, j0, j1;
};

// A line of items with these numbers of units, `fixed` more for each, over `ctas` of `grid` CTAs: the pieces of each item, by the kernels' arithmetic.
template <int BITS>
static std::vector<std::vector<Piece>> pieces_of(const std::vector<int>& units, int fixed, long long total, long long ctas) {
  std::vector<std::vector<Piece>> out(units.size());
  size_t item = 0;
  long long at = 0;  // where the item begins
  if (kvq_cut<BITS>(total, ctas, 0) != 0 || kvq_cut<BITS>(total, ctas, (unsigned)ctas) != total) found("the cuts leave something out", total, ctas);
  for (int c = 0; c < ctas; c++) {
    const long long lo = kvq_cut<BITS>(total, ctas, c), hi = kvq_cut<BITS>(total, ctas, c + 1);
    if (hi <= lo) found("an empty stretch", c, lo);
    for (long long u = lo; u < hi;) {
      const long long span = units[item] + fixed;
      const int j0 = (int)(u - at > fixed ? u - at - fixed : 0);
      u = at + span < hi ? at + span : hi;
      const int j1 = (int)(u - at > fixed ? u - at - fixed : 0);
      if (j0 < j1) out[item].push_back({c, j0, j1});
      if (u == at + span) { at += span; item++; }
    }
  }
  if (item != units.size()) found("items left over", (long long)item, (long long)units.size());
  return out;
}

struct Shared {  // what a launch shares, by its address: whose it is
  std::map<int, int> slots;
  std::map<int, std::pair<int, int>> tickets;  // item, group
  int slot_limit, ticket_limit;
  void slot(int at, int piece) {
    if (at < 0 || at >= slot_limit) found("a slot outside the workspace", at, slot_limit);
    if (!slots.emplace(at, piece).second) found("two pieces in one slot", at, piece);
  }
  void ticket(int at, int item, int group) {
    if (at < 0 || at >= ticket_limit) found("a ticket outside the workspace", at, ticket_limit);
    const auto r = tickets.emplace(at, std::make_pair(item, group));
    if (!r.second && r.first->second != std::make_pair(item, group)) found("two sums count at one ticket", at, item);
  }
};

static bool covered(const std::vector<Piece>& p, int n, int item) {
  int next = 0;
  for (const Piece& x : p) {
    if (x.j0 != next) { found("units that nobody has, or two", item, x.j0); return false; }
    next = x.j1;
  }
  if (next != n) { found("units at the end that nobody has", item, next); return false; }
  return true;
}

// Contexts of `heads` kv heads each, in units, over `sms` * `per` CTAs, or as many as there are units in the contexts.
static void walk_few(const std::vector<int>& units, int heads, int groups, int sms, int per, bool tight = false) {
  const int fixed = ks_fixed(groups);
  std::vector<int> items;
  long long total = 0, most = 0;
  for (int n : units)
    for (int g = 0; g < heads; g++) { items.push_back(n); total += n + fixed; most += n; }
  const int grid = (int)(tight && most < sms * per ? most : sms * per);
  const long long ctas = total < grid ? total : grid;
  const auto pieces = pieces_of<KS_BITS>(items, fixed, total, ctas);
  Shared s;
  s.slot_limit = 2 * 3 * sms;
  s.ticket_limit = 6 * sms;
  long long at = 0;
  std::set<int> grouped_from, alone;
  for (size_t i = 0; i < items.size(); i++) {
    const auto& p = pieces[i];
    const long long begin = at + fixed, last = begin + items[i] - 1;
    at += items[i] + fixed;
    if (!covered(p, items[i], (int)i) || p.size() == 1) continue;
    const int c_lo = kvq_owner(total, ctas, begin), n = kvq_owner(total, ctas, last) - c_lo + 1;
    if (c_lo != p[0].cta || n != (int)p.size()) { found("an item's CTAs", c_lo, n); continue; }
    std::map<int, int> arrived, due;
    for (int k = 0; k < n; k++) {
      if (p[k].cta != c_lo + k) found("a piece's CTA", p[k].cta, k);
      s.slot(kvq_slot(p[k].cta, p[k].j0 == 0), (int)i * 1000 + k);
      if (kvq_slot(p[k].cta, p[k].j0 == 0) != kvq_slot(c_lo + k, k == 0)) found("a piece is looked for elsewhere", k, p[k].cta);
      const KsGroup g = ks_group(k, n, c_lo);
      if (k < g.from || k >= g.to || g.from % g.step != 0 || (g.step == 1) != (n <= KS_GROUP + KS_GROUP / 2)) found("a group", k, g.from);
      if (g.ticket >= 0) {
        s.ticket(g.ticket, (int)i, g.from);
        arrived[g.ticket]++;
        due[g.ticket] = g.to - g.from;
      } else if (g.to - g.from != 1) {
        found("a group of several without a ticket", k, g.from);
      }
      if (k == g.from) {  // one CTA of each group arrives at the end
        const int end = ks_last_ticket(grid, c_lo);
        s.ticket(end, (int)i, -1);
        arrived[end]++;
        due[end] = ks_groups(n, g.step);
        if (g.step > 1) { if (k == 0) grouped_from.insert(c_lo); if (g.to - g.from == 1) alone.insert(c_lo + k); }
      }
    }
    for (const auto& d : due)
      if (arrived[d.first] != d.second) found("not as many arrive as are waited for", d.first, arrived[d.first]);
  }
  for (int c : alone) neighbours += grouped_from.count(c);
}

// Items of `tiles` key tiles, `heads` of each, over `sms` CTAs.
static void walk_chunk(const std::vector<int>& tiles, int heads, int sms) {
  std::vector<int> items;
  long long total = 0;
  for (int n : tiles)
    for (int g = 0; g < heads; g++) { items.push_back(n); total += n + KC_FIXED; }
  long long ctas = total / KC_GRAIN < sms ? total / KC_GRAIN : sms;
  if (ctas < 1) ctas = 1;
  const auto pieces = pieces_of<KC_BITS>(items, KC_FIXED, total, ctas);
  Shared s;
  s.slot_limit = 2 * sms;
  s.ticket_limit = 6 * sms;
  long long at = 0;
  for (size_t i = 0; i < items.size(); i++) {
    const auto& p = pieces[i];
    const long long begin = at + KC_FIXED;
    at += items[i] + KC_FIXED;
    if (!covered(p, items[i], (int)i) || p.size() == 1) continue;
    const int c_lo = kvq_owner(total, ctas, begin), n = kvq_owner(total, ctas, begin + items[i] - 1) - c_lo + 1;
    if (c_lo != p[0].cta || n != (int)p.size()) { found("an item's CTAs", c_lo, n); continue; }
    for (int k = 0; k < n; k++) {
      if (p[k].cta != c_lo + k) found("a piece's CTA", p[k].cta, k);
      s.slot(kvq_slot(p[k].cta, p[k].j0 == 0), (int)i * 1000 + k);
      if (kvq_slot(p[k].cta, p[k].j0 == 0) != kvq_slot(c_lo + k, k == 0)) found("a piece is looked for elsewhere", k, p[k].cta);
    }
    s.ticket(kc_ticket(c_lo), (int)i, 0);
    s.ticket(kc_done_ticket(sms, c_lo), (int)i, 1);
  }
}

static std::vector<int> units_of(const std::vector<int>& positions, int unit) {
  std::vector<int> out;
  for (int n : positions) out.push_back(n > unit ? (n + unit - 1) / unit : 1);
  return out;
}

int main() {
  // contexts whose items lie so that a CTA with the last piece of one, a group by itself, has the first piece of the next
  struct { std::vector<int> positions; int heads, groups; const char* name; } listed[] = {
      {{20724, 7137, 3324, 4400}, 8, 1, "four conversations, 8 kv heads"}, {{16527, 12298}, 8, 1, "two conversations, 8 kv heads"},
      {{131000}, 5, 1, "131000 positions, 5 kv heads"}, {{59054, 7135}, 8, 2, "two conversations, two column groups"},
      {std::vector<int>(7, 8000), 4, 1, "7 x 8000, 4 kv heads"}, {{20000, 15000}, 8, 1, "20000 and 15000, 8 kv heads"}};
  for (const auto& l : listed) {
    where = l.name;
    const long long before = neighbours;
    walk_few(units_of(l.positions, KS_UNIT), l.heads, l.groups, 148, l.groups == 1 ? 3 : 2);
    if (neighbours == before) found("no such CTA: the case shows nothing", 0, 0);
  }
  std::mt19937 rng(1);
  auto spread = [&](double lo, double hi) { return (int)exp(std::uniform_real_distribution<double>(log(lo), log(hi))(rng)); };
  for (int i = 0; i < 6000; i++) {
    where = "a drawn batch";
    std::vector<int> n;
    const int longest = spread(64, 200000);
    for (int b = spread(1, 70); b > 0; b--) n.push_back(spread(1, longest + 1));
    const int heads = 1 + (int)(rng() % 8), sms = i % 5 ? 148 : 1 + (int)(rng() % 160);
    walk_few(units_of(n, KS_UNIT), heads, 1, sms, 3, i & 1);
    walk_few(units_of(n, KS_UNIT), heads, 2 + (int)(rng() % 2), sms, 2, i & 1);
    walk_chunk(units_of(n, KC_KEYS), heads, sms);
  }
  for (int i = 0; i < 40; i++) {  // lines on either side of 2^20 units and of 2^23 tiles, and far beyond
    where = "a long line";
    const int heads = 1 + (int)(rng() % 8);
    std::vector<int> n;
    for (int b = 1 + (int)(rng() % 4); b > 0; b--) n.push_back(spread(1 << 16, 1 << 24));
    walk_few(units_of(n, KS_UNIT), heads, 1, 148, 3);
    walk_few(units_of(n, KS_UNIT), heads, 2, 148, 2);
    n.resize(n.size() * 20, 1 << 24);
    walk_chunk(units_of(n, KC_KEYS), heads, 148);
  }
  for (int near : {(1 << KS_BITS) - 4, (1 << KS_BITS) - 3, (1 << KS_BITS) - 2}) walk_few({near}, 1, 1, 148, 3);
  for (int near : {(1 << KC_BITS) - 3, (1 << KC_BITS) - 2, (1 << KC_BITS) - 1}) walk_chunk({near}, 1, 148);
  if (findings) printf("%d findings\n", findings);
  return findings != 0;
}
