// Who holds which page of a paged KV cache: host code, no kernels.
//
// Pages are counted (a page that several sequences share is held by each of them) and taken
// lowest first.  A call checks everything and reserves what it needs before it changes
// anything, so a refused one leaves the table as it was; the rows that have to move on the
// device are left as (source slot, destination slot) pairs in groups for rspx_kv_move.  What a
// call changed is noted, so that it can be taken back where its rows could not be moved.
#include <stdint.h>

#include <algorithm>
#include <new>
#include <vector>

#include "respect_amd.h"

struct rspx_pages {
  int pages, page;
  int free_pages, lowest;             // no free page below `lowest`
  std::vector<int32_t> refs;          // sequences that hold each page
  std::vector<std::vector<int32_t>> held;
  std::vector<int64_t> len;           // rows of each sequence, -1: no such sequence
  std::vector<uint32_t> seen;         // stamp of the call that named it last
  uint32_t stamp = 0;
  std::vector<int32_t> groups, moves; // of the last call
  std::vector<int32_t> left;          // pages that the call gives up
  struct Before {
    int32_t seq, pages;
    int64_t len;
  };
  struct Own {
    int32_t seq, at, old;             // held[seq][at] was `old`
  };
  std::vector<Before> before;         // of the last call: its sequences as they were,
  std::vector<Own> owned;             // and the shared pages that they left
};

namespace {

using Pages = rspx_pages;

constexpr int kMostMembers = 4096;    // of a group of sequences that begin alike: bounds the search

int64_t pages_for(const Pages& p, int64_t rows) { return (rows + p.page - 1) / p.page; }

int check_ids(Pages& p, const int32_t* ids, int n, bool distinct) {
  if (n < 0 || (n > 0 && !ids)) return RSPX_EINVAL;
  if (++p.stamp == 0) {
    std::fill(p.seen.begin(), p.seen.end(), 0u);
    p.stamp = 1;
  }
  for (int i = 0; i < n; ++i) {
    if (ids[i] < 0 || ids[i] >= (int)p.len.size() || p.len[ids[i]] < 0) return RSPX_EINVAL;
    if (distinct && p.seen[ids[i]] == p.stamp) return RSPX_EINVAL;
    p.seen[ids[i]] = p.stamp;
  }
  return RSPX_OK;
}

// The lowest free page; there is one.
int32_t take(Pages& p) {
  int i = p.lowest;
  while (p.refs[i] != 0) ++i;
  p.refs[i] = 1;
  p.lowest = i + 1;
  --p.free_pages;
  return i;
}

void drop(Pages& p, int32_t page) {
  if (--p.refs[page] == 0) {
    ++p.free_pages;
    p.lowest = std::min(p.lowest, (int)page);
  }
}

// A call's begin: the last one's moves and notes are forgotten.
void begin(Pages& p) {
  p.groups.clear();
  p.moves.clear();
  p.before.clear();
  p.owned.clear();
}

void note(Pages& p, int32_t seq) { p.before.push_back({seq, (int32_t)p.held[seq].size(), p.len[seq]}); }

int32_t slot(const Pages& p, const std::vector<int32_t>& held, int64_t row) {
  return held[row / p.page] * p.page + (int32_t)(row % p.page);
}

// Held pages with rows in [lo, hi) that others hold too.
int64_t shared(const Pages& p, const std::vector<int32_t>& held, int64_t lo, int64_t hi) {
  int64_t n = 0;
  if (hi > lo)
    for (int64_t i = lo / p.page; i < std::min<int64_t>(pages_for(p, hi), held.size()); ++i) n += p.refs[held[i]] > 1;
  return n;
}

// Gives the sequence pages of its own where it shares the ones with rows in [lo, hi), and
// copies the rows before lo that they hold.  Room for pages, moves and notes is there.  The pages
// left count as held until the call ends (leave): what its moves read is neither taken nor,
// by another sequence of the call that holds it then alone, written.
void own(Pages& p, int32_t seq, int64_t lo, int64_t hi) {
  std::vector<int32_t>& held = p.held[seq];
  if (hi <= lo) return;
  for (int64_t i = lo / p.page; i < std::min<int64_t>(pages_for(p, hi), held.size()); ++i) {
    const int32_t old = held[i];
    if (p.refs[old] <= 1) continue;
    held[i] = take(p);
    p.left.push_back(old);
    p.owned.push_back({seq, (int32_t)i, old});
    for (int64_t r = 0; r < std::min<int64_t>(p.page, lo - i * p.page); ++r) {
      p.moves.push_back(old * p.page + (int32_t)r);
      p.moves.push_back(held[i] * p.page + (int32_t)r);
    }
  }
}

void leave(Pages& p) {
  for (const int32_t page : p.left) drop(p, page);
  p.left.clear();
}

void end_group(Pages& p) {
  if (p.groups.empty()) p.groups.push_back(0);
  if ((int32_t)(p.moves.size() / 2) > p.groups.back()) p.groups.push_back((int32_t)(p.moves.size() / 2));
}

// No exception may cross the C boundary.
template <class F>
int guarded(F&& f) {
  try {
    return f();
  } catch (...) {
    return RSPX_ENOMEM;
  }
}

}  // namespace

extern "C" rspx_pages* rspx_pages_new(int pages, int page, int sequences) {
  if (pages < 1 || page < 1 || (page & (page - 1)) || sequences < 1 || (int64_t)pages * page > INT32_MAX) return nullptr;
  try {
    rspx_pages* p = new rspx_pages;
    try {
      p->pages = pages, p->page = page, p->free_pages = pages, p->lowest = 0;
      p->refs.assign(pages, 0);
      p->held.resize(sequences);
      p->len.assign(sequences, -1);
      p->seen.assign(sequences, 0);
    } catch (...) {
      delete p;
      throw;
    }
    return p;
  } catch (...) {
    return nullptr;
  }
}

extern "C" void rspx_pages_delete(rspx_pages* p) { delete p; }

extern "C" int rspx_pages_available(const rspx_pages* p) { return p ? p->free_pages : RSPX_EINVAL; }

extern "C" int64_t rspx_pages_length(const rspx_pages* p, int seq) {
  return p && seq >= 0 && seq < (int)p->len.size() ? p->len[seq] : -1;
}

extern "C" int rspx_pages_add(rspx_pages* p, const int64_t* lengths, int n, int32_t* ids) {
  if (!p || n < 0 || (n > 0 && (!lengths || !ids))) return RSPX_EINVAL;
  return guarded([&] {
    begin(*p);
    int64_t need = 0;
    for (int i = 0; i < n; ++i) {
      if (lengths[i] < 0) return RSPX_EINVAL;
      if (lengths[i] > (int64_t)p->pages * p->page) return RSPX_EFULL;
      need += pages_for(*p, lengths[i]);
    }
    if (need > p->free_pages) return RSPX_EFULL;
    int got = 0;
    for (int s = 0; s < (int)p->len.size() && got < n; ++s)
      if (p->len[s] < 0) {
        p->held[s].reserve(pages_for(*p, lengths[got]));
        ids[got++] = s;
      }
    if (got < n) return RSPX_EFULL;
    for (int i = 0; i < n; ++i) {
      p->len[ids[i]] = lengths[i];
      for (int64_t k = 0; k < pages_for(*p, lengths[i]); ++k) p->held[ids[i]].push_back(take(*p));
    }
    return RSPX_OK;
  });
}

extern "C" int rspx_pages_extend(rspx_pages* p, const int32_t* ids, int n, const int64_t* counts) {
  if (!p || (n > 0 && !counts)) return RSPX_EINVAL;
  return guarded([&] {
    begin(*p);
    if (const int rc = check_ids(*p, ids, n, true)) return rc;
    int64_t need = 0, copied = 0;
    for (int i = 0; i < n; ++i) {
      if (counts[i] < 0) return RSPX_EINVAL;
      const int64_t len = p->len[ids[i]], room = (int64_t)p->pages * p->page;
      if (counts[i] > room || len + counts[i] > room) return RSPX_EFULL;
      const int64_t own_pages = shared(*p, p->held[ids[i]], len, len + counts[i]);
      copied += own_pages;
      need += own_pages + std::max<int64_t>(0, pages_for(*p, len + counts[i]) - (int64_t)p->held[ids[i]].size());
    }
    if (need > p->free_pages) return RSPX_EFULL;
    for (int i = 0; i < n; ++i) p->held[ids[i]].reserve(pages_for(*p, p->len[ids[i]] + counts[i]));
    p->moves.reserve(2 * copied * p->page);
    p->groups.reserve(n + 1);
    p->left.reserve(copied);
    p->owned.reserve(copied);
    p->before.reserve(n);
    for (int i = 0; i < n; ++i) {
      std::vector<int32_t>& held = p->held[ids[i]];
      int64_t& len = p->len[ids[i]];
      note(*p, ids[i]);
      own(*p, ids[i], len, len + counts[i]);
      end_group(*p);
      len += counts[i];
      while ((int64_t)held.size() < pages_for(*p, len)) held.push_back(take(*p));
    }
    leave(*p);
    return RSPX_OK;
  });
}

extern "C" int rspx_pages_fork(rspx_pages* p, const int32_t* ids, int n, int copies, int32_t* out) {
  if (!p || copies < 0 || (n > 0 && copies > 0 && !out)) return RSPX_EINVAL;
  return guarded([&] {
    begin(*p);
    if (const int rc = check_ids(*p, ids, n, false)) return rc;
    const int64_t all = (int64_t)n * copies;
    if (all > (int64_t)p->len.size()) return RSPX_EFULL;
    int64_t need = 0, rows = 0;
    for (int i = 0; i < n; ++i) {
      const int64_t begun = p->len[ids[i]] % p->page;
      need += begun ? copies : 0;
      rows += begun * copies;
    }
    if (need > p->free_pages) return RSPX_EFULL;
    int got = 0;
    for (int s = 0; s < (int)p->len.size() && got < all; ++s)
      if (p->len[s] < 0) {
        p->held[s].reserve(pages_for(*p, p->len[ids[got / copies]]));
        out[got++] = s;
      }
    if (got < all) return RSPX_EFULL;
    p->moves.reserve(2 * rows);
    p->groups.reserve(all + 1);
    p->before.reserve(all);
    for (int64_t k = 0; k < all; ++k) {
      const int32_t src = ids[k / copies];
      note(*p, out[k]);
      std::vector<int32_t>& held = p->held[out[k]];
      const int64_t len = p->len[src], whole = len / p->page, begun = len % p->page;
      for (int64_t i = 0; i < whole; ++i) {
        held.push_back(p->held[src][i]);
        ++p->refs[held.back()];
      }
      if (begun) {
        const int32_t from = p->held[src][whole], to = take(*p);
        held.push_back(to);
        for (int64_t r = 0; r < begun; ++r) {
          p->moves.push_back(from * p->page + (int32_t)r);
          p->moves.push_back(to * p->page + (int32_t)r);
        }
      }
      p->len[out[k]] = len;
      end_group(*p);
    }
    return RSPX_OK;
  });
}

extern "C" int rspx_pages_compact(rspx_pages* p, const int32_t* ids, int n, const int64_t* starts, const int64_t* paths,
                                  const int64_t* ends) {
  if (!p || (n > 0 && (!starts || !ends))) return RSPX_EINVAL;
  return guarded([&] {
    begin(*p);
    if (const int rc = check_ids(*p, ids, n, true)) return rc;
    int64_t need = 0, rows = 0;
    for (int i = 0; i < n; ++i) {
      const int64_t a = i ? ends[i - 1] : 0, b = ends[i], len = p->len[ids[i]];
      if (b < a || a < 0 || starts[i] < 0 || starts[i] > len || (b > a && !paths)) return RSPX_EINVAL;
      int64_t still = 0;   // the rows that stay: path[i] == i on a first stretch only
      for (int64_t k = a; k < b; ++k) {
        if (paths[k] < 0 || paths[k] >= len - starts[i] || (k > a && paths[k] <= paths[k - 1])) return RSPX_EINVAL;
        still += paths[k] == k - a;
      }
      const int64_t copied = shared(*p, p->held[ids[i]], starts[i] + still, starts[i] + b - a);
      need += copied;
      rows += b - a - still + copied * p->page;
    }
    if (need > p->free_pages) return RSPX_EFULL;
    p->moves.reserve(2 * rows);
    p->groups.reserve(n + 1);
    p->left.reserve(need);
    p->owned.reserve(need);
    p->before.reserve(n);
    for (int i = 0; i < n; ++i) {
      const int64_t a = i ? ends[i - 1] : 0, b = ends[i];
      std::vector<int32_t>& held = p->held[ids[i]];
      note(*p, ids[i]);
      int64_t still = 0;
      while (a + still < b && paths[a + still] == still) ++still;
      // Sources in the pages as they were: a shared one is copied from, never written.  Every
      // destination lies at or before its source, and a copy's destination is a new page, so no
      // move writes what a later one reads.
      const size_t first = p->moves.size();
      for (int64_t k = a + still; k < b; ++k) {
        p->moves.push_back(slot(*p, held, starts[i] + paths[k]));
        p->moves.push_back(0);
      }
      const size_t last = p->moves.size();
      own(*p, ids[i], starts[i] + still, starts[i] + b - a);
      for (size_t m = first, k = still; m < last; m += 2, ++k) p->moves[m + 1] = slot(*p, held, starts[i] + (int64_t)k);
      end_group(*p);
      p->len[ids[i]] = starts[i] + b - a;
    }
    leave(*p);
    return RSPX_OK;
  });
}

extern "C" int rspx_pages_trim(rspx_pages* p, const int32_t* ids, int n) {
  if (!p) return RSPX_EINVAL;
  begin(*p);
  if (const int rc = check_ids(*p, ids, n, true)) return rc;
  for (int i = 0; i < n; ++i) {
    std::vector<int32_t>& held = p->held[ids[i]];
    while ((int64_t)held.size() > pages_for(*p, p->len[ids[i]])) {
      drop(*p, held.back());
      held.pop_back();
    }
  }
  return RSPX_OK;
}

extern "C" int rspx_pages_free(rspx_pages* p, const int32_t* ids, int n) {
  if (!p) return RSPX_EINVAL;
  begin(*p);
  if (const int rc = check_ids(*p, ids, n, true)) return rc;
  for (int i = 0; i < n; ++i) {
    for (const int32_t page : p->held[ids[i]]) drop(*p, page);
    p->held[ids[i]].clear();
    p->len[ids[i]] = -1;
  }
  return RSPX_OK;
}

// Every page's count is what it was, hence so are the free pages; `lowest` may lie lower.
extern "C" int rspx_pages_undo(rspx_pages* p) {
  if (!p) return RSPX_EINVAL;
  for (size_t i = p->owned.size(); i-- > 0;) {
    const rspx_pages::Own& o = p->owned[i];
    int32_t& page = p->held[o.seq][o.at];
    if (p->refs[o.old]++ == 0) --p->free_pages;
    drop(*p, page);
    page = o.old;
  }
  for (size_t i = p->before.size(); i-- > 0;) {
    const rspx_pages::Before& b = p->before[i];
    std::vector<int32_t>& held = p->held[b.seq];
    for (; (int32_t)held.size() > b.pages; held.pop_back()) drop(*p, held.back());
    p->len[b.seq] = b.len;
  }
  begin(*p);
  return RSPX_OK;
}

extern "C" int rspx_pages_moves(const rspx_pages* p, int32_t* n_groups, int32_t* n_moves) {
  if (!p || !n_groups || !n_moves) return RSPX_EINVAL;
  *n_groups = p->groups.empty() ? 0 : (int32_t)p->groups.size() - 1;
  *n_moves = (int32_t)(p->moves.size() / 2);
  return RSPX_OK;
}

extern "C" int rspx_pages_copy_moves(const rspx_pages* p, int32_t* out) {
  if (!p || (!out && !p->groups.empty())) return RSPX_EINVAL;
  std::copy(p->groups.begin(), p->groups.end(), out);
  std::copy(p->moves.begin(), p->moves.end(), out + p->groups.size());
  return RSPX_OK;
}

extern "C" int rspx_pages_width(rspx_pages* p, const int32_t* ids, int n) {
  if (!p) return RSPX_EINVAL;
  if (const int rc = check_ids(*p, ids, n, false)) return rc;
  size_t w = 0;
  for (int i = 0; i < n; ++i) w = std::max(w, p->held[ids[i]].size());
  return (int)w;
}

extern "C" int rspx_pages_table(rspx_pages* p, const int32_t* ids, int n, int width, int32_t* table, int32_t* lens) {
  if (!p || width < 0) return RSPX_EINVAL;
  if (const int rc = check_ids(*p, ids, n, false)) return rc;
  if (n > 0 && (!lens || (width > 0 && !table))) return RSPX_EINVAL;
  for (int i = 0; i < n; ++i) {
    const std::vector<int32_t>& held = p->held[ids[i]];
    if ((int)held.size() > width) return RSPX_EINVAL;
    int32_t* row = table + (int64_t)i * width;
    std::fill(std::copy(held.begin(), held.end(), row), row + width, -1);
    lens[i] = (int32_t)p->len[ids[i]];
  }
  return RSPX_OK;
}

extern "C" int rspx_pages_slots(rspx_pages* p, const int32_t* ids, int n, const int64_t* first, const int64_t* counts,
                                int32_t* out) {
  if (!p || (n > 0 && (!first || !counts))) return RSPX_EINVAL;
  if (const int rc = check_ids(*p, ids, n, false)) return rc;
  int64_t all = 0;
  for (int i = 0; i < n; ++i) {
    if (first[i] < 0 || counts[i] < 0 || first[i] > p->len[ids[i]] || counts[i] > p->len[ids[i]] - first[i]) return RSPX_EINVAL;
    all += counts[i];
  }
  if (all > 0 && !out) return RSPX_EINVAL;
  for (int i = 0; i < n; ++i)
    for (int64_t r = first[i]; r < first[i] + counts[i]; ++r) *out++ = slot(*p, p->held[ids[i]], r);
  return RSPX_OK;
}

extern "C" int rspx_pages_shared(rspx_pages* p, const int32_t* ids, int n, int64_t least, int64_t* members, int64_t* keys) {
  if (!p || least < 0) return RSPX_EINVAL;
  if (const int rc = check_ids(*p, ids, n, false)) return rc;
  if (n > 0 && (!members || !keys)) return RSPX_EINVAL;
  return guarded([&] {
    // alike[i]: the full pages that sequences i - 1 and i begin with alike.
    std::vector<int64_t> alike(n, 0), best(n + 1, 0);
    std::vector<int32_t> from(n + 1, 0);
    for (int i = 1; i < n; ++i) {
      const std::vector<int32_t>&a = p->held[ids[i - 1]], &b = p->held[ids[i]];
      const int64_t most = std::min(p->len[ids[i - 1]], p->len[ids[i]]) / p->page;
      int64_t& k = alike[i];
      while (k < most && a[k] == b[k]) ++k;
    }
    // best[j]: the most keys that need not be read again, of the sequences before j.
    for (int j = 1; j <= n; ++j) {
      best[j] = best[j - 1], from[j] = j - 1;
      int64_t common = INT64_MAX;
      for (int i = j - 2; i >= 0 && j - i <= kMostMembers; --i) {
        common = std::min(common, alike[i + 1]);
        if (common == 0) break;
        const int64_t saved = common * p->page * (j - i - 1);
        if (common * p->page >= least && best[i] + saved > best[j]) best[j] = best[i] + saved, from[j] = i;
      }
    }
    int groups = 0;
    for (int j = n; j > 0; j = from[j]) ++groups;
    int at = groups;
    for (int j = n; j > 0; j = from[j]) {
      int64_t common = j - from[j] > 1 ? INT64_MAX : 0;
      for (int i = from[j] + 1; i < j; ++i) common = std::min(common, alike[i]);
      members[--at] = j - from[j], keys[at] = common * p->page;
    }
    return groups;
  });
}

extern "C" int rspx_pages_alike(rspx_pages* p, const int32_t* ids, int n, const int64_t* members, const int64_t* keys, int groups) {
  if (!p || groups < 0 || (groups > 0 && (!members || !keys))) return RSPX_EINVAL;
  if (const int rc = check_ids(*p, ids, n, false)) return rc;
  int64_t at = 0;
  for (int i = 0; i < groups; ++i) {
    if (members[i] < 0 || keys[i] < 0 || members[i] > n - at) return RSPX_EINVAL;
    at += members[i];
  }
  if (at != n) return RSPX_EINVAL;
  for (int i = 0; i < groups; ids += members[i++]) {
    const int32_t* first = nullptr;   // the pages of the first one that is long enough
    for (int64_t k = 0; k < members[i]; ++k) {
      if (p->len[ids[k]] < keys[i]) continue;
      const int32_t* held = p->held[ids[k]].data();
      if (!first) first = held;
      else if (!std::equal(first, first + pages_for(*p, keys[i]), held)) return 0;
    }
  }
  return 1;
}
