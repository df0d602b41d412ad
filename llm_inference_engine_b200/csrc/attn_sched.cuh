// How the attention over the paged cache is dealt to workers. Pure integer arithmetic, the same on host and device:
// the kernels use it, and so does the host entry that replays a plan.
//
// A sequence b with n new tokens and `len` tokens in all has group * n query rows per KV head, row r = token * group +
// head in the group, cut into tiles of `tile` rows. An ENTRY is a (sequence, row tile); its rows see the tokens from
// `lo` to `hi` (causal, window), that is `pages` pages from `page0`; an entry with rows that see nothing counts one
// page, so that somebody writes its zeros. A UNIT is an entry's KV head. The units form one list, entry-major, then
// head, of ITEMS: ATTN_HEAD head items, which stand for what a unit costs beside its pages (bringing in q, the masked
// last page, gate and output rows: two pages' time in a busy batch), and the unit's pages. The list is cut into equal ranges, one per worker; a unit whose pages
// are split between workers leaves partial sums that a second kernel adds up in page order.
#pragma once

namespace muse {

constexpr int ATTN_PAGE = 64;   // tokens per page
constexpr int ATTN_HEAD = 2;    // head items of a unit

struct AttnEntry {
  int first, n;      // rows of the batch that hold the sequence's new tokens
  int pos;           // position of the first of them
  int row0, rows;    // this tile's rows (token * group + head in group)
  int page0, pages;  // pages its rows see; rows > 0 and nothing seen: one page that is masked whole
  int last;          // last position its rows see (-1: none)
};
// Items of a unit of the entry.
__host__ __device__ inline int attn_items(const AttnEntry& e) { return e.pages > 0 ? e.pages + ATTN_HEAD : 0; }

// cu0, cu1: the sequence's bounds in the batch as the caller gave them; len: its tokens, the new ones included.
__host__ __device__ inline AttnEntry attn_entry(int cu0, int cu1, int len, int m, int max_q, int capacity, int group, int tile, int rt,
                                                int window) {
  AttnEntry e;
  if (len < 0) len = 0;
  if (len > capacity) len = capacity;
  e.first = cu0 < 0 ? 0 : cu0 > m ? m : cu0;
  const int end = cu1 > m ? m : cu1;
  e.n = end > e.first ? end - e.first : 0;
  if (e.n > max_q) e.n = max_q;
  e.pos = len - e.n;
  const int all = e.n * group;
  e.row0 = rt * tile;
  e.rows = all - e.row0;
  if (e.rows > tile) e.rows = tile;
  e.page0 = 0;
  e.pages = 0;
  e.last = -1;
  if (e.rows <= 0) {
    e.rows = 0;
    return e;
  }
  const int p_lo = e.pos + e.row0 / group, p_hi = e.pos + (e.row0 + e.rows - 1) / group;
  if (p_hi < 0) {
    e.pages = 1;
    return e;
  }
  e.last = p_hi;
  int lo = window > 0 && p_lo >= window ? p_lo - window + 1 : 0;
  e.page0 = lo / ATTN_PAGE;
  e.pages = p_hi / ATTN_PAGE - e.page0 + 1;
  return e;
}

// `total` items dealt to `workers` in equal ranges: the first `rem` workers get one more. With fewer items than workers
// only `total` workers take part, with one item each.
struct AttnDeal {   // (the host sees to it that a call's items fit 31 bits)
  int total, base, rem;
  int workers;   // those that take part
};
__host__ __device__ inline AttnDeal attn_deal(int total, int workers) {
  AttnDeal d;
  d.total = total;
  d.workers = total < workers ? total : workers;
  d.base = d.workers > 0 ? static_cast<int>(static_cast<unsigned>(total) / static_cast<unsigned>(d.workers)) : 0;
  d.rem = total - d.base * d.workers;
  return d;
}
// First item of worker w's range (w = workers: the end).
__host__ __device__ inline int attn_range(const AttnDeal& d, int w) { return d.base * w + (w < d.rem ? w : d.rem); }
// The worker whose range holds item f.
__host__ __device__ inline int attn_worker(const AttnDeal& d, int f) {
  const int big = d.rem * (d.base + 1);   // below total
  const unsigned div = static_cast<unsigned>(f < big ? d.base + 1 : d.base), from = static_cast<unsigned>(f < big ? f : f - big);
  return (f < big ? 0 : d.rem) + static_cast<int>(from / div);
}
// Where worker w left its partial sums of the unit whose first page is item u0 (the caller knows that w has some of its
// pages, and not all): a worker has at most two partial segments, one of a unit whose first page lies at or before its
// range (slot 0) and one of a unit that begins inside it (slot 1).
__host__ __device__ inline int attn_slot_of(const AttnDeal& d, int w, int u0) { return 2 * w + (attn_range(d, w) >= u0 ? 0 : 1); }
// Workers that are the warps of a CTA, `per` of them from w on (a multiple of per), add their sums up on chip when
// nothing but this one unit's pages [u0, u1) is theirs; the sums are then in the first one's slot 0.
__host__ __device__ inline bool attn_merged(const AttnDeal& d, int w, int per, int u0, int u1) {
  return per > 1 && w + per <= d.workers && attn_range(d, w) >= u0 && attn_range(d, w + per) <= u1;
}
// The partial sums of a split unit, in page order: slot(i) for i = 0 .. parts - 1. Workers w0 .. w1 have the unit's
// pages; whole groups of `per` in between count once.
struct AttnParts {
  int w0, w1, per;
  int head, groups, parts;   // single workers in front, groups behind them; the rest is single again
  int first_slot;
};
__host__ __device__ inline AttnParts attn_parts(const AttnDeal& d, int per, int u0, int pages) {
  AttnParts p;
  p.per = per;
  p.w0 = attn_worker(d, u0);
  p.w1 = attn_worker(d, u0 + pages - 1);
  p.first_slot = attn_slot_of(d, p.w0, u0);
  const int n = p.w1 - p.w0 + 1;
  p.head = (per - p.w0 % per) % per;   // to the first group boundary
  if (p.head == 0 && !attn_merged(d, p.w0, per, u0, u0 + pages)) p.head = per;   // w0's CTA begins ahead of the unit
  if (p.head > n) p.head = n;
  p.groups = 0;
  if (per > 1 && n > p.head) {
    p.groups = (n - p.head) / per;
    // the last group may reach beyond the unit
    if (p.groups > 0 && !attn_merged(d, p.w0 + p.head + (p.groups - 1) * per, per, u0, u0 + pages)) --p.groups;
  }
  p.parts = n - p.groups * (per - 1);
  return p;
}
__host__ __device__ inline int attn_part_slot(const AttnParts& p, int i) {
  if (i == 0 && p.head > 0) return p.first_slot;
  if (i < p.head) return 2 * (p.w0 + i);
  const int g = i - p.head;
  return g < p.groups ? 2 * (p.w0 + p.head + g * p.per) : 2 * (p.w0 + p.head + p.groups * p.per + g - p.groups);
}

}  // namespace muse
