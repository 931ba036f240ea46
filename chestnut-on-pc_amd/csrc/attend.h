// The kernels of attention of packed sequences of queries over their K/V rows, contiguous or in a
// paged cache; causal or full, through a sliding window, or with first pages that sequences share;
// query heads in groups that share a K/V head.
//
//   s_ij = scale * q_i . k_j,   o_i = sum_j softmax(s_i)_j v_j
// over the keys j < kv_len that query i may see (causal: j <= i + kv_len - q_len, the queries
// being the last places of their sequence).  A query that sees no key gets zeros.
//
// Rows.  The queries of the G heads that share a K/V head are the rows of one product:
// row r of a sequence is query r / G of head g = r % G, so that K and V pass once for all
// of them.  A wave owns 32 rows (or 16: Rows16):
//   S^T = K Q^T (v_mfma 32x32x16, A = 32 keys, B = 32 rows): lane l holds row l % 32 and
//     the keys 8 (i / 4) + 4 (l / 32) + i % 4, i < 16, of a block of 32;
//   the softmax needs the other half of the wave for its maximum and sum only;
//   O^T = V^T P^T: the lane's own exponentials, rounded to the element type, are the B operand
//     as they stand; V^T's operand takes its keys in the same order through transposed LDS reads.
// The running maximum and sum and O are f32; the weights and the output are rounded to the
// element type, the weights because the matrix product takes them so.
//
// Two forms.  WHOLE: a row sees all keys below its limit.  RANGE: it sees the keys from a lower limit
// on and the first `sinks` ones,
//   sliding window:  j > i' - window or j < sinks, i' = i + kv_len - q_len (the query's own place);
//   shared pages:    the sequences of a group hold their first keys in the same pages.  These keys
//                    and all the group's queries are one piece of work (the front), the keys behind
//                    them one for each sequence; a row's sums of both are joined.
// RANGE walks a list of blocks of 64 keys that need not follow one another, with one more limit a row, and
// keeps a bit a key, not the first key alone, of the infinities and NaN of V that it takes out of a tile.
// The kernels (their figures stand at each):
//   attend_tile_kernel  128 or 256 rows, tiles of 64 keys in LDS: prompts and chunks of one;
//                       bound by the matrix cores, the vector unit's exponentials and the
//                       tiles' loads, which run side by side in part only;
//   attend_few_kernel   16 or 32 rows, the keys over four waves: tokens one by one; bound by memory;
//   attend_join_kernel  joins the parts of rows whose keys were split over workgroups;
//   attend_join_shared_kernel  the same for the parts of shared pages and of a sequence's own keys.
#pragma once

#include <algorithm>
#include <type_traits>

#include "common.h"
#include "elem16.h"
#include "kernels.h"
#include "lanes_scan.h"

namespace ck {

struct AttendParams {
  const void* q;
  void* out;
  long q_st, q_sh, o_st, o_sh;
  const void *k, *v;
  long k_st, k_sh, v_st, v_sh;      // KV_ROWS: element strides
  const uint8_t *ks, *vs;           // KV_E4M3
  const int *table, *cu_q, *kv;     // kv: KV_ROWS: first rows [B + 1], else lengths [B]
  int B, Tq, Tk, Hkv, G, table_w, page_shift, n_pages, causal;
  float scale_log2e;
  int target, min_blocks, items;    // see Item; items: at most, and what the workspace holds
  float* ws;
  long part_rows;
  // RANGE: the window (at most 2^30) and the first keys that stay visible, or N > 0 groups of sequences
  // cu_s[g] .. cu_s[g + 1] that share their first s_lens[g] keys (as far as these fill pages)
  int window, sinks;
  int N;
  const int *cu_s, *s_lens;
  int front_items, own_items;       // N > 0: of each kind at most, by the rows that the workspace holds
};

namespace {

constexpr int AT_KEYS = 64;   // keys per tile
constexpr float AT_LOG2E = 1.4426950408889634f;

// where a sequence's K/V rows are
enum KvKind { KV_ROWS = 0, KV_PAGES = 1, KV_E4M3 = 2 };
enum Form { WHOLE = 0, RANGE = 1 };

struct Seq {
  int q0, nq, k0, nk;
};
// sequence b, held to the tensors whatever the index tensors say
template <int KV>
__device__ __forceinline__ Seq sequence(const AttendParams& p, int b) {
  Seq s;
  s.q0 = min(max(p.cu_q[b], 0), p.Tq);
  s.nq = min(max(p.cu_q[b + 1], s.q0), p.Tq) - s.q0;
  if (KV == KV_ROWS) {
    s.k0 = min(max(p.kv[b], 0), p.Tk);
    s.nk = min(max(p.kv[b + 1], s.k0), p.Tk) - s.k0;
  } else {
    s.k0 = 0;
    s.nk = (int)min((long)max(p.kv[b], 0), (long)p.table_w << p.page_shift);
  }
  return s;
}

// RANGE.  The keys that group g shares, held to whole pages of the table.
__device__ __forceinline__ int shared_keys(const AttendParams& p, int g) {
  return (int)min((long)max(p.s_lens[g], 0), (long)p.table_w << p.page_shift) >> p.page_shift << p.page_shift;
}
// The group of sequence b, or -1 (groups that do not ascend name some group or none).
__device__ __forceinline__ int group_of(const AttendParams& p, int b) {
  int lo = 0, hi = p.N;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.cu_s[mid] <= b) lo = mid;
    else hi = mid;
  }
  return p.cu_s[lo] <= b && b < p.cu_s[lo + 1] ? lo : -1;
}
// ---- which part of the work a workgroup does -------------------------------------------
// A sequence's rows make tiles of BM; a tile's keys make chunks of `c` blocks of 64, so that
// about `target` items of equal length per K/V head fill the card whatever the lengths are:
// every workgroup adds up the lengths (64 sequences a step) and finds its own item.  The
// items of a tile with one chunk write the output, the others partial sums, item by item.
// The lengths are the device's, so a captured call follows them, and no launch, counter or
// copy to the host stands before the first load.  A causal tile's items are counted as if its
// rows saw all keys; counting what they see makes shorter chunks, and more sums to join: one
// prompt of 3000 tokens, 16 heads on 4 of 64, 50 -> 43 us, four of 1371 and less 45 -> 51, mixed
// chunks 78 -> 83.  Dividing all blocks of keys exactly, with several pieces a workgroup,
// measured no faster for single tokens and 80 -> 115 us for mixed chunks (the loop over pieces
// costs the tile loop its registers).
// Where the parts of a sequence's group are: its first item, chunks, first query, rows; nch 0: no group.
struct Front {
  int base, nch, q0;
  long rows;
};
struct Item {
  int b, tile, chunk, nch, c, base;   // base: the tile's first item; b: the row of the table
  Seq s;
  // shared pages: front: the keys that the sequences b .. s1 share (s: their queries); whole: every row of every front sees
  // all of its keys.  Else first: the keys below are the front's, of which f says where its parts are; rank: the
  // tile's number among the sequences' own ones; fronts: items of all fronts
  bool front, whole;
  int s1, first, rank, fronts;
  Front f;
};

template <int KV, int BM>
__device__ __forceinline__ int tiles_of(const Seq& s, int G) {
  return (int)(((long)s.nq * G + BM - 1) / BM);
}
__device__ __forceinline__ int blocks_of(int keys) { return (keys + AT_KEYS - 1) / AT_KEYS; }
// through a window: the most blocks that a tile of BM rows of a sequence has
template <int BM>
__device__ __forceinline__ int window_blocks(const AttendParams& p, const Seq& s) {
  // its rows are of (BM - 1) / G + 2 neighbouring tokens at most, and see this many keys together, from any place on
  const int tokens = min(s.nq, (BM - 1) / p.G + 2);
  return min(blocks_of(s.nk), blocks_of(min(p.sinks, s.nk)) + (p.window + tokens + 2 * AT_KEYS - 3) / AT_KEYS);
}

// index counts items, or tiles where TILES.  False: there are not so many.
template <int KV, int BM, bool TILES, int FORM>
__device__ __forceinline__ bool find_item(const AttendParams& p, int index, Item& it) {
  const int lane = threadIdx.x & 63;
  // the first 64 sequences, one a lane
  Seq s{};
  int tiles = 0, blocks = 0;
  auto get = [&](int b0) {
    s = Seq{};
    tiles = blocks = 0;
    if (b0 + lane < p.B) {
      s = sequence<KV>(p, b0 + lane);
      tiles = tiles_of<KV, BM>(s, p.G);
      blocks = FORM == RANGE ? window_blocks<BM>(p, s) : blocks_of(s.nk);
    }
  };
  get(0);
  int c = 1 << 30;
  if (BM <= 128 && p.target) {   // tiles of 256 keep their keys whole
    float work = readlane_f32(lanes_scan((float)tiles * (float)blocks), 63);
    // (offsets that do not ascend may name 2^26 tiles of few rows or 2^30 of 128 in 64 sequences, and more
    // than an int holds in all; past 2^29 the number itself does not count)
    constexpr int MOST = 1 << 29;
    int all = min(lane63(lanes_scan(tiles)), MOST);
    for (int b0 = 64; b0 < p.B; b0 += 64) {
      get(b0);
      work += readlane_f32(lanes_scan((float)tiles * (float)blocks), 63);
      all = min(all + lane63(lanes_scan(tiles)), MOST);
    }
    // each tile adds up to one item that is not full
    const int full = max(p.target - all, (p.target + 1) >> 1);
    if (work < 16777216.f) {   // a whole number
      const int w = (int)work;
      c = max(p.min_blocks, (w + full - 1) / full);
      if (p.B <= 16) {
        // few sequences: lane i counts the items that chunks of c0 + i blocks make, and the shortest
        // chunk that does not make too many is taken (eight chunks and tokens, 80 -> 76 us)
        const int c0 = max(p.min_blocks, (w + p.target - 1) / p.target), ci = c0 + lane;
        const float inv = __builtin_amdgcn_rcpf((float)ci);
        int items = 0;
        for (int b = 0; b < p.B; ++b) {
          const int nb = __builtin_amdgcn_readlane(blocks, b), nt = __builtin_amdgcn_readlane(tiles, b);
          const int q = (int)((float)nb * inv + 0.5f);   // nb / ci to the nearest: the ceiling is it or the next
          items += nt * max(1, q + (q * ci < nb ? 1 : 0));
        }
        const unsigned long long fits = __ballot(items <= p.target);
        if (fits) c = min(c, c0 + __ffsll(fits) - 1);
      }
    } else {
      c = max(p.min_blocks, (int)fminf(work / (float)full * 1.0001f, 1e9f) + 1);
    }
    c = __builtin_amdgcn_readfirstlane(c);
    if (p.B > 64) get(0);
  }
  int base = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    if (b0) get(b0);
    const int nch = max(1, (blocks + c - 1) / c), items = tiles * nch;
    const int si = lanes_scan(items), su = TILES ? lanes_scan(tiles) : si;
    const unsigned long long m = __ballot(su > index);
    if (m) {
      const int w = __ffsll(m) - 1;
      const int local = __builtin_amdgcn_readlane(index - (su - (TILES ? tiles : items)), w);
      it.b = b0 + w;
      it.nch = __builtin_amdgcn_readlane(nch, w);
      it.tile = TILES ? local : local / it.nch;
      it.chunk = TILES ? 0 : local - it.tile * it.nch;
      it.c = c;
      it.base = base + __builtin_amdgcn_readlane(si - items, w) + it.tile * it.nch;
      it.s.q0 = __builtin_amdgcn_readlane(s.q0, w);
      it.s.nq = __builtin_amdgcn_readlane(s.nq, w);
      it.s.k0 = __builtin_amdgcn_readlane(s.k0, w);
      it.s.nk = __builtin_amdgcn_readlane(s.nk, w);
      // the compiler does not see that these are the same for all lanes
      for (int* x : {&it.b, &it.tile, &it.chunk, &it.nch, &it.c, &it.base, &it.s.q0, &it.s.nq, &it.s.k0, &it.s.nk})
        *x = __builtin_amdgcn_readfirstlane(*x);
      if (FORM == RANGE) it.front = it.whole = false;
      return true;
    }
    index -= lane63(su);
    base += lane63(si);
  }
  return false;
}

// keys that query tok of a sequence sees: all below this
__device__ __forceinline__ int keys_of(const AttendParams& p, const Seq& s, int tok) {
  return p.causal ? min(s.nk, max(0, tok + 1 + s.nk - s.nq)) : s.nk;
}

// Shared pages: the pieces are what the groups share (fronts, tiles of BMF rows) and the keys behind
// that of every sequence (tiles of BM), the fronts' items first.  All loads of the first 64 groups and 64 sequences are
// sent for together, and their answers stay in registers: what a workgroup does before its first key counts
// for as much as several blocks of keys (64 streams on two groups' pages 52.4 us where the lengths were read again and
// again, 47.3 so).  tiles_all: own tiles of all.
template <int KV, int BM, int BMF>
__device__ __forceinline__ bool find_shared(const AttendParams& p, int index, Item& it, int& tiles_all) {
  const int lane = threadIdx.x & 63;
  constexpr int MOST = 1 << 29;   // as in find_item
  it = Item{};
  // a group a lane
  int c0 = 0, c1 = 0, share = 0, s0 = 0, s1 = 0, ftiles = 0;
  Seq fs{};
  auto get_fronts = [&](int g0) {
    c0 = c1 = share = s0 = s1 = ftiles = 0;
    fs = Seq{};
    if (g0 + lane < p.N) {
      c0 = p.cu_s[g0 + lane];
      c1 = p.cu_s[g0 + lane + 1];
      share = shared_keys(p, g0 + lane);
    }
  };
  auto get_fronts_queries = [&](int g0) {
    if (g0 + lane < p.N) {
      s0 = min(max(c0, 0), p.B);
      s1 = min(max(c1, s0), p.B);
      fs.q0 = min(max(p.cu_q[s0], 0), p.Tq);
      fs.nq = min(max(p.cu_q[s1], fs.q0), p.Tq) - fs.q0;
      fs.nk = share;
      ftiles = tiles_of<KV, BMF>(fs, p.G);
    }
  };
  // a sequence a lane
  Seq s{};
  int g = -1, first = 0, tiles = 0, blocks = 0;
  auto get_own = [&](int b0) {
    s = Seq{};
    if (b0 + lane < p.B) s = sequence<KV>(p, b0 + lane);
  };
  auto group_own = [&](int b0) {
    g = -1;
    first = tiles = blocks = 0;
    if (p.N <= 64) {
      for (int j = 0; j < p.N; ++j)
        if (b0 + lane >= __builtin_amdgcn_readlane(c0, j) && b0 + lane < __builtin_amdgcn_readlane(c1, j)) {
          g = j;
          first = __builtin_amdgcn_readlane(share, j);
        }
    } else if (b0 + lane < p.B) {
      g = group_of(p, b0 + lane);
      if (g >= 0) first = shared_keys(p, g);
    }
    if (b0 + lane < p.B) {
      tiles = tiles_of<KV, BM>(s, p.G);
      blocks = max(0, blocks_of(s.nk) - first / AT_KEYS);
    }
  };
  get_fronts(0);
  get_own(0);
  get_fronts_queries(0);
  group_own(0);
  // how long a chunk is, whether every query of every group sees all that its group shares, and how many own tiles there are.
  // (One answer for all groups: a single sequence that ends within the shared keys sends all fronts' tiles through the masked
  // path; the 64 streams of two groups with one such 104.6 us for 39.2, and 41.2 with that one in no group.)
  float work = readlane_f32(lanes_scan((float)ftiles * (float)blocks_of(fs.nk)), 63);
  for (int g0 = 64; g0 < p.N; g0 += 64) {
    get_fronts(g0);
    get_fronts_queries(g0);
    work += readlane_f32(lanes_scan((float)ftiles * (float)blocks_of(fs.nk)), 63);
  }
  bool whole = true;
  tiles_all = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    if (b0) {
      get_own(b0);
      group_own(b0);
    }
    work += readlane_f32(lanes_scan((float)tiles * (float)blocks), 63);
    tiles_all = min(tiles_all + lane63(lanes_scan(tiles)), MOST);
    whole = whole && __all(g < 0 || s.nq <= 0 || keys_of(p, s, 0) >= first);
  }
  int c = 1 << 30;
  if (p.target)
    c = max(p.min_blocks, work < 16777216.f ? ((int)work + p.target - 1) / p.target : (int)fminf(work / (float)p.target * 1.0001f, 1e9f) + 1);
  auto chunks = [&](int blocks) { return max(1, (blocks + c - 1) / c); };
  // up to half as long again where no more items than run at once come of it (a second round begins anew: 32 tokens on
  // 37376 shared keys 36.0 -> 34.4 us, 64 on two groups' 47.4 -> 44; twice as long, with many tiny tiles, 37 -> 41)
  if (p.target && p.N <= 64 && p.B <= 64) {
    const int least = c;
#pragma unroll 1
    for (int i = 4; i <= 6; ++i) {
      c = max(least * i / 4, least + (i > 4));
      if (lane63(lanes_scan(ftiles * chunks(blocks_of(fs.nk)) + tiles * chunks(blocks))) <= p.target) break;
      if (i == 6) {
        c = least;
        break;
      }
    }
  }
  c = __builtin_amdgcn_readfirstlane(c);
  // the fronts
  it.c = c;
  it.whole = __builtin_amdgcn_readfirstlane(whole ? 1 : 0);
  bool found = false;
  int base = 0, fbase = 0, fnch = 0;
  for (int g0 = 0; g0 < p.N; g0 += 64) {
    if (p.N > 64) {
      get_fronts(g0);
      get_fronts_queries(g0);
    }
    fnch = chunks(blocks_of(fs.nk));
    const int items = ftiles * fnch, si = lanes_scan(items);
    fbase = base + si - items;
    const unsigned long long m = __ballot(base + si > index);
    if (m && !found) {
      const int w = __ffsll(m) - 1, local = index - __builtin_amdgcn_readlane(fbase, w);
      found = true;
      it.front = true;
      it.nch = __builtin_amdgcn_readlane(fnch, w);
      // all tiles' first chunks, then their second ones ...: the last ones are short.  R chunks at a time, so that the tiles
      // of one chunk, R workgroups a K/V head apart, are on one XCD, which workgroups go to in turn (those 64 streams
      // 121 -> 93 MB read, 45.9 -> 44.9 us)
      const int nt = __builtin_amdgcn_readlane(ftiles, w), R = p.Hkv < 8 ? 8 / p.Hkv : 1;
      const int at = local / (nt * R), in = local - at * nt * R, r = min(R, it.nch - at * R);
      it.tile = in / r;
      it.chunk = at * R + in - it.tile * r;
      it.base = __builtin_amdgcn_readlane(fbase, w) + it.chunk * (nt - 1) + it.tile;   // (+ chunk: where its sums go)
      it.b = min(__builtin_amdgcn_readlane(s0, w), p.B - 1);
      it.s1 = __builtin_amdgcn_readlane(s1, w);
      it.s.q0 = __builtin_amdgcn_readlane(fs.q0, w);
      it.s.nq = __builtin_amdgcn_readlane(fs.nq, w);
      it.s.k0 = 0;
      it.s.nk = __builtin_amdgcn_readlane(fs.nk, w);
      it.first = it.rank = 0;
    }
    base += lane63(si);
  }
  it.fronts = base;
  // the sequences' own keys
  int rank = 0;
  for (int b0 = 0; b0 < p.B && !found; b0 += 64) {
    if (p.B > 64) {
      get_own(b0);
      group_own(b0);
    }
    const int nch = chunks(blocks), items = tiles * nch, si = lanes_scan(items), so = lanes_scan(tiles);
    const unsigned long long m = __ballot(base + si > index);
    if (m) {
      const int w = __ffsll(m) - 1, before = base + __builtin_amdgcn_readlane(si - items, w), local = index - before;
      found = true;
      it.front = false;
      it.nch = __builtin_amdgcn_readlane(nch, w);
      it.tile = local / it.nch;
      it.chunk = local - it.tile * it.nch;
      it.base = before + it.tile * it.nch;
      it.b = b0 + w;
      it.s1 = 0;
      it.s.q0 = __builtin_amdgcn_readlane(s.q0, w);
      it.s.nq = __builtin_amdgcn_readlane(s.nq, w);
      it.s.k0 = 0;
      it.s.nk = __builtin_amdgcn_readlane(s.nk, w);
      it.first = __builtin_amdgcn_readlane(first, w);
      it.rank = rank + __builtin_amdgcn_readlane(so - tiles, w) + it.tile;
      it.f = Front{};
      int of = __builtin_amdgcn_readlane(g, w);
      if (of >= 0 && it.first > 0) {
        if (p.N > 64) {   // the group's items, from the first one's on
          int at = 0;
          for (int g0 = 0; g0 <= of; g0 += 64) {
            get_fronts(g0);
            get_fronts_queries(g0);
            fnch = chunks(blocks_of(fs.nk));
            const int n = ftiles * fnch, sn = lanes_scan(n);
            fbase = at + sn - n;
            at += lane63(sn);
          }
          of &= 63;
        }
        it.f.base = __builtin_amdgcn_readlane(fbase, of);
        it.f.nch = __builtin_amdgcn_readlane(fnch, of);
        it.f.q0 = __builtin_amdgcn_readlane(fs.q0, of);
        it.f.rows = (long)__builtin_amdgcn_readlane(fs.nq, of) * p.G;
        if (it.f.base < 0) it.f.nch = 0;
      }
    }
    base += lane63(si);
    rank += lane63(so);
  }
  // the compiler does not see that these are the same for all lanes
  for (int* x : {&it.b, &it.tile, &it.chunk, &it.nch, &it.base, &it.s.q0, &it.s.nq, &it.s.nk, &it.s1, &it.first, &it.rank, &it.fronts,
                 &it.f.base, &it.f.nch, &it.f.q0})
    *x = __builtin_amdgcn_readfirstlane(*x);
  it.front = __builtin_amdgcn_readfirstlane(it.front ? 1 : 0);
  return found;
}

// RANGE: the keys that a row sees: those below lim that are from lo on, or below the sinks.
struct Sees {
  int lim, lo;
};
template <int KV>
__device__ __forceinline__ Sees sees(const AttendParams& p, const Item& it, int tok) {
  if (!it.front) {
    const int lim = keys_of(p, it.s, tok);
    return Sees{lim, p.N ? it.first : max(0, lim - p.window)};
  }
  if (it.whole) return Sees{it.s.nk, 0};
  const int t = it.s.q0 + tok;
  int lo = it.b, hi = max(it.s1, it.b + 1);   // the last sequence of the group that begins at or before t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.cu_q[mid] <= t) lo = mid;
    else hi = mid;
  }
  const Seq s = sequence<KV>(p, lo);
  const int at = t - s.q0;
  return Sees{at < 0 || at >= s.nq ? 0 : min(it.s.nk, keys_of(p, s, at)), 0};
}
// RANGE: the blocks of 64 keys that a tile's rows see together: the first sn, then those from
// block w0 on, nb in all.  Of these its rows all see all keys of the blocks below fs and of fa .. fb.
struct Blocks {
  int sn, w0, nb, fs, fa, fb, lim;   // lim: no row sees a key from here on
  __device__ __forceinline__ int key(int v) const { return (v < sn ? v : v - sn + w0) * AT_KEYS; }
};
template <int KV>
__device__ __forceinline__ Blocks blocks(const AttendParams& p, const Item& it, int tok0, int tok1) {
  int lim_lo, lo_lo = 0, lo_hi = 0;
  Blocks x;
  if (it.front) {
    lim_lo = it.whole ? it.s.nk : 0;
    x.lim = it.s.nk;
  } else {
    lim_lo = keys_of(p, it.s, tok0);
    x.lim = keys_of(p, it.s, tok1);
    lo_lo = p.N ? it.first : max(0, lim_lo - p.window);
    lo_hi = p.N ? it.first : max(0, x.lim - p.window);
  }
  x.sn = blocks_of(min(p.sinks, x.lim));
  x.w0 = max(lo_lo / AT_KEYS, x.sn);
  x.nb = x.sn + max(0, blocks_of(x.lim) - x.w0);
  x.fs = min(min(p.sinks, lim_lo) / AT_KEYS, x.sn);
  x.fa = max(blocks_of(lo_hi), x.w0) - x.w0 + x.sn;
  x.fb = lim_lo / AT_KEYS - x.w0 + x.sn;
  // (the compiler does not see that these are the same for all lanes)
  for (int* i : {&x.sn, &x.w0, &x.nb, &x.fs, &x.fa, &x.fb, &x.lim}) *i = __builtin_amdgcn_readfirstlane(*i);
  return x;
}

// ---- LDS tiles --------------------------------------------------------------------------
// Element offsets of 16-byte chunk c of a row: K's fragments are one chunk of 16 consecutive
// rows, V's four chunks of 4 consecutive rows (Rows16: two of 8); all hit every bank once this way.
template <int HD>
__device__ __forceinline__ int k_at(int key, int c) {
  return HD == 128 ? key * HD + ((c ^ (key & 15)) << 3) : key * HD + ((c ^ ((key >> 1) & 7)) << 3);
}
template <int HD>
__device__ __forceinline__ int v_at(int key, int c) {
  return key * HD + ((c ^ (HD == 128 ? (key & 3) << 2 : (key & 2) << 1) ^ ((key >> 1) & 2)) << 3);
}

// KEYS rows of K or V on their way to LDS by NT threads.  Places behind the last key repeat
// it.  A wave's rows of one load lie in one group of 16, so on one page.
// ONCE: this workgroup alone reads them, past the caches.  JUMPS: a tile need not follow the one before.
template <typename T, int HD, int KV, int KEYS, int NT, bool V, bool ONCE = false, bool JUMPS = false>
struct Stage {
  typedef typename Elem<T>::v2 v2;
  typedef typename Elem<T>::v8 v8;
  static constexpr int EPL = KV == KV_E4M3 && KEYS * HD / 16 >= NT ? 16 : 8;   // elements per load
  static constexpr int CPR = HD / EPL, N = KEYS * CPR / NT, RPL = NT / CPR;
  static constexpr int BPL = KV == KV_E4M3 ? EPL : 16;                         // bytes per load
  typedef std::conditional_t<BPL == 16, u32x4_t, u32x2_t> raw;
  static_assert(N * NT == KEYS * CPR && (RPL >= 16 || 16 % RPL == 0), "tile");
  raw x[N];
  unsigned scale[N];
  // lane l: the page of group l (of 16 keys) of the window of 1024 keys that is read, and of the next
  int page, later, window;

  static __device__ __forceinline__ int at(int key, int c) { return V ? v_at<HD>(key, c) : k_at<HD>(key, c); }
  __device__ __forceinline__ int pages(const AttendParams& p, const Item& it, int w, int lane) const {
    const int key = min(w * 1024 + lane * 16, it.s.nk - 1);
    return p.table[(long)it.b * p.table_w + (key >> p.page_shift)];
  }
  // Load i brings the rows from first(key0, i) on to a wave: their place in the cache (or among
  // the packed rows) is the same for all lanes but for lane_row() rows of `pitch` bytes.
  static __device__ __forceinline__ int lane_row(int lane) { return lane / CPR; }
  static __device__ __forceinline__ int first(int key0, int i, int wave) { return key0 + i * RPL + wave * (64 / CPR); }
  // place of a key; of: the load's first row, whose group of 16 it is in (or the last key's)
  __device__ __forceinline__ long row_of(const AttendParams& p, const Item& it, int hk, int key, int of) const {
    if constexpr (KV == KV_ROWS) return it.s.k0 + key;
    const long pg = min(max(__builtin_amdgcn_readlane(page, (of >> 4) & 63), 0), p.n_pages - 1);
    return ((pg * p.Hkv + hk) << p.page_shift) + (key & ((1 << p.page_shift) - 1));
  }
  static __device__ __forceinline__ const char* base(const AttendParams& p, int hk) {
    const char* b = static_cast<const char*>(V ? p.v : p.k);
    if constexpr (KV == KV_ROWS) b += (long)hk * (V ? p.v_sh : p.k_sh) * 2;
    return b;
  }
  static __device__ __forceinline__ long pitch(const AttendParams& p) {
    if constexpr (KV == KV_ROWS) return (V ? p.v_st : p.k_st) * 2;
    return HD / EPL * BPL;
  }
  // bytes from a load's first row to the lane's piece, and of the piece within its row; KV_ROWS:
  // the first row of the next tile, which is `ahead` keys after this one, and bytes between loads
  unsigned lane_off;
  int piece;
  uintptr_t next;
  long between, ahead;
  __device__ __forceinline__ void begin(const AttendParams& p, const Item& it, int hk, int key0, int keys_ahead, int lane,
                                        int wave, bool swizzled) {
    // straight to LDS a wave's 64 pieces of 16 bytes land side by side, so each lane fetches the
    // chunk that belongs in its place
    piece = swizzled ? (at(first(0, 0, wave) + lane_row(lane), lane % CPR) >> 3) % CPR * 16 : lane % CPR * BPL;
    lane_off = lane_row(lane) * (unsigned)pitch(p) + piece;
    asm volatile("" : "+v"(lane_off));
    if constexpr (KV == KV_ROWS) {
      next = (uintptr_t)base(p, hk) + (it.s.k0 + first(key0, 0, wave)) * pitch(p);
      between = RPL * pitch(p);
      ahead = keys_ahead * pitch(p);
    } else {
      window = key0 >> 10;
      page = pages(p, it, window, lane);
      later = pages(p, it, window + 1, lane);
    }
  }
  // f(i, address of the lane's piece, its row's number) for every load of the next tile
  template <typename F>
  __device__ __forceinline__ void rows(const AttendParams& p, const Item& it, int hk, int key0, int lane, int wave, F f) {
    typedef const __attribute__((address_space(1))) char* glob_t;
    if constexpr (KV != KV_ROWS) {
      if (key0 >> 10 != window) {
        page = later;
        if (JUMPS && key0 >> 10 != window + 1) page = pages(p, it, key0 >> 10, lane);
        window = key0 >> 10;
        later = pages(p, it, window + 1, lane);
      }
    } else if constexpr (JUMPS) {
      next = (uintptr_t)base(p, hk) + (it.s.k0 + first(key0, 0, wave)) * pitch(p);
    }
    if (key0 + KEYS <= it.s.nk) {
      uintptr_t a = next;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        long row = 0;
        if constexpr (KV != KV_ROWS) {
          row = row_of(p, it, hk, first(key0, i, wave), first(key0, i, wave));
          a = (uintptr_t)(base(p, hk) + row * pitch(p));
        }
        // in scalar registers: the same address in vector ones costs four multiplications
        const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)a), hi = __builtin_amdgcn_readfirstlane((unsigned)(a >> 32));
        f(i, (glob_t)(((uintptr_t)hi << 32) | lo) + lane_off, row + lane_row(lane));
        if constexpr (KV == KV_ROWS) a += between;
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const long row = row_of(p, it, hk, min(first(key0, i, wave) + lane_row(lane), it.s.nk - 1), first(key0, i, wave));
        f(i, (glob_t)(base(p, hk) + row * pitch(p) + piece), row);
      }
    }
    if constexpr (KV == KV_ROWS && !JUMPS) next += ahead;
  }
  // sends for the rows; store() leaves them (e4m3: as values of T) in LDS
  __device__ __forceinline__ void load(const AttendParams& p, const Item& it, int hk, int key0, int lane, int wave) {
    rows(p, it, hk, key0, lane, wave, [&](int i, auto at, long row) {
      const auto from = (const __attribute__((address_space(1))) raw*)at;
      x[i] = ONCE ? __builtin_nontemporal_load(from) : *from;
      if constexpr (KV == KV_E4M3) scale[i] = (V ? p.vs : p.ks)[row];
    });
  }
  // load() straight into LDS, as store() would leave it
  __device__ __forceinline__ void dma(const AttendParams& p, const Item& it, int hk, int key0, int lane, int wave, T* t) {
    typedef const __attribute__((address_space(1))) void* src_t;
    static_assert(RPL % 16 == 0, "the chunk of a lane is that of every load");
    rows(p, it, hk, key0, lane, wave, [&](int i, auto from, long) {
      __builtin_amdgcn_global_load_lds((src_t)from, (lds_ptr_t)(t + (i * NT + wave * 64) * 8), 16, 0, 0);
    });
  }
  static __device__ __forceinline__ v8 values(unsigned lo, unsigned hi, float s) {
    v2 a, b, c, d;
    if constexpr (std::is_same_v<T, half_t>) {
      a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, s, false);
      b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, s, true);
      c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, s, false);
      d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, s, true);
    } else {
      a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false);
      b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true);
      c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false);
      d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true);
    }
    return v8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
  __device__ __forceinline__ void store(T* t, int tid) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int key = i * RPL + tid / CPR, c = tid % CPR;
      if constexpr (KV != KV_E4M3) {
        *reinterpret_cast<raw*>(t + at(key, c)) = x[i];
      } else {
        const float f = __builtin_bit_cast(float, scale[i] << 23);
#pragma unroll
        for (int j = 0; j < EPL / 8; ++j)
          *reinterpret_cast<v8*>(t + at(key, c * (EPL / 8) + j)) = values(x[i][2 * j], x[i][2 * j + 1], f);
      }
    }
  }
};

// f(integral_constant<int, 0>) ... f(integral_constant<int, N - 1>)
template <typename F, int... I>
__device__ __forceinline__ void each_of(F& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void each(F& f) {
  each_of(f, std::make_integer_sequence<int, N>{});
}

// LDS accesses of one wave complete in order; this keeps the compiler to that order.
__device__ __forceinline__ void wave_order() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_wave_barrier();
  asm volatile("" ::: "memory");
}

// The maximum of lanes l and l ^ 32, in both.  (The swap's results are copied to scalars
// first: a bit cast of a vector's element reads the vector's first one.)
__device__ __forceinline__ float half_max(float v) {
  const unsigned u = __builtin_bit_cast(unsigned, v);
  const auto x = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const unsigned a = x[0], b = x[1];
  return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}

// The maximum of lanes l and l ^ 16, in both.
__device__ __forceinline__ float quarter_max(float v) {
  const unsigned u = __builtin_bit_cast(unsigned, v);
  const auto x = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const unsigned a = x[0], b = x[1];
  return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}

// RANGE: the keys from key0 on that a row sees, one bit each.
template <typename M>
__device__ __forceinline__ M bits_seen(int lim, int lo, int sinks, int key0) {
  constexpr int N = 8 * sizeof(M);
  auto below = [&](int n) -> M { return n - key0 >= N ? ~(M)0 : n <= key0 ? (M)0 : ((M)1 << (n - key0)) - 1; };
  return below(lim) & (~below(lo) | below(sinks));
}

// ---- 32 rows of a wave ------------------------------------------------------------------
template <typename T, int HD, int FORM = WHOLE>
struct Rows {
  typedef typename Elem<T>::v2 v2;
  typedef typename Elem<T>::v4 v4;
  typedef typename Elem<T>::v8 v8;
  static constexpr int BM = 32, KS = HD / 16, CT = HD / 32, VA = CT;
  v8 qf[KS];
  float16_t o[CT];
  float m, l;         // running maximum of the raw scores; this half's part of the sum
  int lim, tok, g;    // keys that the row sees; its query and head within the group (tok < 0: no row)
  int lo, sinks;      // RANGE: from lo on, or below sinks

  template <int KV>
  __device__ __forceinline__ void begin(const AttendParams& p, const Item& it, int hk, int row, int lane) {
    tok = row / p.G;
    g = row - tok * p.G;
    const bool valid = tok < it.s.nq;
    if constexpr (FORM == RANGE) {
      const Sees x = valid ? sees<KV>(p, it, tok) : Sees{0, 0};
      lim = x.lim;
      lo = x.lo;
      sinks = p.sinks;
    } else {
      lim = valid ? keys_of(p, it.s, tok) : 0;
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = v8{};
    if (valid) {
      const T* q = static_cast<const T*>(p.q) + (long)(it.s.q0 + tok) * p.q_st + (long)(hk * p.G + g) * p.q_sh;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const v8*>(q + ks * 16 + (lane >> 5) * 8);
    } else {
      tok = -1;
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) o[ct] = float16_t{};
    m = -INFINITY;
    l = 0.f;
  }

  __device__ __forceinline__ void arrived() {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qf[ks]));
  }

  // S^T of NB blocks of 32 keys in LDS
  template <int NB>
  __device__ __forceinline__ void scores(float16_t (&s)[NB], const T* kt, int lane) const {
#pragma unroll
    for (int kb = 0; kb < NB; ++kb) {
      s[kb] = float16_t{};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const v8 kf = *reinterpret_cast<const v8*>(kt + k_at<HD>(kb * 32 + (lane & 31), ks * 2 + (lane >> 5)));
        s[kb] = Elem<T>::mfma32(kf, qf[ks], s[kb]);
      }
    }
  }
  // nothing of the keys from key0 on that the row does not see
  template <int NB>
  __device__ __forceinline__ void mask(float16_t (&s)[NB], int key0, int lane) const {
    const int left = lim - key0 - 4 * (lane >> 5);
    const int from = lo - key0 - 4 * (lane >> 5), to = sinks - key0 - 4 * (lane >> 5);
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int j = kb * 32 + 8 * (i >> 2) + (i & 3);
        if (j >= left || (FORM == RANGE && j < from && j >= to)) s[kb][i] = -INFINITY;
      }
  }
  template <int NB>
  static __device__ __forceinline__ float top(const float16_t (&s)[NB]) {
    float mx = s[0][0];
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kb][i]);
    return half_max(mx);
  }
  // The maximum that the exponents are taken from may lag behind the true one by 2^8: O and l
  // are rescaled only when some row's has moved further, so hardly ever after the first tiles.
  __device__ __forceinline__ void raise(float mx, float c) {
    if (__any((mx - m) * c > 8.0f || (m == -INFINITY && mx > -INFINITY))) {
      const float mn = fmaxf(m, mx), f = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * c);
      m = mn;
      l *= f;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) o[ct] *= f;
    }
  }
  // the weights, rounded, as the product takes them; the sum is that of the rounded ones, so
  // their rounding cancels where few keys rule.  All are 2^LIFT times what they would be from m.
  __device__ __forceinline__ float origin(float c) const { return m == -INFINITY ? 0.f : __builtin_fmaf(m, c, -Elem<T>::LIFT); }
  template <int NB>
  __device__ __forceinline__ void weigh(v8 (&pf)[2 * NB], const float16_t (&s)[NB], int pair, float c, float mc) {
    const int kb = pair >> 3, i = (pair & 7) * 2;
    const v2 u = pack2<T>(__builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][i], c, -mc)),
                          __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][i + 1], c, -mc)));
    l = Elem<T>::add2(u, l);
    pf[pair >> 2][i & 7] = u[0];
    pf[pair >> 2][(i & 7) + 1] = u[1];
  }
  template <int NB>
  __device__ __forceinline__ void weights(v8 (&pf)[2 * NB], const float16_t (&s)[NB], float c) {
    const float mc = origin(c);
#pragma unroll
    for (int pair = 0; pair < 8 * NB; ++pair) weigh<NB>(pf, s, pair, c, mc);
  }
  // V^T's operands of 16 keys, transposed on their way from LDS.  va: values_at(); OFF: the
  // keys' bytes from there.  In asm with its own wait: the compiler holds the builtin back
  // until every load to LDS that is under way has landed, which is the whole next tile.
  static __device__ __forceinline__ void values_at(unsigned (&va)[CT], const T* vt, int lane) {
    const int key = 4 * (lane >> 5) + ((lane >> 2) & 3), d = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
      va[ct] = (unsigned)(uintptr_t)(lds_ptr_t)(const_cast<T*>(vt) + v_at<HD>(key, (ct * 32 + d) >> 3) + (d & 7));
  }
  template <int OFF>
  static __device__ __forceinline__ void read_values(v8 (&vf)[CT], const unsigned (&va)[CT]) {
    u32x2_t x[2 * CT];
    if constexpr (CT == 4) {
      asm volatile(
          "ds_read_b64_tr_b16 %0, %8 offset:%12\n\t"
          "ds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
          "ds_read_b64_tr_b16 %2, %9 offset:%12\n\t"
          "ds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
          "ds_read_b64_tr_b16 %4, %10 offset:%12\n\t"
          "ds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
          "ds_read_b64_tr_b16 %6, %11 offset:%12\n\t"
          "ds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
          "s_waitcnt lgkmcnt(0)"
          : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(x[4]), "=&v"(x[5]), "=&v"(x[6]), "=&v"(x[7])
          : "v"(va[0]), "v"(va[1]), "v"(va[CT - 2]), "v"(va[CT - 1]), "n"(OFF), "n"(OFF + 8 * HD * 2));
    } else {
      asm volatile(
          "ds_read_b64_tr_b16 %0, %4 offset:%6\n\t"
          "ds_read_b64_tr_b16 %1, %4 offset:%7\n\t"
          "ds_read_b64_tr_b16 %2, %5 offset:%6\n\t"
          "ds_read_b64_tr_b16 %3, %5 offset:%7\n\t"
          "s_waitcnt lgkmcnt(0)"
          : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3])
          : "v"(va[0]), "v"(va[1]), "n"(OFF), "n"(OFF + 8 * HD * 2));
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
      vf[ct] = __builtin_bit_cast(v8, u32x4_t{x[2 * ct][0], x[2 * ct][1], x[2 * ct + 1][0], x[2 * ct + 1][1]});
  }
  // The same of one block of 32 features by the builtin, for tiles that come through registers.
  template <int OFF>
  static __device__ __forceinline__ v8 read_value(unsigned va) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4* at_t;
    const v4 a = __builtin_bit_cast(v4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_t)(uintptr_t)(va + OFF)));
    const v4 b = __builtin_bit_cast(v4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_t)(uintptr_t)(va + OFF + 8 * HD * 2)));
    return v8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  }
  // O^T += V^T P^T
  template <int NB, int OFF, int KK = 0>
  __device__ __forceinline__ void values(const unsigned (&va)[CT], const v8 (&pf)[2 * NB]) {
    if constexpr (KK < 2 * NB) {
      v8 vf[CT];
      read_values<OFF + KK * 16 * HD * 2>(vf, va);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) o[ct] = Elem<T>::mfma32(vf[ct], pf[KK], o[ct]);
      values<NB, OFF, KK + 1>(va, pf);
    }
  }
  // One step of the pipeline: n = K Q^T of the next tile beside the weights of s, then
  // O^T += V^T P^T beside the next tile's maximum, which is returned.  The order is pinned: a
  // wave issues in order, and MFMAs on end leave the vector unit idle.
  template <int VOFF, bool ASM>
  __device__ __forceinline__ float step(float16_t (&n)[2], const float16_t (&s)[2], const T* kt, const unsigned (&va)[CT],
                                        float c, int lane) {
    constexpr int NK = 2 * KS, AHEAD = ASM ? 4 : 2, PPM = 16 / NK;
    const float mc = origin(c);
    auto key = [&](int i) {
      return *reinterpret_cast<const v8*>(kt + k_at<HD>((i / KS) * 32 + (lane & 31), (i % KS) * 2 + (lane >> 5)));
    };
    constexpr int VR = ASM ? 2 * CT : 3;   // V fragments held
    v8 kf[AHEAD], pf[4], vf[VR];
    auto value = [&](auto I) {   // fragment I = kk * CT + ct
      constexpr int i = decltype(I)::value;
      if constexpr (!ASM && i < 4 * CT) vf[i % VR] = read_value<VOFF + (i / CT) * 16 * HD * 2>(va[i % CT]);
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) kf[i] = key(i);
    n[0] = float16_t{};
    n[1] = float16_t{};
    __builtin_amdgcn_sched_barrier(0);
    auto qk = [&](auto I) {
      constexpr int i = decltype(I)::value;
      n[i / KS] = Elem<T>::mfma32(kf[i % AHEAD], qf[i % KS], n[i / KS]);
      if constexpr (i + AHEAD < NK) kf[i % AHEAD] = key(i + AHEAD);
      if constexpr (!ASM && i >= NK - VR) value(std::integral_constant<int, i - (NK - VR)>{});
#pragma unroll
      for (int j = 0; j < PPM; ++j) weigh<2>(pf, s, i * PPM + j, c, mc);
      if constexpr (ASM && i == NK - 2) read_values<VOFF>(*reinterpret_cast<v8 (*)[CT]>(&vf[0]), va);
      __builtin_amdgcn_sched_barrier(0);
    };
    each<NK>(qk);
    float mx = -INFINITY;
    auto pv = [&](auto I) {
      constexpr int i = decltype(I)::value, kk = i / CT, ct = i % CT;
      o[ct] = Elem<T>::mfma32(vf[i % VR], pf[kk], o[ct]);
      value(std::integral_constant<int, i + VR>{});
      // the next tile's scores: 8 of them here, those of the second block last
#pragma unroll
      for (int j = 0; j < 8 / CT; ++j) mx = fmaxf(mx, n[kk >> 1][(kk & 1) * 8 + ct * (8 / CT) + j]);
      if constexpr (ASM && ct == CT / 2 - 1 && kk < 3)
        read_values<VOFF + (kk < 3 ? kk + 1 : 3) * 16 * HD * 2>(*reinterpret_cast<v8 (*)[CT]>(&vf[((kk + 1) & 1) * CT]), va);
      __builtin_amdgcn_sched_barrier(0);
    };
    each<4 * CT>(pv);
    return half_max(mx);
  }
  // bad[k][d]: the first key whose V is +inf, -inf or NaN (k = 0, 1, 2) in feature d
  __device__ __forceinline__ void add_odd(const int (*bad)[HD], int, int lane) {
    typedef const __attribute__((address_space(3))) int* lds_int_t;
    unsigned at = (unsigned)(uintptr_t)(lds_int_t)&bad[0][4 * (lane >> 5)];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        asm volatile("" : "+v"(at)::"memory");   // one element at a time: a rare path, and no registers for it
        const lds_int_t k = (lds_int_t)(uintptr_t)at + ct * 32 + 8 * (i >> 2) + (i & 3);
        float add = k[0] < lim ? INFINITY : 0.f;
        add += k[HD] < lim ? -INFINITY : 0.f;
        add += k[2 * HD] < lim ? NAN : 0.f;
        asm volatile("" : "+v"(add)::"memory");
        o[ct][i] += add;
      }
  }
  // the same of the keys of the tile at key0, one bit each
  template <typename M>
  __device__ __forceinline__ void add_odd(const M (*bad)[HD], int key0, int lane) {
    const M seen = bits_seen<M>(lim, lo, sinks, key0);
    typedef const __attribute__((address_space(3))) M* lds_m_t;
    unsigned at = (unsigned)(uintptr_t)(lds_m_t)&bad[0][4 * (lane >> 5)];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        asm volatile("" : "+v"(at)::"memory");
        const lds_m_t k = (lds_m_t)(uintptr_t)at + ct * 32 + 8 * (i >> 2) + (i & 3);
        float add = k[0] & seen ? INFINITY : 0.f;
        add += k[HD] & seen ? -INFINITY : 0.f;
        add += k[2 * HD] & seen ? NAN : 0.f;
        asm volatile("" : "+v"(add)::"memory");
        o[ct][i] += add;
      }
  }
  // For a wave by itself: S^T of the 32 keys from key0 on; part: some row does not see all of them
  typedef float16_t scores_t[1];
  __device__ __forceinline__ void look(scores_t& s, const T* kt, bool part, int key0, int lane) const {
    scores<1>(s, kt, lane);
    if (part) mask<1>(s, key0, lane);
  }
  // and O^T += V^T P^T of them
  __device__ __forceinline__ void take(const scores_t& s, const unsigned (&va)[VA], float c, int lane) {
    v8 pf[2];
    raise(top<1>(s), c);
    weights<1>(pf, s, c);
    values<1, 0>(va, pf);
  }
  __device__ __forceinline__ float sum() const { return l + __shfl_xor(l, 32); }
  // f(chunk, values) for every four features of the row in this lane
  template <typename F>
  __device__ __forceinline__ void chunks(int lane, F f) const {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        f(ct * 8 + (i >> 1) + (lane >> 5), float4_t{o[ct][i], o[ct][i + 1], o[ct][i + 2], o[ct][i + 3]});
  }
  // the output rows, O / l
  __device__ __forceinline__ void finish(const AttendParams& p, const Item& it, int hk, int lane) const {
    const float t = sum(), r = t == 0.f ? 0.f : 1.0f / t;
    if (tok < 0) return;
    T* out = static_cast<T*>(p.out) + (long)(it.s.q0 + tok) * p.o_st + (long)(hk * p.G + g) * p.o_sh + 4 * (lane >> 5);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const v2 a = pack2<T>(o[ct][i] * r, o[ct][i + 1] * r), b = pack2<T>(o[ct][i + 2] * r, o[ct][i + 3] * r);
        *reinterpret_cast<v4*>(out + ct * 32 + 2 * i) = v4{a[0], a[1], b[0], b[1]};
      }
  }
};

// ---- 16 rows of a wave ------------------------------------------------------------------
// The same with 16x16x32 products, where 32 rows would stand half empty: half the registers.  Lane
// l holds row l % 16, of a block of 16 keys those 4 (l / 16) + i, i < 4; two blocks make the second
// product's operand.  Steps of 32 keys.
template <typename T, int HD, int FORM = WHOLE>
struct Rows16 {
  typedef typename Elem<T>::v2 v2;
  typedef typename Elem<T>::v4 v4;
  typedef typename Elem<T>::v8 v8;
  static constexpr int BM = 16, KS = HD / 32, CT = HD / 16, VA = HD / 32;
  v8 qf[KS];
  float4_t o[CT];
  float m, l;
  int lim, lo, sinks;

  template <int KV>
  __device__ __forceinline__ void begin(const AttendParams& p, const Item& it, int hk, int row, int lane) {
    const int tok = row / p.G, g = row - tok * p.G;
    const bool valid = tok < it.s.nq;
    if constexpr (FORM == RANGE) {
      const Sees x = valid ? sees<KV>(p, it, tok) : Sees{0, 0};
      lim = x.lim;
      lo = x.lo;
      sinks = p.sinks;
    } else {
      lim = valid ? keys_of(p, it.s, tok) : 0;
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = v8{};
    if (valid) {
      const T* q = static_cast<const T*>(p.q) + (long)(it.s.q0 + tok) * p.q_st + (long)(hk * p.G + g) * p.q_sh;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const v8*>(q + ks * 32 + (lane >> 4) * 8);
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) o[ct] = float4_t{};
    m = -INFINITY;
    l = 0.f;
  }
  __device__ __forceinline__ void arrived() {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qf[ks]));
  }
  static __device__ __forceinline__ void values_at(unsigned (&va)[VA], const T* vt, int lane) {
    const int key = 4 * (lane >> 4) + ((lane >> 2) & 3), d = 4 * (lane & 3);
#pragma unroll
    for (int i = 0; i < VA; ++i)
      va[i] = (unsigned)(uintptr_t)(lds_ptr_t)(const_cast<T*>(vt) + v_at<HD>(key, (i * 32 + d) >> 3) + (d & 7));
  }
  typedef float4_t scores_t[2];
  // S^T of the 32 keys from key0 on; part: some row does not see all of them
  __device__ __forceinline__ void look(scores_t& s, const T* kt, bool part, int key0, int lane) const {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      s[kb] = float4_t{};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        s[kb] = Elem<T>::mfma16(*reinterpret_cast<const v8*>(kt + k_at<HD>(kb * 16 + (lane & 15), ks * 4 + (lane >> 4))), qf[ks], s[kb]);
    }
    if (part) {
      const int left = lim - key0 - 4 * (lane >> 4);
      const int from = lo - key0 - 4 * (lane >> 4), to = sinks - key0 - 4 * (lane >> 4);
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (kb * 16 + i >= left || (FORM == RANGE && kb * 16 + i < from && kb * 16 + i >= to)) s[kb][i] = -INFINITY;
    }
  }
  // O^T += V^T P^T of them
  __device__ __forceinline__ void take(const scores_t& s, const unsigned (&va)[VA], float c, int lane) {
    float mx = s[0][0];
#pragma unroll
    for (int i = 1; i < 8; ++i) mx = fmaxf(mx, s[i >> 2][i & 3]);
    mx = half_max(quarter_max(mx));
    if (__any((mx - m) * c > 8.0f || (m == -INFINITY && mx > -INFINITY))) {   // as Rows::raise
      const float mn = fmaxf(m, mx), f = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * c);
      m = mn;
      l *= f;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) o[ct] *= f;
    }
    const float mc = m == -INFINITY ? 0.f : __builtin_fmaf(m, c, -Elem<T>::LIFT);
    v8 pf;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const v2 u = pack2<T>(__builtin_amdgcn_exp2f(__builtin_fmaf(s[i >> 2][i & 3], c, -mc)),
                            __builtin_amdgcn_exp2f(__builtin_fmaf(s[i >> 2][(i & 3) + 1], c, -mc)));
      l = Elem<T>::add2(u, l);
      pf[i] = u[0];
      pf[i + 1] = u[1];
    }
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4* at_t;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const unsigned at = va[ct >> 1] ^ ((ct & 1) * 32);   // 16-byte chunk c and c ^ 2
      const v4 a = __builtin_bit_cast(v4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_t)(uintptr_t)at));
      const v4 b = __builtin_bit_cast(v4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_t)(uintptr_t)(at + 16 * HD * 2)));
      o[ct] = Elem<T>::mfma16(v8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}, pf, o[ct]);
    }
  }
  // as Rows::add_odd
  __device__ __forceinline__ void add_odd(const int (*bad)[HD], int, int lane) {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int* k = &bad[0][ct * 16 + 4 * (lane >> 4) + i];
        float add = k[0] < lim ? INFINITY : 0.f;
        add += k[HD] < lim ? -INFINITY : 0.f;
        add += k[2 * HD] < lim ? NAN : 0.f;
        o[ct][i] += add;
      }
  }
  template <typename M>
  __device__ __forceinline__ void add_odd(const M (*bad)[HD], int key0, int lane) {
    const M seen = bits_seen<M>(lim, lo, sinks, key0);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const M* k = &bad[0][ct * 16 + 4 * (lane >> 4) + i];
        float add = k[0] & seen ? INFINITY : 0.f;
        add += k[HD] & seen ? -INFINITY : 0.f;
        add += k[2 * HD] & seen ? NAN : 0.f;
        o[ct][i] += add;
      }
  }
  __device__ __forceinline__ float sum() const {
    const float t = l + __shfl_xor(l, 16);
    return t + __shfl_xor(t, 32);
  }
  // f(chunk, values) for every four features of the row in this lane
  template <typename F>
  __device__ __forceinline__ void chunks(int lane, F f) const {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) f(ct * 4 + (lane >> 4), o[ct]);
  }
};

// Whether this thread's part of a tile in LDS holds an infinity or a NaN.
template <typename T, int TILE, int NT>
__device__ __forceinline__ bool any_odd(const T* vt, int tid) {
  unsigned acc = 0;
#pragma unroll
  for (int i = 0; i < TILE / 8 / NT; ++i) {
    const u32x4_t u = reinterpret_cast<const u32x4_t*>(vt)[i * NT + tid];
#pragma unroll
    for (int j = 0; j < 4; ++j) acc |= (u[j] & Elem<T>::EXP) + Elem<T>::LOW;
  }
  return acc & 0x80008000u;
}

// Takes infinities and NaN out of a V tile in LDS: zero in their places, the first key of
// each kind and feature in bad.  For the rows that do not see them (0 * inf is not 0).
template <typename T, int HD, int KEYS, int NT>
__device__ __forceinline__ void take_out_odd(T* vt, int (*bad)[HD], int key0, int tid) {
  for (int i = tid; i < KEYS * HD; i += NT) {
    const int key = i / HD, d = i % HD, at = v_at<HD>(key, d >> 3) + (d & 7);
    const float x = (float)vt[at];
    if (!(fabsf(x) < INFINITY)) {
      atomicMin(&bad[x > 0 ? 0 : x < 0 ? 1 : 2][d], key0 + key);
      vt[at] = (T)0.f;
    }
  }
}

// The same where a row may see any of the keys: all of each kind and feature, one bit a key.
template <typename T, int HD, int KEYS, int NT, typename M>
__device__ __forceinline__ void take_out_odd(T* vt, M (*bad)[HD], int tid) {
  for (int i = tid; i < KEYS * HD; i += NT) {
    const int key = i / HD, d = i % HD, at = v_at<HD>(key, d >> 3) + (d & 7);
    const float x = (float)vt[at];
    if (!(fabsf(x) < INFINITY)) {
      atomicOr(&bad[x > 0 ? 0 : x < 0 ? 1 : 2][d], (M)1 << key);
      vt[at] = (T)0.f;
    }
  }
}

// Where the partial sums of an item's rows are: O f32 [items][rows][HD], then (maximum in the
// log2 domain, sum) [items][rows][2].
template <int HD>
__device__ __forceinline__ float* part_o(const AttendParams& p, long row) { return p.ws + row * HD; }
template <int HD>
__device__ __forceinline__ float2_t* part_ml(const AttendParams& p, long row) {
  return reinterpret_cast<float2_t*>(p.ws + p.part_rows * HD) + row;
}

// Where the row q of an item's partial sums is, or -1 (offsets that do not ascend may name more rows than
// there are).  Shared pages: the fronts' items, of BMF rows each, then the sequences' own.
template <int BM, int BMF, int FORM>
__device__ __forceinline__ long part_row(const AttendParams& p, const Item& it, int hk, int q) {
  const int item = it.base + it.chunk;
  if constexpr (FORM == RANGE)
    if (p.N) {
      if (it.front) return item < 0 || item >= p.front_items ? -1 : ((long)item * p.Hkv + hk) * BMF + q;
      const int own = item - it.fronts;
      if (it.fronts < 0 || it.fronts > p.front_items || own < 0 || own >= p.own_items) return -1;
      return (long)it.fronts * p.Hkv * BMF + ((long)own * p.Hkv + hk) * BM + q;
    }
  return ((long)item * p.Hkv + hk) * BM + q;
}
// Shared pages: what the joining launch has to know of a sequence's own tile, so that it need not look for it.
struct Parts {
  int q0, row0, rows;          // the sequence's first query; the tile's first row, its rows
  int own, nch;                // its first item among the own ones, items (0: none)
  int front, fnch, frow0;      // the group's first item, chunks (0: no group), the group's row that is row0
  int frows, pad[3];           // the group's rows
};
// The workspace behind the sums: how many own tiles there are and how many items of fronts, then Parts for each tile.
template <int HD>
__device__ __forceinline__ int* parts_head(const AttendParams& p) { return reinterpret_cast<int*>(p.ws + p.part_rows * (HD + 2)); }
template <int HD>
__device__ __forceinline__ Parts* parts_at(const AttendParams& p) { return reinterpret_cast<Parts*>(parts_head<HD>(p) + 4); }

// By one lane: the Parts of an own tile's first item.
template <int HD, int BM>
__device__ __forceinline__ void leave_parts(const AttendParams& p, const Item& it, int hk, int tile) {
  if (it.front || it.chunk || hk || it.rank < 0 || it.rank >= p.own_items) return;
  Parts x{};
  x.q0 = it.s.q0;
  x.row0 = tile * BM;
  x.rows = (int)min((long)BM, (long)it.s.nq * p.G - (long)tile * BM);
  x.own = it.base - it.fronts;
  x.nch = it.nch;
  x.front = it.f.base;
  x.fnch = it.f.nch;
  x.frows = (int)min(it.f.rows, 0x7FFFFFFFl);
  x.frow0 = (int)max(((long)it.s.q0 - it.f.q0) * p.G + (long)tile * BM, -1l);
  parts_at<HD>(p)[it.rank] = x;
}
// By one lane of the first workgroup: how many own tiles and items of fronts there are.
template <int HD>
__device__ __forceinline__ void leave_head(const AttendParams& p, const Item& it, int tiles) {
  parts_head<HD>(p)[0] = min(tiles, p.own_items);
  parts_head<HD>(p)[1] = it.fronts;
}

// ---- many rows: NW waves of 32 rows over the same keys -----------------------------------
// Tiles of 64 keys.  A wave computes the scores of one tile while it turns those of the tile
// before into weights, so that the matrix cores and the vector unit work at the same time:
//   step j:  S(j+1) = K(j+1) Q^T  beside  P(j) = 2^(S(j) - m);
//            O += V(j)^T P(j)     beside  max S(j+1).
// K is therefore one tile ahead of V.  Both have two buffers in LDS; step j sends for V(j+1)
// and K(j+2) (f16, bf16: straight to LDS; e4m3: through registers, where it is turned into
// values).
// 256 rows (two waves a SIMD, one workgroup a CU): prompts of 9001, 5120 and 2263 tokens, 16
// heads on 4 of 128, bf16, 447 us a call (443 the kernel) = 1.03 PFLOP/s, where a product of
// 8192^3 reaches 1.55; 128 rows 460.  At 471 us it took 392 without its loads, 369 without
// barrier and LDS reads as well, 316 without the softmax too = the matrix cores at the clock
// their power leaves: of the 155 us over those, half are the loads and a third the softmax.
// Slower were the compiler's own order (sched groups 517-535 against 508 then), rings of four
// tiles (467 against 455) and f16 tiles by way of registers (466).
// 128 rows with the keys split: 512 tokens on 12800 keys, 16 heads of 128, f16, 69 us and 8 to
// join them, 680 TFLOP/s by the call; from an e4m3 cache, eight sequences of 1 to 511 tokens, 65
// and 10 us, 545 by the call, though with 128 features that kernel spills 43 registers (tiles
// of 256 rows: 19; without codes to turn into values: 1).  Short prompts (40 of 1 to 239 tokens,
// 8 heads of 64) 12.4 us.
// RANGE, 128 rows: prompts of 9001, 5120 and 2263 through 2048 keys and 4 first ones, 16 heads on 4 of 128, bf16, 268.5 us:
// 224 GFLOP seen, 236 issued, 0.88 PFLOP/s of these (through all keys 471 us, 465 issued, 0.99; WHOLE takes 460 a call with 128
// rows).  256 rows: 288.  Six chunks of 1 to 512 tokens on 12800 shared keys, f16, 227 us and 11.5 to join them, 178 GFLOP, 0.78
// PFLOP/s.
// Masked tiles in the pipeline with the others: prompts 272 -> 270, but e4m3 spills in the loop (46 -> 70 below).
template <typename T, int HD, int FORM>
struct TileLds {
  // (bad: WHOLE, the first key of a kind and feature; RANGE, a bit for each key of the tile)
  typedef std::conditional_t<FORM == RANGE, unsigned long long, int> bad_t;
  static constexpr int TILE = AT_KEYS * HD, BAD = 3 * HD * sizeof(bad_t), BYTES = 4 * TILE * 2 + BAD + 16;
};
// BMO: rows of the tiles of sequences' own keys, where this is a front's
template <typename T, int HD, int KV, int NW, int FORM, int BMO = 32 * NW>
__device__ __forceinline__ void tile_item(const AttendParams& p, Item& it, const int hk, char* const lds) {
  constexpr int BM = 32 * NW, TILE = AT_KEYS * HD, NT = 64 * NW;
  constexpr bool SPLIT = NW == 4;   // a tile's keys may be split over workgroups
  constexpr bool DMA = KV != KV_E4M3;
  typedef typename TileLds<T, HD, FORM>::bad_t bad_t;
  constexpr int BAD = TileLds<T, HD, FORM>::BAD;
  auto kt = [&](int buf) { return reinterpret_cast<T*>(lds) + buf * TILE; };
  auto vt = [&](int buf) { return reinterpret_cast<T*>(lds) + (2 + buf) * TILE; };
  bad_t (*const bad)[HD] = reinterpret_cast<bad_t (*)[HD]>(lds + 4 * TILE * 2);
  int& odd = *reinterpret_cast<int*>(lds + 4 * TILE * 2 + BAD);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tile = tiles_of<KV, BM>(it.s, p.G) - 1 - it.tile;   // the longest first
  const int tok0 = tile * BM / p.G, tok1 = min(it.s.nq - 1, (tile * BM + BM - 1) / p.G);
  // WHOLE: the keys of the tile's first and last rows, and of this chunk
  int klo = 0, kbeg = 0, kend = 0;
  // RANGE: its blocks of keys, and those of this chunk
  Blocks bl;
  int vbeg = 0, vend = 0;
  if constexpr (FORM == RANGE) {
    if (KV != KV_ROWS && p.N && tid == 0) leave_parts<HD, BMO>(p, it, hk, tile);
    bl = blocks<KV>(p, it, tok0, tok1);
    vbeg = SPLIT && it.nch > 1 ? it.chunk * it.c : 0;
    vend = SPLIT && it.nch > 1 ? min(bl.nb, vbeg + it.c) : bl.nb;
    kbeg = bl.key(vbeg);
    kend = vbeg < vend ? kbeg + 1 : kbeg;   // (whether there is any)
  } else {
    klo = keys_of(p, it.s, tok0);
    const int khi = keys_of(p, it.s, tok1);
    kbeg = SPLIT && it.nch > 1 ? it.chunk * it.c * AT_KEYS : 0;
    kend = SPLIT && it.nch > 1 ? min(khi, kbeg + it.c * AT_KEYS) : khi;
  }

  Stage<T, HD, KV, AT_KEYS, NT, false, false, FORM == RANGE> ks;
  Stage<T, HD, KV, AT_KEYS, NT, true, false, FORM == RANGE> vs;
  auto send = [&](auto& st, int key0, T* t) {
    if constexpr (DMA) st.dma(p, it, hk, key0, lane, wave, t);
    else st.load(p, it, hk, key0, lane, wave);
  };
  // what was sent for has landed, here and (barrier) in the other waves
  auto landed = [&] {
    wait_vm_lgkm0<0>();
    lds_barrier();
  };
  Rows<T, HD, FORM> r;
  unsigned va[Rows<T, HD>::CT];
  r.values_at(va, vt(0), lane);
  const float c = p.scale_log2e;
  if (tid == 0) odd = 0;
  float16_t sa[2], sb[2];
  if (kbeg < kend) {
    ks.begin(p, it, hk, kbeg, AT_KEYS, lane, wave, DMA);
    vs.begin(p, it, hk, kbeg, AT_KEYS, lane, wave, DMA);
    r.template begin<KV>(p, it, hk, tile * BM + wave * 32 + (lane & 31), lane);
    send(ks, kbeg, kt(0));
    send(vs, kbeg, vt(0));
    if constexpr (!DMA) ks.store(kt(0), tid);
    send(ks, FORM == RANGE ? bl.key(vbeg + 1) : kbeg + AT_KEYS, kt(1));
    if constexpr (!DMA) {
      vs.store(vt(0), tid);
      ks.store(kt(1), tid);
    }
    landed();
    r.arrived();   // so that no wait in the loop counts Q's loads
    r.template scores<2>(sa, kt(0), lane);
  } else {
    r.template begin<KV>(p, it, hk, tile * BM + wave * 32 + (lane & 31), lane);
  }
  // step j begins: K(j+1) and V(j) are there, K(j)'s and V(j-1)'s buffers free
  auto next = [&](int key1, int key2, int cur) {
    landed();
    send(vs, key1, vt(cur ^ 1));
    send(ks, key2, kt(cur));
  };
  auto keep = [&](int cur) {
    if constexpr (!DMA) {
      vs.store(vt(cur ^ 1), tid);
      ks.store(kt(cur), tid);
    }
  };
  int key0 = kbeg, cur = 0;
  // The infinities and NaN of this tile's V taken out, if there are any.
  auto take_out = [&](int tid_) {
    if (any_odd<T, TILE, NT>(vt(cur), tid_)) odd = 1;
    __syncthreads();
    const bool fix = odd;
    if (fix) {
      for (int i = tid_; i < 3 * HD; i += NT) (&bad[0][0])[i] = FORM == RANGE ? 0 : 0x7FFFFFFF;
      __syncthreads();
      if constexpr (FORM == RANGE) take_out_odd<T, HD, AT_KEYS, NT>(vt(cur), bad, tid_);
      else take_out_odd<T, HD, AT_KEYS, NT>(vt(cur), bad, key0, tid_);
      __syncthreads();
    }
    return fix;
  };
  // A tile whose scores are in sa by itself; part: some row does not see all of it, and an infinity
  // or NaN of V must not reach that row.
  auto alone = [&](bool part, bool more) {
    int lane_ = lane, tid_ = tid;
    if constexpr (FORM == RANGE)   // or the addresses of this rarer path stay in registers through the other one
      asm volatile("" : "+v"(lane_), "+v"(tid_));
    bool fix = false;
    if (part) {
      r.template mask<2>(sa, key0, lane_);
      fix = take_out(tid_);
    }
    r.raise(r.template top<2>(sa), c);
    typename Elem<T>::v8 pf[4];
    r.template weights<2>(pf, sa, c);
    unsigned vc[Rows<T, HD>::CT];
#pragma unroll
    for (int ct = 0; ct < Rows<T, HD>::CT; ++ct) vc[ct] = va[ct] + cur * TILE * 2;
    r.template values<2, 0>(vc, pf);
    if (fix) {
      r.add_odd(bad, key0, lane_);
      __syncthreads();
      if (tid_ == 0) odd = 0;
    }
    if (more) {
      r.template scores<2>(sa, kt(cur ^ 1), lane_);
      keep(cur);
    }
  };
  if constexpr (FORM == RANGE) {
    auto whole = [&](int v) { return v < bl.fs || (v >= bl.fa && v < bl.fb); };
    if ((long)tile * BM + wave * 32 >= (long)it.s.nq * p.G) {
      // a wave without a row only brings tiles, and leaves the CU's units to the others
      for (int v = vbeg; v < vend; ++v, cur ^= 1) {
        next(bl.key(v + 1), bl.key(v + 2), cur);
        if (!whole(v) && take_out(tid)) __syncthreads();   // (as below, behind add_odd)
        if (v + 1 < vend) keep(cur);
      }
      wait_vm_lgkm0<0>();
      return;
    }
    for (int v = vbeg; v < vend; ++v, cur ^= 1) {
      // runs of tiles of which every row sees all
      const int run = min(v < bl.fs ? bl.fs : v >= bl.fa ? bl.fb : v, vend);
      if (v + 1 < run) {
        float mx = r.template top<2>(sa);
        auto step = [&](float16_t (&s)[2], float16_t (&n)[2], auto CUR) {
          constexpr int cu = decltype(CUR)::value;
          next(bl.key(v + 1), bl.key(v + 2), cu);
          r.raise(mx, c);
          mx = r.template step<cu * TILE * 2, DMA>(n, s, kt(cu ^ 1), va, c, lane);
          keep(cu);
          ++v;
        };
        if (cur) {
          step(sa, sb, std::integral_constant<int, 1>{});
          sa[0] = sb[0];
          sa[1] = sb[1];
          cur = 0;
        }
        while (v + 2 < run) {
          step(sa, sb, std::integral_constant<int, 0>{});
          step(sb, sa, std::integral_constant<int, 1>{});
        }
        if (v + 1 < run) {
          step(sa, sb, std::integral_constant<int, 0>{});
          cur = 1;
          sa[0] = sb[0];
          sa[1] = sb[1];
        }
      }
      key0 = bl.key(v);
      next(bl.key(v + 1), bl.key(v + 2), cur);
      alone(!whole(v), v + 1 < vend);
    }
  } else {
    // while every row sees all of this tile and of the next one
    const int kfull = min(klo, kend) - 2 * AT_KEYS;
    if (key0 <= kfull) {
      float mx = r.template top<2>(sa);
      auto step = [&](float16_t (&s)[2], float16_t (&n)[2], auto CUR) {
        constexpr int cu = decltype(CUR)::value;
        next(key0 + AT_KEYS, key0 + 2 * AT_KEYS, cu);
        r.raise(mx, c);
        mx = r.template step<cu * TILE * 2, DMA>(n, s, kt(cu ^ 1), va, c, lane);
        keep(cu);
        key0 += AT_KEYS;
      };
      while (key0 + AT_KEYS <= kfull) {
        step(sa, sb, std::integral_constant<int, 0>{});
        step(sb, sa, std::integral_constant<int, 1>{});
      }
      if (key0 <= kfull) {
        step(sa, sb, std::integral_constant<int, 0>{});
        cur = 1;
        sa[0] = sb[0];
        sa[1] = sb[1];
      }
    }
    // the rest one by one
    for (; key0 < kend; key0 += AT_KEYS, cur ^= 1) {
      next(key0 + AT_KEYS, key0 + 2 * AT_KEYS, cur);
      alone(key0 + AT_KEYS > klo, key0 + AT_KEYS < kend);
    }
  }
  wait_vm_lgkm0<0>();   // the loads past the last tile land before this workgroup's LDS is another's

  // (the parts of shared pages are always joined)
  if ((!SPLIT || it.nch == 1) && (FORM != RANGE || KV == KV_ROWS || !p.N)) {
    r.finish(p, it, hk, lane);
    return;
  }
  const float t = r.sum();
  if (r.tok < 0) return;
  const long row = part_row<BMO, BM, FORM>(p, it, hk, wave * 32 + (lane & 31));
  if (FORM == RANGE && row < 0) return;
  if (lane < 32) *part_ml<HD>(p, row) = float2_t{r.m * p.scale_log2e, t};
  if (kbeg >= kend) return;
  float* o = part_o<HD>(p, row) + 4 * (lane >> 5);
#pragma unroll
  for (int ct = 0; ct < HD / 32; ++ct)
#pragma unroll
    for (int i = 0; i < 16; i += 4)
      *reinterpret_cast<float4_t*>(o + ct * 32 + 2 * i) = float4_t{r.o[ct][i], r.o[ct][i + 1], r.o[ct][i + 2], r.o[ct][i + 3]};
}

template <typename T, int HD, int KV, int NW, int FORM>
__global__ __launch_bounds__(64 * NW, 2) void attend_tile_kernel(const AttendParams p) {
  // one array: with several, the compiler holds every read of one back until all loads to the
  // others have landed
  __shared__ __attribute__((aligned(1024))) char lds[TileLds<T, HD, FORM>::BYTES];
  const int hk = blockIdx.x % p.Hkv, index = blockIdx.x / p.Hkv;
  Item it;
  if (FORM == RANGE && KV != KV_ROWS && p.N) {
    int tiles;
    const bool some = find_shared<KV, 32 * NW, 32 * NW>(p, index, it, tiles);
    if (blockIdx.x == 0 && threadIdx.x == 0) leave_head<HD>(p, it, tiles);
    if (!some) return;
  } else if (!find_item<KV, 32 * NW, false, FORM>(p, index, it)) {
    return;
  }
  tile_item<T, HD, KV, NW, FORM>(p, it, hk, lds);
}

// ---- few rows: 16 or 32 of them, the keys over the waves -----------------------------------
// Every wave streams its own blocks of 32 keys (w, w + 4, ...) through LDS of its own; nothing
// waits for another wave until the end, where the waves' sums are joined.  Bound by memory: the
// rows come past the caches, K and V of the next step under way during this one's products.
// What helps is workgroups on a CU: 16 rows leave registers for more of them.  32 tokens on 1025
// to 32701 keys, 16 heads on 4 of 128, e4m3: 120 us with 32 rows, 115 with 16, 110 with three
// workgroups a CU, 5.9 TB/s, where plain reads of this kind reach 7.1 and the card's copy 4.9;
// 16 such on 8 heads of 64 84, 64, and 62 with K's next rows sent for before V's are stored.  Two
// steps ahead are slower: 116 for 115, and 77 for 64.
// One token on 6144 keys, 8 heads of 64, f16: 6.1 to 6.4 us.
constexpr int FEW_WAVES = 4;

// workgroups a CU
constexpr int few_at_once(int bm, int hd, bool e4m3) { return hd == 64 ? (bm == 16 ? 4 : 3) : bm == 16 && e4m3 ? 3 : 2; }

// RANGE: one token of 32 streams through 4096 keys and 16 first ones, 16 heads on 4 of 128, e4m3, 133 MB: 29.9 us = 4.4
// TB/s, of which about 8 are a workgroup's beginning (lengths, then the table, then keys, each a wait for memory), and 4.7 to
// join them; one token through 512 keys, 8 heads of 64, whole: 10.0 us.
// MIXED (shared pages, single tokens): the groups' fronts by tiles of 128 rows, the sequences' own keys by few rows.
// 64 streams on 24576 and 12800 shared keys and 1 to 1500 of their own, 16 heads on 4 of 128, e4m3, 87 MB: 39.2 us and 5.3 to
// join them (all by tiles 62 and 5.5).  Bound by the waits for memory: a step of e4m3 tiles takes 1.6 us where the next
// tile's keys come from HBM, and two workgroups a CU are all that registers allow.  Own keys two steps ahead: 46.6 us a
// call for 45.7; in chunks twice as long 46.0, four times 63.
template <typename T, int HD, int KV, typename R, int FORM, bool MIXED = false>
__global__ __launch_bounds__(64 * FEW_WAVES, MIXED ? 2 : few_at_once(R::BM, HD, KV == KV_E4M3)) void attend_few_kernel(const AttendParams p) {
  constexpr int BM = R::BM, KEYS = 32, TILE = KEYS * HD, NW = FEW_WAVES, BMF = MIXED ? 128 : BM;
  // 1: V takes K's place in LDS, so that three workgroups of 128 features fit a CU
  constexpr int PARTS = HD == 128 && few_at_once(BM, HD, KV == KV_E4M3) == 3 ? 1 : 2;
  constexpr int FRONT = MIXED ? (TileLds<T, HD, RANGE>::BYTES / 2 / NW + 511) / 512 * 512 : 0;   // of each wave's part; rows stay aligned
  static_assert(!MIXED || FRONT * NW * 2 >= TileLds<T, HD, RANGE>::BYTES, "a tile's LDS");
  __shared__ __attribute__((aligned(1024))) T lds[NW][PARTS * TILE > FRONT ? PARTS * TILE : FRONT];   // at the end: O f32 [NW][BM][HD]
  __shared__ float2_t ml[NW][BM];
  typedef std::conditional_t<FORM == RANGE, unsigned, int> bad_t;   // as TileLds
  __shared__ bad_t bad[NW][3][HD];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hk = blockIdx.x % p.Hkv, index = blockIdx.x / p.Hkv;
  Item it;
  if (FORM == RANGE && KV != KV_ROWS && BM == 16 && (MIXED || p.N)) {
    int tiles;
    const bool some = find_shared<KV, BM, BMF>(p, index, it, tiles);
    if (blockIdx.x == 0 && tid == 0) leave_head<HD>(p, it, tiles);
    if (!some) return;
  } else if (!find_item<KV, BM, false, FORM>(p, index, it)) {
    return;
  }
  if constexpr (MIXED)
    if (it.front) {
      tile_item<T, HD, KV, 4, RANGE, BM>(p, it, hk, reinterpret_cast<char*>(&lds));
      return;
    }
  R r;
  r.template begin<KV>(p, it, hk, it.tile * BM + lane % BM, lane);
  const int tok0 = it.tile * BM / p.G, tok1 = min(it.s.nq - 1, (it.tile * BM + BM - 1) / p.G);
  // WHOLE: steps are keys; RANGE: halves of the tile's blocks, of which those that no row sees are left out
  Blocks bl;
  int klo = 0, kbeg, kend, at, lo_lo = 0;
  if constexpr (FORM == RANGE) {
    bl = blocks<KV>(p, it, tok0, tok1);
    lo_lo = it.front ? 0 : p.N ? it.first : max(0, keys_of(p, it.s, tok0) - p.window);
    kbeg = it.nch > 1 ? 2 * it.chunk * it.c : 0;
    kend = it.nch > 1 ? min(2 * bl.nb, kbeg + 2 * it.c) : 2 * bl.nb;
    at = kbeg + wave;
  } else {
    klo = keys_of(p, it.s, tok0);
    const int khi = keys_of(p, it.s, tok1);
    kbeg = it.nch > 1 ? it.chunk * it.c * AT_KEYS : 0;
    kend = it.nch > 1 ? min(khi, kbeg + it.c * AT_KEYS) : khi;
    at = kbeg + wave * KEYS;
  }
  constexpr int STEP = FORM == RANGE ? NW : NW * KEYS;
  auto key_at = [&](int at) { return FORM == RANGE ? bl.key(at >> 1) + (at & 1) * KEYS : at; };
  auto seen_from = [&](int at) {   // the wave's first step from `at` on with a key that some row sees
    if constexpr (FORM == RANGE)
      while (at < kend) {
        const int key = key_at(at);
        if (key < bl.lim && (key + KEYS > lo_lo || key < p.sinks)) break;
        at += STEP;
      }
    return at;
  };
  at = seen_from(at);

  r.arrived();
  Stage<T, HD, KV, KEYS, 64, false, true, FORM == RANGE> ks;
  Stage<T, HD, KV, KEYS, 64, true, true, FORM == RANGE> vs;
  T* const kt = lds[wave];
  T* const vt = kt + (PARTS - 1) * TILE;
  if (at < kend) {
    ks.begin(p, it, hk, key_at(at), NW * KEYS, lane, 0, false);
    vs.begin(p, it, hk, key_at(at), NW * KEYS, lane, 0, false);
  }
  unsigned va[R::VA];
  r.values_at(va, vt, lane);
  if (at < kend) {
    ks.load(p, it, hk, key_at(at), lane, 0);
    vs.load(p, it, hk, key_at(at), lane, 0);
  }
  for (; at < kend;) {
    const int key0 = key_at(at), then = seen_from(at + STEP);
    const bool part = FORM == RANGE ? !((at >> 1) < bl.fs || ((at >> 1) >= bl.fa && (at >> 1) < bl.fb)) : key0 + KEYS > klo;
    wave_order();
    typename R::scores_t s;
    const bool more = then < kend;
    ks.store(kt, lane);
    if (more) ks.load(p, it, hk, key_at(then), lane, 0);
    if constexpr (PARTS == 1) {
      wave_order();
      r.look(s, kt, part, key0, lane);
      wave_order();
    }
    vs.store(vt, lane);
    if (more) vs.load(p, it, hk, key_at(then), lane, 0);
    wave_order();
    if constexpr (PARTS == 2) r.look(s, kt, part, key0, lane);
    const bool fix = part && __any(any_odd<T, TILE, 64>(vt, lane));
    if (fix) {
      for (int i = lane; i < 3 * HD; i += 64) (&bad[wave][0][0])[i] = FORM == RANGE ? 0 : 0x7FFFFFFF;
      wave_order();
      if constexpr (FORM == RANGE) take_out_odd<T, HD, KEYS, 64>(vt, bad[wave], lane);
      else take_out_odd<T, HD, KEYS, 64>(vt, bad[wave], key0, lane);
      wave_order();
    }
    r.take(s, va, p.scale_log2e, lane);
    if (fix) r.add_odd(bad[wave], key0, lane);
    at = then;
  }

  // ---- join the waves ----
  __syncthreads();
  const int rows = min(BM, it.s.nq * p.G - it.tile * BM);
  float* const ob = reinterpret_cast<float*>(&lds[0][0]);
  const float t = r.sum();
  if (lane < BM) ml[wave][lane] = float2_t{r.m * p.scale_log2e, t};
  if (lane % BM < rows) {
    // 16-byte chunk c of row q at c ^ (q & 7): 8 rows of a chunk in 8 different places
    float* o = ob + (wave * BM + lane % BM) * HD;
    r.chunks(lane, [&](int c, float4_t x) { *reinterpret_cast<float4_t*>(o + ((c ^ (lane & 7)) << 2)) = x; });
  }
  __syncthreads();
  for (int i = tid; i < rows * (HD / 4); i += 64 * NW) {
    const int q = i / (HD / 4), c = i % (HD / 4);
    float M = ml[0][q][0];
#pragma unroll
    for (int w = 1; w < NW; ++w) M = fmaxf(M, ml[w][q][0]);
    float sum = 0.f;
    float4_t a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float2_t x = ml[w][q];
      if (x[1] == 0.f) continue;   // saw no key; a maximum of -inf alone may stand for scores of NaN, and so does its sum
      const float f = __builtin_amdgcn_exp2f(x[0] - M);
      sum += f * x[1];
      a += f * *reinterpret_cast<const float4_t*>(ob + (w * BM + q) * HD + ((c ^ (q & 7)) << 2));
    }
    if (it.nch == 1 && (FORM != RANGE || KV == KV_ROWS || !p.N)) {
      const float rs = sum == 0.f ? 0.f : 1.0f / sum;
      const int row = it.tile * BM + q, tok = row / p.G;
      T* out = static_cast<T*>(p.out) + (long)(it.s.q0 + tok) * p.o_st + (long)(hk * p.G + row - tok * p.G) * p.o_sh + c * 4;
      const auto x = pack2<T>(a[0] * rs, a[1] * rs), y = pack2<T>(a[2] * rs, a[3] * rs);
      *reinterpret_cast<typename Elem<T>::v4*>(out) = typename Elem<T>::v4{x[0], x[1], y[0], y[1]};
    } else {
      const long row = part_row<BM, BMF, FORM>(p, it, hk, q);
      if (FORM == RANGE && row < 0) continue;
      *reinterpret_cast<float4_t*>(part_o<HD>(p, row) + c * 4) = a;
      if (c == 0) *part_ml<HD>(p, row) = float2_t{M, sum};
    }
  }
  if (FORM == RANGE && KV != KV_ROWS && p.N && tid == 0) leave_parts<HD, BM>(p, it, hk, it.tile);
}

// One group's (cg of CG) share of nch parts of a row, the first at `row`, added to a (chunk c), its sum and maximum.
template <int HD, int CG>
__device__ __forceinline__ void add_parts(const AttendParams& p, long row, long pitch, int nch, int cg, int c, float& M, float& sum, float4_t& a) {
  // four at a time, their loads together
  constexpr int AT = 4;
  for (int n0 = cg; n0 < nch; n0 += AT * CG) {
    float2_t x[AT];
    float4_t y[AT];
#pragma unroll
    for (int i = 0; i < AT; ++i) {
      const long at = row + (long)min(n0 + i * CG, nch - 1) * pitch;
      x[i] = *part_ml<HD>(p, at);
      y[i] = *reinterpret_cast<const float4_t*>(part_o<HD>(p, at) + c * 4);
    }
    float m = M;
#pragma unroll
    for (int i = 0; i < AT; ++i) {
      if (n0 + i * CG >= nch) x[i] = float2_t{-INFINITY, 0.f};
      m = fmaxf(m, x[i][0]);
    }
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - m);
    M = m;
    sum *= f;
    a *= f;
#pragma unroll
    for (int i = 0; i < AT; ++i) {
      if (x[i][1] == 0.f) continue;   // saw no key, has no O
      const float h = __builtin_amdgcn_exp2f(x[i][0] - m);
      sum += x[i][1] * h;
      a += y[i] * h;
    }
  }
}

// ---- the chunks of a tile joined ----------------------------------------------------------
// HD / 4 lanes a row, RP rows and CG groups of chunks a workgroup of 256.  Its work is small (4
// to 10 us); a launch of its own, as the last workgroup of a tile doing it needs counters that
// are zero at the start, and the workspace comes with whatever it held.
template <typename T, int HD, int KV, int BM, int FORM>
__global__ __launch_bounds__(256) void attend_join_kernel(const AttendParams p) {
  constexpr int LPR = HD / 4, CG = BM <= 32 ? 256 / LPR : 1, RP = 256 / LPR / CG;
  __shared__ float4_t so[CG][LPR];
  __shared__ float2_t sm[CG];
  const int hk = blockIdx.x % p.Hkv, index = blockIdx.x / p.Hkv;
  Item it;
  // (offsets that do not ascend may name more rows than there are: what has no item has no sums)
  if (!find_item<KV, BM, true, FORM>(p, index, it) || it.nch == 1 || it.base < 0 || it.base + it.nch > p.items) return;
  const int c = threadIdx.x % LPR, cg = CG > 1 ? threadIdx.x / LPR : 0;
  const int q = blockIdx.y * RP + (CG > 1 ? 0 : threadIdx.x / LPR);
  const int tile = BM <= 32 ? it.tile : tiles_of<KV, BM>(it.s, p.G) - 1 - it.tile;
  const bool in = (long)tile * BM + q < (long)it.s.nq * p.G;
  if (CG > 1 && !in) return;
  float M = -INFINITY, sum = 0.f;
  float4_t a = {0.f, 0.f, 0.f, 0.f};
  if (in) add_parts<HD, CG>(p, ((long)it.base * p.Hkv + hk) * BM + q, (long)p.Hkv * BM, it.nch, cg, c, M, sum, a);
  if constexpr (CG > 1) {
    so[cg][c] = a;
    if (c == 0) sm[cg] = float2_t{M, sum};
    __syncthreads();
    if (cg) return;
#pragma unroll
    for (int w = 1; w < CG; ++w) M = fmaxf(M, sm[w][0]);
    sum = 0.f;
    a = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < CG; ++w) {
      if (sm[w][1] == 0.f) continue;
      const float f = __builtin_amdgcn_exp2f(sm[w][0] - M);
      sum += f * sm[w][1];
      a += f * so[w][c];
    }
  }
  if (!in) return;
  const float rs = sum == 0.f ? 0.f : 1.0f / sum;
  const int row = tile * BM + q, tok = row / p.G;
  T* out = static_cast<T*>(p.out) + (long)(it.s.q0 + tok) * p.o_st + (long)(hk * p.G + row - tok * p.G) * p.o_sh + c * 4;
  const auto x = pack2<T>(a[0] * rs, a[1] * rs), y = pack2<T>(a[2] * rs, a[3] * rs);
  *reinterpret_cast<typename Elem<T>::v4*>(out) = typename Elem<T>::v4{x[0], x[1], y[0], y[1]};
}

// Shared pages: a sequence's own parts and those of its group's front, by the Parts that the launch before left.
template <typename T, int HD, int BM, int BMF>
__global__ __launch_bounds__(256) void attend_join_shared_kernel(const AttendParams p) {
  constexpr int LPR = HD / 4, CG = BM <= 32 ? 256 / LPR : 1, RP = 256 / LPR / CG;
  __shared__ float4_t so[CG][LPR];
  __shared__ float2_t sm[CG];
  const int hk = blockIdx.x % p.Hkv, index = blockIdx.x / p.Hkv;
  const int tiles = parts_head<HD>(p)[0], fronts = parts_head<HD>(p)[1];
  const Parts x = parts_at<HD>(p)[index];
  const int c = threadIdx.x % LPR, cg = CG > 1 ? threadIdx.x / LPR : 0;
  const int q = blockIdx.y * RP + (CG > 1 ? 0 : threadIdx.x / LPR);
  // (offsets that do not ascend may name more rows than there are; a tile without an item then has no Parts, and what
  // stands there is held to the tensors)
  const bool sound = index < tiles && fronts >= 0 && fronts <= p.front_items && x.nch > 0 && x.own >= 0 && x.own <= p.own_items - x.nch &&
                     x.rows <= BM && x.row0 >= 0 && x.q0 >= 0 && (long)x.q0 * p.G + x.row0 + x.rows <= (long)p.Tq * p.G;
  const bool in = sound && q < x.rows;
  if (CG > 1 && !in) return;
  float M = -INFINITY, sum = 0.f;
  float4_t a = {0.f, 0.f, 0.f, 0.f};
  if (in) {
    add_parts<HD, CG>(p, (long)fronts * p.Hkv * BMF + ((long)x.own * p.Hkv + hk) * BM + q, (long)p.Hkv * BM, x.nch, cg, c, M, sum, a);
    const long of = (long)x.frow0 + q;
    if (x.fnch > 0 && x.frow0 >= 0 && of < x.frows && x.frows <= (long)p.Tq * p.G) {
      // its tile of the group's rows (those of 128 come last first), chunk by chunk
      const long ftiles = ((long)x.frows + BMF - 1) / BMF, ft = of / BMF, item = x.front + (BMF <= 32 ? ft : ftiles - 1 - ft);
      if (item >= 0 && item + (x.fnch - 1) * ftiles < fronts)
        add_parts<HD, CG>(p, (item * p.Hkv + hk) * BMF + of % BMF, ftiles * p.Hkv * BMF, x.fnch, cg, c, M, sum, a);
    }
  }
  if constexpr (CG > 1) {
    so[cg][c] = a;
    if (c == 0) sm[cg] = float2_t{M, sum};
    __syncthreads();
    if (cg) return;
#pragma unroll
    for (int w = 1; w < CG; ++w) M = fmaxf(M, sm[w][0]);
    sum = 0.f;
    a = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < CG; ++w) {
      if (sm[w][1] == 0.f) continue;
      const float f = __builtin_amdgcn_exp2f(sm[w][0] - M);
      sum += f * sm[w][1];
      a += f * so[w][c];
    }
  }
  if (!in) return;
  const float rs = sum == 0.f ? 0.f : 1.0f / sum;
  const int row = x.row0 + q, tok = row / p.G;
  T* out = static_cast<T*>(p.out) + (long)(x.q0 + tok) * p.o_st + (long)(hk * p.G + row - tok * p.G) * p.o_sh + c * 4;
  const auto u = pack2<T>(a[0] * rs, a[1] * rs), v = pack2<T>(a[2] * rs, a[3] * rs);
  *reinterpret_cast<typename Elem<T>::v4*>(out) = typename Elem<T>::v4{u[0], u[1], v[0], v[1]};
}

// ---- host ---------------------------------------------------------------------------------
// The form of a call: rows per tile, items per K/V head to aim at (0: keys are not split).
struct Plan {
  int bm, target, min_blocks;
  int bmf;             // shared pages: rows of the fronts' tiles
  long front_items, own_items;
  long tiles, items;   // at most
};
template <typename T, int HD, int KV>
void launch_shared(const AttendParams& p, const Plan& pl, hipStream_t s) {
  const dim3 grid((unsigned)(pl.items * p.Hkv));
  const unsigned tiles = (unsigned)(pl.tiles * p.Hkv);
  if (pl.bmf == 16) {
    CK_LAUNCH((attend_few_kernel<T, HD, KV, Rows16<T, HD, RANGE>, RANGE>), grid, dim3(256), 0, s, p);
    CK_LAUNCH((attend_join_shared_kernel<T, HD, 16, 16>), dim3(tiles, 16), dim3(256), 0, s, p);
  } else if (pl.bm == 16) {
    CK_LAUNCH((attend_few_kernel<T, HD, KV, Rows16<T, HD, RANGE>, RANGE, true>), grid, dim3(256), 0, s, p);
    CK_LAUNCH((attend_join_shared_kernel<T, HD, 16, 128>), dim3(tiles, 16), dim3(256), 0, s, p);
  } else {
    CK_LAUNCH((attend_tile_kernel<T, HD, KV, 4, RANGE>), grid, dim3(256), 0, s, p);
    CK_LAUNCH((attend_join_shared_kernel<T, HD, 128, 128>), dim3(tiles, 128 / (1024 / HD)), dim3(256), 0, s, p);
  }
}
template <typename T, int HD, int KV, int FORM>
void launch_kv(const AttendParams& p, const Plan& pl, hipStream_t s) {
  if constexpr (FORM == RANGE && KV != KV_ROWS)
    if (p.N) return launch_shared<T, HD, KV>(p, pl, s);
  const dim3 grid((unsigned)(pl.items * p.Hkv));
  if (pl.bm == 16) CK_LAUNCH((attend_few_kernel<T, HD, KV, Rows16<T, HD, FORM>, FORM>), grid, dim3(64 * FEW_WAVES), 0, s, p);
  else if (pl.bm == 32) CK_LAUNCH((attend_few_kernel<T, HD, KV, Rows<T, HD, FORM>, FORM>), grid, dim3(64 * FEW_WAVES), 0, s, p);
  else if (pl.bm == 128) CK_LAUNCH((attend_tile_kernel<T, HD, KV, 4, FORM>), grid, dim3(256), 0, s, p);
  else if constexpr (FORM == WHOLE) CK_LAUNCH((attend_tile_kernel<T, HD, KV, 8, FORM>), grid, dim3(512), 0, s, p);
  if (!pl.target) return;
  const unsigned tiles = (unsigned)(pl.tiles * p.Hkv);
  if (pl.bm == 16) CK_LAUNCH((attend_join_kernel<T, HD, KV, 16, FORM>), dim3(tiles, 16), dim3(256), 0, s, p);
  else if (pl.bm == 32) CK_LAUNCH((attend_join_kernel<T, HD, KV, 32, FORM>), dim3(tiles, 32), dim3(256), 0, s, p);
  else CK_LAUNCH((attend_join_kernel<T, HD, KV, 128, FORM>), dim3(tiles, 128 / (1024 / HD)), dim3(256), 0, s, p);
}
template <typename T, int HD, int FORM>
void launch_hd(const AttendParams& p, int kv, const Plan& pl, hipStream_t s) {
  if (kv == KV_ROWS) launch_kv<T, HD, KV_ROWS, FORM>(p, pl, s);
  else if (kv == KV_PAGES) launch_kv<T, HD, KV_PAGES, FORM>(p, pl, s);
  else launch_kv<T, HD, KV_E4M3, FORM>(p, pl, s);
}

// The checks of a call, and its part of the parameters; false: there is nothing to do.
inline bool attend_begin(const std::string& w, AttendParams& p, const AttendQuery& a) {
  CK_REQUIRE(a.dtype == DT_F16 || a.dtype == DT_BF16, w + ": q must be f16 or bf16");
  CK_REQUIRE(a.head_dim == 64 || a.head_dim == 128, w + ": head_dim must be 64 or 128");
  CK_REQUIRE(a.n_heads > 0 && p.Hkv > 0 && a.n_heads % p.Hkv == 0 && a.n_heads <= 1024,
             w + ": query heads (up to 1024) must be a multiple of the K/V heads");
  CK_REQUIRE(a.T >= 0 && a.B >= 0 && (long)a.T * a.n_heads < (1L << 31) && a.B < (1 << 20), w + ": bad sizes");
  // (the exponents are of 2: past 2.3e38 their factor is infinite)
  CK_REQUIRE(a.scale > 0.f && a.scale * AT_LOG2E < INFINITY, w + ": scale must be positive and finite, and under 2e38");
  if (a.T == 0 || a.B == 0) return false;
  CK_REQUIRE(a.q && a.out && a.cu_q && p.kv, w + ": null pointer");
  // a lane's bytes from its wave's first row are counted in 32 bits
  CK_REQUIRE(p.k_st < (1L << 24) && p.v_st < (1L << 24) && p.k_st >= 0 && p.v_st >= 0, w + ": token strides must be under 2^24");
  CK_REQUIRE(((a.q_st | a.q_sh) & 7) == 0 && ((a.o_st | a.o_sh) & 3) == 0 && (reinterpret_cast<uintptr_t>(a.q) & 15) == 0 &&
                 (reinterpret_cast<uintptr_t>(a.out) & 7) == 0,
             w + ": q rows must be 16-byte and out rows 8-byte aligned");
  p.q = a.q;
  p.out = a.out;
  p.q_st = a.q_st;
  p.q_sh = a.q_sh;
  p.o_st = a.o_st;
  p.o_sh = a.o_sh;
  p.cu_q = a.cu_q;
  p.B = a.B;
  p.Tq = a.T;
  p.G = a.n_heads / p.Hkv;
  p.causal = a.causal;
  p.scale_log2e = a.scale * AT_LOG2E;
  return true;
}
// The workspace (floats) checked, the launches.
template <int FORM>
void attend_launch(const std::string& w, AttendParams& p, const AttendQuery& a, int kv, const Plan& pl, size_t need, hipStream_t s) {
  // (a launch has under 2^32 threads)
  CK_REQUIRE(pl.items * p.Hkv < (1L << 32) / std::max(256, 2 * pl.bm), w + ": too many sequences and rows for one launch");
  if (need) {
    CK_REQUIRE(a.ws && a.ws_floats >= need,
               w + ": workspace too small (" + (FORM == RANGE ? "ck_attention_range_workspace" : "ck_attention_workspace") + ")");
    CK_REQUIRE((reinterpret_cast<uintptr_t>(a.ws) & 15) == 0, w + ": workspace must be 16-byte aligned");
  }
  p.target = pl.target;
  p.min_blocks = pl.min_blocks;
  p.ws = a.ws;
  p.items = (int)pl.items;
  p.part_rows = p.N ? (pl.front_items * pl.bmf + pl.own_items * pl.bm) * p.Hkv : pl.items * p.Hkv * pl.bm;
  p.front_items = (int)pl.front_items;
  p.own_items = (int)pl.own_items;
  if (a.dtype == DT_F16) {
    if (a.head_dim == 64) launch_hd<half_t, 64, FORM>(p, kv, pl, s);
    else launch_hd<half_t, 128, FORM>(p, kv, pl, s);
  } else {
    if (a.head_dim == 64) launch_hd<bf16_t, 64, FORM>(p, kv, pl, s);
    else launch_hd<bf16_t, 128, FORM>(p, kv, pl, s);
  }
  CK_LAUNCHED(w);
}

}  // namespace

// The calls of attend_range.hip.
size_t attend_range_floats(int B, int Tq, long keys, int n_heads, int n_kv, int head_dim, int window, int sinks, int groups);
void launch_attend_range(const char* what, AttendParams& p, const AttendQuery& a, int kv, long keys, hipStream_t s);

}  // namespace ck
