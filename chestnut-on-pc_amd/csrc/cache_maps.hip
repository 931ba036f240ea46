// The index tensors of a step over the paged cache, from the lengths of its requests: new[b] new
// tokens behind the kv[b] places that request b has.
//   cu[b + 1] = cu[b] + new[b],   kv_out[b] = kv[b] + new[b]
//   request b takes need[b] = ceil(kv_out[b] / page) - ceil(kv[b] / page) pages, in the order of the
//   requests and of their places, from free[taken] on; taken_out = taken + sum need
//   row t = cu[b] + i: place = kv[b] + i, its page table[b][place / page] (old, or one just taken),
//   slot = page * size + place % size; no page: -1.  Rows behind the last request: place 0, slot -1.
//
// Bound by latency: one load of the lengths, their scan, one load of a page index, the stores.
// Every workgroup of 1024 threads scans all lengths by itself (two loads a thread and 1024
// requests) and then has 1024 rows: a launch more would cost more than that does.  The last
// request that begins at or before a row in its workgroup is its own: requests leave their data
// in LDS at the row they begin at, and a row finds the last such place by a ballot.  A new page
// goes to the table by the row that comes first on it.  32 requests of a token each
// 3.2 us; 700 requests, 359400 rows, 2.9 MB, 7.1 us (64-bit sums by shuffles 8.9).  In two
// launches (MapsMode): those 700 with their lengths or the list's cursor in place 2.5 and 5.2 us, 5000
// requests of a token each 9.8 and 4.7.
#include "common.h"
#include "elem16.h"
#include "kernels.h"
#include "lanes_scan.h"

namespace ck {
namespace {

constexpr int CM_ROWS = 1024, CM_WAVES = CM_ROWS / 64;
constexpr long CM_MOST = 0x7FFFFFFF;   // sums are held at this

struct MapsParams {
  const int *new_lens, *kv;
  int* table;
  const int *free_pages, *taken;
  int *cu, *kv_out, *positions, *slots, *taken_out;
  int *old, *first;       // two launches: each request's places before (kv may be overwritten) and first page in the list, [B]
  int B, width, shift, T, n_free;
};

struct Scan {
  long rows, pages;
};
// Sums over lanes 0..l, in lane l: by DPP where 32 bits hold them, as they do but for lengths that make no sense.
__device__ __forceinline__ Scan wave_scan(int rows, int pages, int lane) {
  if (!__any(rows >= 1 << 24 || pages >= 1 << 24)) return Scan{lanes_scan(rows), lanes_scan(pages)};
  Scan v{rows, pages};
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const long r = __shfl_up(v.rows, d), g = __shfl_up(v.pages, d);
    if (lane >= d) v = Scan{v.rows + r, v.pages + g};
  }
  return v;
}
__device__ __forceinline__ int held(long v) { return (int)min(v, CM_MOST); }
__device__ __forceinline__ int pages_of(long places, int shift) { return (int)((places + (1 << shift) - 1) >> shift); }

// What a request leaves for its rows: place - row within the workgroup, pages that it had, and
// where in the list the page of column 0 would stand.
struct Mine {
  int b, delta, have, list;
};

enum MapsMode { MAPS_ALL = 0, MAPS_SCAN = 1, MAPS_ROWS = 2 };

// MAPS_ALL: everything; MAPS_SCAN, MAPS_ROWS: the requests by one workgroup, then the rows, where
// kv or taken is overwritten (the others would read it late) or the requests are too many to
// scan once a workgroup.
template <MapsMode MODE>
__global__ __launch_bounds__(CM_ROWS) void cache_maps_kernel(const MapsParams p) {
  __shared__ Scan part[CM_WAVES];
  __shared__ Mine mine[CM_ROWS];
  __shared__ unsigned long long marks[CM_WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const bool writes = MODE == MAPS_SCAN || (MODE == MAPS_ALL && blockIdx.x == 0);
  const long t0 = (long)blockIdx.x * CM_ROWS;
  const long taken = p.taken ? max(*p.taken, 0) : 0;
  if (MODE != MAPS_SCAN) mine[tid].b = -1;
  __syncthreads();
  // request b's rows from `start` on, n of them, its places from `old` on, its pages from `first` on
  auto leave = [&](int b, long start, int n, int old, long first) {
    if (n <= 0 || start >= t0 + CM_ROWS || start + n <= t0) return;
    const int at = (int)max(start - t0, 0l), have = pages_of(old, p.shift);
    mine[at] = Mine{b, (int)min((long)old + (t0 - start), CM_MOST), have, (int)max(min(first - have, CM_MOST), -CM_MOST)};
  };
  long rows = 0;    // of all requests
  if (MODE != MAPS_ROWS) {
    Scan sum{0, taken};
    for (int b0 = 0; b0 < p.B; b0 += CM_ROWS) {
      const int b = b0 + tid;
      int n = 0, old = 0;
      if (b < p.B) {
        n = max(p.new_lens[b], 0);
        old = max(p.kv[b], 0);
      }
      const int need = pages_of((long)old + n, p.shift) - pages_of(old, p.shift);
      const Scan s = wave_scan(n, need, lane);
      if (b0) __syncthreads();   // part of the requests before has been read
      if (lane == 63) part[wave] = s;
      __syncthreads();
      Scan before = sum;
      for (int w = 0; w < CM_WAVES; ++w) {
        if (w < wave) before = Scan{before.rows + part[w].rows, before.pages + part[w].pages};
        sum = Scan{sum.rows + part[w].rows, sum.pages + part[w].pages};
      }
      const long start = before.rows + s.rows - n, first = before.pages + s.pages - need;
      if (MODE == MAPS_ALL) leave(b, start, n, old, first);
      if (writes && b < p.B) {
        p.cu[b + 1] = held(start + n);
        p.kv_out[b] = held((long)old + n);
        if (MODE == MAPS_SCAN) {
          p.old[b] = old;
          p.first[b] = held(first);
        }
      }
    }
    rows = sum.rows;
    if (writes && tid == 0) {
      p.cu[0] = 0;
      if (p.taken_out) *p.taken_out = held(sum.pages);
    }
  } else {
    // the first request that ends behind t0: every wave looks for it alone, 64 places a step
    int lo = 0, hi = p.B;   // it is in lo .. hi, hi: none
    while (hi > lo) {
      const int step = (hi - lo + 63) / 64, b = lo + lane * step;
      const unsigned long long m = __ballot(b < hi && p.cu[min(b, p.B - 1) + 1] > t0);
      // those before the first of a set bit end at or before t0
      const int f = m ? __ffsll(m) - 1 : (hi - lo + step - 1) / step;
      const int last = min(lo + f * step, hi);
      lo = f ? min(lo + (f - 1) * step + 1, hi) : lo;
      hi = last;
    }
    rows = p.cu[p.B];
    for (int b = lo + tid; b < p.B; b += CM_ROWS) {
      const long start = p.cu[b];
      if (start >= t0 + CM_ROWS) break;
      // (n and old not from cu's and kv_out's differences: these are held at 2^31 - 1)
      leave(b, start, max(p.new_lens[b], 0), p.old[b], p.first[b]);
    }
  }
  if (MODE == MAPS_SCAN) return;
  __syncthreads();
  const unsigned long long m = __ballot(mine[tid].b >= 0);
  if (lane == 0) marks[wave] = m;
  __syncthreads();
  const long t = t0 + tid;
  if (t >= p.T) return;
  int place = 0, slot = -1;
  if (t < rows) {
    int at = -1;
    const unsigned long long up_to = m & (~0ull >> (63 - lane));
    if (up_to) at = wave * 64 + 63 - __clzll(up_to);
    else
      for (int w = wave - 1; w >= 0 && at < 0; --w)
        if (marks[w]) at = w * 64 + 63 - __clzll(marks[w]);
    if (at >= 0) {
      const Mine x = mine[at];
      place = (int)min((long)x.delta + tid, CM_MOST);
      const int col = place >> p.shift, in = place & ((1 << p.shift) - 1);
      int page = -1;
      if (col < p.width) {
        int* const entry = p.table + (long)x.b * p.width + col;
        if (col < x.have || !p.free_pages) {
          page = *entry;
        } else {
          const long i = (long)x.list + col;
          if (i >= 0 && i < p.n_free) page = p.free_pages[i];
          if (in == 0) *entry = page;
        }
      }
      const long s = ((long)page << p.shift) + in;
      if (page >= 0 && s <= CM_MOST) slot = (int)s;
    }
  }
  p.positions[t] = place;
  p.slots[t] = slot;
}

// Both launches where something is overwritten that other workgroups read, or where more than 4096
// requests would be scanned by each of them.
bool in_two(int B, int tokens, bool in_place) { return B > 0 && tokens > CM_ROWS && (in_place || B > 4096); }

}  // namespace

size_t cache_maps_workspace(int B, int tokens, bool in_place) {
  CK_REQUIRE(B >= 0 && tokens >= 0, "cache_maps: bad sizes");
  return in_two(B, tokens, in_place) ? 2 * sizeof(int) * (size_t)B : 0;
}

void launch_cache_maps(const CacheMaps& m, hipStream_t s) {
  CK_REQUIRE(m.B >= 0 && m.B < (1 << 20) && m.width >= 0 && m.tokens >= 0 && m.tokens < (1 << 30) && m.n_free >= 0,
             "cache_maps: bad sizes (under 2^20 requests and 2^30 rows)");
  CK_REQUIRE(m.page >= 16 && m.page <= 1024 && (m.page & (m.page - 1)) == 0, "cache_maps: page size must be a power of two from 16 to 1024");
  CK_REQUIRE((long)m.width * m.page <= (1L << 30), "cache_maps: at most 2^30 places a request");
  CK_REQUIRE(m.cu && (!m.B || (m.new_lens && m.kv && m.kv_out)) && (!m.B || !m.width || m.table) &&
                 (!m.tokens || (m.positions && m.slots)),
             "cache_maps: null pointer");
  CK_REQUIRE(!m.free_pages == !m.taken && !m.taken == !m.taken_out, "cache_maps: free pages need the number of them that is taken");
  const bool two = in_two(m.B, m.tokens, m.kv_out == m.kv || (m.taken && m.taken_out == m.taken));
  CK_REQUIRE(!two || (m.ws && m.ws_bytes >= 2 * sizeof(int) * (size_t)m.B), "cache_maps: workspace too small (ck_cache_maps_workspace)");
  MapsParams p{};
  p.new_lens = m.new_lens;
  p.kv = m.kv;
  p.table = m.table;
  p.free_pages = m.free_pages;
  p.taken = m.taken;
  p.cu = m.cu;
  p.kv_out = m.kv_out;
  p.positions = m.positions;
  p.slots = m.slots;
  p.taken_out = m.taken_out;
  p.old = m.ws;
  p.first = m.ws + m.B;
  p.B = m.B;
  p.width = m.width;
  p.shift = page_shift(m.page);
  p.T = m.tokens;
  p.n_free = m.n_free;
  const dim3 grid(std::max(1, ceil_div(m.tokens, CM_ROWS))), block(CM_ROWS);
  if (two) {
    CK_LAUNCH(cache_maps_kernel<MAPS_SCAN>, dim3(1), block, 0, s, p);
    CK_LAUNCH(cache_maps_kernel<MAPS_ROWS>, grid, block, 0, s, p);
  } else {
    CK_LAUNCH(cache_maps_kernel<MAPS_ALL>, grid, block, 0, s, p);
  }
  CK_LAUNCHED("cache_maps");
}

}  // namespace ck
