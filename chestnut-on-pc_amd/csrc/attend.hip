// Attention of packed sequences and over a paged cache, every row seeing all keys below its limit
// (attend.h; a sliding window and shared pages: attend_range.hip).
#include "attend.h"

namespace ck {
namespace {

// keys: the most that the sequences can have, all together; few3: three workgroups of few rows
// run on a CU.  (The workspace is asked for without that: the larger of the two counts.)
Plan plan_of(int B, int Tq, long keys, int n_heads, int n_kv, bool few3 = false) {
  Plan pl{};
  const int G = n_heads / n_kv;
  const long rows = (long)Tq * G;
  // 16 or 32 rows where a sequence has that many on average: bound by the keys, not by the rows.
  // 256 rows where they fill the 256 CUs at least twice without splitting keys (prompts of 16384
  // tokens, 446 us against 460 with 128); with fewer, tiles of 256 with their keys split take
  // 80 us against 82 (512 tokens on 12800 keys) and 81 against 77 (eight mixed chunks).
  pl.bm = rows <= 16L * B ? 16 : rows <= 32L * B ? 32 : (rows / 256 + B) * n_kv >= 512 ? 256 : 128;
  pl.tiles = rows / pl.bm + B;       // sum of ceil(rows_b / bm) is at most this
  // items to aim at: workgroups that run at once, two a CU (tiles of 128, three, four, six
  // a CU in place of two: 512 tokens on 12800 keys 99, 104, 119 for 86 us); of few rows twice as
  // many, as their chunks come out uneven (32 ragged histories 127 -> 122 us; three times 125),
  // or as many where three run on a CU (768 items 110 us, 1024 136, 1536 113; where two do, 16 of
  // the histories, 768 110 and 1024 104)
  const long slots = pl.bm == 128 ? 512 : pl.bm == 16 && few3 ? 768 : 1024;
  pl.min_blocks = pl.bm <= 32 ? 2 : 4;
  // keys stay whole where the tiles fill the card twice, or the sequences have too few to pay for
  // the second launch (prompts of 548, 652 and less, 128 features, split 31 us, whole 20; one of
  // 1031 with two short ones 20 and 26, but the host knows the average only)
  const bool many = pl.bm == 256 || (pl.bm == 128 && pl.tiles * n_kv >= 2 * slots);
  if (!many && keys / B > 2 * pl.min_blocks * AT_KEYS) pl.target = (int)std::max(1L, slots / n_kv);
  pl.items = pl.tiles + pl.target;
  return pl;
}

void launch_attend(const char* what, AttendParams& p, const AttendQuery& a, int kv, long keys, hipStream_t s) {
  if (a.window || a.groups) return launch_attend_range(what, p, a, kv, keys, s);
  if (!attend_begin(what, p, a)) return;
  const Plan pl = plan_of(a.B, a.T, keys, a.n_heads, p.Hkv, a.head_dim == 128 && kv == KV_E4M3);
  const size_t need = pl.target ? attention_workspace(a.B, a.T, keys, a.n_heads, p.Hkv, a.head_dim) : 0;
  attend_launch<WHOLE>(what, p, a, kv, pl, need, s);
}

}  // namespace

size_t attention_workspace(int B, int Tq, long keys, int n_heads, int n_kv, int head_dim, int window, int sinks, int groups) {
  CK_REQUIRE(B >= 0 && Tq >= 0 && keys >= 0 && n_kv > 0 && n_heads > 0 && n_heads % n_kv == 0 && head_dim > 0,
             "attention_workspace: bad sizes");
  CK_REQUIRE(window >= 0 && sinks >= 0 && groups >= 0 && groups < (1 << 20), "attention_workspace: bad sizes");
  if (B == 0 || Tq == 0) return 0;
  if (window || groups) return attend_range_floats(B, Tq, keys, n_heads, n_kv, head_dim, window, sinks, groups);
  const Plan pl = plan_of(B, Tq, keys, n_heads, n_kv);
  return pl.target ? (size_t)pl.items * n_kv * pl.bm * (head_dim + 2) : 0;
}

void launch_attention_varlen(const AttendQuery& a, const void* k, const void* v, long kst, long ksh, long vst, long vsh,
                             const int* cu_k, int Tk, int n_kv, hipStream_t s) {
  AttendParams p{};
  CK_REQUIRE(Tk >= 0 && Tk <= (1 << 30) && n_kv > 0, "attention_varlen: bad sizes");
  CK_REQUIRE(a.T == 0 || Tk == 0 || (k && v), "attention_varlen: null pointer");
  CK_REQUIRE(((kst | ksh | vst | vsh) & 7) == 0 && ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0,
             "attention_varlen: k and v rows must be 16-byte aligned");
  p.k = k;
  p.v = v;
  p.k_st = kst;
  p.k_sh = ksh;
  p.v_st = vst;
  p.v_sh = vsh;
  p.kv = cu_k;
  p.Tk = Tk;
  p.Hkv = n_kv;
  launch_attend("attention_varlen", p, a, KV_ROWS, Tk, s);
}

void launch_attention_paged(const AttendQuery& a, const PagedCache& c, const int* table, int table_w, const int* kv_lens,
                            hipStream_t s) {
  check_pages("attention_paged", c);
  CK_REQUIRE(c.dtype == a.dtype || c.dtype == DT_E4M3, "attention_paged: the cache must be of q's type or e4m3");
  CK_REQUIRE(c.head_dim == a.head_dim, "attention_paged: the cache's head_dim must be q's");
  CK_REQUIRE(table_w >= 0 && (table || !table_w || !a.B || !a.T), "attention_paged: null block table");
  CK_REQUIRE((long)table_w * c.page <= (1L << 30), "attention_paged: at most 2^30 places a sequence");
  AttendParams p{};
  p.k = c.k;
  p.v = c.v;
  p.ks = c.k_scale;
  p.vs = c.v_scale;
  p.table = table;
  p.table_w = table_w;
  p.kv = kv_lens;
  p.Hkv = c.n_kv;
  p.page_shift = page_shift(c.page);
  p.n_pages = c.n_pages;
  launch_attend("attention_paged", p, a, c.dtype == DT_E4M3 ? KV_E4M3 : KV_PAGES,
                (long)a.B * table_w * c.page, s);
}

}  // namespace ck
