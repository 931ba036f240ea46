// Attention through a sliding window, and of sequences that share their first pages (attend.h).
#include "attend.h"

namespace ck {
namespace {

constexpr int MOST_KEYS = 1 << 30;   // of a sequence: a window of as many is none

// As plan_of (attend.hip) where window and groups are 0.
Plan range_plan(int B, int Tq, long keys, int n_heads, int n_kv, int window, int sinks, int groups, bool few3 = false) {
  Plan pl{};
  const int G = n_heads / n_kv;
  const long rows = (long)Tq * G;
  if (groups) {
    // the rows that share keys are a group's: tiles where it has more than 16 on average (24 tokens on 12800 shared keys, 8
    // heads of 64, 22.0 us by 32 few rows, 18.6 by tiles; 12 of 4 heads a K/V head of 128, f16, 32.1 and 20.1; of up to 16
    // rows, 4 such tokens, 17.8 by few and 18.9 by tiles), and single tokens' own keys by few rows beside them
    pl.bmf = rows <= 16L * groups ? 16 : 128;
    pl.bm = rows <= 16L * (pl.bmf == 16 ? groups : B) ? 16 : 128;
    pl.tiles = rows / pl.bm + B;                // the sequences' own
    const long fronts = rows / pl.bmf + groups, slots = pl.bmf == 128 ? 512 : pl.bmf == 16 && few3 ? 768 : 1024;
    pl.min_blocks = pl.bmf == 16 ? 2 : 4;
    const bool many = pl.bmf == 128 && (fronts + pl.tiles) * n_kv >= 2 * slots;
    if (!many && keys / B > 2 * pl.min_blocks * AT_KEYS) pl.target = (int)std::max(1L, slots / n_kv);
    pl.front_items = fronts + pl.target;
    pl.own_items = pl.tiles + pl.target;
    pl.items = fronts + pl.tiles + pl.target;
    return pl;
  }
  pl.bm = rows <= 16L * B ? 16 : rows <= 32L * B ? 32 : 128;
  pl.tiles = rows / pl.bm + B;
  const long slots = pl.bm == 128 ? 512 : pl.bm == 16 && few3 ? 768 : 1024;
  pl.min_blocks = pl.bm <= 32 ? 2 : 4;
  const bool many = pl.bm == 128 && pl.tiles * n_kv >= 2 * slots;
  const long each = std::min(keys / B, (long)window + sinks + pl.bm / G);
  // few rows through up to 768 keys: six steps of the few-row kernel, and one launch (516 keys 18.0 -> 13.9 us a call,
  // 1028 keys of e4m3, 128 features, 18.7 and whole 19.8)
  if (!many && each > (pl.bm <= 32 ? 768 : 2 * pl.min_blocks * AT_KEYS)) pl.target = (int)std::max(1L, slots / n_kv);
  pl.items = pl.tiles + pl.target;
  return pl;
}

}  // namespace

size_t attend_range_floats(int B, int Tq, long keys, int n_heads, int n_kv, int head_dim, int window, int sinks, int groups) {
  const Plan pl = range_plan(B, Tq, keys, n_heads, n_kv, window, sinks, groups);
  if (groups)
    return (size_t)(pl.front_items * pl.bmf + pl.own_items * pl.bm) * n_kv * (head_dim + 2) + 4 + (size_t)pl.own_items * (sizeof(Parts) / 4);
  return pl.target ? (size_t)pl.items * n_kv * pl.bm * (head_dim + 2) : 0;
}

void launch_attend_range(const char* what, AttendParams& p, const AttendQuery& a, int kv, long keys, hipStream_t s) {
  const std::string w(what);
  CK_REQUIRE(a.window >= 0 && a.sinks >= 0 && a.groups >= 0 && a.groups < (1 << 20), w + ": window, sinks and groups (under 2^20) must not be negative");
  CK_REQUIRE(!a.window || a.causal, w + ": a window belongs to causal attention");
  CK_REQUIRE(a.window || !a.sinks, w + ": sinks belong to a window");
  CK_REQUIRE(!a.window || !a.groups, w + ": a window and shared pages exclude each other");
  CK_REQUIRE(!a.groups || kv != KV_ROWS, w + ": shared pages belong to a cache");
  if (!attend_begin(w, p, a)) return;
  CK_REQUIRE(!a.groups || (a.cu_shared && a.shared_lens), w + ": null pointer");
  p.window = std::min(a.window, MOST_KEYS);
  p.sinks = std::min(a.sinks, MOST_KEYS);
  p.N = a.groups;
  p.cu_s = a.cu_shared;
  p.s_lens = a.shared_lens;
  const Plan pl = range_plan(a.B, a.T, keys, a.n_heads, p.Hkv, a.window, a.sinks, a.groups, a.head_dim == 128 && kv == KV_E4M3);
  const size_t need = pl.target || a.groups ? attend_range_floats(a.B, a.T, keys, a.n_heads, p.Hkv, a.head_dim, a.window, a.sinks, a.groups) : 0;
  attend_launch<RANGE>(w, p, a, kv, pl, need, s);
}

}  // namespace ck
