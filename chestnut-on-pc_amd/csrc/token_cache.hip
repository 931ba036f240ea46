// Writing and reading a paged cache of K and V rows.
//
// A cache is `n_pages` pages of [Hkv][page][hd] elements, K and V apart: the rows of one
// head on one page lie together, which is what attention reads in one go.  The elements
// are the model's (f16, bf16) or e4m3 with one scale a row, a power of two kept as its
// biased exponent: the least 2^e with amax <= 448 * 2^e.  A power of two makes the
// scaling and its undoing exact, so the one rounding is the one to e4m3 (nearest even);
// a float format gains nothing from a finer scale but the last bits of its range.
//
// Bound by memory: every row is read and written once.
#include "common.h"
#include "elem16.h"
#include "kernels.h"

namespace ck {
namespace {

struct WriteParams {
  const void *k, *v;
  void *kp, *vp;
  uint8_t *ks, *vs;
  const int* slots;
  long kst, ksh, vst, vsh;
  int T, Hkv, hd, page_shift;
  long n_slots;
  unsigned rows;   // T * Hkv
};

// Rows in the cache: slot's page, head h, place.
__device__ __forceinline__ long cache_row(long page, int h, int place, int Hkv, int page_shift) {
  return ((page * Hkv + h) << page_shift) + place;
}

// The maximum over the LPR lanes (a power of two) of a row, in each of them.
template <int LPR>
__device__ __forceinline__ float row_max(float v) {
  v = fmaxf(v, dpp_mov<DPP_QUAD_1032>(v));
  v = fmaxf(v, dpp_mov<DPP_QUAD_2301>(v));
  if (LPR > 4) v = fmaxf(v, dpp_mov<DPP_ROW_HALF_MIRROR>(v));
  if (LPR > 8) v = fmaxf(v, dpp_mov<DPP_ROW_MIRROR>(v));
  if (LPR > 16) v = fmaxf(v, __shfl_xor(v, 16));
  return v;
}

// LPR lanes a row (those behind its end idle), E elements each, K and V of a row together:
// four 16-byte loads a thread are under way at once.  12288 tokens of 16 x 128, bf16 to e4m3,
// 151 MB: 32.4 us = 4.7 TB/s, the card's copy rate (K and V apart, 8 elements a lane: 38); to
// bf16, 201 MB: 41.1 us = 4.9 TB/s; 32 tokens of 4 x 128: 3.7 us, a launch.
template <typename T, bool Q, int E, int LPR>
__global__ __launch_bounds__(256) void cache_write_kernel(const WriteParams p) {
  typedef typename Elem<T>::v8 v8;
  const int c = threadIdx.x % LPR;
  const unsigned r = blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  if (r >= p.rows) return;
  const unsigned t = r / (unsigned)p.Hkv, h = r - t * p.Hkv;
  const bool in = c * E < p.hd;
  v8 x[2][E / 8];
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    const T* src = static_cast<const T*>(v ? p.v : p.k) + t * (v ? p.vst : p.kst) + h * (v ? p.vsh : p.ksh) + c * E;
#pragma unroll
    for (int i = 0; i < E / 8; ++i) {
      x[v][i] = v8{};
      if (in) x[v][i] = __builtin_nontemporal_load(reinterpret_cast<const v8*>(src) + i);
    }
  }
  const int slot = p.slots[t];
  if (slot < 0 || slot >= p.n_slots) return;
  const long row = cache_row(slot >> p.page_shift, h, slot & ((1 << p.page_shift) - 1), p.Hkv, p.page_shift);
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    void* const dst = v ? p.vp : p.kp;
    if constexpr (!Q) {
#pragma unroll
      for (int i = 0; i < E / 8; ++i)
        if (in) *(reinterpret_cast<v8*>(static_cast<T*>(dst) + row * p.hd + c * E) + i) = x[v][i];
    } else {
      // values that four significant bits would carry past the type's range are held at its top; NaN stays
      float f[E], amax = 0.f;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        f[j] = (float)x[v][j / 8][j % 8];
        f[j] = f[j] > Elem<T>::top ? Elem<T>::top : f[j] < -Elem<T>::top ? -Elem<T>::top : f[j];
        amax = fmaxf(amax, fabsf(f[j]));
      }
      const unsigned bits = __builtin_bit_cast(unsigned, row_max<LPR>(amax));
      const int e = max(1, (int)(bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000 ? 1 : 0));
      const float inv = __builtin_bit_cast(float, (unsigned)(254 - e) << 23);
      typedef unsigned codes __attribute__((ext_vector_type(E / 4)));
      codes w;
#pragma unroll
      for (int j = 0; j < E; j += 4) {
        const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[j] * inv, f[j + 1] * inv, 0, false);
        w[j / 4] = __builtin_amdgcn_cvt_pk_fp8_f32(f[j + 2] * inv, f[j + 3] * inv, lo, true);
      }
      if (in) *reinterpret_cast<codes*>(static_cast<uint8_t*>(dst) + row * p.hd + c * E) = w;
      if (c == 0) (v ? p.vs : p.ks)[row] = (uint8_t)e;
    }
  }
}

struct ReadParams {
  const void *kp, *vp;
  const uint8_t *ks, *vs;
  void *k, *v;
  const int *table, *cu;
  int B, table_w, tokens, Hkv, hd, page_shift, n_pages;
  int pieces, lanes;   // a token's pieces of 8 elements; threads side by side on them (a power of two up to 256)
};

constexpr int READ_TOK = 16;   // tokens per workgroup

// Token t's sequence: the last b with cu[b] <= t (cu[0] is taken as 0); -1 behind the last sequence.
__device__ __forceinline__ int sequence_of(const int* cu, int B, int t) {
  if (t >= cu[B]) return -1;
  int lo = 0, hi = B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Eight elements a thread and token (16 leave every other 16 bytes to a second store: 203 against
// 174 us below).  NT: past the caches, for an output that the L2s do not hold (8 x 4 MiB): 71822
// tokens of 16 x 128 from e4m3, 885 MB in all, 180 -> 174 us = 5.1 TB/s; from f16, 1177 MB,
// 248 us = 4.8 TB/s.
template <typename T, bool Q, bool NT>
__global__ __launch_bounds__(256) void cache_read_kernel(const ReadParams p) {
  __shared__ long base[READ_TOK];   // page * Hkv * page size + place; -1: no such token
  const int t0 = blockIdx.x * READ_TOK;
  const bool isv = blockIdx.y;
  if (threadIdx.x < READ_TOK) {
    const int t = t0 + threadIdx.x;
    long at = -1;
    if (t < p.tokens) {
      const int b = sequence_of(p.cu, p.B, t);
      if (b >= 0) {
        const int i = t - p.cu[b];
        const int pi = i >> p.page_shift;
        if (i >= 0 && pi < p.table_w) {
          const long page = min(max(p.table[(long)b * p.table_w + pi], 0), p.n_pages - 1);
          at = cache_row(page, 0, i & ((1 << p.page_shift) - 1), p.Hkv, p.page_shift);
        }
      }
    }
    base[threadIdx.x] = at;
  }
  __syncthreads();
  typedef typename Elem<T>::v8 v8;
  const int ch = p.hd / 8;
  for (int r = threadIdx.x & (p.lanes - 1); r < p.pieces; r += p.lanes) {
    const int h = r / ch, c = r - h * ch;
#pragma unroll 4
    for (int t = threadIdx.x / p.lanes; t < READ_TOK; t += 256 / p.lanes) {
      if (base[t] < 0) continue;
      const long row = base[t] + ((long)h << p.page_shift);
      v8 y;
      if constexpr (!Q) {
        y = *reinterpret_cast<const v8*>(static_cast<const T*>(isv ? p.vp : p.kp) + row * p.hd + c * 8);
      } else {
        const u32x2_t w = *reinterpret_cast<const u32x2_t*>(static_cast<const uint8_t*>(isv ? p.vp : p.kp) + row * p.hd + c * 8);
        // 2^(byte - 127); of the type's ends, 0 is the f32 subnormal 2^-127 and 255 is NaN
        const unsigned byte = (isv ? p.vs : p.ks)[row];
        const float s = __builtin_bit_cast(float, byte << 23 | (((byte + 1) & 255) < 2 ? 0x400000u : 0u));
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int u = w[j];
          const float2_t a = __builtin_amdgcn_cvt_pk_f32_fp8(u, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(u, true);
          y[4 * j] = (T)(a[0] * s);
          y[4 * j + 1] = (T)(a[1] * s);
          y[4 * j + 2] = (T)(b[0] * s);
          y[4 * j + 3] = (T)(b[1] * s);
        }
      }
      v8* to = reinterpret_cast<v8*>(static_cast<T*>(isv ? p.v : p.k) + ((long)(t0 + t) * p.Hkv + h) * p.hd + c * 8);
      if (NT) __builtin_nontemporal_store(y, to);
      else *to = y;
    }
  }
}

template <typename T, bool Q>
void write_t(const WriteParams& p, hipStream_t s) {
  auto go = [&](auto kernel, int lpr) { CK_LAUNCH(kernel, dim3(ceil_div(p.rows, 256 / lpr)), dim3(256), 0, s, p); };
  if (p.hd % 16) go(cache_write_kernel<T, Q, 8, 32>, 32);
  else if (p.hd <= 64) go(cache_write_kernel<T, Q, 16, 4>, 4);
  else if (p.hd <= 128) go(cache_write_kernel<T, Q, 16, 8>, 8);
  else go(cache_write_kernel<T, Q, 16, 16>, 16);
}

template <typename T>
void read_t(const ReadParams& p, bool q, bool large, hipStream_t s) {
  auto go = [&](auto kernel) { CK_LAUNCH(kernel, dim3(ceil_div(p.tokens, READ_TOK), 2), dim3(256), 0, s, p); };
  if (large) q ? go(cache_read_kernel<T, true, true>) : go(cache_read_kernel<T, false, true>);
  else q ? go(cache_read_kernel<T, true, false>) : go(cache_read_kernel<T, false, false>);
}

}  // namespace

int page_shift(int page) {
  int s = 0;
  while ((1 << s) < page) ++s;
  return s;
}

void check_pages(const char* what, const PagedCache& c) {
  const std::string w(what);
  CK_REQUIRE(c.k && c.v, w + ": null cache");
  CK_REQUIRE(c.dtype == DT_F16 || c.dtype == DT_BF16 || c.dtype == DT_E4M3, w + ": the cache must be f16, bf16 or e4m3");
  CK_REQUIRE(c.n_pages > 0 && c.n_kv > 0 && c.n_kv <= 1024, w + ": pages and K/V heads (up to 1024) must be positive");
  CK_REQUIRE(c.page >= 16 && c.page <= 1024 && (c.page & (c.page - 1)) == 0,
             w + ": page size must be a power of two from 16 to 1024");
  CK_REQUIRE((long)c.n_pages * c.page < (1L << 31), w + ": the cache must have under 2^31 slots");
  CK_REQUIRE(c.head_dim > 0 && c.head_dim % 8 == 0 && c.head_dim <= 256, w + ": head_dim must be a multiple of 8 up to 256");
  CK_REQUIRE(c.dtype != DT_E4M3 || (c.k_scale && c.v_scale), w + ": an e4m3 cache needs its scales");
  CK_REQUIRE(((reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v)) & 15) == 0,
             w + ": pages must be 16-byte aligned");
}

void launch_cache_write(const void* k, const void* v, const PagedCache& c, const int* slots, int T, long kst, long ksh,
                        long vst, long vsh, int dtype, hipStream_t s) {
  CK_REQUIRE(dtype == DT_F16 || dtype == DT_BF16, "cache_write: rows must be f16 or bf16");
  check_pages("cache_write", c);
  CK_REQUIRE(c.dtype == dtype || c.dtype == DT_E4M3, "cache_write: the cache must be of the rows' type or e4m3");
  // (a launch has under 2^32 threads, of which a row takes up to 32)
  CK_REQUIRE(T >= 0 && (long)T * c.n_kv < (1L << 27), "cache_write: under 2^27 rows");
  if (T == 0) return;
  CK_REQUIRE(k && v && slots, "cache_write: null pointer");
  CK_REQUIRE(((kst | ksh | vst | vsh) & 7) == 0 && ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0,
             "cache_write: rows must be 16-byte aligned");
  WriteParams p{};
  p.k = k;
  p.v = v;
  p.kp = c.k;
  p.vp = c.v;
  p.ks = c.k_scale;
  p.vs = c.v_scale;
  p.slots = slots;
  p.kst = kst;
  p.ksh = ksh;
  p.vst = vst;
  p.vsh = vsh;
  p.T = T;
  p.Hkv = c.n_kv;
  p.hd = c.head_dim;
  p.page_shift = page_shift(c.page);
  p.n_slots = (long)c.n_pages * c.page;
  p.rows = (unsigned)T * c.n_kv;
  if (dtype == DT_F16) {
    if (c.dtype == DT_E4M3) write_t<half_t, true>(p, s);
    else write_t<half_t, false>(p, s);
  } else {
    if (c.dtype == DT_E4M3) write_t<bf16_t, true>(p, s);
    else write_t<bf16_t, false>(p, s);
  }
  CK_LAUNCHED("cache_write");
}

void launch_cache_read(const PagedCache& c, const int* table, int table_w, const int* cu, int B, int tokens, void* k,
                       void* v, int dtype, hipStream_t s) {
  CK_REQUIRE(dtype == DT_F16 || dtype == DT_BF16, "cache_read: rows must be f16 or bf16");
  check_pages("cache_read", c);
  CK_REQUIRE(c.dtype == dtype || c.dtype == DT_E4M3, "cache_read: the cache must be of the rows' type or e4m3");
  CK_REQUIRE(tokens >= 0 && B >= 0 && table_w >= 0 && tokens < (1 << 28) && (long)tokens * c.n_kv < (1L << 31),
             "cache_read: under 2^28 tokens and 2^31 rows");
  if (tokens == 0 || B == 0 || table_w == 0) return;
  CK_REQUIRE(table && cu && k && v, "cache_read: null pointer");
  CK_REQUIRE(((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0, "cache_read: rows must be 16-byte aligned");
  ReadParams p{};
  p.kp = c.k;
  p.vp = c.v;
  p.ks = c.k_scale;
  p.vs = c.v_scale;
  p.k = k;
  p.v = v;
  p.table = table;
  p.cu = cu;
  p.B = B;
  p.table_w = table_w;
  p.tokens = tokens;
  p.Hkv = c.n_kv;
  p.hd = c.head_dim;
  p.page_shift = page_shift(c.page);
  p.n_pages = c.n_pages;
  p.pieces = c.n_kv * c.head_dim / 8;
  p.lanes = 1;
  while (p.lanes < 256 && p.lanes < p.pieces) p.lanes *= 2;
  const bool large = (long)tokens * c.n_kv * c.head_dim * 2 > (32L << 20);   // each of K and V
  if (dtype == DT_F16) read_t<half_t>(p, c.dtype == DT_E4M3, large, s);
  else read_t<bf16_t>(p, c.dtype == DT_E4M3, large, s);
  CK_LAUNCHED("cache_read");
}

}  // namespace ck
