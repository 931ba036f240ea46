// Attention of packed sequences of queries over their K/V rows, contiguous or in a paged
// cache; causal or full; query heads in groups that share a K/V head.
//
//   s_ij = scale * q_i . k_j,   o_i = sum_j softmax(s_i)_j v_j
// over the keys j < kv_len that query i may see (causal: j <= i + kv_len - q_len, the queries
// being the last places of their sequence).  A query that sees no key gets zeros.
//
// Rows.  The queries of the G heads that share a K/V head are the rows of one product:
// row r of a sequence is query r / G of head g = r % G, so that K and V pass once for all
// of them.  A wave owns 32 rows, a workgroup 128, over tiles of 64 keys in LDS:
//   S^T = K Q^T (v_mfma 32x32x16, A = 32 keys, B = 32 rows): lane l holds row l % 32 and
//     the keys 8 (i / 4) + 4 (l / 32) + i % 4, i < 16, of a block of 32;
//   the softmax needs the other half of the wave for its maximum and sum only;
//   O^T = V^T P^T: the lane's own exponentials, rounded to the element type, are the B operand
//     as they stand; V^T's operand takes its keys in the same order through transposed LDS reads.
// The running maximum and sum and O are f32.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "elem16.h"
#include "kernels.h"

namespace ck {
namespace {

constexpr int AT_KEYS = 64;   // keys per tile
constexpr float AT_LOG2E = 1.4426950408889634f;

// where a sequence's K/V rows are
enum KvKind { KV_ROWS = 0, KV_PAGES = 1, KV_E4M3 = 2 };

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
};

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

// ---- which part of the work a workgroup does -------------------------------------------
// A sequence's rows make tiles of BM; a tile's keys make chunks of `c` blocks of 64, so that
// about `target` items of equal length per K/V head fill the card whatever the lengths are:
// every workgroup adds up the lengths (64 sequences a step) and finds its own item.  The
// items of a tile with one chunk write the output, the others partial sums, item by item.
struct Item {
  int b, tile, chunk, nch, c, base;   // base: the tile's first item
  Seq s;
};

template <int KV, int BM>
__device__ __forceinline__ int tiles_of(const Seq& s, int G) {
  return (int)(((long)s.nq * G + BM - 1) / BM);
}
__device__ __forceinline__ int blocks_of(int keys) { return (keys + AT_KEYS - 1) / AT_KEYS; }

// index counts items, or tiles where TILES.  False: there are not so many.
template <int KV, int BM, bool TILES>
__device__ __forceinline__ bool find_item(const AttendParams& p, int index, Item& it) {
  const int lane = threadIdx.x & 63;
  int c = 1 << 30;
  if (p.target) {
    long work = 0;
    int tiles = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64)
      if (b0 + lane < p.B) {
        const Seq s = sequence<KV>(p, b0 + lane);
        const int n = tiles_of<KV, BM>(s, p.G);
        tiles += n;
        work += (long)n * blocks_of(s.nk);
      }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      tiles += __shfl_xor(tiles, o);
      work += __shfl_xor(work, o);
    }
    // each tile adds up to one item that is not full
    const int full = max(p.target - tiles, (p.target + 1) >> 1);
    c = max(p.min_blocks, (int)min((work + full - 1) / full, 1L << 30));
  }
  int base = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    int tiles = 0, nch = 1;
    Seq s{};
    if (b0 + lane < p.B) {
      s = sequence<KV>(p, b0 + lane);
      tiles = tiles_of<KV, BM>(s, p.G);
      nch = max(1, (blocks_of(s.nk) + c - 1) / c);
    }
    int items = tiles * nch, units = TILES ? tiles : items, su = units, si = items;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(su, o), z = __shfl_up(si, o);
      if (lane >= o) su += y, si += z;
    }
    const unsigned long long m = __ballot(su > index);
    if (m) {
      const int w = __ffsll(m) - 1;
      const int local = __builtin_amdgcn_readlane(index - (su - units), w);
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
      return true;
    }
    index -= __builtin_amdgcn_readlane(su, 63);
    base += __builtin_amdgcn_readlane(si, 63);
  }
  return false;
}

// keys that query tok of a sequence sees: all below this
__device__ __forceinline__ int keys_of(const AttendParams& p, const Seq& s, int tok) {
  return p.causal ? min(s.nk, max(0, tok + 1 + s.nk - s.nq)) : s.nk;
}

// ---- LDS tiles --------------------------------------------------------------------------
// Element offsets of 16-byte chunk c of a row: K's fragments are one chunk of 16 consecutive
// rows, V's four chunks of 4 consecutive rows; both hit every bank once this way.
template <int HD>
__device__ __forceinline__ int k_at(int key, int c) {
  return HD == 128 ? key * HD + ((c ^ (key & 15)) << 3) : key * HD + ((c ^ ((key >> 1) & 7)) << 3);
}
template <int HD>
__device__ __forceinline__ int v_at(int key, int c) {
  return HD == 128 ? key * HD + ((c ^ ((key & 3) << 2)) << 3) : key * HD + ((c ^ ((key & 2) << 1)) << 3);
}

// KEYS rows of K and V on their way through the registers of NT threads: load() sends for
// them, store() leaves them (e4m3: as values of T) in LDS.  Places behind the last key
// repeat it.  A wave's rows of one load lie in one group of 16, so on one page.
template <typename T, int HD, int KV, int KEYS, int NT>
struct Stage {
  typedef typename Elem<T>::v2 v2;
  typedef typename Elem<T>::v8 v8;
  static constexpr int EPL = KV == KV_E4M3 && KEYS * HD / 16 >= NT ? 16 : 8;   // elements per load
  static constexpr int CPR = HD / EPL, N = KEYS * CPR / NT, RPL = NT / CPR;
  static constexpr int BPL = KV == KV_E4M3 ? EPL : 16;                         // bytes per load
  typedef std::conditional_t<BPL == 16, u32x4_t, u32x2_t> raw;
  static_assert(N * NT == KEYS * CPR && (RPL >= 16 || 16 % RPL == 0), "tile");
  raw k[N], v[N];
  unsigned ks[N], vs[N];
  int page[N];

  // the pages of the keys from key0 on
  __device__ __forceinline__ void pages(const AttendParams& p, const Item& it, int key0, int wave) {
    if constexpr (KV != KV_ROWS) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int key = min(key0 + ((i * RPL + wave * (64 / CPR)) & ~15), it.s.nk - 1);
        page[i] = p.table[(long)it.b * p.table_w + (key >> p.page_shift)];
      }
    }
  }
  __device__ __forceinline__ void load(const AttendParams& p, const Item& it, int hk, int key0, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int key = min(key0 + i * RPL + tid / CPR, it.s.nk - 1), c = tid % CPR;
      if constexpr (KV == KV_ROWS) {
        k[i] = *reinterpret_cast<const raw*>(static_cast<const T*>(p.k) + (long)(it.s.k0 + key) * p.k_st + (long)hk * p.k_sh + c * 8);
        v[i] = *reinterpret_cast<const raw*>(static_cast<const T*>(p.v) + (long)(it.s.k0 + key) * p.v_st + (long)hk * p.v_sh + c * 8);
      } else {
        const long pg = min(max(page[i], 0), p.n_pages - 1);
        const long at = ((pg * p.Hkv + hk) << p.page_shift) + (key & ((1 << p.page_shift) - 1));
        const long off = at * (HD / EPL * BPL) + c * BPL;
        k[i] = *reinterpret_cast<const raw*>(static_cast<const char*>(p.k) + off);
        v[i] = *reinterpret_cast<const raw*>(static_cast<const char*>(p.v) + off);
        if constexpr (KV == KV_E4M3) {
          ks[i] = p.ks[at];
          vs[i] = p.vs[at];
        }
      }
    }
  }
  // load() straight into LDS, as store() would leave it: a wave's 64 pieces of 16 bytes land side by
  // side, so each lane fetches the chunk that belongs in its place
  __device__ __forceinline__ void dma(const AttendParams& p, const Item& it, int hk, int key0, int tid, int wave, T* kt, T* vt) const {
    typedef const __attribute__((address_space(1))) void* src_t;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int row = i * RPL + tid / CPR, pos = tid % CPR, key = min(key0 + row, it.s.nk - 1);
      const int ck = (k_at<HD>(row, pos) >> 3) % CPR, cv = (v_at<HD>(row, pos) >> 3) % CPR;
      const T *kb, *vb;
      if constexpr (KV == KV_ROWS) {
        kb = static_cast<const T*>(p.k) + (long)(it.s.k0 + key) * p.k_st + (long)hk * p.k_sh;
        vb = static_cast<const T*>(p.v) + (long)(it.s.k0 + key) * p.v_st + (long)hk * p.v_sh;
      } else {
        const long pg = min(max(page[i], 0), p.n_pages - 1);
        const long at = ((pg * p.Hkv + hk) << p.page_shift) + (key & ((1 << p.page_shift) - 1));
        kb = static_cast<const T*>(p.k) + at * HD;
        vb = static_cast<const T*>(p.v) + at * HD;
      }
      __builtin_amdgcn_global_load_lds((src_t)(kb + ck * 8), (lds_ptr_t)(kt + (i * NT + wave * 64) * 8), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((src_t)(vb + cv * 8), (lds_ptr_t)(vt + (i * NT + wave * 64) * 8), 16, 0, 0);
    }
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
  __device__ __forceinline__ void store(T* kt, T* vt, int tid) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int key = i * RPL + tid / CPR, c = tid % CPR;
      if constexpr (KV != KV_E4M3) {
        *reinterpret_cast<raw*>(kt + k_at<HD>(key, c)) = k[i];
        *reinterpret_cast<raw*>(vt + v_at<HD>(key, c)) = v[i];
      } else {
        const float fk = __builtin_bit_cast(float, ks[i] << 23), fv = __builtin_bit_cast(float, vs[i] << 23);
#pragma unroll
        for (int j = 0; j < EPL / 8; ++j) {
          const int cc = c * (EPL / 8) + j;
          *reinterpret_cast<v8*>(kt + k_at<HD>(key, cc)) = values(k[i][2 * j], k[i][2 * j + 1], fk);
          *reinterpret_cast<v8*>(vt + v_at<HD>(key, cc)) = values(v[i][2 * j], v[i][2 * j + 1], fv);
        }
      }
    }
  }
};

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

// ---- 32 rows of a wave ------------------------------------------------------------------
template <typename T, int HD>
struct Rows {
  typedef typename Elem<T>::v2 v2;
  typedef typename Elem<T>::v4 v4;
  typedef typename Elem<T>::v8 v8;
  static constexpr int KS = HD / 16, CT = HD / 32;
  v8 qf[KS];
  float16_t o[CT];
  float m, l;         // running maximum of the raw scores; this half's part of the sum
  int lim, tok, g;    // keys that the row sees; its query and head within the group (tok < 0: no row)

  __device__ __forceinline__ void begin(const AttendParams& p, const Item& it, int hk, int row, int lane) {
    tok = row / p.G;
    g = row - tok * p.G;
    const bool valid = tok < it.s.nq;
    lim = valid ? keys_of(p, it.s, tok) : 0;
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

  // NB blocks of 32 keys from key0 on, in LDS.  part: some row may not see all of them.
  template <int NB>
  __device__ __forceinline__ void step(const T* kt, const T* vt, int key0, bool part, float c, int lane) {
    const int half = lane >> 5, r32 = lane & 31;
    float16_t s[NB];
#pragma unroll
    for (int kb = 0; kb < NB; ++kb) {
      s[kb] = float16_t{};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const v8 kf = *reinterpret_cast<const v8*>(kt + k_at<HD>(kb * 32 + r32, ks * 2 + half));
        s[kb] = Elem<T>::mfma32(kf, qf[ks], s[kb]);
      }
    }
    if (part) {
      const int left = lim - key0 - 4 * half;
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (kb * 32 + 8 * (i >> 2) + (i & 3) >= left) s[kb][i] = -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kb][i]);
    mx = half_max(mx);
    // The maximum that the exponents are taken from may lag behind the true one by 2^8: O and l
    // are rescaled only when some row's has moved further, so hardly ever after the first tiles.
    if (__any((mx - m) * c > 8.0f || (m == -INFINITY && mx > -INFINITY))) {
      const float mn = fmaxf(m, mx), f = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * c);
      m = mn;
      l *= f;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) o[ct] *= f;
    }
    const float mc = m == -INFINITY ? 0.f : m * c;
    v8 pf[2 * NB];
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][i], c, -mc));
        const float d = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][i + 1], c, -mc));
        // the sum is that of the rounded weights, so their rounding cancels where few keys rule
        const v2 u = pack2<T>(a, d);
        l = Elem<T>::add2(u, l);
        pf[kb * 2 + (i >> 3)][i & 7] = u[0];
        pf[kb * 2 + (i >> 3)][(i & 7) + 1] = u[1];
      }
    // O^T += V^T P^T
    const int va = 4 * half + ((lane >> 2) & 3), vd = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
    for (int kk = 0; kk < 2 * NB; ++kk)
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        v8 vf;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int key = kk * 16 + e * 8 + va, d = ct * 32 + vd;
          typedef short s16x4 __attribute__((ext_vector_type(4)));
          const v4 x = __builtin_bit_cast(v4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                  (__attribute__((address_space(3))) s16x4*)(vt + v_at<HD>(key, d >> 3) + (d & 7))));
#pragma unroll
          for (int j = 0; j < 4; ++j) vf[e * 4 + j] = x[j];
        }
        o[ct] = Elem<T>::mfma32(vf, pf[kk], o[ct]);
      }
  }
  // bad[k][d]: the first key whose V is +inf, -inf or NaN (k = 0, 1, 2) in feature d
  __device__ __forceinline__ void add_odd(const int (*bad)[HD], int lane) {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int d = ct * 32 + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3);
        float add = bad[0][d] < lim ? INFINITY : 0.f;
        add += bad[1][d] < lim ? -INFINITY : 0.f;
        add += bad[2][d] < lim ? NAN : 0.f;
        asm volatile("" : "+v"(add)::"memory");   // one element at a time: a rare path, and no registers for it
        o[ct][i] += add;
      }
  }
  __device__ __forceinline__ float sum() const { return l + __shfl_xor(l, 32); }
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

// Where the partial sums of an item's rows are: O f32 [items][rows][HD], then (maximum in the
// log2 domain, sum) [items][rows][2].
template <int HD>
__device__ __forceinline__ float* part_o(const AttendParams& p, long row) { return p.ws + row * HD; }
template <int HD>
__device__ __forceinline__ float2_t* part_ml(const AttendParams& p, long row) {
  return reinterpret_cast<float2_t*>(p.ws + p.part_rows * HD) + row;
}

// ---- many rows: NW waves of 32 rows over the same keys -----------------------------------
// Tiles of 64 keys in two buffers: the next one is under way (f16, bf16: straight to LDS;
// e4m3: through registers, where it is turned into values) while this one is used.
template <typename T, int HD, int KV, int NW>
__global__ __launch_bounds__(64 * NW, 2) void attend_tile_kernel(const AttendParams p) {
  constexpr int BM = 32 * NW, TILE = AT_KEYS * HD, NT = 64 * NW;
  constexpr bool DMA = KV != KV_E4M3;
  __shared__ __attribute__((aligned(1024))) T kt[2][TILE], vt[2][TILE];
  __shared__ int bad[3][HD], odd;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hk = blockIdx.x % p.Hkv, index = blockIdx.x / p.Hkv;
  Item it;
  if (!find_item<KV, BM, false>(p, index, it)) return;
  const int tile = tiles_of<KV, BM>(it.s, p.G) - 1 - it.tile;   // the longest first
  // the keys of the tile's first and last rows, and of this chunk
  const int klo = keys_of(p, it.s, tile * BM / p.G);
  const int khi = keys_of(p, it.s, min(it.s.nq - 1, (tile * BM + BM - 1) / p.G));
  const int kbeg = it.nch > 1 ? it.chunk * it.c * AT_KEYS : 0;
  const int kend = it.nch > 1 ? min(khi, kbeg + it.c * AT_KEYS) : khi;

  Stage<T, HD, KV, AT_KEYS, NT> st;
  if (tid == 0) odd = 0;
  if (kbeg < kend) {
    st.pages(p, it, kbeg, wave);
    if constexpr (DMA) st.dma(p, it, hk, kbeg, tid, wave, kt[0], vt[0]);
    else st.load(p, it, hk, kbeg, tid);
    st.pages(p, it, kbeg + AT_KEYS, wave);
  }
  Rows<T, HD> r;
  r.begin(p, it, hk, tile * BM + wave * 32 + (lane & 31), lane);
  // Q has arrived before the loop, whose waits would otherwise count its loads every time
  r.arrived();
  if (!DMA && kbeg < kend) st.store(kt[0], vt[0], tid);
  for (int key0 = kbeg, cur = 0; key0 < kend; key0 += AT_KEYS, cur ^= 1) {
    const bool more = key0 + AT_KEYS < kend;
    __syncthreads();   // this tile is there, and the other buffer is free
    if (more) {
      if constexpr (DMA) st.dma(p, it, hk, key0 + AT_KEYS, tid, wave, kt[cur ^ 1], vt[cur ^ 1]);
      else st.load(p, it, hk, key0 + AT_KEYS, tid);
      st.pages(p, it, key0 + 2 * AT_KEYS, wave);
    }
    // A tile that some row sees in part: an infinity or NaN of V must not reach that row.
    const bool part = key0 + AT_KEYS > klo;
    bool fix = false;
    if (part) {
      if (any_odd<T, TILE, NT>(vt[cur], tid)) odd = 1;
      __syncthreads();
      fix = odd;
      if (fix) {
        for (int i = tid; i < 3 * HD; i += NT) (&bad[0][0])[i] = 0x7FFFFFFF;
        __syncthreads();
        take_out_odd<T, HD, AT_KEYS, NT>(vt[cur], bad, key0, tid);
        __syncthreads();
      }
    }
    r.template step<2>(kt[cur], vt[cur], key0, part, p.scale_log2e, lane);
    if (fix) {
      r.add_odd(bad, lane);
      __syncthreads();
      if (tid == 0) odd = 0;
    }
    if (!DMA && more) st.store(kt[cur ^ 1], vt[cur ^ 1], tid);
  }

  if (it.nch == 1) {
    r.finish(p, it, hk, lane);
    return;
  }
  const float t = r.sum();
  if (r.tok < 0) return;
  const long row = ((long)(it.base + it.chunk) * p.Hkv + hk) * BM + wave * 32 + (lane & 31);
  if (lane < 32) *part_ml<HD>(p, row) = float2_t{r.m * p.scale_log2e, t};
  if (kbeg >= kend) return;
  float* o = part_o<HD>(p, row) + 4 * (lane >> 5);
#pragma unroll
  for (int ct = 0; ct < HD / 32; ++ct)
#pragma unroll
    for (int i = 0; i < 16; i += 4)
      *reinterpret_cast<float4_t*>(o + ct * 32 + 2 * i) = float4_t{r.o[ct][i], r.o[ct][i + 1], r.o[ct][i + 2], r.o[ct][i + 3]};
}

// ---- few rows: 32 of them, the keys over the waves ----------------------------------------
// Every wave streams its own blocks of 32 keys (w, w + 4, ...) through LDS of its own; nothing
// waits for another wave until the end, where the waves' sums are joined.
constexpr int FEW_WAVES = 4;

template <typename T, int HD, int KV>
__global__ __launch_bounds__(64 * FEW_WAVES, 2) void attend_few_kernel(const AttendParams p) {
  constexpr int BM = 32, KEYS = 32, TILE = KEYS * HD, NW = FEW_WAVES;
  __shared__ __attribute__((aligned(16))) T lds[NW][2 * TILE];   // at the end: O f32 [NW][32][HD]
  __shared__ float2_t ml[NW][BM];
  __shared__ int bad[NW][3][HD];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hk = blockIdx.x % p.Hkv, index = blockIdx.x / p.Hkv;
  Item it;
  if (!find_item<KV, BM, false>(p, index, it)) return;
  Rows<T, HD> r;
  r.begin(p, it, hk, it.tile * BM + (lane & 31), lane);
  const int klo = keys_of(p, it.s, it.tile * BM / p.G);
  const int khi = keys_of(p, it.s, min(it.s.nq - 1, (it.tile * BM + BM - 1) / p.G));
  const int kbeg = it.nch > 1 ? it.chunk * it.c * AT_KEYS : 0;
  const int kend = it.nch > 1 ? min(khi, kbeg + it.c * AT_KEYS) : khi;

  r.arrived();
  Stage<T, HD, KV, KEYS, 64> st;
  T* const kt = lds[wave];
  T* const vt = kt + TILE;
  int key0 = kbeg + wave * KEYS;
  if (key0 < kend) {
    st.pages(p, it, key0, 0);
    st.load(p, it, hk, key0, lane);
    st.pages(p, it, key0 + NW * KEYS, 0);
  }
  for (; key0 < kend; key0 += NW * KEYS) {
    const bool part = key0 + KEYS > klo;
    wave_order();
    st.store(kt, vt, lane);
    if (key0 + NW * KEYS < kend) {
      st.load(p, it, hk, key0 + NW * KEYS, lane);
      st.pages(p, it, key0 + 2 * NW * KEYS, 0);
    }
    wave_order();
    const bool fix = part && __any(any_odd<T, TILE, 64>(vt, lane));
    if (fix) {
      for (int i = lane; i < 3 * HD; i += 64) (&bad[wave][0][0])[i] = 0x7FFFFFFF;
      wave_order();
      take_out_odd<T, HD, KEYS, 64>(vt, bad[wave], key0, lane);
      wave_order();
    }
    r.template step<1>(kt, vt, key0, part, p.scale_log2e, lane);
    if (fix) r.add_odd(bad[wave], lane);
  }

  // ---- join the waves ----
  __syncthreads();
  const int rows = min(BM, it.s.nq * p.G - it.tile * BM);
  float* const ob = reinterpret_cast<float*>(&lds[0][0]);
  const float t = r.sum();
  if (lane < 32) ml[wave][lane] = float2_t{r.m * p.scale_log2e, t};
  if ((lane & 31) < rows) {
    // 16-byte chunk c of row q at c ^ (q & 7): 8 rows of a chunk in 8 different places
    float* o = ob + (wave * BM + (lane & 31)) * HD;
#pragma unroll
    for (int ct = 0; ct < HD / 32; ++ct)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *reinterpret_cast<float4_t*>(o + (((ct * 8 + (i >> 1) + (lane >> 5)) ^ (lane & 7)) << 2)) =
            float4_t{r.o[ct][i], r.o[ct][i + 1], r.o[ct][i + 2], r.o[ct][i + 3]};
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
      if (x[0] == -INFINITY) continue;   // saw no key
      const float f = __builtin_amdgcn_exp2f(x[0] - M);
      sum += f * x[1];
      a += f * *reinterpret_cast<const float4_t*>(ob + (w * BM + q) * HD + ((c ^ (q & 7)) << 2));
    }
    if (it.nch == 1) {
      const float rs = sum == 0.f ? 0.f : 1.0f / sum;
      const int row = it.tile * BM + q, tok = row / p.G;
      T* out = static_cast<T*>(p.out) + (long)(it.s.q0 + tok) * p.o_st + (long)(hk * p.G + row - tok * p.G) * p.o_sh + c * 4;
      const auto x = pack2<T>(a[0] * rs, a[1] * rs), y = pack2<T>(a[2] * rs, a[3] * rs);
      *reinterpret_cast<typename Elem<T>::v4*>(out) = typename Elem<T>::v4{x[0], x[1], y[0], y[1]};
    } else {
      const long row = ((long)(it.base + it.chunk) * p.Hkv + hk) * BM + q;
      *reinterpret_cast<float4_t*>(part_o<HD>(p, row) + c * 4) = a;
      if (c == 0) *part_ml<HD>(p, row) = float2_t{M, sum};
    }
  }
}

// ---- the chunks of a tile joined ----------------------------------------------------------
// HD / 4 lanes a row, RP rows and CG groups of chunks a workgroup of 256.
template <typename T, int HD, int KV, int BM>
__global__ __launch_bounds__(256) void attend_join_kernel(const AttendParams p) {
  constexpr int LPR = HD / 4, CG = BM == 32 ? 256 / LPR : 1, RP = 256 / LPR / CG;
  __shared__ float4_t so[CG][LPR];
  __shared__ float2_t sm[CG];
  const int hk = blockIdx.x % p.Hkv, index = blockIdx.x / p.Hkv;
  Item it;
  // (offsets that do not ascend may name more rows than there are: what has no item has no sums)
  if (!find_item<KV, BM, true>(p, index, it) || it.nch == 1 || it.base + it.nch > p.items) return;
  const int c = threadIdx.x % LPR, cg = CG > 1 ? threadIdx.x / LPR : 0;
  const int q = blockIdx.y * RP + (CG > 1 ? 0 : threadIdx.x / LPR);
  const int tile = BM == 32 ? it.tile : tiles_of<KV, BM>(it.s, p.G) - 1 - it.tile;
  const bool in = (long)tile * BM + q < (long)it.s.nq * p.G;
  if (CG > 1 && !in) return;
  float M = -INFINITY, sum = 0.f;
  float4_t a = {0.f, 0.f, 0.f, 0.f};
  if (in) {
    const long row = ((long)it.base * p.Hkv + hk) * BM + q;
    for (int n = cg; n < it.nch; n += CG) {
      const float2_t x = *part_ml<HD>(p, row + (long)n * p.Hkv * BM);
      if (x[0] == -INFINITY) continue;   // saw no key, has no O
      const float4_t y = *reinterpret_cast<const float4_t*>(part_o<HD>(p, row + (long)n * p.Hkv * BM) + c * 4);
      const float m = fmaxf(M, x[0]), f = __builtin_amdgcn_exp2f(M - m), h = __builtin_amdgcn_exp2f(x[0] - m);
      M = m;
      sum = sum * f + x[1] * h;
      a = a * f + y * h;
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
      if (sm[w][0] == -INFINITY) continue;
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

// ---- host ---------------------------------------------------------------------------------
// The form of a call: rows per tile, items per K/V head to aim at (0: keys are not split).
struct Plan {
  int bm, target, min_blocks;
  long tiles, items;   // at most
};
Plan plan_of(int B, int Tq, long max_keys, int n_heads, int n_kv) {
  Plan pl{};
  const int G = n_heads / n_kv;
  const long rows = (long)Tq * G;
  pl.bm = rows <= 32L * B ? 32 : 128;
  pl.tiles = rows / pl.bm + B;       // sum of ceil(rows_b / bm) is at most this
  const long slots = 512;            // workgroups that run at once, two a CU
  const long blocks = (max_keys + AT_KEYS - 1) / AT_KEYS;
  pl.min_blocks = pl.bm == 32 ? 2 : 4;
  if (blocks > pl.min_blocks && (pl.bm == 32 || pl.tiles * n_kv < 2 * slots)) pl.target = (int)std::max(1L, slots / n_kv);
  pl.items = pl.tiles + pl.target;
  return pl;
}

template <typename T, int HD, int KV>
void launch_kv(const AttendParams& p, const Plan& pl, hipStream_t s) {
  const dim3 grid((unsigned)(pl.items * p.Hkv));
  if (pl.bm == 32) CK_LAUNCH((attend_few_kernel<T, HD, KV>), grid, dim3(64 * FEW_WAVES), 0, s, p);
  else CK_LAUNCH((attend_tile_kernel<T, HD, KV, 4>), grid, dim3(256), 0, s, p);
  if (!pl.target) return;
  const unsigned tiles = (unsigned)(pl.tiles * p.Hkv);
  if (pl.bm == 32) CK_LAUNCH((attend_join_kernel<T, HD, KV, 32>), dim3(tiles, 32), dim3(256), 0, s, p);
  else CK_LAUNCH((attend_join_kernel<T, HD, KV, 128>), dim3(tiles, 128 / (1024 / HD)), dim3(256), 0, s, p);
}
template <typename T, int HD>
void launch_hd(const AttendParams& p, int kv, const Plan& pl, hipStream_t s) {
  if (kv == KV_ROWS) launch_kv<T, HD, KV_ROWS>(p, pl, s);
  else if (kv == KV_PAGES) launch_kv<T, HD, KV_PAGES>(p, pl, s);
  else launch_kv<T, HD, KV_E4M3>(p, pl, s);
}

void launch_attend(const char* what, AttendParams& p, const AttendQuery& a, int kv, long max_keys, hipStream_t s) {
  const std::string w(what);
  CK_REQUIRE(a.dtype == DT_F16 || a.dtype == DT_BF16, w + ": q must be f16 or bf16");
  CK_REQUIRE(a.head_dim == 64 || a.head_dim == 128, w + ": head_dim must be 64 or 128");
  CK_REQUIRE(a.n_heads > 0 && p.Hkv > 0 && a.n_heads % p.Hkv == 0 && a.n_heads <= 1024,
             w + ": query heads (up to 1024) must be a multiple of the K/V heads");
  CK_REQUIRE(a.T >= 0 && a.B >= 0 && (long)a.T * a.n_heads < (1L << 31) && a.B < (1 << 20), w + ": bad sizes");
  CK_REQUIRE(a.scale > 0.f && a.scale < INFINITY, w + ": scale must be positive and finite");
  if (a.T == 0 || a.B == 0) return;
  CK_REQUIRE(a.q && a.out && a.cu_q && p.kv, w + ": null pointer");
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
  const Plan pl = plan_of(a.B, a.T, max_keys, a.n_heads, p.Hkv);
  CK_REQUIRE(pl.items * p.Hkv < (1L << 31), w + ": too many rows");
  if (pl.target) {
    const size_t need = attention_workspace(a.B, a.T, max_keys, a.n_heads, p.Hkv, a.head_dim);
    CK_REQUIRE(a.ws && a.ws_floats >= need, w + ": workspace too small (ck_attention_workspace)");
    CK_REQUIRE((reinterpret_cast<uintptr_t>(a.ws) & 15) == 0, w + ": workspace must be 16-byte aligned");
  }
  p.target = pl.target;
  p.min_blocks = pl.min_blocks;
  p.ws = a.ws;
  p.items = (int)pl.items;
  p.part_rows = pl.items * p.Hkv * pl.bm;
  if (a.dtype == DT_F16) {
    if (a.head_dim == 64) launch_hd<half_t, 64>(p, kv, pl, s);
    else launch_hd<half_t, 128>(p, kv, pl, s);
  } else {
    if (a.head_dim == 64) launch_hd<bf16_t, 64>(p, kv, pl, s);
    else launch_hd<bf16_t, 128>(p, kv, pl, s);
  }
  CK_LAUNCHED(what);
}

}  // namespace

size_t attention_workspace(int B, int Tq, long max_keys, int n_heads, int n_kv, int head_dim) {
  CK_REQUIRE(B >= 0 && Tq >= 0 && max_keys >= 0 && n_kv > 0 && n_heads > 0 && n_heads % n_kv == 0 && head_dim > 0,
             "attention_workspace: bad sizes");
  if (B == 0 || Tq == 0) return 0;
  const Plan pl = plan_of(B, Tq, max_keys, n_heads, n_kv);
  return pl.target ? (size_t)pl.items * n_kv * pl.bm * (head_dim + 2) : 0;
}

void launch_attention_varlen(const AttendQuery& a, const void* k, const void* v, long kst, long ksh, long vst, long vsh,
                             const int* cu_k, int Tk, int n_kv, hipStream_t s) {
  AttendParams p{};
  CK_REQUIRE(Tk >= 0 && n_kv > 0, "attention_varlen: bad sizes");
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
                (long)table_w * c.page, s);
}

}  // namespace ck
