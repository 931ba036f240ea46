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

template <typename T, int HD, int KV>
__global__ __launch_bounds__(256) void attend_kernel(const AttendParams p) {
  typedef typename Elem<T>::v2 v2;
  typedef typename Elem<T>::v4 v4;
  typedef typename Elem<T>::v8 v8;
  constexpr int CH = HD / 8, KS = HD / 16, CT = HD / 32, BM = 128;
  __shared__ __attribute__((aligned(16))) T kt[AT_KEYS * HD], vt[AT_KEYS * HD];
  __shared__ int bad[3][HD], any_bad;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, r32 = lane & 31;

  // ---- the workgroup's K/V head, sequence and row tile ----
  const int hk = blockIdx.x % p.Hkv;
  int t = blockIdx.x / p.Hkv, b = -1;
  Seq sq{};
  for (int b0 = 0; b0 < p.B && b < 0; b0 += 64) {
    int n = 0;
    Seq s{};
    if (b0 + lane < p.B) {
      s = sequence<KV>(p, b0 + lane);
      n = (int)(((long)s.nq * p.G + BM - 1) / BM);
    }
    int sum = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(sum, o);
      if (lane >= o) sum += y;
    }
    const int total = __shfl(sum, 63);
    if (t < total) {
      const int w = __ffsll((unsigned long long)__ballot(sum > t)) - 1;
      b = b0 + w;
      t -= __shfl(sum - n, w);
      sq.q0 = __shfl(s.q0, w);
      sq.nq = __shfl(s.nq, w);
      sq.k0 = __shfl(s.k0, w);
      sq.nk = __shfl(s.nk, w);
    } else {
      t -= total;
    }
  }
  if (b < 0) return;

  // ---- this lane's row ----
  const int row = t * BM + wave * 32 + r32;
  const int tok = row / p.G, g = row - tok * p.G;
  const bool valid = tok < sq.nq;
  const int lim = !valid ? 0 : p.causal ? min(sq.nk, max(0, tok + 1 + sq.nk - sq.nq)) : sq.nk;
  // keys of the tile's first and last rows
  const int tok0 = t * BM / p.G, tok1 = min(sq.nq - 1, (t * BM + BM - 1) / p.G);
  const int klo = p.causal ? min(sq.nk, max(0, tok0 + 1 + sq.nk - sq.nq)) : sq.nk;
  const int khi = p.causal ? min(sq.nk, max(0, tok1 + 1 + sq.nk - sq.nq)) : sq.nk;

  v8 qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) qf[ks] = v8{};
  if (valid) {
    const T* q = static_cast<const T*>(p.q) + (long)(sq.q0 + tok) * p.q_st + (long)(hk * p.G + g) * p.q_sh;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const v8*>(q + ks * 16 + half * 8);
  }

  // LDS places of 16-byte chunk c of a row: K's fragments are one chunk of 16 consecutive
  // rows, V's four chunks of 4 consecutive rows; both hit every bank once this way
  auto k_at = [](int key, int c) {
    return HD == 128 ? key * HD + ((c ^ (key & 15)) << 3) : key * HD + ((c ^ ((key >> 1) & 7)) << 3);
  };
  auto v_at = [](int key, int c) {
    return HD == 128 ? key * HD + ((c ^ ((key & 3) << 2)) << 3) : key * HD + ((c ^ ((key & 2) << 1)) << 3);
  };

  float16_t o[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) o[ct] = float16_t{};
  float m = -INFINITY, l = 0.f;
  if (tid == 0) any_bad = 0;

  for (int key0 = 0; key0 < khi; key0 += AT_KEYS) {
    __syncthreads();
    // ---- the tile into LDS; places behind the last key repeat it ----
    for (int i = tid; i < AT_KEYS * CH; i += 256) {
      const int key = i / CH, c = i % CH, kk = min(key0 + key, sq.nk - 1);
      v8 kx, vx;
      if constexpr (KV == KV_ROWS) {
        kx = *reinterpret_cast<const v8*>(static_cast<const T*>(p.k) + (long)(sq.k0 + kk) * p.k_st + (long)hk * p.k_sh + c * 8);
        vx = *reinterpret_cast<const v8*>(static_cast<const T*>(p.v) + (long)(sq.k0 + kk) * p.v_st + (long)hk * p.v_sh + c * 8);
      } else {
        const long page = min(max(p.table[(long)b * p.table_w + (kk >> p.page_shift)], 0), p.n_pages - 1);
        const long at = ((page * p.Hkv + hk) << p.page_shift) + (kk & ((1 << p.page_shift) - 1));
        if constexpr (KV == KV_PAGES) {
          kx = *reinterpret_cast<const v8*>(static_cast<const T*>(p.k) + at * HD + c * 8);
          vx = *reinterpret_cast<const v8*>(static_cast<const T*>(p.v) + at * HD + c * 8);
        } else {
          auto dequant = [&](const void* base, const uint8_t* sc) {
            const u32x2_t w = *reinterpret_cast<const u32x2_t*>(static_cast<const uint8_t*>(base) + at * HD + c * 8);
            const float s = __builtin_bit_cast(float, (unsigned)sc[at] << 23);
            v8 y;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[j], false), d = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[j], true);
              const v2 u = pack2<T>(a[0] * s, a[1] * s), x = pack2<T>(d[0] * s, d[1] * s);
              y[4 * j] = u[0];
              y[4 * j + 1] = u[1];
              y[4 * j + 2] = x[0];
              y[4 * j + 3] = x[1];
            }
            return y;
          };
          kx = dequant(p.k, p.ks);
          vx = dequant(p.v, p.vs);
        }
      }
      *reinterpret_cast<v8*>(kt + k_at(key, c)) = kx;
      *reinterpret_cast<v8*>(vt + v_at(key, c)) = vx;
    }
    __syncthreads();

    // ---- a tile that some row sees in part: an infinity or NaN of V in a place that a row
    // does not see must not reach it (0 * inf), so such values are taken out of the tile and
    // added to the rows that do see them ----
    const bool part = key0 + AT_KEYS > klo;
    bool fix = false;
    if (part) {
      unsigned acc = 0;
      for (int i = tid; i < AT_KEYS * HD / 2; i += 256) acc |= (reinterpret_cast<const unsigned*>(vt)[i] & Elem<T>::EXP) + Elem<T>::LOW;
      if (acc & 0x80008000u) any_bad = 1;
      __syncthreads();
      fix = any_bad;
      if (fix) {
        for (int i = tid; i < 3 * HD; i += 256) (&bad[0][0])[i] = 0x7FFFFFFF;
        __syncthreads();
        for (int i = tid; i < AT_KEYS * HD; i += 256) {
          const int key = i / HD, d = i % HD, at = v_at(key, d >> 3) + (d & 7);
          const float x = (float)vt[at];
          if (!(fabsf(x) < INFINITY)) {
            atomicMin(&bad[x > 0 ? 0 : x < 0 ? 1 : 2][d], key0 + key);
            vt[at] = (T)0.f;
          }
        }
        __syncthreads();
      }
    }

    // ---- S^T ----
    float16_t s[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      s[kb] = float16_t{};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const v8 kf = *reinterpret_cast<const v8*>(kt + k_at(kb * 32 + r32, ks * 2 + half));
        s[kb] = Elem<T>::mfma32(kf, qf[ks], s[kb]);
      }
    }
    if (part) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (key0 + kb * 32 + 8 * (i >> 2) + 4 * half + (i & 3) >= lim) s[kb][i] = -INFINITY;
    }
    // ---- running softmax ----
    float mx = m;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kb][i]);
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    const float ms = mx == -INFINITY ? 0.f : mx * p.scale_log2e;
    const float f = __builtin_amdgcn_exp2f(m * p.scale_log2e - ms);
    m = mx;
    l *= f;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) o[ct] *= f;
    v8 pf[4];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][i], p.scale_log2e, -ms));
        const float d = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][i + 1], p.scale_log2e, -ms));
        l += a + d;
        const v2 u = pack2<T>(a, d);
        pf[kb * 2 + (i >> 3)][i & 7] = u[0];
        pf[kb * 2 + (i >> 3)][(i & 7) + 1] = u[1];
      }
    // ---- O^T += V^T P^T ----
    const int va = (lane >> 2) & 3, vb = lane & 3;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        v8 vf;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int key = kk * 16 + e * 8 + 4 * half + va, d = ct * 32 + 16 * ((lane >> 4) & 1) + 4 * vb;
          typedef short s16x4 __attribute__((ext_vector_type(4)));
          const v4 x = __builtin_bit_cast(v4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                  (__attribute__((address_space(3))) s16x4*)(vt + v_at(key, d >> 3) + (d & 7))));
#pragma unroll
          for (int j = 0; j < 4; ++j) vf[e * 4 + j] = x[j];
        }
        o[ct] = Elem<T>::mfma32(vf, pf[kk], o[ct]);
      }
    if (fix) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int d = ct * 32 + 8 * (i >> 2) + 4 * half + (i & 3);
          if (bad[0][d] < lim) o[ct][i] += INFINITY;
          if (bad[1][d] < lim) o[ct][i] -= INFINITY;
          if (bad[2][d] < lim) o[ct][i] = NAN;
        }
      __syncthreads();
      if (tid == 0) any_bad = 0;
    }
  }

  if (!valid) return;
  l += __shfl_xor(l, 32);
  const float rl = l == 0.f ? 0.f : 1.0f / l;
  T* out = static_cast<T*>(p.out) + (long)(sq.q0 + tok) * p.o_st + (long)(hk * p.G + g) * p.o_sh;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const v2 a = pack2<T>(o[ct][i] * rl, o[ct][i + 1] * rl), c = pack2<T>(o[ct][i + 2] * rl, o[ct][i + 3] * rl);
      *reinterpret_cast<v4*>(out + ct * 32 + 2 * i + 4 * half) = v4{a[0], a[1], c[0], c[1]};
    }
}

template <typename T, int HD>
void launch_kv(const AttendParams& p, int kv, int grid, hipStream_t s) {
  if (kv == KV_ROWS) CK_LAUNCH((attend_kernel<T, HD, KV_ROWS>), dim3(grid), dim3(256), 0, s, p);
  else if (kv == KV_PAGES) CK_LAUNCH((attend_kernel<T, HD, KV_PAGES>), dim3(grid), dim3(256), 0, s, p);
  else CK_LAUNCH((attend_kernel<T, HD, KV_E4M3>), dim3(grid), dim3(256), 0, s, p);
}

void launch_attend(const char* what, AttendParams& p, const AttendQuery& a, int kv, hipStream_t s) {
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
  // sum over sequences of ceil(rows / 128) is at most this
  const long tiles = (long)a.T * p.G / 128 + a.B;
  CK_REQUIRE(tiles * p.Hkv < (1L << 31), w + ": too many rows");
  const int grid = (int)(tiles * p.Hkv);
  if (a.dtype == DT_F16) {
    if (a.head_dim == 64) launch_kv<half_t, 64>(p, kv, grid, s);
    else launch_kv<half_t, 128>(p, kv, grid, s);
  } else {
    if (a.head_dim == 64) launch_kv<bf16_t, 64>(p, kv, grid, s);
    else launch_kv<bf16_t, 128>(p, kv, grid, s);
  }
  CK_LAUNCHED(what);
}

}  // namespace

size_t attention_workspace(int, int, long, int, int, int) { return 0; }

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
  launch_attend("attention_varlen", p, a, KV_ROWS, s);
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
  launch_attend("attention_paged", p, a, c.dtype == DT_E4M3 ? KV_E4M3 : KV_PAGES, s);
}

}  // namespace ck
