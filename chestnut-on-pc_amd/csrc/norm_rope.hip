// Norms of query and key heads with the position rotation in the same pass:
//   y = w x / sqrt(mean(x^2) + eps),  then the first `rot` elements of y turned as rope.hip turns them,
// mean over the elements of one head, weights w of their own for queries and keys.  The squares
// are summed in f32 and nothing is rounded but the output (a norm that rounds before the
// rotation rounds twice).
//
// Bound by memory: every element is read and written once.  The head_dim / 16 lanes of a head
// hold 16 elements each, both halves of eight pairs, so that the sum takes shuffles within a
// few lanes and the rotation none; a lane holds the same pairs of every head that it comes
// across, and their weights in registers.  The angles belong to a token: a workgroup computes
// those of its tokens once into LDS.  A lane's heads are sent for together, before the angles: 12288
// tokens of 32 heads of 128, half of each turned, 201 MB, by calls one after another 59 us with one head
// under way, 41.6 with four, 38.9 with six = 5.2 TB/s, 39 with eight, 67 with twelve (a kernel trace:
// 40.9, least 38.2).
#include "common.h"
#include "elem16.h"
#include "kernels.h"
#include "rope_angles.h"

namespace ck {
namespace {

constexpr int NR_LDS = 1024;   // pairs of a workgroup's tokens: cos and sin in 8 KB
constexpr int NR_HEADS = 6;      // of a lane, that are under way together

struct NormRopeParams {
  NormRopeHeads q, k;
  RopeAngles a;
  int T, H, hd, tpw;           // H: heads of q and k together; tpw: tokens per workgroup
  unsigned m_H;                // div_magic of H
  int interleaved, wtype, w_aligned;
  float eps, inv_hd;
};

__device__ __forceinline__ float weight_at(const void* w, int type, int i) {
  if (!w) return 1.0f;
  return type == DT_F16 ? (float)static_cast<const half_t*>(w)[i] : type == DT_BF16 ? (float)static_cast<const bf16_t*>(w)[i] :
                                                                                      static_cast<const float*>(w)[i];
}

// The sum over LPR lanes (a power of two), in each of them.
template <int LPR>
__device__ __forceinline__ float lanes_sum(float v) {
  if (LPR > 1) v += dpp_mov<DPP_QUAD_1032>(v);
  if (LPR > 2) v += dpp_mov<DPP_QUAD_2301>(v);
  if (LPR > 4) v += dpp_mov<DPP_ROW_HALF_MIRROR>(v);
  if (LPR > 8) v += dpp_mov<DPP_ROW_MIRROR>(v);
  if (LPR > 16) v += __shfl_xor(v, 16);
  return v;
}

// Eight weights from element i on (a multiple of 8).
__device__ __forceinline__ void weights_at(float (&f)[8], const void* w, int type, int i, bool aligned) {
  if (!w || !aligned) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = weight_at(w, type, i + j);
  } else if (type == DT_F16) {
    const half8_t v = *reinterpret_cast<const half8_t*>(static_cast<const half_t*>(w) + i);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (float)v[j];
  } else if (type == DT_BF16) {
    const bf16x8_t v = *reinterpret_cast<const bf16x8_t*>(static_cast<const bf16_t*>(w) + i);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (float)v[j];
  } else {
    const float4_t *v = reinterpret_cast<const float4_t*>(static_cast<const float*>(w) + i), x = v[0], y = v[1];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[j] = x[j];
      f[4 + j] = y[j];
    }
  }
}

template <typename T, int LPR, bool NT>
__global__ __launch_bounds__(256) void norm_rope_kernel(const NormRopeParams p) {
  typedef typename Elem<T>::v8 v8;
  constexpr int U = NR_HEADS, STEP = 256 / LPR;   // STEP: heads side by side
  __shared__ float2_t cs[NR_LDS];
  const int t0 = blockIdx.x * p.tpw, nt = min(p.tpw, p.T - t0), half = p.a.half;
  const unsigned n = nt * p.H;
  const int e = (int)(threadIdx.x % LPR) * 8;   // the lane's first pair
  const bool turn = e < half;
  // its two runs of eight elements: both halves of eight pairs, else two that lie apart, so that neighbouring lanes
  // have neighbouring runs; where interleaved, each is turned by itself
  const int from = p.interleaved ? 0 : 2 * half, a = turn && !p.interleaved ? e : from + e - (p.interleaved ? 0 : half);
  const int b = turn && !p.interleaved ? e + half : a + (p.hd - from) / 2;
  v8 v0[U], v1[U];
  auto load = [&](unsigned r0) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const unsigned r = min(r0 + i * STEP, n - 1), t = div_by(r, p.m_H), h = r - t * p.H;
      const bool isk = (int)h >= p.q.heads;
      const long g = isk ? (int)h - p.q.heads : (int)h;
      const T* x = static_cast<const T*>(isk ? p.k.x : p.q.x) + (t0 + t) * (isk ? p.k.x_st : p.q.x_st) + g * (isk ? p.k.x_sh : p.q.x_sh);
      v0[i] = *reinterpret_cast<const v8*>(x + a);
      v1[i] = *reinterpret_cast<const v8*>(x + b);
    }
  };
  unsigned r0 = threadIdx.x / LPR;
  load(r0);
  float wq[2][8], wk[2][8];
  weights_at(wq[0], p.q.weight, p.wtype, a, p.w_aligned);
  weights_at(wq[1], p.q.weight, p.wtype, b, p.w_aligned);
  weights_at(wk[0], p.k.weight, p.wtype, a, p.w_aligned);
  weights_at(wk[1], p.k.weight, p.wtype, b, p.w_aligned);
  rope_angles<256>(p.a, t0, nt, cs, threadIdx.x);
  __syncthreads();
  auto put = [](T* to, v8 v) {
    if (NT) __builtin_nontemporal_store(v, reinterpret_cast<v8*>(to));
    else *reinterpret_cast<v8*>(to) = v;
  };
  for (; r0 < n; r0 += U * STEP) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const unsigned r = r0 + i * STEP;
      if (r >= n) break;
      const unsigned t = div_by(r, p.m_H), h = r - t * p.H;
      const bool isk = (int)h >= p.q.heads;
      const long g = isk ? (int)h - p.q.heads : (int)h;
      T* y = static_cast<T*>(isk ? p.k.out : p.q.out) + (t0 + t) * (isk ? p.k.o_st : p.q.o_st) + g * (isk ? p.k.o_sh : p.q.o_sh);
      float f[16], sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        f[j] = (float)v0[i][j];
        f[8 + j] = (float)v1[i][j];
        sum = __builtin_fmaf(f[j], f[j], sum);
        sum = __builtin_fmaf(f[8 + j], f[8 + j], sum);
      }
      const float inv = 1.0f / sqrtf(__builtin_fmaf(lanes_sum<LPR>(sum), p.inv_hd, p.eps));
#pragma unroll
      for (int j = 0; j < 16; ++j) f[j] *= inv * (isk ? wk[j / 8][j % 8] : wq[j / 8][j % 8]);
      if (p.interleaved) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int at = k ? b : a;
          if (at < 2 * half) {
            const float2_t* c = cs + t * half + at / 2;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2_t u = c[j];
              const float x0 = f[8 * k + 2 * j], x1 = f[8 * k + 2 * j + 1];
              f[8 * k + 2 * j] = x0 * u[0] - x1 * u[1];
              f[8 * k + 2 * j + 1] = x1 * u[0] + x0 * u[1];
            }
          }
        }
      } else if (turn) {
        const float2_t* c = cs + t * half + e;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2_t u = c[j];
          const float x0 = f[j], x1 = f[8 + j];
          f[j] = x0 * u[0] - x1 * u[1];
          f[8 + j] = x1 * u[0] + x0 * u[1];
        }
      }
      v8 y0, y1;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        y0[j] = (T)f[j];
        y1[j] = (T)f[8 + j];
      }
      put(y + a, y0);
      put(y + b, y1);
    }
    if (r0 + U * STEP < n) load(r0 + U * STEP);
  }
}

// Any head_dim up to 512, any alignment: a wave a head, pair by pair.  Bound by its loads and stores of 2 bytes a lane: 12288
// tokens of 32 heads of 96, 24 pairs turned, 151 MB, 135 us = 1.1 TB/s (heads of 64 and of 128 in the form above 28.6 and 39.8).
template <typename T>
__global__ __launch_bounds__(256) void norm_rope_any_kernel(const NormRopeParams p) {
  constexpr int PAIRS = 512 / 2 / 64;   // of a lane
  __shared__ float2_t cs[NR_LDS];
  const int t0 = blockIdx.x * p.tpw, nt = min(p.tpw, p.T - t0), half = p.a.half, lane = threadIdx.x & 63;
  rope_angles<256>(p.a, t0, nt, cs, threadIdx.x);
  __syncthreads();
  for (unsigned r = threadIdx.x / 64; r < (unsigned)(nt * p.H); r += 4) {
    const unsigned t = div_by(r, p.m_H), h = r - t * p.H;
    const bool isk = (int)h >= p.q.heads;
    const NormRopeHeads& s = isk ? p.k : p.q;
    const long g = isk ? (int)h - p.q.heads : (int)h;
    const T* x = static_cast<const T*>(s.x) + (t0 + t) * s.x_st + g * s.x_sh;
    T* y = static_cast<T*>(s.out) + (t0 + t) * s.o_st + g * s.o_sh;
    float f[2 * PAIRS], sum = 0.f;
    // pair i: elements of the rotated part, then two neighbours behind it
    auto at = [&](int i, int second) {
      return i >= half ? 2 * i + second : p.interleaved ? 2 * i + second : i + second * half;
    };
#pragma unroll
    for (int n = 0; n < PAIRS; ++n) {
      const int i = lane + 64 * n;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        f[2 * n + k] = at(i, k) < p.hd && 2 * i < p.hd ? (float)x[at(i, k)] : 0.f;
        sum = __builtin_fmaf(f[2 * n + k], f[2 * n + k], sum);
      }
    }
    const float inv = 1.0f / sqrtf(__builtin_fmaf(wave_sum(sum), p.inv_hd, p.eps));
#pragma unroll
    for (int n = 0; n < PAIRS; ++n) {
      const int i = lane + 64 * n;
      if (2 * i >= p.hd) continue;
      const int i0 = at(i, 0), i1 = at(i, 1);
      float a = f[2 * n] * (inv * weight_at(s.weight, p.wtype, i0)), b = 0.f;
      if (i1 < p.hd) b = f[2 * n + 1] * (inv * weight_at(s.weight, p.wtype, i1));
      if (i < half) {
        const float2_t u = cs[t * half + i];
        const float c = a * u[0] - b * u[1];
        b = b * u[0] + a * u[1];
        a = c;
      }
      y[i0] = (T)a;
      if (i1 < p.hd) y[i1] = (T)b;
    }
  }
}

}  // namespace

void launch_norm_rope(const NormRopeHeads& q, const NormRopeHeads& k, const int* positions, int n_axes, const int* axes,
                      const double* inv_freq, int T, int hd, int rot, int dtype, int weight_dtype, float eps,
                      bool interleaved, float scale, hipStream_t s) {
  CK_REQUIRE(T >= 0 && q.heads >= 0 && k.heads >= 0 && q.heads + k.heads > 0 && hd > 0, "norm_rope: sizes must be positive");
  CK_REQUIRE(rot > 0 && rot % 2 == 0 && rot <= hd, "norm_rope: 2 * len(inv_freq) must be even and at most head_dim");
  CK_REQUIRE(dtype == DT_F16 || dtype == DT_BF16, "norm_rope: f16 or bf16");
  CK_REQUIRE(weight_dtype == DT_F16 || weight_dtype == DT_BF16 || weight_dtype == 0, "norm_rope: weights must be f32, f16 or bf16");
  CK_REQUIRE(q.heads <= 1024 && k.heads <= 1024 && hd <= 512 && (long)(q.heads + k.heads) * hd <= 65536,
             "norm_rope: head_dim up to 512, heads up to 1024, 65536 elements a token");
  CK_REQUIRE(eps >= 1.17549435e-38f && eps < INFINITY, "norm_rope: eps must be a normal positive number");
  if (T == 0) return;
  CK_REQUIRE(positions && inv_freq && (!q.heads || (q.x && q.out)) && (!k.heads || (k.x && k.out)), "norm_rope: null pointer");
  NormRopeParams p{};
  p.q = q;
  p.k = k;
  p.a = rope_angles_of("norm_rope", positions, n_axes, axes, inv_freq, T, rot, scale, false);
  p.T = T;
  p.H = q.heads + k.heads;
  p.hd = hd;
  p.m_H = div_magic(p.H);
  p.interleaved = interleaved;
  p.wtype = weight_dtype;
  p.eps = eps;
  p.inv_hd = 1.0f / hd;
  long strides = 0;
  uintptr_t ends = 0;
  for (const NormRopeHeads* x : {&q, &k})
    if (x->heads) {
      CK_REQUIRE(x->x != x->out || (x->x_st == x->o_st && x->x_sh == x->o_sh), "norm_rope: in place, out must be laid out as x");
      strides |= x->x_st | x->x_sh | x->o_st | x->o_sh;
      ends |= reinterpret_cast<uintptr_t>(x->x) | reinterpret_cast<uintptr_t>(x->out);
    }
  const bool wide = rot % 16 == 0 && hd >= 64 && (hd & (hd - 1)) == 0 && (strides & 7) == 0 && (ends & 15) == 0;
  p.w_aligned = ((reinterpret_cast<uintptr_t>(q.weight) | reinterpret_cast<uintptr_t>(k.weight)) & 15) == 0;
  // a lane's heads loaded at once, but enough workgroups to fill the CUs twice first
  int tpw = std::max(1, std::min<int>(NR_HEADS * (wide ? 4096 / hd : 4) / p.H, ceil_div(T, 512)));
  tpw = std::max(1, std::min(tpw, NR_LDS / (rot / 2)));
  p.tpw = tpw;
  const dim3 grid(ceil_div(T, tpw)), block(256);
  CK_REQUIRE(grid.x < (1u << 24), "norm_rope: too many tokens for one launch");   // of under 2^32 threads
  const bool large = (long)T * p.H * hd * 2 > (32L << 20);
  auto go = [&](auto kernel) { CK_LAUNCH(kernel, grid, block, 0, s, p); };
  auto of = [&](auto t) {
    typedef decltype(t) E;
    if (!wide) go(norm_rope_any_kernel<E>);
    else if (hd == 64) large ? go(norm_rope_kernel<E, 4, true>) : go(norm_rope_kernel<E, 4, false>);
    else if (hd == 128) large ? go(norm_rope_kernel<E, 8, true>) : go(norm_rope_kernel<E, 8, false>);
    else if (hd == 256) large ? go(norm_rope_kernel<E, 16, true>) : go(norm_rope_kernel<E, 16, false>);
    else large ? go(norm_rope_kernel<E, 32, true>) : go(norm_rope_kernel<E, 32, false>);
  };
  if (dtype == DT_F16) of(half_t{});
  else of(bf16_t{});
  CK_LAUNCHED("norm_rope");
}

}  // namespace ck
