// Rotary positions.  Pair i of a head's first `rot` elements is turned by the angle
// a = position * inv_freq[i]:
//   y0 = s (x0 cos a - x1 sin a),  y1 = s (x1 cos a + x0 sin a),
// pairs (i, i + rot/2), or (2i, 2i + 1) where interleaved; the elements behind `rot`
// are copied.  With axes (time, row, column, ...) there is a position for each, and a pair's
// angle goes by the one that axes[i] names.
//
// Bound by memory: every element is read and written once.  The angles belong to a
// token, not to its heads, so a workgroup computes those of its tokens once into LDS
// and then passes over the heads, 32 bytes a thread and step.
#include "common.h"
#include "elem16.h"
#include "kernels.h"
#include "rope_angles.h"

namespace ck {
namespace {

constexpr int ROPE_LDS = 1024;   // pairs of a workgroup's tokens: cos and sin in 8 KB

struct RopeParams {
  const void* x;
  void* out;
  RopeAngles a;
  long xst, xsh, ost, osh;   // element strides of tokens and heads
  int T, H, hd, rot, tpw;    // tpw: tokens per workgroup
  unsigned per_tok, m_tok;   // items (2V elements) per token and its div_magic
  unsigned per_head, m_head; // items per head and its div_magic
  int interleaved, copy;     // copy: the elements behind rot are to be copied (out is not x)
};

// V: pairs per item.  8 where rows and strides are whole 16-byte chunks and rot a multiple of 16, else 1.
// NT: written past the caches, for an output that the L2s do not hold (8 x 4 MiB): 12288 tokens of
// 20 heads of 128, 126 MB in all, 29.6 -> 23.3 us = 5.4 TB/s (loads past
// them too: 32.9).  4 tokens of 8 heads of 64: 2.4 us, a launch.
// APART (calls with axes; the others stay as they were, to the bit): where pairs are neighbours, and behind rot, an
// item's two runs lie half a head apart, so that neighbouring lanes have neighbouring runs: 12288 tokens of 20 heads of
// 128, all turned, neighbouring pairs, 126 MB, 27.5 -> 22.5 us; with two items a thread in place of four, 20.7 = 6.1 TB/s.
// 256 tokens of 16 heads of 64: 3.0 us.
template <typename T, int V, bool NT, bool APART>
__global__ __launch_bounds__(256) void rope_kernel(const RopeParams p) {
  __shared__ float2_t cs[ROPE_LDS];
  const int t0 = blockIdx.x * p.tpw, nt = min(p.tpw, p.T - t0), half = p.rot >> 1;
  rope_angles<256>(p.a, t0, nt, cs, threadIdx.x);
  __syncthreads();
  const T* x = static_cast<const T*>(p.x);
  T* out = static_cast<T*>(p.out);
  typedef T vec __attribute__((ext_vector_type(V)));
  auto put = [](T* to, vec v) {
    if (NT) __builtin_nontemporal_store(v, reinterpret_cast<vec*>(to));
    else *reinterpret_cast<vec*>(to) = v;
  };
  for (unsigned i = threadIdx.x; i < nt * p.per_tok; i += 256) {
    const unsigned t = div_by(i, p.m_tok), r = i - t * p.per_tok, h = div_by(r, p.m_head);
    const int e = (int)(r - h * p.per_head) * V;   // first pair of the item; elements 2e.. behind rot
    const T* xr = x + (t0 + t) * p.xst + h * p.xsh;
    T* yr = out + (t0 + t) * p.ost + h * p.osh;
    if (APART && (e >= half || p.interleaved)) {
      const int from = p.interleaved ? 0 : 2 * half, i = p.interleaved ? e : e - half;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int at = from + i + (k ? (p.hd - from) / 2 : 0);
        const bool turn = p.interleaved && at < 2 * half;
        if (!turn && !p.copy) continue;
        vec v = *reinterpret_cast<const vec*>(xr + at);
        if (turn) {
          const float2_t* c = cs + t * half + at / 2;
#pragma unroll
          for (int j = 0; j < V / 2; ++j) {
            const float2_t u = c[j];
            const float a0 = (float)v[2 * j], a1 = (float)v[2 * j + 1];
            v[2 * j] = (T)(a0 * u[0] - a1 * u[1]);
            v[2 * j + 1] = (T)(a1 * u[0] + a0 * u[1]);
          }
        }
        put(yr + at, v);
      }
      continue;
    }
    if (e >= half) {
      if (!p.copy) continue;
      if constexpr (V == 1) {
        yr[2 * e] = xr[2 * e];
        if (2 * e + 1 < p.hd) yr[2 * e + 1] = xr[2 * e + 1];
      } else {
        const vec v0 = *reinterpret_cast<const vec*>(xr + 2 * e), v1 = *reinterpret_cast<const vec*>(xr + 2 * e + V);
        put(yr + 2 * e, v0);
        put(yr + 2 * e + V, v1);
      }
      continue;
    }
    const float2_t* c = cs + t * half + e;
    const int a = p.interleaved ? 2 * e : e, b = p.interleaved ? 2 * e + V : e + half;
    vec v0 = *reinterpret_cast<const vec*>(xr + a), v1 = *reinterpret_cast<const vec*>(xr + b);
    vec y0, y1;
    if (V > 1 && p.interleaved) {
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        const float2_t u = c[j], w = c[V / 2 + j];
        const float a0 = (float)v0[2 * j], a1 = (float)v0[2 * j + 1], b0 = (float)v1[2 * j], b1 = (float)v1[2 * j + 1];
        y0[2 * j] = (T)(a0 * u[0] - a1 * u[1]);
        y0[2 * j + 1] = (T)(a1 * u[0] + a0 * u[1]);
        y1[2 * j] = (T)(b0 * w[0] - b1 * w[1]);
        y1[2 * j + 1] = (T)(b1 * w[0] + b0 * w[1]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float2_t u = c[j];
        const float a0 = (float)v0[j], a1 = (float)v1[j];
        y0[j] = (T)(a0 * u[0] - a1 * u[1]);
        y1[j] = (T)(a1 * u[0] + a0 * u[1]);
      }
    }
    put(yr + a, y0);
    put(yr + b, y1);
  }
}

}  // namespace

RopeAngles rope_angles_of(const char* what, const int* positions, int n_axes, const int* axes, const double* inv_freq,
                          int T, int rot, float scale, bool inverse) {
  CK_REQUIRE(n_axes >= 1 && (axes || n_axes == 1), std::string(what) + ": positions of several axes need every pair's axis");
  RopeAngles a{};
  a.pos = positions;
  a.inv_freq = inv_freq;
  a.axes = axes;
  a.n_axes = n_axes;
  a.T = T;
  a.half = rot / 2;
  a.scale = scale;
  a.sign = inverse ? -1.0f : 1.0f;
  return a;
}

void launch_rope(const void* x, void* out, const int* positions, int n_axes, const int* axes, const double* inv_freq,
                 int T, int H, int hd, int rot, long xst, long xsh, long ost, long osh, int dtype, bool interleaved,
                 float scale, bool inverse, hipStream_t s) {
  CK_REQUIRE(T >= 0 && H > 0 && hd > 0, "rope: sizes must be positive");
  CK_REQUIRE(rot > 0 && rot % 2 == 0 && rot <= hd, "rope: 2 * len(inv_freq) must be even and at most head_dim");
  CK_REQUIRE(dtype == DT_F16 || dtype == DT_BF16, "rope: f16 or bf16");
  CK_REQUIRE(hd <= 512 && H <= 1024 && (long)H * hd <= 65536, "rope: head_dim up to 512, heads up to 1024, 65536 elements a token");
  if (T == 0) return;
  CK_REQUIRE(x && out && positions && inv_freq, "rope: null pointer");
  CK_REQUIRE(x != out || (xst == ost && xsh == osh), "rope: in place, out must be laid out as x");
  RopeParams p{};
  p.x = x;
  p.out = out;
  p.a = rope_angles_of("rope", positions, n_axes, axes, inv_freq, T, rot, scale, inverse);
  p.xst = xst;
  p.xsh = xsh;
  p.ost = ost;
  p.osh = osh;
  p.T = T;
  p.H = H;
  p.hd = hd;
  p.rot = rot;
  p.interleaved = interleaved;
  p.copy = rot < hd && x != out;
  const bool wide = rot % 16 == 0 && hd % 16 == 0 && ((xst | xsh | ost | osh) & 7) == 0 &&
                    ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  p.per_head = wide ? hd / 16 : (hd + 1) / 2;
  p.per_tok = p.per_head * H;
  p.m_head = div_magic(p.per_head);
  p.m_tok = div_magic(p.per_tok);
  // four items a thread (APART: two), but enough workgroups to fill the CUs twice first
  const bool apart = axes && wide;
  int tpw = std::max(1, std::min<int>((apart ? 512 : 1024) / (int)p.per_tok, ceil_div(T, 512)));
  tpw = std::max(1, std::min(tpw, ROPE_LDS / (rot / 2)));
  p.tpw = tpw;
  const dim3 grid(ceil_div(T, tpw)), block(256);
  CK_REQUIRE(grid.x < (1u << 24), "rope: too many tokens for one launch");   // of under 2^32 threads
  const bool large = (long)T * H * hd * 2 > (32L << 20);
  auto go = [&](auto kernel) { CK_LAUNCH(kernel, grid, block, 0, s, p); };
  auto of = [&](auto t) {
    typedef decltype(t) E;
    if (!wide) go(rope_kernel<E, 1, false, false>);
    else if (apart) large ? go(rope_kernel<E, 8, true, true>) : go(rope_kernel<E, 8, false, true>);
    else large ? go(rope_kernel<E, 8, true, false>) : go(rope_kernel<E, 8, false, false>);
  };
  if (dtype == DT_F16) of(half_t{});
  else of(bf16_t{});
  CK_LAUNCHED("rope");
}

}  // namespace ck
