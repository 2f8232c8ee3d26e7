// What the kernels of shaped attention share: scores that are capped, lowered by distance and masked to an interval of positions per token.
//
//     x_ij = scale q_i . k_j;   x <- cap tanh(x / cap)  (cap > 0);   x <- x - slope_h |pos_i - pos_j|
//     visible: first_i <= pos_j <= last_i
//
// Causal attention, windows, documents behind one another and prefixes that every token sees are all such intervals, so one pair of
// numbers per token stands for the mask.  Cached tokens lie in the order of their positions, which ``key_pos`` lists once tokens have
// been shed from a cache (null: token j of a row has position j); an interval of positions is then a run of the row.
// Positions stay below 2^24, exact in fp32; scores are kept in the base of the exponent, x log2(e).
#pragma once
#include "common.cuh"

namespace smc {

constexpr int SH_POS_END = 1 << 24;
constexpr float SH_LOG2E = 1.4426950408889634f, SH_LN2 = 0.6931471805599453f;

struct ShapedCache {
  const int* block_table;        // [bt_rows, bt_stride] page of every cached token
  const int* key_pos;            // [bt_rows, kp_stride] its position, ascending, or null
  const int2* bounds;            // per query token: first and last visible position, or null: all up to its own
  const float* slopes;           // per query head, or null
  int bt_stride, bt_rows, kp_stride, n_pages;
  float scale, cap;
};

// One sequence of a call: block-table row, tokens held before the new ones, index of the first new one in q, new tokens.
struct ShapedRun { int row, held, at, n; };

// A run whose numbers leave the tables or q counts as empty and raises the status bit.
__device__ __forceinline__ ShapedRun shaped_run(const ShapedCache& c, const int4* runs, int s, int T, int* status) {
  const int4 v = runs[s];
  ShapedRun r{v.x, v.y, v.z, v.w};
  if (r.n <= 0) { r.n = 0; return r; }
  if (r.row < 0 || r.row >= c.bt_rows || r.held < 0 || r.at < 0 || r.at > T - r.n || r.held > c.bt_stride - r.n) {
    atomicOr(status, SMC_ERR_BOUNDS);
    r.n = 0;
  }
  return r;
}

// Visible positions of query token t of q, whose own position is pos; [POS_END, -1] where it sees nothing.
__device__ __forceinline__ int2 shaped_bounds(const ShapedCache& c, int t, int pos) {
  if (c.bounds == nullptr) return make_int2(0, pos);
  const int2 b = c.bounds[t];
  const int lo = max(b.x, 0), hi = min(b.y, SH_POS_END - 1);
  return lo <= hi ? make_int2(lo, hi) : make_int2(SH_POS_END, -1);
}

// First index of the ascending list p[0, n) whose value is >= v (n if none), found by a whole warp: 32 probes at a time.
__device__ __forceinline__ int shaped_lower_bound(const int* p, int n, int v) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = n;                                  // p[lo - 1] < v <= p[hi]
  while (hi - lo > 32) {
    const int step = (hi - lo) / 33 + 1, at = lo + (lane + 1) * step - 1;
    const bool below = at < hi && p[at] < v;
    const int k = __popc(__ballot_sync(0xffffffffu, below));       // ascending: the first k probes lie below
    const int end = lo + (k + 1) * step - 1;
    lo += k * step;
    hi = min(hi, end);
  }
  const bool below = lo + lane < hi && p[lo + lane] < v;
  return lo + __popc(__ballot_sync(0xffffffffu, below));
}

// exp2 of non-positive numbers and a few above
__device__ __forceinline__ float shaped_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Registers of a warpgroup, moved between those that need few and those that need many (all of a warpgroup's warps call it; the sum over
// the block is at most what it was launched with).
template <int N> __device__ __forceinline__ void regs_fewer() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_more() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

// two fp32 operations at once
__device__ __forceinline__ uint64_t f2_pair(float a, float b) {
  uint64_t y;
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float2 f2_unpair(uint64_t v) {
  float2 y;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(y.x), "=f"(y.y) : "l"(v));
  return y;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t y;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y) : "l"(a), "l"(b), "l"(c));
  return y;
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t y;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
  return y;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t y;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
  return y;
}
__device__ __forceinline__ float shaped_max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// tanh u = u P(u^2) for u^2 <= SH_TANH_MAX: minimax polynomials of tanh(sqrt y) / sqrt y on [0, 0.625^2], found by an exchange
// algorithm in double precision; largest relative error 2.7e-6 with four coefficients (behind it stand probabilities of eight
// bits) and 3.7e-9 with six (32-bit results).  Scores beyond, rare at the usual caps, take 1 - 2 / (1 + e^2|u|).
constexpr float SH_TANH_MAX = 0.390625f;
template <int N>
__host__ __device__ constexpr float tanh_coef(int k) {
  constexpr float c4[4] = {0.9999972581863403f, -0.333099901676178f, 0.13020624220371246f, -0.04011745750904083f};
  constexpr float c6[6] = {1.0f, -0.3333326280117035f, 0.13331185281276703f, -0.0537252314388752f, 0.020603151991963387f, -0.005672425962984562f};
  static_assert(N == 4 || N == 6, "four or six coefficients");
  return N == 4 ? c4[k] : c6[k];
}
__device__ __forceinline__ float shaped_tanh_far(float u) {
  return copysignf(1.0f - __fdividef(2.0f, 1.0f + shaped_ex2(2.0f * SH_LOG2E * fabsf(u))), u);
}
// cap log2(e) tanh(x in) of one number
__device__ __forceinline__ float shaped_cap(float x, float in, float out) {
  const float u = x * in, y = u * u;
  float t;
  if (y > SH_TANH_MAX) {
    t = shaped_tanh_far(u);
  } else {
    t = tanh_coef<6>(5);
#pragma unroll
    for (int i = 4; i >= 0; --i) t = fmaf(t, y, tanh_coef<6>(i));
    t *= u;
  }
  return t * out;
}
// the same of the 2 W numbers x, two at a time, N coefficients
template <int N, int W>
__device__ __forceinline__ void shaped_cap_pairs(uint64_t (&x)[W], float in, float out) {
  const uint64_t in2 = f2_pair(in, in);
  uint64_t u[W];
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    u[i] = f2_mul(x[i], in2);
    const uint64_t y = f2_mul(u[i], u[i]);
    const float2 yy = f2_unpair(y);
    top = shaped_max3(top, yy.x, yy.y);
    uint64_t t = f2_pair(out * tanh_coef<N>(N - 1), out * tanh_coef<N>(N - 1));
#pragma unroll
    for (int k = N - 2; k >= 0; --k) t = f2_fma(t, y, f2_pair(out * tanh_coef<N>(k), out * tanh_coef<N>(k)));
    x[i] = f2_mul(t, u[i]);
  }
  if (top > SH_TANH_MAX) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float2 uu = f2_unpair(u[i]), nn = f2_unpair(x[i]);
      x[i] = f2_pair(uu.x * uu.x > SH_TANH_MAX ? out * shaped_tanh_far(uu.x) : nn.x, uu.y * uu.y > SH_TANH_MAX ? out * shaped_tanh_far(uu.y) : nn.y);
    }
  }
}

}  // namespace smc
