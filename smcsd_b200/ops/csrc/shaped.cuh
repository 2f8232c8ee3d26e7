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
constexpr float SH_TANH3_REACH = 0.35f;                // of a tanh by three or four coefficients, see below
constexpr float SH_LOG2E = 1.4426950408889634f, SH_LN2 = 0.6931471805599453f;

struct ShapedCache {
  const int* block_table;        // [bt_rows, bt_stride] page of every cached token
  const int* key_pos;            // [bt_rows, kp_stride] its position, ascending, or null
  const int2* bounds;            // per query token: first and last visible position, or null: all up to its own
  const float* slopes;           // per query head, or null
  int bt_stride, bt_rows, kp_stride, n_pages;
  float mul;                     // scale log2(e)
  float cap_in, cap_out;         // scale / cap and cap log2(e), 0: no cap
  int bt_cols;                   // of the table, which may be some columns of a wider one; those that a position can name
  float near_reach;              // |tanh's argument| up to which factors folded into three or four coefficients serve; -1: not even zero
};

// The pitch of a block table: from row to row in the low 32 bits, its columns in the high ones (0: as many).
inline long long pitch_stride(long long pitch) { return pitch & 0xffffffffll; }
inline int pitch_cols(long long pitch) { return (int)(pitch >> 32 ? pitch >> 32 : pitch); }
inline bool pitch_fits(long long pitch) { return pitch > 0 && pitch_stride(pitch) <= 0x7fffffff && pitch_cols(pitch) <= pitch_stride(pitch); }

// Scales and caps (0: none) whose factors are fp32 numbers: scale log2(e), scale / cap and cap log2(e).
inline bool shaped_scores_fit(float scale, float cap) {
  auto normal = [](double x) { return x >= 1.2e-38 && x <= 3.4e38; };
  return normal((double)scale * 1.4426950408889634) && (cap == 0.f || (cap > 0.f && normal((double)scale / cap) && normal((double)cap * 1.4426950408889634)));
}

// (in double precision: an error of a factor is one of every score)
inline ShapedCache shaped_cache(const int* block_table, long long bt_pitch, int bt_rows, int n_pages, const int* key_pos, int kp_stride, const int* bounds,
                                const float* slopes, float scale, float cap) {
  const double log2e = 1.4426950408889634, in = cap > 0.f ? (double)scale / cap : 0.0;
  // the folded coefficients hold scale log2(e) (scale / cap)^2k up to k = 3; below 2e-5 they fade
  const float near_reach = in >= 2e-5 && scale * log2e * in * in * in * in * in * in <= 1e37 ? SH_TANH3_REACH : -1.f;
  return ShapedCache{block_table, key_pos, (const int2*)bounds, slopes, (int)pitch_stride(bt_pitch), bt_rows, kp_stride, n_pages, (float)(scale * log2e),
                     cap > 0.f ? (float)((double)scale / cap) : 0.f, cap > 0.f ? (float)(cap * log2e) : 0.f,
                     pitch_cols(bt_pitch) < SH_POS_END ? pitch_cols(bt_pitch) : SH_POS_END, near_reach};
}

// One sequence of a call: block-table row, tokens held before the new ones, index of the first new one in q, new tokens.
struct ShapedRun { int row, held, at, n; };

// A run whose numbers leave the tables or q counts as empty and raises the status bit.
__device__ __forceinline__ ShapedRun shaped_run(const ShapedCache& c, const int4* runs, int s, int T, int* status) {
  const int4 v = runs[s];
  ShapedRun r{v.x, v.y, v.z, v.w};
  if (r.n <= 0) { r.n = 0; return r; }
  if (r.row < 0 || r.row >= c.bt_rows || r.held < 0 || r.at < 0 || r.at > T - r.n || r.held > c.bt_cols - r.n) {
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

__device__ __forceinline__ float shaped_min3(float a, float b, float c) {
  float y;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// tanh u = u P(u^2): minimax polynomials of tanh(sqrt y) / sqrt y on [0, reach^2], found by an exchange algorithm in double precision.
// Largest relative errors, of the coefficients as they stand here in fp32: three up to 0.35 3.0e-6, five up to 0.75 6.3e-7 (the probabilities behind these two are rounded to
// eight bits, but the log-sum-exp of a prompt takes them along: up to 0.35 x 3.0e-6 of a cap, 5e-5 at 50; four and six in their place 8192 tokens 772 -> 872 us);
// four up to 0.35 6.1e-8, six up to 0.625 1.0e-8 (32-bit results).  Scores beyond, rare at the usual caps, take 1 - 2 / (1 + e^2|u|).
constexpr float SH_TANH5_REACH = 0.75f, SH_TANH6_REACH = 0.625f;
template <int N>
__host__ __device__ constexpr float tanh_coef(int k) {
  constexpr float c3[3] = {0.9999971985816956f, -0.33291319012641907f, 0.1239800825715065f};
  constexpr float c4[4] = {0.9999999403953552f, -0.3333243131637573f, 0.13296015560626984f, -0.04897000268101692f};
  constexpr float c5[5] = {0.999999463558197f, -0.33328500390052795f, 0.13261182606220245f, -0.05011862516403198f, 0.012984894216060638f};
  constexpr float c6[6] = {1.0f, -0.3333326280117035f, 0.13331185281276703f, -0.0537252314388752f, 0.020603151991963387f, -0.005672425962984562f};
  static_assert(N >= 3 && N <= 6, "three to six coefficients");
  return N == 3 ? c3[k] : N == 4 ? c4[k] : N == 5 ? c5[k] : c6[k];
}
__device__ __forceinline__ float shaped_tanh_far(float u) {
  return copysignf(1.0f - __fdividef(2.0f, 1.0f + shaped_ex2(2.0f * SH_LOG2E * fabsf(u))), u);
}
// out tanh(x in) of one number
__device__ __forceinline__ float shaped_cap(float x, float in, float out) {
  const float u = x * in, y = u * u;
  float t;
  if (!(y <= SH_TANH6_REACH * SH_TANH6_REACH)) {
    t = shaped_tanh_far(u);
  } else {
    t = tanh_coef<6>(5);
#pragma unroll
    for (int i = 4; i >= 0; --i) t = fmaf(t, y, tanh_coef<6>(i));
    t *= u;
  }
  return t * out;
}
// out tanh(x in) + add of two numbers within reach.  With three or four coefficients the factors are folded into them (N + 1 operations a pair); where the
// powers of `in` leave the range of fp32 (near_reach: -1) it does not serve.  With more, u is made first.
template <int N>
struct ShapedCapNear {
  uint64_t c[N], in2;
  __device__ __forceinline__ ShapedCapNear(float in, float out, float in_out) {
    float f = N <= 4 ? in_out : out;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      c[k] = f2_pair(f * tanh_coef<N>(k), f * tanh_coef<N>(k));
      if (N <= 4) f *= in * in;
    }
    in2 = f2_pair(in, in);
  }
  __device__ __forceinline__ uint64_t operator()(uint64_t x, uint64_t add) const {
    const uint64_t u = N <= 4 ? x : f2_mul(x, in2), y = f2_mul(u, u);
    uint64_t t = f2_fma(c[N - 1], y, c[N - 2]);
#pragma unroll
    for (int k = N - 3; k >= 0; --k) t = f2_fma(t, y, c[k]);
    return f2_fma(t, u, add);
  }
};

}  // namespace smc
