// Attention of single tokens, or a few of each sequence, over the paged cache with capped, distance-biased or interval-masked scores
// (shaped.cuh), and the weight that every cached token collects in it.
//
// What bounds it is the cache: 4 D bytes per key and KV head, read once.  The keys of all sequences, cut into tiles of 64, are one line of
// work per KV head that W workers share in equal parts, wherever sequences begin and end: a batch of ragged contexts keeps every SM busy to the
// end, and a single sequence is spread over all of them.  A CTA gathers its tiles page by page with cp.async, three of them in flight, and
// its warps take 16 keys each (mma.sync: a tile of a dozen rows is short against the gather, and the tensor memory's 128 lanes would stay
// empty).  Where a sequence ends inside a worker's part its state goes to the workspace, and the worker that comes last joins the
// parts of a (sequence, KV head) in the order of its keys, so that results do not depend on the order of arrival.
//
// With ``mass`` the scores of all (row, key) pairs stay in the workspace (4 E G bytes per key and KV head, against 4 D of the cache), and a second
// kernel adds up exp(x - lse) over the rows of each key.  One thread owns a key, so no atomics are needed there either.
#include "shaped.cuh"

namespace smc {

// Registers of 384 threads, 168 each at the start: the loaders leave theirs to the warps that hold outputs.
constexpr int ST_FEW = 40, ST_MANY = 232;
static_assert(128 * ST_FEW + 256 * ST_MANY <= 384 * 168, "the registers of the launch");
constexpr int ST_K = 64, ST_MAX_BS = 1024, ST_LOADERS = 4;
constexpr int ST_COUNTERS = 32768;                     // at the front of every workspace, whatever batch it serves next

struct ShapedStepParams {
  ShapedCache c;
  const __nv_bfloat16* q;        // [bs * E] rows of Hq * D, ld_q apart
  const __nv_bfloat16* k_pool;
  const __nv_bfloat16* v_pool;
  const int* rows;               // [bs] block-table rows
  const int* lens;               // [bs] cached tokens, the new ones included
  __nv_bfloat16* out;
  float* lse;                    // [bs * E, Hq] or null
  float* mass;                   // [bt_rows, Hkv, mass_stride] or null
  // workspace
  int* counters;                 // [row blocks][bs][Hkv], zero between calls
  float* parts;                  // [W][2][Hkv][E G][D + 2]
  float* lse2;                   // [bs * E, Hq] in base 2, +inf where nothing is visible
  float* scores;                 // [Hkv][score_tiles][E G][64]
  long long ld_q, ld_out, mass_stride, score_tiles;
  int bs, E, Hq, Hkv, workers, pdl;
  int* status;
};

// Run of keys [begin, begin + n) of a sequence that any of its tokens may see; with listed positions an outer bound of it: positions are
// distinct, so tokens lie at least as far apart in position as in the row.
struct StepKeys { int row, len, begin, n; };

__device__ __forceinline__ StepKeys step_keys(const ShapedStepParams& p, int s) {
  StepKeys k;
  k.row = p.rows[s];
  k.len = p.lens[s];
  if (k.row < 0 || k.row >= p.c.bt_rows || k.len < 0 || k.len > p.c.bt_stride) {
    atomicOr(p.status, SMC_ERR_BOUNDS);
    k.row = k.len = 0;
  }
  int lo = 0, hi = k.len;
  if (p.c.bounds != nullptr) {
    lo = k.len;
    hi = 0;
    for (int e = 0; e < p.E; ++e) {
      const int idx = k.len - p.E + e;
      if (idx < 0) continue;
      const int pos = p.c.key_pos != nullptr ? p.c.key_pos[(size_t)k.row * p.c.kp_stride + idx] : idx;
      const int2 b = shaped_bounds(p.c, s * p.E + e, pos);
      if (b.x > b.y) continue;
      lo = min(lo, p.c.key_pos == nullptr ? b.x : max(0, b.x <= pos ? idx - (pos - b.x) : idx));
      hi = max(hi, p.c.key_pos == nullptr ? b.y + 1 : b.y >= pos ? idx + 1 + min(b.y - pos, k.len) : min(idx, b.y + 1));
    }
    lo = min(lo, k.len);
    hi = min(hi, k.len);
  }
  k.begin = lo;
  k.n = max(0, hi - lo);
  return k;
}

// first tile of worker w
__device__ __forceinline__ int step_first(int w, int workers, int total) { return (int)((long long)w * total / workers); }
// the worker that has tile x
__device__ __forceinline__ int step_owner(int x, int workers, int total) { return (int)((((long long)x + 1) * workers - 1) / total); }

__device__ __forceinline__ void st_cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void st_cp4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void st_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void st_ldsm(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void st_ldsm_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t st_pack(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Prefix sums of the tiles of all sequences into tiles[0 .. bs], by the whole block.
__device__ __forceinline__ void step_schedule(const ShapedStepParams& p, int* tiles, int* warp_sum) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  int base = 0;
  for (int s0 = 0; s0 < p.bs; s0 += blockDim.x) {
    const int s = s0 + threadIdx.x;
    int sum = s < p.bs ? (step_keys(p, s).n + ST_K - 1) / ST_K : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    if (lane == 31) warp_sum[warp] = sum;
    __syncthreads();
    int all = base;
    for (int w = 0; w < warps; ++w) {
      if (w < warp) sum += warp_sum[w];
      all += warp_sum[w];
    }
    if (s < p.bs) tiles[s + 1] = base + sum;
    base = all;
    __syncthreads();
  }
  if (threadIdx.x == 0) tiles[0] = 0;
  __syncthreads();
}

// sequence of tile x (the last s with tiles[s] <= x)
__device__ __forceinline__ int step_sequence(const int* tiles, int bs, int x) {
  int lo = 0, hi = bs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tiles[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

template <int D, int MT>
struct StCfg {
  // consumers: row tiles of 16 x four groups of 16 keys, twice (tiles in turn) where that makes eight warps
  static constexpr int TURNS = MT == 1 ? 2 : 1, GROUPS = 4 * TURNS, WARPS = GROUPS * MT, THREADS = (WARPS + ST_LOADERS) * 32;
  static constexpr int LD = D + 8;
  static constexpr int STAGES = D == 64 ? 8 : D == 128 ? 5 : MT == 1 ? 3 : 2;
  static constexpr size_t KV = (size_t)ST_K * LD * 2;                // one of K, V
  // stages, a state of [16 MT][D + 4] for the join, positions of the tiles in flight, prefix sums
  static constexpr size_t SMEM = STAGES * 2 * KV + (size_t)16 * MT * (D + 4) * 4 + (size_t)STAGES * ST_K * 4 + (ST_MAX_BS + 1 + 64) * 4;
};

// A place in the line of tiles: the sequence that tile x belongs to.
struct StepCursor {
  int s, seq0, seq1;
  StepKeys key;
  __device__ __forceinline__ void seek(const ShapedStepParams& p, const int* tiles, int x) {
    s = step_sequence(tiles, p.bs, x);
    seq0 = tiles[s];
    seq1 = tiles[s + 1];
    key = step_keys(p, s);
  }
};

struct StShared {
  uint64_t full[8], empty[8];
  int last;
  volatile int abort;
};

__device__ __forceinline__ bool st_wait(StShared& S, int* status, uint64_t* bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  for (;;) {
    for (int i = 0; i < 64; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (S.abort) return false;
    if (clock64() - t0 > SMC_SPIN_CYCLES) {
      atomicOr(status, SMC_ERR_BARRIER_TIMEOUT);
      S.abort = 1;
      return false;
    }
  }
}

template <int D, int MT>
__global__ void __launch_bounds__(StCfg<D, MT>::THREADS, 1) shaped_step_kernel(const ShapedStepParams p) {
  using Cfg = StCfg<D, MT>;
  constexpr int LD = Cfg::LD, STAGES = Cfg::STAGES, THREADS = Cfg::WARPS * 32, CPR = D / 8;
  extern __shared__ __align__(128) uint8_t st_smem[];
  __nv_bfloat16* kv_s = reinterpret_cast<__nv_bfloat16*>(st_smem);   // [stage][K, V][64][LD]
  float* join = reinterpret_cast<float*>(st_smem + STAGES * 2 * Cfg::KV);            // [16 MT][D + 4]
  int* pos_s = reinterpret_cast<int*>(join + 16 * MT * (D + 4));     // [stage][64]
  int* tiles = pos_s + STAGES * ST_K;                                // [bs + 1]
  int* misc = tiles + ST_MAX_BS + 1;                                 // [64]
  __shared__ float ml_s[Cfg::GROUPS][16 * MT][2];
  __shared__ StShared S;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c4 = lane & 3;
  // rows r = token * G + head of this CTA: [m0, M)
  const int G = p.Hq / p.Hkv, m0 = blockIdx.z * 16 * MT, rows_all = p.E * G, M = min(rows_all, m0 + 16 * MT), kvh = blockIdx.y, w = blockIdx.x;
  int* counter = p.counters + ((size_t)blockIdx.z * p.bs) * p.Hkv + kvh;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&S.full[i], ST_LOADERS * 32);
      mbar_init(&S.empty[i], 4 * MT);
    }
    S.abort = 0;
    fence_barrier_init();
  }
  if (p.pdl) { pdl_launch_dependents(); pdl_wait_prior_grid(); }
  step_schedule(p, tiles, misc);
  const int total = tiles[p.bs];
  // sequences without a tile have nobody else to write their rows
  if (w == 0) {
    for (int s = warp; s < p.bs; s += Cfg::THREADS / 32) {
      if (tiles[s + 1] > tiles[s]) continue;
      for (int x = m0 * D + lane; x < M * D; x += 32) {
        const int e = x / (G * D), hd = x - e * G * D;
        p.out[(size_t)(s * p.E + e) * p.ld_out + (size_t)kvh * G * D + hd] = __float2bfloat16(0.f);
      }
      for (int x = m0 + lane; x < M; x += 32) {
        const size_t at = (size_t)(s * p.E + x / G) * p.Hq + kvh * G + x % G;
        if (p.lse != nullptr) p.lse[at] = -INFINITY;
        if (p.scores != nullptr) p.lse2[at] = INFINITY;
      }
    }
  }
  const int W = min(p.workers, total);                               // each of them has a tile
  if (w >= W) return;
  const int t_begin = step_first(w, W, total), t_end = step_first(w + 1, W, total);

  if (warp >= Cfg::WARPS) {
    if constexpr (D == 256) regs_fewer<ST_FEW>();
    // ================================================================= loaders: 16 keys of each tile a warp
    const int lw = warp - Cfg::WARPS, kl0 = lw * 16 + (lane & 15);
    const size_t kv_row = (size_t)p.Hkv * D;
    constexpr int AHEAD = 3;                                         // tiles that page ids are read ahead
    StepCursor cur;
    cur.seq1 = t_begin;
    int page[AHEAD], from[AHEAD];                                    // of this lane's key: page, index of its position or -1
    auto ids = [&](int x, int& pg, int& at) {
      if (x >= t_end) return;
      if (x >= cur.seq1) cur.seek(p, tiles, x);
      const int i = (x - cur.seq0) * ST_K + kl0, idx = cur.key.begin + min(i, cur.key.n - 1);       // keys behind the last repeat it
      pg = p.c.block_table[(size_t)cur.key.row * p.c.bt_stride + idx];
      at = cur.key.row * p.c.kp_stride + idx;
    };
#pragma unroll
    for (int d = 0; d < AHEAD; ++d) ids(t_begin + d, page[d], from[d]);
    for (int x0 = t_begin; x0 < t_end; x0 += AHEAD) {
#pragma unroll
      for (int d = 0; d < AHEAD; ++d) {
        const int x = x0 + d, n = x - t_begin, st = n % STAGES;
        if (x >= t_end) break;
        int pg = page[d];
        const int at = from[d];
        if (pg < 0 || pg > p.c.n_pages) { atomicOr(p.status, SMC_ERR_BOUNDS); pg = 0; }
        ids(x + AHEAD, page[d], from[d]);
        const bool ok = n < STAGES || st_wait(S, p.status, &S.empty[st], (uint32_t)(n / STAGES - 1) & 1u);
        if (!__all_sync(0xffffffffu, ok)) { x0 = t_end; break; }
        const uint32_t k0 = smem_u32(kv_s + (size_t)st * 2 * ST_K * LD);
#pragma unroll 8
        for (int i = lane; i < 16 * CPR; i += 32) {
          const int kl = i / CPR, c = i - kl * CPR;
          const size_t src = (size_t)__shfl_sync(0xffffffffu, pg, kl) * kv_row + (size_t)kvh * D + c * 8;
          const uint32_t dst = k0 + (uint32_t)((lw * 16 + kl) * LD + c * 8) * 2;
          st_cp16(dst, p.k_pool + src);
          st_cp16(dst + (uint32_t)Cfg::KV, p.v_pool + src);
        }
        if (p.c.key_pos != nullptr && lane < 16) st_cp4(smem_u32(pos_s + st * ST_K + kl0), p.c.key_pos + at);
        asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_u32(&S.full[st])) : "memory");       // when all of them have landed
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    return;
  }

  if constexpr (D == 256) regs_more<ST_MANY>();
  const int mt = warp % MT, gi = warp / MT, kg = gi & 3, turn = gi >> 2;             // row tile, group; of it keys and turn
  const float mul = p.c.scale * SH_LOG2E, cap_in = p.c.cap > 0.f ? p.c.scale / p.c.cap : 0.f, cap_out = p.c.cap * SH_LOG2E;
  bool alive = true;
  int x = t_begin;
  while (x < t_end) {
    // ---------------------------------------------------------------- one sequence's tiles of this worker
    const int s = step_sequence(tiles, p.bs, x), seq0 = tiles[s], seq1 = tiles[s + 1], x_end = min(t_end, seq1);
    const StepKeys key = step_keys(p, s);
    uint32_t qa[D / 16][4];
    {
      const int r0 = m0 + mt * 16 + g, r1 = r0 + 8;
      const __nv_bfloat16* q0 = p.q + (size_t)(s * p.E + r0 / G) * p.ld_q + (size_t)(kvh * G + r0 % G) * D + 2 * c4;
      const __nv_bfloat16* q1 = p.q + (size_t)(s * p.E + r1 / G) * p.ld_q + (size_t)(kvh * G + r1 % G) * D + 2 * c4;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        qa[kk][0] = r0 < M ? *reinterpret_cast<const uint32_t*>(q0 + kk * 16) : 0u;
        qa[kk][1] = r1 < M ? *reinterpret_cast<const uint32_t*>(q1 + kk * 16) : 0u;
        qa[kk][2] = r0 < M ? *reinterpret_cast<const uint32_t*>(q0 + kk * 16 + 8) : 0u;
        qa[kk][3] = r1 < M ? *reinterpret_cast<const uint32_t*>(q1 + kk * 16 + 8) : 0u;
      }
    }
    int2 see[2];
    int own_pos[2];
    float slope[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = m0 + mt * 16 + g + 8 * i, e = r / G, idx = key.len - p.E + e;
      own_pos[i] = 0;
      see[i] = make_int2(SH_POS_END, -1);
      slope[i] = 0.f;
      if (r < M && idx >= 0) {
        own_pos[i] = p.c.key_pos != nullptr ? p.c.key_pos[(size_t)key.row * p.c.kp_stride + idx] : idx;
        see[i] = shaped_bounds(p.c, s * p.E + e, own_pos[i]);
        if (p.c.slopes != nullptr) slope[i] = -p.c.slopes[kvh * G + r % G] * SH_LOG2E;
      }
    }
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;

    for (; x < x_end; ++x) {
      const int nth = x - t_begin, st = nth % STAGES;
      if (Cfg::TURNS > 1 && nth % Cfg::TURNS != turn) continue;
      if (alive) alive = __all_sync(0xffffffffu, st_wait(S, p.status, &S.full[st], (uint32_t)(nth / STAGES) & 1u));
      if (!alive) continue;
      const __nv_bfloat16* Kt = kv_s + (size_t)st * 2 * ST_K * LD + kg * 16 * LD;
      const __nv_bfloat16* Vt = Kt + ST_K * LD;
      float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}, sd[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      // matrices of a K fragment: keys 0-7 dims 0-7, keys 0-7 dims 8-15, keys 8-15 dims 0-7, keys 8-15 dims 8-15
      const uint32_t ka = smem_u32(Kt + ((lane & 7) + (lane >> 4) * 8) * LD + ((lane >> 3) & 1) * 8);
#pragma unroll
      for (int kk = 0; kk < D / 16; kk += 2) {                       // two chains of products
        uint32_t b[4], d[4];
        st_ldsm(b, ka + kk * 32);
        st_ldsm(d, ka + kk * 32 + 32);
        st_mma(sc[0], qa[kk], b[0], b[1]);
        st_mma(sc[1], qa[kk], b[2], b[3]);
        st_mma(sd[0], qa[kk + 1], d[0], d[1]);
        st_mma(sd[1], qa[kk + 1], d[2], d[3]);
      }
      const int i0 = (x - seq0) * ST_K + kg * 16;                    // of the sequence's visible keys
      float top[2] = {m[0], m[1]};
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int col = n * 8 + 2 * c4 + (i & 1), r = i >> 1;
          int kp = p.c.key_pos != nullptr ? pos_s[st * ST_K + kg * 16 + col] : key.begin + i0 + col;
          kp = i0 + col < key.n ? kp : -1;
          float v = sc[n][i] + sd[n][i];
          v = p.c.cap > 0.f ? shaped_cap(v, cap_in, cap_out) : v * mul;
          v = fmaf(slope[r], fabsf((float)(kp - own_pos[r])), v);
          v = kp >= see[r].x && kp <= see[r].y ? v : -INFINITY;
          sc[n][i] = v;
          top[r] = fmaxf(top[r], v);
        }
      if (p.scores != nullptr && x < p.score_tiles) {
        float* at = p.scores + (((size_t)kvh * p.score_tiles + x) * rows_all + m0 + mt * 16 + g) * ST_K + kg * 16 + 2 * c4;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          if (m0 + mt * 16 + g < M) *reinterpret_cast<float2*>(at + n * 8) = make_float2(sc[n][0], sc[n][1]);
          if (m0 + mt * 16 + g + 8 < M) *reinterpret_cast<float2*>(at + 8 * ST_K + n * 8) = make_float2(sc[n][2], sc[n][3]);
        }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
      }
      if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float alpha = top[r] == -INFINITY ? 1.f : shaped_ex2(m[r] - top[r]);
          m[r] = top[r];
          l[r] *= alpha;
#pragma unroll
          for (int n = 0; n < D / 8; ++n) { o[n][2 * r] *= alpha; o[n][2 * r + 1] *= alpha; }
        }
      }
      float pr[2][4];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = i >> 1;
          pr[n][i] = m[r] == -INFINITY ? 0.f : shaped_ex2(sc[n][i] - m[r]);
          l[r] += pr[n][i];
        }
      const uint32_t pa[4] = {st_pack(pr[0][0], pr[0][1]), st_pack(pr[0][2], pr[0][3]), st_pack(pr[1][0], pr[1][1]), st_pack(pr[1][2], pr[1][3])};
      // matrices of a V fragment: keys 0-7 dims 0-7, keys 8-15 dims 0-7, keys 0-7 dims 8-15, keys 8-15 dims 8-15
      const uint32_t va = smem_u32(Vt + (lane & 15) * LD + (lane >> 4) * 8);
#pragma unroll
      for (int n = 0; n < D / 16; ++n) {
        uint32_t b[4];
        st_ldsm_t(b, va + n * 32);
        st_mma(o[2 * n], pa, b[0], b[1]);
        st_mma(o[2 * n + 1], pa, b[2], b[3]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&S.empty[st]);
    }
    // ---------------------------------------------------------------- the groups of keys, joined one after the other
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (c4 == 0) {
        ml_s[gi][mt * 16 + g + 8 * r][0] = m[r];
        ml_s[gi][mt * 16 + g + 8 * r][1] = l[r];
      }
    }
    named_bar(1, THREADS);
    float top[2], sum[2], mine[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = mt * 16 + g + 8 * r;
      top[r] = ml_s[0][row][0];
#pragma unroll
      for (int k = 1; k < Cfg::GROUPS; ++k) top[r] = fmaxf(top[r], ml_s[k][row][0]);
      sum[r] = 0.f;
#pragma unroll
      for (int k = 0; k < Cfg::GROUPS; ++k) sum[r] += top[r] == -INFINITY ? 0.f : ml_s[k][row][1] * shaped_ex2(ml_s[k][row][0] - top[r]);
      mine[r] = top[r] == -INFINITY ? 0.f : shaped_ex2(m[r] - top[r]);
    }
    for (int k = 0; k < Cfg::GROUPS; ++k) {
      if (gi == k) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float* at = join + (mt * 16 + g + 8 * r) * (D + 4);
#pragma unroll
          for (int n = 0; n < D / 8; ++n) {
            float2* cell = reinterpret_cast<float2*>(at + n * 8 + 2 * c4);
            const float2 before = k == 0 ? make_float2(0.f, 0.f) : *cell;
            // a row that no key of this group is visible to adds nothing, whatever its values are
            *cell = mine[r] == 0.f ? before : make_float2(before.x + o[n][2 * r] * mine[r], before.y + o[n][2 * r + 1] * mine[r]);
          }
          if (k == Cfg::GROUPS - 1 && c4 == 0) { at[D] = top[r]; at[D + 1] = sum[r]; }
        }
      }
      named_bar(1, THREADS);
    }
    const int w_first = step_owner(seq0, W, total), w_last = step_owner(seq1 - 1, W, total), R = M - m0;
    bool finish = w_first == w_last;
    if (!finish) {
      // part of worker v: row r of [rows_all], value n of [D + 2]
      auto part = [&](int v) {
        return p.parts + ((((size_t)v * 2 + (step_first(v, W, total) >= seq0 ? 0 : 1)) * p.Hkv + kvh) * rows_all + m0) * (D + 2);
      };
      float* to = part(w);
      for (int i = threadIdx.x; i < R * (D + 2); i += THREADS) to[i] = join[i / (D + 2) * (D + 4) + i % (D + 2)];
      __threadfence();
      named_bar(1, THREADS);
      if (threadIdx.x == 0) {
        const int n = w_last - w_first + 1;
        S.last = atomicAdd(counter + s * p.Hkv, 1) == n - 1;
        if (S.last) counter[s * p.Hkv] = 0;
        __threadfence();
      }
      named_bar(1, THREADS);
      finish = S.last != 0;
      if (finish) {                                                  // all parts are there
        for (int r = warp; r < R; r += Cfg::WARPS) {                 // a warp per row
          float big = -INFINITY;
          for (int v = w_first + lane; v <= w_last; v += 32) big = fmaxf(big, __ldcg(part(v) + r * (D + 2) + D));
          big = warp_max(big);
          float acc[D / 32], den = 0.f;
#pragma unroll
          for (int n = 0; n < D / 32; ++n) acc[n] = 0.f;
          for (int v = w_first; v <= w_last; ++v) {
            const float* from = part(v) + r * (D + 2);
            const float pm = __ldcg(from + D), f = pm == -INFINITY ? 0.f : shaped_ex2(pm - big);
            den += f == 0.f ? 0.f : __ldcg(from + D + 1) * f;
#pragma unroll
            for (int n = 0; n < D / 32; ++n) acc[n] += f == 0.f ? 0.f : __ldcg(from + n * 32 + lane) * f;
          }
          float* at = join + r * (D + 4);
#pragma unroll
          for (int n = 0; n < D / 32; ++n) at[n * 32 + lane] = acc[n];
          if (lane == 0) { at[D] = big; at[D + 1] = den; }
        }
        named_bar(1, THREADS);
      }
    }
    if (finish) {
      for (int i = threadIdx.x; i < R * (D / 2); i += THREADS) {
        const int lr = i / (D / 2), r = m0 + lr, d = (i - lr * (D / 2)) * 2;
        const float* at = join + lr * (D + 4);
        const bool none = at[D] == -INFINITY && at[D + 1] == 0.f;
        const float inv = 1.f / at[D + 1];
        *reinterpret_cast<uint32_t*>(p.out + (size_t)(s * p.E + r / G) * p.ld_out + (size_t)(kvh * G + r % G) * D + d) =
            none ? 0u : st_pack(at[d] * inv, at[d + 1] * inv);
      }
      if (p.lse != nullptr || p.scores != nullptr)
        for (int lr = threadIdx.x; lr < R; lr += THREADS) {
          const float* at = join + lr * (D + 4);
          const int r = m0 + lr;
          const bool none = at[D] == -INFINITY && at[D + 1] == 0.f;
          const float v = at[D] + __log2f(at[D + 1]);
          const size_t to = (size_t)(s * p.E + r / G) * p.Hq + kvh * G + r % G;
          if (p.lse != nullptr) p.lse[to] = none ? -INFINITY : SH_LN2 * v;
          if (p.scores != nullptr) p.lse2[to] = none ? INFINITY : v;
        }
    }
    named_bar(1, THREADS);                                                 // `join` is free for the next sequence
  }
}

// mass[row, kvh, j] += sum over the rows of exp2(score - lse)
__global__ void __launch_bounds__(256) shaped_step_mass_kernel(const ShapedStepParams p) {
  extern __shared__ int sm_tiles[];                                  // [bs + 1 + 32]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kvh = blockIdx.y, G = p.Hq / p.Hkv, M = p.E * G;
  pdl_wait_prior_grid();
  step_schedule(p, sm_tiles, sm_tiles + p.bs + 1);
  const int total = sm_tiles[p.bs];
  if (total > p.score_tiles) {                                       // the workspace is too small for these contexts
    if (threadIdx.x == 0 && blockIdx.x == 0) atomicOr(p.status, SMC_ERR_BOUNDS);
    return;
  }
  for (int x = blockIdx.x * 8 + warp; x < total; x += gridDim.x * 8) {
    const int s = step_sequence(sm_tiles, p.bs, x);
    const StepKeys k = step_keys(p, s);
    bool twice = false;                                              // a row listed twice would be added to by two warps at once
    for (int o = lane; o < s; o += 32) twice |= p.rows[o] == k.row && p.lens[o] > 0;
    if (__any_sync(0xffffffffu, twice)) {
      if (lane == 0) atomicOr(p.status, SMC_ERR_BOUNDS);
      continue;
    }
    const int i = (x - sm_tiles[s]) * ST_K + 2 * lane;
    const float* sc = p.scores + ((size_t)kvh * p.score_tiles + x) * M * ST_K + 2 * lane;
    float a = 0.f, b = 0.f;
    for (int r = 0; r < M; ++r) {
      const float top = p.lse2[(size_t)(s * p.E + r / G) * p.Hq + kvh * G + r % G];
      const float2 v = *reinterpret_cast<const float2*>(sc + (size_t)r * ST_K);
      a += shaped_ex2(v.x - top);
      b += shaped_ex2(v.y - top);
    }
    float* to = p.mass + ((size_t)k.row * p.Hkv + kvh) * p.mass_stride + k.begin + i;
    if (i < k.n) to[0] += a;
    if (i + 1 < k.n) to[1] += b;
  }
}

// Parts of the workspace, each from a 256-byte border.
struct StepWork { size_t parts, lse2, scores, bytes; long long score_tiles, counted; int workers; };

// Row tiles of a CTA: a warp's registers hold 16 rows of outputs; more than 32 rows go to further CTAs, which find the keys in L2.
static int step_row_tiles(int M) { return M <= 16 ? 1 : 2; }

static StepWork step_work(int bs, int E, int Hq, int Hkv, int D, long long keys) {
  StepWork w;
  const int M = E * (Hq / Hkv), mt = step_row_tiles(M), blocks = (M + 16 * mt - 1) / (16 * mt);
  w.workers = 148 / (Hkv * blocks) > 0 ? 148 / (Hkv * blocks) : 1;  // a CTA per SM
  w.score_tiles = keys > 0 ? keys / ST_K + bs : 0;                   // every sequence may end inside a tile
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  w.counted = (long long)bs * Hkv * blocks;
  w.parts = (size_t)ST_COUNTERS * 4;
  w.lse2 = w.parts + up((size_t)w.workers * 2 * Hkv * M * (D + 2) * 4);
  w.scores = w.lse2 + up((size_t)bs * E * Hq * 4);
  w.bytes = w.scores + up((size_t)Hkv * w.score_tiles * M * ST_K * 4);
  return w;
}

template <int D, int MT>
static int launch_shaped_step(const ShapedStepParams& p, cudaStream_t st) {
  using Cfg = StCfg<D, MT>;
  static_assert(Cfg::SMEM + Cfg::GROUPS * 16 * MT * 8 + sizeof(StShared) <= 232448, "shared memory");
  CUDA_CHECK_RET(cudaFuncSetAttribute(shaped_step_kernel<D, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg::SMEM));
  if constexpr (D == 256) {                           // what the warps ask for later is there from the start
    static const int regs = [] { cudaFuncAttributes a; return cudaFuncGetAttributes(&a, shaped_step_kernel<D, MT>) == cudaSuccess ? a.numRegs : 0; }();
    if (regs < 168) return -155;
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.workers, (unsigned)p.Hkv, (unsigned)((p.E * (p.Hq / p.Hkv) + 16 * MT - 1) / (16 * MT)));
  cfg.blockDim = dim3(Cfg::THREADS);
  cfg.dynamicSmemBytes = Cfg::SMEM;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = p.pdl ? 1 : 0;
  CUDA_CHECK_RET(cudaLaunchKernelEx(&cfg, shaped_step_kernel<D, MT>, p));
  if (p.mass == nullptr) return 0;
  cfg.gridDim = dim3((unsigned)((296 + p.Hkv - 1) / p.Hkv), (unsigned)p.Hkv);
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = (size_t)(p.bs + 1 + 32) * 4;
  cfg.numAttrs = 1;
  CUDA_CHECK_RET(cudaLaunchKernelEx(&cfg, shaped_step_mass_kernel, p));
  return 0;
}

}  // namespace smc

// Bytes of workspace for steps of bs sequences of E tokens; keys > 0: with the mass, of that many cached tokens in all.
SMC_API long long smc_shaped_step_work(int bs, int E, int Hq, int Hkv, int D, long long keys) {
  if (bs < 1 || E < 1 || Hkv < 1 || Hq < Hkv || Hq % Hkv || E > 64 || Hq / Hkv > 64 / E || (D != 64 && D != 128 && D != 256)) return -1;
  const smc::StepWork w = smc::step_work(bs, E, Hq, Hkv, D, keys);
  return bs > smc::ST_MAX_BS || w.counted > smc::ST_COUNTERS ? -1 : (long long)w.bytes;
}

// q, out: bs * E rows of Hq * D bf16 values, the E tokens of a sequence are the last of its lens[s] cached ones (rows [bs], lens [bs] int32).
// work: zeros at first, smc_shaped_step_work bytes or more; with the mass it has to hold the scores of all cached tokens of the batch.  mass [bt_rows, Hkv, mass_stride] fp32 or null.
SMC_API int smc_shaped_step(const void* q, long long ld_q, const void* k_pool, const void* v_pool, int n_pages, const int* block_table,
                            int bt_stride, int bt_rows, const int* key_pos, int kp_stride, const int* rows, const int* lens, void* out,
                            long long ld_out, float* lse, float* mass, long long mass_stride, int bs, int E, int Hq, int Hkv, int D,
                            float scale, float cap, const float* slopes, const int* bounds, void* work, long long work_bytes,
                            int* status, int pdl, cudaStream_t st) {
  using namespace smc;
  if (bs <= 0) return 0;
  if (smc_shaped_step_work(bs, E, Hq, Hkv, D, 0) < 0) return -150;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 3 || (ld_q & 1) || (ld_out & 1) ||
      ((reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool)) & 15) || (reinterpret_cast<uintptr_t>(work) & 15) ||
      (reinterpret_cast<uintptr_t>(bounds) & 7))
    return -151;
  if (!(cap >= 0.f) || cap > 3e38f || !(scale > 0.f) || scale > 3e38f) return -152;
  if (mass != nullptr && mass_stride < bt_stride) return -153;
  StepWork w = step_work(bs, E, Hq, Hkv, D, 0);
  if (mass != nullptr) w.score_tiles = (work_bytes - (long long)w.scores) / ((long long)Hq * E * ST_K * 4);       // the rest of it
  if (work_bytes < (long long)w.bytes || (mass != nullptr && w.score_tiles < 1)) return -154;
  ShapedStepParams p;
  p.c = ShapedCache{block_table, key_pos, (const int2*)bounds, slopes, bt_stride, bt_rows, kp_stride, n_pages, scale, cap};
  p.q = (const __nv_bfloat16*)q; p.k_pool = (const __nv_bfloat16*)k_pool; p.v_pool = (const __nv_bfloat16*)v_pool;
  p.rows = rows; p.lens = lens; p.out = (__nv_bfloat16*)out; p.lse = lse; p.mass = mass;
  char* base = (char*)work;
  p.counters = (int*)base; p.parts = (float*)(base + w.parts); p.lse2 = (float*)(base + w.lse2);
  p.scores = mass != nullptr ? (float*)(base + w.scores) : nullptr;
  p.ld_q = ld_q; p.ld_out = ld_out; p.mass_stride = mass_stride; p.score_tiles = w.score_tiles;
  p.bs = bs; p.E = E; p.Hq = Hq; p.Hkv = Hkv; p.workers = w.workers; p.pdl = pdl; p.status = status;
  const int mt = step_row_tiles(E * (Hq / Hkv));
#define SMC_SHAPED_STEP(DD)                                      \
  if (D == DD) {                                                 \
    if (mt == 1) return launch_shaped_step<DD, 1>(p, st);        \
    return launch_shaped_step<DD, 2>(p, st);                     \
  }
  SMC_SHAPED_STEP(64)
  SMC_SHAPED_STEP(128)
  SMC_SHAPED_STEP(256)
#undef SMC_SHAPED_STEP
  return -150;
}
