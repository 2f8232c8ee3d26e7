// Attention of single tokens, or a few of each sequence, over the paged cache with capped, distance-biased or interval-masked scores
// (shaped.cuh), and the weight that every cached token collects in it.
//
// What bounds it is the cache: 4 D bytes per key and KV head, read once.  The keys of all sequences, cut into tiles of 64 (128 with D = 64), are one line of
// work per KV head that W workers share in equal parts, wherever sequences begin and end: a batch of ragged contexts keeps every SM busy to the
// end, and a single sequence is spread over all of them.  Four loader warps gather the tiles page by page with cp.async into a ring; the other
// warps take 16 keys each, two tiles in turn, and come to the loaders' ring only through its barriers.
//
// Keys are the rows of the products (mma.sync, 16 x 8 x 16) and queries their eight columns: S^T = K Q^T and O^T += V^T P^T, so that the
// four or eight heads of a group fill a fragment (as rows of sixteen they left half of every product and of the softmax idle: heads of 256, 4 x 57,600 keys
// 110 -> 96 us).  tcgen05 has no such narrow form: with keys in its 128 lanes the softmax would run across lanes, with queries there most of them would be empty.  From 17 rows
// on the products cost more than the cache: 36 rows (nine tokens of groups of four) take 2.7 times as long as four on the same keys.
//
// Microseconds on B200 (device times, graphs replayed; of them at the measured 6.54 TB/s): 4 x 57,600 keys, 8 KV heads of 128, groups of four: 156 (145); of 64: 91 (72); 2 heads of
// 256: 83 (72); with the mass, 48 sequences of 600 to 9000 keys: 190 (147), two of 99,000 and 131,000: 184 (147); a window of 2048 over the 48, thinned out, without the mass:
// 42 (19); one sequence of 701 keys, heads of 64: 9.3, a launch, three dependent reads and a join.  Rows of 512 bytes as bulk copies 96 -> 87, the cache's lines first out of L2 157 -> 154 and 196 -> 190 with the mass.
//
// Where a sequence ends inside a worker's part its state goes to the workspace, and the worker that comes last joins the
// parts of a (sequence, KV head) in the order of its keys, so that results do not depend on the order of arrival.
//
// With ``mass`` the scores of all (row, key) pairs stay in the workspace (4 E G bytes per key and KV head, against 4 D of the cache), and a second
// kernel adds up exp(x - lse) over the rows of each key.  One thread owns a key, so no atomics are needed there either.
#include "shaped.cuh"

namespace smc {

// Registers of 384 threads, 168 each at the start: the loaders leave theirs to the warps that hold outputs.
constexpr int ST_FEW = 40, ST_MANY = 232;
static_assert(128 * ST_FEW + 256 * ST_MANY <= 384 * 168, "the registers of the launch");
constexpr int ST_MAX_BS = 1024, ST_LOADERS = 4;
// Keys of a tile: what a loader warp does besides copying comes once a tile, and 64 keys of 128 bytes were too few to hide it (4 x 57,600 keys of 8 heads of 64:
// 108 us with tiles of 64 keys, 93 with 128).
constexpr int step_tile(int D) { return D == 64 ? 128 : 64; }
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
  float* parts;                  // [W][2][Hkv][E G][D + 4]
  float* lse2;                   // [bs * E, Hq] in base 2, +inf where nothing is visible
  float* scores;                 // [Hkv][score_tiles][tile][pitch], pitch E G rounded up to 4
  long long ld_q, ld_out, mass_stride, score_tiles;
  int bs, E, Hq, Hkv, workers, tile, pdl;
  int* status;
};

// Run of keys [begin, begin + n) of a sequence between the first and the last one that any of its tokens sees.
struct StepKeys { int row, len, begin, n; };

// What the schedule leaves in shared memory: tiles of the sequences ahead of each, [bs + 1], and where its run begins with the keys of its last tile less one, [bs].
struct StepLine { int* tiles; int* spans; };
constexpr int ST_LAST_BITS = 7;                        // keys of a tile: at most 128; a run begins in front of 2^24

// of a sequence that has a tile
__device__ __forceinline__ StepKeys step_keys(const ShapedStepParams& p, const StepLine& line, int s) {
  const int span = line.spans[s];
  return {p.rows[s], p.lens[s], span >> ST_LAST_BITS, (line.tiles[s + 1] - line.tiles[s] - 1) * p.tile + (span & ((1 << ST_LAST_BITS) - 1)) + 1};
}

// The runs of all sequences, each found by L lanes of a warp: tiles into line.tiles[s + 1], beginnings into line.spans[s].  Listed positions are searched for the ends of the
// intervals, L probes at a time, inside what their distances leave: positions are distinct, so tokens lie at least as far apart in position as in the row.
template <int L, bool SEARCH>
__device__ __forceinline__ void step_spans(const ShapedStepParams& p, const StepLine& line) {
  const int lane = threadIdx.x & 31, sub = lane % L, shift = lane / L * L;
  const unsigned group = L == 32 ? 0xffffffffu : (1u << L) - 1u;
  for (int s0 = 0; s0 < p.bs; s0 += (int)blockDim.x / L) {
    const int s = s0 + (int)threadIdx.x / L;
    int row = 0, len = 0;
    if (s < p.bs) {
      row = p.rows[s];
      len = p.lens[s];
      if (row < 0 || row >= p.c.bt_rows || len < 0 || len > p.c.bt_cols) {
        atomicOr(p.status, SMC_ERR_BOUNDS);
        row = len = 0;
      }
    }
    int lo = 0, hi = len;
    if (p.c.bounds != nullptr) {
      const int* kp = p.c.key_pos != nullptr ? p.c.key_pos + (size_t)row * p.c.kp_stride : nullptr;
      int near = SH_POS_END, far = -1;                 // positions that any token sees
      lo = len;
      hi = 0;
      for (int e = sub; e < p.E; e += L) {
        const int idx = len - p.E + e;
        if (idx < 0) continue;
        const int pos = kp != nullptr ? kp[idx] : idx;
        const int2 b = shaped_bounds(p.c, s * p.E + e, pos);
        if (b.x > b.y) continue;
        near = min(near, b.x);
        far = max(far, b.y);
        lo = min(lo, kp == nullptr ? b.x : max(0, b.x <= pos ? idx - (pos - b.x) : idx));
        hi = max(hi, kp == nullptr ? b.y + 1 : b.y >= pos ? idx + 1 + min(b.y - pos, len) : min(idx, b.y + 1));
      }
#pragma unroll
      for (int o = 1; o < L; o <<= 1) {
        lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        near = min(near, __shfl_xor_sync(0xffffffffu, near, o));
        far = max(far, __shfl_xor_sync(0xffffffffu, far, o));
      }
      lo = min(lo, len);
      hi = max(lo, min(hi, len));
      if constexpr (SEARCH) {
        // first indices of [lo, hi) whose positions are >= near and > far; hi if none
        int a0 = lo, a1 = hi, b0 = lo, b1 = hi;
        while (__any_sync(0xffffffffu, a0 < a1 || b0 < b1)) {
          const int sa = (a1 - a0) / (L + 1) + 1, sb = (b1 - b0) / (L + 1) + 1, at = a0 + (sub + 1) * sa - 1, bt = b0 + (sub + 1) * sb - 1;
          const int ka = __popc(__ballot_sync(0xffffffffu, at < a1 && kp[at] < near) >> shift & group);
          const int kb = __popc(__ballot_sync(0xffffffffu, bt < b1 && kp[bt] <= far) >> shift & group);
          a1 = min(a1, a0 + (ka + 1) * sa - 1);
          b1 = min(b1, b0 + (kb + 1) * sb - 1);
          a0 += ka * sa;
          b0 += kb * sb;
        }
        lo = a0;
        hi = max(a0, b0);
      }
    }
    if (s < p.bs && sub == 0) {
      line.tiles[s + 1] = (hi - lo + p.tile - 1) / p.tile;
      line.spans[s] = lo << ST_LAST_BITS | ((hi - lo + p.tile - 1) % p.tile);
    }
  }
}

// first tile of worker w
__device__ __forceinline__ int step_first(int w, int workers, int total) { return (int)((long long)w * total / workers); }
// the worker that has tile x
__device__ __forceinline__ int step_owner(int x, int workers, int total) { return (int)((((long long)x + 1) * workers - 1) / total); }

__device__ __forceinline__ void st_cp16(uint32_t dst, const void* src, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy) : "memory");
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
// an 8 x 8 matrix of bf16 values, two neighbours of a row per lane, transposed
__device__ __forceinline__ uint32_t st_transpose(uint32_t v) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(v));
  return y;
}
__device__ __forceinline__ uint32_t st_pack(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// The line of all sequences, by the whole block.  A run that has to be searched for takes as many lanes as there are: its probes are dependent reads (300 sequences of up to 500
// tokens by eight lanes each, in seven turns, 45 us a step, by one each 38).
__device__ __forceinline__ void step_schedule(const ShapedStepParams& p, const StepLine& line, int* warp_sum) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (p.c.bounds == nullptr || p.c.key_pos == nullptr) step_spans<1, false>(p, line);
  else if (p.bs <= warps) step_spans<32, true>(p, line);
  else if (p.bs <= warps * 4) step_spans<8, true>(p, line);
  else step_spans<1, true>(p, line);
  __syncthreads();
  int base = 0;
  for (int s0 = 0; s0 < p.bs; s0 += blockDim.x) {
    const int s = s0 + threadIdx.x;
    int sum = s < p.bs ? line.tiles[s + 1] : 0;
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
    if (s < p.bs) line.tiles[s + 1] = base + sum;
    base = all;
    __syncthreads();
  }
  if (threadIdx.x == 0) line.tiles[0] = 0;
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

// A warp takes NQ columns of eight rows, MT warps side by side all rows of the CTA.
template <int D, int NQ, int MT>
struct StCfg {
  static constexpr int ROWS = 8 * NQ * MT;
  // groups of keys in a tile, tiles in turn: eight consumer warps; four with D = 256, whose 16 keys a warp holds while it works are 16 KB
  static constexpr int KT = step_tile(D), TURNS = MT == 1 && D == 128 ? 2 : 1, GW = MT == 1 ? (D == 64 ? 8 : 4) : MT == 2 ? 4 : 2, SUB = KT / 16 / GW;
  static constexpr int GROUPS = GW * TURNS, WARPS = GROUPS * MT, THREADS = (WARPS + ST_LOADERS) * 32;
  static constexpr int LD = D + 8;
  static constexpr int STAGES = D == 64 ? 4 : D == 128 ? 5 : MT == 1 ? 3 : 2;
  // rows of 512 bytes come as one bulk copy each (19 cycles a copy, whatever its size); shorter ones in pieces of 16 bytes
  static constexpr bool BULK = D == 256;
  static constexpr int SLOTS = D == 256 ? (ROWS == 8 ? 2 : 1) : 64 / ROWS;           // states that groups leave at once when they are joined
  static constexpr size_t KV = (size_t)KT * LD * 2;                // one of K, V
  // stages, states, positions of the tiles in flight, the line of tiles
  static constexpr size_t SMEM = STAGES * 2 * KV + (size_t)SLOTS * ROWS * (D + 4) * 4 + (size_t)STAGES * KT * 4 + (2 * ST_MAX_BS + 1 + 64) * 4;
};

// A place in the line of tiles: the sequence that tile x belongs to.
struct StepCursor {
  int s, seq0, seq1;
  StepKeys key;
  __device__ __forceinline__ void seek(const ShapedStepParams& p, const StepLine& line, int x) {
    s = step_sequence(line.tiles, p.bs, x);
    seq0 = line.tiles[s];
    seq1 = line.tiles[s + 1];
    key = step_keys(p, line, s);
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

template <int D, int NQ, int MT>
__global__ void __launch_bounds__(StCfg<D, NQ, MT>::THREADS, 1) shaped_step_kernel(const ShapedStepParams p) {
  using Cfg = StCfg<D, NQ, MT>;
  constexpr int LD = Cfg::LD, KT = Cfg::KT, KW = KT / ST_LOADERS, STAGES = Cfg::STAGES, THREADS = Cfg::WARPS * 32;
  [[maybe_unused]] constexpr int CPR = D / 8;
  extern __shared__ __align__(128) uint8_t st_smem[];
  __nv_bfloat16* kv_s = reinterpret_cast<__nv_bfloat16*>(st_smem);   // [stage][K, V][KT][LD]
  float* join = reinterpret_cast<float*>(st_smem + STAGES * 2 * Cfg::KV);            // [slot][ROWS][D + 4]
  int* pos_s = reinterpret_cast<int*>(join + Cfg::SLOTS * Cfg::ROWS * (D + 4));      // [stage][KT]
  int* tiles = pos_s + STAGES * KT;                                  // [bs + 1]
  const StepLine line{tiles, tiles + ST_MAX_BS + 1};
  int* misc = line.spans + ST_MAX_BS;                                // [64]
  __shared__ float ml_s[Cfg::GROUPS][Cfg::ROWS][2];
  __shared__ float4 row_s[Cfg::ROWS];                                // of a row: first and last visible position, its own, slope
  __shared__ StShared S;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c4 = lane & 3;
  const int G = p.Hq / p.Hkv, M = p.E * G, kvh = blockIdx.y, w = blockIdx.x;         // rows r = token * G + head
  int* counter = p.counters + kvh;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&S.full[i], Cfg::BULK ? ST_LOADERS : ST_LOADERS * (p.c.key_pos != nullptr ? 33 : 32));
      mbar_init(&S.empty[i], Cfg::GW * MT);
    }
    S.abort = 0;
    fence_barrier_init();
  }
  // a mass kernel behind this one reads rows and lengths ahead of its wait: they have to be there before it may start
  if (p.pdl) pdl_wait_prior_grid();
  pdl_launch_dependents();
  step_schedule(p, line, misc);
  const int total = tiles[p.bs];
  // sequences without a tile have nobody else to write their rows
  if (w == 0) {
    for (int s = warp; s < p.bs; s += Cfg::THREADS / 32) {
      if (tiles[s + 1] > tiles[s]) continue;
      for (int x = lane; x < M * D; x += 32) {
        const int e = x / (G * D), hd = x - e * G * D;
        p.out[(size_t)(s * p.E + e) * p.ld_out + (size_t)kvh * G * D + hd] = __float2bfloat16(0.f);
      }
      for (int x = lane; x < M; x += 32) {
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
    if constexpr (D == 256 && Cfg::THREADS == 384) regs_fewer<ST_FEW>();
    // ================================================================= loaders: KW keys of each tile a warp
    const int lw = warp - Cfg::WARPS, kl0 = lw * KW + lane % KW;
    const long long row_bytes = (long long)p.Hkv * D * 2;
    const uint64_t policy = l2_policy_evict_first();                 // read once: L2 is for the scores
    // what this lane copies: with BULK a row of K or V, else chunk lane % CPR of the rows lane / CPR, + 32 / CPR, ...
    const int c = Cfg::BULK ? 0 : lane % CPR, r0 = Cfg::BULK ? lane & 15 : lane / CPR;
    const char* from_k = reinterpret_cast<const char*>((Cfg::BULK && lane >= 16 ? p.v_pool : p.k_pool) + (size_t)kvh * D + c * 8);
    const char* from_v = reinterpret_cast<const char*>(p.v_pool + (size_t)kvh * D + c * 8);
    const uint32_t to0 = smem_u32(kv_s) + (uint32_t)((lw * KW + r0) * LD + c * 8) * 2 + (Cfg::BULK && lane >= 16 ? (uint32_t)Cfg::KV : 0u);
    constexpr int AHEAD = 4;                                         // tiles that page ids are read ahead
    int page[AHEAD], kpos[AHEAD];                                    // of this lane's key
    int next = t_begin, seq_end = t_begin, i = 0, n = 0;             // next tile to read ids of; this lane's key among the n of its sequence
    const int* bt = nullptr;
    const int* kp = nullptr;
    auto ids = [&](int& pg, int& pos) {
      if (next >= t_end) return;
      if (next >= seq_end) {
        StepCursor cur;
        cur.seek(p, line, next);
        seq_end = cur.seq1;
        n = cur.key.n;
        i = (next - cur.seq0) * KT + kl0;
        bt = p.c.block_table + (size_t)cur.key.row * p.c.bt_stride + cur.key.begin;
        if (p.c.key_pos != nullptr) kp = p.c.key_pos + (size_t)cur.key.row * p.c.kp_stride + cur.key.begin;
      }
      const int at = min(i, n - 1);                                  // keys behind the last repeat it
      pg = bt[at];
      if (kp != nullptr) pos = kp[at];
      i += KT;
      ++next;
    };
#pragma unroll
    for (int d = 0; d < AHEAD; ++d) ids(page[d], kpos[d]);
    int st = 0, left = t_end - t_begin;
    uint32_t phase = 1;                                              // of the stage's last release; the first use waits for none
    bool ok = true;
    while (left > 0 && ok) {
#pragma unroll
      for (int d = 0; d < AHEAD; ++d) {
        if (left <= 0) break;
        int pg = page[d];
        const int pos = kpos[d];
        if ((unsigned)pg > (unsigned)p.c.n_pages) { atomicOr(p.status, SMC_ERR_BOUNDS); pg = 0; }
        ids(page[d], kpos[d]);
        ok = __all_sync(0xffffffffu, st_wait(S, p.status, &S.empty[st], phase));
        if (!ok) break;
        if (kp != nullptr && lane < KW) pos_s[st * KT + kl0] = pos;
        const uint32_t to = to0 + (uint32_t)st * (uint32_t)(2 * Cfg::KV);
        if constexpr (Cfg::BULK) {
          __syncwarp();
          if (lane == 0) mbar_expect_tx(&S.full[st], 32 * D * 2);
          __syncwarp();
          asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;"
                       ::"r"(to), "l"(from_k + pg * row_bytes), "r"(D * 2), "r"(smem_u32(&S.full[st])), "l"(policy) : "memory");
        } else {
#pragma unroll
          for (int r = 0; r < KW; r += 32 / CPR) {
            const long long off = __shfl_sync(0xffffffffu, pg, r0 + r) * row_bytes;
            st_cp16(to + (uint32_t)(r * LD * 2), from_k + off, policy);
            st_cp16(to + (uint32_t)(r * LD * 2) + (uint32_t)Cfg::KV, from_v + off, policy);
          }
          __syncwarp();                                              // each lane arrives once its own copies have landed, which says nothing of positions
          if (kp != nullptr && lane == 0) mbar_arrive(&S.full[st]);
          asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_u32(&S.full[st])) : "memory");
        }
        --left;
        if (++st == STAGES) { st = 0; phase ^= 1u; }
      }
    }
    if constexpr (Cfg::BULK) {
      // a CTA that gave up keeps its shared memory until the copies in flight have landed
      const int issued = t_end - t_begin - left;
      if (S.abort)
        for (int k = max(0, issued - STAGES); k < issued; ++k) (void)mbar_wait(&S.full[k % STAGES], (uint32_t)(k / STAGES) & 1u);
    } else {
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
    return;
  }

  if constexpr (D == 256 && Cfg::THREADS == 384) regs_more<ST_MANY>();
  const int mt = warp % MT, gi = warp / MT, kg = gi % Cfg::GW, turn = gi / Cfg::GW;  // row set, group; of it keys and turn
  const float mul = p.c.mul, cap_in = p.c.cap_in, cap_out = p.c.cap_out;
  const int pitch = (M + 3) / 4 * 4;
  bool alive = true;
  int x = t_begin;
  while (x < t_end) {
    // ---------------------------------------------------------------- one sequence's tiles of this worker
    const int s = step_sequence(tiles, p.bs, x), seq0 = tiles[s], seq1 = tiles[s + 1], x_end = min(t_end, seq1);
    const StepKeys key = step_keys(p, line, s);
    for (int r = threadIdx.x; r < Cfg::ROWS; r += THREADS) {
      const int idx = key.len - p.E + r / G;
      float4 v = make_float4((float)SH_POS_END, -1.f, 0.f, 0.f);
      if (r < M && idx >= 0) {
        const int pos = p.c.key_pos != nullptr ? p.c.key_pos[(size_t)key.row * p.c.kp_stride + idx] : idx;
        const int2 see = shaped_bounds(p.c, s * p.E + r / G, pos);
        v = make_float4((float)see.x, (float)see.y, (float)pos, p.c.slopes != nullptr ? -p.c.slopes[kvh * G + r % G] * SH_LOG2E : 0.f);
      }
      row_s[r] = v;
    }
    uint32_t qb[NQ][D / 16][2];                                      // Q^T fragments: row g of each column set
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const int r = (mt * NQ + q) * 8 + g;
      const __nv_bfloat16* q0 = p.q + (size_t)(s * p.E + r / G) * p.ld_q + (size_t)(kvh * G + r % G) * D + 2 * c4;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        qb[q][kk][0] = r < M ? *reinterpret_cast<const uint32_t*>(q0 + kk * 16) : 0u;
        qb[q][kk][1] = r < M ? *reinterpret_cast<const uint32_t*>(q0 + kk * 16 + 8) : 0u;
      }
    }
    named_bar(1, THREADS);                                           // rows are known
    // keys between these are seen by all of this warp's rows
    const int my_row = mt * NQ * 8 + lane;
    const bool has_row = lane < NQ * 8 && my_row < M;
    const float seen_from = warp_max(has_row ? row_s[my_row].x : -1.f), seen_to = -warp_max(has_row ? -row_s[my_row].y : -(float)SH_POS_END);
    float m[NQ][2], l[NQ][2], o[NQ][D / 16][4];                      // of columns 2 c4, 2 c4 + 1
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      m[q][0] = m[q][1] = -INFINITY;
      l[q][0] = l[q][1] = 0.f;
#pragma unroll
      for (int n = 0; n < D / 16; ++n) o[q][n][0] = o[q][n][1] = o[q][n][2] = o[q][n][3] = 0.f;
    }

    for (; x < x_end; ++x) {
      const int nth = x - t_begin, st = nth % STAGES;
      if (Cfg::TURNS > 1 && nth % Cfg::TURNS != turn) continue;
      if (alive) alive = __all_sync(0xffffffffu, st_wait(S, p.status, &S.full[st], (uint32_t)(nth / STAGES) & 1u));
      if (!alive) continue;
#pragma unroll
      for (int sub = 0; sub < Cfg::SUB; ++sub) {
        const int k0 = (kg * Cfg::SUB + sub) * 16;
        const __nv_bfloat16* Kt = kv_s + (size_t)st * 2 * KT * LD + k0 * LD;
        const __nv_bfloat16* Vt = Kt + KT * LD;
        float sc[NQ][4], sd[NQ][4];                                  // two chains of products
#pragma unroll
        for (int q = 0; q < NQ; ++q) sc[q][0] = sc[q][1] = sc[q][2] = sc[q][3] = sd[q][0] = sd[q][1] = sd[q][2] = sd[q][3] = 0.f;
        // matrices of a K fragment: keys 0-7 dims 0-7, keys 8-15 dims 0-7, keys 0-7 dims 8-15, keys 8-15 dims 8-15
        const uint32_t ka = smem_u32(Kt + (lane & 15) * LD + (lane >> 4) * 8);
#pragma unroll
        for (int kk = 0; kk < D / 16; kk += 2) {
          uint32_t a[4], b[4];
          st_ldsm(a, ka + kk * 32);
          st_ldsm(b, ka + kk * 32 + 32);
#pragma unroll
          for (int q = 0; q < NQ; ++q) {
            st_mma(sc[q], a, qb[q][kk][0], qb[q][kk][1]);
            st_mma(sd[q], b, qb[q][kk + 1][0], qb[q][kk + 1][1]);
          }
        }
        const int i0 = (x - seq0) * KT + k0 + g;                     // of the sequence's visible keys: this lane's, and the one 8 behind
        float kp[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int pos = p.c.key_pos != nullptr ? pos_s[st * KT + k0 + g + 8 * h] : key.begin + i0 + 8 * h;
          kp[h] = i0 + 8 * h < key.n ? (float)pos : -1.f;
        }
        const bool plain = p.c.slopes == nullptr && __all_sync(0xffffffffu, kp[0] >= seen_from && kp[1] >= 0.f && kp[1] <= seen_to);
        uint32_t pb[NQ][2];
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          float top[2] = {m[q][0], m[q][1]};
          if (plain) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float v = sc[q][i] + sd[q][i];
              sc[q][i] = cap_in > 0.f ? shaped_cap(v, cap_in, cap_out) : v * mul;
              top[i & 1] = fmaxf(top[i & 1], sc[q][i]);
            }
          } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 row = row_s[(mt * NQ + q) * 8 + 2 * c4 + (i & 1)];
            float v = sc[q][i] + sd[q][i];
            v = cap_in > 0.f ? shaped_cap(v, cap_in, cap_out) : v * mul;
            v = fmaf(row.w, fabsf(kp[i >> 1] - row.z), v);
            v = kp[i >> 1] >= row.x && kp[i >> 1] <= row.y ? v : -INFINITY;
            sc[q][i] = v;
            top[i & 1] = fmaxf(top[i & 1], v);
          }
          }
          if (p.scores != nullptr && x < p.score_tiles) {
            const int r = (mt * NQ + q) * 8 + 2 * c4;
            float* at = p.scores + (((size_t)kvh * p.score_tiles + x) * KT + k0 + g) * pitch + r;
            if (r < pitch) {
              *reinterpret_cast<float2*>(at) = make_float2(sc[q][0], sc[q][1]);
              *reinterpret_cast<float2*>(at + 8 * pitch) = make_float2(sc[q][2], sc[q][3]);
            }
          }
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int sh = 4; sh < 32; sh <<= 1) top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], sh));
          if (__any_sync(0xffffffffu, top[0] > m[q][0] || top[1] > m[q][1])) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const float alpha = top[c] == -INFINITY ? 1.f : shaped_ex2(m[q][c] - top[c]);
              m[q][c] = top[c];
              l[q][c] *= alpha;
#pragma unroll
              for (int n = 0; n < D / 16; ++n) { o[q][n][c] *= alpha; o[q][n][2 + c] *= alpha; }
            }
          }
          const float ref[2] = {m[q][0] == -INFINITY ? 0.f : m[q][0], m[q][1] == -INFINITY ? 0.f : m[q][1]};
          float pr[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            pr[i] = shaped_ex2(sc[q][i] - ref[i & 1]);
            l[q][i & 1] += pr[i];
          }
          pb[q][0] = st_transpose(st_pack(pr[0], pr[1]));
          pb[q][1] = st_transpose(st_pack(pr[2], pr[3]));
        }
        // matrices of a V^T fragment: dims 0-7 keys 0-7, dims 8-15 keys 0-7, dims 0-7 keys 8-15, dims 8-15 keys 8-15
        const uint32_t va = smem_u32(Vt + ((lane & 7) + (lane >> 4) * 8) * LD + ((lane >> 3) & 1) * 8);
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
          uint32_t a[4];
          st_ldsm_t(a, va + n * 32);
#pragma unroll
          for (int q = 0; q < NQ; ++q) st_mma(o[q][n], a, pb[q][0], pb[q][1]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&S.empty[st]);
    }
    // ---------------------------------------------------------------- the groups of keys, joined in their order
#pragma unroll
    for (int q = 0; q < NQ; ++q)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int sh = 4; sh < 32; sh <<= 1) l[q][c] += __shfl_xor_sync(0xffffffffu, l[q][c], sh);
        if (g == 0) {
          ml_s[gi][(mt * NQ + q) * 8 + 2 * c4 + c][0] = m[q][c];
          ml_s[gi][(mt * NQ + q) * 8 + 2 * c4 + c][1] = l[q][c];
        }
      }
    named_bar(1, THREADS);
    float mine[NQ][2];
#pragma unroll
    for (int q = 0; q < NQ; ++q)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int row = (mt * NQ + q) * 8 + 2 * c4 + c;
        float top = ml_s[0][row][0];
#pragma unroll
        for (int k = 1; k < Cfg::GROUPS; ++k) top = fmaxf(top, ml_s[k][row][0]);
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < Cfg::GROUPS; ++k) sum += top == -INFINITY ? 0.f : ml_s[k][row][1] * shaped_ex2(ml_s[k][row][0] - top);
        mine[q][c] = top == -INFINITY ? 0.f : shaped_ex2(m[q][c] - top);
        if (gi == 0 && g == 0) {
          join[row * (D + 4) + D] = top;
          join[row * (D + 4) + D + 1] = sum;
        }
      }
    for (int k0 = 0; k0 < Cfg::GROUPS; k0 += Cfg::SLOTS) {
      if (gi >= k0 && gi < k0 + Cfg::SLOTS) {
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int row = (mt * NQ + q) * 8 + 2 * c4 + c;
            if (row >= M) continue;
            float* at = join + ((gi - k0) * Cfg::ROWS + row) * (D + 4) + g;
            const float f = mine[q][c];
#pragma unroll
            for (int n = 0; n < D / 16; ++n)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                // a group none of whose keys is visible adds nothing, whatever its values are
                const float v = f == 0.f ? 0.f : o[q][n][2 * h + c] * f;
                at[n * 16 + 8 * h] = k0 == 0 ? v : at[n * 16 + 8 * h] + v;
              }
          }
      }
      named_bar(1, THREADS);
    }
    if (Cfg::SLOTS > 1) {
      for (int i = threadIdx.x; i < M * (D / 4); i += THREADS) {
        float4* at = reinterpret_cast<float4*>(join + i / (D / 4) * (D + 4)) + i % (D / 4);
        float4 v = *at;
#pragma unroll
        for (int k = 1; k < Cfg::SLOTS; ++k) {
          const float4 u = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(at) + k * Cfg::ROWS * (D + 4));
          v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
        }
        *at = v;
      }
      named_bar(1, THREADS);
    }
    const int w_first = step_owner(seq0, W, total), w_last = step_owner(seq1 - 1, W, total);
    bool finish = w_first == w_last;
    if (!finish) {
      // part of worker v: row r of [rows_all], values [D], maximum and sum
      const bool ahead = step_first(w_first, W, total) < seq0;       // the first worker came from the sequence before
      auto part = [&](int v) { return p.parts + ((size_t)(v * 2 + (v == w_first && ahead ? 1 : 0)) * p.Hkv + kvh) * M * (D + 4); };
      float4* to = reinterpret_cast<float4*>(part(w));
      for (int i = threadIdx.x; i < M * (D + 4) / 4; i += THREADS) to[i] = reinterpret_cast<const float4*>(join)[i];
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
      if (finish) {                                                  // all parts are there; a warp per row, many loads in flight
        for (int r = warp; r < M; r += Cfg::WARPS) {
          constexpr int V = (148 + 31) / 32, B = 8, W4 = D / 128 > 0 ? D / 128 : 1;  // parts whose factors a lane holds, parts read at once
          const int n = w_last - w_first + 1;
          float f[V], den = 0.f, big = -INFINITY;
#pragma unroll
          for (int k = 0; k < V; ++k) {
            const int v = k * 32 + lane;
            f[k] = v < n ? __ldcg(part(w_first + v) + r * (D + 4) + D) : -INFINITY;
            big = fmaxf(big, f[k]);
          }
          big = warp_max(big);
#pragma unroll
          for (int k = 0; k < V; ++k) {
            const int v = k * 32 + lane;
            f[k] = f[k] == -INFINITY ? 0.f : shaped_ex2(f[k] - big);
            if (f[k] != 0.f) den += __ldcg(part(w_first + v) + r * (D + 4) + D + 1) * f[k];
          }
          den = warp_sum(den);
          float4 acc[W4];
#pragma unroll
          for (int k = 0; k < W4; ++k) acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
          const bool mine = D >= 128 || lane < D / 4;
#pragma unroll
          for (int k = 0; k < V; ++k)
            for (int v0 = k * 32; v0 < min(n, k * 32 + 32); v0 += B) {
              float4 got[B][W4];
#pragma unroll
              for (int i = 0; i < B; ++i)
#pragma unroll
                for (int c = 0; c < W4; ++c)
                  got[i][c] = mine ? __ldcg(reinterpret_cast<const float4*>(part(w_first + min(v0 + i, n - 1)) + r * (D + 4)) + c * 32 + lane) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
              for (int i = 0; i < B; ++i) {
                const float fi = __shfl_sync(0xffffffffu, f[k], (v0 + i) & 31);        // zero behind the last part
                if (fi != 0.f) {
#pragma unroll
                  for (int c = 0; c < W4; ++c) {
                    acc[c].x = fmaf(got[i][c].x, fi, acc[c].x);
                    acc[c].y = fmaf(got[i][c].y, fi, acc[c].y);
                    acc[c].z = fmaf(got[i][c].z, fi, acc[c].z);
                    acc[c].w = fmaf(got[i][c].w, fi, acc[c].w);
                  }
                }
              }
            }
          float* at = join + r * (D + 4);
          if (mine) {
#pragma unroll
            for (int c = 0; c < W4; ++c) reinterpret_cast<float4*>(at)[c * 32 + lane] = acc[c];
          }
          if (lane == 0) { at[D] = big; at[D + 1] = den; }
        }
        named_bar(1, THREADS);
      }
    }
    if (finish) {
      for (int i = threadIdx.x; i < M * (D / 2); i += THREADS) {
        const int r = i / (D / 2), d = (i - r * (D / 2)) * 2;
        const float* at = join + r * (D + 4);
        const bool none = at[D] == -INFINITY && at[D + 1] == 0.f;
        const float inv = 1.f / at[D + 1];
        *reinterpret_cast<uint32_t*>(p.out + (size_t)(s * p.E + r / G) * p.ld_out + (size_t)(kvh * G + r % G) * D + d) =
            none ? 0u : st_pack(at[d] * inv, at[d + 1] * inv);
      }
      if (p.lse != nullptr || p.scores != nullptr)
        for (int r = threadIdx.x; r < M; r += THREADS) {
          const float* at = join + r * (D + 4);
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

// mass[row, kvh, j] += sum over the rows of exp2(score - lse).  Every warp takes an equal run of tiles, a lane a key; four keys of a lane are in
// flight at once (one tile after the other, each looked up anew: 27 us for 230,000 keys and 8 heads, 10 so, of them 4.5 at the memory's rate).
constexpr int SM_WARPS = 8;

__global__ void __launch_bounds__(SM_WARPS * 32) shaped_step_mass_kernel(const ShapedStepParams p) {
  extern __shared__ int sm_tiles[];                                  // [bs + 1], [bs], [32]
  __shared__ __align__(16) float top_s[SM_WARPS][64];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kvh = blockIdx.y, G = p.Hq / p.Hkv, M = p.E * G, pitch = (M + 3) / 4 * 4;
  const StepLine line{sm_tiles, sm_tiles + p.bs + 1};
  step_schedule(p, line, line.spans + p.bs);                         // from what was there before the first kernel
  const int total = sm_tiles[p.bs], many = gridDim.x * SM_WARPS, me = blockIdx.x * SM_WARPS + warp;
  // on every path: whoever follows waits for this grid alone, which must not end ahead of the first kernel
  pdl_wait_prior_grid();
  if (total > p.score_tiles) {                                       // the workspace is too small for these contexts
    if (threadIdx.x == 0 && blockIdx.x == 0) atomicOr(p.status, SMC_ERR_BOUNDS);
    return;
  }
  const int x_end = step_first(me + 1, many, total);
  int x = step_first(me, many, total);
  while (x < x_end) {
    StepCursor cur;
    cur.seek(p, line, x);
    const int end = min(x_end, cur.seq1);
    bool twice = false;                                              // a row listed twice would be added to by two warps at once
    for (int o = lane; o < cur.s; o += 32) twice |= p.rows[o] == cur.key.row && p.lens[o] > 0;
    if (__any_sync(0xffffffffu, twice)) {
      if (lane == 0) atomicOr(p.status, SMC_ERR_BOUNDS);
      x = end;
      continue;
    }
    __syncwarp();
    for (int r = lane; r < pitch; r += 32)
      top_s[warp][r] = r < M ? p.lse2[(size_t)(cur.s * p.E + r / G) * p.Hq + kvh * G + r % G] : INFINITY;
    __syncwarp();
    const float* sc = p.scores + ((size_t)kvh * p.score_tiles + cur.seq0) * p.tile * pitch;
    float* to = p.mass + ((size_t)cur.key.row * p.Hkv + kvh) * p.mass_stride + cur.key.begin;
    const int i_end = min((end - cur.seq0) * p.tile, cur.key.n);
    for (int i = (x - cur.seq0) * p.tile + lane; i < i_end; i += 128) {
      float sum[4] = {0.f, 0.f, 0.f, 0.f}, before[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) before[k] = i + 32 * k < i_end ? to[i + 32 * k] : 0.f;
      for (int r = 0; r < pitch; r += 4) {
        const float4 top = *reinterpret_cast<const float4*>(&top_s[warp][r]);
        float4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<const float4*>(sc + (size_t)min(i + 32 * k, i_end - 1) * pitch + r);
#pragma unroll
        for (int k = 0; k < 4; ++k) {                                // columns behind the last row were never written
          sum[k] += shaped_ex2(v[k].x - top.x);
          sum[k] += r + 1 < M ? shaped_ex2(v[k].y - top.y) : 0.f;
          sum[k] += r + 2 < M ? shaped_ex2(v[k].z - top.z) : 0.f;
          sum[k] += r + 3 < M ? shaped_ex2(v[k].w - top.w) : 0.f;
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + 32 * k < i_end) to[i + 32 * k] = before[k] + sum[k];
    }
    x = end;
  }
}

// Parts of the workspace, each from a 256-byte border.
struct StepWork { size_t parts, lse2, scores, bytes; long long score_tiles, counted; int workers; };

static StepWork step_work(int bs, int E, int Hq, int Hkv, int D, long long keys) {
  StepWork w;
  const int M = E * (Hq / Hkv);
  w.workers = 148 / Hkv > 0 ? 148 / Hkv : 1;           // a CTA per SM
  w.score_tiles = keys > 0 ? keys / step_tile(D) + bs : 0;                   // every sequence may end inside a tile
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  w.counted = (long long)bs * Hkv;
  w.parts = (size_t)ST_COUNTERS * 4;
  w.lse2 = w.parts + up((size_t)w.workers * 2 * Hkv * M * (D + 4) * 4);
  w.scores = w.lse2 + up((size_t)bs * E * Hq * 4);
  w.bytes = w.scores + up((size_t)Hkv * w.score_tiles * ((M + 3) / 4 * 4) * step_tile(D) * 4);
  return w;
}

template <int D, int NQ, int MT>
static int launch_shaped_step(const ShapedStepParams& p, cudaStream_t st) {
  using Cfg = StCfg<D, NQ, MT>;
  auto kernel = shaped_step_kernel<D, NQ, MT>;
  static_assert(Cfg::SMEM + Cfg::GROUPS * Cfg::ROWS * 8 + Cfg::ROWS * 16 + sizeof(StShared) <= 232448, "shared memory");
  CUDA_CHECK_RET(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg::SMEM));
  if constexpr (D == 256 && Cfg::THREADS == 384) {     // what the warps ask for later is there from the start
    static const int regs = [&] { cudaFuncAttributes a; return cudaFuncGetAttributes(&a, kernel) == cudaSuccess ? a.numRegs : 0; }();
    if (regs < 168) return -155;
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.workers, (unsigned)p.Hkv);
  cfg.blockDim = dim3(Cfg::THREADS);
  cfg.dynamicSmemBytes = Cfg::SMEM;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = p.pdl ? 1 : 0;
  CUDA_CHECK_RET(cudaLaunchKernelEx(&cfg, kernel, p));
  if (p.mass == nullptr) return 0;
  cfg.gridDim = dim3((unsigned)((148 * 4 + p.Hkv - 1) / p.Hkv), (unsigned)p.Hkv);
  cfg.blockDim = dim3(SM_WARPS * 32);
  cfg.dynamicSmemBytes = (size_t)(2 * p.bs + 1 + 32) * 4;
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
                            long long bt_pitch, int bt_rows, const int* key_pos, int kp_stride, const int* rows, const int* lens, void* out,
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
  if (!shaped_scores_fit(scale, cap)) return -152;
  if (!pitch_fits(bt_pitch) || n_pages < 0 || (mass != nullptr && mass_stride < pitch_cols(bt_pitch))) return -153;
  StepWork w = step_work(bs, E, Hq, Hkv, D, 0);
  if (mass != nullptr) w.score_tiles = (work_bytes - (long long)w.scores) / ((long long)Hkv * ((E * (Hq / Hkv) + 3) / 4 * 4) * step_tile(D) * 4);       // the rest of it
  if (work_bytes < (long long)w.bytes || (mass != nullptr && w.score_tiles < 1)) return -154;
  ShapedStepParams p;
  p.c = shaped_cache(block_table, bt_pitch, bt_rows, n_pages, key_pos, kp_stride, bounds, slopes, scale, cap);
  p.q = (const __nv_bfloat16*)q; p.k_pool = (const __nv_bfloat16*)k_pool; p.v_pool = (const __nv_bfloat16*)v_pool;
  p.rows = rows; p.lens = lens; p.out = (__nv_bfloat16*)out; p.lse = lse; p.mass = mass;
  char* base = (char*)work;
  p.counters = (int*)base; p.parts = (float*)(base + w.parts); p.lse2 = (float*)(base + w.lse2);
  p.scores = mass != nullptr ? (float*)(base + w.scores) : nullptr;
  p.ld_q = ld_q; p.ld_out = ld_out; p.mass_stride = mass_stride; p.score_tiles = w.score_tiles;
  p.bs = bs; p.E = E; p.Hq = Hq; p.Hkv = Hkv; p.workers = w.workers; p.tile = step_tile(D); p.pdl = pdl; p.status = status;
  const int rows_each = E * (Hq / Hkv);
#define SMC_SHAPED_STEP(DD)                                                  \
  if (D == DD) {                                                             \
    if (rows_each <= 8) return launch_shaped_step<DD, 1, 1>(p, st);          \
    if (rows_each <= 16) return launch_shaped_step<DD, 2, 1>(p, st);         \
    if (rows_each <= 32) return launch_shaped_step<DD, 2, 2>(p, st);         \
    return launch_shaped_step<DD, 2, 4>(p, st);                              \
  }
  SMC_SHAPED_STEP(64)
  SMC_SHAPED_STEP(128)
  SMC_SHAPED_STEP(256)
#undef SMC_SHAPED_STEP
  return -150;
}
