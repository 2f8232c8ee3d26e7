// The weight that every cached token collects from a prompt's tokens, on tcgen05:
//     mass[row, kvh, j] += sum over the tokens i and the query heads of the group of exp(x_ij - lse_i)
// with the scores of shaped.cuh and the log-sum-exp that the attention pass left.
//
// A CTA takes NT tiles of 128 keys of one KV head as the left operand, so that a key is a lane of the tensor memory and a thread adds up its
// own key's weight: no reduction across threads, no atomics, one order of the sum.  The query rows that may see the keys stream
// through a ring in steps of 128 (tokens x heads of the group), with their log-sum-exp, positions, bounds and slopes as columns in shared memory:
//     S_t = K_t Q^T      UMMA 128 x 128 x D, two buffers per key tile in tensor memory
//     sum                four warps per key tile: exp2(x - lse) of 128 columns, masked by the key's position where a column does not see all keys
// What bounds it is the exponential, one per (token, head, key) pair; the product is half of the attention's.  A step of 128 columns takes 2700 cycles of the 2048 its
// exponentials take on the two warps of a scheduler, 4400 with a cap; a key tile 8 us from its pages to its first sum.  Microseconds on B200 (device times,
// graphs replayed): 4096 tokens of 32 heads on 8: heads of 128 133, capped 202, distance bias 154, both 235; the last 33 to 64 tokens of four prompts of 20,000, heads of 64 119.
// The grid is persistent: key tiles of all sequences, those with most tokens behind them first; the next tile's keys are fetched while one is worked on.  Where sequences bring
// many tokens the two blocks of a cluster take the steps of a tile by turns and add up their sums through shared memory in their order.
#include <atomic>
#include <type_traits>

#include "shaped.cuh"

namespace smc {

constexpr int MS_LOADERS = 4, MS_Q = 128;
// A sequence that brings so many steps and has no more key tiles, over all heads, than the device has SMs: two blocks share each of them.  Its own numbers decide, so that
// the order of its sums does not hang on what else a call brings.  Heads of 128, 8 KV heads, capped, us with one block and with two: 1500 tokens (48 tiles) 155 and 84, 4096
// (128) 356 and 195, 9000 (288) 759 and 772, two of 400 behind 6000 (208 each) 131 and 161: a tile costs 8 us before its first sum in every block.
constexpr int MS_SHARED_STEPS = 16, MS_SHARED_TILES = 148;

template <int D> struct MsCfg;                        // key tiles of a CTA, slots of the ring of query steps, of them in flight, sets of keys in shared memory
template <> struct MsCfg<64> { static constexpr int NT = 2, QU = 6, LAG = 3, KB = 2; };
template <> struct MsCfg<128> { static constexpr int NT = 2, QU = 4, LAG = 2, KB = 1; };
template <> struct MsCfg<256> { static constexpr int NT = 1, QU = 2, LAG = 1, KB = 1; };

struct ShapedMassParams {
  ShapedCache c;
  const __nv_bfloat16* q;
  const __nv_bfloat16* k_pool;
  const int4* runs;
  const float* lse;              // [T, Hq]
  float* mass;                   // [bt_rows, Hkv, mass_stride]
  long long ld_q, mass_stride;
  int n_runs, T, Hq, Hkv, pdl, cluster, share_from;                  // blocks of a cluster; new tokens of a sequence whose tiles two of them share
  int* status;
};

// What a step's query rows bring along, by column
struct alignas(16) MsColumns {
  float neg_lse[MS_Q], pos[MS_Q], first[MS_Q], last[MS_Q], slope[MS_Q];
  float max_first[4], min_last[4], min_pos4[4];       // over 32 columns each: a key between the first two is seen by every column
};

template <int D> struct MsShared {
  static constexpr int SLOTS = MsCfg<D>::QU + 2;      // a step's columns are read until its sums are done, two products behind the ring
  MsColumns col[SLOTS];
  uint64_t q_full[MsCfg<D>::QU], q_empty[MsCfg<D>::QU], col_full[SLOTS], k_full[2], k_empty[2], s_full[2][2], s_empty[2][2];
  float sum[MsCfg<D>::NT * 128];                      // of this block, for the cluster
  uint32_t tmem_slot;
  int lo[16], hi[16];
  volatile int abort;
};

template <typename Shared>
__device__ __forceinline__ bool ms_wait(Shared& S, int* status, uint64_t* bar, uint32_t parity) {
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

// All tiles of KT keys of the sequences whose tiles two blocks share, or of the others, those with most tokens behind their first key in front; used by whole warps.
template <int KT>
struct MsTiles {
  const ShapedMassParams& p;
  const bool shared;
  ShapedRun mine;
  __device__ MsTiles(const ShapedMassParams& params, const ShapedRun& of_lane, bool of_shared) : p(params), shared(of_shared), mine(this_kind(of_lane)) {}
  __device__ static ShapedRun any_run(const ShapedMassParams& p, int s) { return s < p.n_runs ? shaped_run(p.c, p.runs, s, p.T, p.status) : ShapedRun{0, 0, 0, 0}; }
  __device__ ShapedRun this_kind(ShapedRun r) const {
    const bool is_shared = p.cluster > 1 && r.n >= p.share_from && (long long)((r.held + r.n - 1) / KT + 1) * p.Hkv <= MS_SHARED_TILES;
    if (is_shared != shared) r.n = 0;
    return r;
  }
  __device__ ShapedRun run_of(int s) const { return this_kind(any_run(p, s)); }
  // tiles of run r with at least `tokens` of its new tokens at or behind their first key: the first ones of the row
  __device__ int of_run(const ShapedRun& r, int tokens) const { return tokens > r.n ? 0 : (int)((unsigned)(r.held + r.n - tokens) / KT) + 1; }
  __device__ int count(int tokens) const {
    int n = of_run(mine, tokens);
    for (int s = (threadIdx.x & 31) + 32; s < p.n_runs; s += 32) n += of_run(run_of(s), tokens);
    return (int)__reduce_add_sync(0xffffffffu, (unsigned)n);
  }
  // tile number `want`: its run, the run's number and the tile inside it
  __device__ bool find(int want, ShapedRun& run, int& number, int& tile) const {
    const int lane = threadIdx.x & 31;
    int most = mine.n;
    for (int s = lane + 32; s < p.n_runs; s += 32) most = max(most, run_of(s).n);
    int lo = 1, hi = __reduce_max_sync(0xffffffffu, most) + 1;        // count(lo) > want >= count(hi)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (count(mid) > want) lo = mid; else hi = mid;
    }
    int left = want - count(lo + 1);
    for (int s0 = 0; s0 < p.n_runs; s0 += 32) {
      const ShapedRun r = s0 == 0 ? mine : run_of(s0 + lane);
      const int more = of_run(r, lo + 1), n = of_run(r, lo) - more;
      int sum = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, left >= sum - n && left < sum);
      if (hit) {
        const int src = __ffs(hit) - 1;
        run.row = __shfl_sync(0xffffffffu, r.row, src);
        run.held = __shfl_sync(0xffffffffu, r.held, src);
        run.at = __shfl_sync(0xffffffffu, r.at, src);
        run.n = __shfl_sync(0xffffffffu, r.n, src);
        tile = __shfl_sync(0xffffffffu, more + left - (sum - n), src);
        number = s0 + src;
        return true;
      }
      left -= __shfl_sync(0xffffffffu, sum, 31);
    }
    return false;
  }
};

template <int D, bool CAP, bool BIAS>
__global__ void __launch_bounds__((5 * MsCfg<D>::NT + MS_LOADERS) * 32, 1) shaped_mass_kernel(const ShapedMassParams p) {
  constexpr int NT = MsCfg<D>::NT, QU = MsCfg<D>::QU, LAG = MsCfg<D>::LAG, KB = MsCfg<D>::KB;
  constexpr int NPAN = D / 64, PANEL = 128 * 128, TILE = NPAN * PANEL, CPR = D / 8;
  using Shared = MsShared<D>;
  constexpr int SLOTS = Shared::SLOTS;
  extern __shared__ uint8_t ms_smem_raw[];
  __shared__ Shared S;
  const uint32_t raw = smem_u32(ms_smem_raw);
  uint8_t* smem = ms_smem_raw + (((raw + 1023u) & ~1023u) - raw);
  uint8_t* q_s = smem + KB * NT * TILE;               // [QU] query steps behind [KB][NT] keys
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int LOAD_WARP = 4 * NT, MMA_WARP = LOAD_WARP + MS_LOADERS;
  const int G = p.Hq / p.Hkv, TT = 128 / G;           // tokens of a step
  if (warp == MMA_WARP) {
    tmem_alloc(&S.tmem_slot, 512);
    tmem_relinquish();
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < QU; ++i) {
      mbar_init(&S.q_full[i], MS_LOADERS);
      mbar_init(&S.q_empty[i], NT);
    }
    for (int i = 0; i < SLOTS; ++i) mbar_init(&S.col_full[i], MS_LOADERS);
    for (int i = 0; i < KB; ++i) {
      mbar_init(&S.k_full[i], MS_LOADERS);
      mbar_init(&S.k_empty[i], NT);
    }
    for (int t = 0; t < NT; ++t)
      for (int i = 0; i < 2; ++i) {
        mbar_init(&S.s_full[t][i], 1);
        mbar_init(&S.s_empty[t][i], 4);
      }
    S.abort = 0;
    fence_barrier_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = S.tmem_slot;
  if (p.pdl) { pdl_launch_dependents(); pdl_wait_prior_grid(); }

  bool dead = false;                                  // a wait of this warp ran out: it goes on to the end without work
  uint32_t u0 = 0, k_use = 0;                         // steps and key tiles so far: barriers run on from item to item
  using Tiles = MsTiles<NT * 128>;
  const ShapedRun of_lane = Tiles::any_run(p, lane);
  // tiles that two blocks share, then the others (at most the table's entries over 128, times the heads)
  const int together = p.cluster > 1 ? Tiles(p, of_lane, true).count(1) * p.Hkv : 0, items = together + Tiles(p, of_lane, false).count(1) * p.Hkv;
  for (int base = 0, round = 0; base < items; ++round) {
    const bool shared = base < together;
    const int C = shared ? p.cluster : 1, rank = C > 1 ? (int)cluster_ctarank() : 0, groups = gridDim.x / C, group = blockIdx.x / C;
    // every second round runs backwards, so that who had a long tile gets a short one
    const int item = base + (round & 1 ? groups - 1 - group : group), end = shared ? together : items, first = shared ? 0 : together;
    base = min(base + groups, end);
    ShapedRun run{0, 0, 0, 0};
    int number = 0, tile = 0;
    bool have = item < end && Tiles(p, of_lane, shared).find((item - first) / p.Hkv, run, number, tile);
    if (have) {
      bool twice = false;                             // a row listed twice would be added to by two blocks at once
      for (int o = lane; o < number; o += 32) twice |= p.runs[o].x == run.row && p.runs[o].w > 0;
      if (__any_sync(0xffffffffu, twice)) {
        if (threadIdx.x == 0) atomicOr(p.status, SMC_ERR_BOUNDS);
        have = false;
      }
    }
    const int kvh = item % p.Hkv, hbase = kvh * G, keys = run.held + run.n, k0 = tile * NT * 128;
    const int* kp = p.c.key_pos != nullptr ? p.c.key_pos + (size_t)run.row * p.c.kp_stride : nullptr;
    auto pos_of = [&](int idx) { return kp != nullptr ? kp[idx] : idx; };
    // new tokens [ta, tb) of the run that may see one of the keys
    int ta = max(0, k0 - run.held), tb = have ? run.n : 0;
    if (p.c.bounds != nullptr) {
      int lo = run.n, hi = 0;
      if (have) {
        const int near = pos_of(k0), far = pos_of(min(k0 + NT * 128, keys) - 1);
        for (int i = threadIdx.x; i < run.n; i += blockDim.x) {
          const int2 b = shaped_bounds(p.c, run.at + i, 0);
          if (b.x <= far && b.y >= near && b.x <= b.y) { lo = min(lo, i); hi = max(hi, i + 1); }
        }
      }
      lo = __reduce_min_sync(0xffffffffu, lo);
      hi = __reduce_max_sync(0xffffffffu, hi);
      __syncthreads();                                // the item before has read its range
      if (lane == 0) { S.lo[warp] = lo; S.hi[warp] = hi; }
      __syncthreads();
      ta = run.n;
      tb = 0;
      for (int w = 0; w < (int)(blockDim.x >> 5); ++w) { ta = min(ta, S.lo[w]); tb = max(tb, S.hi[w]); }
    }
    const int all_steps = tb > ta ? (tb - ta + TT - 1) / TT : 0, n_steps = (all_steps - rank + C - 1) / C;     // this block's: rank, rank + C, ...
    uint8_t* k_s = smem + (k_use % KB) * NT * TILE;
    float total = 0.f;
    if (n_steps <= 0 || dead) {
    } else if (warp >= LOAD_WARP && warp < MMA_WARP) {
      // ================================================================= loaders
      const int lw = warp - LOAD_WARP;
      bool go = k_use < KB || ms_wait(S, p.status, &S.k_empty[k_use % KB], (k_use / KB - 1) & 1u);     // products with the keys before are done
      go = __all_sync(0xffffffffu, go);
      dead = !go;
      if (go) {                                       // keys: this warp's 32 of each tile
        const int* bt = p.c.block_table + (size_t)run.row * p.c.bt_stride;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int mine = k0 + t * 128 + lw * 32 + lane;
          int page = mine < keys ? bt[mine] : -1;
          if (page > p.c.n_pages || (page < 0 && mine < keys)) { atomicOr(p.status, SMC_ERR_BOUNDS); page = 0; }
          const uint32_t dst0 = smem_u32(k_s + t * TILE);
#pragma unroll 4
          for (int idx = lane; idx < 32 * CPR; idx += 32) {
            const int kl = idx / CPR, c = idx % CPR, r = lw * 32 + kl;
            const int pg = __shfl_sync(0xffffffffu, page, kl);
            const uint32_t dst = dst0 + (uint32_t)((c >> 3) * PANEL + r * 128 + (((c & 7) ^ (r & 7)) << 4));
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(p.k_pool + (size_t)max(pg, 0) * p.Hkv * D + (size_t)kvh * D + c * 8), "r"(pg >= 0 ? 16 : 0) : "memory");
          }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      }
      // this lane's column of a step, read one step ahead
      const int cl = lw * 32 + lane, ct = cl / G, h = hbase + cl % G;
      const int row_off = ct * (int)p.ld_q + cl % G * D;               // of its query row, from the step's first token on (tokens of a step: at most 128)
      struct Column { float lse; int pos; int2 see; bool live; } next;
      const float slope = BIAS && cl < TT * G ? -p.c.slopes[h] * SH_LOG2E : 0.f;
      auto column = [&](int j) {
        const int tok = ta + (rank + j * C) * TT + ct;
        Column c{-INFINITY, 0, make_int2(0, SH_POS_END), cl < TT * G && tok < tb && j < n_steps};
        if (c.live) {
          c.lse = p.lse[(size_t)(run.at + tok) * p.Hq + h];
          c.pos = pos_of(run.held + tok);
          c.see = shaped_bounds(p.c, run.at + tok, c.pos);
        }
        return c;
      };
      if (go) next = column(0);
      for (int j = 0; go && j < n_steps; ++j) {
        const uint32_t u = u0 + j, st = u % QU;
        const int step0 = ta + (rank + j * C) * TT;
        const Column mine = next;
        next = column(j + 1);
        const bool live = mine.live, seen = mine.lse != -INFINITY;
        const float nl = seen ? -mine.lse * SH_LOG2E : -INFINITY, posf = (float)mine.pos;
        // a token that has seen nothing sees no key
        const float first = !live || seen ? (float)mine.see.x : (float)SH_POS_END, last = !live || seen ? (float)mine.see.y : -1.f;
        const bool ok = u < QU || ms_wait(S, p.status, &S.q_empty[st], (u / QU - 1) & 1u);
        if (!__all_sync(0xffffffffu, ok)) { go = false; dead = true; break; }
        MsColumns& col = S.col[u % SLOTS];
        col.neg_lse[cl] = nl;
        col.pos[cl] = posf;
        // columns without a token see nothing (a key that is not finite makes NaN of their zeros), but do not send their step the long way
        col.first[cl] = live ? first : (float)SH_POS_END;
        col.last[cl] = live ? last : -1.f;
        if (BIAS) col.slope[cl] = slope;
        const float mf = warp_max(first), ml = -warp_max(-last);
        const float mp = BIAS ? -warp_max(live ? -posf : -(float)SH_POS_END) : 0.f;
        if (lane == 0) { col.max_first[lw] = mf; col.min_last[lw] = ml; col.min_pos4[lw] = mp; }
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.col_full[u % SLOTS]);
        // the row of every lane's column, 16 bytes a lane: chunk lane % CPR of the rows lane / CPR, + 32 / CPR, ...
        const __nv_bfloat16* q0 = p.q + (size_t)(run.at + step0) * p.ld_q + (size_t)hbase * D + lane % CPR * 8;
        const uint32_t dst0 = smem_u32(q_s + (size_t)st * TILE) + (uint32_t)((lane % CPR >> 3) * PANEL);
#pragma unroll
        for (int r0 = 0; r0 < 32; r0 += 32 / CPR) {
          const int rl = r0 + lane / CPR, r = lw * 32 + rl;
          const int off = __shfl_sync(0xffffffffu, live ? row_off : -1, rl);
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                       ::"r"(dst0 + (uint32_t)(r * 128 + (((lane % CPR & 7) ^ (r & 7)) << 4))), "l"(q0 + max(off, 0)), "r"(off >= 0 ? 16 : 0) : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (j >= LAG - 1) {                           // the keys, then step j - LAG, have landed: hand them over
          asm volatile("cp.async.wait_group %0;" ::"n"(LAG) : "memory");
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(j == LAG - 1 ? &S.k_full[k_use % KB] : &S.q_full[(u - LAG) % QU]);
        }
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      fence_proxy_async();
      __syncwarp();
      if (go && lane == 0) {
        if (n_steps < LAG) mbar_arrive(&S.k_full[k_use % KB]);
        for (int j = max(0, n_steps - LAG); j < n_steps; ++j) mbar_arrive(&S.q_full[(u0 + j) % QU]);
      }
    } else if (warp >= MMA_WARP) {
      // ================================================================= MMA issuers (one thread per key tile)
      const int t = warp - MMA_WARP;
      bool ok = true;
      if (elect_one()) {
        constexpr uint32_t idesc = umma_idesc_bf16(128, MS_Q);
        const uint32_t k_addr = smem_u32(k_s) + t * TILE;
        ok = ms_wait(S, p.status, &S.k_full[k_use % KB], (k_use / KB) & 1u);
        for (int j = 0; ok && j < n_steps; ++j) {
          const uint32_t u = u0 + j, st = u % QU, buf = u & 1u;
          ok = ms_wait(S, p.status, &S.q_full[st], (u / QU) & 1u) && (u < 2 || ms_wait(S, p.status, &S.s_empty[t][buf], (u / 2 - 1) & 1u));
          if (!ok) break;
          tc_fence_after();
          const uint32_t q_addr = smem_u32(q_s + (size_t)st * TILE);
#pragma unroll
          for (int pan = 0; pan < NPAN; ++pan)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_bf16_ss(tmem_base + (uint32_t)(t * 2 + buf) * 128u, umma_desc_k_sw128(k_addr + pan * PANEL) + 2 * k,
                           umma_desc_k_sw128(q_addr + pan * PANEL) + 2 * k, idesc, (pan | k) ? 1u : 0u);
          umma_commit(&S.s_full[t][buf]);
          umma_commit(&S.q_empty[st]);
          if (j == n_steps - 1) umma_commit(&S.k_empty[k_use % KB]);
        }
      }
      dead = !__all_sync(0xffffffffu, ok);
    } else {
      // ================================================================= sums (one key per thread)
      const int t = warp >> 2, r = (warp & 3) * 32 + lane, k = k0 + t * 128 + r;
      const uint32_t ts = tmem_base + (uint32_t)t * 256u + (((uint32_t)((warp & 3) * 32)) << 16);
      const float kpos = k < keys ? (float)pos_of(k) : -1.f;
      const float mul = p.c.mul, cap_in = p.c.cap_in, cap_out = p.c.cap_out;
      const uint64_t mul2 = f2_pair(mul, mul), ahead2 = f2_pair(-kpos, -kpos);
      const ShapedCapNear<4> near(cap_in, cap_out, mul);
      float* to = p.mass + ((size_t)run.row * p.Hkv + kvh) * p.mass_stride + k;
      const float before = C == 1 && k < keys ? *to : 0.f;          // long back when the sum is there
      for (int j = 0; j < n_steps; ++j) {
        const uint32_t u = u0 + j, buf = u & 1u;
        const MsColumns& col = S.col[u % SLOTS];
        if (!__all_sync(0xffffffffu, ms_wait(S, p.status, &S.s_full[t][buf], (u / 2) & 1u) &&
                                         ms_wait(S, p.status, &S.col_full[u % SLOTS], (u / SLOTS) & 1u))) { dead = true; break; }
        tc_fence_after();
        const float4 mf = *reinterpret_cast<const float4*>(col.max_first), ml = *reinterpret_cast<const float4*>(col.min_last);
        const bool full = __all_sync(0xffffffffu, kpos >= fmaxf(fmaxf(mf.x, mf.y), fmaxf(mf.z, mf.w)) && kpos <= fminf(fminf(ml.x, ml.y), fminf(ml.z, ml.w)));
        const float4 mp = *reinterpret_cast<const float4*>(col.min_pos4);
        uint64_t part[2] = {0ull, 0ull};              // a step's sum in four parts ahead of the running one: short chains of additions
        const bool behind = !BIAS || __all_sync(0xffffffffu, kpos <= fminf(fminf(mp.x, mp.y), fminf(mp.z, mp.w)));    // every column lies behind this key
        // exp2 of what `shaped` makes of pairs of scores and what is added to them; `plain`: every key is in front of every token and seen by it
        auto add_up = [&](const uint32_t (&w)[32], int c0, auto plain, auto shaped) {
          constexpr bool PLAIN = decltype(plain)::value;
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const ulonglong2 nl = *reinterpret_cast<const ulonglong2*>(&col.neg_lse[c0 + i]);
            uint64_t off[2] = {nl.x, nl.y};
            if (BIAS) {                               // (the distance itself first, exact: shares of it from some point between would cancel across a gap in the positions)
              const ulonglong2 sl = *reinterpret_cast<const ulonglong2*>(&col.slope[c0 + i]), at = *reinterpret_cast<const ulonglong2*>(&col.pos[c0 + i]);
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                uint64_t far = f2_add(k ? at.y : at.x, ahead2);
                if constexpr (!PLAIN) {
                  const float2 v = f2_unpair(far);
                  far = f2_pair(fabsf(v.x), fabsf(v.y));
                }
                off[k] = f2_fma(far, k ? sl.y : sl.x, off[k]);
              }
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int c = c0 + i + 2 * k;
              const float2 v = f2_unpair(shaped(f2_pair(__uint_as_float(w[i + 2 * k]), __uint_as_float(w[i + 2 * k + 1])), off[k]));
              float e0 = shaped_ex2(v.x), e1 = shaped_ex2(v.y);
              if constexpr (!PLAIN) {
                e0 = kpos >= col.first[c] && kpos <= col.last[c] ? e0 : 0.f;
                e1 = kpos >= col.first[c + 1] && kpos <= col.last[c + 1] ? e1 : 0.f;
              }
              part[k] = f2_add(part[k], f2_pair(e0, e1));
            }
          }
        };
        auto number_by_number = [&](uint64_t x, uint64_t off) {
          const float2 v = f2_unpair(x);
          return f2_add(CAP ? f2_pair(shaped_cap(v.x, cap_in, cap_out), shaped_cap(v.y, cap_in, cap_out)) : f2_mul(x, mul2), off);
        };
#pragma unroll 1
        for (int c0 = 0; c0 < MS_Q; c0 += 64) {
          uint32_t w[2][32];
#pragma unroll
          for (int k = 0; k < 4; ++k) tmem_ld_32x32b_x16(ts + buf * 128u + c0 + 16 * k, *reinterpret_cast<uint32_t(*)[16]>(&w[k >> 1][(k & 1) * 16]));
          tmem_ld_wait();
          bool reach = true;
          if (CAP) {
            float far = 0.f;
#pragma unroll
            for (int i = 0; i < 64; i += 2) far = shaped_max3(far, fabsf(__uint_as_float(w[i >> 5][i & 31])), fabsf(__uint_as_float(w[i >> 5][(i & 31) + 1])));
            reach = __all_sync(0xffffffffu, far * cap_in <= p.c.near_reach);
          }
          if (full && reach && behind) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
              add_up(w[h], c0 + 32 * h, std::true_type(), [&](uint64_t x, uint64_t off) { return CAP ? near(x, off) : f2_fma(x, mul2, off); });
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) add_up(w[h], c0 + 32 * h, std::false_type(), number_by_number);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.s_empty[t][buf]);
        const float2 a = f2_unpair(part[0]), b = f2_unpair(part[1]);
        total += (a.x + a.y) + (b.x + b.y);
      }
      if (C == 1 && !dead && k < keys) *to = before + total;
    }
    if (C > 1 && all_steps > 0) {                     // the blocks' sums in their order, a part of the keys by each block
      if (warp < LOAD_WARP) S.sum[threadIdx.x] = dead ? 0.f : total;
      cluster_sync();
      const int share = NT * 128 / C, i = rank * share + threadIdx.x;
      if (threadIdx.x < share && k0 + i < keys) {
        float all_of = 0.f;
        for (int c = 0; c < C; ++c) all_of += ld_dsmem_f32(smem_u32(&S.sum[i]), c);
        p.mass[((size_t)run.row * p.Hkv + kvh) * p.mass_stride + k0 + i] += all_of;
      }
      cluster_sync();
    }
    if (n_steps <= 0) continue;
    u0 += n_steps;
    ++k_use;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) tmem_dealloc(tmem_base, 512);
}

template <int D, bool CAP, bool BIAS>
static int launch_shaped_mass(const ShapedMassParams& p, cudaStream_t st) {
  constexpr size_t smem = (size_t)(MsCfg<D>::KB * MsCfg<D>::NT + MsCfg<D>::QU) * D * 256 + 1024;
  static_assert(smem + sizeof(MsShared<D>) <= 232448, "shared memory");
  CUDA_CHECK_RET(cudaFuncSetAttribute(shaped_mass_kernel<D, CAP, BIAS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3((5 * MsCfg<D>::NT + MS_LOADERS) * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  // as many clusters as the device holds at once (fewer than its SMs would make: a cluster stays inside a GPC), looked up once for each device
  static std::atomic<int> held[64][3];
  int dev = 0;
  CUDA_CHECK_RET(cudaGetDevice(&dev));
  int clusters = dev < 64 ? held[dev][p.cluster].load(std::memory_order_relaxed) : 0;
  if (clusters == 0) {
    cfg.gridDim = dim3((unsigned)p.cluster);
    cfg.numAttrs = 1;
    CUDA_CHECK_RET(cudaOccupancyMaxActiveClusters(&clusters, shaped_mass_kernel<D, CAP, BIAS>, &cfg));
    if (clusters < 1) return -164;
    if (dev < 64) held[dev][p.cluster].store(clusters, std::memory_order_relaxed);
  }
  cfg.gridDim = dim3((unsigned)(clusters * p.cluster));
  cfg.numAttrs = p.pdl ? 2 : 1;
  CUDA_CHECK_RET(cudaLaunchKernelEx(&cfg, shaped_mass_kernel<D, CAP, BIAS>, p));
  return 0;
}

}  // namespace smc

// q [T] rows of Hq * D bf16 values with their lse [T, Hq]; runs as in smc_shaped_prompt, every row once; mass [bt_rows, Hkv, mass_stride] fp32.
SMC_API int smc_shaped_mass(const void* q, long long ld_q, const void* k_pool, int n_pages, const int* block_table, long long bt_pitch, int bt_rows,
                            const int* key_pos, int kp_stride, const int* runs, int n_runs, const float* lse, float* mass, long long mass_stride,
                            int T, int Hq, int Hkv, int D, float scale, float cap, const float* slopes, const int* bounds, int* status, int pdl,
                            cudaStream_t st) {
  using namespace smc;
  if (n_runs <= 0 || T <= 0) return 0;
  if (Hkv < 1 || Hq < Hkv || Hq % Hkv || Hq / Hkv > 128 || (D != 64 && D != 128 && D != 256)) return -160;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(runs)) & 15 || (ld_q & 7) || ld_q > (1 << 23) ||
      (reinterpret_cast<uintptr_t>(bounds) & 7))
    return -161;
  if (!shaped_scores_fit(scale, cap)) return -162;
  if (!pitch_fits(bt_pitch) || n_pages < 0 || mass_stride < pitch_cols(bt_pitch)) return -163;
  ShapedMassParams p;
  p.c = shaped_cache(block_table, bt_pitch, bt_rows, n_pages, key_pos, kp_stride, bounds, slopes, scale, cap);
  p.q = (const __nv_bfloat16*)q; p.k_pool = (const __nv_bfloat16*)k_pool; p.runs = (const int4*)runs; p.lse = lse; p.mass = mass;
  p.ld_q = ld_q; p.mass_stride = mass_stride; p.n_runs = n_runs; p.T = T; p.Hq = Hq; p.Hkv = Hkv; p.pdl = pdl; p.status = status;
  p.share_from = MS_SHARED_STEPS * (128 / (Hq / Hkv));
  p.cluster = T >= p.share_from ? 2 : 1;      // clusters only where a sequence may bring that many steps
#define SMC_SHAPED_MASS(DD)                                                                                            \
  if (D == DD) {                                                                                                       \
    if (cap > 0.f) return slopes ? launch_shaped_mass<DD, true, true>(p, st) : launch_shaped_mass<DD, true, false>(p, st); \
    return slopes ? launch_shaped_mass<DD, false, true>(p, st) : launch_shaped_mass<DD, false, false>(p, st);          \
  }
  SMC_SHAPED_MASS(64)
  SMC_SHAPED_MASS(128)
  SMC_SHAPED_MASS(256)
#undef SMC_SHAPED_MASS
  return -160;
}
