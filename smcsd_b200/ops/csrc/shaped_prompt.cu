// Attention of prompts over the paged cache with capped, distance-biased or interval-masked scores (shaped.cuh), on tcgen05.
//
// A CTA takes NT tiles of 128 query rows of one KV head (consecutive tokens of a sequence x the query heads that share the KV head)
// and walks the keys that any of its tokens sees in steps of BK:
//     S_t = Q_t K^T      UMMA 128 x BK x D, scores in tensor memory
//     softmax            four warps per row tile, one query row per thread: the shape of the scores, then P = exp2(x - m_ref) as bf16 over the
//                        scores, in tensor memory
//     O_t += P_t V       UMMA 128 x D x BK accumulating in tensor memory, P its left operand there
// m_ref moves only when the row maximum has grown by more than 2^8.  Sums stay in fp32 ahead of the rounding of P to bf16.
// The shape of the scores costs little beside the exponential: a tanh is a polynomial whose last operation also takes the reference off (four
// operations a pair of scores instead of one), a distance is linear over a step from its nearest key on and one operation more; only steps that a row sees in part, and
// scores far beyond the polynomial, are shaped number by number.  (Shaped in a pass of their own ahead of the maximum: 8192 tokens capped 986 us, folded 772.)  What a
// tanh still costs is in part registers: with heads of 64 and 128 the capped variants spill some 350 bytes a thread, the others up to 12.
//
// What bounds it is the chain of a step: 4700 cycles for 128 keys and two row tiles, of which the exponentials take 2048 and the products, with heads of
// 128, 2048.  A row tile waits 1750 cycles for P V and the next scores (the second waits for the first: the probabilities lie over
// the scores, tensor memory holds no more), reads and takes the maximum in 650 and its exponentials in 1450; the two tiles take turns at those, and the first half of
// P goes to the tensor cores while the second is made.  Taken back: half a row per thread on twice the warps (heads of 128 654 -> 785 us, of 64 555 -> 523),
// steps of 64 keys with two score buffers and the next scores shaped between the exponentials (654 -> 810), probabilities beside the scores for heads of
// 64 and 256 (555 -> 586, 658 -> 849), a quarter of the exponentials by polynomial (610 -> 600).
// Microseconds on B200 (device times, graphs replayed), 8192 causal tokens: 32/8 heads of 128 646 (0.85 PFLOP/s), capped 772, distance bias 811, both 941; of 64 553 and 687 capped;
// 16/2 heads of 256 719 and 871.  Tokens behind a thinned-out cache (pages in any order): two portions of 411 and 512 behind 6000, heads of 256, 63; three turns of 37 to 181
// tokens 17, of them 4.5 until the first scores.
// Tiles are found on the device, the longest walks first: nothing but the number of tokens and sequences has to be known at the launch.
// Every mbarrier wait is bounded; a timeout raises a status bit and all roles unwind.
#include "shaped.cuh"
#include "tmap_host.h"

namespace smc {

constexpr int SP_LOADERS = 4;
// Two row tiles: 512 threads start with 128 registers each; a softmax thread, which holds 128 scores, takes some from the others.
constexpr int SP_FEW = 56, SP_MANY = 200;
static_assert(256 * SP_FEW + 256 * SP_MANY <= 512 * 128, "the registers of the launch");

// Row tiles of a CTA, keys of a step, score buffers of a row tile, slots of the ring (each K or V of a step).
template <int D> struct SpCfg;
template <> struct SpCfg<64> { static constexpr int NT = 2, BK = 128, SB = 1, UNITS = 8; };
template <> struct SpCfg<128> { static constexpr int NT = 2, BK = 128, SB = 1, UNITS = 5; };
template <> struct SpCfg<256> { static constexpr int NT = 1, BK = 64, SB = 2, UNITS = 5; };

constexpr float SP_NONE = -67108864.f;                // below any position, whatever is added

struct ShapedPromptParams {
  ShapedCache c;
  const __nv_bfloat16* q;        // [T] rows of Hq * D, ld_q apart
  const __nv_bfloat16* k_pool;   // [pages + 1, Hkv * D]
  const __nv_bfloat16* v_pool;
  const int4* runs;
  __nv_bfloat16* out;            // [T] rows of Hq * D, ld_out apart
  float* lse;                    // [T, Hq] or null
  long long ld_q, ld_out;
  int n_runs, T, Hq, Hkv, pdl;
  int* status;
};

template <int D> struct SpShared {
  static constexpr int SLOTS = SpCfg<D>::UNITS / 2 + 1;               // steps whose keys' positions are held
  uint64_t kv_full[SpCfg<D>::UNITS], kv_empty[SpCfg<D>::UNITS], q_full[2], s_full[2][2], p_full[2][2][2], o_done[2][2], pos_full[SLOTS], turn[2][4];
  alignas(16) float pos[SLOTS][SpCfg<D>::BK];         // of a step's keys, less that of the first or, with distances, of the one nearest the tile's tokens; SP_NONE behind the last
  float pos_near[SLOTS];
  uint32_t tmem_slot;
  int lo[8], hi[8], begin, end[2];
  volatile int abort;
};

template <typename Shared>
__device__ __forceinline__ bool sp_wait(Shared& S, int* status, uint64_t* bar, uint32_t parity) {
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

__device__ __forceinline__ uint32_t sp_pack(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// D[tmem] (+)= A[tmem] * B[smem]: A rows are lanes, two bf16 values of K to a column
__device__ __forceinline__ void sp_umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n"
      ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Tile number `want` (0: most steps) of all tiles of `tokens` tokens, by a whole warp; run number and tile inside it, or false behind the
// last.  The tiles of a sequence with at least c steps of `bk` keys are its last ones, so counting them is arithmetic and c of the
// wanted one is found by bisection.
__device__ __forceinline__ bool sp_find_tile(const ShapedCache& c, const int4* runs, int n_runs, int T, int* status, int tokens, int bk, int launched, int want,
                                             ShapedRun& run, int& tile) {
  const int lane = threadIdx.x & 31;
  const ShapedRun mine = lane < n_runs ? shaped_run(c, runs, lane, T, status) : ShapedRun{0, 0, 0, 0};
  // tiles of run r with at least `cost` steps
  auto of_run = [&](const ShapedRun& r, int cost) {
    const long long y = (long long)(cost - 1) * bk - r.held;         // tokens ahead of these tiles' ends, less one
    if (r.n <= 0 || y >= r.n) return 0;
    return (r.n + tokens - 1) / tokens - (y > 0 ? (int)(y / tokens) : 0);
  };
  auto count = [&](int cost) {
    int n = of_run(mine, cost);
    for (int s = lane + 32; s < n_runs; s += 32) n += of_run(shaped_run(c, runs, s, T, status), cost);
    return (int)__reduce_add_sync(0xffffffffu, (unsigned)n);
  };
  const int tiles = count(1);
  if (tiles > launched && want == 0 && threadIdx.x == 0) atomicOr(status, SMC_ERR_BOUNDS);      // tokens of q in two runs: more tiles than q has
  if (tiles <= want) return false;
  int lo = 1, hi = c.bt_cols / bk + 2;                                // count(lo) > want >= count(hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (count(mid) > want) lo = mid; else hi = mid;
  }
  int left = want - count(lo + 1);                                    // which of the tiles with exactly `lo` steps
  for (int s0 = 0; s0 < n_runs; s0 += 32) {
    const ShapedRun r = s0 == 0 ? mine : s0 + lane < n_runs ? shaped_run(c, runs, s0 + lane, T, status) : ShapedRun{0, 0, 0, 0};
    const int with = of_run(r, lo), n = with - of_run(r, lo + 1);
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
      tile = __shfl_sync(0xffffffffu, (r.n + tokens - 1) / tokens - with + left - (sum - n), src);
      return true;
    }
    left -= __shfl_sync(0xffffffffu, sum, 31);
  }
  return false;
}

template <int D, bool CAP, bool BIAS>
__global__ void __launch_bounds__(SpCfg<D>::NT == 2 ? 512 : 384, 1)
shaped_prompt_kernel(const ShapedPromptParams p, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV) {
  constexpr int NT = SpCfg<D>::NT, UNITS = SpCfg<D>::UNITS, BK = SpCfg<D>::BK, SB = SpCfg<D>::SB;
  constexpr int HALVES = BK / 64;                     // parts of a step's probabilities that are handed over on their own
  constexpr int KPW = BK / SP_LOADERS, KL = BK / 32;  // keys gathered by one loader warp; keys whose page a lane knows
  constexpr int NPAN = D / 64;                        // 64-element (128-byte) panels along the head dimension
  constexpr int PANEL_Q = 128 * 128, PANEL_KV = BK * 128;
  constexpr int Q_BYTES = NPAN * PANEL_Q, KV_BYTES = NPAN * PANEL_KV;
  constexpr int CPR = D / 8;                          // 16-byte chunks per row
  constexpr uint32_t COL_O = NT * SB * BK;            // tensor memory: scores (t * SB + buffer) * BK, probabilities over them, outputs behind
  static_assert(COL_O + NT * D <= 512, "tensor memory");
  using Shared = SpShared<D>;
  constexpr int SLOTS = Shared::SLOTS;
  extern __shared__ uint8_t sp_smem_raw[];
  __shared__ Shared S;
  const uint32_t raw = smem_u32(sp_smem_raw);
  uint8_t* smem = sp_smem_raw + (((raw + 1023u) & ~1023u) - raw);
  uint8_t* q_s = smem;
  uint8_t* kv_s = q_s + NT * Q_BYTES;                 // [unit]: K of step 0, V of step 0, K of step 1, ...

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int LOAD_WARP = 4 * NT, MMA_WARP = 4 * NT + SP_LOADERS;      // softmax, loaders, one issuer per row tile
  const int G = p.Hq / p.Hkv, TT = 128 / G;           // tokens of a row tile
  const int kvh = blockIdx.x % p.Hkv, hbase = kvh * G;
  if (p.pdl) { pdl_launch_dependents(); pdl_wait_prior_grid(); }

  ShapedRun run;
  int tile;
  if (!sp_find_tile(p.c, p.runs, p.n_runs, p.T, p.status, NT * TT, BK, gridDim.x / p.Hkv, blockIdx.x / p.Hkv, run, tile)) return;
  const int first = run.held + tile * NT * TT, tok0 = run.at + tile * NT * TT;       // index in the row and in q of the first token
  const int count = min(NT * TT, run.n - tile * NT * TT), keys = run.held + run.n;
  const int* kp = p.c.key_pos != nullptr ? p.c.key_pos + (size_t)run.row * p.c.kp_stride : nullptr;

  if (threadIdx.x == 0) {
    for (int s = 0; s < UNITS; ++s) {
      mbar_init(&S.kv_full[s], SP_LOADERS);
      mbar_init(&S.kv_empty[s], NT);
    }
    for (int s = 0; s < SLOTS; ++s) mbar_init(&S.pos_full[s], SP_LOADERS);
    for (int t = 0; t < NT; ++t) {
      mbar_init(&S.q_full[t], 4);
      for (int q = 0; q < 4; ++q) mbar_init(&S.turn[t][q], 1);
      for (int i = 0; i < SB; ++i) {
        mbar_init(&S.s_full[t][i], 1);
        mbar_init(&S.p_full[t][i][0], 4);
        mbar_init(&S.p_full[t][i][1], 4);
        mbar_init(&S.o_done[t][i], 1);
      }
    }
    S.abort = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == MMA_WARP) {
    tmem_alloc(&S.tmem_slot, 512);
    tmem_relinquish();
  }
  // positions of this thread's query row, the interval it sees, and the union over each row tile
  const int t_row = warp >> 2, r = (warp & 3) * 32 + lane, tk = t_row * TT + r / G;
  const bool live = warp < LOAD_WARP && r < TT * G && tk < count;
  int2 see = make_int2(SH_POS_END, -1);
  float pos_row = 0.f;
  if (live) {
    const int pos = kp != nullptr ? kp[first + tk] : first + tk;
    see = shaped_bounds(p.c, tok0 + tk, pos);
    pos_row = (float)pos;
  }
  if (warp < LOAD_WARP) {
    const int lo = __reduce_min_sync(0xffffffffu, see.x), hi = __reduce_max_sync(0xffffffffu, see.y);
    if (lane == 0) { S.lo[warp] = lo; S.hi[warp] = hi; }
  }
  __syncthreads();
  if (warp < 1 + NT) {                                // positions -> run of the row
    int lo = SH_POS_END, hi = -1;
    for (int w = 0; w < 4 * NT; ++w) {
      if (warp == 0 || (w >> 2) == warp - 1) { lo = min(lo, S.lo[w]); hi = max(hi, S.hi[w]); }
    }
    const int v = warp == 0 ? lo : hi + 1;
    const int at = kp != nullptr ? shaped_lower_bound(kp, keys, v) : min(v, keys);
    if (lane == 0) {
      if (warp == 0) S.begin = at; else S.end[warp - 1] = at;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = S.tmem_slot;
  const int begin = S.begin, end_all = max(S.end[0], S.end[NT - 1]);
  int n_of[2];                                        // key steps of each row tile
  n_of[0] = max(0, (S.end[0] - begin + BK - 1) / BK);
  n_of[1] = NT > 1 ? max(0, (S.end[NT - 1] - begin + BK - 1) / BK) : 0;
  const int n_steps = max(n_of[0], n_of[1]);

  if (warp >= LOAD_WARP && warp < MMA_WARP) {
    // ================================================================= loaders
    if constexpr (NT == 2) regs_fewer<SP_FEW>();
    const int lw = warp - LOAD_WARP;
    const int* bt = p.c.block_table + (size_t)run.row * p.c.bt_stride;
    const size_t kv_row = (size_t)p.Hkv * D;
    // every loader warp reads all page ids of a step (lane l: keys l, l + 32, ...) and comes to the same decision for each 64 of them
    auto checked = [&](int page) {
      if (page >= 0 && page <= p.c.n_pages) return page;
      atomicOr(p.status, SMC_ERR_BOUNDS);
      return 0;
    };
    constexpr int LAG = 1, PD = 2;                     // gathered units in flight behind the newest (a unit is handed over LAG later, when as many more slots are free); steps that page ids are read ahead
    int issued = 0;
    uint32_t gathered = 0;                            // bit (u & 31): this warp's part of unit u went through cp.async (arrival still owed)
    int pg[PD][KL], pk[PD], pn[PD];
    auto ahead = [&](int step, int (&ids)[KL], int& pos, int& near_pos) {
#pragma unroll
      for (int i = 0; i < KL; ++i) ids[i] = step < n_steps ? bt[min(begin + step * BK + i * 32 + lane, end_all - 1)] : 0;
      const int k0 = begin + step * BK, k = k0 + lw * KPW + lane;      // the positions this warp hands over
      pos = lane < KPW && k < end_all ? (kp != nullptr ? kp[k] : k) : -1;
      const int k_near = !BIAS || k0 >= first ? k0 : min(k0 + BK, end_all) - 1;  // keys in front of the tile's tokens: the last one
      near_pos = k0 < end_all ? (kp != nullptr ? kp[k_near] : k_near) : 0;
    };
#pragma unroll
    for (int d = 0; d < PD; ++d) ahead(d, pg[d], pk[d], pn[d]);
    bool go = true;
    const uint64_t pol = l2_policy_evict_last();      // the other row tiles of this KV head read the same keys
    for (int j0 = 0; go && j0 < n_steps; j0 += PD) {
#pragma unroll
      for (int d = 0; d < PD; ++d) {
        const int j = j0 + d;
        if (!go || j >= n_steps) break;
        int page[KL];
#pragma unroll
        for (int i = 0; i < KL; ++i) page[i] = checked(pg[d][i]);
        const float pos = pk[d] < 0 ? SP_NONE : (float)(pk[d] - pn[d]), pos_near = (float)pn[d];
        ahead(j + PD, pg[d], pk[d], pn[d]);
        int base[KL / 2];
        bool rows_run[KL / 2];
#pragma unroll
        for (int h = 0; h < KL / 2; ++h) {            // 64 consecutive pages come by TMA
          base[h] = __shfl_sync(0xffffffffu, page[2 * h], 0);
          rows_run[h] = __all_sync(0xffffffffu, page[2 * h] == base[h] + lane && page[2 * h + 1] == base[h] + 32 + lane) && base[h] >= 1;
        }
        const int half = lw * KPW / 64;
        const bool mine_run = KL == 2 || half == 0 ? rows_run[0] : rows_run[KL / 2 - 1];
        const bool lead = lw * KPW % 64 == 0;         // issues its half's copies
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const int u = 2 * j + kv, st = u % UNITS, use = u / UNITS;
          const bool ok = use < 1 || sp_wait(S, p.status, &S.kv_empty[st], (uint32_t)(use - 1) & 1u);
          if (!__all_sync(0xffffffffu, ok)) { go = false; break; }
          if (kv == 0) {                              // the ring of positions turns with the keys
            if (lane < KPW) S.pos[j % SLOTS][lw * KPW + lane] = pos;
            if (lw == 0 && lane == 0) S.pos_near[j % SLOTS] = pos_near;
            __syncwarp();
            if (lane == 0) mbar_arrive(&S.pos_full[j % SLOTS]);
          }
          uint8_t* ptr = kv_s + (size_t)st * KV_BYTES;
          if (mine_run) {
            if (lane == 0) {
              if (lead) {
                const int b0 = KL == 2 || half == 0 ? base[0] : base[KL / 2 - 1];
                mbar_expect_tx(&S.kv_full[st], NPAN * 64 * 128);
#pragma unroll
                for (int pan = 0; pan < NPAN; ++pan)
                  tma_load_2d(ptr + pan * PANEL_KV + half * 64 * 128, kv ? &tmV : &tmK, &S.kv_full[st], kvh * D + pan * 64, b0, pol);
              } else {
                mbar_arrive(&S.kv_full[st]);
              }
            }
            gathered &= ~(1u << (u & 31));
          } else {
            const uint32_t dst0 = smem_u32(ptr);
            const __nv_bfloat16* pool = kv ? p.v_pool : p.k_pool;
#pragma unroll 4
            for (int idx = lane; idx < KPW * CPR; idx += 32) {
              const int kl = idx / CPR, c = idx % CPR, key = lw * KPW + kl;
              int mine = page[0];
#pragma unroll
              for (int i = 1; i < KL; ++i) mine = lw * KPW / 32 == i ? page[i] : mine;
              const int pgi = __shfl_sync(0xffffffffu, mine, key & 31);
              const uint32_t dst = dst0 + (uint32_t)((c >> 3) * PANEL_KV + key * 128 + (((c & 7) ^ (key & 7)) << 4));
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(pool + (size_t)pgi * kv_row + (size_t)kvh * D + c * 8) : "memory");
            }
            gathered |= 1u << (u & 31);
          }
          asm volatile("cp.async.commit_group;" ::: "memory");     // one group per unit (empty for a TMA unit)
          if (u >= LAG && ((gathered >> ((u - LAG) & 31)) & 1u)) { // gathered unit u - LAG has landed: hand it over
            asm volatile("cp.async.wait_group %0;" ::"n"(LAG) : "memory");
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&S.kv_full[(u - LAG) % UNITS]);
          }
          ++issued;
        }
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    fence_proxy_async();
    __syncwarp();
    if (lane == 0)
      for (int u = max(0, issued - LAG); u < issued; ++u)
        if ((gathered >> (u & 31)) & 1u) mbar_arrive(&S.kv_full[u % UNITS]);
    // an aborted CTA keeps its shared memory until the copies in flight have landed
    if (S.abort && lane == 0 && lw * KPW % 64 == 0)
      for (int u = max(0, issued - UNITS); u < issued; ++u)
        if (!((gathered >> (u & 31)) & 1u)) (void)mbar_wait(&S.kv_full[u % UNITS], (uint32_t)(u / UNITS) & 1u);
  } else if (warp >= MMA_WARP) {
    // ================================================================= MMA issuers (one thread per row tile)
    if constexpr (NT == 2) regs_fewer<SP_FEW>();
    const int t = warp - MMA_WARP;
    if (t < NT && elect_one()) {
      const int n = n_of[t];
      constexpr uint32_t idesc_s = umma_idesc_bf16(128, BK);
      constexpr uint32_t idesc_o = umma_idesc_bf16(128, D) | (1u << 16);       // B operand (V) is MN-major
      const uint32_t q_addr = smem_u32(q_s) + t * Q_BYTES;
      const uint32_t tS = tmem_base + (uint32_t)(t * SB * BK), tO = tmem_base + COL_O + t * D;
      auto wait_unit = [&](int u) { return sp_wait(S, p.status, &S.kv_full[u % UNITS], (uint32_t)(u / UNITS) & 1u); };
      auto issue_s = [&](int j) -> bool {
        if (!wait_unit(2 * j)) return false;
        // the buffer is free once the product of the probabilities that it holds is done
        if (j >= SB && !sp_wait(S, p.status, &S.o_done[t][j % SB], (uint32_t)(j / SB - 1) & 1u)) return false;
        tc_fence_after();
        const uint32_t k_addr = smem_u32(kv_s + (size_t)(2 * j % UNITS) * KV_BYTES);
#pragma unroll
        for (int pan = 0; pan < NPAN; ++pan)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_bf16_ss(tS + (uint32_t)(j % SB) * BK, umma_desc_k_sw128(q_addr + pan * PANEL_Q) + 2 * k,
                         umma_desc_k_sw128(k_addr + pan * PANEL_KV) + 2 * k, idesc_s, (pan | k) ? 1u : 0u);
        umma_commit(&S.s_full[t][j % SB]);
        umma_commit(&S.kv_empty[2 * j % UNITS]);
        return true;
      };
      bool ok = n == 0 || sp_wait(S, p.status, &S.q_full[t], 0);
      for (int j = 0; ok && j < min(n, SB); ++j) ok = issue_s(j);
      for (int j = 0; ok && j < n; ++j) {
        if (!wait_unit(2 * j + 1)) { ok = false; break; }
        const uint32_t v_addr = smem_u32(kv_s + (size_t)((2 * j + 1) % UNITS) * KV_BYTES);
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {            // the first half of the keys while the second takes its exponentials
          if (!ok || !(ok = sp_wait(S, p.status, &S.p_full[t][j % SB][h], (uint32_t)(j / SB) & 1u))) break;
          tc_fence_after();
#pragma unroll
          for (int k = h * 4; k < h * 4 + 4; ++k)
            sp_umma_ts(tO, tS + (uint32_t)(j % SB) * BK + 8 * k, umma_desc_mn_sw128(v_addr + k * 2048, PANEL_KV), idesc_o, (j | k) ? 1u : 0u);
        }
        if (!ok) break;
        umma_commit(&S.o_done[t][j % SB]);            // O_t holds the sum over steps 0..j
        umma_commit(&S.kv_empty[(2 * j + 1) % UNITS]);
        if (j + SB < n) ok = issue_s(j + SB);
      }
      // steps that only the other tile's rows see
      for (int u = 2 * n; ok && u < 2 * n_steps; ++u) {
        ok = wait_unit(u);
        if (ok) mbar_arrive(&S.kv_empty[u % UNITS]);
      }
    }
    __syncwarp();
  } else if (warp < LOAD_WARP) {
    // ================================================================= softmax (one query row per thread)
    if constexpr (NT == 2) regs_more<SP_MANY>();
    const int t = t_row, n = n_of[t];
    const uint32_t lane_off = ((uint32_t)((warp & 3) * 32)) << 16;
    const uint32_t tO = tmem_base + COL_O + t * D + lane_off;
    // this tile's query rows r = token * G + head, zero padded to 128, into swizzled K-major panels: a row per thread
    {
      const uint4* src = reinterpret_cast<const uint4*>(p.q + (size_t)(tok0 + tk) * p.ld_q + (size_t)(hbase + r % G) * D);
      uint8_t* dst = q_s + t * Q_BYTES + r * 128;
#pragma unroll
      for (int c0 = 0; c0 < CPR; c0 += 8) {
        uint4 v[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] = live ? src[c0 + c] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(dst + (c0 >> 3) * PANEL_Q + ((c ^ (r & 7)) << 4)) = v[c];
      }
    }
    fence_proxy_async();                              // generic-proxy writes before the tensor core reads them
    __syncwarp();
    if (lane == 0) mbar_arrive(&S.q_full[t]);
    // rows behind the last token mask nothing, so that they do not send their warp the long way
    const float first_seen = live ? (float)see.x : 0.f, last_seen = live ? (float)see.y : (float)SH_POS_END;
    const float mul = p.c.mul, cap_in = p.c.cap_in, cap_out = p.c.cap_out;
    const float slope = BIAS && live ? -p.c.slopes[hbase + r % G] * SH_LOG2E : 0.f;
    const ShapedCapNear<3> near(cap_in, cap_out, mul);
    float m_ref = -INFINITY;                          // exponent reference of the row (log2 domain); -inf until it has seen a key
    uint64_t sum[2] = {0ull, 0ull};                   // its running sum, in four parts
    bool alive = true;
    for (int j = 0; j < n; ++j) {
      if (!__all_sync(0xffffffffu, sp_wait(S, p.status, &S.s_full[t][j % SB], (uint32_t)(j / SB) & 1u) &&
                                       sp_wait(S, p.status, &S.pos_full[j % SLOTS], (uint32_t)(j / SLOTS) & 1u))) { alive = false; break; }
      tc_fence_after();
      const float* pos = S.pos[j % SLOTS];
      const uint32_t ts = tmem_base + (uint32_t)((t * SB + j % SB) * BK) + lane_off;
      // Where the step lies, ahead of its scores where distances make this longer.  Its keys ascend, those behind the last (position -1) come at its end.
      float nearest, pos0, pos1;
      bool plain, behind = false;
      auto place = [&] {
        nearest = S.pos_near[j % SLOTS];
        pos0 = BIAS ? nearest + pos[0] : nearest;
        pos1 = nearest + pos[BK - 1];
        bool mine = pos0 >= first_seen && pos1 >= 0.f && pos1 <= last_seen;
        if (BIAS) {
          // A distance is linear over the step from its nearest key on; taken from the farthest one, beyond a gap in the positions, the near ones would be differences of
          // large numbers.  So the row has to lie beyond that key (one inside the step looks both ways), and where far keys gain the step has to be short.
          behind = nearest == pos1;
          mine = mine && (slope == 0.f || (behind ? pos_row >= pos1 : pos_row <= pos0)) && slope * (pos1 - pos0) <= 16.f;
        }
        plain = __all_sync(0xffffffffu, mine);
      };
      if (BIAS) place();
      uint32_t x[BK];
#pragma unroll
      for (int c0 = 0; c0 < BK; c0 += 16) tmem_ld_32x32b_x16(ts + c0, *reinterpret_cast<uint32_t(*)[16]>(&x[c0]));
      tmem_ld_wait();
      auto val = [&](int i) { return __uint_as_float(x[i]); };
      auto pair = [&](int i) { return f2_pair(val(i), val(i + 1)); };
      // The shape of the scores is folded into the exponentials below: a tanh is monotone and a distance costs most at one end of the step, so the
      // largest score and the distance of that end give a reference that no score exceeds, by no more than the step's scores differ.
      float mx[2] = {-INFINITY, -INFINITY}, mn[2] = {INFINITY, INFINITY};
#pragma unroll
      for (int i = 0; i < BK; i += 4) {
        mx[0] = shaped_max3(mx[0], val(i), val(i + 1));
        mx[1] = shaped_max3(mx[1], val(i + 2), val(i + 3));
        if (CAP || BIAS) {
          mn[0] = shaped_min3(mn[0], val(i), val(i + 1));
          mn[1] = shaped_min3(mn[1], val(i + 2), val(i + 3));
        }
      }
      const float most = fmaxf(mx[0], mx[1]), least = fminf(mn[0], mn[1]), reach = fmaxf(most, -least) * cap_in;
      if (!BIAS) place();
      // 0: scores as they are after this; 1: tanh by three coefficients (or none); 2: by five
      int way = 1;
      if (!plain || (BIAS && __any_sync(0xffffffffu, !((most - least) * mul < 60.f)))) way = 0;
      else if (CAP && __any_sync(0xffffffffu, !(reach <= p.c.near_reach))) way = __any_sync(0xffffffffu, !(reach <= SH_TANH5_REACH)) ? 0 : 2;
      float top;
      if (way != 0) {
        top = CAP ? shaped_cap(most, cap_in, cap_out) : most * mul;
        if (BIAS) {
          const float a = fabsf(pos0 - pos_row), b = fabsf(pos1 - pos_row);
          top += slope * (slope > 0.f ? fmaxf(a, b) : fminf(a, b));
        }
      } else {
        // (the few scores beyond reach in a loop of their own: between the others their code would lie 64 times in the way, 10 us of a first step)
        const ShapedCapNear<5> by_five(cap_in, cap_out, mul);
        if (CAP && __any_sync(0xffffffffu, !(reach <= SH_TANH5_REACH))) {
#pragma unroll
          for (int i = 0; i < BK; ++i) x[i] = __float_as_uint(shaped_cap(val(i), cap_in, cap_out));
        } else {
#pragma unroll
          for (int i = 0; i < BK; i += 2) {
            const float2 v = f2_unpair(CAP ? by_five(pair(i), 0ull) : f2_mul(pair(i), f2_pair(mul, mul)));
            x[i] = __float_as_uint(v.x);
            x[i + 1] = __float_as_uint(v.y);
          }
        }
        top = -INFINITY;
#pragma unroll
        for (int i = 0; i < BK; ++i) {
          const float at = nearest + pos[i];
          float v = val(i);
          if (BIAS) v = fmaf(fabsf(at - pos_row), slope, v);
          v = at >= first_seen && at <= last_seen ? v : -INFINITY;    // probability zero
          x[i] = __float_as_uint(v);
          top = fmaxf(top, v);
        }
      }
      const bool grow = top > m_ref + 8.f;            // also true for the first visible key (m_ref = -inf)
      if (j >= 1 && __any_sync(0xffffffffu, grow)) {
        // rare after the first steps: PV of step j - 1 must have completed before O is rescaled in tensor memory
        if (!__all_sync(0xffffffffu, sp_wait(S, p.status, &S.o_done[t][(j - 1) % SB], (uint32_t)((j - 1) / SB) & 1u))) { alive = false; break; }
        tc_fence_after();
        const float alpha = grow ? exp2f(m_ref - top) : 1.f;
#pragma unroll
        for (int c0 = 0; c0 < D; c0 += 16) {
          uint32_t o[16];
          tmem_ld_32x32b_x16(tO + c0, o);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
          tmem_st_32x32b_x16(tO + c0, o);
        }
        tmem_st_wait();
        const uint64_t alpha2 = f2_pair(alpha, alpha);
        sum[0] = f2_mul(sum[0], alpha2);
        sum[1] = f2_mul(sum[1], alpha2);
      }
      if (grow) m_ref = top;
      const float ref = m_ref == -INFINITY ? 0.f : m_ref;             // a row that has seen nothing yet: every probability is exp2(-inf)
      // The two warps that share a scheduler (same quarter of either tile) take turns at the exponentials, tile 0 first: one waits for its scores and
      // looks for its maxima meanwhile.
      if (NT > 1) {
        const int q = warp & 3;
        const bool in_turn = t ? j >= n_of[0] || sp_wait(S, p.status, &S.turn[1][q], (uint32_t)j & 1u)
                               : j == 0 || j > n_of[1] || sp_wait(S, p.status, &S.turn[0][q], (uint32_t)(j - 1) & 1u);
        if (!__all_sync(0xffffffffu, in_turn)) { alive = false; break; }
      }
      // exp2 of what `shaped` makes of the pairs, 64 keys after the other
      auto exponentials = [&](auto shaped) {
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
#pragma unroll
          for (int c0 = h * 64; c0 < h * 64 + 64; c0 += 32) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const float2 e = f2_unpair(shaped(c0 + i));
              const float p0 = shaped_ex2(e.x), p1 = shaped_ex2(e.y);
              sum[(i >> 1) & 1] = f2_add(sum[(i >> 1) & 1], f2_pair(p0, p1));
              pk[i >> 1] = sp_pack(p0, p1);
            }
            tmem_st_32x32b_x16(ts + (c0 >> 1), pk);
          }
          if (NT > 1 && h == HALVES - 1 && lane == 0) mbar_arrive(&S.turn[t ^ 1][warp & 3]);
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&S.p_full[t][j % SB][h]);
        }
      };
      const uint64_t mul2 = f2_pair(mul, mul), off = f2_pair(-ref, -ref);
      // distance's share less the reference, from the nearest key on
      const float per = behind ? -slope : slope, start = fmaf(slope, fabsf(nearest - pos_row), -ref);
      const uint64_t per2 = f2_pair(per, per), start2 = f2_pair(start, start);
      auto away = [&](int i) {
        if (!BIAS) return off;
        uint64_t at;                                  // volatile: read where it is used, the scores leave no room for all of them
        asm volatile("ld.shared.b64 %0, [%1];" : "=l"(at) : "r"(smem_u32(pos + i)));
        return f2_fma(at, per2, start2);
      };
      if (way == 0) exponentials([&](int i) { return f2_add(pair(i), off); });
      else if (!CAP) exponentials([&](int i) { return f2_fma(pair(i), mul2, away(i)); });
      else if (way == 1) exponentials([&](int i) { return near(pair(i), away(i)); });
      else {
        const ShapedCapNear<5> far(cap_in, cap_out, mul);
        exponentials([&](int i) { return far(pair(i), away(i)); });
      }
    }
    // the last product is done: read the accumulated O once
    if (alive && n > 0)
      alive = __all_sync(0xffffffffu, sp_wait(S, p.status, &S.o_done[t][(n - 1) % SB], (uint32_t)((n - 1) / SB) & 1u));
    tc_fence_after();
    if (alive) {
      const size_t at = (size_t)(tok0 + tk) * p.ld_out + (size_t)(hbase + r % G) * D;
      const float2 s0 = f2_unpair(sum[0]), s1 = f2_unpair(sum[1]);
      const float total = (s0.x + s0.y) + (s1.x + s1.y);
      const bool none = m_ref == -INFINITY && total == 0.f;           // nothing visible
      const float inv = 1.f / total;
      if (live && p.lse != nullptr)
        p.lse[(size_t)(tok0 + tk) * p.Hq + hbase + r % G] = none ? -INFINITY : SH_LN2 * (m_ref + __log2f(total));
#pragma unroll
      for (int c0 = 0; c0 < D; c0 += 32) {
        uint32_t o[32];
        if (n > 0) {
          tmem_ld_32x32b_x16(tO + c0, *reinterpret_cast<uint32_t(*)[16]>(&o[0]));
          tmem_ld_32x32b_x16(tO + c0 + 16, *reinterpret_cast<uint32_t(*)[16]>(&o[16]));
          tmem_ld_wait();
        }
        if (live) {
          float v[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = none ? 0.f : __uint_as_float(o[i]) * inv;
          uint4* dst = reinterpret_cast<uint4*>(p.out + at + c0);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            dst[i] = make_uint4(sp_pack(v[8 * i], v[8 * i + 1]), sp_pack(v[8 * i + 2], v[8 * i + 3]), sp_pack(v[8 * i + 4], v[8 * i + 5]),
                                sp_pack(v[8 * i + 6], v[8 * i + 7]));
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) tmem_dealloc(tmem_base, 512);
}

template <int D, bool CAP, bool BIAS>
static int launch_shaped_prompt(const ShapedPromptParams& p, int n_tiles, const CUtensorMap& tmK, const CUtensorMap& tmV, cudaStream_t st) {
  constexpr int NT = SpCfg<D>::NT;
  constexpr size_t smem = (size_t)NT * D * 256 + (size_t)SpCfg<D>::UNITS * SpCfg<D>::BK * D * 2 + 1024;
  static_assert(smem + sizeof(SpShared<D>) <= 232448, "shared memory");
  auto kernel = shaped_prompt_kernel<D, CAP, BIAS>;
  CUDA_CHECK_RET(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  if constexpr (NT == 2) {                            // what the warpgroups ask for later is there from the start
    static const int regs = [&] { cudaFuncAttributes a; return cudaFuncGetAttributes(&a, kernel) == cudaSuccess ? a.numRegs : 0; }();
    if (regs < 128) return -145;
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(n_tiles * p.Hkv));
  cfg.blockDim = dim3(NT == 2 ? 512 : 384);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = p.pdl ? 1 : 0;
  CUDA_CHECK_RET(cudaLaunchKernelEx(&cfg, kernel, p, tmK, tmV));
  return 0;
}

}  // namespace smc

// q, out: T rows of Hq * D bf16 values; runs [n_runs][4] int32 {block-table row, tokens held, index of the first new token in q, new tokens}:
// all tokens of a sequence, the new ones included, are in the pages of its row.  bounds [T][2], slopes [Hq], key_pos, lse [T, Hq] may be null.
SMC_API int smc_shaped_prompt(const void* q, long long ld_q, const void* k_pool, const void* v_pool, int n_pages, const int* block_table,
                              long long bt_pitch, int bt_rows, const int* key_pos, int kp_stride, const int* runs, int n_runs, void* out,
                              long long ld_out, float* lse, int T, int Hq, int Hkv, int D, float scale, float cap, const float* slopes,
                              const int* bounds, int* status, int pdl, cudaStream_t st) {
  using namespace smc;
  if (n_runs <= 0 || T <= 0) return 0;
  if (Hkv < 1 || Hq < Hkv || Hq % Hkv || Hq / Hkv > 128 || (D != 64 && D != 128 && D != 256)) return -140;
  // rows of queries and outputs move in pieces of 16 bytes, a run's numbers in one, a token's bounds in one; the tensor maps look at the pools
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(runs) | reinterpret_cast<uintptr_t>(k_pool) |
       reinterpret_cast<uintptr_t>(v_pool)) & 15)
    return -141;
  if (!pitch_fits(bt_pitch) || n_pages < 0 || (ld_q & 7) || (ld_out & 7) || (reinterpret_cast<uintptr_t>(bounds) & 7)) return -142;
  if (!shaped_scores_fit(scale, cap)) return -143;
  ShapedPromptParams p;
  p.c = shaped_cache(block_table, bt_pitch, bt_rows, n_pages, key_pos, kp_stride, bounds, slopes, scale, cap);
  p.q = (const __nv_bfloat16*)q; p.k_pool = (const __nv_bfloat16*)k_pool; p.v_pool = (const __nv_bfloat16*)v_pool;
  p.runs = (const int4*)runs; p.out = (__nv_bfloat16*)out; p.lse = lse; p.ld_q = ld_q; p.ld_out = ld_out;
  p.n_runs = n_runs; p.T = T; p.Hq = Hq; p.Hkv = Hkv; p.pdl = pdl; p.status = status;
  CUtensorMap tmK, tmV;
  int rc = pool_tmap(&tmK, k_pool, (long long)n_pages + 1, (long long)Hkv * D);
  if (rc == 0) rc = pool_tmap(&tmV, v_pool, (long long)n_pages + 1, (long long)Hkv * D);
  if (rc) return rc;
  const int tokens = (D == 256 ? 1 : 2) * (128 / (Hq / Hkv)), n_tiles = T / tokens + n_runs;     // at most that many
  if ((long long)n_tiles * Hkv > 0x7fffffff) return -144;
#define SMC_SHAPED_PROMPT(DD)                                                                                          \
  if (D == DD) {                                                                                                       \
    if (cap > 0.f) return slopes ? launch_shaped_prompt<DD, true, true>(p, n_tiles, tmK, tmV, st)                      \
                                 : launch_shaped_prompt<DD, true, false>(p, n_tiles, tmK, tmV, st);                    \
    return slopes ? launch_shaped_prompt<DD, false, true>(p, n_tiles, tmK, tmV, st)                                    \
                  : launch_shaped_prompt<DD, false, false>(p, n_tiles, tmK, tmV, st);                                  \
  }
  SMC_SHAPED_PROMPT(64)
  SMC_SHAPED_PROMPT(128)
  SMC_SHAPED_PROMPT(256)
#undef SMC_SHAPED_PROMPT
  return -140;
}
