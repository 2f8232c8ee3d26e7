// Rows of the block table brought down to a budget: the tokens that hold the most attention weight stay.
//
// Of the n tokens of a row the first `first`, the last `last` and, of those between, the ones with the highest weight stay, `keep` in all; equal
// weights go to the lower index.  A token's weight is the fp32 sum over the KV heads in their order.  The kept tokens move up in their order - page ids,
// positions and weights, no key or value - into the same row, whose other tokens lose their references, or into another row, for which
// references are taken.  Pages without a reference go on the free stack, the lowest on top, as the host's form leaves them.
//
// Two kernels.  The first finds out who stays: a cluster of eight blocks to a row (one block alone for a short one; rows with the same source share the
// first one's answer), pieces of 512 tokens going round its blocks.  The n-th highest weight is found by three histograms of 11, 11 and 10 bits over
// order-preserving integers in shared memory, joined over the cluster; a token's place is the number of tokens in front of it that stay, counted by
// warps and joined over all pieces by one scan.  The second moves: a block to a row and head (or to its pages and positions), whose reads of a
// run of places end before its writes, which lie in front of all later reads - so it may be the same row.
// What bounds it: 4 bytes per token and head read once, then barriers and dependent reads; the row that takes longest decides.  (In one kernel, the moves of a cluster
// kept in step by barriers between heads: 115 us for 16 rows of 65,000 tokens and 8 heads from two sources, 50 so; 16 rows of 2,100
// tokens 26: reads of the weights 5, three histograms 5, places 4, moves 5, launches.  In place the block that comes last also looks through the marks of dead pages, a bit for
// every page of the allocator: 16 rows of 2176 tokens to 2048 40 us with 40,000 pages, 57 with 400,000, 184 with 4 million.)
#include "shaped.cuh"

namespace smc {

constexpr int EV_CL = 8, EV_T = 512, EV_BINS = 2048, EV_SOLO = 8192, EV_PIECES = 512;
constexpr int EV_ENTRIES = 4096;                       // rows of a call
constexpr int EV_MOVE = 8;                             // places of a thread between two barriers of the second kernel

struct EvictParams {
  int* table;
  int* key_pos;                                        // or null
  float* mass;                                         // [rows, heads, mass_stride]
  int* lens;                                           // [rows]
  const int* src;
  const int* dst;
  int* kept;                                           // [n_rows, keep]
  int* refcount;
  int* free_stack;
  int* free_count;
  unsigned* done;                                      // workspace: blocks done, pages dead, a bit for every dead page; zero between calls
  unsigned* dead;
  unsigned* bits;
  int* old;                                            // [EV_ENTRIES] what the second kernel has to know: the row's length before, -1: leave it alone
  long long bt_stride, kp_stride, mass_stride;
  int cols, n_rows, rows, heads, n_pages, keep, first, last, capacity;
  int* status;
};

// Order-preserving integer of a weight: NaN above all, both zeros alike.
__device__ __forceinline__ unsigned ev_key(float f) {
  const unsigned u = __float_as_uint(f + 0.0f);
  if (f != f) return 0xffffffffu;
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

struct EvShared {
  alignas(16) unsigned hist[EV_BINS], total[2][EV_BINS];           // of this block; of the cluster, in its first block, for every other pass
  int eq_of[EV_PIECES / EV_CL][EV_T / 32], sure_of[EV_PIECES / EV_CL][EV_T / 32];     // of a piece's warps: ties with the border, tokens that stay anyhow; then those ahead
  int eq[EV_PIECES / EV_CL], sure[EV_PIECES / EV_CL];   // of this block's pieces; then those ahead
  int warp[32];
  unsigned digit;
  int left, last;
};

// exclusive sum of v over the block; every thread also gets the whole sum
__device__ __forceinline__ int ev_scan(int v, int* warp_sum, int& all) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int sum = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += up;
  }
  if (lane == 31) warp_sum[warp] = sum;
  __syncthreads();
  const int mine = lane < EV_T / 32 ? warp_sum[lane] : 0;
  const int ahead = __reduce_add_sync(0xffffffffu, lane < warp ? mine : 0);
  all = __reduce_add_sync(0xffffffffu, mine);
  __syncthreads();
  return ahead + sum - v;
}
// add to a word of the cluster's first block
__device__ __forceinline__ void ev_add_first(unsigned* word, unsigned v) {
  asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(dsmem_map(smem_u32(word), 0)), "r"(v) : "memory");
}

__global__ void __launch_bounds__(EV_T, 2) evict_kernel(const EvictParams p) {
  extern __shared__ unsigned ev_keys[];                // [capacity]: piece i of this block at i * EV_T
  __shared__ EvShared S;
  const int t = threadIdx.x, rank = (int)cluster_ctarank(), b = blockIdx.x / EV_CL;
  const int src = p.src[b], dst = p.dst[b];
  bool fine = src >= 0 && src < p.rows && dst >= 0 && dst < p.rows;
  // nobody else may write this entry's rows, nor read the one that it writes
  bool clash = false;
  for (int o = t; o < p.n_rows; o += EV_T)
    if (o != b) clash |= p.dst[o] == dst || p.dst[o] == src || p.src[o] == dst;
  fine = !__syncthreads_or(clash) && fine;             // (a value known to the whole cluster: every block asks the same)
  bool shared = false;                                 // an earlier entry has the same source: its answer serves
  for (int o = t; o < b; o += EV_T) shared |= p.src[o] == src;
  shared = __syncthreads_or(shared);
  int n = src >= 0 && src < p.rows ? p.lens[src] : -1;
  const int old = fine ? p.lens[dst] : 0;
  const bool known = n >= 0 && n <= p.cols;            // (an entry that clashes still answers for those that share its source)
  n = known ? n : 0;
  fine = fine && known && old >= 0 && old <= p.cols;
  const bool solo = n <= EV_SOLO, in_place = src == dst;
  const int CL = solo ? 1 : EV_CL;
  auto barrier = [&] { if (solo) __syncthreads(); else cluster_sync(); };
  if (!fine && rank == 0 && t == 0) atomicOr(p.status, SMC_ERR_BOUNDS);
  if (known && !shared && !(solo && rank > 0)) {
    const int pieces = (n + EV_T - 1) / EV_T, steps = (pieces + CL - 1) / CL;
    const bool all = n <= p.keep;
    const int m = min(n, p.keep), lo = p.first, hi = n - p.last, want = p.keep - p.first - p.last;      // want of [lo, hi) stay
    auto index = [&](int i) { return (i * CL + rank) * EV_T + t; };                                     // of this thread in step i
    unsigned border = 0;
    int need = 0;                                      // tokens at the border that stay
    if (!all) {
      for (int i0 = 0; i0 < steps; i0 += 4) {          // 32 reads of a thread in flight
        float sum[4];
        for (int h0 = 0; h0 < p.heads; h0 += 8) {
          float w[4][8];
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int h = 0; h < 8; ++h) {
              const int idx = index(i0 + u);
              w[u][h] = idx < n && h0 + h < p.heads ? p.mass[((size_t)src * p.heads + h0 + h) * p.mass_stride + idx] : 0.f;
            }
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int h = 0; h < 8; ++h)
              if (h0 + h < p.heads) sum[u] = h0 + h == 0 ? w[u][h] : sum[u] + w[u][h];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (index(i0 + u) < n) ev_keys[(i0 + u) * EV_T + t] = ev_key(sum[u]);
      }
      need = want;
      if (want > 0) {
        int shift = 32;
        for (int i = t; i < EV_BINS; i += EV_T) S.total[0][i] = 0;
        for (int pass = 0; pass < 3; ++pass) {
          const int bits = pass < 2 ? 11 : 10;
          const unsigned known = shift < 32 ? border >> shift : 0u;
          unsigned* hist = solo ? S.total[pass & 1] : S.hist;
          if (!solo)
            for (int i = t; i < EV_BINS; i += EV_T) S.hist[i] = 0;
          __syncthreads();
          for (int i = 0; i < steps; ++i) {
            const int idx = index(i);
            const unsigned k = idx >= lo && idx < hi ? ev_keys[i * EV_T + t] : 0u;
            const bool counts = idx >= lo && idx < hi && (shift == 32 || k >> shift == known);
            const unsigned digit = k >> (shift - bits) & ((1u << bits) - 1u);
            if (pass == 0) {                           // most tokens share a few exponents: one addition for all lanes of a digit
              const unsigned same = __match_any_sync(0xffffffffu, counts ? digit : 0xffffffffu);
              if (counts && (threadIdx.x & 31) == __ffs(same) - 1) atomicAdd(&hist[digit], (unsigned)__popc(same));
            } else if (counts) {
              atomicAdd(&hist[digit], 1u);
            }
          }
          barrier();
          if (!solo)
            for (int i = t; i < EV_BINS; i += EV_T)
              if (S.hist[i] != 0u) ev_add_first(&S.total[pass & 1][i], S.hist[i]);
          for (int i = t; i < EV_BINS; i += EV_T) S.total[(pass & 1) ^ 1][i] = 0;
          barrier();
          // four bins a thread, the highest first
          constexpr int B = EV_BINS / EV_T;
          int count[B], mine = 0;
          static_assert(B == 4, "a thread's bins are read at once");
          {
            const uint32_t at = dsmem_map(smem_u32(&S.total[pass & 1][EV_BINS - 4 - 4 * t]), solo ? cluster_ctarank() : 0);
            asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(count[3]), "=r"(count[2]), "=r"(count[1]), "=r"(count[0]) : "r"(at) : "memory");
            mine = count[0] + count[1] + count[2] + count[3];
          }
          int sum, before = ev_scan(mine, S.warp, sum);
#pragma unroll
          for (int i = 0; i < B; ++i) {
            if (before < need && need <= before + count[i]) {
              S.digit = (unsigned)(EV_BINS - 1 - (B * t + i));
              S.left = need - before;
            }
            before += count[i];
          }
          __syncthreads();
          shift -= bits;
          border |= S.digit << shift;
          need = S.left;
          __syncthreads();
        }
      } else {
        border = 0xffffffffu;                          // ties with it: `need` is zero
      }
    }
    // what stays of each piece
    auto flags = [&](int i, bool& sure, bool& tie) {
      const int idx = index(i);
      const unsigned k = !all && idx < n ? ev_keys[i * EV_T + t] : 0u;
      const bool inner = idx >= lo && idx < hi;
      sure = idx < n && (all || !inner || (want > 0 && k > border));
      tie = idx < n && !all && inner && k == border;
    };
    const int warp = t >> 5, lane = t & 31;
    const unsigned below = (1u << lane) - 1u;
    for (int i = 0; i < steps; ++i) {
      bool sure, tie;
      flags(i, sure, tie);
      const unsigned a = __ballot_sync(0xffffffffu, sure), e = __ballot_sync(0xffffffffu, tie);
      if (lane == 0) { S.sure_of[i][warp] = __popc(a); S.eq_of[i][warp] = __popc(e); }
    }
    __syncthreads();
    if (t < steps) {                                   // warps of a piece -> those ahead of each
      int a = 0, e = 0;
#pragma unroll
      for (int w = 0; w < EV_T / 32; ++w) {
        const int wa = S.sure_of[t][w], we = S.eq_of[t][w];
        S.sure_of[t][w] = a;
        S.eq_of[t][w] = e;
        a += wa;
        e += we;
      }
      S.sure[t] = a;
      S.eq[t] = e;
    }
    barrier();
    {                                                  // pieces of the row -> those ahead of each
      int sure = 0, eq = 0, sum;
      if (t < pieces) {
        sure = solo ? S.sure[t] : (int)ld_dsmem_u32(smem_u32(&S.sure[t / CL]), t % CL);
        eq = solo ? S.eq[t] : (int)ld_dsmem_u32(smem_u32(&S.eq[t / CL]), t % CL);
      }
      const int sure_at = ev_scan(sure, S.warp, sum), eq_at = ev_scan(eq, S.warp, sum);
      barrier();                                       // all blocks have read the counts
      if (t < pieces && t % CL == rank) { S.sure[t / CL] = sure_at; S.eq[t / CL] = eq_at; }
      __syncthreads();
    }
    for (int i = 0; i < steps; ++i) {
      const int idx = index(i);
      bool sure, tie;
      flags(i, sure, tie);
      const unsigned a = __ballot_sync(0xffffffffu, sure), e = __ballot_sync(0xffffffffu, tie);
      // in front of a token stay the sure ones and the first `need` ties
      const int eq = S.eq[i] + S.eq_of[i][warp] + __popc(e & below);
      if (sure || (tie && eq < need)) {
        p.kept[(size_t)b * p.keep + S.sure[i] + S.sure_of[i][warp] + __popc(a & below) + min(eq, need)] = idx;
      } else if (fine && in_place && idx < n) {        // it leaves the row
        const int page = p.table[(size_t)src * p.bt_stride + idx];
        if (page < 0 || page > p.n_pages) {
          atomicOr(p.status, SMC_ERR_BOUNDS);
        } else if (page > 0) {
          const int before = atomicSub(&p.refcount[page], 1);
          if (before == 1) {
            atomicOr(&p.bits[page >> 5], 1u << (page & 31));
            atomicAdd(p.dead, 1u);
          } else if (before < 1) {
            atomicAdd(&p.refcount[page], 1);           // nobody held it
          }
        }
      }
    }
    for (int i = m + rank * EV_T + t; i < p.keep; i += CL * EV_T) p.kept[(size_t)b * p.keep + i] = -1;
    barrier();                                         // no block leaves while its counts are read, and all have read the lengths
  }
  if (rank == 0 && t == 0) {
    p.old[b] = fine ? old : -1;
    if (fine) p.lens[dst] = min(n, p.keep);
  }
  // the block that comes last puts dead pages on the free stack
  __syncthreads();
  if (t == 0) {
    __threadfence();
    S.last = atomicAdd(p.done, 1u) == gridDim.x - 1;
    __threadfence();
  }
  __syncthreads();
  if (!S.last) return;
  if (t == 0) {
    S.left = (int)atomicAdd(p.dead, 0u);
    *p.done = 0;
    *p.dead = 0;
  }
  __syncthreads();
  if (S.left == 0) return;
  const int words = p.n_pages / 32 + 1, per = (words + EV_T - 1) / EV_T;
  const int top = words - 1 - t * per;                 // this thread's words, the highest pages first
  int mine = 0, sum;
  for (int i = 0; i < per; ++i)
    if (top - i >= 0) mine += __popc(__ldcg(p.bits + top - i));
  const int at = ev_scan(mine, S.warp, sum), base = *p.free_count;
  int put = base + at;
  for (int i = 0; i < per; ++i) {
    if (top - i < 0) break;
    unsigned w = __ldcg(p.bits + top - i);
    if (w != 0u) p.bits[top - i] = 0u;
    while (w != 0u) {
      const int bit = 31 - __clz(w);
      w ^= 1u << bit;
      if (put >= 0 && put < p.n_pages) p.free_stack[put] = (top - i) * 32 + bit;
      else atomicOr(p.status, SMC_ERR_BOUNDS);         // a count below zero, or more free pages than there are
      ++put;
    }
  }
  __syncthreads();
  if (t == 0) *p.free_count = min(base + sum, p.n_pages);
}

// Part 0 of an entry: pages with their references, positions, the list of an entry that shares another one's answer; part 1 + h: the weights of a head.
__global__ void __launch_bounds__(EV_T) evict_move_kernel(const EvictParams p) {
  const int t = threadIdx.x, b = blockIdx.x / (p.heads + 1), part = blockIdx.x % (p.heads + 1) - 1;
  const int src = p.src[b], dst = p.dst[b];
  int leader = b;
  for (int o = t; o < b; o += EV_T)
    if (p.src[o] == src) { leader = o; break; }
  __shared__ int s_leader;
  if (t == 0) s_leader = b;
  __syncthreads();
  if (leader < b) atomicMin(&s_leader, leader);
  __syncthreads();
  leader = s_leader;
  pdl_wait_prior_grid();
  const int old = p.old[b];
  if (old < 0) return;
  const int m = p.lens[dst];
  const int* list = p.kept + (size_t)leader * p.keep;
  // every thread EV_MOVE places of a run; between its reads and its writes a barrier where the row is its own source
  auto move = [&](auto* from, auto* to, auto also) {
    for (int p0 = 0; p0 < m; p0 += EV_T * EV_MOVE) {
      int idx[EV_MOVE];
      decltype(*from + 0) v[EV_MOVE];
#pragma unroll
      for (int u = 0; u < EV_MOVE; ++u) idx[u] = p0 + u * EV_T + t < m ? list[p0 + u * EV_T + t] : -1;
#pragma unroll
      for (int u = 0; u < EV_MOVE; ++u)
        if (idx[u] >= 0) v[u] = from[idx[u]];
      if (src == dst) __syncthreads();
#pragma unroll
      for (int u = 0; u < EV_MOVE; ++u)
        if (idx[u] >= 0) {
          to[p0 + u * EV_T + t] = v[u];
          also(p0 + u * EV_T + t, idx[u], v[u]);
        }
    }
  };
  if (part < 0) {
    move(p.table + (size_t)src * p.bt_stride, p.table + (size_t)dst * p.bt_stride, [&](int at, int idx, int page) {
      if (page < 0 || page > p.n_pages) atomicOr(p.status, SMC_ERR_BOUNDS);
      else if (page > 0 && src != dst) atomicAdd(&p.refcount[page], 1);
      if (leader != b) p.kept[(size_t)b * p.keep + at] = idx;
    });
    if (p.key_pos != nullptr)
      move(p.key_pos + (size_t)src * p.kp_stride, p.key_pos + (size_t)dst * p.kp_stride, [](int, int, int) {});
    if (leader != b)
      for (int i = m + t; i < p.keep; i += EV_T) p.kept[(size_t)b * p.keep + i] = -1;
  } else {
    float* to = p.mass + ((size_t)dst * p.heads + part) * p.mass_stride;
    move(p.mass + ((size_t)src * p.heads + part) * p.mass_stride, to, [](int, int, float) {});
    __syncthreads();
    for (int i = m + t; i < old; i += EV_T) to[i] = 0.f;              // no weight behind the kept tokens, up to the row's old length
  }
}

}  // namespace smc

// Bytes of workspace (zeros at first) for an allocator of n_pages pages.
SMC_API long long smc_evict_work(int n_pages) { return n_pages < 1 ? -1 : 256 + smc::EV_ENTRIES * 4 + ((long long)n_pages / 32 + 1) * 4; }

// src, dst [n_rows] int32 rows of table [rows, columns], key_pos [rows, kp_stride] or null and mass [rows, heads, mass_stride] fp32, with lens [rows]; a
// row is written by one entry at most and then read by no other.  kept [n_rows, keep].
SMC_API int smc_evict(int* table, long long bt_pitch, int* key_pos, long long kp_stride, float* mass, long long mass_stride, int* lens, int rows,
                      const int* src, const int* dst, int n_rows, int heads, int keep, int first, int last, int* kept, int* refcount, int* free_stack,
                      int* free_count, int n_pages, void* work, long long work_bytes, int* status, cudaStream_t st) {
  using namespace smc;
  if (n_rows <= 0) return 0;
  if (n_rows > EV_ENTRIES || kept == nullptr || heads < 1 || keep < 1 || first < 0 || last < 0 || first > keep || last > keep - first) return -170;
  const int cols = pitch_cols(bt_pitch);
  if (!pitch_fits(bt_pitch) || cols > EV_PIECES * EV_T || mass_stride < cols || (key_pos != nullptr && kp_stride < cols)) return -171;
  if (n_pages < 1 || work_bytes < smc_evict_work(n_pages) || (reinterpret_cast<uintptr_t>(work) & 3)) return -172;
  EvictParams p;
  p.table = table; p.key_pos = key_pos; p.mass = mass; p.lens = lens; p.src = src; p.dst = dst; p.kept = kept;
  p.refcount = refcount; p.free_stack = free_stack; p.free_count = free_count;
  p.done = (unsigned*)work; p.dead = p.done + 1; p.old = (int*)(p.done + 64); p.bits = p.done + 64 + EV_ENTRIES;
  p.bt_stride = pitch_stride(bt_pitch); p.cols = cols; p.kp_stride = kp_stride; p.mass_stride = mass_stride;
  p.n_rows = n_rows; p.rows = rows; p.heads = heads; p.n_pages = n_pages; p.keep = keep; p.first = first; p.last = last; p.status = status;
  const int per = (cols + EV_CL * EV_T - 1) / (EV_CL * EV_T) * EV_T, alone = cols < EV_SOLO ? (cols + EV_T - 1) / EV_T * EV_T : EV_SOLO;
  p.capacity = per > alone ? per : alone;
  const size_t smem = (size_t)p.capacity * 4;
  CUDA_CHECK_RET(cudaFuncSetAttribute(evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = EV_CL;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(n_rows * EV_CL));
  cfg.blockDim = dim3(EV_T);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  CUDA_CHECK_RET(cudaLaunchKernelEx(&cfg, evict_kernel, p));
  // (rows and lists that the second kernel reads ahead of its wait are the caller's: the first kernel lets it start at its end only)
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)(n_rows * (heads + 1)));
  cfg.dynamicSmemBytes = 0;
  CUDA_CHECK_RET(cudaLaunchKernelEx(&cfg, evict_move_kernel, p));
  return 0;
}
