// Rows of the block table brought down to a budget: the tokens that hold the most attention weight stay.
//
// Of the n tokens of a row the first `first`, the last `last` and, of those between, the ones with the highest weight stay, `keep` in all; equal
// weights go to the lower index.  A token's weight is the fp32 sum over the KV heads in their order.  The kept tokens move up in their order - page ids,
// positions and weights, no key or value - into the same row, whose other tokens lose their references, or into another row, for which
// references are taken.  Pages without a reference go on the free stack, the lowest on top, as the host's form leaves them.
//
// A cluster of eight blocks serves a row (one block alone a short one): blocks of 1024 tokens go round the cluster, so that one step
// covers a run of the row and, with a barrier between its reads and its writes, compaction in place never overwrites what a later step reads.  The
// n-th highest weight is found by three histograms of 11, 11 and 10 bits over order-preserving integers in shared memory, joined over the cluster.
// What bounds it: 4 bytes per token and head read once, then barriers; the row that takes longest decides.
#include "common.cuh"

namespace smc {

constexpr int EV_CL = 8, EV_T = 1024, EV_BINS = 2048, EV_SOLO = 8192, EV_BLOCKS = 512;
constexpr int EV_HEADS = 8;                            // heads moved between two barriers

struct EvictParams {
  int* table;
  int* key_pos;                                        // or null
  float* mass;                                         // [rows, heads, mass_stride]
  int* lens;                                           // [rows]
  const int* src;
  const int* dst;
  int* kept;                                           // [n_rows, keep] or null
  int* refcount;
  int* free_stack;
  int* free_count;
  unsigned* done;                                      // workspace: blocks done, pages dead, a bit for every dead page; zero between calls
  unsigned* dead;
  unsigned* bits;
  long long bt_stride, kp_stride, mass_stride;
  int n_rows, rows, heads, n_pages, keep, first, last, capacity;
  int* status;
};

// Order-preserving integer of a weight: NaN above all, both zeros alike.
__device__ __forceinline__ unsigned ev_key(float f) {
  const unsigned u = __float_as_uint(f + 0.0f);
  if (f != f) return 0xffffffffu;
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

struct EvShared {
  unsigned hist[EV_BINS];
  int eq[EV_BLOCKS / EV_CL], sure[EV_BLOCKS / EV_CL];   // of this block's pieces: ties with the border, tokens that stay anyhow
  int eq_at[EV_BLOCKS / EV_CL], kept_at[EV_BLOCKS / EV_CL];
  int warp[32], warp2[32];
  unsigned digit;
  int left, total;
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
  const int mine = warp_sum[lane];
  const int ahead = __reduce_add_sync(0xffffffffu, lane < warp ? mine : 0);
  all = __reduce_add_sync(0xffffffffu, mine);
  __syncthreads();
  return ahead + sum - v;
}

__global__ void __launch_bounds__(EV_T, 1) evict_kernel(const EvictParams p) {
  extern __shared__ unsigned ev_keys[];                // [capacity]: piece i of this block at i * EV_T
  __shared__ EvShared S;
  const int t = threadIdx.x, rank = (int)cluster_ctarank(), b = blockIdx.x / EV_CL;
  const int src = p.src[b], dst = p.dst[b];
  bool fine = src >= 0 && src < p.rows && dst >= 0 && dst < p.rows;
  // nobody else may write this entry's rows, nor read the one that it writes
  bool clash = false;
  for (int o = t; o < p.n_rows; o += EV_T)
    if (o != b) clash |= p.dst[o] == dst || p.dst[o] == src || p.src[o] == dst;
  fine = !__syncthreads_or(clash) && fine;
  const int n = fine ? p.lens[src] : 0, old = fine ? p.lens[dst] : 0;
  fine = fine && n >= 0 && n <= p.bt_stride && old >= 0 && old <= p.bt_stride;
  const bool solo = n <= EV_SOLO, in_place = src == dst;
  const int CL = solo ? 1 : EV_CL;
  auto barrier = [&] { if (solo) __syncthreads(); else cluster_sync(); };
  const bool idle = solo && rank > 0;
  if (!fine && rank == 0 && t == 0) atomicOr(p.status, SMC_ERR_BOUNDS);
  if (fine && !idle) {
    const int pieces = (n + EV_T - 1) / EV_T, steps = (pieces + CL - 1) / CL;
    const bool all = n <= p.keep;
    const int m = min(n, p.keep), lo = p.first, hi = n - p.last, want = p.keep - p.first - p.last;      // want of [lo, hi) stay
    auto index = [&](int i) { return (i * CL + rank) * EV_T + t; };                                     // of this thread in step i
    unsigned border = 0;
    int need = 0;                                      // tokens at the border that stay
    if (!all) {
      for (int i = 0; i < steps; ++i) {
        const int idx = index(i);
        if (idx < n) {
          const float* w = p.mass + (size_t)src * p.heads * p.mass_stride + idx;
          float sum = w[0];
#pragma unroll 8
          for (int h = 1; h < p.heads; ++h) sum += w[(size_t)h * p.mass_stride];
          ev_keys[i * EV_T + t] = ev_key(sum);
        }
      }
      need = want;
      if (want > 0) {
        int shift = 32;
        for (int pass = 0; pass < 3; ++pass) {
          const int bits = pass < 2 ? 11 : 10;
          const unsigned known = shift < 32 ? border >> shift : 0u;
          for (int i = t; i < EV_BINS; i += EV_T) S.hist[i] = 0;
          __syncthreads();
          for (int i = 0; i < steps; ++i) {
            const int idx = index(i);
            if (idx >= lo && idx < hi) {
              const unsigned k = ev_keys[i * EV_T + t];
              if (shift == 32 || k >> shift == known) atomicAdd(&S.hist[k >> (shift - bits) & ((1u << bits) - 1u)], 1u);
            }
          }
          barrier();
          // two bins a thread, the highest first, over all blocks of the cluster
          int count[2] = {0, 0};
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int bin = EV_BINS - 1 - (2 * t + i);
            if (solo) count[i] = (int)S.hist[bin];
            else
              for (int c = 0; c < EV_CL; ++c) count[i] += (int)ld_dsmem_u32(smem_u32(&S.hist[bin]), c);
          }
          int sum;
          const int ahead = ev_scan(count[0] + count[1], S.warp, sum);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int before = ahead + (i ? count[0] : 0);
            if (before < need && need <= before + count[i]) {
              S.digit = (unsigned)(EV_BINS - 1 - (2 * t + i));
              S.left = need - before;
            }
          }
          barrier();                                   // the histograms are read, the digit is there
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
    for (int i = 0; i < steps; ++i) {
      bool sure, tie;
      flags(i, sure, tie);
      const int a = __syncthreads_count(sure), e = __syncthreads_count(tie);
      if (t == 0) { S.sure[i] = a; S.eq[i] = e; }
    }
    barrier();
    {
      int sure = 0, eq = 0, all_eq, all_kept;
      if (t < pieces) {
        const int c = t % CL, i = t / CL;
        sure = solo ? S.sure[i] : (int)ld_dsmem_u32(smem_u32(&S.sure[i]), c);
        eq = solo ? S.eq[i] : (int)ld_dsmem_u32(smem_u32(&S.eq[i]), c);
      }
      const int eq_at = ev_scan(eq, S.warp, all_eq);
      const int kept_at = ev_scan(sure + max(0, min(eq, need - eq_at)), S.warp2, all_kept);
      if (t < pieces && t % CL == rank) { S.eq_at[t / CL] = eq_at; S.kept_at[t / CL] = kept_at; }
      __syncthreads();
    }
    for (int i = 0; i < steps; ++i) {
      bool sure, tie;
      flags(i, sure, tie);
      const int idx = index(i);
      const bool mine = i * CL + rank < pieces;        // uniform over the block
      int sum, at = 0;
      bool stay = false;
      if (mine) {
        const int eq_at = S.eq_at[i] + ev_scan(tie, S.warp, sum);
        stay = sure || (tie && eq_at < need);
        at = S.kept_at[i] + ev_scan(stay, S.warp2, sum);
        if (stay && p.kept != nullptr) p.kept[(size_t)b * p.keep + at] = idx;
      }
      if (all && in_place) continue;                   // nothing moves
      int page = 0, pos = 0;
      if (mine && idx < n) {
        page = p.table[(size_t)src * p.bt_stride + idx];
        if (p.key_pos != nullptr) pos = p.key_pos[(size_t)src * p.kp_stride + idx];
        if (page < 0 || page > p.n_pages) {
          atomicOr(p.status, SMC_ERR_BOUNDS);
        } else if (page > 0) {
          if (in_place && !stay) {
            const int before = atomicSub(&p.refcount[page], 1);
            if (before == 1) {
              atomicOr(&p.bits[page >> 5], 1u << (page & 31));
              atomicAdd(p.dead, 1u);
            } else if (before < 1) {
              atomicAdd(&p.refcount[page], 1);         // nobody held it
            }
          } else if (!in_place && stay) {
            atomicAdd(&p.refcount[page], 1);
          }
        }
      }
      for (int h0 = 0; h0 < p.heads; h0 += EV_HEADS) {
        float w[EV_HEADS];
#pragma unroll
        for (int h = 0; h < EV_HEADS; ++h)
          if (stay && h0 + h < p.heads) w[h] = p.mass[((size_t)src * p.heads + h0 + h) * p.mass_stride + idx];
        if (in_place) barrier();
        if (stay) {
          if (h0 == 0) {
            p.table[(size_t)dst * p.bt_stride + at] = page;
            if (p.key_pos != nullptr) p.key_pos[(size_t)dst * p.kp_stride + at] = pos;
          }
#pragma unroll
          for (int h = 0; h < EV_HEADS; ++h)
            if (h0 + h < p.heads) p.mass[((size_t)dst * p.heads + h0 + h) * p.mass_stride + at] = w[h];
        }
      }
    }
    if (in_place) barrier();                           // everything has been read
    // behind the kept tokens: no weight up to the row's old length, no index
    const int step = CL * EV_T, t0 = rank * EV_T + t;
    for (int h = 0; h < p.heads; ++h)
      for (int i = m + t0; i < old; i += step) p.mass[((size_t)dst * p.heads + h) * p.mass_stride + i] = 0.f;
    if (p.kept != nullptr)
      for (int i = m + t0; i < p.keep; i += step) p.kept[(size_t)b * p.keep + i] = -1;
    barrier();                                         // all blocks have read the lengths, and no block leaves while its counts are read
    if (rank == 0 && t == 0) p.lens[dst] = m;
  }
  // the block that comes last puts dead pages on the free stack
  __syncthreads();
  if (t == 0) {
    __threadfence();
    S.total = atomicAdd(p.done, 1u) == gridDim.x - 1;
    __threadfence();
  }
  __syncthreads();
  if (!S.total) return;
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
      if (put < p.n_pages) p.free_stack[put] = (top - i) * 32 + bit;
      else atomicOr(p.status, SMC_ERR_BOUNDS);         // more free pages than there are
      ++put;
    }
  }
  __syncthreads();
  if (t == 0) *p.free_count = min(base + sum, p.n_pages);
}

}  // namespace smc

// Bytes of workspace (zeros at first) for an allocator of n_pages pages.
SMC_API long long smc_evict_work(int n_pages) { return n_pages < 1 ? -1 : 256 + ((long long)n_pages / 32 + 1) * 4; }

// src, dst [n_rows] int32 rows of table [rows, bt_stride], key_pos [rows, kp_stride] or null and mass [rows, heads, mass_stride] fp32, with lens [rows]; a
// row is written by one entry at most and then read by no other.  kept [n_rows, keep] or null.
SMC_API int smc_evict(int* table, long long bt_stride, int* key_pos, long long kp_stride, float* mass, long long mass_stride, int* lens, int rows,
                      const int* src, const int* dst, int n_rows, int heads, int keep, int first, int last, int* kept, int* refcount, int* free_stack,
                      int* free_count, int n_pages, void* work, long long work_bytes, int* status, cudaStream_t st) {
  using namespace smc;
  if (n_rows <= 0) return 0;
  if (heads < 1 || keep < 1 || first < 0 || last < 0 || first > keep || last > keep - first) return -170;
  if (bt_stride < 1 || bt_stride > EV_BLOCKS * EV_T / 2 || mass_stride < bt_stride || (key_pos != nullptr && kp_stride < bt_stride)) return -171;
  if (work_bytes < smc_evict_work(n_pages) || (reinterpret_cast<uintptr_t>(work) & 3)) return -172;
  EvictParams p;
  p.table = table; p.key_pos = key_pos; p.mass = mass; p.lens = lens; p.src = src; p.dst = dst; p.kept = kept;
  p.refcount = refcount; p.free_stack = free_stack; p.free_count = free_count;
  p.done = (unsigned*)work; p.dead = p.done + 1; p.bits = p.done + 64;
  p.bt_stride = bt_stride; p.kp_stride = kp_stride; p.mass_stride = mass_stride;
  p.n_rows = n_rows; p.rows = rows; p.heads = heads; p.n_pages = n_pages; p.keep = keep; p.first = first; p.last = last; p.status = status;
  const long long per = (bt_stride + EV_CL * EV_T - 1) / (EV_CL * EV_T) * EV_T, alone = (bt_stride < EV_SOLO ? (bt_stride + EV_T - 1) / EV_T * EV_T : EV_SOLO);
  p.capacity = (int)(per > alone ? per : alone);
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
  return 0;
}
