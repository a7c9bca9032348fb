// kvcu_evict.cu — bounding a paged cache: which rows stay, and moving them.
//
// k_evict_select: per (layer, entry) the positions that stay under a budget: the
//   first n_sink, the last n_recent, and of those between the largest masses,
//   ties to the lowest position, as an ascending list.  A radix select on the
//   masses' 32-bit order (11 + 11 + 10 bits): the row is read once into shared
//   memory while the first histogram is formed, the other passes run there.
//   Bound: one read of the masses (4 B per position).
// k_evict_compact: row j of a sequence := its row keep[j], in place through the
//   block table, in every layer, and the masses with it.  Bound: one read and
//   one write of the kept rows.
#include <cuda_runtime.h>

#include "kvcu_internal.h"

namespace {

// ------------------------------------------------------------------ cluster helpers
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// Every thread of every CTA of the cluster arrives, then waits for all; orders
// the reads and writes before it against those after it.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A 32-bit word of CTA `rank`'s shared memory at this CTA's address p.
__device__ __forceinline__ uint32_t ld_cluster(const uint32_t* p, uint32_t rank) {
  uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(p)), v;
  asm volatile("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(a) : "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

// ------------------------------------------------------------------ select
struct SelectArgs {
  const float* mass;
  uint64_t mass_lstride, mass_stride;
  uint32_t n, n_seqs;
  const uint32_t* seq_ids;
  const uint32_t* lens;
  uint32_t budget, n_sink, n_recent;
  uint32_t* keep;
  uint64_t keep_lstride, keep_stride;
  uint32_t* counts;
  uint32_t* status;
  uint32_t cap;  // positions a CTA's shared memory holds
};

constexpr uint32_t BINS = 2048;

// Ascending 32-bit order of the values; -0 and +0 are one value, NaN is below
// everything.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 0u;
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Inclusive sum over the block of one value per thread.  `part` holds one word
// per warp; ends with a barrier before `part` may be reused.
template <int NT>
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* part) {
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= (uint32_t)o) v += y;
  }
  if (lane == 31) part[warp] = v;
  __syncthreads();
  uint32_t before = 0;
  for (uint32_t w = 0; w < warp; ++w) before += part[w];
  __syncthreads();
  return v + before;
}

// One row per cluster of C CTAs; each CTA holds an equal share of the row's
// middle, in order.
template <int C, int NT>
__global__ void __launch_bounds__(NT) k_evict_select(SelectArgs a) {
  extern __shared__ uint32_t cache[];  // [cap] order keys of this CTA's share
  __shared__ uint32_t hist[BINS], total[BINS];
  __shared__ uint32_t part[NT / 32], part2[NT / 32];
  __shared__ uint32_t s_bin, s_above, s_tot[2];
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  const uint32_t rank = C > 1 ? cluster_rank() : 0u;
  const uint32_t row = blockIdx.x / C, layer = row / a.n, b = row % a.n;
  const uint32_t s = a.seq_ids ? a.seq_ids[b] : b;
  uint32_t len = 0;
  if (s < a.n_seqs) {
    len = a.lens[s];
    if (len > a.mass_stride) {
      if (tid == 0) atomicOr(a.status, KVCU_STATUS_BAD_LEN);
      len = (uint32_t)a.mass_stride;
    }
  } else if (tid == 0) {
    atomicOr(a.status, KVCU_STATUS_BAD_SEQ);
  }
  uint32_t* keep = a.keep + layer * a.keep_lstride + b * a.keep_stride;
  if (layer == 0 && rank == 0 && tid == 0) a.counts[b] = min(len, a.budget);
  if (len <= a.budget) {  // all stay (the whole cluster takes this way)
    for (uint32_t j = rank * NT + tid; j < a.budget; j += C * NT) keep[j] = j < len ? j : KVCU_NO_POSITION;
    return;
  }
  // the two ends that always stay
  for (uint32_t j = rank * NT + tid; j < a.n_sink; j += C * NT) keep[j] = j;
  for (uint32_t j = rank * NT + tid; j < a.n_recent; j += C * NT)
    keep[a.budget - a.n_recent + j] = len - a.n_recent + j;
  const uint32_t lo = a.n_sink, hi = len - a.n_recent;
  uint32_t need = a.budget - a.n_sink - a.n_recent;  // of the hi - lo > need positions between
  if (need == 0) return;
  const uint32_t share = (hi - lo + C - 1) / C;
  const uint32_t p0 = min(lo + rank * share, hi), p1 = min(p0 + share, hi), cnt = p1 - p0;
  const float* mass = a.mass + layer * a.mass_lstride + b * a.mass_stride + p0;
  auto key_at = [&](uint32_t i) { return i < a.cap ? cache[i] : order_key(mass[i]); };

  // ---- radix select of the need-th largest key
  uint32_t prefix = 0, above = 0;  // keys above the prefix's range: all kept
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t mask = pass == 2 ? 1023u : 2047u;
    for (uint32_t i = tid; i < BINS; i += NT) hist[i] = 0;
    __syncthreads();
    if (pass == 0) {
      for (uint32_t i = tid; i < cnt; i += NT) {
        const uint32_t k = order_key(mass[i]);
        if (i < a.cap) cache[i] = k;
        atomicAdd(&hist[k >> 21], 1u);
      }
    } else {
      const int top = pass == 1 ? 21 : 10;
      for (uint32_t i = tid; i < cnt; i += NT) {
        const uint32_t k = key_at(i);
        if ((k >> top) == prefix) atomicAdd(&hist[(k >> shift) & mask], 1u);
      }
    }
    const uint32_t* h = hist;
    if constexpr (C > 1) {
      cluster_sync();
      for (uint32_t i = tid; i <= mask; i += NT) {
        uint32_t t = 0;
#pragma unroll
        for (int r = 0; r < C; ++r) t += ld_cluster(&hist[i], r);
        total[i] = t;
      }
      h = total;
      cluster_sync();  // no CTA clears its histogram while another reads it
    } else {
      __syncthreads();
    }
    // from the top bin down: the bin that holds the need-th largest
    constexpr uint32_t PER = BINS / NT;  // bins of a thread, highest first
    uint32_t mine = 0, own[PER];
#pragma unroll
    for (uint32_t j = 0; j < PER; ++j) {
      const uint32_t bin = BINS - 1 - (tid * PER + j);
      own[j] = bin <= mask ? h[bin] : 0u;
      mine += own[j];
    }
    const uint32_t upto = block_scan<NT>(mine, part);
    uint32_t run = above + upto - mine;
    if (run < need && need <= above + upto) {
#pragma unroll
      for (uint32_t j = 0; j < PER; ++j) {
        if (run < need && need <= run + own[j]) {
          s_bin = BINS - 1 - (tid * PER + j);
          s_above = run;
        }
        run += own[j];
      }
    }
    __syncthreads();
    prefix = (prefix << (pass == 2 ? 10 : 11)) | s_bin;
    above = s_above;
    __syncthreads();
  }
  const uint32_t ties = need - above;  // of the positions equal to the threshold, the first `ties`

  // ---- the kept positions in order: each warp takes a run of the share
  const uint32_t run = ((cnt + NT / 32 - 1) / (NT / 32) + 31u) & ~31u;
  const uint32_t w0 = min(warp * run, cnt), w1 = min(w0 + run, cnt);
  uint32_t gt = 0, eq = 0;
  for (uint32_t i = w0 + lane; i < w1; i += 32) {
    const uint32_t k = key_at(i);
    gt += k > prefix;
    eq += k == prefix;
  }
  gt = __reduce_add_sync(0xffffffffu, gt);
  eq = __reduce_add_sync(0xffffffffu, eq);
  if (lane == 0) {
    part[warp] = gt;
    part2[warp] = eq;
  }
  __syncthreads();
  uint32_t gt0 = 0, eq0 = 0;
  for (uint32_t w = 0; w < warp; ++w) {
    gt0 += part[w];
    eq0 += part2[w];
  }
  if constexpr (C > 1) {
    if (tid == NT - 1) {
      s_tot[0] = gt0 + gt;
      s_tot[1] = eq0 + eq;
    }
    cluster_sync();
    for (uint32_t r = 0; r < rank; ++r) {
      gt0 += ld_cluster(&s_tot[0], r);
      eq0 += ld_cluster(&s_tot[1], r);
    }
    cluster_sync();  // no CTA leaves while another reads its shared memory
  }
  const uint32_t below = (1u << lane) - 1u;
  for (uint32_t i0 = w0; i0 < w1; i0 += 32) {
    const uint32_t i = i0 + lane;
    const uint32_t k = i < w1 ? key_at(i) : 0u;
    const bool g = i < w1 && k > prefix, e = i < w1 && k == prefix;
    const uint32_t mg = __ballot_sync(0xffffffffu, g), me = __ballot_sync(0xffffffffu, e);
    const uint32_t gi = gt0 + __popc(mg & below), ei = eq0 + __popc(me & below);
    if (g || (e && ei < ties)) keep[a.n_sink + gi + min(ei, ties)] = p0 + i;
    gt0 += __popc(mg);
    eq0 += __popc(me);
  }
}

// ------------------------------------------------------------------ compact
struct CompactArgs {
  char* a;  // the pool's two arrays: payload / latent, scales / rope
  char* b;
  uint32_t row_a, row_b;  // bytes of a row
  uint64_t layer_rows;    // rows of a layer
  uint32_t num_blocks, block_size, layer, n, n_seqs;
  const uint32_t* seq_ids;
  const uint32_t* toff;
  const uint32_t* tables;
  const uint32_t* keep;
  uint64_t keep_lstride, keep_stride;
  const uint32_t* counts;
  float* mass;
  uint64_t mass_lstride, mass_stride;
  uint32_t* lens;
  uint32_t* status;
  uint32_t tile;  // rows of a CTA's tile
};

constexpr int CT = 256;              // threads
constexpr uint32_t MAX_TILE = 64;    // rows
constexpr uint64_t NO_ROW = ~0ull;

template <int U>
__device__ __forceinline__ void copy_in(uint32_t dst, const char* src) {
  if constexpr (U == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  } else if constexpr (U == 4) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
  } else {
    uint16_t v;
    asm volatile("ld.global.cg.u16 %0, [%1];" : "=h"(v) : "l"(src) : "memory");
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(dst), "h"(v) : "memory");
  }
}
template <int U>
__device__ __forceinline__ void copy_out(char* dst, const char* src) {
  if constexpr (U == 16) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
  else if constexpr (U == 4) *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(src);
  else *reinterpret_cast<uint16_t*>(dst) = *reinterpret_cast<const uint16_t*>(src);
}

// One (layer, entry) per cluster.  Its kept rows go in waves of C * tile rows,
// tile by tile over the CTAs: a wave's rows are all read into shared memory,
// the cluster meets, then they are written.  In place without a second copy:
// keep ascends, so keep[j] >= j, and row r is the source of some j <= r only.
// The rows a wave overwrites, [w, w + 1) * C * tile, are therefore sources of
// this wave and earlier ones, which have been read; the next wave's sources lie
// behind them, so its reads are already in flight meanwhile.
template <int UA, int UB>
__global__ void __launch_bounds__(CT) k_evict_compact(CompactArgs a, uint32_t C) {
  extern __shared__ __align__(16) char smem[];  // two stages of [tile][row_a] and [tile][row_b padded]
  __shared__ uint64_t src_row[2][MAX_TILE], dst_row[2][MAX_TILE];
  __shared__ float mval[2][MAX_TILE];
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  const uint32_t rank = C > 1 ? cluster_rank() : 0u;
  const uint32_t pair = blockIdx.x / C, layer = pair / a.n, b = pair % a.n;
  const uint32_t s = a.seq_ids ? a.seq_ids[b] : b;
  if (s >= a.n_seqs) {
    if (tid == 0) atomicOr(a.status, KVCU_STATUS_BAD_SEQ);
    return;
  }
  uint32_t count = a.counts[b];
  if (count > a.keep_stride) {
    if (tid == 0) atomicOr(a.status, KVCU_STATUS_BAD_LEN);
    count = (uint32_t)a.keep_stride;
  }
  if (a.lens && layer == 0 && rank == 0 && tid == 0) a.lens[s] = count;
  const uint32_t* keep = a.keep + layer * a.keep_lstride + b * a.keep_stride;
  if (count == 0 || keep[count - 1] == count - 1) return;  // ascending: every row is in its place
  const uint32_t t0 = a.toff[s], t1 = max(a.toff[s + 1], t0);
  float* mass = a.mass ? a.mass + layer * a.mass_lstride + b * a.mass_stride : nullptr;
  const uint64_t base = (uint64_t)(a.layer + layer) * a.layer_rows;
  const uint32_t pad_b = (a.row_b + 15u) & ~15u;
  const uint32_t stage = a.tile * (a.row_a + pad_b);
  const uint32_t waves = (count + C * a.tile - 1) / (C * a.tile);

  auto row_of = [&](uint32_t p) -> uint64_t {
    const uint32_t bi = p / a.block_size;
    if (bi >= t1 - t0) {
      atomicOr(a.status, KVCU_STATUS_BAD_TABLE);
      return NO_ROW;
    }
    const uint32_t blk = a.tables[t0 + bi];
    if (blk >= a.num_blocks) {
      atomicOr(a.status, KVCU_STATUS_BAD_BLOCK);
      return NO_ROW;
    }
    return base + (uint64_t)blk * a.block_size + p % a.block_size;
  };
  auto load = [&](uint32_t w) {
    const uint32_t f = w & 1u;
    const uint32_t j0 = (w * C + rank) * a.tile;
    if (tid < a.tile) {
      uint64_t src = NO_ROW, dst = NO_ROW;
      const uint32_t j = j0 + tid;
      if (j < count) {
        const uint32_t p = keep[j];
        if (p != j) {
          src = row_of(p);
          dst = row_of(j);
          if (src == NO_ROW) dst = NO_ROW;
          if (mass) mval[f][tid] = p < a.mass_stride ? __ldcg(mass + p) : 0.0f;
        }
      }
      src_row[f][tid] = src;
      dst_row[f][tid] = dst;
    }
    __syncthreads();
    char* st = smem + f * stage;
    const uint32_t sa = static_cast<uint32_t>(__cvta_generic_to_shared(st));
    for (uint32_t r = warp; r < a.tile; r += CT / 32) {
      const uint64_t src = src_row[f][r];
      if (dst_row[f][r] == NO_ROW) continue;
      for (uint32_t o = lane * UA; o < a.row_a; o += 32 * UA) copy_in<UA>(sa + r * a.row_a + o, a.a + src * a.row_a + o);
      const uint32_t sb = sa + a.tile * a.row_a + r * pad_b;
      for (uint32_t o = lane * UB; o < a.row_b; o += 32 * UB) copy_in<UB>(sb + o, a.b + src * a.row_b + o);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  load(0);
  for (uint32_t w = 0; w < waves; ++w) {
    if (w + 1 < waves) {
      load(w + 1);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    // the whole wave is in shared memory
    if (C > 1) cluster_sync();
    else __syncthreads();
    const uint32_t f = w & 1u;
    const char* st = smem + f * stage;
    for (uint32_t r = warp; r < a.tile; r += CT / 32) {
      const uint64_t dst = dst_row[f][r];
      if (dst == NO_ROW) continue;
      for (uint32_t o = lane * UA; o < a.row_a; o += 32 * UA) copy_out<UA>(a.a + dst * a.row_a + o, st + r * a.row_a + o);
      const char* sb = st + a.tile * a.row_a + r * pad_b;
      for (uint32_t o = lane * UB; o < a.row_b; o += 32 * UB) copy_out<UB>(a.b + dst * a.row_b + o, sb + o);
    }
    if (mass && tid < a.tile && src_row[f][tid] != NO_ROW) {
      const uint32_t j = (w * C + rank) * a.tile + tid;
      if (j < a.mass_stride) mass[j] = mval[f][tid];
    }
    __syncthreads();  // the stage may be filled again
  }
}

struct DevScope {
  int prev = -1, rc = 0;
  explicit DevScope(int dev) {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    if (prev != dev) rc = kvcu_check_cuda(cudaSetDevice(dev), "cudaSetDevice");
  }
  ~DevScope() {
    int cur = -1;
    if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev) cudaSetDevice(prev);
  }
};

template <typename... KArgs, typename... Args>
int launch_clusters(void (*kernel)(KArgs...), uint32_t clusters, uint32_t C, int threads, size_t smem, cudaStream_t st,
                    const char* what, Args... args) {
  const int rc = kvcu_configure_once(
      reinterpret_cast<const void*>(kernel),
      [](const void* k) {
        return kvcu_check_cuda(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, KVCU_EVICT_SMEM),
                               "cudaFuncSetAttribute(evict)");
      },
      reinterpret_cast<const void*>(kernel));
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(clusters * C);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return kvcu_check_cuda(cudaLaunchKernelEx(&cfg, kernel, args...), what);
}

template <int C>
int launch_select(const SelectArgs& a, uint32_t rows, cudaStream_t st) {
  return launch_clusters(k_evict_select<C, 1024>, rows, C, 1024, (size_t)a.cap * 4, st, "evict select launch", a);
}

template <int UA>
int launch_compact(const CompactArgs& a, uint32_t pairs, uint32_t C, size_t smem, cudaStream_t st) {
  if (a.row_b % 4 == 0)
    return launch_clusters(k_evict_compact<UA, 4>, pairs, C, CT, smem, st, "evict compact launch", a, C);
  return launch_clusters(k_evict_compact<UA, 2>, pairs, C, CT, smem, st, "evict compact launch", a, C);
}

}  // namespace

extern "C" int kvcu_evict_select(kvcu_pool* pool, uint32_t n_layers, uint32_t n, const uint32_t* seq_ids, uint32_t n_seqs,
                                 const uint32_t* lens, uint32_t budget, uint32_t n_sink, uint32_t n_recent,
                                 const float* mass, uint64_t mass_layer_stride, uint64_t mass_stride, uint32_t* keep,
                                 uint64_t keep_layer_stride, uint64_t keep_stride, uint32_t* keep_counts, void* stream) {
  if (!pool || !(pool->kv || pool->qs)) return KVCU_ERR_INVALID_ARG;
  if (budget == 0 || (uint64_t)n_sink + n_recent > budget || budget == KVCU_NO_POSITION) {
    kvcu_set_error("kvcu_evict_select: budget %u with %u first and %u last positions", budget, n_sink, n_recent);
    return KVCU_ERR_INVALID_ARG;
  }
  if (!n || !n_layers) return KVCU_OK;
  if (!lens || !mass || !keep || !keep_counts) {
    kvcu_set_error("kvcu_evict_select: null pointer argument");
    return KVCU_ERR_INVALID_ARG;
  }
  const uint64_t rows = (uint64_t)n * n_layers;
  if (keep_stride < budget || (n_layers > 1 && keep_layer_stride < (n - 1) * keep_stride + budget) || !mass_stride ||
      rows > 0x7FFFFFFu) {
    kvcu_set_error("kvcu_evict_select: strides or %llu rows out of range", (unsigned long long)rows);
    return KVCU_ERR_INVALID_ARG;
  }
  DevScope d(pool->device);
  if (d.rc) return d.rc;
  // CTAs of a row: a long row is shared until its keys fit the shared memory or
  // the shares get short; few rows are shared to occupy more SMs.
  const uint64_t sms = (uint64_t)kvcu_current_sm_count();
  uint32_t C = 1;
  while (C < 8 && (mass_stride / C > KVCU_EVICT_SMEM / 4 || (rows * C * 2 <= sms && mass_stride / C > 4096))) C *= 2;
  SelectArgs a = {mass, mass_layer_stride, mass_stride, n, n_seqs, seq_ids, lens, budget, n_sink, n_recent, keep,
                  keep_layer_stride, keep_stride, keep_counts, pool->status, 0};
  const uint64_t share = (mass_stride + C - 1) / C;
  a.cap = share < KVCU_EVICT_SMEM / 4 ? (uint32_t)share : (uint32_t)(KVCU_EVICT_SMEM / 4);
  const cudaStream_t st = (cudaStream_t)stream;
  if (C == 1) return launch_select<1>(a, (uint32_t)rows, st);
  if (C == 2) return launch_select<2>(a, (uint32_t)rows, st);
  if (C == 4) return launch_select<4>(a, (uint32_t)rows, st);
  return launch_select<8>(a, (uint32_t)rows, st);
}

extern "C" int kvcu_evict_compact(kvcu_pool* pool, uint32_t layer, uint32_t n_layers, uint32_t n, const uint32_t* seq_ids,
                                  uint32_t n_seqs, const uint32_t* table_offsets, const uint32_t* tables,
                                  const uint32_t* keep, uint64_t keep_layer_stride, uint64_t keep_stride,
                                  const uint32_t* keep_counts, float* mass, uint64_t mass_layer_stride,
                                  uint64_t mass_stride, uint32_t* lens, void* stream) {
  if (!pool || !(pool->kv || pool->qs)) return KVCU_ERR_INVALID_ARG;
  if (n_layers == 0 || layer >= pool->n_layers || n_layers > pool->n_layers - layer) {
    kvcu_set_error("kvcu_evict_compact: layers [%u, %u + %u) outside the pool's %u", layer, layer, n_layers,
                   pool->n_layers);
    return KVCU_ERR_LAYER_OOB;
  }
  if (!n) return KVCU_OK;
  if (!table_offsets || !tables || !keep || !keep_counts) {
    kvcu_set_error("kvcu_evict_compact: null pointer argument");
    return KVCU_ERR_INVALID_ARG;
  }
  const uint64_t pairs = (uint64_t)n * n_layers;
  if (pairs > 0x7FFFFFFu || !keep_stride) {
    kvcu_set_error("kvcu_evict_compact: %llu (layer, entry) pairs, keep stride %llu", (unsigned long long)pairs,
                   (unsigned long long)keep_stride);
    return KVCU_ERR_INVALID_ARG;
  }
  DevScope d(pool->device);
  if (d.rc) return d.rc;
  CompactArgs a = {};
  if (pool->quantized) {
    a.a = reinterpret_cast<char*>(pool->qs);
    a.b = reinterpret_cast<char*>(pool->sc);
    a.row_a = pool->nblk * 32;
    a.row_b = pool->nblk * 2;
  } else {
    a.a = reinterpret_cast<char*>(pool->kv);
    a.b = reinterpret_cast<char*>(pool->pe);
    a.row_a = pool->kv_rank * 4;
    a.row_b = pool->rope_dim * 4;
  }
  a.layer_rows = (uint64_t)pool->num_blocks * pool->block_size;
  a.num_blocks = pool->num_blocks;
  a.block_size = pool->block_size;
  a.layer = layer;
  a.n = n;
  a.n_seqs = n_seqs;
  a.seq_ids = seq_ids;
  a.toff = table_offsets;
  a.tables = tables;
  a.keep = keep;
  a.keep_lstride = keep_layer_stride;
  a.keep_stride = keep_stride;
  a.counts = keep_counts;
  a.mass = mass;
  a.mass_lstride = mass_layer_stride;
  a.mass_stride = mass_stride;
  a.lens = lens;
  a.status = pool->status;
  // two stages of about 20 KB, so that several CTAs share an SM
  const uint32_t row = a.row_a + ((a.row_b + 15u) & ~15u);
  uint32_t tile = 20480u / row;
  tile = tile < 1 ? 1 : tile > MAX_TILE ? MAX_TILE : tile;
  const size_t smem = 2ull * tile * row;
  if (smem > KVCU_EVICT_SMEM) {
    kvcu_set_error("kvcu_evict_compact: rows of %u bytes are too long", row);
    return KVCU_ERR_UNSUPPORTED;
  }
  a.tile = tile;
  // CTAs of a pair: more while the grid stays within four CTAs an SM
  const uint64_t sms = (uint64_t)kvcu_current_sm_count();
  uint32_t C = 1;
  while (C < 8 && pairs * C * 2 <= 4 * sms && (uint64_t)C * tile < keep_stride) C *= 2;
  const cudaStream_t st = (cudaStream_t)stream;
  if (a.row_a % 16 == 0) return launch_compact<16>(a, (uint32_t)pairs, C, smem, st);
  return launch_compact<4>(a, (uint32_t)pairs, C, smem, st);
}
