// kvcu_evict.cu — bounding a paged cache: which rows stay, and moving them.
//
// k_evict_select: per (layer, entry) the positions that stay under a budget: the
//   first n_sink, the last n_recent, and of those between the largest masses,
//   ties to the lowest position, as an ascending list.  A radix select on the
//   masses' 32-bit order (11 + 11 + 10 bits): the row is read once into shared
//   memory while the first histogram is formed, the other passes run there.
//   Floor: one read of the masses (4 B per position); bound: the instructions of three
//   passes, and the longest row, which one CTA has alone where there are more rows than
//   SMs (64,784 positions, as many as an SM's whole share).  512 rows of 1.5k to 65k
//   positions, 2,048 kept: 57 us (35.9 MB read once).  The first pass has four bins to an
//   octave: masses that all lie within one or two octaves share a few bins, whose atomics
//   collide and whose keys overflow the list, 101 us for the same rows.
// k_evict_compact: row j of a sequence := its row keep[j], in place through the
//   block table, in every layer, and the masses with it.  Bound: one read and
//   one write of the kept rows.  512 pairs of 2,048 rows of 612 B: 252 us, 4.3 TB/s; of
//   2,304 B (f32): 128 pairs 372 us, 256 pairs 725 us, 3.3 TB/s.
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
  uint32_t n_layers, n, n_seqs;
  const uint32_t* seq_ids;
  const uint32_t* lens;
  uint32_t budget, n_sink, n_recent;
  uint32_t* keep;
  uint64_t keep_lstride, keep_stride;
  uint32_t* counts;
  uint32_t* status;
  uint32_t cap;  // groups of four positions a CTA's shared memory holds
};

constexpr uint32_t BINS = 2048;
constexpr uint32_t LIST = 2048;
constexpr uint32_t ORDERED = 512;  // entries up to which rows are taken longest first
constexpr uint32_t SHARED_KEYS = 18432;  // 72 KB
constexpr int SELECT_THREADS = 512;

// Ascending 32-bit order of the values; -0 and +0 are one value, NaN is below
// everything.
__device__ __forceinline__ uint32_t order_key(float v) {
  const int b = __float_as_int(v + 0.0f);
  return v == v ? (uint32_t)(b ^ ((b >> 31) | (int)0x80000000)) : 0u;
}

__device__ __forceinline__ uint32_t warp_scan(uint32_t v, uint32_t lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= (uint32_t)o) v += y;
  }
  return v;
}

// Sum of the block's earlier warps' words part[w] (every warp scans them for itself).
template <int NT>
__device__ __forceinline__ uint32_t before_warp(const uint32_t* part, uint32_t warp, uint32_t lane) {
  const uint32_t p = lane < NT / 32 ? part[lane] : 0u;
  return __shfl_sync(0xffffffffu, warp_scan(p, lane) - p, warp);
}

// One row per cluster of C CTAs; each CTA holds an equal share of the row's
// middle, in order.
template <int C, int NT>
__global__ void __launch_bounds__(NT, 2) k_evict_select(SelectArgs a) {
  extern __shared__ uint4 cache[];  // [cap] order keys of this CTA's share, four positions each
  __shared__ uint32_t hist[BINS], total[BINS];
  __shared__ uint32_t part[NT / 32], part2[NT / 32];
  __shared__ uint2 list[LIST];  // (key, position in the share) of the threshold's first bin
  __shared__ uint32_t s_bin, s_above, s_listed, s_tot[2];
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  const uint32_t rank = C > 1 ? cluster_rank() : 0u;
  const uint32_t row = blockIdx.x / C;
  uint32_t layer = row / a.n, b = row % a.n;
  if (a.n > 1 && a.n <= ORDERED) {
    // long rows first, so that none starts when the others end: all layers of the
    // entry whose length has rank row / layers (a few loads and compares per CTA)
    for (uint32_t i = tid; i < a.n; i += NT) {
      const uint32_t q = a.seq_ids ? a.seq_ids[i] : i;
      total[i] = q < a.n_seqs ? a.lens[q] : 0u;
    }
    __syncthreads();
    layer = row % a.n_layers;
    for (uint32_t i = tid; i < a.n; i += NT) {
      const uint32_t mine = total[i];
      uint32_t rank_i = 0;
      for (uint32_t k = 0; k < a.n; ++k) rank_i += total[k] > mine || (total[k] == mine && k < i);
      if (rank_i == row / a.n_layers) s_bin = i;
    }
    __syncthreads();
    b = s_bin;
  }
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
  // The share in groups of four positions that are 16-byte aligned in memory: position
  // v = 4 g + j - off of it, which the first and last group may only have in part.
  const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(mass) >> 2) & 3u;
  const uint32_t groups = (cnt + off + 3) / 4;
  auto read = [&](uint32_t g) -> float4 {
    const uint32_t v = 4 * g - off;
    if (v < cnt && v + 4 <= cnt) return *reinterpret_cast<const float4*>(mass + v);
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (v < cnt) x.x = mass[v];
    if (v + 1 < cnt) x.y = mass[v + 1];
    if (v + 2 < cnt) x.z = mass[v + 2];
    if (v + 3 < cnt) x.w = mass[v + 3];
    return x;
  };
  auto keys_of = [&](float4 x) {
    return make_uint4(order_key(x.x), order_key(x.y), order_key(x.z), order_key(x.w));
  };
  auto keys_at = [&](uint32_t g) -> uint4 { return g < a.cap ? cache[g] : keys_of(read(g)); };
  auto whole = [&](uint32_t g) {
    const uint32_t v = 4 * g - off;
    return v < cnt && v + 4 <= cnt;
  };
  // f(key, position in the share) for the group's positions that are there
  auto each = [&](uint32_t g, const uint4& k, auto&& f) {
    const uint32_t v = 4 * g - off;
    if (v + 4 <= cnt && v < cnt) {
      f(k.x, v);
      f(k.y, v + 1);
      f(k.z, v + 2);
      f(k.w, v + 3);
      return;
    }
    if (v < cnt) f(k.x, v);
    if (v + 1 < cnt) f(k.y, v + 1);
    if (v + 2 < cnt) f(k.z, v + 2);
    if (v + 3 < cnt) f(k.w, v + 3);
  };

  // ---- radix select of the need-th largest key
  // Warps take runs of the groups in order.  The first pass over the share forms the
  // histogram of the keys' top 11 bits.  The second, knowing the threshold's bin,
  // counts each run's keys above it and lists those in it, so that the finer
  // histograms and the rest of the counts need only the list (where it overflows,
  // they go over the whole share).  The last pass writes.
  const uint32_t run = (groups + NT - 1) / NT * 32u;
  const uint32_t w0 = min(warp * run, groups), w1 = min(w0 + run, groups);
  if (tid == 0) s_listed = 0;
  if (tid < NT / 32) part2[tid] = 0;
  for (uint32_t i = tid; i < BINS; i += NT) hist[i] = 0;
  __syncthreads();
  constexpr uint32_t U = 4;  // groups of a thread in flight
  for (uint32_t g0 = w0 + lane; g0 < w1; g0 += U * 32) {
    float4 x[U];
#pragma unroll
    for (uint32_t j = 0; j < U; ++j)
      if (g0 + j * 32 < w1) x[j] = read(g0 + j * 32);
#pragma unroll
    for (uint32_t j = 0; j < U; ++j) {
      const uint32_t g = g0 + j * 32;
      if (g >= w1) break;
      const uint4 key = keys_of(x[j]);
      if (g < a.cap) cache[g] = key;
      each(g, key, [&](uint32_t v, uint32_t) { atomicAdd(&hist[v >> 21], 1u); });
    }
  }
  uint32_t prefix = 0, above = 0;  // keys above the prefix's range: all kept
  uint32_t sure = 0;               // this lane's keys above the first bin
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, top = pass == 1 ? 21 : 10;
    const uint32_t mask = pass == 2 ? 1023u : 2047u;
    if (pass) {
      for (uint32_t i = tid; i < BINS; i += NT) hist[i] = 0;
      if (pass == 1) {
        const uint32_t lo = prefix << 21;
        for (uint32_t g0 = w0 + lane; g0 < w1; g0 += U * 32) {
          uint4 k[U];
#pragma unroll
          for (uint32_t j = 0; j < U; ++j)
            if (g0 + j * 32 < w1) k[j] = keys_at(g0 + j * 32);
#pragma unroll
          for (uint32_t j = 0; j < U; ++j)
            if (g0 + j * 32 < w1) {
              const uint32_t g = g0 + j * 32, last = lo | 0x1FFFFFu;  // the bin's last key
              auto in_bin = [&](uint32_t v) { return v >= lo && v <= last; };
              auto note = [&](uint32_t v, uint32_t at) {
                if (!in_bin(v)) return;
                const uint32_t n = atomicAdd(&s_listed, 1u);
                if (n < LIST) list[n] = make_uint2(v, at);
              };
              if (whole(g)) {  // few keys are in the bin: one branch for the group
                sure += (k[j].x > last) + (k[j].y > last) + (k[j].z > last) + (k[j].w > last);
                if (in_bin(k[j].x) || in_bin(k[j].y) || in_bin(k[j].z) || in_bin(k[j].w)) each(g, k[j], note);
              } else {
                each(g, k[j], [&](uint32_t v, uint32_t at) {
                  sure += v > last;
                  note(v, at);
                });
              }
            }
        }
      }
      __syncthreads();
      auto add = [&](uint32_t v) {
        if ((v >> top) == prefix) atomicAdd(&hist[(v >> shift) & mask], 1u);
      };
      if (s_listed <= LIST) {
        for (uint32_t i = tid; i < s_listed; i += NT) add(list[i].x);
      } else {
#pragma unroll 4
        for (uint32_t g = w0 + lane; g < w1; g += 32) each(g, keys_at(g), [&](uint32_t v, uint32_t) { add(v); });
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
    const uint32_t in_warp = warp_scan(mine, lane);
    if (lane == 31) part[warp] = in_warp;
    __syncthreads();
    uint32_t upto = above + before_warp<NT>(part, warp, lane) + in_warp - mine;
    if (upto < need && need <= upto + mine) {
#pragma unroll
      for (uint32_t j = 0; j < PER; ++j) {
        if (upto < need && need <= upto + own[j]) {
          s_bin = BINS - 1 - (tid * PER + j);
          s_above = upto;
        }
        upto += own[j];
      }
    }
    __syncthreads();
    prefix = (prefix << (pass == 2 ? 10 : 11)) | s_bin;
    above = s_above;
  }
  const uint32_t ties = need - above;  // of the positions equal to the threshold, the first `ties`

  // ---- how many each run keeps: keys above the threshold, and equal ones
  if (s_listed > LIST) {
    uint32_t eq = 0;
    sure = 0;
#pragma unroll 4
    for (uint32_t g = w0 + lane; g < w1; g += 32)
      each(g, keys_at(g), [&](uint32_t v, uint32_t) {
        sure += v > prefix;
        eq += v == prefix;
      });
    eq = __reduce_add_sync(0xffffffffu, eq);
    if (lane == 0) part2[warp] = eq;
  }
  sure = __reduce_add_sync(0xffffffffu, sure);
  if (lane == 0) part[warp] = sure;
  __syncthreads();
  if (s_listed <= LIST) {
    for (uint32_t i = tid; i < s_listed; i += NT) {
      const uint2 e = list[i];
      if (e.x >= prefix) atomicAdd(e.x > prefix ? &part[(e.y + off) / 4 / run] : &part2[(e.y + off) / 4 / run], 1u);
    }
    __syncthreads();
  }
  uint32_t gt0 = before_warp<NT>(part, warp, lane), eq0 = before_warp<NT>(part2, warp, lane);
  if constexpr (C > 1) {
    if (tid == NT - 1) {
      s_tot[0] = gt0 + part[warp];
      s_tot[1] = eq0 + part2[warp];
    }
    cluster_sync();
    for (uint32_t r = 0; r < rank; ++r) {
      gt0 += ld_cluster(&s_tot[0], r);
      eq0 += ld_cluster(&s_tot[1], r);
    }
    cluster_sync();  // no CTA leaves while another reads its shared memory
  }

  // ---- the kept positions in order.  Counts go in pairs, those above the threshold in
  // the low half of a word, equal ones in the high.
  uint32_t* out = keep + a.n_sink;
#pragma unroll 2
  for (uint32_t g0 = w0; g0 < w1; g0 += 32) {
    const uint32_t g = g0 + lane;
    uint4 k = make_uint4(0, 0, 0, 0);
    uint32_t n = 0;
    if (g < w1) {
      k = keys_at(g);
      each(g, k, [&](uint32_t v, uint32_t) { n += v < prefix ? 0u : v == prefix ? 0x10000u : 1u; });
    }
    const uint32_t upto = warp_scan(n, lane), all = __shfl_sync(0xffffffffu, upto, 31);
    if (n) {
      uint32_t gi = gt0 + ((upto - n) & 0xFFFFu), ei = eq0 + ((upto - n) >> 16);
      each(g, k, [&](uint32_t v, uint32_t at) {
        if (v > prefix) {
          out[gi + min(ei, ties)] = p0 + at;
          ++gi;
        } else if (v == prefix) {
          if (ei < ties) out[gi + ei] = p0 + at;
          ++ei;
        }
      });
    }
    gt0 += all & 0xFFFFu;
    eq0 += all >> 16;
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
  uint64_t mass_lstride, mass_stride, mass_row;  // mass_row: positions of a row of sums
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

  // Thread r < tile has row r of the CTA's tile.  Its numbers run ahead of the
  // copies: the list is read three waves, the block table two waves before they are
  // needed, and neither is waited for until then.
  auto row_j = [&](uint32_t w) { return (w * C + rank) * a.tile + tid; };
  uint32_t pos, at = KVCU_NO_POSITION, blk_src = 0, blk_dst = 0;  // position fetched; position resolved, its blocks
  float val = 0.0f;
  auto fetch = [&](uint32_t w) { pos = tid < a.tile && row_j(w) < count ? keep[row_j(w)] : KVCU_NO_POSITION; };
  auto resolve = [&](uint32_t w) {
    const uint32_t j = row_j(w);
    at = pos == j ? KVCU_NO_POSITION : pos;  // a row that is in its place stays there
    if (at == KVCU_NO_POSITION) return;
    if (at / a.block_size >= t1 - t0 || j / a.block_size >= t1 - t0) {
      atomicOr(a.status, KVCU_STATUS_BAD_TABLE);
      at = KVCU_NO_POSITION;
      return;
    }
    blk_src = a.tables[t0 + at / a.block_size];
    blk_dst = a.tables[t0 + j / a.block_size];
    if (!mass) return;
    val = 0.0f;
    if (at < a.mass_row) val = __ldcg(mass + at);
    else atomicOr(a.status, KVCU_STATUS_BAD_LEN);
  };
  auto load = [&](uint32_t w) {  // the copies of wave w, resolved before
    const uint32_t f = w & 1u;
    if (tid < a.tile) {
      uint64_t src = NO_ROW, dst = NO_ROW;
      if (at != KVCU_NO_POSITION) {
        if (blk_src < a.num_blocks && blk_dst < a.num_blocks) {
          src = base + (uint64_t)blk_src * a.block_size + at % a.block_size;
          dst = base + (uint64_t)blk_dst * a.block_size + row_j(w) % a.block_size;
        } else {
          atomicOr(a.status, KVCU_STATUS_BAD_BLOCK);
        }
      }
      src_row[f][tid] = src;
      dst_row[f][tid] = dst;
      mval[f][tid] = val;
    }
    __syncthreads();
    if (w + 1 < waves) resolve(w + 1);
    if (w + 2 < waves) fetch(w + 2);
    char* st = smem + f * stage;
    const uint32_t sa = static_cast<uint32_t>(__cvta_generic_to_shared(st));
    for (uint32_t r = warp; r < a.tile; r += CT / 32) {
      const uint64_t src = src_row[f][r];
      if (src == NO_ROW) continue;
      for (uint32_t o = lane * UA; o < a.row_a; o += 32 * UA) copy_in<UA>(sa + r * a.row_a + o, a.a + src * a.row_a + o);
      const uint32_t sb = sa + a.tile * a.row_a + r * pad_b;
      for (uint32_t o = lane * UB; o < a.row_b; o += 32 * UB) copy_in<UB>(sb + o, a.b + src * a.row_b + o);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  fetch(0);
  resolve(0);
  if (waves > 1) fetch(1);
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
      if (j < a.mass_row) mass[j] = mval[f][tid];
    }
    __syncthreads();  // the stage may be filled again
  }
}

// ---- the same through registers: a thread has the same pieces of a tile's rows in
// every wave (up to three of 32 bytes and two of 4), so a wave costs it a handful of
// 256-bit loads and stores and no pass through shared memory; the next wave's loads
// are in flight while one is written.
//
// A piece is one word: its byte in the row, its row of the tile from bit 16, and
// whether it lies in the second array.
constexpr uint32_t SECOND = 0x80000000u, NO_PIECE = 0xFFFFFFFFu;
constexpr int WIDE = 3, WORDS = 2;  // three CTAs an SM; with four pieces and two CTAs 348 us where this takes 251
constexpr uint32_t REG_TILE = 56;  // rows at most

struct Wave {
  uint32_t wide[WIDE][8];
  uint32_t word[WORDS];
};

__device__ __forceinline__ void ld256(uint32_t (&v)[8], const char* p) {
  asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "l"(p)
               : "memory");
}
__device__ __forceinline__ void st256(char* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
               "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

__global__ void __launch_bounds__(CT, 3) k_evict_compact_wide(CompactArgs a, uint32_t C) {
  __shared__ uint64_t src_row[2][REG_TILE], dst_row[2][REG_TILE];
  const uint32_t tid = threadIdx.x;
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
  const uint32_t waves = (count + C * a.tile - 1) / (C * a.tile);
  // this thread's pieces: 32-byte ones of the first array, then of the second where its rows have
  // such; 4-byte words of the second otherwise
  const uint32_t ca = a.row_a / 32, cb = a.row_b % 32 ? 0u : a.row_b / 32, wb = cb ? 0u : a.row_b / 4;
  uint32_t wide[WIDE], word[WORDS];
#pragma unroll
  for (int i = 0; i < WIDE; ++i) {
    const uint32_t k = tid + i * CT, na = a.tile * ca;
    if (k < na) wide[i] = k / ca << 16 | k % ca * 32;
    else if (k - na < a.tile * cb) wide[i] = SECOND | (k - na) / cb << 16 | (k - na) % cb * 32;
    else wide[i] = NO_PIECE;
  }
#pragma unroll
  for (int i = 0; i < WORDS; ++i) {
    const uint32_t k = tid + i * CT;
    word[i] = k < a.tile * wb ? k / wb << 16 | k % wb * 4 : NO_PIECE;
  }
  auto row_in = [](uint32_t piece) { return piece >> 16 & 0xFFu; };
  auto wide_at = [&](uint32_t piece, uint64_t r) {
    return (piece & SECOND ? a.b + r * a.row_b : a.a + r * a.row_a) + (piece & 0xFFFFu);
  };
  auto word_at = [&](uint32_t piece, uint64_t r) {
    return reinterpret_cast<volatile uint32_t*>(a.b + r * a.row_b + (piece & 0xFFFFu));
  };
  // Thread r < tile has row r of the CTA's tile.  Its numbers run ahead of the
  // copies: the list is read three waves, the block table two waves before they are
  // needed, and neither is waited for until then.
  auto row_j = [&](uint32_t w) { return (w * C + rank) * a.tile + tid; };
  uint32_t pos = KVCU_NO_POSITION, at = KVCU_NO_POSITION, blk_src = 0, blk_dst = 0;
  float val[2] = {0.0f, 0.0f}, val_next = 0.0f;
  auto fetch = [&](uint32_t w) {
    pos = w < waves && tid < a.tile && row_j(w) < count ? keep[row_j(w)] : KVCU_NO_POSITION;
  };
  auto resolve = [&](uint32_t w) {
    const uint32_t j = row_j(w);
    at = pos == j ? KVCU_NO_POSITION : pos;  // a row that is in its place stays there
    if (at == KVCU_NO_POSITION) return;
    if (at / a.block_size >= t1 - t0 || j / a.block_size >= t1 - t0) {
      atomicOr(a.status, KVCU_STATUS_BAD_TABLE);
      at = KVCU_NO_POSITION;
      return;
    }
    blk_src = a.tables[t0 + at / a.block_size];
    blk_dst = a.tables[t0 + j / a.block_size];
    if (!mass) return;
    val_next = 0.0f;
    if (at < a.mass_row) val_next = __ldcg(mass + at);
    else atomicOr(a.status, KVCU_STATUS_BAD_LEN);
  };
  auto publish = [&](uint32_t w, float& v) {
    if (tid >= a.tile) return;
    uint64_t src = NO_ROW, dst = NO_ROW;
    if (at != KVCU_NO_POSITION) {
      if (blk_src < a.num_blocks && blk_dst < a.num_blocks) {
        src = base + (uint64_t)blk_src * a.block_size + at % a.block_size;
        dst = base + (uint64_t)blk_dst * a.block_size + row_j(w) % a.block_size;
      } else {
        atomicOr(a.status, KVCU_STATUS_BAD_BLOCK);
      }
    }
    src_row[w & 1u][tid] = src;
    dst_row[w & 1u][tid] = dst;
    v = val_next;
  };
  auto load = [&](uint32_t w, Wave& v) {
#pragma unroll
    for (int i = 0; i < WIDE; ++i) {
      if (wide[i] == NO_PIECE) continue;
      const uint64_t r = src_row[w & 1u][row_in(wide[i])];
      if (r != NO_ROW) ld256(v.wide[i], wide_at(wide[i], r));
    }
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      if (word[i] == NO_PIECE) continue;
      const uint64_t r = src_row[w & 1u][row_in(word[i])];
      if (r != NO_ROW) v.word[i] = *word_at(word[i], r);
    }
  };
  auto store = [&](uint32_t w, const Wave& v, float m) {
#pragma unroll
    for (int i = 0; i < WIDE; ++i) {
      if (wide[i] == NO_PIECE) continue;
      const uint64_t r = dst_row[w & 1u][row_in(wide[i])];
      if (r != NO_ROW) st256(wide_at(wide[i], r), v.wide[i]);
    }
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      if (word[i] == NO_PIECE) continue;
      const uint64_t r = dst_row[w & 1u][row_in(word[i])];
      if (r != NO_ROW) *word_at(word[i], r) = v.word[i];
    }
    if (mass && tid < a.tile && dst_row[w & 1u][tid] != NO_ROW && row_j(w) < a.mass_row) mass[row_j(w)] = m;
  };
  Wave even, odd;
  fetch(0);
  resolve(0);
  fetch(1);
  publish(0, val[0]);
  __syncthreads();
  load(0, even);
  resolve(1);
  fetch(2);
  // one wave: the next one's loads are sent, the cluster meets with this one's in registers, it is written
  auto step = [&](uint32_t w, Wave& now, Wave& next, float& v, float& v_next) {
    if (w + 1 < waves) {
      publish(w + 1, v_next);
      __syncthreads();
      load(w + 1, next);
      resolve(w + 2);
      fetch(w + 3);
    }
    if (C > 1) cluster_sync();
    else __syncthreads();
    store(w, now, v);
    __syncthreads();  // this wave's row numbers may be replaced
  };
  for (uint32_t w = 0; w < waves; w += 2) {
    step(w, even, odd, val[0], val[1]);
    if (w + 1 < waves) step(w + 1, odd, even, val[1], val[0]);
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
  return launch_clusters(k_evict_select<C, SELECT_THREADS>, rows, C, SELECT_THREADS, (size_t)a.cap * 16, st, "evict select launch", a);
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
  // CTAs of a row: few rows are shared to occupy the SMs, while the shares are not too short
  const uint64_t sms = (uint64_t)kvcu_current_sm_count();
  uint32_t C = 1;
  while (C < 8 && rows * C <= sms && mass_stride / C > 4096) C *= 2;
  SelectArgs a = {mass, mass_layer_stride, mass_stride, n_layers, n, n_seqs, seq_ids, lens, budget, n_sink, n_recent, keep,
                  keep_layer_stride, keep_stride, keep_counts, pool->status, 0};
  const uint64_t share = (mass_stride + C - 1) / C;
  // keys held in shared memory: with more CTAs than SMs two share an SM's, longer
  // shares are read again from L2 in each pass
  const uint64_t most = rows * C > sms ? SHARED_KEYS / 4 : KVCU_EVICT_SMEM / 16, need = share / 4 + 2;
  a.cap = (uint32_t)(need < most ? need : most);
  const cudaStream_t st = (cudaStream_t)stream;
  if (C == 1) return launch_select<1>(a, (uint32_t)rows, st);
  if (C == 2) return launch_select<2>(a, (uint32_t)rows, st);
  if (C == 4) return launch_select<4>(a, (uint32_t)rows, st);
  return launch_select<8>(a, (uint32_t)rows, st);
}

uint64_t kvcu_mass_row(uint32_t n_layers, uint32_t n, uint64_t layer_stride, uint64_t stride) {
  if (n_layers <= 1) return stride;
  const uint64_t small = layer_stride < stride ? layer_stride : stride, large = layer_stride < stride ? stride : layer_stride;
  if (n <= 1) return small;
  // the rows of the smaller stride lie between two of the larger
  const uint64_t steps = (layer_stride < stride ? n_layers : n) - 1u;
  if (small == 0 || large / steps < small || large == steps * small) return 0;
  const uint64_t last = large - steps * small;
  return small < last ? small : last;
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
  const uint64_t mass_row = mass ? kvcu_mass_row(n_layers, n, mass_layer_stride, mass_stride) : 0;
  if (mass && !mass_row) {
    kvcu_set_error("kvcu_evict_compact: rows of sums overlap at strides %llu (layers) and %llu (entries)",
                   (unsigned long long)mass_layer_stride, (unsigned long long)mass_stride);
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
  a.mass_row = mass_row;
  a.lens = lens;
  a.status = pool->status;
  const uint64_t sms = (uint64_t)kvcu_current_sm_count();
  const cudaStream_t st = (cudaStream_t)stream;
  // Rows of whole 32-byte pieces, with a second array of such or of whole words (every
  // Q8_0 pool of an even number of blocks, f32 pools of ranks divisible by 8), go through registers;
  // 512 pairs of 2,048 kept rows of 612 B: 251 us against 371 us through shared memory.
  const uint32_t pieces = a.row_a / 32 + (a.row_b % 32 ? 0u : a.row_b / 32);
  if (a.row_a % 32 == 0 && a.row_b % 4 == 0 && pieces <= WIDE * CT && a.row_a <= 65536 && a.row_b <= 65536) {
    a.tile = WIDE * CT / pieces;
    if (a.row_b % 32 && a.tile > WORDS * CT / (a.row_b / 4)) a.tile = WORDS * CT / (a.row_b / 4);
    if (a.tile > REG_TILE) a.tile = REG_TILE;
    if (a.tile > 0) {
      uint32_t C = 1;
      while (C < 8 && pairs * C * 2 <= 4 * sms && (uint64_t)C * a.tile < keep_stride) C *= 2;
      return launch_clusters(k_evict_compact_wide, (uint32_t)pairs, C, CT, 0, st, "evict compact launch", a, C);
    }
  }
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
  uint32_t C = 1;
  while (C < 8 && pairs * C * 2 <= 4 * sms && (uint64_t)C * tile < keep_stride) C *= 2;
  if (a.row_a % 16 == 0) return launch_compact<16>(a, (uint32_t)pairs, C, smem, st);
  return launch_compact<4>(a, (uint32_t)pairs, C, smem, st);
}
