// kvcu_mass.cu — the attention weight each cached position received.
//
// For entry b with queries i < n_q (the newest n_q positions' queries) and heads h
//   mass[b][p] = (p < old_lens[b] ? decay * mass[b][p] : 0)
//                + sum over i, h with p < len - (n_q - 1 - i) of exp(scale * q_ih . row_p - lse_ih)
// over the sequence's cached rows read through the block table; lse is the
// decode's log-sum-exp of the same scores, so the exponentials are the softmax
// weights themselves and a position's sum depends on no other position: no
// running maximum and nothing to join when a sequence is split over CTAs.
// CTAs take the ranges of the decode plan the caller made for the step, whose
// cost line (tokens, and a little per item) fits here too.
//
// The scores need f32-level accuracy (an error of the score is a relative error
// of the weight), so the products keep q's and the row's full precision.
#include <cuda_runtime.h>
#include <math.h>

#include "kvcu_internal.h"
#include "kvcu_numeric.cuh"

namespace {

constexpr int R = 512, P = 64, W = R + P;
constexpr uint32_t NBLK = W / 32;  // 32-value blocks of a Q8_0 row

struct MassArgs {
  uint32_t layer, num_blocks, block_size;
  const float* kv;
  const float* pe;
  const int8_t* qs;
  const uint16_t* sc;
  uint32_t* status;
  uint32_t n, n_seqs;
  const uint32_t* seq_ids;
  const uint32_t* toff;
  const uint32_t* tables;
  const uint32_t* lens;
  const uint32_t* entry_lens;
  const kvcu_item* items;
  const uint32_t* meta;
  const uint32_t* ranges;
  uint32_t n_q, n_heads;
  const float* q;
  const float* lse;
  float scale, decay;
  const uint32_t* old_lens;
  float* mass;
  uint64_t mass_stride;
};

// Work item `it`'s entry: its block table, length and the queries' limits.
struct Entry {
  uint32_t b, t0, t1, len, old;
};

__device__ __forceinline__ Entry entry_of(const MassArgs& a, uint32_t b, bool report) {
  Entry e = {b, 0, 0, 0, 0};
  const uint32_t s = a.seq_ids ? a.seq_ids[b] : b;
  if (b >= a.n || s >= a.n_seqs) {
    if (report) atomicOr(a.status, KVCU_STATUS_BAD_SEQ);
    return e;
  }
  e.t0 = a.toff[s];
  e.t1 = max(a.toff[s + 1], e.t0);
  uint64_t len = a.lens[s];
  if (a.entry_lens) len = min(len, (uint64_t)a.entry_lens[b]);
  const uint64_t most = min((uint64_t)(e.t1 - e.t0) * a.block_size, a.mass_stride);
  if (len > most) {
    if (report) atomicOr(a.status, KVCU_STATUS_BAD_LEN);
    len = most;
  }
  e.len = (uint32_t)len;
  e.old = a.old_lens ? a.old_lens[b] : e.len;
  return e;
}

// ------------------------------------------------------------------ CUDA cores
// Tiles of 64 rows in f32 in shared memory; lane l has tokens l and l + 32, warp w
// the columns (query, head) w, w + 8, ... of a chunk of 32.  Packed f32 FMAs.
constexpr int NT = 256, TT = 64, KS = W + 4, CC = 32;
constexpr int CC_SMEM = (TT * KS + CC * W + 8 * TT) * 4;

template <bool QUANT>
__global__ void __launch_bounds__(NT, 1) k_mass(MassArgs a) {
  extern __shared__ __align__(16) float smem[];
  float* k_s = smem;             // [TT][KS]
  float* q_s = k_s + TT * KS;    // [CC][W]
  float* red = q_s + CC * W;     // [8][TT]
  __shared__ long long rows[TT];
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  const uint32_t n_items = a.meta[0], n_ranges = a.meta[1];
  if (blockIdx.x == 0 && tid == 0 && n_ranges > gridDim.x) atomicOr(a.status, KVCU_STATUS_BAD_PLAN);
  const uint32_t it0 = blockIdx.x < n_ranges ? min(a.ranges[blockIdx.x], n_items) : n_items;
  const uint32_t it1 = blockIdx.x < n_ranges ? min(a.ranges[blockIdx.x + 1], n_items) : n_items;
  const uint32_t cols = a.n_q * a.n_heads;
  for (uint32_t it = it0; it < it1; ++it) {
    const kvcu_item item = a.items[it];
    const Entry e = entry_of(a, item.b, tid == 0);
    const uint32_t end = min(item.end, e.len);
    const float* qb = a.q + (uint64_t)item.b * cols * W;
    const float* lse = a.lse + (uint64_t)item.b * cols;
    bool q_loaded = false;
    for (uint32_t p0 = item.start; p0 < end; p0 += TT) {
      __syncthreads();
      if (tid < TT) {
        const uint32_t p = p0 + tid;
        long long r = -1;
        if (p < end) {
          const uint32_t blk = a.tables[e.t0 + p / a.block_size];
          if (blk < a.num_blocks)
            r = (long long)(((uint64_t)a.layer * a.num_blocks + blk) * a.block_size + p % a.block_size);
          else
            atomicOr(a.status, KVCU_STATUS_BAD_BLOCK);
        }
        rows[tid] = r;
      }
      __syncthreads();
      for (uint32_t t = warp; t < TT; t += NT / 32) {
        const long long r = rows[t];
        float4* dst = reinterpret_cast<float4*>(k_s + t * KS);
        if (r < 0) {
          for (uint32_t w = lane; w < W / 4; w += 32) dst[w] = make_float4(0.f, 0.f, 0.f, 0.f);
        } else if constexpr (QUANT) {
          const char4* src = reinterpret_cast<const char4*>(a.qs + (uint64_t)r * W);
          const uint16_t* sc = a.sc + (uint64_t)r * NBLK;
          for (uint32_t w = lane; w < W / 4; w += 32) {
            const char4 v = src[w];
            const float d = kvcu::f16_to_f32(sc[w / 8]);
            dst[w] = make_float4(d * v.x, d * v.y, d * v.z, d * v.w);
          }
        } else {
          const float4* kv = reinterpret_cast<const float4*>(a.kv + (uint64_t)r * R);
          const float4* pe = reinterpret_cast<const float4*>(a.pe + (uint64_t)r * P);
          for (uint32_t w = lane; w < W / 4; w += 32) dst[w] = w < R / 4 ? kv[w] : pe[w - R / 4];
        }
      }
      float sum = 0.f;  // of token tid
      for (uint32_t c0 = 0; c0 < cols; c0 += CC) {
        if (!q_loaded || cols > CC) {
          __syncthreads();
          for (uint32_t i = tid; i < CC * (W / 4); i += NT) {
            const uint32_t c = c0 + i / (W / 4);
            reinterpret_cast<float4*>(q_s)[i] =
                c < cols ? reinterpret_cast<const float4*>(qb + (uint64_t)c0 * W)[i] : make_float4(0.f, 0.f, 0.f, 0.f);
          }
          q_loaded = true;
        }
        __syncthreads();
        float2 acc[4][2];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j][0] = acc[j][1] = make_float2(0.f, 0.f);
        const float4* k0 = reinterpret_cast<const float4*>(k_s + lane * KS);
        const float4* k1 = reinterpret_cast<const float4*>(k_s + (lane + 32) * KS);
        const float4* qw = reinterpret_cast<const float4*>(q_s + warp * W);
        if (c0 + warp < cols) {
#pragma unroll 4
          for (int k = 0; k < W / 4; ++k) {
            const float4 u = k0[k], v = k1[k];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float4 x = qw[j * 8 * (W / 4) + k];
              const float2 xl = make_float2(x.x, x.y), xh = make_float2(x.z, x.w);
              acc[j][0] = __ffma2_rn(make_float2(u.x, u.y), xl, acc[j][0]);
              acc[j][0] = __ffma2_rn(make_float2(u.z, u.w), xh, acc[j][0]);
              acc[j][1] = __ffma2_rn(make_float2(v.x, v.y), xl, acc[j][1]);
              acc[j][1] = __ffma2_rn(make_float2(v.z, v.w), xh, acc[j][1]);
            }
          }
        }
        float w0 = 0.f, w1 = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t c = c0 + warp + 8 * j;
          if (c >= cols) continue;
          const float l = lse[c];
          if (l == -INFINITY) continue;  // a query that saw nothing
          const uint32_t back = a.n_q - 1 - c / a.n_heads;  // positions behind this query
          const uint32_t seen = e.len > back ? e.len - back : 0u;
          if (p0 + lane < seen) w0 += expf(fmaf(acc[j][0].x + acc[j][0].y, a.scale, -l));
          if (p0 + lane + 32 < seen) w1 += expf(fmaf(acc[j][1].x + acc[j][1].y, a.scale, -l));
        }
        red[warp * TT + lane] = w0;
        red[warp * TT + lane + 32] = w1;
        __syncthreads();
        if (tid < TT)
          for (int w = 0; w < 8; ++w) sum += red[w * TT + tid];
      }
      if (tid < TT && rows[tid] >= 0) {
        float* m = a.mass + (uint64_t)item.b * a.mass_stride + p0 + tid;
        *m = p0 + tid < e.old ? fmaf(a.decay, *m, sum) : sum;
      }
    }
  }
}

template <bool QUANT>
int launch_mass(const MassArgs& a, uint32_t grid, cudaStream_t st) {
  const int rc = kvcu_configure_once(
      reinterpret_cast<const void*>(k_mass<QUANT>),
      [](const void*) {
        return kvcu_check_cuda(
            cudaFuncSetAttribute(k_mass<QUANT>, cudaFuncAttributeMaxDynamicSharedMemorySize, CC_SMEM),
            "cudaFuncSetAttribute(mass)");
      },
      nullptr);
  if (rc) return rc;
  k_mass<QUANT><<<grid, NT, CC_SMEM, st>>>(a);
  return kvcu_check_cuda(cudaGetLastError(), "attention mass launch");
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

}  // namespace

extern "C" int kvcu_attn_mass(kvcu_decode_ws* ws, kvcu_pool* pool, uint32_t layer, uint32_t n, const uint32_t* seq_ids,
                              uint32_t n_seqs, const uint32_t* table_offsets, const uint32_t* tables,
                              const uint32_t* lens, uint32_t n_q, const float* q, const float* lse, uint32_t n_heads,
                              float scale, float decay, const uint32_t* old_lens, float* mass, uint64_t mass_stride,
                              void* stream) {
  if (!ws || !pool || !(pool->kv || pool->qs)) return KVCU_ERR_INVALID_ARG;
  if (ws->device != pool->device) {
    kvcu_set_error("kvcu_attn_mass: workspace on device %d, pool on %d", ws->device, pool->device);
    return KVCU_ERR_INVALID_ARG;
  }
  if (layer >= pool->n_layers) {
    kvcu_set_error("kvcu_attn_mass: layer %u >= n_layers %u", layer, pool->n_layers);
    return KVCU_ERR_LAYER_OOB;
  }
  if (pool->kv_rank != (uint32_t)R || pool->rope_dim != (uint32_t)P || n_heads == 0 || n_heads > 32) {
    kvcu_set_error("kvcu_attn_mass: kernels are built for kv_rank=%d, rope_dim=%d, 1..32 heads (got %u, %u, %u)", R, P,
                   pool->kv_rank, pool->rope_dim, n_heads);
    return KVCU_ERR_UNSUPPORTED;
  }
  if (!n) return KVCU_OK;
  if (n != ws->plan_n || ws->plan_layers != 1) {
    kvcu_set_error("kvcu_attn_mass: batch of %u entries, the workspace's last plan covers %u in %u layers", n, ws->plan_n,
                   ws->plan_layers);
    return KVCU_ERR_INVALID_ARG;
  }
  if (!table_offsets || !tables || !lens || !q || !lse || !mass || !mass_stride || ((uintptr_t)q & 15u)) {
    kvcu_set_error("kvcu_attn_mass: null pointer, zero stride, or q not 16-byte aligned");
    return KVCU_ERR_INVALID_ARG;
  }
  if (n_q == 0 || n_q > 65536u) {
    kvcu_set_error("kvcu_attn_mass: %u queries per entry, 1 .. 65536 supported", n_q);
    return KVCU_ERR_INVALID_ARG;
  }
  DevScope d(pool->device);
  if (d.rc) return d.rc;
  MassArgs a = {};
  a.layer = layer;
  a.num_blocks = pool->num_blocks;
  a.block_size = pool->block_size;
  a.kv = pool->kv;
  a.pe = pool->pe;
  a.qs = pool->qs;
  a.sc = pool->sc;
  a.status = pool->status;
  a.n = n;
  a.n_seqs = n_seqs;
  a.seq_ids = seq_ids;
  a.toff = table_offsets;
  a.tables = tables;
  a.lens = lens;
  a.entry_lens = ws->entry_lens;
  a.items = ws->items;
  a.meta = ws->meta;
  a.ranges = ws->ranges;
  a.n_q = n_q;
  a.n_heads = n_heads;
  a.q = q;
  a.lse = lse;
  a.scale = scale;
  a.decay = decay;
  a.old_lens = old_lens;
  a.mass = mass;
  a.mass_stride = mass_stride;
  const cudaStream_t st = (cudaStream_t)stream;
  const uint32_t grid = (uint32_t)ws->decode_ctas;
  return pool->quantized ? launch_mass<true>(a, grid, st) : launch_mass<false>(a, grid, st);
}
