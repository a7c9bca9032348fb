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
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>

#include "kvcu_internal.h"
#include "kvcu_tcgen05.cuh"

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

// ------------------------------------------------------------------ CUDA cores, f32 rows
// Tiles of 64 rows in f32 in shared memory; lane l has tokens l and l + 32, warp w
// the columns (query, head) w, w + 8, ... of a chunk of 32.  Packed f32 FMAs.
constexpr int NT = 256, TT = 64, KS = W + 4, CC = 32;
constexpr int CC_SMEM = (TT * KS + CC * W + 8 * TT) * 4;

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

// ------------------------------------------------------------------ tensor cores, Q8_0 rows
// A Q8_0 row is 18 blocks of 32 int8 values with a scale each.  int8 values are exact
// in f16, so per block and column D = sum of value * q runs on tcgen05 kind::f16 with
// M = 128 rows, and one f32 FMA with the row's block scale adds D to the row's score.
// q's columns are brought to [2^13, 2^14) by a power of two and split into two f16
// parts (22 bits), both accumulated into D, so the scores have f32's accuracy;
// rounding row or query to one f16 would cost 2e-3 of the weight.
//
// A thread owns one of a tile's 128 rows: it unpacks the row's blocks to f16 straight
// into TMEM (the MMA's A operand), reads the block sums back from its own TMEM lane
// and keeps the row's scores in registers.  Two warpgroups share a tile, each with
// half of the blocks: in a step one unpacks two blocks, hands them to the issuer
// (8 MMAs) and scales the sums of the step before, so unpacking, MMAs and scaling
// overlap.  At the tile's end they swap halves of the columns through shared memory,
// take the exponentials of their half, and the first adds the two sums to the mass.
//
//   warps 0-7   the two warpgroups
//   warp 8      producer: TMA boxes of 128 B x <= 128 rows (a "unit": four blocks of
//               every row of the tile; the fifth unit is the last two) through a ring
//               of five, scales and tile descriptions through a ring of two
//   warps 9-10  issue the MMAs, one for each warpgroup
//   warp 11     the next chunk's q parts into the other of two buffers (the first
//               chunk is prepared by all warps but the producer)
// More columns (queries x heads) than an instance has go in chunks: the item's rows
// are streamed again, from L2, for each.
//
// An earlier form on mma.sync, the sums of six slices of a row meeting in shared
// memory, took 492 us where this one takes MASS_LARGE us (192 sequences, 2.0 M rows).
constexpr int TC_THREADS = 384, TCT = 128, UNITS = 5;
constexpr uint32_t UNIT_BYTES = TCT * 128;
constexpr long long DRAIN_LIMIT = 1ll << 31;  // clocks a role that gives up waits for its own copies and MMAs
constexpr uint32_t TM_WG = 192, TM_D = 64, TM_COLS = 512;  // TMEM columns: of a warpgroup, start of its D, allocated
constexpr int COMPUTE = 8, PRODUCER = 8, ISSUER = 9 /* two */, FILLER = 11;

enum Bar : int {
  B_TF = 0,                // tile description and scales: full
  B_TE = B_TF + 2,         //   read
  B_UF = B_TE + 2,         // unit: full
  B_UE = B_UF + UNITS,     //   read
  B_Q0 = B_UE + UNITS,     // the first chunk's q parts
  B_QF = B_Q0 + 1,         // q parts: full
  B_QE = B_QF + 2,         //   done with
  B_AF = B_QE + 2,         // unpacked blocks in TMEM, per warpgroup and buffer
  B_DF = B_AF + 4,         // block sums ready, per warpgroup and buffer
  B_X = B_DF + 4,          // both warpgroups' scores swapped
  B_FINAL = B_X + 1,       // all MMAs of an issuer retired
  NUM_BARS = B_FINAL + 2
};

struct Tile {
  uint32_t b, p0, end, c0, old, ok;  // ok: bits of the boxes that were loaded
  uint32_t chunk;                    // counts the chunks of the CTA; q buffer chunk % 2
  uint32_t flags;                    // TILE_*
};
constexpr uint32_t TILE_LIVE = 1, TILE_FIRST = 2, TILE_LAST = 4;  // of its chunk

template <int NC>  // columns of a chunk
struct Map {
  static constexpr int HC = NC / 2;
  static constexpr int RB = (NC + 7) / 8 * 8;          // rows of a q part
  static constexpr uint32_t N = (RB + 15) / 16 * 16;   // MMA columns: the surplus reads rows of the next part
  static constexpr uint32_t REGION = 2 * RB * 128;     // 64 elements of the hi rows, then of the lo rows
  static constexpr uint32_t QBUF = (W / 64) * REGION;
  static constexpr uint32_t RING = 2 * QBUF;           // 1024-aligned, as every region and unit
  static constexpr uint32_t SC = RING + UNITS * UNIT_BYTES;
  static constexpr uint32_t X = SC + 2 * TCT * NBLK * 2;      // [2][warpgroup][HC][128] scores given away
  static constexpr uint32_t S = X + 2 * 2 * HC * TCT * 4;     // [2][128] the second warpgroup's sums
  static constexpr uint32_t COL = S + 2 * TCT * 4;            // [2][RB] scale, lse, limit
  static constexpr uint32_t TILES = COL + 2 * RB * 12;
  static constexpr uint32_t BARS = (TILES + 2 * sizeof(Tile) + 7) / 8 * 8;
  static constexpr uint32_t MISC = BARS + NUM_BARS * 8;       // TMEM base, abort flag
  static constexpr uint32_t ALLOC = MISC + 16 + 1024;
  static_assert(ALLOC <= 232448, "shared memory budget");
  static_assert(REGION % 1024 == 0 && NC % 4 == 0 && TM_D + 4 * N <= TM_WG, "layout");
};

struct TcMass {
  MassArgs m;
  uint32_t box_rows;
  long long wait_limit;
};

// Bounded wait: false after `limit` clocks or when another role has given up.
__device__ __forceinline__ bool wait_slow(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag, long long limit) {
  const long long t0 = clock64();
  while (!kvtc::mbar_try(bar, parity))
    if (*abort_flag || clock64() - t0 > limit) {
      *abort_flag = 1u;
      return false;
    }
  return true;
}
// One verdict for the converged warp.
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag, long long limit) {
  const bool ok = kvtc::mbar_try(bar, parity) || wait_slow(bar, parity, abort_flag, limit);
  return __all_sync(0xffffffffu, ok);
}

__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
// D (+)= A B with A in TMEM, f16 x f16 -> f32
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Four int8 values as two f16 pairs, exact: a biased byte u in the low mantissa of
// 1024 is 1024 + u; minus 1152 leaves u - 128.
__device__ __forceinline__ void int8_to_f16(uint32_t w, uint32_t* out) {
  const uint32_t u = w ^ 0x80808080u;
  const __half2 bias = __half2half2(__ushort_as_half(0x6480));
  const uint32_t x = __byte_perm(u, 0x64646464u, 0x4140), y = __byte_perm(u, 0x64646464u, 0x4342);
  const __half2 r0 = __hsub2(*reinterpret_cast<const __half2*>(&x), bias);
  const __half2 r1 = __hsub2(*reinterpret_cast<const __half2*>(&y), bias);
  out[0] = *reinterpret_cast<const uint32_t*>(&r0);
  out[1] = *reinterpret_cast<const uint32_t*>(&r1);
}

__device__ __forceinline__ uint32_t pack_half(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Rows first, first + step, ... of the q parts of (entry b, columns from c0) and their
// columns' scales, by one warp; the next row is loaded while one is split.
template <int NC>
__device__ __forceinline__ void fill_rows(const MassArgs& a, char* sm, uint32_t buf, uint32_t first, uint32_t step,
                                          uint32_t b, uint32_t c0, uint32_t cols, uint32_t lane) {
  using M = Map<NC>;
  float* col = reinterpret_cast<float*>(sm + M::COL) + buf * 3 * M::RB;
  char* q = sm + buf * M::QBUF;
  float4 x[5], nx[5];
  auto load = [&](uint32_t r, float4* v) {
    const bool live = r < NC && c0 + r < cols;
    const float4* src = reinterpret_cast<const float4*>(a.q + ((uint64_t)b * cols + c0 + r) * W);
#pragma unroll
    for (int i = 0; i < 5; ++i) {
      const uint32_t f = lane + 32 * i;
      v[i] = live && f < W / 4 ? src[f] : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  load(first, nx);
  for (uint32_t r = first; r < (uint32_t)M::RB; r += step) {
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 5; ++i) {
      x[i] = nx[i];
      amax = fmaxf(fmaxf(fmaxf(amax, fabsf(x[i].x)), fmaxf(fabsf(x[i].y), fabsf(x[i].z))), fabsf(x[i].w));
    }
    if (r + step < (uint32_t)M::RB) load(r + step, nx);
    // all values are >= 0: their bits order as integers
    const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(amax));
    // 2^(13 - exponent of the maximum); 1 for a column of zeros or with an infinity
    const uint32_t eb = top >> 23;
    const uint32_t f2 = top == 0u || eb == 255u ? 127u : min(max(267 - (int)eb, 1), 253);
    const float up = __uint_as_float(f2 << 23);
    if (lane == 0) col[r] = a.scale * __uint_as_float((254u - f2) << 23);
#pragma unroll
    for (int i = 0; i < 5; ++i) {
      const uint32_t f = lane + 32 * i;  // elements 4f .. 4f + 3
      if (f >= W / 4) continue;
      const float y0 = x[i].x * up, y1 = x[i].y * up, y2 = x[i].z * up, y3 = x[i].w * up;
      const uint2 hi = make_uint2(pack_half(y0, y1), pack_half(y2, y3));
      const float2 h0 = __half22float2(*reinterpret_cast<const __half2*>(&hi.x));
      const float2 h1 = __half22float2(*reinterpret_cast<const __half2*>(&hi.y));
      char* at = q + (f / 16) * M::REGION;
      *reinterpret_cast<uint2*>(at + kvtc::sw128_off(r, (f % 16) * 8)) = hi;
      *reinterpret_cast<uint2*>(at + kvtc::sw128_off(M::RB + r, (f % 16) * 8)) =
          make_uint2(pack_half(y0 - h0.x, y1 - h0.y), pack_half(y2 - h1.x, y3 - h1.y));
    }
  }
}

// Each column's lse and the positions below which it counts, a lane each.
template <int NC>
__device__ __forceinline__ void fill_columns(const MassArgs& a, char* sm, uint32_t buf, uint32_t b, uint32_t c0,
                                             uint32_t len, uint32_t cols, uint32_t lane) {
  using M = Map<NC>;
  const uint32_t c = c0 + lane;
  if (lane >= (uint32_t)M::RB) return;
  const float l = lane < NC && c < cols ? a.lse[(uint64_t)b * cols + c] : -INFINITY;
  const uint32_t behind = a.n_q - 1 - c / a.n_heads;  // positions behind the column's query
  float* col = reinterpret_cast<float*>(sm + M::COL) + buf * 3 * M::RB;
  col[M::RB + lane] = l;
  // a column past the last, or a query that saw nothing, has no positions
  reinterpret_cast<uint32_t*>(col)[2 * M::RB + lane] = l == -INFINITY || len <= behind ? 0u : len - behind;
}

// The CTA's items one after another, 32 at a time so that their chains of dependent
// loads (item, sequence, length and table) run side by side.  All lanes of a warp.
struct Items {
  uint32_t it, it1, at;  // next item; end; items of the batch used
  kvcu_item mine;
  Entry me;
  uint32_t b, start, end, len, old, t0;  // the current item
  __device__ __forceinline__ bool next(const MassArgs& a, uint32_t lane, bool report) {
    while (it < it1) {
      const uint32_t k = at & 31u;
      if (k == 0) {
        mine = {0, 0, 0, 0};
        me = {0, 0, 0, 0, 0};
        if (it + lane < it1) {
          mine = a.items[it + lane];
          me = entry_of(a, mine.b, report);
        }
      }
      b = __shfl_sync(0xffffffffu, mine.b, k);
      start = __shfl_sync(0xffffffffu, mine.start, k);
      len = __shfl_sync(0xffffffffu, me.len, k);
      old = __shfl_sync(0xffffffffu, me.old, k);
      t0 = __shfl_sync(0xffffffffu, me.t0, k);
      end = min(__shfl_sync(0xffffffffu, mine.end, k), len);
      ++it;
      ++at;
      if (start < end) return true;
    }
    return false;
  }
};

template <int NC>
__global__ void __launch_bounds__(TC_THREADS, 1)
    k_mass_tc(const __grid_constant__ CUtensorMap wide, const __grid_constant__ CUtensorMap tail, const TcMass t) {
  using M = Map<NC>;
  const MassArgs& a = t.m;
  extern __shared__ char raw[];
  char* sm = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  const uint32_t base = kvtc::smem_u32(sm);
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(sm + M::MISC + 4);
  auto bar = [&](int i) { return base + M::BARS + 8u * (uint32_t)i; };
  auto wait = [&](int i, uint32_t parity) { return wait_bar(bar(i), parity, abort_flag, t.wait_limit); };
  if (tid == 0) {
    const int counts[NUM_BARS] = {1, 1, COMPUTE + 2, COMPUTE + 2, 1, 1, 1, 1, 1, COMPUTE, COMPUTE, COMPUTE, COMPUTE, COMPUTE,
                                  COMPUTE + 3, 1, 1, COMPUTE, COMPUTE, 4, 4, 4, 4, 1, 1, 1, 1, COMPUTE, 1, 1};
    for (int i = 0; i < NUM_BARS; ++i) kvtc::mbar_init(bar(i), counts[i]);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == ISSUER) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + M::MISC), "r"(TM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  kvcu_pdl_wait();  // launched programmatically: the set-up above overlaps the previous kernel's tail
  kvtc::tc_fence_before();
  __syncthreads();
  kvtc::tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(sm + M::MISC);
  const uint32_t cols = a.n_q * a.n_heads;
  const uint32_t n_items = a.meta[0], n_ranges = a.meta[1];
  Items items = {};
  items.it = blockIdx.x < n_ranges ? min(a.ranges[blockIdx.x], n_items) : n_items;
  items.it1 = blockIdx.x < n_ranges ? min(a.ranges[blockIdx.x + 1], n_items) : n_items;
  const Tile* tiles = reinterpret_cast<const Tile*>(sm + M::TILES);
  // the q parts of chunk c of the CTA: the first has a barrier of its own
  auto wait_q = [&](uint32_t c) { return c == 0 ? wait(B_Q0, 0) : wait(B_QF + (c & 1u), ((c >> 1) - (c & 1u ? 0 : 1)) & 1u); };

  if (warp == PRODUCER) {
    // ---------------------------------------------------------------- producer
    if (blockIdx.x == 0 && lane == 0 && n_ranges > gridDim.x) atomicOr(a.status, KVCU_STATUS_BAD_PLAN);
    const uint32_t boxes = TCT / t.box_rows;
    uint32_t ti = 0, ui = 0, chunk = 0;
    bool ok = true;
    while (ok && items.next(a, lane, true)) {
      auto block_at = [&](uint32_t p0) -> uint32_t {  // of this lane's box
        const uint32_t p = p0 + lane * t.box_rows;
        return lane < boxes && p < items.end ? a.tables[items.t0 + p / a.block_size] : 0xFFFFFFFFu;
      };
      for (uint32_t c0 = 0; ok && c0 < cols; c0 += NC, ++chunk) {
        uint32_t next = block_at(items.start);
        for (uint32_t p0 = items.start; ok && p0 < items.end; p0 += TCT, ++ti) {
          const uint32_t blk = next, p = p0 + lane * t.box_rows;
          next = block_at(p0 + TCT < items.end ? p0 + TCT : items.end);
          const bool in = lane < boxes && p < items.end, good = in && blk < a.num_blocks;
          if (in && !good && c0 == 0) atomicOr(a.status, KVCU_STATUS_BAD_BLOCK);
          const uint32_t votes = __ballot_sync(0xffffffffu, good);
          const uint64_t row = ((uint64_t)a.layer * a.num_blocks + blk) * a.block_size + p % a.block_size;
          const uint32_t ts = ti & 1u;
          if (!(ok = wait(B_TE + ts, ((ti >> 1) & 1u) ^ 1u))) break;
          if (lane == 0) {
            const uint32_t flags = TILE_LIVE | (p0 == items.start ? TILE_FIRST : 0u) |
                                   (p0 + TCT >= items.end ? TILE_LAST : 0u);
            *reinterpret_cast<Tile*>(sm + M::TILES + ts * sizeof(Tile)) = {items.b, p0, items.end, c0, items.old, votes,
                                                                           chunk, flags};
            kvtc::mbar_arrive_tx(bar(B_TF + ts), __popc(votes) * t.box_rows * NBLK * 2);
          }
          __syncwarp();
          if (good)
            bulk_load(base + M::SC + (ts * TCT + lane * t.box_rows) * NBLK * 2, a.sc + row * NBLK, t.box_rows * NBLK * 2,
                      bar(B_TF + ts));
          for (uint32_t u = 0; u < UNITS; ++u, ++ui) {
            const uint32_t slot = ui % UNITS, width = u < 4 ? 128u : 64u;
            if (!(ok = wait(B_UE + slot, ((ui / UNITS) & 1u) ^ 1u))) break;
            if (lane == 0) kvtc::mbar_arrive_tx(bar(B_UF + slot), __popc(votes) * t.box_rows * width);
            __syncwarp();
            if (good)
              tma_2d(base + M::RING + slot * UNIT_BYTES + lane * t.box_rows * width, u < 4 ? &wide : &tail, (int)(u * 128),
                     (int)row, bar(B_UF + slot));
          }
        }
      }
    }
    if (ok && (ok = wait(B_TE + (ti & 1u), ((ti >> 1) & 1u) ^ 1u)) && lane == 0) {
      reinterpret_cast<Tile*>(sm + M::TILES)[ti & 1u].flags = 0;
      kvtc::mbar_arrive(bar(B_TF + (ti & 1u)));
    }
    if (!ok) {
      // the copies in flight must land before the CTA leaves
      const long long t0 = clock64();
      for (uint32_t k = ui > UNITS ? ui - UNITS : 0; k < ui; ++k)
        while (!kvtc::mbar_try(bar(B_UF + k % UNITS), (k / UNITS) & 1u) && clock64() - t0 <= DRAIN_LIMIT) {
        }
      for (uint32_t k = ti > 2 ? ti - 2 : 0; k < ti; ++k)
        while (!kvtc::mbar_try(bar(B_TF + (k & 1u)), (k >> 1) & 1u) && clock64() - t0 <= DRAIN_LIMIT) {
        }
    }
  } else {
    // ---------------------------------------------------------------- the first chunk's q parts
    const bool any = items.next(a, lane, false);
    if (any) {
      const uint32_t me = warp < COMPUTE ? warp : warp - 1;
      if (me == 0) fill_columns<NC>(a, sm, 0, items.b, 0, items.len, cols, lane);
      fill_rows<NC>(a, sm, 0, me, COMPUTE + 3, items.b, 0, cols, lane);
      kvtc::fence_proxy_async();
      __syncwarp();
      if (lane == 0) kvtc::mbar_arrive(bar(B_Q0));
    }
    if (warp == FILLER) {
      // -------------------------------------------------------------- the later chunks' q parts
      uint32_t c0 = NC, chunk = 1;
      bool ok = any;
      while (ok) {
        if (c0 >= cols) {
          if (!items.next(a, lane, false)) break;
          c0 = 0;
        }
        if (!(ok = wait(B_QE + (chunk & 1u), ((chunk >> 1) & 1u) ^ 1u))) break;
        fill_columns<NC>(a, sm, chunk & 1u, items.b, c0, items.len, cols, lane);
        fill_rows<NC>(a, sm, chunk & 1u, 0, 1, items.b, c0, cols, lane);
        kvtc::fence_proxy_async();
        __syncwarp();
        if (lane == 0) kvtc::mbar_arrive(bar(B_QF + (chunk & 1u)));
        c0 += NC;
        ++chunk;
      }
    } else if (warp >= ISSUER) {
      // -------------------------------------------------------------- MMA issuers, one per warpgroup
      // kind::f16: D f32 (bit 4), A and B f16, both K-major, N >> 3 at bit 17, M >> 4 at bit 24
      constexpr uint32_t IDESC = (1u << 4) | ((M::N >> 3) << 17) | ((uint32_t)(TCT >> 4) << 24);
      const uint32_t g = warp - ISSUER;
      uint32_t j = 0;
      bool ok = true;
      for (uint32_t ti = 0; ok; ++ti) {
        if (!wait(B_TF + (ti & 1u), (ti >> 1) & 1u)) break;
        const uint32_t flags = tiles[ti & 1u].flags, chunk = tiles[ti & 1u].chunk;
        __syncwarp();
        if (lane == 0) kvtc::mbar_arrive(bar(B_TE + (ti & 1u)));
        if (!(flags & TILE_LIVE)) break;
        if ((flags & TILE_FIRST) && !wait_q(chunk)) break;
        // a descriptor's address field counts 16 bytes: offsets are added to the buffer's
        const uint64_t q = kvtc::smem_desc(base + (chunk & 1u) * M::QBUF, 16, 1024, kvtc::LAYOUT_SW128);
#pragma unroll
        for (uint32_t u = 0; u < UNITS; ++u, ++j) {
          const uint32_t f = j & 1u;
          if (!(ok = wait(B_AF + 2 * g + f, (j >> 1) & 1u))) break;
          kvtc::tc_fence_after();
          if (kvtc::elect_one()) {
            const uint32_t ta = tmem + g * TM_WG + f * 32u, td = tmem + g * TM_WG + TM_D + f * 2u * M::N;
            // block 4u + 2g + e, the last 16 + g; two blocks to a region of 64 elements
            const uint64_t at = q + (u < 4 ? (2 * u + g) * M::REGION : 8 * M::REGION + g * 64u) / 16;
#pragma unroll
            for (uint32_t e = 0; e < (u < 4 ? 2u : 1u); ++e)
#pragma unroll
              for (uint32_t ks = 0; ks < 2; ++ks) {
                mma_ts(td + e * M::N, ta + e * 16u + ks * 8u, at + (e * 64u + ks * 32u) / 16, IDESC, ks);
                mma_ts(td + e * M::N, ta + e * 16u + ks * 8u, at + (M::RB * 128u + e * 64u + ks * 32u) / 16, IDESC, 1u);
              }
            kvtc::mma_commit(bar(B_DF + 2 * g + f));
          }
          __syncwarp();
        }
      }
      // all issued MMAs retire before TMEM is freed
      if (kvtc::elect_one()) kvtc::mma_commit(bar(B_FINAL + g));
      __syncwarp();
      const long long t0 = clock64();
      while (!kvtc::mbar_try(bar(B_FINAL + g), 0) && clock64() - t0 <= DRAIN_LIMIT) {
      }
    } else {
      // -------------------------------------------------------------- the warpgroups
      constexpr int HC = M::HC;
      const uint32_t g = warp >> 2, r = (warp & 3u) * 32u + lane;
      const uint32_t tw = tmem + ((warp & 3u) * 32u << 16) + g * TM_WG;
      float* xs = reinterpret_cast<float*>(sm + M::X);
      float* sums = reinterpret_cast<float*>(sm + M::S);
      uint32_t j = 0, ui = 0, ti = 0;
      // the first warpgroup: the tile before, whose mass is written once the other's sum is there
      float* out = nullptr;
      float keep_old = 0.f, factor = 1.f, own = 0.f;
      bool ok = true;
      float2 tot[NC / 2];
      Tile d = {};        // the tile whose scores are being formed
      uint32_t last = 0;  // its last block's scale
#pragma unroll
      for (int c = 0; c < NC / 2; ++c) tot[c] = make_float2(0.f, 0.f);
      // adds the sums of step jj (`blocks` of them) to the scores
      auto drain = [&](uint32_t jj, int blocks, uint32_t scales) -> bool {
        const uint32_t f = jj & 1u;
        if (!wait(B_DF + 2 * g + f, (jj >> 1) & 1u)) return false;
        kvtc::tc_fence_after();
        const float2 sc = __half22float2(*reinterpret_cast<const __half2*>(&scales));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (e < blocks) {
            uint32_t v[NC];
            kvtc::tmem_ld<NC>(tw + TM_D + f * 2u * M::N + e * M::N, v);
            kvtc::tmem_wait_ld();
            kvtc::reg_fence(v);
            const float de = e ? sc.y : sc.x;
#pragma unroll
            for (int c = 0; c < NC / 2; ++c)
              tot[c] = __ffma2_rn(make_float2(__uint_as_float(v[2 * c]), __uint_as_float(v[2 * c + 1])),
                                  make_float2(de, de), tot[c]);
          }
        }
        return true;
      };
      // tile d, number k of the CTA, whose last step is j1: the rest of its scores, their weights, its sums
      auto finish = [&](uint32_t k, uint32_t j1) -> bool {
        if (!drain(j1, 1, last)) return false;
        if ((d.flags & TILE_FIRST) && !wait_q(d.chunk)) return false;  // its columns' scales
        // each warpgroup gives away the other's half of the columns
        const uint32_t ts = k & 1u;
        float* give = xs + (ts * 2 + g) * HC * TCT + r;
        const float* got = xs + (ts * 2 + (g ^ 1u)) * HC * TCT + r;
        float mine[HC];
#pragma unroll
        for (int c = 0; c < HC; ++c) {
          const float lo = c & 1 ? tot[c / 2].y : tot[c / 2].x;
          const int c2 = c + HC;
          const float hi = c2 & 1 ? tot[c2 / 2].y : tot[c2 / 2].x;
          mine[c] = g ? hi : lo;
          give[c * TCT] = g ? lo : hi;
        }
        __syncwarp();
        if (lane == 0) kvtc::mbar_arrive(bar(B_X));
        if (!wait(B_X, k & 1u)) return false;
        if (out) *out = fmaf(factor, keep_old, own + sums[(ts ^ 1u) * TCT + r]);
        const uint32_t qb = d.chunk & 1u, p = d.p0 + r;
        const float* col = reinterpret_cast<const float*>(sm + M::COL) + qb * 3 * M::RB + g * HC;
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < HC; ++c) {
          const float s = mine[c] + got[c * TCT];
          if (p < reinterpret_cast<const uint32_t*>(col)[2 * M::RB + c]) sum += expf(fmaf(s, col[c], -col[M::RB + c]));
        }
        if (g) {
          sums[ts * TCT + r] = sum;
        } else {
          own = sum;
          out = nullptr;
          keep_old = 0.f;
          if (p < d.end && (d.ok >> (r / t.box_rows) & 1u)) {
            out = a.mass + (uint64_t)d.b * a.mass_stride + p;
            factor = d.c0 ? 1.f : a.decay;
            if (d.c0 || p < d.old) keep_old = *out;
          }
        }
        if (d.flags & TILE_LAST) {
          __syncwarp();
          if (lane == 0) kvtc::mbar_arrive(bar(B_QE + qb));
        }
#pragma unroll
        for (int c = 0; c < NC / 2; ++c) tot[c] = make_float2(0.f, 0.f);
        return true;
      };
      while (true) {
        const uint32_t ts = ti & 1u;
        if (!(ok = wait(B_TF + ts, (ti >> 1) & 1u))) break;
        const Tile now = tiles[ts];
        uint32_t scales[5];  // of this warpgroup's blocks: pairs 2u, 2u + 1 of unit u; the last is one block
        const uint32_t* sp = reinterpret_cast<const uint32_t*>(sm + M::SC + (ts * TCT + r) * NBLK * 2);
#pragma unroll
        for (int u = 0; u < 4; ++u) scales[u] = sp[2 * u + g];
        scales[4] = g ? sp[8] >> 16 : sp[8];
        __syncwarp();
        if (lane == 0) kvtc::mbar_arrive(bar(B_TE + ts));
        if (!(now.flags & TILE_LIVE)) break;
#pragma unroll
        for (int u = 0; u < UNITS; ++u, ++ui, ++j) {
          const uint32_t slot = ui % UNITS;
          if (!(ok = wait(B_UF + slot, (ui / UNITS) & 1u))) break;
          const char* st = sm + M::RING + slot * UNIT_BYTES;
          uint32_t af[32];
          const uint32_t ta = tw + (j & 1u) * 32u;
          if (u < 4) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint4 w = *reinterpret_cast<const uint4*>(st + kvtc::sw128_off(r, (g * 4 + k) * 16));
              int8_to_f16(w.x, af + 8 * k);
              int8_to_f16(w.y, af + 8 * k + 2);
              int8_to_f16(w.z, af + 8 * k + 4);
              int8_to_f16(w.w, af + 8 * k + 6);
            }
            kvtc::tmem_st<32>(ta, af);
          } else {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const uint4 w = *reinterpret_cast<const uint4*>(st + kvtc::sw64_off(r, (g * 2 + k) * 16));
              int8_to_f16(w.x, af + 8 * k);
              int8_to_f16(w.y, af + 8 * k + 2);
              int8_to_f16(w.z, af + 8 * k + 4);
              int8_to_f16(w.w, af + 8 * k + 6);
            }
            kvtc::tmem_st<16>(ta, af);
          }
          kvtc::tmem_wait_st();
          kvtc::tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            kvtc::mbar_arrive(bar(B_UE + slot));
            kvtc::mbar_arrive(bar(B_AF + 2 * g + (j & 1u)));
          }
          // the step before: of this tile, or the last of the tile before, which is then finished
          // while this tile's first MMAs run
          if (u > 0) ok = drain(j - 1, 2, scales[u > 0 ? u - 1 : 0]);
          else if (ti > 0) ok = finish(ti - 1, j - 1);
          if (!ok) break;
          if (u == 0) {
            d = now;
            last = scales[4];
          }
        }
        if (!ok) break;
        ++ti;
      }
      if (ok && ti > 0) ok = finish(ti - 1, j - 1);
      if (ok) {  // the last tile's sums
        __syncwarp();
        if (lane == 0) kvtc::mbar_arrive(bar(B_X));
        if (wait(B_X, ti & 1u) && out) *out = fmaf(factor, keep_old, own + sums[((ti & 1u) ^ 1u) * TCT + r]);
      }
    }
  }
  // ---- teardown
  kvcu_pdl_trigger();
  __syncwarp();
  kvtc::tc_fence_before();
  __syncthreads();
  if (tid == 0 && *abort_flag) atomicOr(a.status, KVCU_STATUS_TIMEOUT);
  if (warp == ISSUER) {
    kvtc::tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TM_COLS) : "memory");
  }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Boxes of a row's 128-byte pieces (bytes 0 .. 511) and of its last 64 bytes.
int make_maps(const kvcu_pool* p, uint32_t box_rows, CUtensorMap* wide, CUtensorMap* tail) {
  static EncodeTiledFn enc = []() -> EncodeTiledFn {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return nullptr;
    return reinterpret_cast<EncodeTiledFn>(f);
  }();
  if (!enc) {
    kvcu_set_error("cuTensorMapEncodeTiled unavailable");
    return KVCU_ERR_CUDA;
  }
  const cuuint64_t dims[2] = {(cuuint64_t)W, (cuuint64_t)p->rows()};
  const cuuint64_t strides[1] = {(cuuint64_t)W};
  const cuuint32_t estr[2] = {1, 1}, box_wide[2] = {128, box_rows}, box_tail[2] = {64, box_rows};
  const CUresult r = enc(wide, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, p->qs, dims, strides, box_wide, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  const CUresult r2 = enc(tail, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, p->qs, dims, strides, box_tail, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS || r2 != CUDA_SUCCESS) {
    kvcu_set_error("cuTensorMapEncodeTiled failed: %d, %d", (int)r, (int)r2);
    return KVCU_ERR_CUDA;
  }
  return KVCU_OK;
}

template <int NC>
int launch_mass_tc(const kvcu_pool* pool, const MassArgs& a, uint32_t grid, long long wait_limit, cudaStream_t st) {
  const int rc = kvcu_configure_once(
      reinterpret_cast<const void*>(k_mass_tc<NC>),
      [](const void*) {
        return kvcu_check_cuda(
            cudaFuncSetAttribute(k_mass_tc<NC>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Map<NC>::ALLOC),
            "cudaFuncSetAttribute(mass)");
      },
      nullptr);
  if (rc) return rc;
  TcMass t = {a, 128, wait_limit};
  while (pool->block_size % t.box_rows) t.box_rows /= 2;  // block sizes are multiples of 16
  CUtensorMap wide, tail;
  const int rm = make_maps(pool, t.box_rows, &wide, &tail);
  if (rm) return rm;
  return kvcu_check_cuda(
      kvcu_launch_pdl(k_mass_tc<NC>, dim3(grid), dim3(TC_THREADS), Map<NC>::ALLOC, st, wide, tail, t),
      "attention mass launch");
}

int launch_mass(const MassArgs& a, uint32_t grid, cudaStream_t st) {
  const int rc = kvcu_configure_once(
      reinterpret_cast<const void*>(k_mass),
      [](const void*) {
        return kvcu_check_cuda(cudaFuncSetAttribute(k_mass, cudaFuncAttributeMaxDynamicSharedMemorySize, CC_SMEM),
                               "cudaFuncSetAttribute(mass)");
      },
      nullptr);
  if (rc) return rc;
  k_mass<<<grid, NT, CC_SMEM, st>>>(a);
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
  if (!pool->quantized) return launch_mass(a, grid, st);
  if (pool->rows() > 0x7FFFFFFFull) {
    kvcu_set_error("kvcu_attn_mass: %llu rows, TMA coordinates reach 2^31 - 1", (unsigned long long)pool->rows());
    return KVCU_ERR_UNSUPPORTED;
  }
  const long long limit = ws->wait_limit ? (long long)ws->wait_limit : (1ll << 31);
  // columns of a chunk: a chunk costs its columns' scaling and exponentials and,
  // whatever their number, the rows' unpacking (as much as about 30 columns)
  const uint32_t cols = n_q * n_heads;
  auto cost = [&](uint32_t nc) { return (uint64_t)((cols + nc - 1) / nc) * (nc + 30); };
  if (cost(8) <= cost(16) && cost(8) <= cost(20) && cost(8) <= cost(24)) return launch_mass_tc<8>(pool, a, grid, limit, st);
  if (cost(16) <= cost(20) && cost(16) <= cost(24)) return launch_mass_tc<16>(pool, a, grid, limit, st);
  if (cost(20) <= cost(24)) return launch_mass_tc<20>(pool, a, grid, limit, st);
  return launch_mass_tc<24>(pool, a, grid, limit, st);
}
