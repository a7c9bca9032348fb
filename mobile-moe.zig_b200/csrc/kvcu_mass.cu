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
// A Q8_0 row is 18 blocks of 32 int8 values with a scale each, and int8 values are
// exact in f16: per block, mma.sync m16n8k16 (f16, f32 accumulation) of 16 rows'
// values against 8 columns of q, then one f32 FMA with the row's block scale.  q is
// brought to [2^13, 2^14) by a power of two per column and slice and split into two
// f16 parts (22 bits), so the scores have f32's accuracy at two MMAs per product;
// rounding row or query to one f16 would cost 2e-3 of the weight.  tcgen05 does
// not help here: its accumulators live in TMEM, and the 18 block sums of every
// (row, column) would have to be read back from there before they can be scaled,
// where mma.sync leaves them in the registers that scale them.
//
// One CTA per SM, 12 compute warps and a producer.  A compute warp has 3 of the 18
// blocks (its q parts stay in registers for a whole item) and 32 of a tile's 64
// rows; the 6 slices' partial scores meet in shared memory, where 256 threads add
// them, take the exponentials and sum over the columns while the other warps are
// already in the next tile.  The producer streams rows in with bulk copies (576 B,
// padded to 608 B in shared memory: the 8-byte fragment loads then touch every bank
// once) through three stages, and runs ahead with the items, lengths and block
// tables.  More than 24 columns (several queries, more heads) go in chunks: the
// item's rows are streamed again, from L2, for each.
constexpr int TC_WARPS = 12, TC_THREADS = (TC_WARPS + 4) * 32, SLICES = 6, BPS = 3;  // blocks per slice
// Registers: launched with 128 a thread; the producer's four warps (three idle) give
// theirs to the compute warps, whose q parts take 72.
constexpr int TC_LAUNCH_REGS = 128, TC_PRODUCER_REGS = 56, TC_COMPUTE_REGS = 152;
static_assert(TC_WARPS * TC_COMPUTE_REGS + 4 * TC_PRODUCER_REGS <= (TC_WARPS + 4) * TC_LAUNCH_REGS,
              "register split exceeds the launch allocation");
constexpr int TCT = 64, ROW = 608, STAGES = 3;
constexpr uint32_t STAGE_BYTES = TCT * ROW + TCT * NBLK * 2;
constexpr uint32_t GROUP = 16, GROUP_TX = GROUP * (W + NBLK * 2);

struct Desc {
  uint32_t b, p0, end, c0, old, len, ok, live;  // ok: bits of the 16-row groups; live: 0 ends the CTA's work
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// Wait for phase `parity`, at most `limit` clocks.
__device__ __forceinline__ bool bounded_wait(uint32_t bar, uint32_t parity, long long limit) {
  if (kvtc::mbar_try(bar, parity)) return true;
  const long long t0 = clock64();
  while (!kvtc::mbar_try(bar, parity))
    if (clock64() - t0 > limit) return false;
  return true;
}

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four int8 values as two f16 pairs, exact: a biased byte u in the low mantissa of
// 1024 is 1024 + u; minus 1152 leaves u - 128.
__device__ __forceinline__ void int8_to_f16(uint32_t w, uint32_t* lo, uint32_t* hi) {
  const uint32_t u = w ^ 0x80808080u;
  const __half2 bias = __half2half2(__ushort_as_half(0x6480));
  const uint32_t x = __byte_perm(u, 0x64646464u, 0x4140), y = __byte_perm(u, 0x64646464u, 0x4342);
  const __half2 r0 = __hsub2(*reinterpret_cast<const __half2*>(&x), bias);
  const __half2 r1 = __hsub2(*reinterpret_cast<const __half2*>(&y), bias);
  *lo = *reinterpret_cast<const uint32_t*>(&r0);
  *hi = *reinterpret_cast<const uint32_t*>(&r1);
}

__device__ __forceinline__ uint32_t pack_half(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <int NTL>  // column tiles of 8 in a chunk
struct TcLayout {
  static constexpr int COLS = NTL * 8;
  static constexpr int LD = NTL == 2 ? 24 : COLS;  // floats of a row of partial scores (a stride of 16 would conflict)
  static constexpr uint32_t RED = STAGES * STAGE_BYTES;
  static constexpr uint32_t RED_BYTES = SLICES * TCT * LD * 4;
  static constexpr uint32_t TOTAL = RED + 2 * RED_BYTES;
};

template <int NTL>
__global__ void __launch_bounds__(TC_THREADS, 1) k_mass_tc(MassArgs a, long long wait_limit) {
  using L = TcLayout<NTL>;
  extern __shared__ __align__(128) char sm[];
  __shared__ __align__(8) uint64_t bars[2 * STAGES];
  __shared__ Desc descs[STAGES];
  __shared__ uint32_t s_abort[2];
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  const uint32_t full = kvtc::smem_u32(bars), empty = full + 8 * STAGES, base = kvtc::smem_u32(sm);
  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) {
      kvtc::mbar_init(full + 8 * i, 1);
      kvtc::mbar_init(empty + 8 * i, TC_WARPS);
    }
    s_abort[0] = s_abort[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  const uint32_t cols = a.n_q * a.n_heads;

  if (warp >= TC_WARPS) {
    // ---------------------------------------------------------------- producer
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(TC_PRODUCER_REGS));
    if (warp > TC_WARPS) return;
    const uint32_t n_items = a.meta[0], n_ranges = a.meta[1];
    if (blockIdx.x == 0 && lane == 0 && n_ranges > gridDim.x) atomicOr(a.status, KVCU_STATUS_BAD_PLAN);
    const uint32_t it0 = blockIdx.x < n_ranges ? min(a.ranges[blockIdx.x], n_items) : n_items;
    const uint32_t it1 = blockIdx.x < n_ranges ? min(a.ranges[blockIdx.x + 1], n_items) : n_items;
    uint32_t g = 0;  // stage uses so far
    bool ok = true;
    for (uint32_t base_it = it0; ok && base_it < it1; base_it += 32) {
      // 32 items' entries at once: one chain of dependent loads for all
      kvcu_item mine = {0, 0, 0, 0};
      Entry me = {0, 0, 0, 0, 0};
      if (base_it + lane < it1) {
        mine = a.items[base_it + lane];
        me = entry_of(a, mine.b, true);
      }
      const uint32_t here = min(32u, it1 - base_it);
      for (uint32_t k = 0; ok && k < here; ++k) {
        const uint32_t b = __shfl_sync(0xffffffffu, mine.b, k), start = __shfl_sync(0xffffffffu, mine.start, k);
        const uint32_t len = __shfl_sync(0xffffffffu, me.len, k), old = __shfl_sync(0xffffffffu, me.old, k);
        const uint32_t t0 = __shfl_sync(0xffffffffu, me.t0, k);
        const uint32_t end = min(__shfl_sync(0xffffffffu, mine.end, k), len);
        const uint32_t grp = lane >> 3;  // this lane's two rows, 2 * lane and 2 * lane + 1, lie in one 16-row group
        auto block_at = [&](uint32_t p0) -> uint32_t {
          const uint32_t p = p0 + grp * GROUP;
          return p < end ? a.tables[t0 + p / a.block_size] : 0xFFFFFFFFu;
        };
        for (uint32_t c0 = 0; ok && c0 < cols; c0 += L::COLS) {
          uint32_t next = block_at(start);
          for (uint32_t p0 = start; p0 < end; p0 += TCT, ++g) {
            const uint32_t blk = next, s = g % STAGES;
            next = block_at(p0 + TCT < end ? p0 + TCT : end);
            const bool in = p0 + grp * GROUP < end, good = in && blk < a.num_blocks;
            if (in && !good && c0 == 0 && (lane & 7u) == 0) atomicOr(a.status, KVCU_STATUS_BAD_BLOCK);
            const uint32_t votes = __ballot_sync(0xffffffffu, good && (lane & 7u) == 0);
            ok = bounded_wait(empty + 8 * s, ((g / STAGES) & 1u) ^ 1u, wait_limit);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const uint32_t mask = (votes & 1u) | (votes >> 7 & 2u) | (votes >> 14 & 4u) | (votes >> 21 & 8u);
            if (lane == 0) {
              descs[s] = {b, p0, end, c0, old, len, mask, 1u};
              kvtc::mbar_arrive_tx(full + 8 * s, __popc(mask) * GROUP_TX);
            }
            __syncwarp();
            if (good) {
              const uint64_t row = ((uint64_t)a.layer * a.num_blocks + blk) * a.block_size + (p0 + grp * GROUP) % a.block_size;
              const uint32_t st = base + s * STAGE_BYTES;
              const uint32_t r = 2 * lane;
              const int8_t* src = a.qs + (row + (r & 15u)) * W;
              bulk_load(st + r * ROW, src, W, full + 8 * s);
              bulk_load(st + (r + 1) * ROW, src + W, W, full + 8 * s);
              if ((lane & 7u) == 0)
                bulk_load(st + TCT * ROW + grp * GROUP * NBLK * 2, a.sc + row * NBLK, GROUP * NBLK * 2, full + 8 * s);
            }
          }
        }
      }
    }
    const uint32_t s = g % STAGES;
    if (ok) ok = __all_sync(0xffffffffu, bounded_wait(empty + 8 * s, ((g / STAGES) & 1u) ^ 1u, wait_limit));
    if (ok) {
      if (lane == 0) {
        descs[s].live = 0;
        kvtc::mbar_arrive(full + 8 * s);
      }
    } else {
      if (lane == 0) atomicOr(a.status, KVCU_STATUS_TIMEOUT);
      // the copies in flight must land before the CTA leaves
      for (uint32_t k = g > STAGES ? g - STAGES : 0; k < g; ++k)
        bounded_wait(full + 8 * (k % STAGES), (k / STAGES) & 1u, wait_limit);
    }
    return;
  }

  // ------------------------------------------------------------------ compute
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(TC_COMPUTE_REGS));
  const uint32_t slice = warp % SLICES, half = warp / SLICES;
  const uint32_t gr = lane >> 2, t = lane & 3u;
  uint32_t bh[BPS][2][NTL][2], bl[BPS][2][NTL][2];  // q parts: [block][k step][column tile][pair]
  float back[NTL][2];                               // 2^-e of the columns this lane's sums belong to
  // the adding threads: row tid / 4 of a tile, 2 * NTL columns
  constexpr int CPT = 2 * NTL;
  const uint32_t er = tid >> 2, ec = (tid & 3u) * CPT;
  const bool adds = tid < 4 * TCT;
  float lse[CPT];
  uint32_t lim[CPT];  // positions below it count
  float before = 0.f;
  Desc prev = {};
  uint32_t have_b = 0xFFFFFFFFu, have_c = 0;
  for (uint32_t g = 0;; ++g) {
    const uint32_t s = g % STAGES;
    if (!bounded_wait(full + 8 * s, (g / STAGES) & 1u, wait_limit)) *(volatile uint32_t*)&s_abort[g & 1u] = 1u;
    const Desc d = descs[s];
    asm volatile("bar.sync 1, %0;" ::"n"(TC_WARPS * 32) : "memory");
    // every partial score of tile g - 1 is in shared memory
    const bool stop = *(volatile uint32_t*)&s_abort[g & 1u] != 0;
    if (adds && prev.live) {
      const float* red = reinterpret_cast<const float*>(sm + L::RED + ((g - 1) & 1u) * L::RED_BYTES);
      const uint32_t p = prev.p0 + er;
      float sc[CPT];
#pragma unroll
      for (int j = 0; j < CPT; ++j) sc[j] = 0.f;
#pragma unroll
      for (int k = 0; k < SLICES; ++k)
#pragma unroll
        for (int j = 0; j < CPT; j += 2) {
          const float2 v = *reinterpret_cast<const float2*>(red + (k * TCT + er) * L::LD + ec + j);
          sc[j] += v.x;
          sc[j + 1] += v.y;
        }
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < CPT; ++j)
        if (p < lim[j]) sum += expf(fmaf(sc[j], a.scale, -lse[j]));
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      if ((tid & 3u) == 0 && p < prev.end && (prev.ok >> (er >> 4) & 1u)) {
        float* m = a.mass + (uint64_t)prev.b * a.mass_stride + p;
        if (prev.c0) *m = before + sum;
        else *m = p < prev.old ? fmaf(a.decay, before, sum) : sum;
      }
    }
    if (stop || !d.live) {
      if (stop && tid == 0) atomicOr(a.status, KVCU_STATUS_TIMEOUT);
      break;
    }
    if (d.b != have_b || d.c0 != have_c) {
      have_b = d.b;
      have_c = d.c0;
      const float* qb = a.q + (uint64_t)d.b * cols * W;
      float inv[NTL];
#pragma unroll
      for (int nt = 0; nt < NTL; ++nt) {
        const uint32_t c = d.c0 + nt * 8 + gr;
        float x[BPS][8];
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < BPS; ++i) {
          float4 u = make_float4(0.f, 0.f, 0.f, 0.f), v = u;
          if (c < cols) {
            const float4* src = reinterpret_cast<const float4*>(qb + (uint64_t)c * W + (slice * BPS + i) * 32 + t * 8);
            u = src[0];
            v = src[1];
          }
          x[i][0] = u.x, x[i][1] = u.y, x[i][2] = u.z, x[i][3] = u.w;
          x[i][4] = v.x, x[i][5] = v.y, x[i][6] = v.z, x[i][7] = v.w;
#pragma unroll
          for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(x[i][j]));
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // 2^(13 - exponent of amax); 1 for a column of zeros or with an infinity
        const uint32_t eb = __float_as_uint(amax) >> 23;
        const uint32_t f = amax == 0.f || eb == 255u ? 127u : min(max(267 - (int)eb, 1), 253);
        const float up = __uint_as_float(f << 23);
        inv[nt] = __uint_as_float((254u - f) << 23);
#pragma unroll
        for (int i = 0; i < BPS; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {  // elements 2j, 2j + 1: k step j / 2, pair j % 2
            const float y0 = x[i][2 * j] * up, y1 = x[i][2 * j + 1] * up;
            const uint32_t h = pack_half(y0, y1);
            const float2 hf = __half22float2(*reinterpret_cast<const __half2*>(&h));
            bh[i][j >> 1][nt][j & 1] = h;
            bl[i][j >> 1][nt][j & 1] = pack_half(y0 - hf.x, y1 - hf.y);
          }
        back[nt][0] = __shfl_sync(0xffffffffu, inv[nt], t * 8);
        back[nt][1] = __shfl_sync(0xffffffffu, inv[nt], t * 8 + 4);
      }
      if (adds) {
#pragma unroll
        for (int j = 0; j < CPT; ++j) {
          const uint32_t c = d.c0 + ec + j;
          lse[j] = c < cols ? a.lse[(uint64_t)d.b * cols + c] : -INFINITY;
          const uint32_t behind = a.n_q - 1 - c / a.n_heads;
          // a column past the last, or a query that saw nothing, has no positions
          lim[j] = lse[j] == -INFINITY || d.len <= behind ? 0u : d.len - behind;
        }
      }
    }
    if (adds && (tid & 3u) == 0) {
      const uint32_t p = d.p0 + er;
      before = p < d.end && (d.c0 || p < d.old) ? a.mass[(uint64_t)d.b * a.mass_stride + p] : 0.f;
    }
    const char* st = sm + s * STAGE_BYTES;
    float* red = reinterpret_cast<float*>(sm + L::RED + (g & 1u) * L::RED_BYTES);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const uint32_t r0 = half * 32 + m * 16 + gr, r1 = r0 + 8;
      float tot[NTL][4];
#pragma unroll
      for (int nt = 0; nt < NTL; ++nt) tot[nt][0] = tot[nt][1] = tot[nt][2] = tot[nt][3] = 0.f;
#pragma unroll
      for (int i = 0; i < BPS; ++i) {
        const uint32_t blk = slice * BPS + i;
        const uint2 w0 = *reinterpret_cast<const uint2*>(st + r0 * ROW + blk * 32 + t * 8);
        const uint2 w1 = *reinterpret_cast<const uint2*>(st + r1 * ROW + blk * 32 + t * 8);
        const __half* sc = reinterpret_cast<const __half*>(st + TCT * ROW);
        const float d0 = __half2float(sc[r0 * NBLK + blk]), d1 = __half2float(sc[r1 * NBLK + blk]);
        uint32_t af[2][4];
        int8_to_f16(w0.x, &af[0][0], &af[0][2]);
        int8_to_f16(w1.x, &af[0][1], &af[0][3]);
        int8_to_f16(w0.y, &af[1][0], &af[1][2]);
        int8_to_f16(w1.y, &af[1][1], &af[1][3]);
#pragma unroll
        for (int nt = 0; nt < NTL; ++nt) {
          float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) {
            mma16816(acc, af[ks], bl[i][ks][nt][0], bl[i][ks][nt][1]);
            mma16816(acc, af[ks], bh[i][ks][nt][0], bh[i][ks][nt][1]);
          }
          tot[nt][0] = fmaf(acc[0], d0, tot[nt][0]);
          tot[nt][1] = fmaf(acc[1], d0, tot[nt][1]);
          tot[nt][2] = fmaf(acc[2], d1, tot[nt][2]);
          tot[nt][3] = fmaf(acc[3], d1, tot[nt][3]);
        }
      }
#pragma unroll
      for (int nt = 0; nt < NTL; ++nt) {
        float* o = red + (slice * TCT + r0) * L::LD + nt * 8 + t * 2;
        *reinterpret_cast<float2*>(o) = make_float2(tot[nt][0] * back[nt][0], tot[nt][1] * back[nt][1]);
        *reinterpret_cast<float2*>(o + 8 * L::LD) = make_float2(tot[nt][2] * back[nt][0], tot[nt][3] * back[nt][1]);
      }
    }
    __syncwarp();
    if (lane == 0) kvtc::mbar_arrive(empty + 8 * s);
    prev = d;
  }
}

template <int NTL>
int launch_mass_tc(const MassArgs& a, uint32_t grid, long long wait_limit, cudaStream_t st) {
  const int rc = kvcu_configure_once(
      reinterpret_cast<const void*>(k_mass_tc<NTL>),
      [](const void*) {
        // the register split assumes exactly this many at launch: with fewer, setmaxnreg.inc would wait for ever
        cudaFuncAttributes fa;
        KVCU_CUDA(cudaFuncGetAttributes(&fa, k_mass_tc<NTL>));
        if (fa.numRegs != TC_LAUNCH_REGS) {
          kvcu_set_error("attn_mass: built with %d registers per thread, the register split needs %d", fa.numRegs,
                         TC_LAUNCH_REGS);
          return KVCU_ERR_UNSUPPORTED;
        }
        return kvcu_check_cuda(
            cudaFuncSetAttribute(k_mass_tc<NTL>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcLayout<NTL>::TOTAL),
            "cudaFuncSetAttribute(mass)");
      },
      nullptr);
  if (rc) return rc;
  k_mass_tc<NTL><<<grid, TC_THREADS, TcLayout<NTL>::TOTAL, st>>>(a, wait_limit);
  return kvcu_check_cuda(cudaGetLastError(), "attention mass launch");
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
  const long long limit = ws->wait_limit ? (long long)ws->wait_limit : (1ll << 31);
  // column tiles per chunk: a chunk costs its tiles and, whatever their number, the
  // rows' unpacking (about three half tiles)
  const uint32_t cols = n_q * n_heads;
  auto cost = [&](uint32_t nt) { return ((cols + 8 * nt - 1) / (8 * nt)) * (2 * nt + 3); };
  const uint32_t nt = cost(1) <= cost(2) && cost(1) <= cost(3) ? 1u : cost(2) <= cost(3) ? 2u : 3u;
  if (nt == 1) return launch_mass_tc<1>(a, grid, limit, st);
  if (nt == 2) return launch_mass_tc<2>(a, grid, limit, st);
  return launch_mass_tc<3>(a, grid, limit, st);
}
