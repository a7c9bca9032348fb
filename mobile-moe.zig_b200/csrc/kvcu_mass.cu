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
#include "kvcu_mass.cuh"

using namespace kvmass;

namespace {

// ------------------------------------------------------------------ tensor cores
// The scores run on tcgen05 kind::f16 with M = 128 rows, in f32's accuracy:
//   Q8_0 rows are 18 blocks of 32 int8 values with a scale each; int8 values are exact
//     in f16, so D = sum of value * q per block and column, and one f32 FMA with the
//     row's block scale adds D to the row's score;
//   f32 rows are treated as such blocks, with the power of two that brings the block
//     to [2^13, 2^14) for the scale and the values split into two f16 parts (22 bits);
//   q's columns are scaled and split the same way, one power of two to a column.
// The parts' products (two per Q8_0 value, three per f32 value; low times low stays
// below 2^-22) accumulate into one D.  Rounding row or query to one f16 would cost
// 2e-3 of the weight.
//
// A thread owns one of 128 rows: it unpacks the row's blocks to f16 straight into
// TMEM (the MMA's A operand), reads the block sums back from its own TMEM lane and
// keeps the row's scores in registers.  A tile is 256 rows, two pairs of warpgroups
// with 128 rows each; in a pair each warpgroup has half of the blocks.  In a step a
// warpgroup unpacks one block, hands it to its pair's issuer and scales the sums of
// the step before, so unpacking, MMAs and scaling overlap; a tile is finished while
// the next one's first MMAs run: the pair's warpgroups swap halves of the columns
// through shared memory, take the exponentials of their half, and the first adds the
// two sums to the mass.
//
//   warps 0-15   the four warpgroups; before a chunk they also prepare its q parts
//   warp 16      producer: TMA boxes of 128 B x <= 128 rows (a "unit": of each of a
//                pair's rows four Q8_0 blocks, the fifth unit two; or one f32 block)
//                through rings, and each tile's description and scales
//   warps 17-18  issue the MMAs, one for each pair
// More columns (queries x heads) than an instance has go in chunks: the item's rows
// are streamed again for each, from L2 where all items' rows fit there, else from memory
// (Q8_0 rows only below 48 columns: kvcu_mass_wide.cu).  192 sequences of 2.0M rows in all:
// 336 us with 20 heads, 608 us with 32 (two chunks); f32, 16 sequences of 8,000 rows: 77 us
// for one query of 20 heads, 389 us for eight (seven chunks).
// Bound: waits.  A Q8_0 row takes an SM 46 clocks, where the loads alone take 28 (6.2 TB/s)
// and issuing its 98 warp instructions 24.5: no pipe is saturated (issue 48%, memory 35%,
// tensor 18%), and each of a warpgroup's nine steps waits for its TMEM stores, for the MMAs
// of the step before and for their sums.  Measured with 20 heads: 64 sequences to 32k rows
// 68-69 us (3.0 TB/s), 192 to 65k 392 us (3.4 TB/s), one of 777 rows 10.8 us; f32, 16
// sequences to 8k 43 us, 64 of 8,192 rows 6.0-6.2 TB/s.
constexpr int COMPUTE = 16, PRODUCER = 16, ISSUER = 17;  // warps; two issuers
constexpr int TC_THREADS = (COMPUTE + 4) * 32;
// Registers: launched with 96 a thread; the last warpgroup gives to the four others.
constexpr int LAUNCH_REGS = 96, SERVICE_REGS = 64, COMPUTE_REGS = 104;
static_assert(COMPUTE * COMPUTE_REGS + 4 * SERVICE_REGS <= (COMPUTE + 4) * LAUNCH_REGS,
              "register split exceeds the launch allocation");
constexpr uint32_t HALF = 128, TILE = 2 * HALF;  // rows of a pair, of a tile
constexpr uint32_t UNIT_BYTES = HALF * 128;
constexpr int STEPS = 9;                         // blocks of a warpgroup
constexpr long long DRAIN_LIMIT = 1ll << 31;     // clocks a role that gives up waits for its own copies and MMAs
constexpr uint32_t TM_WG = 128, TM_COLS = 512;   // TMEM columns of a warpgroup, allocated

struct Tile {
  uint32_t b, p0, end, c0, old, ok;  // ok: bits of the boxes that were loaded
  uint32_t chunk;                    // counts the chunks of the CTA
  uint32_t flags;                    // TILE_*
  uint32_t len;
};
constexpr uint32_t TILE_LIVE = 1, TILE_FIRST = 2;  // FIRST: of its chunk

template <bool Q8, int NC>  // NC: columns of a chunk
struct Map {
  static constexpr int HC = NC / 2;
  static constexpr int RB = (NC + 7) / 8 * 8;          // rows of a q part
  static constexpr uint32_t N = (RB + 15) / 16 * 16;   // MMA columns: the surplus reads rows of the next part
  static constexpr uint32_t REGION = 2 * RB * 128;     // 64 elements of the hi rows, then of the lo rows
  static constexpr uint32_t UNITS = Q8 ? 5 : 18;       // of a pair's rows
  // Units go through rings of their own for each group of warps that reads them: a
  // pair's (Q8_0: both warpgroups read every unit) or a warpgroup's (f32: one reads a
  // block).  A barrier's parity tells only neighbouring phases apart, so whoever waits
  // on a slot has to see every one of its phases.
  static constexpr int RINGS = Q8 ? 2 : 4, DEPTH = Q8 ? 4 : 2, SLOTS = RINGS * DEPTH;
  static constexpr uint32_t A_COLS = Q8 ? 16 : 32;     // TMEM columns of an unpacked block: its parts
  static constexpr uint32_t TM_D = 2 * A_COLS;         // block sums, two buffers of N columns
  static constexpr uint32_t RING = (W / 64) * REGION;  // 1024-aligned, as every region and unit
  static constexpr uint32_t SC = RING + SLOTS * UNIT_BYTES;
  static constexpr uint32_t X = SC + (Q8 ? TILE * NBLK * 2 : 0);  // [pair][warpgroup][HC][128] scores given away
  static constexpr uint32_t S = X + 2 * 2 * HC * HALF * 4;            // [pair][2][128] the second warpgroup's sums
  static constexpr uint32_t COL = S + 2 * 2 * HALF * 4;               // [RB] (scale, -lse), then limits
  static constexpr uint32_t TILES = COL + RB * 12;
  static constexpr uint32_t BARS = (TILES + sizeof(Tile) + 7) / 8 * 8;
  // barriers
  static constexpr int B_TF = 0;            // tile description and scales: full
  static constexpr int B_TE = B_TF + 1;     //   read
  static constexpr int B_UF = B_TE + 1;     // unit: full
  static constexpr int B_UE = B_UF + SLOTS;  //   read
  static constexpr int B_QF = B_UE + SLOTS;  // q parts of a chunk: full (two barriers in turn)
  static constexpr int B_QE = B_QF + 2;     //   done with
  static constexpr int B_AF = B_QE + 1;     // unpacked block in TMEM, per warpgroup and buffer
  static constexpr int B_DF = B_AF + 8;     // block sums ready, per warpgroup and buffer
  static constexpr int B_X = B_DF + 8;      // scores swapped, per pair
  static constexpr int B_XE = B_X + 2;      //   read
  static constexpr int B_FINAL = B_XE + 2;  // all MMAs of an issuer retired
  static constexpr int NUM_BARS = B_FINAL + 2;
  static constexpr uint32_t MISC = BARS + NUM_BARS * 8;  // TMEM base, abort flag
  static constexpr uint32_t ALLOC = MISC + 16 + 1024;
  static_assert(ALLOC <= 232448, "shared memory budget");
  static_assert(REGION % 1024 == 0 && NC % 4 == 0 && TM_D + 2 * N <= TM_WG, "layout");
};

struct TcMass {
  MassArgs m;
  uint32_t box_rows;
  long long wait_limit;
  uint32_t withhold_plus1;  // test hook: 0, or 1 + the tile of each CTA whose first units are withheld
};

// The q parts of (entry b, columns from c0) and each column's scale, -lse and limit,
// rows dealt to the compute warps.
template <bool Q8, int NC>
__device__ __forceinline__ void fill_q(const MassArgs& a, char* sm, uint32_t warp, uint32_t lane, uint32_t b, uint32_t c0,
                                       uint32_t len, uint32_t cols) {
  using M = Map<Q8, NC>;
  float* col = reinterpret_cast<float*>(sm + M::COL);
#pragma unroll 1
  for (uint32_t r = warp; r < (uint32_t)M::RB; r += COMPUTE) {
    const uint32_t c = c0 + r;
    const bool live = r < NC && c < cols;
    const float4* src = reinterpret_cast<const float4*>(a.q + ((uint64_t)b * cols + c) * W);
    float4 x[5];
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 5; ++i) {
      const uint32_t f = lane + 32 * i;  // elements 4f .. 4f + 3
      x[i] = live && f < W / 4 ? src[f] : make_float4(0.f, 0.f, 0.f, 0.f);
      amax = fmaxf(fmaxf(fmaxf(amax, fabsf(x[i].x)), fmaxf(fabsf(x[i].y), fabsf(x[i].z))), fabsf(x[i].w));
    }
    // magnitudes order as integers
    const uint32_t f2 = scale_field(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));
    const float up = __uint_as_float(f2 << 23);
#pragma unroll
    for (int i = 0; i < 5; ++i) {
      const uint32_t f = lane + 32 * i;
      if (f >= W / 4) continue;
      uint2 hi, lo;
      split(x[i].x * up, x[i].y * up, &hi.x, &lo.x);
      split(x[i].z * up, x[i].w * up, &hi.y, &lo.y);
      char* at = sm + (f / 16) * M::REGION;
      *reinterpret_cast<uint2*>(at + kvtc::sw128_off(r, (f % 16) * 8)) = hi;
      *reinterpret_cast<uint2*>(at + kvtc::sw128_off(M::RB + r, (f % 16) * 8)) = lo;
    }
    if (lane == 0) {
      const float l = live ? a.lse[(uint64_t)b * cols + c] : -INFINITY;
      const uint32_t behind = a.n_q - 1 - c / a.n_heads;  // positions behind the column's query
      // exp(s - lse) = 2^(s log2 e - lse log2 e)
      constexpr double LOG2E = 1.4426950408889634;
      col[2 * r] = (float)(a.scale * LOG2E) * __uint_as_float((254u - f2) << 23);
      col[2 * r + 1] = (float)(-l * LOG2E);
      // a column past the last, or a query that saw nothing, has no positions
      reinterpret_cast<uint32_t*>(col)[2 * M::RB + r] = l == -INFINITY || len <= behind ? 0u : len - behind;
    }
  }
}

template <bool Q8, int NC>
__global__ void __launch_bounds__(TC_THREADS, 1)
    k_mass(const __grid_constant__ CUtensorMap wide, const __grid_constant__ CUtensorMap tail, const TcMass t) {
  using M = Map<Q8, NC>;
  const MassArgs& a = t.m;
  extern __shared__ char raw[];
  char* sm = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  const uint32_t base = kvtc::smem_u32(sm);
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(sm + M::MISC + 4);
  auto bar = [&](int i) { return base + M::BARS + 8u * (uint32_t)i; };
  auto wait = [&](int i, uint32_t parity) { return wait_bar(bar(i), parity, abort_flag, t.wait_limit); };
  if (tid == 0) {
    auto init = [&](int first, int n, uint32_t count) {
      for (int i = 0; i < n; ++i) kvtc::mbar_init(bar(first + i), count);
    };
    init(M::B_TF, 1, 1);
    init(M::B_TE, 1, COMPUTE + 2);
    init(M::B_UF, M::SLOTS, 1);
    init(M::B_UE, M::SLOTS, Q8 ? 8 : 4);
    init(M::B_QF, 2, COMPUTE);
    init(M::B_QE, 1, COMPUTE);
    init(M::B_AF, 8, 4);
    init(M::B_DF, 8, 1);
    init(M::B_X, 2, 8);
    init(M::B_XE, 2, 8);
    init(M::B_FINAL, 2, 1);
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
  Tile* tile = reinterpret_cast<Tile*>(sm + M::TILES);

  if (warp >= COMPUTE) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(SERVICE_REGS));
    if (warp == PRODUCER) {
      // -------------------------------------------------------------- producer
      const uint32_t n_items = a.meta[0], n_ranges = a.meta[1];
      if (blockIdx.x == 0 && lane == 0 && n_ranges > gridDim.x) atomicOr(a.status, KVCU_STATUS_BAD_PLAN);
      const uint32_t it0 = blockIdx.x < n_ranges ? min(a.ranges[blockIdx.x], n_items) : n_items;
      const uint32_t it1 = blockIdx.x < n_ranges ? min(a.ranges[blockIdx.x + 1], n_items) : n_items;
      const uint32_t boxes = TILE / t.box_rows, pair = lane * t.box_rows / HALF;  // this lane's box
      uint32_t ti = 0, chunk = 0, filled[2] = {0, 0};  // filled: units into a ring (of the pair; f32: both alike, in turn)
      uint32_t sent = 0;  // lane k: units sent through slot k
      bool ok = true;
      kvcu_item mine = {0, 0, 0, 0};
      Entry me = {0, 0, 0, 0, 0};
      for (uint32_t it = it0; ok && it < it1; ++it) {
        const uint32_t k = (it - it0) & 31u;
        if (k == 0 && it + lane < it1) {  // 32 items at a time: their chains of dependent loads run side by side
          mine = a.items[it + lane];
          me = entry_of(a, mine.b, true);
        }
        const uint32_t b = __shfl_sync(0xffffffffu, mine.b, k), start = __shfl_sync(0xffffffffu, mine.start, k);
        const uint32_t len = __shfl_sync(0xffffffffu, me.len, k), old = __shfl_sync(0xffffffffu, me.old, k);
        const uint32_t t0 = __shfl_sync(0xffffffffu, me.t0, k);
        const uint32_t end = min(__shfl_sync(0xffffffffu, mine.end, k), len);
        auto block_at = [&](uint32_t p0) -> uint32_t {
          const uint32_t p = p0 + lane * t.box_rows;
          return lane < boxes && p < end ? a.tables[t0 + p / a.block_size] : 0xFFFFFFFFu;
        };
        for (uint32_t c0 = 0; ok && c0 < cols && start < end; c0 += NC, ++chunk) {
          uint32_t next = block_at(start);
          for (uint32_t p0 = start; ok && p0 < end; p0 += TILE) {
            const uint32_t blk = next, p = p0 + lane * t.box_rows;
            next = block_at(p0 + TILE < end ? p0 + TILE : end);
            const bool in = lane < boxes && p < end, good = in && blk < a.num_blocks;
            if (in && !good && c0 == 0) atomicOr(a.status, KVCU_STATUS_BAD_BLOCK);
            const uint32_t votes = __ballot_sync(0xffffffffu, good);
            const uint32_t of[2] = {votes & ((1u << (HALF / t.box_rows)) - 1u), votes >> (HALF / t.box_rows)};
            const uint64_t row = ((uint64_t)a.layer * a.num_blocks + blk) * a.block_size + p % a.block_size;
            if (!(ok = wait(M::B_TE, (ti & 1u) ^ 1u))) break;
            if (lane == 0) {
              *tile = {b, p0, end, c0, old, votes, chunk, TILE_LIVE | (p0 == start ? TILE_FIRST : 0u), len};
              kvtc::mbar_arrive_tx(bar(M::B_TF), Q8 ? __popc(votes) * t.box_rows * NBLK * 2 : 0u);
            }
            ++ti;
            __syncwarp();
            if (Q8 && good)
              bulk_load(base + M::SC + lane * t.box_rows * NBLK * 2, a.sc + row * NBLK, t.box_rows * NBLK * 2,
                        bar(M::B_TF));
            const uint32_t pairs = p0 + HALF < end ? 2u : 1u;
            for (uint32_t u = 0; ok && u < M::UNITS; ++u)
              for (uint32_t pr = 0; pr < pairs; ++pr) {
                // f32: blocks alternate between the pair's two rings, STEPS to each in a tile
                const uint32_t nth = Q8 ? filled[pr] + u : filled[pr] + u / 2, ring = Q8 ? pr : 2 * pr + (u & 1u);
                const uint32_t slot = ring * M::DEPTH + nth % M::DEPTH, width = Q8 && u == 4 ? 64u : 128u;
                if (!(ok = wait(M::B_UE + slot, ((nth / M::DEPTH) & 1u) ^ 1u))) break;
                if (u == 0 && ti == t.withhold_plus1) continue;  // no copy and no arrival: its readers' waits run out
                if (lane == 0) kvtc::mbar_arrive_tx(bar(M::B_UF + slot), __popc(of[pr]) * t.box_rows * width);
                __syncwarp();
                if (good && pair == pr) {
                  const uint32_t dst = base + M::RING + slot * UNIT_BYTES + (lane * t.box_rows - pr * HALF) * width;
                  const bool second = u >= (Q8 ? 4u : 16u);
                  const int x = Q8 ? (int)(u * 128) : (int)((second ? u - 16 : u) * 32);
                  tma_2d(dst, second ? &tail : &wide, x, (int)row, bar(M::B_UF + slot));
                }
                sent += lane == slot;
              }
            for (uint32_t pr = 0; pr < pairs; ++pr) filled[pr] += Q8 ? M::UNITS : STEPS;
          }
        }
      }
      if (ok && (ok = wait(M::B_TE, (ti & 1u) ^ 1u)) && lane == 0) {
        tile->flags = 0;
        kvtc::mbar_arrive(bar(M::B_TF));
      }
      // The copies in flight must land before the CTA leaves, also where only their readers have given up: the
      // last of each slot, and the last scales (which a tile that was handed back has had).
      const long long t0 = clock64();
      while (sent && !kvtc::mbar_try(bar(M::B_UF + (int)lane), (sent - 1) & 1u) && clock64() - t0 <= DRAIN_LIMIT) {
      }
      __syncwarp();
      while (!ok && ti && !kvtc::mbar_try(bar(M::B_TF), (ti - 1) & 1u) && clock64() - t0 <= DRAIN_LIMIT) {
      }
    } else if (warp < ISSUER + 2) {
      // -------------------------------------------------------------- MMA issuers, one per pair
      // kind::f16: D f32 (bit 4), A and B f16, both K-major, N >> 3 at bit 17, M >> 4 at bit 24
      constexpr uint32_t IDESC = (1u << 4) | ((M::N >> 3) << 17) | ((HALF >> 4) << 24);
      // a descriptor's address field counts 16 bytes: offsets are added to the buffer's
      const uint64_t q = kvtc::smem_desc(base, 16, 1024, kvtc::LAYOUT_SW128);
      const uint32_t pair = warp - ISSUER;
      uint32_t j = 0;
      bool ok = true;
      for (uint32_t ti = 0; ok; ++ti) {
        if (!wait(M::B_TF, ti & 1u)) break;
        const Tile d = *tile;
        if (!(d.flags & TILE_LIVE)) break;
        // every chunk's, also where this pair has no rows: the phase of a barrier tells only the last two
        // apart.  The tile is handed back after it, so the other roles stay within one chunk of this one.
        if ((d.flags & TILE_FIRST) && !wait(M::B_QF + (d.chunk & 1u), (d.chunk >> 1) & 1u)) break;
        __syncwarp();
        if (lane == 0) kvtc::mbar_arrive(bar(M::B_TE));
        if (d.p0 + pair * HALF >= d.end) continue;
        // the warpgroups' blocks as they come
        uint32_t done[2] = {0, 0};  // steps issued
        long long t0 = 0;
        while (done[0] + done[1] < 2 * STEPS) {
          bool any = false;
#pragma unroll
          for (uint32_t g = 0; g < 2; ++g) {
            const uint32_t wg = 2 * pair + g, s = done[g], f = (j + s) & 1u;
            if (s == STEPS || !try_all(bar(M::B_AF + 2 * wg + f), ((j + s) >> 1) & 1u)) continue;
            any = true;
            ++done[g];
            kvtc::tc_fence_after();
            if (kvtc::elect_one()) {
              const uint32_t ta = tmem + wg * TM_WG + f * M::A_COLS, td = tmem + wg * TM_WG + M::TM_D + f * M::N;
              // the step's block; two blocks to a region of 64 elements
              const uint32_t blk = Q8 ? (s == 8 ? 16 + g : (s >> 1) * 4 + 2 * g + (s & 1u)) : 2 * s + g;
              const uint64_t at = q + ((blk >> 1) * M::REGION + (blk & 1u) * 64u) / 16;
#pragma unroll
              for (uint32_t ks = 0; ks < 2; ++ks) {
                mma_ts(td, ta + ks * 8u, at + ks * 2u, IDESC, ks);
                mma_ts(td, ta + ks * 8u, at + M::RB * 8u + ks * 2u, IDESC, 1u);
                if (!Q8) mma_ts(td, ta + 16u + ks * 8u, at + ks * 2u, IDESC, 1u);
              }
              kvtc::mma_commit(bar(M::B_DF + 2 * wg + f));
            }
            __syncwarp();
          }
          if (any) {
            t0 = 0;
          } else if (t0 == 0) {
            t0 = clock64();
          } else if (__any_sync(0xffffffffu, *abort_flag || clock64() - t0 > t.wait_limit)) {
            *abort_flag = 1u;
            ok = false;
            break;
          }
        }
        j += STEPS;
      }
      // all issued MMAs retire before TMEM is freed
      if (kvtc::elect_one()) kvtc::mma_commit(bar(M::B_FINAL + pair));
      __syncwarp();
      const long long t0 = clock64();
      while (!kvtc::mbar_try(bar(M::B_FINAL + pair), 0) && clock64() - t0 <= DRAIN_LIMIT) {
      }
    }
  } else {
    // ---------------------------------------------------------------- the warpgroups
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(COMPUTE_REGS));
    constexpr int HC = M::HC;
    const uint32_t wg = warp >> 2, pair = wg >> 1, g = wg & 1u, r = (warp & 3u) * 32u + lane;
    const uint32_t tw = tmem + ((warp & 3u) * 32u << 16) + wg * TM_WG;
    float* give = reinterpret_cast<float*>(sm + M::X) + wg * HC * HALF + r;
    const float* got = reinterpret_cast<const float*>(sm + M::X) + (wg ^ 1u) * HC * HALF + r;
    float* sums = reinterpret_cast<float*>(sm + M::S) + pair * 2 * HALF + r;
    const float2* col = reinterpret_cast<const float2*>(sm + M::COL) + g * HC;  // scale, -lse in powers of two
    const uint32_t* limit = reinterpret_cast<const uint32_t*>(sm + M::COL) + 2 * M::RB + g * HC;
    uint32_t j = 0, ui = 0, xi = 0;  // steps of the warpgroup, units of its ring, finished tiles of the pair
    // the first warpgroup: the tile before, whose mass is written once the other's sum is there
    float* out = nullptr;
    float keep_old = 0.f, factor = 1.f, own = 0.f;
    bool ok = true, open = false;  // open: a tile of this pair waits to be finished
    float2 tot[NC / 2];
    uint32_t d_b = 0, d_p = 0, d_c0 = 0, d_old = 0, d_fl = 0, d_chunk = 0;  // that tile, for this thread's row
    float last = 0.f;                                                        // its last block's scale
#pragma unroll
    for (int c = 0; c < NC / 2; ++c) tot[c] = make_float2(0.f, 0.f);
    // adds step jj's block sums times the block's scale to the scores
    auto drain = [&](uint32_t jj, float scale) -> bool {
      const uint32_t f = jj & 1u;
      if (!wait(M::B_DF + 2 * wg + f, (jj >> 1) & 1u)) return false;
      kvtc::tc_fence_after();
      uint32_t v[NC];
      kvtc::tmem_ld<NC>(tw + M::TM_D + f * M::N, v);
      kvtc::tmem_wait_ld();
      kvtc::reg_fence(v);
#pragma unroll
      for (int c = 0; c < NC / 2; ++c)
        tot[c] = __ffma2_rn(make_float2(__uint_as_float(v[2 * c]), __uint_as_float(v[2 * c + 1])),
                            make_float2(scale, scale), tot[c]);
      return true;
    };
    // the open tile: the rest of its scores, their weights, its sums
    auto finish = [&]() -> bool {
      if (!drain(j - 1, last)) return false;
      if ((d_fl & TILE_FIRST) && !wait(M::B_QF + (d_chunk & 1u), (d_chunk >> 1) & 1u)) return false;  // its columns' scales
      // each warpgroup gives away the other's half of the columns
      if (!wait(M::B_XE + pair, (xi & 1u) ^ 1u)) return false;
      float mine[HC];
#pragma unroll
      for (int c = 0; c < HC; ++c) {
        const float lo = c & 1 ? tot[c / 2].y : tot[c / 2].x;
        const int c2 = c + HC;
        const float hi = c2 & 1 ? tot[c2 / 2].y : tot[c2 / 2].x;
        mine[c] = g ? hi : lo;
        give[c * HALF] = g ? lo : hi;
      }
      __syncwarp();
      if (lane == 0) kvtc::mbar_arrive(bar(M::B_X + pair));
      if (!wait(M::B_X + pair, xi & 1u)) return false;
      if (out) *out = fmaf(factor, keep_old, own + sums[((xi & 1u) ^ 1u) * HALF]);
#pragma unroll
      for (int c = 0; c < HC; ++c) mine[c] += got[c * HALF];
      __syncwarp();
      if (lane == 0) kvtc::mbar_arrive(bar(M::B_XE + pair));
      float sum = 0.f;
      // a column that is not there has -lse = +inf and limit 0; with one query all others' limit is the length
#pragma unroll
      for (int c = 0; c < HC; ++c) {
        const float2 k = col[c];
        const float w = exp2_approx(fmaf(mine[c], k.x, k.y));
        sum += (a.n_q == 1 ? k.y != INFINITY : d_p < limit[c]) ? w : 0.f;
      }
      if (g) {
        sums[(xi & 1u) * HALF] = sum;
      } else {
        own = sum;
        out = nullptr;
        keep_old = 0.f;
        if (d_fl & 4u) {  // the row is there
          out = a.mass + (uint64_t)d_b * a.mass_stride + d_p;
          factor = d_c0 ? 1.f : a.decay;
          if (d_c0 || d_p < d_old) keep_old = *out;
        }
      }
      ++xi;
      open = false;
#pragma unroll
      for (int c = 0; c < NC / 2; ++c) tot[c] = make_float2(0.f, 0.f);
      return true;
    };
    for (uint32_t ti = 0;; ++ti) {
      if (!(ok = wait(M::B_TF, ti & 1u))) break;
      const Tile d = *tile;
      uint32_t scales[5];  // Q8_0: of this warpgroup's blocks: pairs of unit u; the last is one block
      if (Q8) {
        const uint32_t* sp = reinterpret_cast<const uint32_t*>(sm + M::SC + (pair * HALF + r) * NBLK * 2);
#pragma unroll
        for (int u = 0; u < 4; ++u) scales[u] = sp[2 * u + g];
        scales[4] = g ? sp[8] >> 16 : sp[8];
      }
      __syncwarp();
      if (lane == 0) kvtc::mbar_arrive(bar(M::B_TE));
      if (!(d.flags & TILE_LIVE)) break;
      // the tile before, and before a chunk its q parts, while this tile's first MMA runs or waits for them
      auto between = [&]() -> bool {
        if (open && !finish()) return false;
        if (d.flags & TILE_FIRST) {
          __syncwarp();
          if (lane == 0) kvtc::mbar_arrive(bar(M::B_QE));
          if (!wait(M::B_QE, d.chunk & 1u)) return false;  // nobody uses the parts of the chunk before
          fill_q<Q8, NC>(a, sm, warp, lane, d.b, d.c0, d.len, cols);
          kvtc::fence_proxy_async();
          __syncwarp();
          if (lane == 0) kvtc::mbar_arrive(bar(M::B_QF + (d.chunk & 1u)));
        }
        return true;
      };
      if (d.p0 + pair * HALF >= d.end) {  // no rows for this pair
        if (!(ok = between())) break;
        continue;
      }
      float before = 0.f;  // the step before's scale
#pragma unroll
      for (int s = 0; s < STEPS; ++s, ++j) {
        const uint32_t nth = ui + (Q8 ? (uint32_t)s / 2 : (uint32_t)s);
        const uint32_t slot = (Q8 ? pair : wg) * M::DEPTH + nth % M::DEPTH;
        if (!Q8 || s % 2 == 0) {
          if (!(ok = wait(M::B_UF + slot, (nth / M::DEPTH) & 1u))) break;
        }
        const char* st = sm + M::RING + slot * UNIT_BYTES;
        const uint32_t ta = tw + (j & 1u) * M::A_COLS;
        float scale;
        if constexpr (Q8) {
          uint32_t af[16];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t piece = (s < 8 ? g * 4 + (s & 1) * 2 : g * 2) + k;  // of 16 bytes
            const uint4 w = *reinterpret_cast<const uint4*>(
                st + (s < 8 ? kvtc::sw128_off(r, piece * 16) : kvtc::sw64_off(r, piece * 16)));
            int8_to_f16(w.x, af + 8 * k);
            int8_to_f16(w.y, af + 8 * k + 2);
            int8_to_f16(w.z, af + 8 * k + 4);
            int8_to_f16(w.w, af + 8 * k + 6);
          }
          kvtc::tmem_st<16>(ta, af);
          const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&scales[s / 2]));
          scale = s & 1 ? h.y : h.x;
        } else {
          float4 x[8];
          float amax = 0.f;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            x[k] = *reinterpret_cast<const float4*>(st + kvtc::sw128_off(r, k * 16));
            amax = fmaxf(fmaxf(fmaxf(amax, fabsf(x[k].x)), fmaxf(fabsf(x[k].y), fabsf(x[k].z))), fabsf(x[k].w));
          }
          const uint32_t f2 = scale_field(__float_as_uint(amax));
          const float up = __uint_as_float(f2 << 23);
          scale = __uint_as_float((254u - f2) << 23);
#pragma unroll
          for (int k = 0; k < 8; k += 4) {
            uint32_t hi[8], lo[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              split(x[k + i].x * up, x[k + i].y * up, hi + 2 * i, lo + 2 * i);
              split(x[k + i].z * up, x[k + i].w * up, hi + 2 * i + 1, lo + 2 * i + 1);
            }
            kvtc::tmem_st<8>(ta + 2 * k, hi);
            kvtc::tmem_st<8>(ta + 16 + 2 * k, lo);
          }
        }
        kvtc::tmem_wait_st();
        kvtc::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (!Q8 || s % 2 == 1 || s == 8) kvtc::mbar_arrive(bar(M::B_UE + slot));
          kvtc::mbar_arrive(bar(M::B_AF + 2 * wg + (j & 1u)));
        }
        if (s == 0) {
          if (!(ok = between())) break;
          open = true;
          d_b = d.b;
          d_p = d.p0 + pair * HALF + r;
          d_c0 = d.c0;
          d_old = d.old;
          d_chunk = d.chunk;
          d_fl = d.flags | (d_p < d.end && (d.ok >> ((pair * HALF + r) / t.box_rows) & 1u) ? 4u : 0u);
        } else if (!(ok = drain(j - 1, before))) {
          break;
        }
        before = scale;
      }
      if (!ok) break;
      last = before;
      ui += Q8 ? M::UNITS : STEPS;
    }
    if (ok && open) ok = finish();
    if (ok) {  // the last tile's sums
      __syncwarp();
      if (lane == 0) kvtc::mbar_arrive(bar(M::B_X + pair));
      if (wait(M::B_X + pair, xi & 1u) && out) *out = fmaf(factor, keep_old, own + sums[((xi & 1u) ^ 1u) * HALF]);
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

// Boxes of `box_cols` x `box_rows` elements of a row-major [rows][width] array; 64B swizzle for
// 64-byte boxes, else 128B.
int make_map(CUtensorMap* map, CUtensorMapDataType type, uint32_t elt, const void* at, uint64_t rows, uint32_t width,
             uint32_t box_cols, uint32_t box_rows) {
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
  const cuuint64_t dims[2] = {width, rows}, strides[1] = {(cuuint64_t)width * elt};
  const cuuint32_t estr[2] = {1, 1}, boxes[2] = {box_cols, box_rows};
  const CUresult r = enc(map, type, 2, const_cast<void*>(at), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         box_cols * elt == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r == CUDA_SUCCESS) return KVCU_OK;
  kvcu_set_error("cuTensorMapEncodeTiled failed: %d", (int)r);
  return KVCU_ERR_CUDA;
}

// Boxes of 128-byte pieces of the rows: Q8_0 bytes 0 .. 511 and the last 64; f32 latents and rope parts.
int make_maps(const kvcu_pool* p, uint32_t box_rows, CUtensorMap* wide, CUtensorMap* tail) {
  const CUtensorMapDataType u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8, f32 = CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  const int rc = p->quantized ? make_map(wide, u8, 1, p->qs, p->rows(), W, 128, box_rows)
                              : make_map(wide, f32, 4, p->kv, p->rows(), R, 32, box_rows);
  if (rc) return rc;
  return p->quantized ? make_map(tail, u8, 1, p->qs, p->rows(), W, 64, box_rows)
                      : make_map(tail, f32, 4, p->pe, p->rows(), P, 32, box_rows);
}

template <bool Q8, int NC>
int launch_mass(const kvcu_pool* pool, const MassArgs& a, const kvcu_decode_ws* ws, cudaStream_t st) {
  const int rc = kvcu_configure_once(
      reinterpret_cast<const void*>(k_mass<Q8, NC>),
      [](const void*) {
        // the register split assumes exactly this many at launch: with fewer, setmaxnreg.inc would wait for ever
        cudaFuncAttributes fa;
        KVCU_CUDA(cudaFuncGetAttributes(&fa, k_mass<Q8, NC>));
        if (fa.numRegs != LAUNCH_REGS) {
          kvcu_set_error("attn_mass: built with %d registers per thread, the register split needs %d", fa.numRegs,
                         LAUNCH_REGS);
          return KVCU_ERR_UNSUPPORTED;
        }
        return kvcu_check_cuda(
            cudaFuncSetAttribute(k_mass<Q8, NC>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Map<Q8, NC>::ALLOC),
            "cudaFuncSetAttribute(mass)");
      },
      nullptr);
  if (rc) return rc;
  TcMass t = {a, HALF, ws->wait_limit ? (long long)ws->wait_limit : (1ll << 31), ws->withhold_plus1};
  while (pool->block_size % t.box_rows) t.box_rows /= 2;  // block sizes are multiples of 16
  CUtensorMap wide, tail;
  const int rm = make_maps(pool, t.box_rows, &wide, &tail);
  if (rm) return rm;
  return kvcu_check_cuda(
      kvcu_launch_pdl(k_mass<Q8, NC>, dim3((uint32_t)ws->decode_ctas), dim3(TC_THREADS), Map<Q8, NC>::ALLOC, st, wide, tail, t),
      "attention mass launch");
}

// Columns of a chunk: a chunk costs its columns' scaling and exponentials and, whatever
// their number, the rows' unpacking (as much as about 30 columns).
template <bool Q8>
int launch_chunks(const kvcu_pool* pool, const MassArgs& a, const kvcu_decode_ws* ws, cudaStream_t st) {
  const uint32_t cols = a.n_q * a.n_heads;
  auto cost = [&](uint32_t nc) { return (uint64_t)((cols + nc - 1) / nc) * (nc + 30); };
  if (cost(8) <= cost(16) && cost(8) <= cost(20) && cost(8) <= cost(24))
    return launch_mass<Q8, 8>(pool, a, ws, st);
  if (cost(16) <= cost(20) && cost(16) <= cost(24)) return launch_mass<Q8, 16>(pool, a, ws, st);
  if (cost(20) <= cost(24)) return launch_mass<Q8, 20>(pool, a, ws, st);
  return launch_mass<Q8, 24>(pool, a, ws, st);
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
  if (pool->rows() > 0x7FFFFFFFull) {
    kvcu_set_error("kvcu_attn_mass: %llu rows, TMA coordinates reach 2^31 - 1", (unsigned long long)pool->rows());
    return KVCU_ERR_UNSUPPORTED;
  }
  ws->mass_launches = 1;
  if (!pool->quantized) return launch_chunks<false>(pool, a, ws, st);
  // Many columns: the wide kernel, in as few passes over the queries as the workspace's
  // decode partials (idle outside a decode) hold their parts for.
  const uint64_t room = (uint64_t)ws->max_layers * ws->max_items * ws->max_heads * R * 4;
  uint32_t passes = 1, count = n_q;
  while (count * n_heads >= WIDE_MIN_COLS && wide_scratch(n, count * n_heads) > room) count = (n_q + passes) / (passes + 1), ++passes;
  if (count * n_heads < WIDE_MIN_COLS) return launch_chunks<true>(pool, a, ws, st);
  ws->mass_launches = 0;
  for (uint32_t q0 = 0; q0 < n_q; q0 += count) {
    ws->mass_launches += 2;  // the columns' parts, and the sums
    const int rc = launch_wide(pool, a, q0, n_q - q0 < count ? n_q - q0 : count, ws->part_o, ws, st);
    if (rc) return rc;
  }
  return KVCU_OK;
}
