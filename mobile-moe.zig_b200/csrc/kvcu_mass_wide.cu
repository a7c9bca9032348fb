// kvcu_mass_wide.cu — the attention mass of Q8_0 rows for many columns (queries x heads).
//
// k_mass (kvcu_mass.cu) adds a row's 18 block sums in f32, exact int8 values times q:
// the best for a step's few columns, but its scaling grows with the columns and its
// chunks re-unpack the rows.  Here a row's value, int8 times its block's scale (19 bits),
// is the exact sum of two f16 parts, so one accumulator serves all of K = 576: a GEMM
//   S[row][column] = A_hi B_hi + A_lo B_hi + A_hi B_lo       (low times low < 2^-22)
// with 128 rows to a tile (A, unpacked into TMEM), up to 128 columns to a chunk (B, q's
// parts made by k_mass_wide_q) and the exponentials as its epilogue.
//   A row's scales are brought to at most 2^8 by a power of two of the row; its parts
// are exact for blocks with scales down to 2^-21 of the row's largest, and within
// 2^-39 of the row's largest value below that.  The tensor cores' f32 accumulation drops
// bits of each addend, so the low parts' products have an accumulator of their own, where
// that does not matter, and the main one is taken out after every third of K and added in
// registers: 12 additions of the tensor core to a sum.
//
// A unit is (tile, chunk), 9 stages of 64 elements each.  Per stage of N columns the
// MMAs take 12 x N/2 clocks; B is streamed from L2, 256 N bytes to a stage (43 B a clock
// of the 71 an SM can take), as a chunk of all of K would not fit in shared memory.
// Bound: the tensor cores, with the hand-overs around each stage (about 1,400 clocks a
// stage of 128 columns for 768 of MMAs).  Measured with 20 heads: 32 queries over 28.7k rows
// 77 us, 8 over them 36 us (chunked k_mass: 238 and 66).
//   warps 0-7    drain: each thread the sums of one row and half of the columns, their
//                exponentials, and the row's mass
//   warps 8-15   unpack every second stage to f16 parts in its TMEM buffer: four threads to
//                a row's 64 bytes (a thread to a row took four times the L1 passes, and held up
//                the MMAs' reads of shared memory), and an order of B's K that fits
//   warp 16      producer: bulk copies of 64 elements of N columns of one part, laid out for the MMA
//   warps 17-18  issue the MMAs of the main accumulator, and of the low parts'
#include "kvcu_mass.cuh"

using namespace kvmass;

namespace {

constexpr int DRAIN = 8, UNPACK = 16, PRODUCER = 16, ISSUER = 17, THREADS = 20 * 32;  // warps up to DRAIN, UNPACK
// Registers: launched with 96 a thread; the last warpgroup gives to the others.
constexpr int LAUNCH_REGS = 96, DRAIN_REGS = 120, UNPACK_REGS = 88, SERVICE_REGS = 64;
static_assert(8 * DRAIN_REGS + 8 * UNPACK_REGS + 4 * SERVICE_REGS <= 20 * LAUNCH_REGS,
              "register split exceeds the launch allocation");
static_assert(DRAIN_REGS > LAUNCH_REGS && UNPACK_REGS < LAUNCH_REGS && SERVICE_REGS < LAUNCH_REGS,
              "an increase to fewer registers, or a decrease to more, is an illegal instruction");
constexpr uint32_t ROWS = 128, STAGES = W / 64;
constexpr uint32_t MAX_N = 128, MAX_BLOCKS = MAX_N / 32;  // columns of a chunk; blocks of 16 a thread drains
constexpr uint32_t COL_BYTES = 12;  // constants of a column: scale and -lse, two columns' to 16 bytes; then the limits
constexpr uint32_t GROUP = 3;                             // stages to a drain
constexpr uint32_t RING_BYTES = 12 * MAX_N * 128, SLOTS = 12;  // of the ring: high parts in the even ones
constexpr uint32_t TM_X = 2 * MAX_N, TM_A = 3 * MAX_N, TM_COLS = 512;  // TMEM: two main sums, the low parts', two stages of 64
constexpr uint32_t COL = RING_BYTES;  // [2] a chunk's constants
constexpr uint32_t SUMS = COL + 2 * MAX_N * COL_BYTES;                // [2][ROWS]
// barriers
constexpr int B_BF = 0, B_BE = SLOTS, B_AF = 2 * SLOTS, B_AE = B_AF + 2, B_DF = B_AE + 2, B_DE = B_DF + 2,
              B_SF = B_DE + 2, B_SE = B_SF + 2, B_CF = B_SE + 2, B_CE = B_CF + 2, B_XF = B_CE + 2, B_XE = B_XF + 1, B_FINAL = B_XE + 1, NUM_BARS = B_FINAL + 1;
constexpr uint32_t BARS = SUMS + 2 * ROWS * 4, MISC = BARS + NUM_BARS * 8, ALLOC = MISC + 16 + 1024;
static_assert(ALLOC <= 232448 && TM_A + 2 * 64 <= TM_COLS, "budgets");
constexpr long long DRAIN_LIMIT = 1ll << 31;

struct Wide {
  MassArgs m;
  uint32_t q0, cols, chunks, width, padded;  // of an entry: first query, columns, chunks of `width`, chunks * width
  const char* parts;
  const char* col;                           // [n][chunks][width * COL_BYTES]
  long long wait_limit;
  uint32_t withhold_plus1;  // test hook: 0, or 1 + the tile of each CTA whose first unit of B is withheld
};

void shape(uint32_t cols, uint32_t* chunks, uint32_t* width) {
  *chunks = (cols + MAX_N - 1) / MAX_N;
  *width = ((cols + *chunks - 1) / *chunks + 31) / 32 * 32;
}

constexpr uint64_t NO_ROW = ~0ull;
// 32 columns of 16 TMEM lanes: lane l has columns 8 i + 2 (l % 4) and the next one of rows l / 4
// (v[4 i], v[4 i + 1]) and l / 4 + 8 (v[4 i + 2], v[4 i + 3]).
__device__ __forceinline__ void st_rows(uint32_t to, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(to),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
// The row of the pool that position p of the entry has, NO_ROW behind `end` or in a bad block.
__device__ __forceinline__ uint64_t row_of(const MassArgs& a, const Entry& e, uint32_t p, uint32_t end, bool report) {
  if (p >= end) return NO_ROW;
  const uint32_t blk = a.tables[e.t0 + p / a.block_size];
  if (blk < a.num_blocks) return ((uint64_t)a.layer * a.num_blocks + blk) * a.block_size + p % a.block_size;
  if (report) atomicOr(a.status, KVCU_STATUS_BAD_BLOCK);
  return NO_ROW;
}
// The exponent field of the power of two that brings the row's largest scale to [2^7, 2^8).
__device__ __forceinline__ uint32_t scale_of(const MassArgs& a, uint64_t row) {
  if (row == NO_ROW) return 127u;
  const uint32_t* scales = reinterpret_cast<const uint32_t*>(a.sc + row * NBLK);
  uint32_t top = 0;
#pragma unroll
  for (uint32_t s = 0; s < STAGES; ++s) {
    const uint32_t two = __ldg(scales + s) & 0x7fff7fffu;
    top = max(top, max(two & 0xffffu, two >> 16));
  }
  const uint32_t bits = __float_as_uint(__half2float(__ushort_as_half((unsigned short)top)));
  return top == 0u || top >= 0x7c00u ? 127u : 261u - (bits >> 23);  // 7 - exponent, biased
}

// The columns' parts, [n][chunk][stage][hi, lo] units of B as shared memory holds them (`width`
// rows of 64 f16, 128B swizzle), and constants; a warp to a column.
__global__ void __launch_bounds__(256) k_mass_wide_q(const Wide t, char* parts, char* consts) {
  kvcu_pdl_wait();
  const MassArgs& a = t.m;
  const uint64_t id = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const uint32_t lane = threadIdx.x & 31u;
  if (id >= (uint64_t)a.n * t.padded) return;
  const uint32_t b = (uint32_t)(id / t.padded), c = (uint32_t)(id % t.padded);
  const bool live = c < t.cols;
  const uint32_t i = t.q0 + c / a.n_heads;
  const uint64_t column = ((uint64_t)b * a.n_q + i) * a.n_heads + c % a.n_heads;
  const float4* src = reinterpret_cast<const float4*>(a.q + column * W);
  float4 x[5];
  float amax = 0.f;
#pragma unroll
  for (int k = 0; k < 5; ++k) {
    const uint32_t f = lane + 32 * k;
    x[k] = live && f < W / 4 ? src[f] : make_float4(0.f, 0.f, 0.f, 0.f);
    amax = fmaxf(fmaxf(fmaxf(amax, fabsf(x[k].x)), fmaxf(fabsf(x[k].y), fabsf(x[k].z))), fabsf(x[k].w));
  }
  const uint32_t field = scale_field(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));
  const float up = __uint_as_float(field << 23);
  char* units = parts + ((uint64_t)b * t.chunks + c / t.width) * STAGES * 2 * (t.width * 128u);
#pragma unroll
  for (int k = 0; k < 5; ++k) {
    const uint32_t f = lane + 32 * k;
    if (f >= W / 4) continue;
    uint2 h, l;
    split(x[k].x * up, x[k].y * up, &h.x, &l.x);
    split(x[k].z * up, x[k].w * up, &h.y, &l.y);
    // 64 elements in the order that the rows' unpacking gives them: piece f / 4, four elements f % 4 of it
    char* to = units + f / 16 * 2 * (t.width * 128u) + kvtc::sw128_off(c % t.width, (f % 4 * 4 + f / 4 % 4) * 8);
    *reinterpret_cast<uint2*>(to) = h;
    *reinterpret_cast<uint2*>(to + t.width * 128u) = l;
  }
  if (lane == 0) {
    constexpr double LOG2E = 1.4426950408889634;
    const float l = live ? a.lse[column] : -INFINITY;
    const uint32_t behind = live ? a.n_q - 1 - i : 0u, len = entry_of(a, b, false).len;
    // a column past the last, or a query that saw nothing, has no positions: its weights are 2^-inf
    const bool none = l == -INFINITY || len <= behind;
    const uint32_t at = c % t.width;
    char* col = consts + ((uint64_t)b * t.chunks + c / t.width) * t.width * COL_BYTES;
    float* pair = reinterpret_cast<float*>(col) + at / 2 * 4 + (at & 1u);
    pair[0] = none ? 0.f : (float)(a.scale * LOG2E) * __uint_as_float((254u - field) << 23);
    pair[2] = none ? -INFINITY : (float)(-l * LOG2E);
    reinterpret_cast<uint32_t*>(col + t.width * 8u)[at] = none ? 0u : len - behind;
  }
}

__global__ void __launch_bounds__(THREADS, 1) k_mass_wide(const Wide t) {
  const MassArgs& a = t.m;
  extern __shared__ char raw[];
  char* sm = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  const uint32_t base = kvtc::smem_u32(sm);
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(sm + MISC + 4);
  auto bar = [&](uint32_t i) { return base + BARS + 8u * i; };
  auto wait = [&](uint32_t i, uint32_t parity) { return wait_bar(bar(i), parity, abort_flag, t.wait_limit); };
  if (tid == 0) {
    auto init = [&](int first, int n, uint32_t count) {
      for (int i = 0; i < n; ++i) kvtc::mbar_init(bar(first + i), count);
    };
    init(B_BF, SLOTS, 1);
    for (int i = 0; i < SLOTS; ++i) kvtc::mbar_init(bar(B_BE + i), i & 1 ? 1 : 2);  // both issuers read a high part
    init(B_AF, 2, 4);
    init(B_AE, 2, 2);
    init(B_DF, 2, 1);
    init(B_DE, 2, DRAIN);
    init(B_SF, 2, 4);
    init(B_SE, 2, 4);
    init(B_CF, 2, 1);
    init(B_CE, 2, DRAIN);
    init(B_XF, 1, 1);
    init(B_XE, 1, DRAIN);
    init(B_FINAL, 1, 2);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == ISSUER) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + MISC), "r"(TM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  kvcu_pdl_wait();
  kvtc::tc_fence_before();
  __syncthreads();
  kvtc::tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(sm + MISC);
  const uint32_t n_items = a.meta[0], n_ranges = a.meta[1];
  const uint32_t it0 = blockIdx.x < n_ranges ? min(a.ranges[blockIdx.x], n_items) : n_items;
  const uint32_t it1 = blockIdx.x < n_ranges ? min(a.ranges[blockIdx.x + 1], n_items) : n_items;
  const uint32_t unit_bytes = t.width * 128u;
  bool ok = true;

  if (warp >= UNPACK) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(SERVICE_REGS));
  if (warp == PRODUCER) {
    // ---------------------------------------------------------------- producer
    if (blockIdx.x == 0 && lane == 0 && n_ranges > gridDim.x) atomicOr(a.status, KVCU_STATUS_BAD_PLAN);
    uint32_t slot = 0, lap = 0, tile = 0, unit = 0;
    uint32_t sent = 0;  // lane k: units of B sent through slot k
    for (uint32_t it = it0; ok && it < it1; ++it) {
      const kvcu_item w = a.items[it];
      const uint32_t end = min(w.end, entry_of(a, w.b, lane == 0).len);
      for (uint32_t p0 = w.start; ok && p0 < end; p0 += ROWS) {
        ++tile;
        for (uint32_t ch = 0; ok && ch < t.chunks; ++ch) {
          if (!(ok = wait(B_CE + (unit & 1u), ((unit >> 1) & 1u) ^ 1u))) break;
          if (lane == 0) {
            kvtc::mbar_arrive_tx(bar(B_CF + (unit & 1u)), t.width * COL_BYTES);
            bulk_load(base + COL + (unit & 1u) * MAX_N * COL_BYTES,
                      t.col + ((uint64_t)w.b * t.chunks + ch) * t.width * COL_BYTES, t.width * COL_BYTES,
                      bar(B_CF + (unit & 1u)));
          }
          __syncwarp();
          ++unit;
          for (uint32_t u = 0; u < 2 * STAGES; ++u) {  // stage u / 2, part u % 2
            if (!(ok = wait(B_BE + slot, (lap & 1u) ^ 1u))) break;
            // test hook: no copy and no arrival, the waits on it run out
            if (!(u == 0 && ch == 0 && tile == t.withhold_plus1)) {
              if (lane == 0) {
                kvtc::mbar_arrive_tx(bar(B_BF + slot), unit_bytes);
                bulk_load(base + slot * unit_bytes,
                          t.parts + (((uint64_t)w.b * t.chunks + ch) * STAGES * 2 + u) * unit_bytes, unit_bytes,
                          bar(B_BF + slot));
              }
              __syncwarp();
              sent += lane == slot;
            }
            if (++slot == SLOTS) slot = 0, ++lap;
          }
        }
      }
    }
    // the copies in flight must land before the CTA leaves, also where only their readers have given up
    const long long t0 = clock64();
    while (sent && !kvtc::mbar_try(bar(B_BF + lane), (sent - 1) & 1u) && clock64() - t0 <= DRAIN_LIMIT) {
    }
    __syncwarp();
    while (unit && !kvtc::mbar_try(bar(B_CF + ((unit - 1) & 1u)), ((unit - 1) >> 1) & 1u) &&
           clock64() - t0 <= DRAIN_LIMIT) {
    }
    __syncwarp();
  } else if (warp == ISSUER || warp == ISSUER + 1) {
    // ---------------------------------------------------------------- MMA issuers
    // Few MMAs queue up behind the running one, not enough for the time that a warp's waits take: two
    // warps, one for each accumulator, wait in turn.
    // kind::f16: D f32 (bit 4), A and B f16, both K-major, N >> 3 at bit 17, M >> 4 at bit 24
    const uint32_t idesc = (1u << 4) | ((t.width >> 3) << 17) | ((ROWS >> 4) << 24);
    const bool main = warp == ISSUER;
    uint32_t x = 0, slot = 0, lap = 0;  // stages, and the ring's place
    for (uint32_t it = it0; ok && it < it1; ++it) {
      const kvcu_item w = a.items[it];
      const uint32_t end = min(w.end, entry_of(a, w.b, false).len);
      const uint32_t units = w.start < end ? (end - w.start + ROWS - 1) / ROWS * t.chunks : 0u;
      for (uint32_t s = 0; s < units * STAGES; ++s, ++x) {
        const uint32_t period = main ? GROUP : STAGES, n = x / period, f = main ? n & 1u : 0u;
        const bool first = x % period == 0, last = x % period == period - 1;
        if (first && !(ok = wait((main ? B_DE : B_XE) + f, ((main ? n >> 1 : n) & 1u) ^ 1u))) break;
        if (!(ok = wait(B_AF + (x & 1u), (x >> 1) & 1u)) || !(ok = wait(B_BF + slot, lap & 1u))) break;
        const uint32_t td = tmem + (main ? 0u : TM_X) + f * MAX_N, ta = tmem + TM_A + (x & 1u) * 64u;
        const uint64_t hi = kvtc::smem_desc(base + slot * unit_bytes, 16, 1024, kvtc::LAYOUT_SW128);
        kvtc::tc_fence_after();
        if (kvtc::elect_one()) {
          // A_hi B_hi, or A_lo B_hi
#pragma unroll
          for (uint32_t ks = 0; ks < 4; ++ks)
            mma_ts(td, ta + (main ? 0u : 32u) + ks * 8u, hi + ks * 2u, idesc, first && ks == 0 ? 0u : 1u);
          kvtc::mma_commit(bar(B_BE + slot));
          if (main) {
            kvtc::mma_commit(bar(B_AE + (x & 1u)));
            if (last) kvtc::mma_commit(bar(B_DF + f));
          }
        }
        __syncwarp();
        if (!main) {
          if (!(ok = wait(B_BF + slot + 1, lap & 1u))) break;
          kvtc::tc_fence_after();
          if (kvtc::elect_one()) {
            const uint64_t lo = kvtc::smem_desc(base + (slot + 1) * unit_bytes, 16, 1024, kvtc::LAYOUT_SW128);
#pragma unroll
            for (uint32_t ks = 0; ks < 4; ++ks) mma_ts(td, ta + ks * 8u, lo + ks * 2u, idesc, 1u);  // A_hi B_lo
            kvtc::mma_commit(bar(B_BE + slot + 1));
            kvtc::mma_commit(bar(B_AE + (x & 1u)));
            if (last) kvtc::mma_commit(bar(B_XF + f));
          }
          __syncwarp();
        }
        slot += 2;
        if (slot == SLOTS) slot = 0, ++lap;
      }
    }
    // all issued MMAs retire before TMEM is freed
    if (kvtc::elect_one()) kvtc::mma_commit(bar(B_FINAL));
    __syncwarp();
    const long long t0 = clock64();
    while (!kvtc::mbar_try(bar(B_FINAL), 0) && clock64() - t0 <= DRAIN_LIMIT) {
    }
  } else if (warp < DRAIN) {
    // ---------------------------------------------------------------- sums
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(DRAIN_REGS));
    const uint32_t g = warp >> 2, r = (warp & 3u) * 32u + lane, half = t.width / 2, blocks = t.width / 32;
    const uint32_t td = tmem + ((warp & 3u) * 32u << 16) + g * half;
    float* sums = reinterpret_cast<float*>(sm + SUMS) + r;
    uint32_t group = 0, unit = 0, tiles = 0;  // of the CTA
    for (uint32_t it = it0; ok && it < it1; ++it) {
      const kvcu_item w = a.items[it];
      const Entry e = entry_of(a, w.b, false);
      const uint32_t end = min(w.end, e.len), old = t.q0 ? e.len : e.old;
      for (uint32_t p0 = w.start; ok && p0 < end; p0 += ROWS, ++tiles) {
        const uint32_t p = p0 + r;
        const uint64_t row = row_of(a, e, p, end, g == 0);
        const float down = __uint_as_float((254u - scale_of(a, row)) << 23);
        float* out = a.mass + (uint64_t)w.b * a.mass_stride + p;
        float before = 0.f;
        float2 run = make_float2(0.f, 0.f);
        if (g == 0 && row != NO_ROW && (t.q0 || p < old)) before = *out;
        for (uint32_t ch = 0; ok && ch < t.chunks; ++ch) {
          float2 tot[MAX_BLOCKS][8];
#pragma unroll 1
          for (uint32_t part = 0; part < STAGES / GROUP; ++part, ++group) {
            const uint32_t f = group & 1u;
            if (!(ok = wait(B_DF + f, (group >> 1) & 1u))) break;
            kvtc::tc_fence_after();
            auto take = [&](uint32_t from, bool start) {
#pragma unroll
              for (uint32_t i = 0; i < MAX_BLOCKS; ++i) {
                if (i >= blocks) continue;
                uint32_t v[16];
                kvtc::tmem_ld<16>(from + i * 16, v);
                kvtc::tmem_wait_ld();
                kvtc::reg_fence(v);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                  const float2 x = make_float2(__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1]));
                  tot[i][k] = start ? x : __fadd2_rn(tot[i][k], x);
                }
              }
            };
            auto done = [&](uint32_t i) {
              kvtc::tc_fence_before();
              __syncwarp();
              if (lane == 0) kvtc::mbar_arrive(bar(i));
            };
            if (part == STAGES / GROUP - 1) {  // the low parts' first: there is one accumulator of them
              if (!(ok = wait(B_XF, unit & 1u))) break;
              kvtc::tc_fence_after();
              take(td + TM_X, false);
              done(B_XE);
            }
            take(td + f * MAX_N, part == 0);
            done(B_DE + f);
          }
          if (!ok) break;
          if (!(ok = wait(B_CF + (unit & 1u), (unit >> 1) & 1u))) break;
          const char* constants = sm + COL + (unit & 1u) * MAX_N * COL_BYTES;
          const float4* col = reinterpret_cast<const float4*>(constants) + g * half / 2;
          const uint2* limit = reinterpret_cast<const uint2*>(constants + t.width * 8u) + g * half / 2;
          // every query's limit is behind the tile, but for the last tiles
          const bool inside = p0 + ROWS + t.m.n_q <= e.len + 1;
          const float2 back = make_float2(down, down);
          auto weigh = [&](uint32_t i, auto&& use) {
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) {
              const float4 c = col[i * 8 + k];  // of two columns
              const float2 s = __ffma2_rn(__fmul2_rn(tot[i][k], back), make_float2(c.x, c.y), make_float2(c.z, c.w));
              use(i * 8 + k, make_float2(exp2_approx(s.x), exp2_approx(s.y)));
            }
          };
          const float2 start = run;
          if (inside) {
#pragma unroll
            for (uint32_t i = 0; i < MAX_BLOCKS; ++i)
              if (i < blocks) weigh(i, [&](uint32_t, float2 weight) { run = __fadd2_rn(run, weight); });
          }
          // also for a row whose infinities or NaN met a column without positions (0 times them is NaN)
          if (!inside || !(run.x + run.y < INFINITY)) {
            run = start;
#pragma unroll
            for (uint32_t i = 0; i < MAX_BLOCKS; ++i)
              if (i < blocks)
                weigh(i, [&](uint32_t k, float2 weight) {
                  const uint2 l = limit[k];
                  run = __fadd2_rn(run, make_float2(p < l.x ? weight.x : 0.f, p < l.y ? weight.y : 0.f));
                });
          }
          __syncwarp();
          if (lane == 0) kvtc::mbar_arrive(bar(B_CE + (unit & 1u)));
          ++unit;
        }
        if (!ok) break;
        // the second half's sum to the first, which writes the mass
        const uint32_t f = tiles & 1u, parity = (tiles >> 1) & 1u;
        if (g) {
          if (!(ok = wait(B_SE + f, parity ^ 1u))) break;
          sums[f * ROWS] = run.x + run.y;
          __syncwarp();
          if (lane == 0) kvtc::mbar_arrive(bar(B_SF + f));
        } else {
          if (!(ok = wait(B_SF + f, parity))) break;
          const float sum = run.x + run.y + sums[f * ROWS];
          __syncwarp();
          if (lane == 0) kvtc::mbar_arrive(bar(B_SE + f));
          if (row != NO_ROW) *out = fmaf(t.q0 ? 1.f : a.decay, before, sum);
        }
      }
    }
  } else if (warp < UNPACK) {
    // ---------------------------------------------------------------- rows
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(UNPACK_REGS));
    const uint32_t pair = (warp - DRAIN) >> 2, r = (warp & 3u) * 32u + lane, piece = lane & 3u;
    const uint32_t ta = tmem + ((warp & 3u) * 32u << 16) + TM_A + pair * 64u;
    uint32_t x = 0;  // stages of the units before
    for (uint32_t it = it0; ok && it < it1; ++it) {
      const kvcu_item w = a.items[it];
      const Entry e = entry_of(a, w.b, false);
      const uint32_t end = min(w.end, e.len);
      for (uint32_t p0 = w.start; ok && p0 < end; p0 += ROWS) {
        const uint64_t own = row_of(a, e, p0 + r, end, false);
        const float own_up = __uint_as_float(scale_of(a, own) << 23);
        uint32_t row[4];
        float up[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          row[m] = __shfl_sync(0xffffffffu, (uint32_t)own, (lane >> 2) + 8 * m);  // rows count to 2^31 at most
          up[m] = __shfl_sync(0xffffffffu, own_up, (lane >> 2) + 8 * m);
        }
        uint4 d[4] = {};
        uint16_t sc[4] = {};
        auto load = [&](uint32_t s) {
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            if (row[m] == (uint32_t)NO_ROW) continue;
            d[m] = __ldg(reinterpret_cast<const uint4*>(a.qs + (uint64_t)row[m] * W + s * 64) + piece);
            sc[m] = __ldg(a.sc + (uint64_t)row[m] * NBLK + s * 2 + piece / 2);
          }
        };
        load((x ^ pair) & 1u);
        for (uint32_t ch = 0; ok && ch < t.chunks; ++ch, x += STAGES)
          for (uint32_t s = (x ^ pair) & 1u; s < STAGES; s += 2) {
            // this pair's buffer's n-th use
            if (!(ok = wait(B_AE + pair, (((x + s) >> 1) & 1u) ^ 1u))) break;
#pragma unroll
            for (int m = 0; m < 4; m += 2) {  // two rows
              uint32_t hi[16], lo[16];
#pragma unroll
              for (int n = 0; n < 2; ++n) {
                const __half2 scale = __float2half2_rn(__half2float(__ushort_as_half(sc[m + n])) * up[m + n]);
                uint32_t y[8];
                int8_to_f16(d[m + n].x, y);
                int8_to_f16(d[m + n].y, y + 2);
                int8_to_f16(d[m + n].z, y + 4);
                int8_to_f16(d[m + n].w, y + 6);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  const __half2 v = *reinterpret_cast<const __half2*>(&y[i]), top = __hmul2_rn(v, scale);
                  const __half2 rest = __hfma2(v, scale, __hneg2(top));
                  hi[i / 2 * 4 + n * 2 + i % 2] = *reinterpret_cast<const uint32_t*>(&top);
                  lo[i / 2 * 4 + n * 2 + i % 2] = *reinterpret_cast<const uint32_t*>(&rest);
                }
              }
              st_rows(ta + ((uint32_t)m * 8u << 16), hi);
              st_rows(ta + ((uint32_t)m * 8u << 16) + 32, lo);
            }
            load(s + 2 < STAGES ? s + 2 : s + 2 - STAGES);  // the next one of this tile, if there is one
            kvtc::tmem_wait_st();
            kvtc::tc_fence_before();
            __syncwarp();
            if (lane == 0) kvtc::mbar_arrive(bar(B_AF + pair));
          }
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

}  // namespace

namespace kvmass {

uint64_t wide_scratch(uint32_t n, uint32_t cols) {
  uint32_t chunks, width;
  shape(cols, &chunks, &width);
  return (uint64_t)n * chunks * width * (2 * W * sizeof(__half) + COL_BYTES);
}

int launch_wide(const kvcu_pool* pool, const MassArgs& a, uint32_t q0, uint32_t count, void* scratch,
                const kvcu_decode_ws* ws, cudaStream_t st) {
  Wide t = {};
  t.m = a;
  t.q0 = q0;
  t.cols = count * a.n_heads;
  shape(t.cols, &t.chunks, &t.width);
  t.padded = t.chunks * t.width;
  const uint64_t columns = (uint64_t)a.n * t.padded;
  char* parts = static_cast<char*>(scratch);
  char* consts = parts + columns * 2 * W * sizeof(__half);
  t.parts = parts;
  t.col = consts;
  t.wait_limit = ws->wait_limit ? (long long)ws->wait_limit : (1ll << 31);
  t.withhold_plus1 = ws->withhold_plus1;
  int rc = kvcu_configure_once(
      reinterpret_cast<const void*>(k_mass_wide),
      [](const void*) {
        // the register split assumes exactly this many at launch: with fewer, setmaxnreg.inc would wait for ever
        cudaFuncAttributes fa;
        KVCU_CUDA(cudaFuncGetAttributes(&fa, k_mass_wide));
        if (fa.numRegs != LAUNCH_REGS) {
          kvcu_set_error("attn_mass: built with %d registers per thread, the register split needs %d", fa.numRegs,
                         LAUNCH_REGS);
          return (int)KVCU_ERR_UNSUPPORTED;
        }
        return kvcu_check_cuda(cudaFuncSetAttribute(k_mass_wide, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ALLOC),
                               "cudaFuncSetAttribute(mass)");
      },
      nullptr);
  if (rc) return rc;
  rc = kvcu_check_cuda(kvcu_launch_pdl(k_mass_wide_q, dim3((uint32_t)((columns + 7) / 8)), dim3(256), 0, st, t, parts, consts),
                       "attention mass columns launch");
  if (rc) return rc;
  return kvcu_check_cuda(kvcu_launch_pdl(k_mass_wide, dim3((uint32_t)ws->decode_ctas), dim3(THREADS), ALLOC, st, t),
                         "attention mass launch");
}

}  // namespace kvmass
