// kvcu_mass.cuh — what the two attention-mass kernels share: their arguments, an
// entry's length and table, waits, and the f16 parts of f32 values.
#pragma once
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>

#include "kvcu_internal.h"
#include "kvcu_tcgen05.cuh"

namespace kvmass {

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

// Whether the phase is over, for the converged warp: all lanes or none.
__device__ __forceinline__ bool try_all(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n"
      " vote.sync.all.pred p, p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded wait of the converged warp: false after `limit` clocks or when another
// role has given up.
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag, long long limit) {
  if (try_all(bar, parity)) return true;
  const long long t0 = clock64();
  while (!try_all(bar, parity))
    if (__any_sync(0xffffffffu, *abort_flag || clock64() - t0 > limit)) {
      *abort_flag = 1u;
      return false;
    }
  return true;
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

// 2^x by the hardware (PTX ex2.approx.f32: relative error below 2^-22).
__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
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
// x and y as f16 pairs hi + lo
__device__ __forceinline__ void split(float x, float y, uint32_t* hi, uint32_t* lo) {
  *hi = pack_half(x, y);
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(hi));
  *lo = pack_half(x - h.x, y - h.y);
}
// The exponent field of the power of two that brings a largest magnitude (its f32
// bits) to [2^13, 2^14); 1 for zeros or an infinity among them.  254 minus it is the
// inverse's.
__device__ __forceinline__ uint32_t scale_field(uint32_t top) {
  const uint32_t eb = top >> 23;
  return top == 0u || eb >= 255u ? 127u : (uint32_t)min(max(267 - (int)eb, 1), 253);
}

// The kernel for many columns (kvcu_mass_wide.cu): queries [q0, q0 + count) of every entry.
// From 48 columns on it is the faster one (14k to 60k rows: 40 columns 22 us against 21, 48 equal, 80 23
// against 37, 320 50 against 126).
constexpr uint32_t WIDE_MIN_COLS = 48;
uint64_t wide_scratch(uint32_t n, uint32_t cols);  // bytes it takes for n entries of `cols` columns
int launch_wide(const kvcu_pool* pool, const MassArgs& a, uint32_t q0, uint32_t count, void* scratch,
                const kvcu_decode_ws* ws, cudaStream_t st);

}  // namespace kvmass
