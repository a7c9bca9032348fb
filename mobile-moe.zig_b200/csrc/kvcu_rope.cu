// kvcu_rope.cu — rotary positions as an operator of their own.
//
// y = m R(pos) x over the pairs of a head's rotary part, R(pos) turning pair i
// by the angle pos * f_i:
//   y_a = m (x_a cos - x_b sin),  y_b = m (x_a sin + x_b cos)
// with (a, b) = (2i, 2i+1) in the interleaved layout (what the reference's
// RoPECache.apply does, src/math.zig:227-238) or (i, i + d/2) in the half
// layout.  The transposed form m R(pos)^T, the same with the sine negated, is
// the gradient of y with respect to x.  f_i = base^(-2i/d), or one of three
// published changes of it for contexts longer than the trained one (see
// kvcu_rope_create).
//
// The angles: pos * f_i reaches millions of radians, where one f32 rounding of
// the product is already a tenth of a radian.  So the table holds turns per
// position, f_i / 2 pi, in 64 bits; the product and its reduction to
// [-1/2, 1/2] turns are done in 64 bits (exact to 1e-16 of the number of
// turns), and only the reduced angle is rounded to f32, for sincospif.
//
// Bound: memory.  Each CTA forms the sines of its tokens once in shared memory
// (a few 64-bit operations per token and pair, shared by all heads), then every
// thread turns V pairs with two 16-byte loads and two 16-byte stores.
// Measured: 4,096 tokens' gradient in f32 (40 heads of 128) 33 us, 5.1 TB/s; one token is
// the launch.  A bf16 prompt of 8,191 tokens takes 14 us, 3.1 TB/s, by latency (issue 39%,
// memory 19%): no row is being loaded until a CTA's sines are there, and after that each
// thread has two loads in flight.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>

#include <new>

#include "kvcu_internal.h"

namespace {

constexpr int ROPE_THREADS = 256;
constexpr uint32_t ROPE_MAX_HEADS = 16384;  // q and k heads together: keeps the 32-bit quotients exact
constexpr uint32_t ROPE_MAX_TOKENS = 8;     // tokens of one CTA

struct RopeTensor {
  const void* x;
  void* y;
  uint64_t x_row, x_head, y_row, y_head;  // elements
  uint32_t heads;
};

struct RopeArgs {
  const uint32_t* pos;
  uint32_t n, half, tokens;    // tokens: per CTA
  uint64_t div_heads, div_chunks;  // ceil(2^32 / d) of the row and chunk counts
  uint32_t heads, chunks;      // q + k heads; chunks of V pairs per head
  float mscale, sign;          // sign: -1 for the transposed form
  RopeTensor t[2];
  double turns[KVCU_ROPE_MAX_PAIRS];  // f_i / (2 pi)
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_f32(float v, float* o) { *o = v; }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16* o) { *o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f32(float v, __half* o) { *o = __float2half_rn(v); }

// x / d for x * d < 2^32, m = ceil(2^32 / d)
__device__ __forceinline__ uint32_t quot(uint32_t x, uint64_t m) { return (uint32_t)((x * m) >> 32); }

// Each thread turns V pairs: V = 16 / sizeof(T) where the addresses allow
// 16-byte accesses, else 1.
template <typename T, bool HALF, int V>
__global__ void __launch_bounds__(ROPE_THREADS) k_rope(const __grid_constant__ RopeArgs a) {
  extern __shared__ float2 cs[];  // [tokens][half] (cos, sin) times the magnitude
  const uint32_t t0 = blockIdx.x * a.tokens;
  const uint32_t tn = min(a.tokens, a.n - t0);
  for (uint32_t i = threadIdx.x; i < tn * a.half; i += ROPE_THREADS) {
    const uint32_t t = i / a.half, p = i - t * a.half;
    double u = (double)a.pos[t0 + t] * a.turns[p];
    u -= rint(u);
    float s, c;
    sincospif(2.0f * (float)u, &s, &c);
    cs[i] = make_float2(c * a.mscale, s * a.mscale * a.sign);
  }
  __syncthreads();
  const uint32_t items = tn * a.heads * a.chunks;
  for (uint32_t i = threadIdx.x; i < items; i += ROPE_THREADS) {
    const uint32_t row = quot(i, a.div_chunks), c = i - row * a.chunks;
    const uint32_t tok = quot(row, a.div_heads);
    uint32_t h = row - tok * a.heads;
    const int w = h >= a.t[0].heads;
    if (w) h -= a.t[0].heads;
    const RopeTensor& r = a.t[w];
    const T* x = static_cast<const T*>(r.x) + (t0 + tok) * r.x_row + h * r.x_head;
    T* y = static_cast<T*>(r.y) + (t0 + tok) * r.y_row + h * r.y_head;
    const uint32_t p0 = c * V;                     // first pair
    const uint32_t o0 = HALF ? p0 : 2 * p0;        // the two 16-byte pieces (V elements each)
    const uint32_t o1 = HALF ? p0 + a.half : 2 * p0 + V;
    __align__(16) T u[V], v[V];
    if constexpr (V > 1) {
      *reinterpret_cast<uint4*>(u) = *reinterpret_cast<const uint4*>(x + o0);
      *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(x + o1);
    } else {
      u[0] = x[o0];
      v[0] = x[o1];
    }
    const float2* f = cs + tok * a.half + p0;
    if constexpr (HALF || V == 1) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float xa = to_f32(u[k]), xb = to_f32(v[k]);
        from_f32(xa * f[k].x - xb * f[k].y, &u[k]);
        from_f32(xa * f[k].y + xb * f[k].x, &v[k]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < V / 2; ++k) {
        const float xa = to_f32(u[2 * k]), xb = to_f32(u[2 * k + 1]);
        from_f32(xa * f[k].x - xb * f[k].y, &u[2 * k]);
        from_f32(xa * f[k].y + xb * f[k].x, &u[2 * k + 1]);
        const float ya = to_f32(v[2 * k]), yb = to_f32(v[2 * k + 1]);
        from_f32(ya * f[V / 2 + k].x - yb * f[V / 2 + k].y, &v[2 * k]);
        from_f32(ya * f[V / 2 + k].y + yb * f[V / 2 + k].x, &v[2 * k + 1]);
      }
    }
    if constexpr (V > 1) {
      *reinterpret_cast<uint4*>(y + o0) = *reinterpret_cast<const uint4*>(u);
      *reinterpret_cast<uint4*>(y + o1) = *reinterpret_cast<const uint4*>(v);
    } else {
      y[o0] = u[0];
      y[o1] = v[0];
    }
  }
}

bool aligned16(const RopeTensor& t, uint32_t size) {
  if (!t.heads) return true;
  const uint64_t bits = (uint64_t)t.x | (uint64_t)t.y | (t.x_row * size) | (t.x_head * size) | (t.y_row * size) |
                        (t.y_head * size);
  return bits % 16 == 0;
}

// Whether the n x heads output segments of `rot` elements are disjoint: of the
// two strides the smaller must clear a segment and the larger everything below.
bool disjoint(uint32_t n, uint32_t heads, uint64_t row, uint64_t head, uint32_t rot) {
  uint64_t small = row, large = head, ns = n, nl = heads;
  if (nl <= 1 || (ns > 1 && head < row)) {
    small = head;
    large = row;
    ns = heads;
    nl = n;
  }
  if (ns > 1 && small < rot) return false;
  const uint64_t span = ns > 1 ? (ns - 1) * small + rot : rot;
  return nl <= 1 || large >= span;
}

template <typename T>
int launch(const RopeArgs& args, bool half, cudaStream_t st) {
  RopeArgs a = args;
  constexpr uint32_t VEC = 16 / sizeof(T);
  const bool vec = a.half % VEC == 0 && aligned16(a.t[0], sizeof(T)) && aligned16(a.t[1], sizeof(T));
  a.chunks = vec ? a.half / VEC : a.half;
  a.div_chunks = ((1ull << 32) + a.chunks - 1) / a.chunks;
  const dim3 grid((a.n + a.tokens - 1) / a.tokens);
  const size_t smem = (size_t)a.tokens * a.half * sizeof(float2);
  if (vec) {
    if (half) k_rope<T, true, (int)VEC><<<grid, ROPE_THREADS, smem, st>>>(a);
    else k_rope<T, false, (int)VEC><<<grid, ROPE_THREADS, smem, st>>>(a);
  } else {
    if (half) k_rope<T, true, 1><<<grid, ROPE_THREADS, smem, st>>>(a);
    else k_rope<T, false, 1><<<grid, ROPE_THREADS, smem, st>>>(a);
  }
  return kvcu_check_cuda(cudaGetLastError(), "rope launch");
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

extern "C" kvcu_rope* kvcu_rope_create(const kvcu_rope_desc* d) {
  if (!d) {
    kvcu_set_error("kvcu_rope_create: null description");
    return nullptr;
  }
  const double fast = d->beta_fast == 0.0 ? 32.0 : d->beta_fast, slow = d->beta_slow == 0.0 ? 1.0 : d->beta_slow;
  const bool scaled = d->scaling != KVCU_ROPE_NONE;
  const char* bad = nullptr;
  if (d->rot_dim < 2 || d->rot_dim % 2 || d->rot_dim > 2 * KVCU_ROPE_MAX_PAIRS) bad = "rot_dim";
  else if (d->layout > KVCU_ROPE_HALF) bad = "layout";
  else if (d->scaling > KVCU_ROPE_YARN) bad = "scaling";
  else if (!(d->base > 1.0) || !isfinite(d->base)) bad = "base";
  else if (scaled && (!(d->factor >= 1.0) || !isfinite(d->factor))) bad = "factor";
  else if (d->scaling == KVCU_ROPE_NTK && d->rot_dim < 4) bad = "rot_dim (NTK scaling needs two pairs)";
  else if (d->scaling == KVCU_ROPE_YARN && (!d->orig_ctx || !(slow > 0.0) || !(fast > slow) || !isfinite(fast)))
    bad = "orig_ctx / beta_fast / beta_slow";
  else if (!isfinite(d->mscale) || d->mscale < 0.0) bad = "mscale";
  if (bad) {
    kvcu_set_error("kvcu_rope_create: unsupported %s", bad);
    return nullptr;
  }
  kvcu_rope* r = new (std::nothrow) kvcu_rope();
  if (!r) {
    kvcu_set_error("kvcu_rope_create: out of memory");
    return nullptr;
  }
  const double pi = 3.14159265358979323846, dim = (double)d->rot_dim;
  r->rot = d->rot_dim;
  r->layout = d->layout;
  double base = d->base;
  if (d->scaling == KVCU_ROPE_NTK) base *= pow(d->factor, dim / (dim - 2.0));
  double low = 0.0, high = 0.0;
  if (d->scaling == KVCU_ROPE_YARN) {
    // the pair that makes `turns` full turns over the trained context; the ramp between the two is linear in
    // the pair's index, as the method's authors' code and the models trained with it have it (their paper
    // describes one over the number of turns)
    auto pair_of = [&](double turns) { return dim * log(d->orig_ctx / (turns * 2.0 * pi)) / (2.0 * log(base)); };
    low = fmax(floor(pair_of(fast)), 0.0);
    high = fmin(ceil(pair_of(slow)), dim - 1.0);
  }
  for (uint32_t i = 0; i < d->rot_dim / 2; ++i) {
    double f = pow(base, -2.0 * i / dim);
    if (d->scaling == KVCU_ROPE_LINEAR) f /= d->factor;
    if (d->scaling == KVCU_ROPE_YARN) {
      const double ramp = fmin(fmax((i - low) / fmax(high - low, 0.001), 0.0), 1.0);
      f = f / d->factor * ramp + f * (1.0 - ramp);
    }
    r->inv_freq[i] = f;
    r->turns[i] = f / (2.0 * pi);
  }
  r->mscale = d->mscale != 0.0 ? d->mscale : d->scaling == KVCU_ROPE_YARN ? 0.1 * log(d->factor) + 1.0 : 1.0;
  return r;
}

extern "C" int kvcu_rope_destroy(kvcu_rope* r) {
  delete r;
  return KVCU_OK;
}

extern "C" int kvcu_rope_frequencies(const kvcu_rope* r, double* inv_freq, double* mscale) {
  if (!r) return KVCU_ERR_INVALID_ARG;
  if (inv_freq)
    for (uint32_t i = 0; i < r->rot / 2; ++i) inv_freq[i] = r->inv_freq[i];
  if (mscale) *mscale = r->mscale;
  return KVCU_OK;
}

extern "C" int kvcu_rope_apply(const kvcu_rope* r, int device, int dtype, int transpose, uint32_t n,
                               const uint32_t* positions, const void* q, uint32_t q_heads, uint64_t q_row_stride,
                               uint64_t q_head_stride, void* q_out, uint64_t q_out_row_stride,
                               uint64_t q_out_head_stride, const void* k, uint32_t k_heads, uint64_t k_row_stride,
                               uint64_t k_head_stride, void* k_out, uint64_t k_out_row_stride,
                               uint64_t k_out_head_stride, void* stream) {
  if (!r || dtype < KVCU_DTYPE_F32 || dtype > KVCU_DTYPE_F16) {
    kvcu_set_error("kvcu_rope_apply: %s", r ? "unknown dtype" : "null rope");
    return KVCU_ERR_INVALID_ARG;
  }
  const uint64_t heads = (uint64_t)q_heads + k_heads;
  if (!n || !heads) return KVCU_OK;
  if (!positions || (q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out))) {
    kvcu_set_error("kvcu_rope_apply: null pointer argument");
    return KVCU_ERR_INVALID_ARG;
  }
  if (heads > ROPE_MAX_HEADS) {
    kvcu_set_error("kvcu_rope_apply: %llu heads, at most %u", (unsigned long long)heads, ROPE_MAX_HEADS);
    return KVCU_ERR_UNSUPPORTED;
  }
  if ((q_heads && !disjoint(n, q_heads, q_out_row_stride, q_out_head_stride, r->rot)) ||
      (k_heads && !disjoint(n, k_heads, k_out_row_stride, k_out_head_stride, r->rot))) {
    kvcu_set_error("kvcu_rope_apply: the output strides overlap");
    return KVCU_ERR_INVALID_ARG;
  }
  const uint64_t size = dtype == KVCU_DTYPE_F32 ? 4 : 2;
  if (((uint64_t)positions % 4) || (q_heads && (((uint64_t)q | (uint64_t)q_out) % size)) ||
      (k_heads && (((uint64_t)k | (uint64_t)k_out) % size))) {
    kvcu_set_error("kvcu_rope_apply: a pointer is not aligned to its type");
    return KVCU_ERR_INVALID_ARG;
  }
  DevScope d(device);
  if (d.rc) return d.rc;
  RopeArgs a = {};
  a.pos = positions;
  a.n = n;
  a.half = r->rot / 2;
  a.heads = (uint32_t)heads;
  a.div_heads = ((1ull << 32) + heads - 1) / heads;
  // up to 8 tokens a CTA, fewer while that leaves SMs without one
  const uint32_t per = n / (2u * (uint32_t)kvcu_current_sm_count());
  a.tokens = per < 1 ? 1 : per > ROPE_MAX_TOKENS ? ROPE_MAX_TOKENS : per;
  a.mscale = (float)r->mscale;
  a.sign = transpose ? -1.0f : 1.0f;
  a.t[0] = {q, q_out, q_row_stride, q_head_stride, q_out_row_stride, q_out_head_stride, q_heads};
  a.t[1] = {k, k_out, k_row_stride, k_head_stride, k_out_row_stride, k_out_head_stride, k_heads};
  for (uint32_t i = 0; i < a.half; ++i) a.turns[i] = r->turns[i];
  const bool half = r->layout == KVCU_ROPE_HALF;
  const cudaStream_t st = (cudaStream_t)stream;
  if (dtype == KVCU_DTYPE_F32) return launch<float>(a, half, st);
  if (dtype == KVCU_DTYPE_BF16) return launch<__nv_bfloat16>(a, half, st);
  return launch<__half>(a, half, st);
}
