// adamw.hip -- AdamW over many tensors in one launch, and the norm of all their gradients.
//
//   g' = s g;  m = b1 m + (1-b1) g';  v = b2 v + (1-b2) g'^2;  p = p (1 - lr wd) - lr/(1-b1^t) m / (sqrt(v)/sqrt(1-b2^t) + eps)
//
// Bound by memory: per value p in and out, g in, m and v in and out -- 28 bytes all in fp32, 10 with 16-bit p and g and
// 8-bit states.  The tensors are cut at create time into chunks whose records (addresses, length, decay) lie in device
// memory, so a workgroup reaches its data by ONE dependent load; a fixed grid walks over the records.  Measured: 201 M bf16 values with
// fp32 copies and states 1116 us (5.0 TB/s), with 8-bit states and no copies 437 us in a kernel trace, 450 - 540 from run to run of calls in a row (3.8 -
// 4.6 TB/s), their norm 70 us where nothing else runs (5.7 TB/s: of 403 MB the chip's last cache keeps a part), 92 - 117 in front of a step; a million
// values of 48 tensors in fp32 6.2 us, which is the chain record -> data -> store.  1280 or 4096 workgroups instead of at most 2048, and
// chunks of 16 passes instead of 4, take the same; chunks of one pass for 201 M values 1220 us.
//
// The update count t has to live on the device (a captured step is replayed) and every workgroup has to read it before any
// changes it.  Each workgroup therefore keeps a copy of its own, {t, b1^t, b2^t}, and advances that: no atomics, no second
// launch.  The products of the powers drift by t ulps of fp64.
//
// 8-bit states: blocks of 256 values = 32 lanes x 8 values, so a block's largest magnitude is a reduction over half a wave.
// It is a maximum of the bit patterns of |x|: a NaN is above all numbers there and reaches the scale, hence the whole block
// (r's codes have no NaN of their own).  What is rounded to 8 bits is the stored state alone; the update of p uses the
// unrounded m and v of this step.  Quotients and roots are the correctly rounded ones (the hardware's reciprocal would save 5 % there).
#include <algorithm>
#include <cmath>
#include <vector>

#include "op_common.h"

struct nerfhip_adamw : nh::OpHandle {};

namespace nh {
namespace {

thread_local std::string g_adamw_error;

constexpr int kThreads = 256;
constexpr int kVec = 8;                      // values per thread and pass
constexpr int kPass = kThreads * kVec;       // values per workgroup and pass (8 blocks of an 8-bit state)
// With 32-bit states a thread's values are two times 4 consecutive ones, kHalf apart: a wave then reads and writes whole lines of fp32 (100 M
// values in fp32 552 us, with 8 in a row 555; a million 7.2 and 7.9).  In 8 bits they are 8 in a row: a block of 256 is 32 lanes.
constexpr int kHalf = kPass / 2;
constexpr int kBlock = 256;
constexpr float kM8 = 448.0f, kR8 = 4032.0f;

struct Chunk {        // one record
  void* p;
  const void* g;
  float* master;
  void* m;
  void* v;
  float* ms;
  float* vs;
  int64_t at;         // where the chunk starts in read_state's buffers
  int32_t n;
  float wd;
};
struct Slot {         // one workgroup's copy of the update count and of the powers of the betas
  int64_t t;
  double b1t, b2t;
};

struct AdamW : nerfhip_adamw {
  nerfhip_adamw_config cfg;
  Chunk* chunks = nullptr;
  Slot* slots = nullptr;
  double* partial = nullptr;
  int32_t n_chunks = 0, grid = 0, norm_grid = 0;
};

struct Hyper {
  double b1, b2, lr;
  float fb1, gb1, fb2, gb2, eps;   // b and 1 - b, each rounded once
};

// The records' addresses are of global memory (not generic ones, whose accesses the compiler would have to order with LDS).
// Global memory takes vector accesses at any address, so a tensor may start anywhere its element may.
#define NH_GLOBAL __attribute__((address_space(1)))
template <class T, int N> struct Vals { typedef T t __attribute__((ext_vector_type(N), aligned(sizeof(T)))); };
typedef uint32_t Codes __attribute__((ext_vector_type(2), aligned(1)));

template <class T, bool FULL, int N> __device__ __forceinline__ void load_vals(const void* base, int at, int n, float (&x)[N]) {
  const NH_GLOBAL T* p = (const NH_GLOBAL T*)base + at;
  if (FULL || n >= N) {
    const typename Vals<T, N>::t a = *(const NH_GLOBAL typename Vals<T, N>::t*)p;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = (float)a[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = i < n ? (float)p[i] : 0.0f;
  }
}
template <class T, bool FULL, int N> __device__ __forceinline__ void store_vals(void* base, int at, int n, const float (&x)[N]) {
  NH_GLOBAL T* p = (NH_GLOBAL T*)base + at;
  if (FULL || n >= N) {
    typename Vals<T, N>::t a;
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] = (T)x[i];
    *(NH_GLOBAL typename Vals<T, N>::t*)p = a;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) if (i < n) p[i] = (T)x[i];
  }
}
// The values of a pass: 8 in a row (8-bit states), 4 in a row, or two times 4 kHalf apart, which are all there.
template <class T, int BITS, bool FULL, int V> __device__ __forceinline__ void load_pass(const void* base, int at, int n, float (&x)[V]) {
  if constexpr (BITS == 8 || V == 4) {
    load_vals<T, FULL>(base, at, n, x);
  } else {
    static_assert(FULL && V == 8, "");
    float a[4], b[4];
    load_vals<T, true>(base, at, 4, a);
    load_vals<T, true>(base, at + kHalf, 4, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[i] = a[i]; x[4 + i] = b[i]; }
  }
}
template <class T, int BITS, bool FULL, int V> __device__ __forceinline__ void store_pass(void* base, int at, int n, const float (&x)[V]) {
  if constexpr (BITS == 8 || V == 4) {
    store_vals<T, FULL>(base, at, n, x);
  } else {
    const float a[4] = {x[0], x[1], x[2], x[3]}, b[4] = {x[4], x[5], x[6], x[7]};
    store_vals<T, true>(base, at, 4, a);
    store_vals<T, true>(base, at + kHalf, 4, b);
  }
}
template <bool FULL> __device__ __forceinline__ Codes load_codes(const void* base, int at, int n) {
  const NH_GLOBAL uint8_t* p = (const NH_GLOBAL uint8_t*)base + at;
  if (FULL || n >= 8) return *(const NH_GLOBAL Codes*)p;
  Codes c = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) if (i < n) c[i >> 2] |= (uint32_t)p[i] << (8 * (i & 3));
  return c;
}
template <bool FULL> __device__ __forceinline__ void store_codes(void* base, int at, int n, Codes c) {
  NH_GLOBAL uint8_t* p = (NH_GLOBAL uint8_t*)base + at;
  if (FULL || n >= 8) { *(NH_GLOBAL Codes*)p = c; return; }
#pragma unroll
  for (int i = 0; i < 8; ++i) if (i < n) p[i] = (uint8_t)(c[i >> 2] >> (8 * (i & 3)));
}

__device__ __forceinline__ float root_value(uint32_t c) {   // code of sqrt(v) -> 0 .. 4032
  const float low = (float)c, high = __builtin_bit_cast(float, (c + (131u << 5)) << 18);
  return c < 32 ? low : high;
}
__device__ __forceinline__ uint32_t root_code(float q) {    // 0 .. 4032 -> nearest code, ties to even; q > 0 never gives 0
  const uint32_t b = __builtin_bit_cast(uint32_t, q);
  const uint32_t high = ((b + 0x1ffffu + ((b >> 18) & 1u)) >> 18) - (131u << 5);
  const uint32_t low = __builtin_bit_cast(uint32_t, q + 8388608.0f) & 0xffu;   // codes are one apart up to 64: the sum rounds to whole numbers
  return max(q < 64.0f ? low : high, min(b, 1u));
}
template <int CTRL> __device__ __forceinline__ uint32_t dpp_max(uint32_t b) {
  return max(b, (uint32_t)__builtin_amdgcn_update_dpp((int)b, (int)b, CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float half_wave_max(uint32_t b) {   // of the 32 lanes that hold one block: rotations within 16 lanes, one exchange
  b = dpp_max<0x121>(b);
  b = dpp_max<0x122>(b);
  b = dpp_max<0x124>(b);
  b = dpp_max<0x128>(b);
  b = max(b, (uint32_t)__shfl_xor((int)b, 16, 64));
  return __builtin_bit_cast(float, b);
}
__device__ __forceinline__ float block_scale(const float (&x)[8], float top_inv) {
  uint32_t b = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) b = max(b, __builtin_bit_cast(uint32_t, x[i]) & 0x7fffffffu);
  const float s = half_wave_max(b) * top_inv;
  return s < 1.17549435e-38f ? 1.17549435e-38f : s;            // an empty block: codes 0, and 1/scale stays finite
}

// m, and v (32 bits) or sqrt(v) (8 bits)
template <int BITS, bool FULL, int V> __device__ __forceinline__ void load_m(const Chunk& k, int at, int n, float (&m)[V]) {
  if constexpr (BITS == 32) {
    load_pass<float, BITS, FULL>(k.m, at, n, m);
  } else {
    const Codes c = load_codes<FULL>(k.m, at, n);
    const float s = FULL || n > 0 ? ((const NH_GLOBAL float*)k.ms)[at / kBlock] : 0.0f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[h], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[h], true);
      m[4 * h] = lo[0] * s; m[4 * h + 1] = lo[1] * s; m[4 * h + 2] = hi[0] * s; m[4 * h + 3] = hi[1] * s;
    }
  }
}
template <int BITS, bool FULL, int V> __device__ __forceinline__ void load_v(const Chunk& k, int at, int n, float (&v)[V]) {
  if constexpr (BITS == 32) {
    load_pass<float, BITS, FULL>(k.v, at, n, v);
  } else {
    const Codes c = load_codes<FULL>(k.v, at, n);
    const float s = FULL || n > 0 ? ((const NH_GLOBAL float*)k.vs)[at / kBlock] : 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = root_value((c[i >> 2] >> (8 * (i & 3))) & 255u) * s;
  }
}

// What a step has in common: read behind the first loads of values, so that the two waits overlap.
struct Common {
  Slot next;
  double lr;
  float gs, step, rs2;
  bool ready, skip;
};
__device__ __forceinline__ void read_common(Common& f, const Slot* slots, const Hyper& hp, const float* lr_dev, const float* grad_scale) {
  if (f.ready) return;
  f.ready = true;
  f.gs = grad_scale ? *grad_scale : 1.0f;
  f.skip = !(__builtin_fabsf(f.gs) < __builtin_inff());        // every workgroup alike: no slot moves
  f.next = slots[blockIdx.x];
  f.next.t += 1;
  f.next.b1t *= hp.b1;
  f.next.b2t *= hp.b2;
  f.lr = lr_dev ? (double)*lr_dev : hp.lr;
  f.step = (float)(f.lr / (1.0 - f.next.b1t));
  f.rs2 = (float)(1.0 / sqrt(1.0 - f.next.b2t));
}

// One pass of V values a thread.  FULL: all of the workgroup's exist; else each thread has n of its V (n may be <= 0).
template <class P, class G, int BITS, bool MASTER, bool FULL, int V, class Read>
__device__ __forceinline__ void update(const Chunk& k, int at, int n, const Hyper& hp, Common& f, const Read& read) {
  float p[V], g[V], m[V], v[V], r[V];
  load_pass<G, BITS, FULL>(k.g, at, n, g);
  if (MASTER) load_pass<float, BITS, FULL>(k.master, at, n, p);
  else load_pass<P, BITS, FULL>(k.p, at, n, p);
  load_m<BITS, FULL>(k, at, n, m);
  load_v<BITS, FULL>(k, at, n, v);
  read();
  if (f.skip) return;
  const float keep = (float)(1.0 - f.lr * (double)k.wd);
  if (BITS == 8)
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = v[i] * v[i];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float gi = g[i] * f.gs;
    m[i] = m[i] * hp.fb1 + gi * hp.gb1;
    v[i] = v[i] * hp.fb2 + (gi * gi) * hp.gb2;
    r[i] = __builtin_sqrtf(v[i]);
    p[i] = p[i] * keep - f.step * (m[i] / (r[i] * f.rs2 + hp.eps));
  }
  if (MASTER) store_pass<float, BITS, FULL>(k.master, at, n, p);
  store_pass<P, BITS, FULL>(k.p, at, n, p);
  if constexpr (BITS == 32) {
    store_pass<float, BITS, FULL>(k.m, at, n, m);
    store_pass<float, BITS, FULL>(k.v, at, n, v);
  } else {
    const float sm = block_scale(m, 1.0f / kM8), sr = block_scale(r, 1.0f / kR8);
    const float im = 1.0f / sm, ir = 1.0f / sr;
    Codes cm = {0, 0}, cr = {0, 0};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int w = __builtin_amdgcn_cvt_pk_fp8_f32(m[4 * h] * im, m[4 * h + 1] * im, 0, false);
      cm[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(m[4 * h + 2] * im, m[4 * h + 3] * im, w, true);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) cr[i >> 2] |= root_code(r[i] * ir) << (8 * (i & 3));
    if (FULL || n > 0) {
      store_codes<FULL>(k.m, at, n, cm);
      store_codes<FULL>(k.v, at, n, cr);
      if ((threadIdx.x & 31) == 0) {
        ((NH_GLOBAL float*)k.ms)[at / kBlock] = sm;
        ((NH_GLOBAL float*)k.vs)[at / kBlock] = sr;
      }
    }
  }
}

template <class P, class G, int BITS, bool MASTER>
__global__ __launch_bounds__(kThreads) void adamw_kernel(const Chunk* __restrict__ chunks, int n_chunks, Slot* __restrict__ slots,
                                                         Hyper hp, const float* __restrict__ lr_dev,
                                                         const float* __restrict__ grad_scale) {
  Common f = {};
  auto read = [&] { read_common(f, slots, hp, lr_dev, grad_scale); };
  for (int c = blockIdx.x; c < n_chunks && !f.skip; c += gridDim.x) {
    const Chunk k = chunks[c];
    if constexpr (BITS == 8) {
      for (int base = 0; base < k.n; base += kPass) {
        const int at = base + (int)threadIdx.x * kVec;
        if (base + kPass <= k.n) update<P, G, 8, MASTER, true, kVec>(k, at, kVec, hp, f, read);
        else update<P, G, 8, MASTER, false, kVec>(k, at, k.n - at, hp, f, read);
      }
    } else {
      int at = (int)threadIdx.x * (kVec / 2), left = k.n;
      for (; left >= kPass; left -= kPass, at += kPass) update<P, G, 32, MASTER, true, kVec>(k, at, 4, hp, f, read);
      for (; left >= kHalf; left -= kHalf, at += kHalf) update<P, G, 32, MASTER, true, kVec / 2>(k, at, 4, hp, f, read);
      if (left > 0) update<P, G, 32, MASTER, false, kVec / 2>(k, at, k.n - at, hp, f, read);
    }
  }
  read();
  __syncthreads();                                             // all waves have read the slot
  if (threadIdx.x == 0 && !f.skip) slots[blockIdx.x] = f.next;
}

__device__ __forceinline__ double block_sum(double x, double* part) {   // of a workgroup's threads, in a fixed order; thread 0's
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
  __syncthreads();
  double s = 0.0;
  if (threadIdx.x == 0)
    for (int w = 0; w < (int)blockDim.x / 64; ++w) s += part[w];
  return s;
}

// Squares in fp64: those of fp32 or bf16 gradients pass fp32's range, and 2^28 of them its precision.
template <class G>
__global__ __launch_bounds__(kThreads) void norm_kernel(const Chunk* __restrict__ chunks, int n_chunks, double* __restrict__ partial) {
  constexpr int kWide = 16 / sizeof(G);      // whole lines
  __shared__ double part[kThreads / 64];
  double s = 0.0;
  for (int c = blockIdx.x; c < n_chunks; c += gridDim.x) {
    const void* g = chunks[c].g;
    const int len = chunks[c].n;
    for (int at = (int)threadIdx.x * kWide; at < len; at += kThreads * kWide) {
      float x[kWide];
      load_vals<G, false>(g, at, len - at, x);
#pragma unroll
      for (int i = 0; i < kWide; ++i) s = fma((double)x[i], (double)x[i], s);
    }
  }
  s = block_sum(s, part);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__global__ __launch_bounds__(kThreads) void norm_final_kernel(const double* __restrict__ partial, int n, double max_norm,
                                                              double inv_scale, float* __restrict__ out) {
  __shared__ double part[kThreads / 64];
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += kThreads) s += partial[i];
  s = block_sum(s, part);
  if (threadIdx.x == 0) {
    const double norm = sqrt(s) * inv_scale;
    double f = 1.0;
    if (max_norm > 0.0 && max_norm < norm + 1e-6) f = max_norm / (norm + 1e-6);
    out[0] = (float)norm;
    out[1] = norm < __builtin_inf() ? (float)(f * inv_scale) : __builtin_nanf("");
  }
}

// Four values of every thread and pass, so that a wave stores whole lines; between a tensor's end and the next multiple of 256 zeros are written.
typedef float Four __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t FourCodes __attribute__((aligned(1)));
template <int BITS, bool ROOT> __device__ __forceinline__ void read_state(const void* state, const float* scale, int len, float* out) {
  const int padded = (len + kBlock - 1) / kBlock * kBlock;
  for (int at = (int)threadIdx.x * 4; at < padded; at += kThreads * 4) {
    const int n = len - at;
    Four x = {0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (BITS == 32) {
      const NH_GLOBAL float* const p = (const NH_GLOBAL float*)state + at;
      if (n >= 4) x = *(const NH_GLOBAL Four*)p;
      else
#pragma unroll
        for (int i = 0; i < 4; ++i) if (i < n) x[i] = p[i];
      if (ROOT)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __builtin_sqrtf(x[i]);
    } else if (n > 0) {
      const NH_GLOBAL uint8_t* const p = (const NH_GLOBAL uint8_t*)state + at;
      uint32_t c = 0;
      if (n >= 4) c = *(const NH_GLOBAL FourCodes*)p;
      else
#pragma unroll
        for (int i = 0; i < 4; ++i) if (i < n) c |= (uint32_t)p[i] << (8 * i);
      const float s = ((const NH_GLOBAL float*)scale)[at / kBlock];
      if (ROOT) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = root_value((c >> (8 * i)) & 255u) * s;
      } else {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
        x[0] = lo[0] * s; x[1] = lo[1] * s; x[2] = hi[0] * s; x[3] = hi[1] * s;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) if (i >= n) x[i] = 0.0f;
    }
    *(NH_GLOBAL Four*)((NH_GLOBAL float*)out + at) = x;
  }
}
template <int BITS>
__global__ __launch_bounds__(kThreads) void read_state_kernel(const Chunk* __restrict__ chunks, int n_chunks, float* __restrict__ m_out,
                                                              float* __restrict__ r_out) {
  for (int c = blockIdx.x; c < n_chunks; c += gridDim.x) {
    const Chunk k = chunks[c];
    if (m_out) read_state<BITS, false>(k.m, k.ms, k.n, m_out + k.at);
    if (r_out) read_state<BITS, true>(k.v, k.vs, k.n, r_out + k.at);
  }
}

__global__ void set_slots_kernel(Slot* slots, int n, Slot s) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n) slots[i] = s;
}

template <class P, class G, int BITS, bool MASTER> hipError_t launch_step(AdamW* a, const Hyper& hp, const float* lr_dev, const float* gs) {
  hipLaunchKernelGGL((adamw_kernel<P, G, BITS, MASTER>), dim3(a->grid), dim3(kThreads), 0, a->stream, a->chunks, a->n_chunks, a->slots, hp,
                     lr_dev, gs);
  return hipGetLastError();
}
template <class P, class G> hipError_t launch_types(AdamW* a, const Hyper& hp, const float* lr_dev, const float* gs) {
  if (a->cfg.master)
    return a->cfg.state_bits == 8 ? launch_step<P, G, 8, true>(a, hp, lr_dev, gs) : launch_step<P, G, 32, true>(a, hp, lr_dev, gs);
  return a->cfg.state_bits == 8 ? launch_step<P, G, 8, false>(a, hp, lr_dev, gs) : launch_step<P, G, 32, false>(a, hp, lr_dev, gs);
}
hipError_t launch_any(AdamW* a, const Hyper& hp, const float* lr_dev, const float* gs) {
  const bool wide = a->cfg.grad_dtype == NERFHIP_F32;
  if (a->cfg.param_dtype == NERFHIP_F32)
    return a->cfg.state_bits == 8 ? launch_step<float, float, 8, false>(a, hp, lr_dev, gs)
                                  : launch_step<float, float, 32, false>(a, hp, lr_dev, gs);
  if (a->cfg.param_dtype == NERFHIP_BF16)
    return wide ? launch_types<__bf16, float>(a, hp, lr_dev, gs) : launch_types<__bf16, __bf16>(a, hp, lr_dev, gs);
  return wide ? launch_types<_Float16, float>(a, hp, lr_dev, gs) : launch_types<_Float16, _Float16>(a, hp, lr_dev, gs);
}

int bad(AdamW* a, const char* msg) { return op_fail(a, g_adamw_error, NERFHIP_E_INVALID, msg); }

hipError_t write_step(AdamW* a, int64_t t) {
  const Slot s{t, std::pow(a->cfg.beta1, (double)t), std::pow(a->cfg.beta2, (double)t)};
  hipLaunchKernelGGL(set_slots_kernel, dim3((a->grid + 255) / 256), dim3(256), 0, a->stream, a->slots, a->grid, s);
  return hipGetLastError();
}

int create(const nerfhip_adamw_config& c, const nerfhip_adamw_tensor* t, int64_t count, AdamW* a) {
  if (!(c.beta1 >= 0.0 && c.beta1 < 1.0 && c.beta2 >= 0.0 && c.beta2 < 1.0)) return bad(nullptr, "beta1 and beta2 must be in [0, 1)");
  if (!(c.eps >= 0.0 && c.eps < 1e30)) return bad(nullptr, "eps must be >= 0 and finite");
  if (!dtype_ok(c.param_dtype)) return bad(nullptr, "param_dtype must be F32, BF16 or F16");
  if (c.grad_dtype != c.param_dtype && c.grad_dtype != NERFHIP_F32) return bad(nullptr, "grad_dtype must be param_dtype or F32");
  if (c.state_bits != 8 && c.state_bits != 32) return bad(nullptr, "state_bits must be 8 or 32");
  if (c.master != 0 && c.master != 1) return bad(nullptr, "master must be 0 or 1");
  if (c.master && c.param_dtype == NERFHIP_F32) return bad(nullptr, "master copies are for 16-bit parameters");
  if (c.reserved[0] || c.reserved[1]) return bad(nullptr, "reserved fields must be 0");
  if (count < 0 || (count > 0 && !t)) return bad(nullptr, "null tensor table or negative count");
  const size_t pb = dtype_bytes(c.param_dtype), gb = dtype_bytes(c.grad_dtype), sb = c.state_bits == 8 ? 1 : 4;
  int64_t total = 0;
  for (int64_t i = 0; i < count; ++i) {
    const nerfhip_adamw_tensor& x = t[i];
    if (x.n < 0 || x.n > (int64_t)1 << 40) return bad(nullptr, "a tensor's n must be in [0, 2^40]");
    if (!(x.weight_decay >= 0.0f && x.weight_decay < 1e30f)) return bad(nullptr, "weight_decay must be >= 0 and finite");
    if (x.reserved != 0.0f) return bad(nullptr, "reserved fields must be 0");
    if (x.n == 0) continue;
    if (!x.param || !x.grad || !x.m || !x.v) return bad(nullptr, "a tensor has a null pointer");
    if ((c.master != 0) != (x.master != nullptr)) return bad(nullptr, "master pointers go with config.master");
    if ((c.state_bits == 8) != (x.m_scale != nullptr) || (c.state_bits == 8) != (x.v_scale != nullptr))
      return bad(nullptr, "m_scale and v_scale go with state_bits 8");
    if ((uintptr_t)x.param % pb || (uintptr_t)x.grad % gb || (uintptr_t)x.master % 4 || (uintptr_t)x.m % sb || (uintptr_t)x.v % sb ||
        (uintptr_t)x.m_scale % 4 || (uintptr_t)x.v_scale % 4)
      return bad(nullptr, "a pointer is not aligned to its element");
    total += x.n;
    if (total > (int64_t)1 << 40) return bad(nullptr, "more than 2^40 values in all");
  }
  struct Piece { uintptr_t lo, hi; bool written; };
  std::vector<Piece> mem;
  for (int64_t i = 0; i < count; ++i) {
    const nerfhip_adamw_tensor& x = t[i];
    auto add = [&](const void* p, int64_t n, size_t bytes, bool written) {
      if (p && n > 0) mem.push_back({(uintptr_t)p, (uintptr_t)p + (uintptr_t)n * bytes, written});
    };
    const int64_t nb = (x.n + kBlock - 1) / kBlock;
    add(x.param, x.n, pb, true);
    add(x.grad, x.n, gb, false);
    add(x.master, x.n, 4, true);
    add(x.m, x.n, sb, true);
    add(x.v, x.n, sb, true);
    add(x.m_scale, nb, 4, true);
    add(x.v_scale, nb, 4, true);
  }
  std::sort(mem.begin(), mem.end(), [](const Piece& a, const Piece& b) { return a.lo < b.lo; });
  uintptr_t end_all = 0, end_written = 0;      // of what starts before
  for (const Piece& p : mem) {
    if (p.lo < end_written || (p.written && p.lo < end_all)) return bad(nullptr, "tensors overlap");
    if (p.hi > end_all) end_all = p.hi;
    if (p.written && p.hi > end_written) end_written = p.hi;
  }
  if (!op_device_ok(c.device)) return op_fail(nullptr, g_adamw_error, NERFHIP_E_HIP, "no such HIP device (libnerfhip has no CPU path)");
  // A chunk is one pass of a workgroup while that fills the chip (256 CUs x 8 workgroups), four where there are more values
  // than that: a quarter of the records to read.  Few values with 32-bit states: half a pass, one load a thread and tensor (a million
  // values in fp32 6.2 us, whole passes 7.2).
  const int64_t fill = 256 * 8, chunk = total > kPass * fill * 4 ? 4 * kPass : c.state_bits == 32 && total <= kHalf * fill ? kHalf : kPass;
  std::vector<Chunk> rec;
  int64_t start = 0;
  for (int64_t i = 0; i < count; ++i) {
    const nerfhip_adamw_tensor& x = t[i];
    for (int64_t at = 0; at < x.n; at += chunk) {
      Chunk k;
      k.p = (char*)x.param + at * (int64_t)pb;
      k.g = (const char*)x.grad + at * (int64_t)gb;
      k.master = x.master ? x.master + at : nullptr;
      k.m = (char*)x.m + at * (int64_t)sb;
      k.v = (char*)x.v + at * (int64_t)sb;
      k.ms = x.m_scale ? x.m_scale + at / kBlock : nullptr;
      k.vs = x.v_scale ? x.v_scale + at / kBlock : nullptr;
      k.at = start + at;
      k.n = (int32_t)(x.n - at < chunk ? x.n - at : chunk);
      k.wd = x.weight_decay;
      rec.push_back(k);
    }
    start += (x.n + kBlock - 1) / kBlock * kBlock;
  }
  a->cfg = c;
  a->device = c.device;
  a->n_chunks = (int32_t)rec.size();
  a->grid = a->n_chunks < 2048 ? (a->n_chunks > 0 ? a->n_chunks : 1) : 2048;
  a->norm_grid = a->grid;
  DeviceScope dev(c.device);
  if (!dev.ok) return op_fail(nullptr, g_adamw_error, NERFHIP_E_HIP, "hipSetDevice failed");
  hipError_t e;
#define ACHK(expr) do { if ((e = (expr)) != hipSuccess) return op_fail_hip(nullptr, g_adamw_error, e, #expr); } while (0)
  ACHK(hipStreamCreateWithFlags(&a->own_stream, hipStreamNonBlocking));
  a->stream = a->own_stream;
  ACHK(hipMalloc((void**)&a->chunks, (rec.empty() ? 1 : rec.size()) * sizeof(Chunk)));
  ACHK(hipMalloc((void**)&a->slots, (size_t)a->grid * sizeof(Slot)));
  ACHK(hipMalloc((void**)&a->partial, (size_t)a->norm_grid * sizeof(double)));
  if (!rec.empty()) ACHK(hipMemcpy(a->chunks, rec.data(), rec.size() * sizeof(Chunk), hipMemcpyHostToDevice));
  ACHK(write_step(a, 0));
  ACHK(hipStreamSynchronize(a->stream));
#undef ACHK
  return NERFHIP_OK;
}

void destroy(AdamW* a) {
  DeviceScope dev(a->device);
  if (a->own_stream) { (void)hipStreamSynchronize(a->own_stream); (void)hipStreamDestroy(a->own_stream); }
  (void)hipFree(a->chunks);     // waits for kernels that still use it, on whichever stream
  (void)hipFree(a->slots);
  (void)hipFree(a->partial);
  delete a;
}

}  // namespace
}  // namespace nh

using namespace nh;

// Runs `body` on the handle's device; no C++ exception crosses the C boundary.
#define ADAMW_ENTRY(h)                                                                                              \
  if (!(h)) return op_fail(nullptr, g_adamw_error, NERFHIP_E_INVALID, "null handle");                               \
  AdamW* const a = static_cast<AdamW*>(h);                                                                          \
  DeviceScope dev_(a->device);                                                                                      \
  if (!dev_.ok) return op_fail(a, g_adamw_error, NERFHIP_E_HIP, "hipSetDevice failed");

extern "C" {

int nerfhip_adamw_create(const nerfhip_adamw_config* cfg, const nerfhip_adamw_tensor* tensors, int64_t count, nerfhip_adamw_t** out) {
  if (!cfg || !out) return op_fail(nullptr, g_adamw_error, NERFHIP_E_INVALID, "null argument");
  *out = nullptr;
  AdamW* a = nullptr;
  try {
    a = new AdamW();
    const int rc = create(*cfg, tensors, count, a);
    if (rc != NERFHIP_OK) { destroy(a); return rc; }
    *out = a;
    return NERFHIP_OK;
  } catch (const std::bad_alloc&) {
    if (a) destroy(a);
    return op_fail(nullptr, g_adamw_error, NERFHIP_E_NOMEM, "out of host memory");
  }
}

void nerfhip_adamw_destroy(nerfhip_adamw_t* h) { if (h) destroy(static_cast<AdamW*>(h)); }

const char* nerfhip_adamw_last_error(const nerfhip_adamw_t* h) { return h ? h->err.c_str() : g_adamw_error.c_str(); }

int nerfhip_adamw_set_stream(nerfhip_adamw_t* h, void* hip_stream) {
  if (!h) return op_fail(nullptr, g_adamw_error, NERFHIP_E_INVALID, "null handle");
  h->stream = op_stream(h, hip_stream);
  return NERFHIP_OK;
}

int nerfhip_adamw_synchronize(nerfhip_adamw_t* h) {
  ADAMW_ENTRY(h)
  const hipError_t e = hipStreamSynchronize(a->stream);
  return e == hipSuccess ? NERFHIP_OK : op_fail_hip(a, g_adamw_error, e, "hipStreamSynchronize");
}

int nerfhip_adamw_step(nerfhip_adamw_t* h, double lr, const float* lr_dev, const float* grad_scale) {
  ADAMW_ENTRY(h)
  if (!lr_dev && !(std::fabs(lr) < 1e30)) return bad(a, "lr must be finite");
  if ((uintptr_t)lr_dev % 4 || (uintptr_t)grad_scale % 4) return bad(a, "a pointer is not aligned to its element");
  const nerfhip_adamw_config& c = a->cfg;
  const Hyper hp{c.beta1, c.beta2, lr, (float)c.beta1, (float)(1.0 - c.beta1), (float)c.beta2, (float)(1.0 - c.beta2), (float)c.eps};
  const hipError_t e = launch_any(a, hp, lr_dev, grad_scale);
  return e == hipSuccess ? NERFHIP_OK : op_fail_hip(a, g_adamw_error, e, "adamw kernel");
}

int nerfhip_adamw_grad_norm(nerfhip_adamw_t* h, double max_norm, double loss_scale, float* out) {
  ADAMW_ENTRY(h)
  if (!out) return bad(a, "null argument");
  if ((uintptr_t)out % 4) return bad(a, "a pointer is not aligned to its element");
  if (!(max_norm >= 0.0 && max_norm < 1e300)) return bad(a, "max_norm must be >= 0 and finite");
  // 1 / loss_scale is a factor in fp32: past its range it would clear or skip every update
  if (!(loss_scale >= 1e-30 && loss_scale <= 1e30)) return bad(a, "loss_scale must be in [1e-30, 1e30]");
  const dim3 grid(a->norm_grid), block(kThreads);
  if (a->cfg.grad_dtype == NERFHIP_F32) hipLaunchKernelGGL((norm_kernel<float>), grid, block, 0, a->stream, a->chunks, a->n_chunks, a->partial);
  else if (a->cfg.grad_dtype == NERFHIP_BF16) hipLaunchKernelGGL((norm_kernel<__bf16>), grid, block, 0, a->stream, a->chunks, a->n_chunks, a->partial);
  else hipLaunchKernelGGL((norm_kernel<_Float16>), grid, block, 0, a->stream, a->chunks, a->n_chunks, a->partial);
  hipLaunchKernelGGL(norm_final_kernel, dim3(1), block, 0, a->stream, a->partial, a->norm_grid, max_norm, 1.0 / loss_scale, out);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? NERFHIP_OK : op_fail_hip(a, g_adamw_error, e, "gradient norm kernels");
}

int nerfhip_adamw_read_state(nerfhip_adamw_t* h, float* m, float* root) {
  ADAMW_ENTRY(h)
  if ((uintptr_t)m % 4 || (uintptr_t)root % 4) return bad(a, "a pointer is not aligned to its element");
  if (!m && !root) return NERFHIP_OK;
  const dim3 grid(a->grid), block(kThreads);
  if (a->cfg.state_bits == 8) hipLaunchKernelGGL((read_state_kernel<8>), grid, block, 0, a->stream, a->chunks, a->n_chunks, m, root);
  else hipLaunchKernelGGL((read_state_kernel<32>), grid, block, 0, a->stream, a->chunks, a->n_chunks, m, root);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? NERFHIP_OK : op_fail_hip(a, g_adamw_error, e, "read_state kernel");
}

int nerfhip_adamw_get_step(nerfhip_adamw_t* h, int64_t* step) {
  ADAMW_ENTRY(h)
  if (!step) return bad(a, "null argument");
  Slot s;
  hipError_t e = hipMemcpyAsync(&s, a->slots, sizeof(s), hipMemcpyDeviceToHost, a->stream);
  if (e == hipSuccess) e = hipStreamSynchronize(a->stream);
  if (e != hipSuccess) return op_fail_hip(a, g_adamw_error, e, "get_step");
  *step = s.t;
  return NERFHIP_OK;
}

int nerfhip_adamw_set_step(nerfhip_adamw_t* h, int64_t step) {
  ADAMW_ENTRY(h)
  if (step < 0) return bad(a, "step must be >= 0");
  hipError_t e = write_step(a, step);
  if (e == hipSuccess) e = hipStreamSynchronize(a->stream);
  return e == hipSuccess ? NERFHIP_OK : op_fail_hip(a, g_adamw_error, e, "set_step");
}

}  // extern "C"
