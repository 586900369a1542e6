// ffn.hip -- the gated feed-forward block: entry points, the plan of launches, and the kernels beside the matrix product
// (ffn_gemm.hip.h): few rows, operand copies, column sums, sums over splits.
//
//   forward    g = x Wg^T + bg, u = x Wu^T + bu, h = a(g) u   one product with d_ff gate and d_ff up columns
//              y = h Wd^T + bd
//   backward   dh = dy Wd                                     fp32, to scratch
//              g, u again; h, dg = dh u a'(g), du = dh a(g)    one product, and the column sums for the biases
//              dx = dg Wg + du Wu                              one product of two segments
//              dWg = dg^T x, dWu = du^T x, dWd = dy^T h
// 16 rows d_model d_ff flop in the backward pass, 4 of them for g and u again: keeping them would cost 2 d_ff values a row from the
// forward to the backward pass, and in 16 bits a rounding more in every gradient.
//
// Roundings to 16 bits (16-bit tensors): h before the second product (of more than 16 rows), dg and du before theirs.  The matrix cores take
// no more, and each adds about what the final rounding of the result does.  dh, g and u stay in fp32.
#include "ffn_gemm.hip.h"

struct nerfhip_ffn : nh::OpHandle {
  nerfhip_ffn_config cfg;
  int n_cu = 256;
};

namespace nh {
namespace {

thread_local std::string g_ffn_error;

// Rows that a pass over the weights takes along, in blocks of 16: up to `few_rows`, and of large weights in 16 bits up to 16.  Here and in tiles
// (us): 20 rows of 1024 -> 4096 in bf16 19 and 23, of 2048 -> 8192 35 and 32; 32 rows 21 and 22, 42 and 32.  In fp32, where tiles need the
// weights in pieces, 64 rows of 1024 -> 4096 59 and 65, of 4096 -> 4096 105 and 210.
constexpr int few_rows(int dtype) { return dtype == NERFHIP_F32 ? 64 : 32; }
bool take_few(const nerfhip_ffn_config& f, int64_t rows) {
  return rows <= 16 || (rows <= few_rows(f.dtype) && (f.dtype == NERFHIP_F32 || (int64_t)f.d_model * f.d_ff < (int64_t)1 << 24));
}

template <class V> __device__ __forceinline__ V load_any(const void* p) {
  V v;
  __builtin_memcpy(&v, p, sizeof(V));
  return v;
}

// ---- few rows: the weights are read once, straight into registers ------------------------------------------------------
// One workgroup: 16 output columns (GATE: of both weights), its NW waves take every NW-th piece of kUnroll x 64 bytes of k; lane (c, g)
// reads 16 bytes of weight row c, k chunk g, which is what the matrix instruction wants.  Bound by the weights' bytes: 8 rows of
// 4096 -> 2 x 16384 -> 4096 in bf16, 403 MB, take 86 us, 50 and 36.
// Where 16 columns each would leave CUs without a workgroup and rows are few, P parts of k take the place of rows and columns: row c of both
// operands is row or column c % (16 / P) of part c / (16 / P), and of the products the P squares on the diagonal count.  One row of
// 4096 -> 1024: 4.5 us with four parts, 8.1 with one; past one workgroup to a CU they lose (2 rows of 4096 -> 4096: 8.5 us with one, 9.0
// with two, 10.3 with four).
// The workgroups start at different k: weight rows lie a power of two apart as a rule, and at the same k all of them would read from the same
// few memory channels (8 rows as above 92 us, one row in f16 87 instead of 79).
// k is cut among the waves of one workgroup only: a cut among workgroups, the last of which adds the parts up, spent four times as
// long on the fences between the chip's caches as on 8 MB of weights.
struct FewArgs {
  const void* x;
  int64_t ldx;
  const void *w, *w2;
  int64_t ldw, ldw2;
  const void *b, *b2;
  int32_t rows, N, K;
  int32_t act;
  void* out;              // GATE: h [rows][ldo] in fp32, or two pieces of it one behind the other; else y
  int64_t ldo;
};

template <class T> __device__ __forceinline__ s16x8 load_k(const T* p, int k, int K) {   // 16 bytes of a row; zeros past K
  constexpr int kN = 16 / sizeof(T);
  if (k + kN <= K) return load_any<s16x8>(p + k);
  T v[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i) v[i] = k + i < K ? p[k + i] : (T)0.0f;
  return __builtin_bit_cast(s16x8, v);
}
template <int DT> __device__ __forceinline__ f32x4 mma_few(s16x8 a, s16x8 b, f32x4 c) {
  if constexpr (DT == NERFHIP_F32) {   // k = 4 g + t in instruction t, for both operands alike
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int t = 0; t < 4; ++t) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[t], y[t], c, 0, 0, 0);
    return c;
  } else {
    return mma<DT>(a, b, c);
  }
}

// Up to 16 rows of 16-bit tensors h goes to the second product as two pieces: 16 bits more than it has as one.  Beyond, one piece: it is read
// by every workgroup, and 32 rows of 8192 -> 2048 took 37 us with two and 24 with one.
constexpr bool few_pieces(int dtype, int blocks) { return dtype != NERFHIP_F32 && blocks == 1; }
template <class T> __device__ __forceinline__ void split2(float v, T& hi, T& lo) {
  hi = (T)v;
  const float rest = v - (float)hi;
  lo = (T)(__builtin_fabsf(rest) < __builtin_inff() ? rest : 0.0f);      // v past the type's range: hi is infinite as it should be
}

// RB: blocks of 16 rows; P: parts of k side by side
template <int DT, bool GATE, int NW, int RB, int kUnroll, int P> __global__ __launch_bounds__(NW * 64) void few_rows_kernel(const FewArgs fa) {
  typedef typename OpType<DT>::t T;
  constexpr bool kPieces = few_pieces(DT, RB) && !GATE;
  constexpr int kStep = 64 / sizeof(T), kCols = 16 / P;
  static_assert(P == 1 || RB == 1, "parts take the place of rows");
  __shared__ float red[GATE ? 2 : 1][NW][256];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, g = lane >> 4;
  const int one = c % kCols, part = c / kCols;
  const int n = (int)blockIdx.x * kCols + one;
  const bool n_ok = n < fa.N;
  // rows and columns past the end read others, whose sums nobody stores
  const T* const w = (const T*)fa.w + (int64_t)(n_ok ? n : 0) * fa.ldw;
  const T* const w2 = GATE ? (const T*)fa.w2 + (int64_t)(n_ok ? n : 0) * fa.ldw2 : w;
  const T* x[RB];
#pragma unroll
  for (int b = 0; b < RB; ++b) x[b] = (const T*)fa.x + (16 * b + one < fa.rows ? 16 * b + one : 0) * fa.ldx;
  const int64_t second = fa.rows * fa.ldx;
  constexpr int kPiece = kStep * kUnroll;
  const int pieces = (fa.K + kPiece * P - 1) / (kPiece * P);
  const int shift = (int)(blockIdx.x * 5 % (uint32_t)pieces);
  f32x4 acc[RB] = {}, acc2[RB] = {};
  for (int p = wave; p < pieces; p += NW) {
    s16x8 fw[kUnroll], fw2[kUnroll];
    const int q = p + shift < pieces ? p + shift : p + shift - pieces;
    const int k = (q * P + part) * kPiece + g * (16 / (int)sizeof(T));
    const bool whole = (q + 1) * (kPiece * P) <= fa.K;
#pragma unroll
    for (int t = 0; t < kUnroll; ++t) {
      fw[t] = whole ? load_any<s16x8>(w + k + t * kStep) : load_k(w, k + t * kStep, fa.K);
      if (GATE) fw2[t] = whole ? load_any<s16x8>(w2 + k + t * kStep) : load_k(w2, k + t * kStep, fa.K);
    }
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      s16x8 fx[kUnroll], fl[kUnroll];
#pragma unroll
      for (int t = 0; t < kUnroll; ++t) {
        if constexpr (kPieces) fl[t] = whole ? load_any<s16x8>(x[b] + second + k + t * kStep) : load_k(x[b] + second, k + t * kStep, fa.K);
        fx[t] = whole ? load_any<s16x8>(x[b] + k + t * kStep) : load_k(x[b], k + t * kStep, fa.K);
      }
#pragma unroll
      for (int t = 0; t < kUnroll; ++t) {
        acc[b] = mma_few<DT>(fw[t], fx[t], acc[b]);
        if constexpr (kPieces) acc[b] = mma_few<DT>(fw[t], fl[t], acc[b]);
        if (GATE) acc2[b] = mma_few<DT>(fw2[t], fx[t], acc2[b]);
      }
    }
  }
  const int col = (int)blockIdx.x * kCols + tid % kCols;
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    if (b > 0) __syncthreads();
#pragma unroll
    for (int r = 0; r < 4; ++r) {      // [row of x, part][column, part]
      red[0][wave][c * 16 + 4 * g + r] = acc[b][r];
      if (GATE) red[GATE ? 1 : 0][wave][c * 16 + 4 * g + r] = acc2[b][r];
    }
    __syncthreads();
    const int m = 16 * b + tid / kCols;
    if (tid < kCols * kCols && m < fa.rows && col < fa.N) {
      float s = 0.0f, u = 0.0f;
#pragma unroll
      for (int v = 0; v < NW; ++v)
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const int at = (i * kCols + tid / kCols) * 16 + i * kCols + tid % kCols;
          s += red[0][v][at];
          if (GATE) u += red[GATE ? 1 : 0][v][at];
        }
      if (fa.b) {
        s += (float)((const T*)fa.b)[col];
        if (GATE) u += (float)((const T*)fa.b2)[col];
      }
      if constexpr (GATE && DT == NERFHIP_F32) {
        ((float*)fa.out)[m * fa.ldo + col] = activation_value(fa.act, s) * u;
      } else if constexpr (GATE) {
        T* const h = (T*)fa.out + m * fa.ldo + col;
        const float v = activation_value(fa.act, s) * u;
        if constexpr (few_pieces(DT, RB)) split2(v, h[0], h[fa.rows * fa.ldo]);
        else h[0] = (T)v;
      }
      if constexpr (!GATE) ((T*)fa.out)[m * fa.ldo + col] = (T)s;
    }
  }
}

// ---- operand copies: fp32 as three bf16 planes; 16-bit rows that are not whole 16-byte pieces as padded rows -------------------
struct PrepJob {
  const void* src;
  int64_t ld, rows;
  int32_t cols;
  uint16_t* dst;
  int64_t ldp, plane;     // ldp: cols rounded up to 8
};
constexpr int kMaxJobs = 5;
struct PrepArgs { PrepJob job[kMaxJobs]; };

template <bool F32> __device__ __forceinline__ void prep_rows(const PrepJob& j) {
  const uint32_t per_row = (uint32_t)(j.ldp / 8);
  const uint64_t total = (uint64_t)j.rows * per_row;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (uint64_t)gridDim.x * 256) {
    const uint64_t row = total >> 32 ? i / per_row : (uint32_t)i / per_row;
    const int c = (int)(i - row * per_row) * 8;
    uint16_t* const d = j.dst + row * j.ldp + c;
    if constexpr (F32) {
      const float* const p = (const float*)j.src + row * j.ld + c;
      float v[8];
      if (c + 8 <= j.cols) __builtin_memcpy(v, p, sizeof(v));
      else
        for (int k = 0; k < 8; ++k) v[k] = c + k < j.cols ? p[k] : 0.0f;
      uint16_t q[8][3];
#pragma unroll
      for (int k = 0; k < 8; ++k) split3(v[k], q[k]);
#pragma unroll
      for (int s = 0; s < 3; ++s) {
        const uint16_t o[8] = {q[0][s], q[1][s], q[2][s], q[3][s], q[4][s], q[5][s], q[6][s], q[7][s]};
        *(s16x8*)(d + s * j.plane) = __builtin_bit_cast(s16x8, o);
      }
    } else {
      const uint16_t* const p = (const uint16_t*)j.src + row * j.ld + c;
      s16x8 v;
      if (c + 8 <= j.cols) v = load_any<s16x8>(p);
      else {
        uint16_t o[8];
        for (int k = 0; k < 8; ++k) o[k] = c + k < j.cols ? p[k] : (uint16_t)0;
        v = __builtin_bit_cast(s16x8, o);
      }
      *(s16x8*)d = v;
    }
  }
}

// ---- column sums of dy: rows in slices, then the slices in order ----------------------------------------------------------------
constexpr int kSumRows = 128;      // rows of a slice: 32 for each wave of a workgroup
struct ColJob {
  const void* x;
  int64_t ld, rows;
  int32_t cols;
  float* part;                     // [slices][cols], or NULL: no sums
};
template <class T> __device__ __forceinline__ void col_sum(const ColJob& j) {
  __shared__ float red[4][64];
  const int across = (j.cols + 63) / 64, w = threadIdx.x >> 6;
  const int64_t many_blocks = (j.rows + kSumRows - 1) / kSumRows * across;
  for (int64_t id = blockIdx.x; id < many_blocks; id += gridDim.x) {
    const int64_t slice = id / across, r0 = slice * kSumRows + w * (kSumRows / 4);
    const int col = (int)(id % across) * 64 + (threadIdx.x & 63);
    const int many = j.rows - r0 < kSumRows / 4 ? (int)(j.rows - r0) : kSumRows / 4;
    const T* const p = (const T*)j.x + r0 * j.ld + col;
    float s = 0.0f;
    if (col < j.cols) {
      if (many == kSumRows / 4) {
#pragma unroll 16
        for (int r = 0; r < kSumRows / 4; ++r) s += (float)p[r * j.ld];
      } else {
        for (int r = 0; r < many; ++r) s += (float)p[r * j.ld];
      }
    }
    red[w][threadIdx.x & 63] = s;
    __syncthreads();
    if (w == 0 && col < j.cols)
      j.part[slice * j.cols + col] = (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]);
    __syncthreads();
  }
}

// What has to be done before the products: copies (blockIdx.y < n) and column sums.
template <class T> __global__ __launch_bounds__(256) void prep_kernel(const PrepArgs pa, int n, const ColJob sum) {
  if ((int)blockIdx.y < n) prep_rows<sizeof(T) == 4>(pa.job[blockIdx.y]);
  else col_sum<T>(sum);
}
struct SumJob {
  const float* part;
  int64_t ld;
  int32_t slices, cols;
  void* out;
};
struct SumArgs {
  SumJob job[3];
  int32_t n;
};
template <class T> __device__ __forceinline__ void slice_sum(const SumJob& j) {   // 16 columns x 16 groups of slices
  __shared__ float red[16][17];
  const int c = threadIdx.x & 15, w = threadIdx.x >> 4;
  for (int b = blockIdx.x; b * 16 < j.cols; b += gridDim.x) {
    const int col = b * 16 + c;
    float s = 0.0f;
    if (col < j.cols) {
#pragma unroll 8
      for (int i = w; i < j.slices; i += 16) s += j.part[(int64_t)i * j.ld + col];
    }
    red[w][c] = s;
    __syncthreads();
    if (w == 0 && col < j.cols) {
      for (int i = 1; i < 16; ++i) s += red[i][c];
      ((T*)j.out)[col] = (T)s;
    }
    __syncthreads();
  }
}

// ---- sum over splits of a product -------------------------------------------------------------------------------------------------
struct SplitSum {
  const float* part;      // [splits][M][ldp], ldp a multiple of 4
  int64_t M, ldp, ldo;
  int32_t N, splits;
  const void* bias;
  void* out;
};
struct SplitSums { SplitSum of[kMaxProblems]; };
template <class T> __device__ __forceinline__ void split_sum(const SplitSum& j) {
  const uint32_t per_row = (uint32_t)(j.ldp / 4);
  const int64_t total = j.M * per_row, slice = j.M * j.ldp;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t m = total >> 32 ? i / per_row : (uint32_t)i / per_row;
    const int n = (int)(i - m * per_row) * 4;
    const float* p = j.part + i * 4;
    f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
    for (int k = 0; k < j.splits; ++k) s += *(const f32x4*)(p + k * slice);
    if (j.bias)
      for (int r = 0; r < 4; ++r) if (n + r < j.N) s[r] += (float)((const T*)j.bias)[n + r];
    const T q[4] = {(T)s[0], (T)s[1], (T)s[2], (T)s[3]};
    T* const o = (T*)j.out + m * j.ldo + n;
    if (n + 4 <= j.N) put(o, q);
    else
#pragma unroll
      for (int r = 0; r < 4; ++r) if (n + r < j.N) o[r] = q[r];      // an index that is not known would put q into scratch memory
  }
}
// The sums over splits (blockIdx.y < n) and the bias gradients' sums over slices, which wait for a launch that they may join.
template <class T> __global__ __launch_bounds__(256) void sums_kernel(const SplitSums all, int n, const SumArgs sa) {
  if ((int)blockIdx.y < n) split_sum<T>(all.of[blockIdx.y]);
  else slice_sum<T>(sa.job[blockIdx.y - n]);
}
// ---- the gate in parts ------------------------------------------------------------------------------------------------------------
// Where the gate's product has few tiles, its k is cut as other products' is: g and u come as fp32 parts (dh too), and this kernel adds them up
// and does what the gate's epilogue does else.  One thread: eight columns of a row; a workgroup: 256 columns of 8 rows.  Bound by reading
// the parts, which the chip's caches still hold.
constexpr int kJoinRows = 8;
struct JoinArgs {
  const float *g, *u, *dh;         // [splits][M][ldh], dh: [dh_splits][M][ldh]
  int32_t splits, dh_splits;
  int64_t M, ldh, plane;
  int32_t N, act;
  const void *bias, *bias2;
  uint16_t *h, *dg, *du;
  float *sum_g, *sum_u;            // [M / 8][ldh], or NULL
};
__device__ __forceinline__ void sum_parts(const float* p, int64_t slice, int splits, float (&v)[8]) {
  f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f}, b = a;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    a += *(const f32x4*)(p + s * slice);
    b += *(const f32x4*)(p + s * slice + 4);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
}
template <int DT> __device__ __forceinline__ void put8(uint16_t* p, int64_t plane, const float (&v)[8]) {
  if constexpr (DT == NERFHIP_F32) {
    uint16_t q[8][3];
#pragma unroll
    for (int k = 0; k < 8; ++k) split3(v[k], q[k]);
#pragma unroll
    for (int s = 0; s < 3; ++s) {
      const uint16_t o[8] = {q[0][s], q[1][s], q[2][s], q[3][s], q[4][s], q[5][s], q[6][s], q[7][s]};
      *(s16x8*)(p + s * plane) = __builtin_bit_cast(s16x8, o);
    }
  } else {
    typedef typename OpType<DT>::t T;
    T q[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) q[k] = (T)v[k];
    *(s16x8*)p = __builtin_bit_cast(s16x8, q);
  }
}
template <int DT, bool BWD> __global__ __launch_bounds__(256) void join_kernel(const JoinArgs j) {
  typedef typename OpType<DT>::t T;
  __shared__ float red[BWD ? 2 : 1][kJoinRows][256];
  const int across = (int)((j.ldh + 255) / 256), c = (threadIdx.x & 31) * 8, r = threadIdx.x >> 5;
  const int64_t slice_id = blockIdx.x / across, m = slice_id * kJoinRows + r;
  const int64_t col = (int64_t)(blockIdx.x % across) * 256 + c;
  const bool in = m < j.M && col < j.ldh;
  float dg[8] = {}, du[8] = {};
  if (in) {
    const int64_t at = m * j.ldh + col, slice = j.M * j.ldh;
    float g[8], u[8], dh[8], h[8];
    sum_parts(j.g + at, slice, j.splits, g);
    sum_parts(j.u + at, slice, j.splits, u);
    if (BWD) sum_parts(j.dh + at, slice, j.dh_splits, dh);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool real = col + i < j.N;           // between N and ldh lie the zeros that the next product's k runs over
      if (j.bias && real) {
        g[i] += (float)((const T*)j.bias)[col + i];
        u[i] += (float)((const T*)j.bias2)[col + i];
      }
      float a, da;
      activation_any<BWD>(j.act, g[i], a, da);
      h[i] = real ? a * u[i] : 0.0f;
      if (BWD) {
        dg[i] = real ? dh[i] * u[i] * da : 0.0f;
        du[i] = real ? dh[i] * a : 0.0f;
      }
    }
    put8<DT>(j.h + at, j.plane, h);
    if (BWD) {
      put8<DT>(j.dg + at, j.plane, dg);
      put8<DT>(j.du + at, j.plane, du);
    }
  }
  if constexpr (BWD) {
    if (!j.sum_g) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      red[0][r][c + i] = dg[i];
      red[1][r][c + i] = du[i];
    }
    __syncthreads();
    const int64_t k = (int64_t)(blockIdx.x % across) * 256 + threadIdx.x;
    if (k >= j.ldh) return;
    float sg = 0.0f, su = 0.0f;
#pragma unroll
    for (int i = 0; i < kJoinRows; ++i) {
      sg += red[0][i][threadIdx.x];
      su += red[1][i][threadIdx.x];
    }
    j.sum_g[slice_id * j.ldh + k] = sg;
    j.sum_u[slice_id * j.ldh + k] = su;
  }
}

template <class T> __global__ void zero_kernel(T* p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) p[i] = (T)0.0f;
}

// ---- the plan --------------------------------------------------------------------------------------------------------------------
int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
int64_t ceil_div(int64_t x, int64_t by) { return (x + by - 1) / by; }

struct Arena {            // scratch memory; without a base it only counts
  char* base;
  int64_t used = 0;
  void* take(int64_t bytes) {
    void* p = base ? base + used : nullptr;
    used += up(bytes, 256);
    return p;
  }
};

struct Operand {          // one matrix as the products read it
  const uint16_t* p;
  int64_t ld, plane;
};

struct Split {
  int tile, splits;
  double us;
};
struct Size { int64_t M, N; };

// Which tile, and into how many parts the sum over k is cut: the plan that takes least by what was measured on bf16 products
// (microseconds, kernels alone on the chip).  A step of 64 k takes a workgroup `alone` on its CU, `together` where `most` share one; with all
// CUs at work the clock falls and memory is shared: `full` is the factor on a step then.  `fixed` covers a workgroup's start, its first loads
// and its epilogue.  Parts are written and read once more in fp32.
// Measured: 256 x 256: 32 workgroups 1.1 a step, 256 of them 1.55; 128 x 128: 0.72, two to a CU 1.06 for both; 64 x 128: 0.42, 0.46.
struct TileCost { int most; double alone, together, full, fixed; };
constexpr TileCost kTileCost[TILE_KINDS] = {{1, 1.1, 1.1, 1.4, 4.0}, {2, 0.72, 0.9, 1.18, 3.0}, {1, 0.42, 0.42, 1.1, 2.5}};
constexpr double kSumBytesPerUs = 5.0e6, kSumFixed = 4.5;

Split choose(const Size* size, int n, int64_t steps, int products, bool may_split, int columns, int n_cu) {
  Split best{TILE_64, 1, 1e30};
  for (int t = 0; t < TILE_KINDS; ++t) {
    const TileCost& c = kTileCost[t];
    int64_t tiles = 0;
    double values = 0.0;
    for (int i = 0; i < n; ++i) {
      tiles += ceil_div(size[i].M, kTileM[t]) * ceil_div(size[i].N * columns, kTileN[t]);
      values += (double)size[i].M * (double)size[i].N;
    }
    for (int s = 1; s <= 128 && s <= steps; s = s < 4 ? s + 1 : s * 5 / 4) {
      const double k = (double)(ceil_div(steps, s) * products);
      const int64_t blocks = tiles * s, round = (int64_t)n_cu * c.most, over = blocks % round;
      const double load = blocks < round ? (double)blocks / (double)round : 1.0, slow = 1.0 + (c.full - 1.0) * load;
      double us = (double)(blocks / round) * (k * c.together * slow + c.fixed);
      if (over > 0) us += k * (over <= n_cu ? c.alone : c.together) * slow + c.fixed;
      if (s > 1) us += kSumFixed + values * s * 8.0 / kSumBytesPerUs;
      if (us < best.us) best = Split{t, s, us};
      if (!may_split) break;
    }
  }
  return best;
}

struct Ctx {
  nerfhip_ffn* h;
  bool run;               // false: count scratch memory only
  hipError_t err = hipSuccess;
  void check(hipError_t e) { if (err == hipSuccess) err = e; }
};

int products(const Ctx& c) { return c.h->cfg.dtype == NERFHIP_F32 ? products_of<NERFHIP_F32>() : 1; }
int pieces(const Ctx& c) { return c.h->cfg.dtype == NERFHIP_F32 ? 3 : 1; }

void gemm_launch(Ctx& c, int kind, int tile, GemmArgs& ga) {
  int64_t blocks = 0;
  for (int i = 0; i < ga.n; ++i) blocks += (int64_t)ga.of[i].tiles_m * ga.of[i].tiles_n * ga.of[i].splits;
  if (blocks > 0x7fffffff) return c.check(hipErrorInvalidConfiguration);
  ga.blocks = (int32_t)blocks;
  ga.n_cu = c.h->n_cu;
  const int dt = c.h->cfg.dtype;
  c.check(dt == NERFHIP_F32 ? ffn_gemm_launch_f32(kind, tile, ga, c.h->stream) : dt == NERFHIP_BF16 ? ffn_gemm_launch_bf16(kind, tile, ga, c.h->stream)
                                                                                                  : ffn_gemm_launch_f16(kind, tile, ga, c.h->stream));
}

// Adds the segment A B^T.
void add_segment(GemmProblem& ga, const Operand& a, const Operand& b, const Operand* b2 = nullptr) {
  ga.seg[ga.nseg++] = GemmSeg{a.p, b.p, b2 ? b2->p : nullptr, a.plane, b.plane, (int32_t)a.ld, (int32_t)b.ld, b2 ? (int32_t)b2->ld : 0};
}

void set_tiles(GemmProblem& ga, const Split& sp, bool gate) {
  ga.tiles_m = (int32_t)ceil_div(ga.M, kTileM[sp.tile]);
  ga.tiles_n = (int32_t)ceil_div((int64_t)ga.N * (gate ? 2 : 1), kTileN[sp.tile]);
  ga.splits = sp.splits;
}
int64_t steps_of(const GemmProblem& ga) { return ceil_div(ga.K, kBK) * ga.nseg; }      // of 64 k: what a split may take

// The gate's product whole, or, with splits > 1, g and u as two products in parts.
Split plan_gate(const Ctx& c, const GemmProblem& ga) {
  const Size two[] = {{ga.M, ga.N}, {ga.M, ga.N}};
  const Split whole = choose(two, 1, steps_of(ga), products(c), false, 2, c.h->n_cu), parts = choose(two, 2, steps_of(ga), products(c), true, 1, c.h->n_cu);
  return parts.splits > 1 && parts.us < whole.us ? parts : whole;
}
template <bool BWD> void join_launch(Ctx& c, const JoinArgs& j) {
  const int64_t blocks = ceil_div(j.ldh, 256) * ceil_div(j.M, kJoinRows);
  if (blocks > 0x7fffff) return c.check(hipErrorInvalidConfiguration);
  const dim3 grid((uint32_t)blocks), block(256);
  if (c.h->cfg.dtype == NERFHIP_F32) hipLaunchKernelGGL((join_kernel<NERFHIP_F32, BWD>), grid, block, 0, c.h->stream, j);
  else if (c.h->cfg.dtype == NERFHIP_BF16) hipLaunchKernelGGL((join_kernel<NERFHIP_BF16, BWD>), grid, block, 0, c.h->stream, j);
  else hipLaunchKernelGGL((join_kernel<NERFHIP_F16, BWD>), grid, block, 0, c.h->stream, j);
  c.check(hipGetLastError());
}
int gate_slices(const Split& sp, int64_t M) {           // of dg's and du's column sums
  return (int)(sp.splits == 1 ? ceil_div(M, kTileM[sp.tile]) * kTileWavesM : ceil_div(M, kJoinRows));
}
// h, and dg, du and their column sums from ga.dh (dh_splits parts of it where the gate is in parts).
template <bool BWD> void run_gate(Ctx& c, const Split& sp, const GemmProblem& ga, const Operand& x, const Operand& wg, const Operand& wu, int dh_splits,
                                  Arena& mem) {
  if (sp.splits == 1) {
    GemmArgs args{};
    args.n = 1;
    args.of[0] = ga;
    set_tiles(args.of[0], sp, true);
    if (c.run) gemm_launch(c, BWD ? GEMM_GATE_BWD : GEMM_GATE, sp.tile, args);
    return;
  }
  const int64_t part = (int64_t)sp.splits * ga.M * ga.ldh;
  float* const parts = (float*)mem.take(part * 2 * 4);
  const JoinArgs j{parts, parts + part, ga.dh, sp.splits, dh_splits, ga.M, ga.ldh, ga.plane, ga.N, ga.act, ga.bias, ga.bias2,
                   ga.h, ga.dg, ga.du, ga.sum_g, ga.sum_u};
  GemmArgs two{};
  two.n = 2;
  for (int i = 0; i < 2; ++i) {
    GemmProblem& p = two.of[i];
    add_segment(p, x, i == 0 ? wg : wu);
    p.K = ga.K; p.M = ga.M; p.N = ga.N; p.out = parts + i * part; p.ldo = ga.ldh;
    set_tiles(p, sp, false);
  }
  if (c.run) {
    gemm_launch(c, GEMM_NT_F32, sp.tile, two);
    join_launch<BWD>(c, j);
  }
}

// C -> out in the tensors' type (+ bias), through fp32 parts where k is cut.  kind: GEMM_.._OUT; GEMM_.._F32 is the one after it.  Products of
// one launch have the same K and the same plan.
Split plan(const Ctx& c, const Size* size, int n, int64_t steps) { return choose(size, n, steps, products(c), true, 1, c.h->n_cu); }
uint32_t grid_of(int64_t threads) { return (uint32_t)(ceil_div(threads, 256) < 8192 ? ceil_div(threads, 256) : 8192); }
void launch_sums(Ctx& c, const SplitSums& sums, int n, int64_t most, SumArgs& sa) {
  for (int i = 0; i < sa.n; ++i) if (16 * (int64_t)sa.job[i].cols > most) most = 16 * (int64_t)sa.job[i].cols;
  const dim3 grid(grid_of(most), (uint32_t)(n + sa.n)), block(256);
  if (c.h->cfg.dtype == NERFHIP_F32) hipLaunchKernelGGL((sums_kernel<float>), grid, block, 0, c.h->stream, sums, n, sa);
  else if (c.h->cfg.dtype == NERFHIP_BF16) hipLaunchKernelGGL((sums_kernel<__bf16>), grid, block, 0, c.h->stream, sums, n, sa);
  else hipLaunchKernelGGL((sums_kernel<_Float16>), grid, block, 0, c.h->stream, sums, n, sa);
  c.check(hipGetLastError());
  sa.n = 0;
}
void launch_products(Ctx& c, GemmArgs& args, int kind, const Split& sp, Arena& mem, SumArgs& waiting) {
  SplitSums sums{};
  int64_t most = 0;
  for (int i = 0; i < args.n; ++i) {
    GemmProblem& ga = args.of[i];
    set_tiles(ga, sp, false);
    if (sp.splits == 1) continue;
    const int64_t ldp = up(ga.N, 4);
    float* const part = (float*)mem.take((int64_t)sp.splits * ga.M * ldp * 4);
    sums.of[i] = SplitSum{part, ga.M, ldp, ga.ldo, ga.N, sp.splits, ga.bias, ga.out};
    ga.out = part;
    ga.ldo = ldp;
    ga.bias = nullptr;
    if (ga.M * ldp / 4 > most) most = ga.M * ldp / 4;
  }
  if (!c.run) return;
  gemm_launch(c, sp.splits == 1 ? kind : kind + 1, sp.tile, args);
  if (sp.splits == 1) return;
  launch_sums(c, sums, args.n, most, waiting);
}

struct Prep {
  PrepArgs pa;
  int n = 0;
  int64_t most = 0;
  // A matrix for the products: as it is, or as a copy.  The scratch memory is set aside either way (its size may not depend on
  // addresses).
  Operand add(const Ctx& c, const void* src, int64_t ld, int64_t rows, int cols, Arena& mem) {
    const int64_t ldp = up(cols, 8), plane = up(rows * ldp, 128);
    uint16_t* const dst = (uint16_t*)mem.take(plane * 2 * pieces(c));
    if (pieces(c) == 1 && cols % 8 == 0 && ld % 8 == 0 && (uintptr_t)src % 16 == 0) return {(const uint16_t*)src, ld, 0};
    pa.job[n++] = PrepJob{src, ld, rows, cols, dst, ldp, plane};
    if (rows * ldp / 8 > most) most = rows * ldp / 8;
    return {dst, ldp, plane};
  }
  void launch(Ctx& c, const ColJob& sum) {
    if (!c.run || (n == 0 && !sum.part)) return;
    if (sum.part) {
      const int64_t threads = ceil_div(sum.cols, 64) * ceil_div(sum.rows, kSumRows) * 256;
      if (threads > most) most = threads;
    }
    const dim3 grid(grid_of(most), (uint32_t)(n + (sum.part ? 1 : 0))), block(256);
    if (c.h->cfg.dtype == NERFHIP_F32) hipLaunchKernelGGL((prep_kernel<float>), grid, block, 0, c.h->stream, pa, n, sum);
    else if (c.h->cfg.dtype == NERFHIP_BF16) hipLaunchKernelGGL((prep_kernel<__bf16>), grid, block, 0, c.h->stream, pa, n, sum);
    else hipLaunchKernelGGL((prep_kernel<_Float16>), grid, block, 0, c.h->stream, pa, n, sum);
    c.check(hipGetLastError());
  }
};

template <int DT, bool GATE, int RB, int UNROLL, int P> void few_launch_rows(Ctx& c, const FewArgs& fa) {
  // waves of a workgroup: until 16 of them work on a CU, or each has one piece of k
  const int64_t blocks = ceil_div(fa.N, 16 / P), pieces = ceil_div((int64_t)fa.K * (int64_t)dtype_bytes(DT), 64 * UNROLL * P);
  int nw = 4;
  while (nw < 16 && nw < pieces && blocks * nw < 16 * c.h->n_cu) nw *= 2;
  const dim3 grid((uint32_t)blocks);
  if (nw == 4) hipLaunchKernelGGL((few_rows_kernel<DT, GATE, 4, RB, UNROLL, P>), grid, dim3(256), 0, c.h->stream, fa);
  else if (nw == 8) hipLaunchKernelGGL((few_rows_kernel<DT, GATE, 8, RB, UNROLL, P>), grid, dim3(512), 0, c.h->stream, fa);
  else hipLaunchKernelGGL((few_rows_kernel<DT, GATE, 16, RB, UNROLL, P>), grid, dim3(1024), 0, c.h->stream, fa);
  c.check(hipGetLastError());
}
// Loads of a weight that a wave issues at a time: two (in fp32 the gate's one: 23 us instead of 25 for 8 rows of 2048 -> 8192), which spreads
// short rows over more waves (519 -> 1411: 7.0 us, with four 8.4); four where every wave has long rows to read and two bytes of h for each
// of the weights (8 rows of 16384 -> 4096: 36 us, with two 39.7).
template <int DT, bool GATE> void few_launch_type(Ctx& c, const FewArgs& fa) {
  constexpr int kOne = GATE && DT == NERFHIP_F32 ? 1 : 2;
  const int64_t blocks = ceil_div(fa.N, 16);
  if (fa.rows > 32) {
    if constexpr (few_rows(DT) > 32) few_launch_rows<DT, GATE, 4, 2, 1>(c, fa);
  } else if (fa.rows > 16) {
    few_launch_rows<DT, GATE, 2, 2, 1>(c, fa);
  } else if (fa.rows <= 4 && blocks * 4 <= c.h->n_cu) {
    few_launch_rows<DT, GATE, 1, kOne, 4>(c, fa);
  } else if (fa.rows <= 8 && blocks * 2 <= c.h->n_cu) {
    few_launch_rows<DT, GATE, 1, kOne, 2>(c, fa);
  } else if (!GATE && DT != NERFHIP_F32 && fa.K >= 8192) {
    if constexpr (!GATE && DT != NERFHIP_F32) few_launch_rows<DT, GATE, 1, 4, 1>(c, fa);
  } else {
    few_launch_rows<DT, GATE, 1, kOne, 1>(c, fa);
  }
}
template <bool GATE> void few_launch(Ctx& c, const FewArgs& fa) {
  const int dt = c.h->cfg.dtype;
  if (dt == NERFHIP_F32) few_launch_type<NERFHIP_F32, GATE>(c, fa);
  else if (dt == NERFHIP_BF16) few_launch_type<NERFHIP_BF16, GATE>(c, fa);
  else few_launch_type<NERFHIP_F16, GATE>(c, fa);
}

struct Call {             // a call's arguments
  const void *x, *dy;
  int64_t ldx, lddy, rows;
  nerfhip_ffn_weights w;
  void *y, *dx;
  int64_t ldy, lddx;
  nerfhip_ffn_grads g;
};

int64_t forward_few(Ctx& c, const Call& k, char* base) {
  const nerfhip_ffn_config& f = c.h->cfg;
  Arena mem{base};
  const int64_t ldh = up(f.d_ff, 8);
  void* const hid = mem.take(k.rows * ldh * 4);
  if (!c.run) return mem.used;
  FewArgs a{};
  a.x = k.x; a.ldx = k.ldx; a.w = k.w.w_gate; a.w2 = k.w.w_up; a.ldw = k.w.ld_gate; a.ldw2 = k.w.ld_up;
  a.b = k.w.b_gate; a.b2 = k.w.b_up; a.rows = (int32_t)k.rows; a.N = f.d_ff; a.K = f.d_model; a.act = f.activation;
  a.out = hid; a.ldo = ldh;
  few_launch<true>(c, a);
  FewArgs b{};
  b.x = hid; b.ldx = ldh; b.w = k.w.w_down; b.ldw = k.w.ld_down; b.b = k.w.b_down; b.rows = (int32_t)k.rows; b.N = f.d_model; b.K = f.d_ff;
  b.out = k.y; b.ldo = k.ldy;
  few_launch<false>(c, b);
  return mem.used;
}

int64_t forward_many(Ctx& c, const Call& k, char* base) {
  const nerfhip_ffn_config& f = c.h->cfg;
  Arena mem{base};
  Prep prep;
  const Operand x = prep.add(c, k.x, k.ldx, k.rows, f.d_model, mem);
  const Operand wg = prep.add(c, k.w.w_gate, k.w.ld_gate, f.d_ff, f.d_model, mem);
  const Operand wu = prep.add(c, k.w.w_up, k.w.ld_up, f.d_ff, f.d_model, mem);
  const Operand wd = prep.add(c, k.w.w_down, k.w.ld_down, f.d_model, f.d_ff, mem);
  prep.launch(c, ColJob{});
  const int64_t ldh = up(f.d_ff, 8), plane = up(k.rows * ldh, 128);
  uint16_t* const hid = (uint16_t*)mem.take(plane * 2 * pieces(c));
  GemmProblem ga{};
  add_segment(ga, x, wg, &wu);
  ga.K = f.d_model; ga.M = (int32_t)k.rows; ga.N = f.d_ff; ga.act = f.activation;
  ga.bias = k.w.b_gate; ga.bias2 = k.w.b_up;
  ga.h = hid; ga.ldh = ldh; ga.plane = plane;
  run_gate<false>(c, plan_gate(c, ga), ga, x, wg, wu, 0, mem);
  GemmArgs down{};
  GemmProblem& gd = down.of[0];
  add_segment(gd, Operand{hid, ldh, plane}, wd);
  gd.K = f.d_ff; gd.M = (int32_t)k.rows; gd.N = f.d_model;
  gd.out = k.y; gd.ldo = k.ldy; gd.bias = k.w.b_down;
  down.n = 1;
  const Size size{gd.M, gd.N};
  SumArgs none{};
  launch_products(c, down, GEMM_NT_OUT, plan(c, &size, 1, steps_of(gd)), mem, none);
  return mem.used;
}

int64_t backward_many(Ctx& c, const Call& k, char* base) {
  const nerfhip_ffn_config& f = c.h->cfg;
  Arena mem{base};
  Prep prep;
  const Operand x = prep.add(c, k.x, k.ldx, k.rows, f.d_model, mem);
  const Operand dy = prep.add(c, k.dy, k.lddy, k.rows, f.d_model, mem);
  const Operand wg = prep.add(c, k.w.w_gate, k.w.ld_gate, f.d_ff, f.d_model, mem);
  const Operand wu = prep.add(c, k.w.w_up, k.w.ld_up, f.d_ff, f.d_model, mem);
  const Operand wd = prep.add(c, k.w.w_down, k.w.ld_down, f.d_model, f.d_ff, mem);
  const int64_t dy_slices = ceil_div(k.rows, kSumRows);
  float* const dy_sums = (float*)mem.take(dy_slices * f.d_model * 4);
  prep.launch(c, ColJob{k.dy, k.lddy, k.rows, f.d_model, k.g.db_down ? dy_sums : nullptr});
  const int64_t ldh = up(f.d_ff, 8), plane = up(k.rows * ldh, 128), bytes = plane * 2 * pieces(c);
  uint16_t* const hid = (uint16_t*)mem.take(bytes);
  uint16_t* const dg = (uint16_t*)mem.take(bytes);
  uint16_t* const du = (uint16_t*)mem.take(bytes);
  const Operand oh{hid, ldh, plane}, og{dg, ldh, plane}, ou{du, ldh, plane};

  GemmProblem b{};                                     // h, dg, du
  add_segment(b, x, wg, &wu);
  b.K = f.d_model; b.M = (int32_t)k.rows; b.N = f.d_ff; b.act = f.activation;
  b.bias = k.w.b_gate; b.bias2 = k.w.b_up;
  b.h = hid; b.dg = dg; b.du = du; b.ldh = ldh; b.plane = plane;
  const Split gate = plan_gate(c, b);

  GemmArgs first{};                                    // dh = dy Wd
  first.n = 1;
  GemmProblem& a = first.of[0];
  add_segment(a, dy, wd);
  const Size dh_size{k.rows, f.d_ff};
  const Split dhs = plan(c, &dh_size, 1, ceil_div(f.d_model, kBK));
  float* const dh = (float*)mem.take(dhs.splits * k.rows * ldh * 4);
  a.K = f.d_model; a.M = (int32_t)k.rows; a.N = f.d_ff; a.out = dh; a.ldo = ldh;
  set_tiles(a, dhs, false);
  if (c.run) {
    gemm_launch(c, GEMM_NN_F32, dhs.tile, first);
    if (dhs.splits > 1 && gate.splits == 1) {          // the gate's epilogue reads whole ones: added up into the first part
      SplitSums all{};
      all.of[0] = SplitSum{dh, k.rows, ldh, ldh, f.d_ff, dhs.splits, nullptr, dh};
      hipLaunchKernelGGL((sums_kernel<float>), dim3(grid_of(k.rows * ldh / 4)), dim3(256), 0, c.h->stream, all, 1, SumArgs{});
      c.check(hipGetLastError());
    }
  }
  b.dh = dh;
  const int slices = gate_slices(gate, k.rows);
  float* const sums = (float*)mem.take(slices * ldh * 2 * 4);
  if (k.g.db_gate || k.g.db_up) { b.sum_g = sums; b.sum_u = sums + slices * ldh; }
  run_gate<true>(c, gate, b, x, wg, wu, dhs.splits, mem);

  SumArgs sa{};
  if (c.run) {
    if (k.g.db_down) sa.job[sa.n++] = SumJob{dy_sums, f.d_model, (int32_t)dy_slices, f.d_model, k.g.db_down};
    if (k.g.db_gate) sa.job[sa.n++] = SumJob{b.sum_g, ldh, slices, f.d_ff, k.g.db_gate};
    if (k.g.db_up) sa.job[sa.n++] = SumJob{b.sum_u, ldh, slices, f.d_ff, k.g.db_up};
  }

  // The two launches below follow one another on the stream and may cut k: they share one piece of scratch memory.
  const int64_t mark = mem.used;
  int64_t peak = mark;
  if (k.dx || !c.run) {
    GemmArgs args{};
    GemmProblem& ga = args.of[0];
    add_segment(ga, og, wg);
    add_segment(ga, ou, wu);
    ga.K = f.d_ff; ga.M = (int32_t)k.rows; ga.N = f.d_model; ga.out = k.dx; ga.ldo = k.lddx;
    args.n = 1;
    const Size size{ga.M, ga.N};
    launch_products(c, args, GEMM_NN_OUT, plan(c, &size, 1, steps_of(ga)), mem, sa);
    peak = mem.used;
    mem.used = mark;
  }
  // Planned as three whichever are asked for: neither the scratch memory nor the bits depend on that.
  const Size three[] = {{f.d_ff, f.d_model}, {f.d_ff, f.d_model}, {f.d_model, f.d_ff}};
  const Split wsp = plan(c, three, 3, ceil_div(k.rows, kBK));
  GemmArgs args{};
  auto weight_grad = [&](const Operand& p, int m, const Operand& q, int n, void* out) {
    if (!out && c.run) return;
    GemmProblem& ga = args.of[args.n++];
    add_segment(ga, p, q);
    ga.K = (int32_t)k.rows; ga.M = m; ga.N = n; ga.out = out; ga.ldo = n;
  };
  weight_grad(og, f.d_ff, x, f.d_model, k.g.dw_gate);
  weight_grad(ou, f.d_ff, x, f.d_model, k.g.dw_up);
  weight_grad(dy, f.d_model, oh, f.d_ff, k.g.dw_down);
  if (args.n > 0) launch_products(c, args, GEMM_TN_OUT, wsp, mem, sa);
  if (c.run && sa.n > 0) launch_sums(c, SplitSums{}, 0, 0, sa);
  return mem.used > peak ? mem.used : peak;
}

constexpr int64_t kMaxRows = ((int64_t)1 << 31) - 1024, kMaxLd = (int64_t)1 << 21;

int64_t scratch(nerfhip_ffn* h, int64_t rows, bool backward) {
  if (rows == 0) return 256;
  Ctx c{h, false};
  Call k{};
  k.rows = rows;
  const int64_t n = backward ? backward_many(c, k, nullptr) : take_few(h->cfg, rows) ? forward_few(c, k, nullptr) : forward_many(c, k, nullptr);
  return up(n, 256);
}

int bad(nerfhip_ffn* h, const char* msg) { return op_fail(h, g_ffn_error, NERFHIP_E_INVALID, msg); }

struct Range { uintptr_t lo, hi, width, pitch; };      // bytes
Range range_of(const void* p, int64_t rows, int64_t cols, int64_t ld, size_t eb) {
  if (!p || rows < 1) return {0, 0, 0, 0};
  return {(uintptr_t)p, (uintptr_t)p + (uintptr_t)((rows - 1) * ld + cols) * eb, (uintptr_t)cols * eb, rows > 1 ? (uintptr_t)ld * eb : 0};
}
bool overlap(const Range& a, const Range& b) {
  if (!(a.lo < b.hi && b.lo < a.hi)) return false;
  if (a.pitch == 0 || a.pitch != b.pitch) return true;
  const uintptr_t at = b.lo >= a.lo ? (b.lo - a.lo) % a.pitch : (a.pitch - (a.lo - b.lo) % a.pitch) % a.pitch;
  return at < a.width || at + b.width > a.pitch;         // else: other columns of the same wide rows
}

// What forward and backward check alike; NULL: fine.
const char* check_call(const nerfhip_ffn* h, const Call& k, bool backward, const void* ws, int64_t ws_bytes) {
  const nerfhip_ffn_config& f = h->cfg;
  const size_t eb = dtype_bytes(f.dtype);
  if (k.rows < 0 || k.rows > kMaxRows) return "rows out of range";
  const nerfhip_ffn_weights& w = k.w;
  if (!w.w_gate || !w.w_up || !w.w_down) return "null weight";
  if (w.ld_gate < f.d_model || w.ld_up < f.d_model || w.ld_down < f.d_ff) return "a weight's ld is smaller than its row";
  if (w.ld_gate > kMaxLd || w.ld_up > kMaxLd || w.ld_down > kMaxLd) return "a weight's ld is larger than 2097152";
  if ((f.bias != 0) != (w.b_gate != nullptr) || (f.bias != 0) != (w.b_up != nullptr) || (!backward && (f.bias != 0) != (w.b_down != nullptr)))
    return "bias pointers go with config.bias";
  const void* ptr[] = {k.x, k.dy, k.y, k.dx, w.w_gate, w.w_up, w.w_down, w.b_gate, w.b_up, w.b_down, k.g.dw_gate, k.g.dw_up, k.g.dw_down, k.g.db_gate, k.g.db_up, k.g.db_down};
  for (const void* p : ptr)
    if ((uintptr_t)p % eb) return "a pointer is not aligned to its element";
  if (k.rows > 0) {
    if (!k.x || (backward ? !k.dy : !k.y)) return "null argument";
    if (k.ldx < f.d_model || (backward ? k.lddy < f.d_model : k.ldy < f.d_model) || (k.dx && k.lddx < f.d_model)) return "a row stride is smaller than d_model";
    if (k.ldx > kMaxLd || k.lddy > kMaxLd || k.ldy > kMaxLd || k.lddx > kMaxLd) return "a row stride is larger than 2097152";
  }
  if (!f.bias && (k.g.db_gate || k.g.db_up || k.g.db_down)) return "bias gradients without biases";
  if (k.rows > 0 && (!ws || (uintptr_t)ws % 256)) return "workspace must be 256-byte aligned";
  if (k.rows > 0 && ws_bytes < scratch(const_cast<nerfhip_ffn*>(h), k.rows, backward)) return "workspace too small (nerfhip_ffn_workspace_bytes)";
  const int64_t d = f.d_model, ff = f.d_ff;
  const Range in[] = {range_of(k.x, k.rows, d, k.ldx, eb), range_of(k.dy, k.rows, d, k.lddy, eb), range_of(w.w_gate, ff, d, w.ld_gate, eb),
                      range_of(w.w_up, ff, d, w.ld_up, eb), range_of(w.w_down, d, ff, w.ld_down, eb), range_of(w.b_gate, 1, ff, ff, eb),
                      range_of(w.b_up, 1, ff, ff, eb), range_of(w.b_down, 1, d, d, eb)};
  const Range out[] = {range_of(k.y, k.rows, d, k.ldy, eb), range_of(k.dx, k.rows, d, k.lddx, eb), range_of(k.g.dw_gate, ff, d, d, eb),
                       range_of(k.g.dw_up, ff, d, d, eb), range_of(k.g.dw_down, d, ff, ff, eb), range_of(k.g.db_gate, 1, ff, ff, eb),
                       range_of(k.g.db_up, 1, ff, ff, eb), range_of(k.g.db_down, 1, d, d, eb), range_of(ws, ws ? 1 : 0, ws_bytes, 0, 1)};
  const int no = (int)(sizeof(out) / sizeof(out[0]));
  for (int i = 0; i < no; ++i) {
    for (const Range& r : in) if (overlap(out[i], r)) return "an output or the workspace overlaps an input";
    for (int j = i + 1; j < no; ++j) if (overlap(out[i], out[j])) return "two outputs, or an output and the workspace, overlap";
  }
  return nullptr;
}

void zero(Ctx& c, void* p, int64_t n) {
  if (!p) return;
  const int64_t blocks = ceil_div(n, 256) < 4096 ? ceil_div(n, 256) : 4096;
  if (c.h->cfg.dtype == NERFHIP_F32) hipLaunchKernelGGL((zero_kernel<float>), dim3((uint32_t)blocks), dim3(256), 0, c.h->stream, (float*)p, n);
  else hipLaunchKernelGGL((zero_kernel<__bf16>), dim3((uint32_t)blocks), dim3(256), 0, c.h->stream, (__bf16*)p, n);
  c.check(hipGetLastError());
}

}  // namespace
}  // namespace nh

using namespace nh;

extern "C" {

int nerfhip_ffn_create(const nerfhip_ffn_config* cfg, nerfhip_ffn_t** out) {
  if (!cfg || !out) return bad(nullptr, "null argument");
  *out = nullptr;
  const nerfhip_ffn_config& c = *cfg;
  if (c.d_model < 1 || c.d_model > 1048576 || c.d_ff < 1 || c.d_ff > 1048576) return bad(nullptr, "d_model and d_ff must be in [1, 1048576]");
  if (!dtype_ok(c.dtype)) return bad(nullptr, "dtype must be F32, BF16 or F16");
  if (c.activation < NERFHIP_ACT_SILU || c.activation > NERFHIP_ACT_RELU) return bad(nullptr, "unknown activation");
  if (c.bias != 0 && c.bias != 1) return bad(nullptr, "bias must be 0 or 1");
  if (c.reserved[0] || c.reserved[1]) return bad(nullptr, "reserved fields must be 0");
  if (!op_device_ok(c.device)) return op_fail(nullptr, g_ffn_error, NERFHIP_E_HIP, "no such HIP device (libnerfhip has no CPU path)");
  nerfhip_ffn* h = nullptr;
  try { h = new nerfhip_ffn(); } catch (const std::bad_alloc&) { return op_fail(nullptr, g_ffn_error, NERFHIP_E_NOMEM, "out of host memory"); }
  h->cfg = c;
  h->device = c.device;
  hipError_t e = hipErrorInvalidDevice;
  {
    DeviceScope dev(c.device);
    if (dev.ok) e = c.dtype == NERFHIP_F32 ? ffn_gemm_prepare_f32() : c.dtype == NERFHIP_BF16 ? ffn_gemm_prepare_bf16() : ffn_gemm_prepare_f16();
    if (e == hipSuccess) e = hipDeviceGetAttribute(&h->n_cu, hipDeviceAttributeMultiprocessorCount, c.device);
    if (e == hipSuccess) e = hipStreamCreateWithFlags(&h->own_stream, hipStreamNonBlocking);
  }
  if (e != hipSuccess) {
    delete h;
    return op_fail_hip(nullptr, g_ffn_error, e, "nerfhip_ffn_create");
  }
  h->stream = h->own_stream;
  *out = h;
  return NERFHIP_OK;
}

void nerfhip_ffn_destroy(nerfhip_ffn_t* h) {
  if (!h) return;
  DeviceScope dev(h->device);
  if (h->own_stream) { (void)hipStreamSynchronize(h->own_stream); (void)hipStreamDestroy(h->own_stream); }
  delete h;
}

const char* nerfhip_ffn_last_error(const nerfhip_ffn_t* h) { return h ? h->err.c_str() : g_ffn_error.c_str(); }

int nerfhip_ffn_set_stream(nerfhip_ffn_t* h, void* hip_stream) {
  if (!h) return bad(nullptr, "null handle");
  h->stream = op_stream(h, hip_stream);
  return NERFHIP_OK;
}

int nerfhip_ffn_synchronize(nerfhip_ffn_t* h) {
  if (!h) return bad(nullptr, "null handle");
  DeviceScope dev(h->device);
  const hipError_t e = hipStreamSynchronize(h->stream);
  return e == hipSuccess ? NERFHIP_OK : op_fail_hip(h, g_ffn_error, e, "hipStreamSynchronize");
}

int64_t nerfhip_ffn_workspace_bytes(const nerfhip_ffn_t* h, int64_t rows, int32_t backward) {
  if (!h || rows < 0 || rows > kMaxRows) return -1;
  return scratch(const_cast<nerfhip_ffn_t*>(h), rows, backward != 0);
}

int nerfhip_ffn_forward(nerfhip_ffn_t* h, const void* x, int64_t ldx, const nerfhip_ffn_weights* w, int64_t rows, void* y, int64_t ldy,
                        void* workspace, int64_t workspace_bytes) {
  if (!h) return bad(nullptr, "null handle");
  if (!w) return bad(h, "null argument");
  Call k{};
  k.x = x; k.ldx = ldx; k.w = *w; k.rows = rows; k.y = y; k.ldy = ldy;
  if (const char* msg = check_call(h, k, false, workspace, workspace_bytes)) return bad(h, msg);
  if (rows == 0) return NERFHIP_OK;
  DeviceScope dev(h->device);
  if (!dev.ok) return op_fail(h, g_ffn_error, NERFHIP_E_HIP, "hipSetDevice failed");
  Ctx c{h, true};
  if (take_few(h->cfg, rows)) forward_few(c, k, (char*)workspace);
  else forward_many(c, k, (char*)workspace);
  return c.err == hipSuccess ? NERFHIP_OK : op_fail_hip(h, g_ffn_error, c.err, "feed-forward kernels");
}

int nerfhip_ffn_backward(nerfhip_ffn_t* h, const void* x, int64_t ldx, const nerfhip_ffn_weights* w, const void* dy, int64_t lddy,
                         int64_t rows, void* dx, int64_t lddx, const nerfhip_ffn_grads* grads, void* workspace,
                         int64_t workspace_bytes) {
  if (!h) return bad(nullptr, "null handle");
  if (!w) return bad(h, "null argument");
  Call k{};
  k.x = x; k.ldx = ldx; k.w = *w; k.dy = dy; k.lddy = lddy; k.rows = rows; k.dx = dx; k.lddx = lddx;
  if (grads) k.g = *grads;
  if (const char* msg = check_call(h, k, true, workspace, workspace_bytes)) return bad(h, msg);
  DeviceScope dev(h->device);
  if (!dev.ok) return op_fail(h, g_ffn_error, NERFHIP_E_HIP, "hipSetDevice failed");
  Ctx c{h, true};
  if (rows == 0) {
    const int64_t d = h->cfg.d_model, f = h->cfg.d_ff;
    zero(c, k.g.dw_gate, d * f); zero(c, k.g.dw_up, d * f); zero(c, k.g.dw_down, d * f);
    zero(c, k.g.db_gate, f); zero(c, k.g.db_up, f); zero(c, k.g.db_down, d);
  } else {
    backward_many(c, k, (char*)workspace);
  }
  return c.err == hipSuccess ? NERFHIP_OK : op_fail_hip(h, g_ffn_error, c.err, "feed-forward kernels");
}

}  // extern "C"
