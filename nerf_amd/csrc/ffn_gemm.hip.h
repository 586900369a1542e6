// ffn_gemm.hip.h -- the matrix product of the feed-forward block's kernels.
//
//   C[m][n] = sum over segments s, over k of  A_s(m, k) B_s(n, k)        16-bit operands, fp32 sums
//
// An operand lies in memory either with its k values consecutive ([m][k]) or with its m values consecutive ([k][m]); both
// occur: forward products read rows of x and W, dx reads W by columns, the weight gradients read both operands by columns.
// A segment is one pair of operands; the sum over segments stays in the accumulators: dx = dg Wg + du Wu is two.  An fp32 operand is three
// planes of bf16 pieces of 8 bits (x = x0 + x1 + x2 exactly, each rounded to nearest), and its product the sum of x2 w0, x0 w2, x1 w1, x1 w0, x0 w1,
// x0 w0, which leaves out at most 2^-24 of the whole, of either sign.  One product after the other, the smallest first, rounds least: sums over
// 65536 rows of what comes out are 3.3e-7 off, and 1.3e-6 with all six for the same 64 k, where every one rounds at the full sum.  The weight gradients take
// the second order all the same: their long k comes from memory, and in the first order each plane two and three times (914 TFLOP/s of the
// six products against 1330 of a single one; 1200 then).  Both stay below what an fp32 sum over so many rows loses.
//
// Staging: 64 k of both tiles per step, global -> LDS directly (16 bytes per lane), two buffers or a ring.  Out-of-range chunks are read
// as zeros by the buffer descriptor's range check, so edges need no code: rows past the end lie past num_records, and in the
// last step the lanes whose k is past the end take an offset past it.
//   [m][k] operands: LDS rows of 128 bytes (64 k); the 16-byte chunk c of row r is stored at c ^ (r & 7), and read as one
//     ds_read_b128 per fragment: 8 lanes cover 8 different chunks, no bank twice.
//   [k][m] operands: LDS rows of BM values for each k; read with ds_read_b64_tr_b16, which hands lane i of a 16-lane group
//     column i of a 4 (k) x 16 (m) block.  The 32-byte unit u of row k is stored at u ^ f(k), f = (k & 3) | (k >> 1 & 4): the
//     eight rows that a half wave reads at once then lie in eight different bank groups.
// A direct load writes LDS linearly in lane order, so the permutations are applied to the lanes' global addresses.
//
// Bound by the matrix unit (and the clock that its power leaves) where sums are long: 8192 rows of 2048 -> 8192 in bf16, dx 1430 TFLOP/s,
// weight gradients 1340, dh, whose 268 MB of fp32 results are stored too, 1170 (kernel trace, calls in a row, on a card where the library's
// product of 8192^3 reaches 1370; 5 % more on the best one).  Short sums leave the epilogue: the gate of 262144
// rows of 256 -> 2 x 1024 in 407 us with gelu and biases is 196 of products, 0.54 GB of h and 64 activations a lane for four steps.
//
// The product is formed as v_mfma_f32_16x16x32 with the B rows as its first operand: a lane then holds four consecutive n of
// one row m, which the epilogues store as one piece.
#pragma once
#include <type_traits>

#include "op_common.h"

namespace nh {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) s16x8 lds_s16x8;

constexpr int kBK = 64;
constexpr int kMaxSeg = 2;
struct GemmSeg {
  const uint16_t* a;
  const uint16_t* b;
  const uint16_t* b2;      // gate epilogues: b = gate rows, b2 = up rows
  int64_t plane_a, plane_b;          // values between the planes of fp32 operands; both weights of a gate have the same
  int32_t lda, ldb, ldb2;
};
// the planes of the six products, two bits each
constexpr int kPlaneA = 2 | 0 << 2 | 1 << 4 | 1 << 6 | 0 << 8 | 0 << 10, kPlaneB = 0 | 2 << 2 | 1 << 4 | 0 << 6 | 1 << 8 | 0 << 10;
template <int DT> constexpr int products_of() { return DT == NERFHIP_F32 ? 6 : 1; }

enum { EPI_OUT = 0,        // C (+ bias) in the tensors' type
       EPI_F32 = 1,        // C in fp32, one slice per split
       EPI_GATE = 2,       // h
       EPI_GATE_BWD = 3 }; // h, dg, du from dh, and column sums of dg, du

constexpr bool gemm_walks(int epi) { return epi != EPI_GATE_BWD; }

struct GemmProblem {
  GemmSeg seg[kMaxSeg];
  int32_t nseg, K;         // every segment has K values
  int32_t M, N;            // gate epilogues: N = d_ff
  int32_t tiles_m, tiles_n, splits;
  int32_t act;
  void* out;               // EPI_OUT / EPI_F32
  int64_t ldo;
  const void* bias;        // EPI_OUT: [N]; gate: b_gate
  const void* bias2;       // gate: b_up
  uint16_t *h, *dg, *du;   // [M][ldh] in 16 bits, or three planes of it `plane` values apart
  int64_t ldh, plane;
  const float* dh;         // [M][ldh]
  float *sum_g, *sum_u;    // column sums of a workgroup's rows, [tiles_m * waves along m][ldh], or NULL
};
constexpr int kMaxProblems = 3;
struct GemmArgs {          // products that share a launch: workgroups are handed out to one after the other
  GemmProblem of[kMaxProblems];
  int32_t n;
  int32_t blocks, n_cu;    // tiles of all splits of all products; of a launch of 256 x 256 tiles n_cu workgroups take them in turn
};

template <int DT> struct OpType;
template <> struct OpType<NERFHIP_BF16> { typedef __bf16 t; };
template <> struct OpType<NERFHIP_F16> { typedef _Float16 t; };
template <> struct OpType<NERFHIP_F32> { typedef float t; };

template <class V> __device__ __forceinline__ void put(void* p, const V& v) { __builtin_memcpy(p, &v, sizeof(V)); }

// a(g) and a'(g).  exp and 1/x are the hardware's (1 ulp); the error function is Abramowitz and Stegun 7.1.26 (absolute error
// 1.5e-7), whose exp(-x^2), x = |g| / sqrt 2, is also the density that the derivative needs.  Where the value alone is wanted (the
// forward pass over ray samples spends more on it than on its products) the tail (1 - erf x) / 2 is 2^-P(|g|): P is a polynomial of degree 7
// fitted to -log2 of the tail on [0, 6] so that the largest error of the tail and of |g| times it is least (9e-8); 16 instead of 22 issue
// slots, 0.1 of 0.5 ms there.
template <int ACT, bool SLOPE> __device__ __forceinline__ void activation(float g, float& a, float& da) {
  constexpr float kLog2e = 1.4426950408889634f;
  if constexpr (ACT == NERFHIP_ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -kLog2e));
    a = g * s;
    da = s * fmaf(g, 1.0f - s, 1.0f);
  } else if constexpr (ACT == NERFHIP_ACT_GELU && !SLOPE) {
    const float s = __builtin_fminf(__builtin_fabsf(g), 6.0f);      // beyond, |g| times the tail is below 6e-9
    float q = fmaf(-6.1192095e-06f, s, 3.2478114e-05f);
    q = fmaf(q, s, 0.000494710985f);
    q = fmaf(q, s, -0.00750828441f);
    q = fmaf(q, s, 0.0527846925f);
    q = fmaf(q, s, 0.459120303f);
    q = fmaf(q, s, 1.15111494f);
    q = fmaf(q, s, 0.999999821f);
    const float top = fmaf(0.5f, __builtin_fabsf(g), 0.5f * g);     // max(g, 0) that keeps a NaN; g + |g| would pass fp32's range
    a = fmaf(-s, __builtin_amdgcn_exp2f(-q), top);
    da = 0.0f;
  } else if constexpr (ACT == NERFHIP_ACT_GELU) {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f * 0.70710678118654752f, __builtin_fabsf(g), 1.0f));
    const float e = __builtin_amdgcn_exp2f(g * (g * (-0.5f * kLog2e)));
    float q = fmaf(0.5f * 1.061405429f, t, 0.5f * -1.453152027f);
    q = fmaf(q, t, 0.5f * 1.421413741f);
    q = fmaf(q, t, 0.5f * -0.284496736f);
    q = fmaf(q, t, 0.5f * 0.254829592f);
    const float tail = q * t * e;                             // (1 - erf(x)) / 2
    const float c = g < 0.0f ? tail : 1.0f - tail;
    a = g * c;
    da = fmaf(g * e, 0.39894228040143268f, c);
  } else if constexpr (ACT == NERFHIP_ACT_GELU_TANH) {
    constexpr float k = 0.79788456080286536f;                 // sqrt(2 / pi)
    const float g2 = __builtin_fminf(g * g, 1e4f);            // tanh is 1 long before; the slope below stays finite for every g
    const float z2 = g * fmaf(2.0f * k * 0.044715f * kLog2e, g2, 2.0f * k * kLog2e);
    const float c = 1.0f - __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(z2) + 1.0f);   // (1 + tanh z) / 2
    a = g * c;
    da = fmaf(a * (1.0f - c), fmaf(6.0f * k * 0.044715f, g2, 2.0f * k), c);
  } else {
    a = g <= 0.0f ? 0.0f : g;                                 // a NaN stays one
    da = g > 0.0f ? 1.0f : 0.0f;
  }
}
template <bool SLOPE> __device__ __forceinline__ void activation_any(int act, float g, float& a, float& da) {
  switch (act) {
    case NERFHIP_ACT_SILU: activation<NERFHIP_ACT_SILU, SLOPE>(g, a, da); break;
    case NERFHIP_ACT_GELU: activation<NERFHIP_ACT_GELU, SLOPE>(g, a, da); break;
    case NERFHIP_ACT_GELU_TANH: activation<NERFHIP_ACT_GELU_TANH, SLOPE>(g, a, da); break;
    default: activation<NERFHIP_ACT_RELU, SLOPE>(g, a, da);
  }
}
__device__ __forceinline__ float activation_value(int act, float g) {
  float a, da;
  activation_any<false>(act, g, a, da);
  return a;
}

// Three bf16 pieces of a float, each what is left rounded to nearest: after the first at most 2^-8, after the second 2^-17 of the power of two
// below |x|, and the third is exact.  The first is kept finite for finite x (what is left of 2^128 - 2^104 has 16 bits); an infinity leaves an
// infinity and then a NaN, a NaN itself.  Cut off instead of rounded, all pieces had x's sign, and the products left out up to 2^-21 of the
// whole, always towards zero.
__device__ __forceinline__ void split3(float x, uint16_t (&p)[3]) {
  constexpr float kTop = 3.38953139e38f;      // the largest bf16
  float y = __builtin_amdgcn_fmed3f(x, -kTop, kTop);
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const __bf16 q = (__bf16)y;
    p[i] = __builtin_bit_cast(uint16_t, q);
    y = x -= (float)q;
  }
}

// Of two neighbouring 16-column fragments a lane holds columns 4g .. 4g+3 each.  Exchanging with the lane 16 further on gives lanes of
// even g eight consecutive columns of the first fragment and lanes of odd g eight of the second: pieces of 16 bytes, and rows of 64.
__device__ __forceinline__ u32x4 exchange(const uint32_t (&first)[2], const uint32_t (&second)[2]) {
  const auto lo = __builtin_amdgcn_permlane16_swap(first[0], second[0], false, false);
  const auto hi = __builtin_amdgcn_permlane16_swap(first[1], second[1], false, false);
  return u32x4{lo[0], hi[0], lo[1], hi[1]};
}
template <int DT> __device__ __forceinline__ void pack4(f32x4 v, uint32_t (&w)[2]) {
  typedef typename OpType<DT>::t T;
  typedef T T2 __attribute__((ext_vector_type(2)));
  w[0] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{v[0], v[1]}), T2));
  w[1] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{v[2], v[3]}), T2));
}
// The values of two neighbouring fragments (columns at, at + 16 of one row, 4 for each lane) in the form that the next product reads:
// 16 bits, or three bf16 planes.  in: the lane's eight columns exist (they are stored or left as a whole).
template <int DT> __device__ __forceinline__ void put_operand(uint16_t* base, int64_t plane, f32x4 x, f32x4 y, bool in) {
  if constexpr (DT == NERFHIP_F32) {
    uint16_t p[4][3], q[4][3];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      split3(x[r], p[r]);
      split3(y[r], q[r]);
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const uint32_t a[2] = {p[0][i] | (uint32_t)p[1][i] << 16, p[2][i] | (uint32_t)p[3][i] << 16};
      const uint32_t b[2] = {q[0][i] | (uint32_t)q[1][i] << 16, q[2][i] | (uint32_t)q[3][i] << 16};
      const u32x4 v = exchange(a, b);
      if (in) *(u32x4*)(base + i * plane) = v;
    }
  } else {
    uint32_t a[2], b[2];
    pack4<DT>(x, a);
    pack4<DT>(y, b);
    const u32x4 v = exchange(a, b);
    if (in) *(u32x4*)base = v;
  }
}

// 16 bytes per lane from the buffer to LDS at base + 16 * lane.  The wait for it is the caller's (vmcnt).
__device__ __forceinline__ void dma16(u32x4 rsrc, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc) : "memory");
}
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }

// What a wave loads of one operand: pieces of 1 KiB a fixed distance apart, step after step.  The lanes' offsets are the same for all
// pieces; the descriptor's base and size move.  Between two matrix instructions a wave has time for about three scalar ones, so all of
// this is kept incremental.
struct Feed {
  uint32_t voff[2];        // the lane's offset in even and odd pieces
  uint32_t kchunk;         // [m][k]: first k of the lane's chunk
  int32_t ld;
  uint64_t next;           // address of the next step's first piece,
  int64_t left;            // bytes from there to the end of the matrix,
  int32_t k_left, k_down;  // and k to the end; what a step takes of it where lanes have to look ([m][k]), or 0
  int64_t stride;          // bytes from step to step
  int32_t apart;           // and from piece to piece
  u32x4 rsrc;              // the next piece: base, bytes, format
  int32_t bytes;
  uint32_t past;           // a bit past every end in lanes whose k is past the end
  uint32_t to;             // its place in LDS

  // plane: bytes to the operand's plane; last: the step's 64 k are done with
  __device__ __forceinline__ void step(uint32_t lds, int64_t plane, bool last) {
    const uint64_t from = next + (uint64_t)plane;
    rsrc[0] = uniform((uint32_t)from);
    rsrc[1] = uniform((uint32_t)(from >> 32));
    rsrc[3] = 0x00020000u;
    // a tile spans less than 2^30 bytes (rows are at most 2^21 values apart), so what the pieces subtract never reaches valid ones
    const int32_t hi = (int32_t)(left >> 31);
    bytes = (int32_t)uniform(hi > 0 ? 0x7fffffffu : (uint32_t)left);
    past = (int)kchunk >= k_left ? 0x80000000u : 0u;
    to = uniform(lds);
    next += last ? (uint64_t)stride : 0;
    left -= last ? stride : 0;
    k_left -= last ? k_down : 0;
  }
  // the descriptor's last word but one: what lies at or past it reads as zero
  __device__ __forceinline__ void size() { rsrc[2] = (uint32_t)max(bytes, 0); }
  __device__ __forceinline__ void load(int i) { dma16(rsrc, voff[i & 1] | past, to); }
  __device__ __forceinline__ void move() {
    const uint64_t b = ((uint64_t)rsrc[1] << 32 | rsrc[0]) + (uint32_t)apart;
    rsrc[0] = (uint32_t)b;
    rsrc[1] = (uint32_t)(b >> 32);
  }
  template <int NW> __device__ __forceinline__ void shrink() {
    bytes -= apart;                   // may fall below zero: then nothing of the piece exists
    to += NW * 1024;
  }
  template <int NW> __device__ __forceinline__ void piece(int i) {
    size();
    load(i);
    move();
    shrink<NW>();
  }
};

// One operand's tile: ROWS (m or n) x 64 k, loaded by NW waves.  GATE: its rows are 16 gate rows, 16 up rows, and so on.
template <int ROWS, int NW, bool KMAJOR, bool GATE> struct TileLoad {
  static constexpr int kLoads = ROWS / 8 / NW;
  static constexpr int kCh = ROWS / 8, kPer = KMAJOR ? 64 / kCh : 1;              // [k][m]: 16-byte chunks of a k row, k rows of a piece
  static constexpr int kApart = KMAJOR ? NW * kPer : GATE ? NW * 4 : NW * 8;      // rows of memory between a wave's pieces
  static_assert(kLoads * 8 * NW == ROWS && NW % 4 == 0, "whole pieces for every wave; gate and up pieces for different waves");
  static_assert(!KMAJOR || NW * kPer % 8 == 0, "from piece to piece f(k) changes in bit 3 of k alone");

  // From step kt of a segment on.  row0: first row of the tile; rows: how many rows the matrix has (GATE: of each half)
  static __device__ __forceinline__ void open(Feed& f, const uint16_t* p, const uint16_t* p2, int32_t l, int32_t l2, int64_t row0, int rows,
                                              int kt, int K, int wave, int lane) {
    const int64_t up_to = rows - row0;
    const int k0 = kt * kBK;
    f.ld = GATE && (wave & 2) ? l2 : l;
    f.apart = kApart * f.ld * 2;
    if constexpr (!KMAJOR) {
      const int r = lane >> 3, c = (lane & 7) ^ r;
      const int row = GATE ? (wave >> 2) * 16 + (wave & 1) * 8 + r : wave * 8 + r;   // pieces 4q, 4q+1: gate; 4q+2, 4q+3: up
      f.voff[0] = f.voff[1] = (uint32_t)row * (uint32_t)f.ld * 2u + (uint32_t)c * 16u;
      f.kchunk = (uint32_t)c * 8u;
      const int K8 = (K + 7) & ~7;      // a row's last piece is whole: sizes that are no multiple of 8 come as padded copies
      f.next = (uint64_t)(uintptr_t)((GATE && (wave & 2) ? p2 : p) + row0 * f.ld + k0);
      f.left = ((up_to - 1) * f.ld + (K8 - k0)) * 2;
      f.stride = kBK * 2;
      f.k_left = K - k0;
      f.k_down = kBK;
    } else {
      const int kw = wave * kPer + lane / kCh, c = lane % kCh;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int k = kw + i * NW * kPer;
        const int sw = ((k & 3) | (k >> 1 & 4)) & (ROWS / 16 - 1);
        const int src = (((c >> 1) ^ sw) << 1) | (c & 1);
        f.voff[i] = (uint32_t)kw * (uint32_t)f.ld * 2u + (uint32_t)src * 16u;
      }
      f.kchunk = 0;
      f.next = (uint64_t)(uintptr_t)(p + (int64_t)k0 * f.ld + row0);
      f.left = ((int64_t)(K - k0 - 1) * f.ld + ((up_to + 7) & ~(int64_t)7)) * 2;
      f.stride = (int64_t)kBK * f.ld * 2;
      f.k_left = 1;
      f.k_down = 0;
    }
  }
};

// Fragments of 16 rows x 32 k out of a staged tile: lane (c, g) gets k = 8g .. 8g+7 of row c.
template <int ROWS, bool KMAJOR, int NT> struct TileRead {
  uint32_t off;
  __device__ __forceinline__ void init(int lane, int row0) {      // row0: a multiple of 16 NT
    const int c = lane & 15, g = lane >> 4;
    if constexpr (!KMAJOR) {
      off = (uint32_t)(row0 + c) * 128u + (uint32_t)((g ^ (c & 7)) << 4);
    } else {
      const int q = c >> 2, p = c & 3, f = (q | ((g & 1) << 2)) & (ROWS / 16 - 1);
      off = (uint32_t)(8 * g + q) * (ROWS * 2u) + (uint32_t)(((row0 / 16) ^ f) << 5) + (uint32_t)p * 8u;
    }
  }
  __device__ __forceinline__ s16x8 frag(lds_char* tile, int j, int ks) const {
    if constexpr (!KMAJOR) {
      return *(lds_s16x8*)(tile + (off ^ (uint32_t)(ks << 6)) + j * 2048);
    } else {
      lds_char* p = tile + (off ^ (uint32_t)(j << 5)) + ks * 32 * (ROWS * 2);      // unit row0 / 16 + j is row0 / 16 ^ j
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * (ROWS * 2)));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

template <int DT> __device__ __forceinline__ f32x4 mma(s16x8 a, s16x8 b, f32x4 c) {
  if constexpr (DT == NERFHIP_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Workgroups are handed to the 8 XCDs in turn: give each XCD a run of consecutive tiles, and walk the tiles in columns of 8 tile
// rows, so that what shares operands shares an L2.
__device__ __forceinline__ void tile_of(int id, int total, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int q = total / 8, r = total % 8, x = id % 8, i = id / 8;
  const int t = x < r ? x * (q + 1) + i : r * (q + 1) + (x - r) * q + i;
  const int per = 8 * tiles_n, grp = t / per, first = grp * 8;
  const int hm = tiles_m - first < 8 ? tiles_m - first : 8;
  tm = first + (t % per) % hm;
  tn = (t % per) / hm;
}

// Two pieces of 16 bytes that lie behind one another in a lane's row go out as whole lines: even rows' from lanes c and c + 1 first, then odd rows'
// (dh of 8192 rows of 2048 -> 8192 235 us, in half lines 254).
// x, y: the lane's first and second piece; after: of the even row (first piece in even lanes, second in odd ones), and of the odd row.
__device__ __forceinline__ void pair_rows(u32x4& x, u32x4& y, bool odd) {
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const uint32_t send = odd ? x[r] : y[r];
    const uint32_t got = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)send, 0xb1, 0xf, 0xf, true);      // lanes 1 0 3 2
    x[r] = odd ? got : x[r];
    y[r] = odd ? y[r] : got;
  }
}

// m, n: first row and column of the wave's part
template <int DT, bool F32, int MT, int NT>
__device__ __forceinline__ void out_epilogue(const GemmProblem& ga, const f32x4 (&acc)[MT][NT], int64_t m, int64_t n, int lane, int split) {
  typedef typename OpType<DT>::t T;
  const int c = lane & 15, g = lane >> 4;
  constexpr bool kWide = F32 || DT == NERFHIP_F32;
  typedef typename std::conditional<kWide, float, T>::type O;
  constexpr int kN = 16 / sizeof(O), kFrag = kWide ? 1 : 2;      // values and fragments of a piece
  static_assert(NT % (2 * kFrag) == 0, "fragments are stored in pairs of pieces");
  O* const out = (O*)ga.out + (F32 ? (int64_t)split * ga.M * ga.ldo : 0);
  const bool odd = c & 1;
#pragma unroll
  for (int j = 0; j < NT; j += 2 * kFrag) {
    const int64_t at = n + 16 * (j + kFrag * (c & 1)) + (kWide ? 4 * g : 16 * (g & 1) + 8 * (g >> 1));
    const int many = ga.N - at < kN ? (int)(ga.N - at) : kN;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      u32x4 v[2];
      if constexpr (kWide) {
        v[0] = __builtin_bit_cast(u32x4, acc[i][j]);
        v[1] = __builtin_bit_cast(u32x4, acc[i][j + 1]);
      } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t px[2], py[2];
          pack4<DT>(acc[i][j + 2 * k], px);
          pack4<DT>(acc[i][j + 2 * k + 1], py);
          v[k] = exchange(px, py);
        }
      }
      pair_rows(v[0], v[1], odd);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int64_t row = m + 16 * i + (c & 14) + k;
        if (row >= ga.M) continue;
        O* const o = out + row * ga.ldo + at;
        if (many == kN) put(o, v[k]);
        else {
          O q[kN];
          __builtin_memcpy(q, &v[k], sizeof(q));
#pragma unroll
          for (int r = 0; r < kN; ++r) if (r < many) o[r] = q[r];
        }
      }
    }
  }
}

// m, f: first row and first column of d_ff of the wave's part; sum_g, sum_u: where the sums of its rows go, or NULL.
// INSIDE: no row and no column of the part is past the end.  dh is read in one go: a load takes as long as a fragment row's work many times over.
template <int DT, int ACT, bool BWD, bool INSIDE, int MT, int NT>
__device__ __forceinline__ void gate_epilogue(const GemmProblem& ga, const f32x4 (&acc)[MT][NT], int64_t m, int64_t f, int lane,
                                              float* sum_g, float* sum_u) {
  const int c = lane & 15, g = lane >> 4;
  constexpr int kHalf = NT / 2;                      // 16-column fragments of d_ff
  static_assert(kHalf % 2 == 0, "fragments are stored in pairs");
  const int64_t step = 16 * ga.ldh;
  const int rows_in = INSIDE ? MT : (int)((ga.M - m - c + 15) / 16);      // fragment rows that exist for this lane
#pragma unroll
  for (int j = 0; j < kHalf; j += 2) {
    f32x4 sg[2] = {}, su[2] = {};
    // the lane's eight columns after the exchange; columns N .. ldh - 1 are the zeros that the next product's k runs over
    const int64_t out = f + 16 * (j + (g & 1)) + 8 * (g >> 1);
    const bool out_in = INSIDE || out < ga.ldh;
    int64_t line = (m + c) * ga.ldh;
    int64_t at[2];
    int cols[2];                                     // how many of the lane's four columns of each fragment exist
    f32x4 dhs[BWD ? MT : 1][2] = {};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      at[k] = f + 16 * (j + k) + 4 * g;
      cols[k] = INSIDE ? 4 : (int)(ga.N - at[k] < 4 ? ga.N - at[k] : 4);
    }
    if (BWD) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k)
          if (INSIDE || (i < rows_in && at[k] < ga.ldh)) __builtin_memcpy(&dhs[i][k], ga.dh + line + i * step + at[k], sizeof(f32x4));
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      f32x4 h[2], dg[2], du[2];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float a, da;
          const float u = acc[i][2 * (j + k) + 1][r];
          activation<ACT, BWD>(acc[i][2 * (j + k)][r], a, da);
          h[k][r] = a * u;
          const float dh = BWD ? dhs[BWD ? i : 0][k][r] : 0.0f;
          dg[k][r] = dh * u * da;
          du[k][r] = dh * a;
          if (!INSIDE && r >= cols[k]) h[k][r] = dg[k][r] = du[k][r] = 0.0f;
        }
      if (BWD && (INSIDE || i < rows_in)) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          sg[k] += dg[k];
          su[k] += du[k];
        }
      }
      const bool in = INSIDE || (i < rows_in && out_in);
      put_operand<DT>(ga.h + line + out, ga.plane, h[0], h[1], in);
      if (BWD) {
        put_operand<DT>(ga.dg + line + out, ga.plane, dg[0], dg[1], in);
        put_operand<DT>(ga.du + line + out, ga.plane, du[0], du[1], in);
      }
      line += step;
      if (BWD) __builtin_amdgcn_sched_barrier(0);
    }
    if (BWD && sum_g) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int d = 1; d < 16; d <<= 1) {
            sg[k][r] += __shfl_xor(sg[k][r], d, 64);
            su[k][r] += __shfl_xor(su[k][r], d, 64);
          }
        if (c == 0 && (INSIDE || at[k] < ga.ldh)) {
          put(sum_g + at[k], sg[k]);
          put(sum_u + at[k], su[k]);
        }
      }
    }
  }
}

// DT: the tensors' type (F32: operands are bf16 pieces); tile BM x BN (B rows; a gate tile has BN / 2 columns of d_ff); WM x WN waves; BUFS buffers
template <int DT, int BM, int BN, int WM, int WN, int BUFS, bool AK, bool BKM, int EPI>
__global__ __launch_bounds__(WM * WN * 64) void ffn_gemm_kernel(const GemmArgs args) {
  constexpr bool GATE = EPI == EPI_GATE || EPI == EPI_GATE_BWD;
  constexpr int NW = WM * WN, MT = BM / WM / 16, NT = BN / WN / 16;
  constexpr int kStage = (BM + BN) * kBK * 2;
  static_assert(!GATE || NT % 2 == 0, "gate and up fragments come in pairs");
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  lds_char* const lds = (lds_char*)smem;
  const uint32_t lds0 = (uint32_t)(uintptr_t)lds;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;

  // ---- the tile: which product, rows, columns, and the steps of its sum.  A step: one of the kSub products of 64 k of a segment; a split
  // takes whole multiples of 64 k.
  constexpr int kSub = products_of<DT>();
  int which = 0;                                   // an index, not a pointer: what is read through it stays in scalar registers
  auto ga = [&]() -> const GemmProblem& { return args.of[which]; };
  int64_t m0 = 0, n0 = 0;
  int tm = 0, split = 0, per_seg = 0, t1 = 0, steps = 0;
  // The step to be loaded next: 64 k number kt of segment s, whose part here is k_from .. k_to, product `sub`.
  constexpr bool kSameK = AK;                      // the products follow one another for the same 64 k, or each has its turn over the part
  int s = 0, k_from = 0, k_to = 0, kt = 0, sub = 0;
  auto locate = [&](int id) {
    which = 0;
    while (which + 1 < args.n) {
      const int here = args.of[which].tiles_m * args.of[which].tiles_n * args.of[which].splits;
      if (id < here) break;
      id -= here;
      ++which;
    }
    const int total = ga().tiles_m * ga().tiles_n;
    int tn;
    split = (int)uniform((uint32_t)(id / total));
    tile_of(id - split * total, total, ga().tiles_m, ga().tiles_n, tm, tn);
    tm = (int)uniform((uint32_t)tm);
    tn = (int)uniform((uint32_t)tn);
    m0 = (int64_t)tm * BM;
    n0 = (int64_t)tn * (GATE ? BN / 2 : BN);
    per_seg = (ga().K + kBK - 1) / kBK;
    const int all = per_seg * ga().nseg, chunk = (int)uniform((uint32_t)((all + ga().splits - 1) / ga().splits)), t0 = split * chunk;
    t1 = t0 + chunk < all ? t0 + chunk : all;
    steps = t1 > t0 ? (t1 - t0) * kSub : 0;
    s = t0 < t1 ? (int)uniform((uint32_t)(t0 / per_seg)) : 0;
    kt = k_from = t0 - s * per_seg;
    k_to = t1 - s * per_seg < per_seg ? t1 - s * per_seg : per_seg;
    sub = 0;
  };
  locate(blockIdx.x);

  constexpr bool kTurns = BM == 256;
  constexpr int NL = kTurns ? 4 : NW;              // waves that load an operand
  typedef TileLoad<BM, NL, AK, false> LA;
  typedef TileLoad<BN, NL, BKM, GATE> LB;
  TileRead<BM, AK, MT> ra;
  TileRead<BN, BKM, NT> rb;
  ra.init(lane, wm * MT * 16);
  rb.init(lane, wn * NT * 16);
  // The sums start from the biases: lane (c, g) holds n = 16 j + 4 g + 0 .. 3 of row 16 i + c.
  constexpr bool kBias = !AK && !BKM && EPI != EPI_F32;
  f32x4 acc[MT][NT];
  // A wave's 64 columns of biases are read one in each lane and handed round: as the 16 that a lane starts its sums from they put registers of
  // the second product into scratch memory, and a kernel that has any takes 12 us longer to start.
  auto start_sums = [&] {
    float mine = 0.0f;
    if constexpr (kBias) {
      static_assert(NT == 4, "a wave has 64 columns");
      typedef typename OpType<DT>::t T;
      const T* const p = (const T*)(GATE && lane >= 32 ? ga().bias2 : ga().bias);
      const int64_t at = n0 + (GATE ? wn * 32 + (lane & 31) : wn * 64 + lane);
      if (p && at < ga().N) mine = (float)p[at];
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      f32x4 b = {0.0f, 0.0f, 0.0f, 0.0f};
      if (kBias)
#pragma unroll
        for (int r = 0; r < 4; ++r) b[r] = __shfl(mine, (GATE ? j % 2 * 32 + j / 2 * 16 : j * 16) + (lane >> 4) * 4 + r, 64);
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[i][j] = b;
    }
  };
  auto plane_a = [&] { return kSub == 1 ? (int64_t)0 : (int64_t)(kPlaneA >> 2 * sub & 3) * ga().seg[s].plane_a * 2; };
  auto plane_b = [&] { return kSub == 1 ? (int64_t)0 : (int64_t)(kPlaneB >> 2 * sub & 3) * ga().seg[s].plane_b * 2; };
  auto onward = [&] { return !kSameK || kSub == 1 || sub == kSub - 1; };      // the step's 64 k are done with
  // behind step n: whether the loaders have to be opened anew
  auto advance = [&](int n) {
    if (kSub > 1 && kSameK) {
      if (++sub < kSub) return false;
      sub = 0;
    }
    if (++kt < k_to || n + 1 >= steps) return false;
    kt = k_from;
    if (kSub > 1 && !kSameK) {
      if (++sub < kSub) return true;
      sub = 0;
    }
    ++s;
    kt = k_from = 0;
    k_to = t1 - s * per_seg < per_seg ? t1 - s * per_seg : per_seg;
    return true;
  };
  // `of`, m0, ...: of the tile that is done; returns whether it lay inside the matrix for this wave (then it stored eight pieces at least)
  auto epilogue = [&](const GemmProblem& of, int64_t m_at, int64_t n_at, int tm_of, int split_of) {
    const int64_t m = m_at + wm * MT * 16;
    if constexpr (GATE) {
      const int64_t f = n_at + wn * NT * 8;
      constexpr bool kBwd = EPI == EPI_GATE_BWD;
      float* const sg = kBwd && of.sum_g ? of.sum_g + ((int64_t)tm_of * WM + wm) * of.ldh : nullptr;
      float* const su = kBwd && of.sum_g ? of.sum_u + ((int64_t)tm_of * WM + wm) * of.ldh : nullptr;
      const bool inside = m + MT * 16 <= of.M && f + NT * 8 <= of.N;
      // one copy of the code for each activation, and for parts that lie inside the matrix: nothing in them branches or is masked
#define NH_GATE(ACT)                                                                                   \
  if (inside) gate_epilogue<DT, ACT, kBwd, true, MT, NT>(of, acc, m, f, lane, sg, su);                 \
  else gate_epilogue<DT, ACT, kBwd, false, MT, NT>(of, acc, m, f, lane, sg, su)
      switch (of.act) {
        case NERFHIP_ACT_SILU: NH_GATE(NERFHIP_ACT_SILU); break;
        case NERFHIP_ACT_GELU: NH_GATE(NERFHIP_ACT_GELU); break;
        case NERFHIP_ACT_GELU_TANH: NH_GATE(NERFHIP_ACT_GELU_TANH); break;
        default: NH_GATE(NERFHIP_ACT_RELU);
      }
#undef NH_GATE
      return inside;
    } else {
      const int64_t n = n_at + wn * NT * 16;
      out_epilogue<DT, EPI == EPI_F32, MT, NT>(of, acc, m, n, lane, split_of);
      return m + MT * 16 <= of.M && n + NT * 16 <= of.N;
    }
  };

  if constexpr (kTurns) {
    // Two waves share a SIMD: waves 0 .. 3 lead, waves 4 .. 7 follow half a step behind.  While one reads its fragments of a step from
    // LDS, the other has the matrix unit and issues loads between its products (issued in one go they would hold a wave for as long as
    // its products take).  Barriers change the turns:
    //   phase 2t      leaders read step t                                    followers multiply step t - 1, load B of step t + 1
    //   phase 2t + 1  leaders multiply step t, load A of step t + 2          followers read step t
    // A ring of five 32-KiB slots, the whole LDS, takes A0 B0 A1 B1 ... in turn.  A(t + 2) and B(t + 1) go where B(t - 1) and A(t - 1)
    // were, whose last readers were the followers in phase 2t - 1.  A loader waits for its pieces before the barrier in front of phase
    // 2t + 2, where the leaders read them: the followers for all, the leaders for all but the 8 of A(t + 2).
    // A workgroup goes from tile to tile (a CU holds no second one whose work would cover the start of a tile): the first loads of the next
    // tile go out in front of the epilogue.  Not with the backward gate's, whose own loads would wait for them and whose registers they
    // would take.
    constexpr bool kWalk = gemm_walks(EPI);
    static_assert(BM == 256 && BN == 256 && kStage * 5 <= 2 * 160 * 1024, "five slots of half a stage");
    constexpr int kSlot = kStage / 2, kPieces = 8;
    const bool lead = wave < 4;
    const int w4 = wave & 3;
    Feed feed;
    uint32_t slot = lead ? 0 : 1;                         // of this wave's operand in the step that is loaded next
    auto segment = [&] {
      const GemmSeg& g = ga().seg[s];
      if (lead) LA::open(feed, g.a, nullptr, g.lda, 0, m0, ga().M, kt, ga().K, w4, lane);
      else LB::open(feed, g.b, g.b2, g.ldb, g.ldb2, n0, ga().N, kt, ga().K, w4, lane);
    };
    bool reopen = false;                                  // the last step's pieces may still be to be loaded: a segment is opened behind them
    auto next_step = [&](int n) {                         // step n, counted from t0; past the last: loads of nothing, which cost no branches
      if (reopen) segment();
      feed.step(lds0 + slot * kSlot + w4 * 1024, lead ? plane_a() : plane_b(), onward());
      if (n >= steps) feed.bytes = 0;
      slot = slot >= 3 ? slot - 3 : slot + 2;
      reopen = n < steps && advance(n);
    };
    auto load_all = [&](int n) {
      next_step(n);
#pragma unroll
      for (int i = 0; i < kPieces; ++i) feed.piece<NL>(i);
    };
    auto begin = [&] {
      slot = lead ? 0 : 1;
      if (steps == 0) return;
      segment();
      reopen = false;
      load_all(0);
      if (lead) load_all(1);
    };
    begin();
    start_sums();
    bool only_loads = true;                               // behind this wave's loads nothing is on its way, or eight stores at least
    for (int id = blockIdx.x;;) {
    if (steps > 0) {
      if (lead) {
        asm volatile("s_waitcnt vmcnt(8)\n\ts_barrier" ::: "memory");
      } else {
        if (only_loads) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
        asm volatile("s_barrier" ::: "memory");
        load_all(1);
        asm volatile("s_barrier" ::: "memory");
      }
    }
    uint32_t slot_a = 0;
    for (int t = 0; t < steps; ++t) {
      const uint32_t slot_b = slot_a == 4 ? 0 : slot_a + 1;
      lds_char* const ta = lds + slot_a * kSlot;
      lds_char* const tb = lds + slot_b * kSlot;
      slot_a = slot_a >= 3 ? slot_a - 3 : slot_a + 2;
      asm volatile("" : "+v"(ra.off), "+v"(rb.off));      // addresses are formed anew: kept over the loop they would not fit the registers
      s16x8 fa[2][MT], fb[2][NT];
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
        for (int j = 0; j < NT; ++j) fb[ks][j] = rb.frag(tb, j, ks);
#pragma unroll
        for (int i = 0; i < MT; ++i) fa[ks][i] = ra.frag(ta, i, ks);
      }
      next_step(t + 2);
      __builtin_amdgcn_sched_barrier(0);
      // followers: B of step t + 1, loaded during their last products, is there
      if (lead) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            acc[i][j] = mma<DT>(fb[ks][j], fa[ks][i], acc[i][j]);
            // a piece for every eight products, a bit of its work behind each
            const int at = i % 2 * NT + j, n = (ks * MT + i) / 2;
            __builtin_amdgcn_sched_barrier(0);
            if (at == 0) feed.size();
            if (at == 2) feed.load(n);
            if (at == 4) feed.move();
            if (at == 6) feed.shrink<NL>();
            __builtin_amdgcn_sched_barrier(0);
          }
      __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_sched_barrier(0);
      if (lead) asm volatile("s_waitcnt vmcnt(8)\n\ts_barrier" ::: "memory");      // A of step t + 1 is there
      else if (t + 1 < steps) asm volatile("s_barrier" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
    }
    // the loads of nothing still write zeros to LDS: behind this barrier all of it is free
    if (steps > 0) asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    const int done = which;
    const int64_t m_of = m0, n_of = n0;
    const int tm_of = tm, split_of = split;
    id += gridDim.x;
    const bool more = kWalk && id < args.blocks;
    if (more) {
      locate(id);
      begin();
    }
    only_loads = !epilogue(args.of[done], m_of, n_of, tm_of, split_of);
    if (!more) break;
    start_sums();
    }
  } else {
    // A ring of kBufs buffers: step t + kBufs - 1 is loaded while step t is multiplied.
    constexpr int kBufs = BUFS, kLoads = LA::kLoads + LB::kLoads;
    Feed from_a, from_b;
    auto segment = [&] {
      const GemmSeg& g = ga().seg[s];
      LA::open(from_a, g.a, nullptr, g.lda, 0, m0, ga().M, kt, ga().K, wave, lane);
      LB::open(from_b, g.b, g.b2, g.ldb, g.ldb2, n0, ga().N, kt, ga().K, wave, lane);
    };
    if (steps > 0) segment();
    auto open = [&](int n) {                              // past the last step: loads of nothing
      const uint32_t at = lds0 + (uint32_t)(n % kBufs) * kStage + wave * 1024;
      from_a.step(at, plane_a(), onward());
      from_b.step(at + BM * kBK * 2, plane_b(), onward());
      if (n >= steps) from_a.bytes = from_b.bytes = 0;
      return n < steps && advance(n);   // the pieces of step n are still to be loaded: the next segment is opened behind them
    };
    auto piece = [&](int i) {
      if (i < LA::kLoads) from_a.piece<NL>(i);
      else from_b.piece<NL>(i - LA::kLoads);
    };
    if (steps > 0)
      for (int n = 0; n < kBufs - 1; ++n) {
        const bool next = open(n);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) piece(i);
        if (next) segment();
      }
    start_sums();
    for (int t = 0; t < steps; ++t) {
      // this step's pieces have landed, and everybody is done reading the buffer of the step before
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((kBufs - 2) * kLoads) : "memory");
      lds_char* const ta = lds + t % kBufs * kStage;
      lds_char* const tb = ta + BM * kBK * 2;
      s16x8 fa[2][MT], fb[2][NT];
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
        for (int j = 0; j < NT; ++j) fb[ks][j] = rb.frag(tb, j, ks);
#pragma unroll
        for (int i = 0; i < MT; ++i) fa[ks][i] = ra.frag(ta, i, ks);
      }
      const bool next = open(t + kBufs - 1);
      __builtin_amdgcn_sched_barrier(0);
      // With two buffers the loads are wanted at the next step: they go out while the fragments come.  With more of them they go out
      // between the products.
      if constexpr (kBufs == 2) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) piece(i);
        __builtin_amdgcn_sched_barrier(0);
      }
      constexpr int kAll = 2 * MT * NT;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            acc[i][j] = mma<DT>(fb[ks][j], fa[ks][i], acc[i][j]);
            if constexpr (kBufs > 2) {
              const int at = (ks * MT + i) * NT + j;
              if ((at + 1) * kLoads / kAll != at * kLoads / kAll) {
                __builtin_amdgcn_sched_barrier(0);
                piece(at * kLoads / kAll);
                __builtin_amdgcn_sched_barrier(0);
              }
            }
          }
      if (next) segment();
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // the loads of nothing still write zeros to LDS
    epilogue(ga(), m0, n0, tm, split);
  }
}

// The products the block is made of, by how their operands lie and what becomes of the sums.
enum { GEMM_GATE = 0, GEMM_GATE_BWD, GEMM_NT_OUT, GEMM_NT_F32, GEMM_NN_OUT, GEMM_NN_F32, GEMM_TN_OUT, GEMM_TN_F32, GEMM_KINDS };
// 256 x 256 with the ring of slots; 128 x 128 with two buffers, two workgroups to a CU; 64 x 128 with four buffers, for products with few
// tiles.  (A 128 x 128 tile with five buffers and a CU to itself gained 15 % there, 64 x 128 with six nothing: a step's chain of LDS reads,
// address arithmetic and products bounds them, not the loads.)
enum { TILE_256 = 0, TILE_128, TILE_64, TILE_KINDS };
constexpr int kTileM[TILE_KINDS] = {256, 128, 64}, kTileN[TILE_KINDS] = {256, 128, 128};
constexpr int kTileBuffers[TILE_KINDS] = {0, 2, 4};
constexpr int kTileWavesM = 2;
constexpr int tile_lds(int tile) { return tile == TILE_256 ? 160 * 1024 : kTileBuffers[tile] * (kTileM[tile] + kTileN[tile]) * kBK * 2; }
// ffn_gemm_inst.hip, compiled once for each type
hipError_t ffn_gemm_launch_f32(int kind, int tile, const GemmArgs& ga, hipStream_t stream);
hipError_t ffn_gemm_launch_bf16(int kind, int tile, const GemmArgs& ga, hipStream_t stream);
hipError_t ffn_gemm_launch_f16(int kind, int tile, const GemmArgs& ga, hipStream_t stream);
hipError_t ffn_gemm_prepare_f32();
hipError_t ffn_gemm_prepare_bf16();
hipError_t ffn_gemm_prepare_f16();

}  // namespace nh
