// Matrix products on tiles of the matrix cores, for the operators of linear.hip and vocab.hip.
//
//   C(m, n) = sum over k of A(m, k) B(n, k)
//
// Each operand lies in memory either with its reduction index contiguous (rows of k) or with its own
// index contiguous (rows of m or n, one per k): a layer's forward product has two of the first kind, the
// gradient of its input one of each, the gradient of its weight two of the second.  A workgroup forms a
// tile of 256 x 256 or 128 x 128, 128 bytes of the reduction at a time, from two LDS stages that are
// filled past the registers (buffer loads to LDS); what lies outside the operand lies past the buffer's end
// and so arrives as zeros.  16-bit operands whose rows do not begin and end on 16 bytes are copied to
// such rows first, and fp32 ones to three planes of bf16.
//
// In LDS the 16-byte pieces of a row are permuted by its index, so that the 64 lanes of a read meet all banks
// (SQ_LDS_BANK_CONFLICT is 0):
//   rows of k:   piece c of row i sits at c ^ ((i >> 1) & 7); a lane reads its 16 bytes of k at once
//   rows of m/n: piece c of row k sits at c ^ swizzle(k); values are transposed by the LDS read itself
//                (ds_read_b64_tr_b16: lane i of 16 gets element i of four rows)
// The products run as B A, so that a lane ends with four consecutive n of one m.  All sums are fp32.
//
// What bounds it: the matrix cores and the power they take.  The four products of 8192 tokens, 32768 words and a width of
// 4096 in bf16 run at 1264 (with the softmax in its epilogue) to 1388 TFLOP/s, where the library's reach 1489, 1214 and
// 1068 in the three layouts; they are busy 55 % of the cycles of a clock that falls to 1.9 GHz.
#pragma once

#include "dnpeff_internal.hpp"

#include <type_traits>

namespace dn {
namespace tl {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));

#define DN_LDS __attribute__((address_space(3)))

template <class V>
__device__ __forceinline__ DN_LDS V* lds_at(unsigned address) {
  return (DN_LDS V*)(uintptr_t)address;
}

template <class T>
struct num;
// piece: 16 bytes of the reduction index of one row, as a lane holds them; op: the type that tiles multiply; TERMS: products of
// it that a product takes.  fp32 goes as three bf16 numbers that add up to it, in the six products that matter next to fp32 (the
// matrix cores multiply fp32 itself at a sixteenth of bf16's rate).
template <>
struct num<float> {
  typedef v4f piece;
  typedef __bf16 op;
  static constexpr int TERMS = 6, PLANES = 3;
};
template <>
struct num<_Float16> {
  typedef v8h piece;
  typedef _Float16 op;
  static constexpr int TERMS = 1, PLANES = 1;
};
template <>
struct num<__bf16> {
  typedef v8b piece;
  typedef __bf16 op;
  static constexpr int TERMS = 1, PLANES = 1;
};
// The planes of the t-th term, the smallest first: low high, high low, middle middle, middle high, high middle, high high.
__device__ __forceinline__ int plane_a(int t) { return (0x0052 >> (2 * t)) & 3; }
__device__ __forceinline__ int plane_b(int t) { return (0x0118 >> (2 * t)) & 3; }

__device__ __forceinline__ v4f mma(v8b a, v8b b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ v4f mma(v8h a, v8h b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
// (any order of k serves as long as both operands have the same: element e of all four lane groups together)
__device__ __forceinline__ v4f mma(v4f a, v4f b, v4f c) {
#pragma unroll
  for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

// ---- activations and their slopes, in fp32 -----------------------------------------------------------------------
// (16-bit results: the reciprocal and the exponential of the hardware, one ulp of fp32 off)
template <bool EXACT>
__device__ __forceinline__ float sigmoid(float z) {
  if (EXACT) return 1.f / (1.f + expf(-z));
  return __builtin_amdgcn_rcpf(1.f + __expf(-z));
}
// (1 + tanh(u)) / 2 = sigmoid(2u): by itself, so that what is left of it below zero is not rounded away next to 1
template <bool EXACT>
__device__ __forceinline__ float gelu_tanh_s(float z) {
  return sigmoid<EXACT>(1.5957691216057308f * (z + 0.044715f * z * z * z));
}
// The normal distribution's Phi(z), and *e = exp(-z^2 / 2).  16-bit results: erfc(x) = exp(-x^2) t Q(t) for x >= 0 with
// t = 1 / (1 + 0.45 x) and Q the polynomial of degree 7 whose largest relative error on [0, 12] is smallest (fitted for this:
// 3.8e-7 with these coefficients, in fp32 6.5e-7), far below half a unit of those types; fp32 takes the library's erfc.
template <bool EXACT>
__device__ __forceinline__ float normal(float z, float* e) {
  if (EXACT) {
    *e = expf(-0.5f * z * z);
    return 0.5f * erfcf(z * -0.70710678118654752f);  // (1 + erf loses what is left of it below zero)
  }
  const float x = fabsf(z) * 0.70710678118654752f, t = __builtin_amdgcn_rcpf(1.f + 0.45f * x);
  *e = __expf(-x * x);
  float y = fmaf(fmaf(fmaf(0.0682241097f, t, -0.246025205f), t, 0.218937039f), t, 0.0308285784f);
  y = fmaf(fmaf(fmaf(fmaf(y, t, 0.193743601f), t, 0.226509377f), t, 0.253890544f), t, 0.253892303f);
  y = 0.5f * *e * t * y;
  return z < 0.f ? y : 1.f - y;
}
template <bool EXACT, int W>
__device__ __forceinline__ void act_of(float* z, int act) {
  if (act == DNPEFF_ACT_RELU) {
#pragma unroll
    for (int t = 0; t < W; t++) z[t] = z[t] > 0.f ? z[t] : (z[t] != z[t] ? z[t] : 0.f);
  } else if (act == DNPEFF_ACT_SILU) {
#pragma unroll
    for (int t = 0; t < W; t++) z[t] *= sigmoid<EXACT>(z[t]);
  } else if (act == DNPEFF_ACT_GELU) {
#pragma unroll
    for (int t = 0; t < W; t++) {
      float e;
      z[t] *= normal<EXACT>(z[t], &e);
    }
  } else if (act == DNPEFF_ACT_GELU_TANH) {
#pragma unroll
    for (int t = 0; t < W; t++) z[t] *= gelu_tanh_s<EXACT>(z[t]);
  }
}
// v *= act'(z)
template <bool EXACT, int W>
__device__ __forceinline__ void slopes_of(float* v, const float* z, int act) {
  if (act == DNPEFF_ACT_RELU) {
#pragma unroll
    for (int t = 0; t < W; t++) v[t] = z[t] > 0.f ? v[t] : v[t] * 0.f;
  } else if (act == DNPEFF_ACT_SILU) {
#pragma unroll
    for (int t = 0; t < W; t++) {
      const float p = sigmoid<EXACT>(z[t]);
      v[t] *= p * (1.f + z[t] * (1.f - p));
    }
  } else if (act == DNPEFF_ACT_GELU) {
#pragma unroll
    for (int t = 0; t < W; t++) {
      float e;
      const float f = normal<EXACT>(z[t], &e);
      v[t] *= f + z[t] * e * 0.39894228040143268f;
    }
  } else if (act == DNPEFF_ACT_GELU_TANH) {
#pragma unroll
    for (int t = 0; t < W; t++) {
      const float s = gelu_tanh_s<EXACT>(z[t]);
      // (z^2 is kept finite: where it would not be, s (1 - s) is zero)
      v[t] *= s + z[t] * (s * (1.f - s)) * 1.5957691216057308f * (1.f + 0.134145f * fminf(z[t] * z[t], 1e30f));
    }
  }
}

// ---- rows in groups ----------------------------------------------------------------------------------------------
// Group g holds rows ends[g] .. ends[g + 1] (the first from row 0, whatever ends[0] says); rows past the last
// end belong to none and count as group `groups`.  Ends outside the rows are taken as the nearest inside, a group whose end
// falls is empty.  Groups may then overlap, and their tiles add up to more than there can be: counts of tiles stop at
// 2^31 - 1, and launches at most_tiles, so no read or write goes by the ends unchecked.
struct group_rows {
  const int64_t* ends;
  int groups;
  int64_t rows;
  __device__ __forceinline__ int64_t at(int g) const {
    if (!ends) return rows;  // one group of all rows
    const int64_t e = ends[g];
    return e < 0 ? 0 : e > rows ? rows : e;
  }
  // (g the same in all lanes: through the scalar cache)
  __device__ __forceinline__ int64_t one_at(int g) const {
    if (!ends) return rows;
    const int64_t e = ((const __attribute__((address_space(4))) int64_t*)ends)[g];
    return e < 0 ? 0 : e > rows ? rows : e;
  }
  __device__ __forceinline__ int64_t one_first(int g) const { return g == 0 ? 0 : one_at(g); }
  __device__ __forceinline__ int64_t one_last(int g) const { return g < groups ? one_at(g + 1) : rows; }
  __device__ __forceinline__ int64_t first(int g) const { return g == 0 ? 0 : at(g); }
  __device__ __forceinline__ int64_t last(int g) const { return g < groups ? at(g + 1) : rows; }
  __device__ __forceinline__ int64_t count(int g) const {
    const int64_t n = last(g) - first(g);
    return n > 0 ? n : 0;
  }
  // Tiles of `tall` rows that groups which do not overlap take at most.
  __host__ __device__ __forceinline__ int64_t most_tiles(int tall) const { return rows / tall + (groups + 1 < rows ? groups + 1 : rows); }
};

__device__ __forceinline__ int add_up(int a, int b) { return __builtin_elementwise_add_sat(a, b); }
__device__ __forceinline__ int wave_scan(int v, int lane) {  // inclusive sum over the lanes, of counts; 2^31 - 1 at most
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int u = __shfl_up(v, d, 64);
    if (lane >= d) v = add_up(v, u);
  }
  return v;
}
// Tiles of `tall` rows that the groups (and the rows of none) take; every wave by itself.
__device__ __forceinline__ int group_tiles(const group_rows& G, int tall, int lane) {
  int sum = 0;
  for (int b = 0; b <= G.groups; b += 64) {
    const int g = b + lane;
    const int t = g <= G.groups ? (int)((G.count(g) + tall - 1) / tall) : 0;
    sum = add_up(sum, __shfl(wave_scan(t, lane), 63, 64));
  }
  const int64_t most = G.most_tiles(tall);
  return sum < most ? sum : (int)most;
}
// The group of tile `tile` of them, and its number within that group.
__device__ __forceinline__ void group_of_tile(const group_rows& G, int tall, int lane, int tile, int* group, int* within) {
  int before = 0;
  for (int b = 0; b <= G.groups; b += 64) {
    const int g = b + lane;
    const int t = g <= G.groups ? (int)((G.count(g) + tall - 1) / tall) : 0;
    const int upto = add_up(before, wave_scan(t, lane));
    const unsigned long long hit = __ballot(tile < upto);
    if (hit) {
      const int l = __ffsll(hit) - 1;
      *group = __builtin_amdgcn_readfirstlane(b + l);
      *within = __builtin_amdgcn_readfirstlane(tile - (l > 0 ? __shfl(upto, l - 1, 64) : before));  // (what is not past `tile` is exact)
      return;
    }
    before = __shfl(upto, 63, 64);
  }
  *group = -1;
  *within = 0;
}

// ---- a product ---------------------------------------------------------------------------------------------------
enum { ONE = 0, BY_ROWS = 1, BY_REDUCTION = 2 };                      // groups: none, of rows of A and C, of the reduction
enum { E_LINEAR = 0, E_STORE = 1, E_LOSS = 2, E_LOSS_GRAD = 3 };     // what becomes of a tile

struct args {
  const void *A, *B;        // (of num<T>::op)
  int64_t lda, ldb;         // elements from one row to the next
  int64_t a_plane, b_plane; // ... from a plane of fp32 to the next
  int64_t M, N, K;          // BY_REDUCTION: K = rows of both operands
  int tm_first, tn_first;   // (ONE) the launch's first tile in either direction
  int64_t b_group;          // BY_ROWS: elements from a group's B to the next one's
  group_rows G;
  int mode, splits;         // splits: of the reduction, for E_STORE to fp32 partial sums
  int64_t split_k;          // k per split
  int64_t c_split, c_group; // elements between the results of splits, of groups (BY_REDUCTION)
  // E_STORE: `sums` (fp32, rows of ldc, a multiple of 4) is read and added where add_sums, and takes the result where
  // out is NULL; else out (T, or fp32 where out_f32; rows of ldo) takes it, times *scale, squared where asked for
  float* sums;
  void* out;
  int64_t ldc, ldo;
  const float* scale;
  int past;  // out is larger than the caches: past them
  int add_sums, out_f32, square;
  // E_LINEAR
  const void *bias, *residual;
  void* pre;
  int64_t ldp, ldr;
  int act;
  // E_LOSS, E_LOSS_GRAD: columns are words, `word0` the first of this piece
  const int32_t* labels;
  const float *lse, *dloss;
  const float* shrink;      // (dloss is multiplied by this; NULL: by 1)
  float2* parts;            // [M][parts_n]: maximum and sum of each tile's words, this launch's from part0 on
  int parts_n, part0;
  float* hit;               // [M] the label's logit
  int64_t word0, words;
};

// A kernel's arguments where they lie: read where they are needed, not kept in registers throughout.
typedef const __attribute__((address_space(4))) args kargs;
__device__ __forceinline__ kargs& again() {
  kargs* p = (kargs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *p;
}

// W consecutive values of a row at once, wherever they begin: the memory pipe takes any alignment of whole elements
// (products of 1999 x 4101 in fp16 68 us with their results value by value, 46 so).
template <class T, int W>
using loose = T __attribute__((ext_vector_type(W), aligned(sizeof(T))));
template <class T, int W>
__device__ __forceinline__ void load_row(const T* p, float* v) {
  const loose<T, W> q = *(const loose<T, W>*)p;
#pragma unroll
  for (int t = 0; t < W; t++) v[t] = (float)q[t];
}
template <class T, int W>
__device__ __forceinline__ void store_row(T* p, const float* v, bool past = false) {
  loose<T, W> q;
#pragma unroll
  for (int t = 0; t < W; t++) q[t] = (T)v[t];
  if (past)
    __builtin_nontemporal_store(q, (loose<T, W>*)p);
  else
    *(loose<T, W>*)p = q;
}

// W consecutive values as an operand of tiles: as they are, or as planes so far apart.
template <class T, int W>
__device__ __forceinline__ void store_op(typename num<T>::op* p, int64_t plane, const float* v) {
  if constexpr (num<T>::PLANES == 1) {
    store_row<T, W>(p, v);
  } else {
    float rest[W];
    loose<__bf16, W> q[3];
#pragma unroll
    for (int t = 0; t < W; t++) {
      // An infinity is (1, 0, infinity) of its sign: of the products of planes only the one with the other's high plane is
      // infinite then, as the product itself is (infinity, 0, 0 would meet low planes of either sign).  Finite values that
      // would round to infinity begin with the largest bf16.
      constexpr float MOST = 0x1.fep127f;
      const bool past = fabsf(v[t]) > MOST, inf = fabsf(v[t]) == INFINITY;
      q[0][t] = (__bf16)(past ? copysignf(inf ? 1.f : MOST, v[t]) : v[t]);
      rest[t] = v[t] - (float)q[0][t];
      q[1][t] = (__bf16)(inf ? 0.f : rest[t]);
      rest[t] -= (float)q[1][t];
      q[2][t] = (__bf16)rest[t];
    }
#pragma unroll
    for (int h = 0; h < 3; h++) *(loose<__bf16, W>*)(p + h * plane) = q[h];
  }
}

// What becomes of W consecutive values of row m from column n on (all of them there).
// held: the row belongs to a group (its product counts); bias, residual: of these values (0 where there is none).
template <class T, int W, class P>
__device__ __forceinline__ void finish_linear(const P& p, int64_t m, int64_t n, float* v, const float* bias, const float* residual, bool held) {
  constexpr bool EXACT = sizeof(T) == 4;
#pragma unroll
  for (int t = 0; t < W; t++) v[t] = held ? v[t] + bias[t] : 0.f;
  if (p.pre) store_row<T, W>((T*)p.pre + m * p.ldp + n, v);
  if (held) act_of<EXACT, W>(v, p.act);
#pragma unroll
  for (int t = 0; t < W; t++) v[t] += residual[t];
  store_row<T, W>((T*)p.out + m * p.ldc + n, v);
}
template <class T, int W, class P>
__device__ __forceinline__ void finish_store(const P& p, int64_t sheet, int64_t m, int64_t n, float* v) {
  const int64_t at = sheet * p.c_split + m * p.ldc + n;
  if (p.add_sums) {
    float r[W];
    load_row<float, W>(p.sums + at, r);
#pragma unroll
    for (int t = 0; t < W; t++) v[t] += r[t];
  }
  if (!p.out) {
    store_row<float, W>(p.sums + at, v);
    return;
  }
  const int64_t to = sheet * p.c_group + m * p.ldo + n;
  const float s = p.scale ? *p.scale : 1.f;
#pragma unroll
  for (int t = 0; t < W; t++) {
    v[t] *= s;
    if (p.square) v[t] *= v[t];
  }
  if (p.out_f32)
    store_row<float, W>((float*)p.out + to, v, p.past);
  else
    store_row<T, W>((T*)p.out + to, v, p.past);
}
// (softmax - label) times the token's weight; the piece's columns past the last word are zero
struct token {
  int label;
  float lse, dloss;
};
template <class T, int W, class P>
__device__ __forceinline__ void finish_grad(const P& p, int64_t m, int64_t n, float* v, const token& t, float shrink) {
  const int32_t label = t.label;
  const float lse = t.lse, w = label >= p.words ? __builtin_nanf("") : t.dloss * shrink;
  const int64_t place = label - (p.word0 + n);
  const int mine = place >= 0 && place < W ? (int)place : -1, there = label < 0 || n >= p.N ? 0 : p.N - n < W ? (int)(p.N - n) : W;
#pragma unroll
  for (int t = 0; t < W; t++) {
    const float g = (__expf(v[t] - lse) - (t == mine ? 1.f : 0.f)) * w;
    v[t] = t < there ? g : 0.f;
  }
  store_op<T, W>((typename num<T>::op*)p.out + m * p.ldc + n, p.M * p.ldc, v);
}
template <class T, int W, class P>
__device__ __forceinline__ void bias_of(const P& p, int64_t n, int group, bool held, float* b) {
#pragma unroll
  for (int t = 0; t < W; t++) b[t] = 0.f;
  if (p.bias && held) load_row<T, W>((const T*)p.bias + (int64_t)group * p.N + n, b);
}

template <class T, int W, class P>
__device__ __forceinline__ void residual_of(const P& p, int64_t m, int64_t n, float* r) {
#pragma unroll
  for (int t = 0; t < W; t++) r[t] = 0.f;
  if (p.residual) load_row<T, W>((const T*)p.residual + m * p.ldr + n, r);
}

// A buffer load of 16 bytes per lane to LDS: lane l's go to lds + 16 l.  The compiler does not see what the load needs: a wait
// state after m0's write, given here, and five after a lane's write of the buffer's words.  These are given before the first
// stages, where the words come from lanes; later ones are scalar work, and a test looks for such writes in the built code
// (given with each load, they cost small fp32 products 2 % and large ones 0.6; once a stage, large ones 0.8).
__device__ __forceinline__ void to_lds(v4i buffer, unsigned lds, int offset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(buffer) : "memory");
}
__device__ __forceinline__ int64_t uniform(int64_t v) {
  const unsigned lo = __builtin_amdgcn_readfirstlane((int)(unsigned)v), hi = __builtin_amdgcn_readfirstlane((int)((uint64_t)v >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}

// One operand's part of a stage: R of its own index, 128 bytes of the reduction, in N loads of 1 KB by each wave.  A stage's
// buffer begins at the wave's first row and ends with the operand: what lies past that arrives as zeros, as do pieces of a row
// past the reduction's end (their offset is past any buffer's).  What is read of the own index between its end and a row's
// makes results that nobody takes.
template <class T, int R, int THREADS, bool ROWS_OF_K>
struct operand {
  static constexpr int S = 2, CH = 8, BK = 64;
  static_assert(sizeof(T) == 2, "operands are of 16 bits");
  static constexpr int PER_ROW = ROWS_OF_K ? 8 : R / 8;  // pieces in a row
  static constexpr int N = R * 8 / THREADS, ROWS = 64 / PER_ROW;
  static constexpr int NOWHERE = (int)0x80000000u;
  int64_t at, end;  // addresses: this wave's first row of the next stage, the operand's end
  int64_t at0, end0;
  int64_t step;     // bytes from a stage to the next
  int offset[N];
  int k[2];         // (rows of k) a lane's place in the reduction, in even and odd loads
  v4i buffer;
  bool in[2];

  __device__ static __forceinline__ int swizzle(int row) {
    if (ROWS_OF_K) return (row >> 1) & 7;
    return (((row & 3) | ((row >> 1) & 4)) << 1) & (PER_ROW - 1);
  }
  // there: how many of the operand's own index exist from own0 on; k_end: the reduction's end.
  __device__ __forceinline__ void start(const T* p, int64_t ld, int64_t own0, int64_t k0, int64_t k_end, int there, int tid) {
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    ld *= S;
    const int64_t first = (int64_t)p + (ROWS_OF_K ? own0 * ld : own0 * S);
    at = uniform(first + (ROWS_OF_K ? k0 * S : k0 * ld) + wave * N * ROWS * ld);
    end = uniform(first + (ROWS_OF_K ? (there - 1) * ld + (k_end + CH - 1) / CH * 16 : (k_end - 1) * ld + (int64_t)(there + CH - 1) / CH * 16));
    at0 = at, end0 = end;
    step = uniform(ROWS_OF_K ? 128 : BK * ld);
#pragma unroll
    for (int e = 0; e < N; e++) {
      const int row = (wave * N + e) * ROWS + lane / PER_ROW, c = (lane % PER_ROW) ^ swizzle(row);
      offset[e] = (int)((e * ROWS + lane / PER_ROW) * ld) + c * 16;
      if (e < 2) k[e] = c * CH;
    }
  }
  // A stage's loads, one by one: begin() says how much of the reduction is left (or nothing: zeros), load() makes the e-th
  // of N, end_stage() goes on to the next.
  __device__ __forceinline__ void begin(int left) {
    const int64_t r = end - at;
    buffer = v4i{(int)(unsigned)(uint64_t)at, (int)(((uint64_t)at >> 32) & 0xffff), r < 0 ? 0 : r > 0x7fffffff ? 0x7fffffff : (int)r, 0x00020000};
#pragma unroll
    for (int h = 0; h < 2; h++) in[h] = !ROWS_OF_K || k[h] < left;
  }
  __device__ __forceinline__ void load(unsigned to, int e) const { to_lds(buffer, to + e * 1024, in[e & 1] ? offset[e] : NOWHERE); }
  __device__ __forceinline__ void end_stage() { at += step; }
  __device__ __forceinline__ void to_plane(int64_t elements) {  // back to the first stage, of another plane
    at = at0 + elements * S;
    end = end0 + elements * S;
  }
};

// How a lane reads an operand's part of a tile: 16 of its index, `own` + 16 i .. + 15, for 64 bytes of the reduction (the s-th half).
template <class T, int R, bool ROWS_OF_K>
struct reader {
  typedef typename num<T>::piece piece;
  unsigned lane_at[2];  // rows of k: by half
  __device__ __forceinline__ void start(int own, int lane) {
    const int q = lane >> 4, i = lane & 15;
    if (ROWS_OF_K) {
      lane_at[0] = (own + i) * 128 + ((q ^ (i >> 1)) << 4);
      lane_at[1] = lane_at[0] ^ 64;
    } else {
      const int r = i >> 2, col = own + (i & 3) * 4, swz = ((r | ((q & 1) << 2)) << 1) & (R / 8 - 1);
      lane_at[0] = (q * 8 + r) * (R * 2) + (((col >> 3) ^ swz) << 4) + (col & 4) * 2;
    }
  }
  __device__ __forceinline__ piece read(unsigned lds, int i, int s) const {
    if (ROWS_OF_K) {
      return *(const DN_LDS piece*)(lds_at<const char>(lds + lane_at[s]) + i * 2048);
    } else {
      DN_LDS char* p = lds_at<char>(lds + (lane_at[0] ^ (i << 5)));
      union {
        v4s h[2];
        piece p;
      } u;
      u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((DN_LDS v4s*)(p + s * 32 * (R * 2)));
      u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((DN_LDS v4s*)(p + (s * 32 + 4) * (R * 2)));
      return u.p;
    }
  }
};

// Everything of this wave's but the last N loads to LDS has arrived, all its LDS reads are done, and so for every wave.
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// A workgroup's tile: sums over k0 .. k_end of rows m0 .. m_end and columns from n0 on.
template <class T>
struct place {
  const typename num<T>::op *A, *B;
  int64_t m0, m_end, n0, k0, k_end;
  int sheet, tn, group;
  bool held;  // (BY_ROWS) the rows belong to a group
};

// What becomes of a tile's sums.
template <class T, int BM, int BN, int WM, int WN, int E>
__device__ __forceinline__ void finish_tile(kargs& p, const place<T>& w, v4f (&acc)[BM / WM / 16][BN / WN / 16], unsigned room, int tid,
                                            int wave) {
  constexpr int FM = BM / WM / 16, FN = BN / WN / 16, THREADS = WM * WN * 64;
  asm volatile("" : "+v"(tid));  // (what follows from it is worked out here, not kept over the products)
  const int lane = tid & 63;
  const int wm = wave / WN, wn = wave % WN, q = lane >> 4;
  const int64_t m_wave = w.m0 + wm * (BM / WM), n_wave = w.n0 + wn * (BN / WN), m_end = w.m_end;
  if constexpr (E != E_LOSS) {
    // Each wave by itself, 64 of its rows at a time: through LDS, so that its lanes take consecutive values of a row, and
    // whole lines go out.  Piece c of row r at c ^ (r & 15).  (The rows go by in a loop: unrolled over all of them the code
    // would not fit the instruction cache.)
    constexpr int COLS = BN / WN, BLOCKS = 4;
    static_assert(COLS == 64 && FM % BLOCKS == 0, "a row of a wave's part is 16 pieces of 16 bytes");
    const unsigned mine = room + wave * (BLOCKS * 4096);
    const int64_t n_end = E == E_LOSS_GRAD ? p.ldc : p.N;
    if (n_wave >= n_end) return;
    const float shrink = E == E_LOSS_GRAD && p.shrink ? *p.shrink : 1.f;
    // Rows m_top .. of 64: W values a lane, `lanes` side by side.  Where the columns end within a wave's part (tail) the last
    // lane begins as much earlier as makes its values whole: both lanes have the same for what they share.
    const int cols = n_end - n_wave < COLS ? (int)(n_end - n_wave) : COLS;
    auto rows_out = [&](auto width, auto lanes, auto tail, int64_t m_top) {
      constexpr int W = decltype(width)::value, PER_ROW = decltype(lanes)::value, STEP = 64 / PER_ROW;
      constexpr int AT_ONCE = STEP >= 16 ? 64 / STEP : 4;
      const int r_lane = lane / PER_ROW, l = lane % PER_ROW * W;
      const bool in = !tail || l < cols;
      const int c = !tail || l + W <= cols ? l : cols - W;
      const int64_t n = n_wave + c;
      const int last = (int)(m_end - m_top - 1);
      typedef loose<T, W> piece;
      float bias[W];
      piece more[AT_ONCE], next[AT_ONCE];  // the residual of a turn's rows, and of the next turn's
      token these[AT_ONCE], those[AT_ONCE];  // what the loss needs of them
      auto fetch = [&](int r0) {
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++) {
          const int r = r0 + u * STEP + r_lane;
          const int64_t m = m_top + (r < last ? r : last);
          if constexpr (E == E_LOSS_GRAD)
            those[u] = token{p.labels[m], p.lse[m], p.dloss[m]};
          else
            next[u] = *(const piece*)((const T*)p.residual + m * p.ldr + n);
        }
      };
      if constexpr (E == E_LINEAR) {
        bias_of<T, W>(p, n, w.group, w.held, bias);
        if (p.residual) fetch(0);
      }
      if constexpr (E == E_LOSS_GRAD) fetch(0);
#pragma unroll 1
      for (int r0 = 0; r0 < 16 * BLOCKS && r0 <= last; r0 += STEP * AT_ONCE) {
        if (E == E_LINEAR && p.residual) {
#pragma unroll
          for (int u = 0; u < AT_ONCE; u++) more[u] = next[u];
          fetch(r0 + STEP * AT_ONCE);
        }
        if constexpr (E == E_LOSS_GRAD) {
#pragma unroll
          for (int u = 0; u < AT_ONCE; u++) these[u] = those[u];
          fetch(r0 + STEP * AT_ONCE);
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++) {
          const int r = r0 + u * STEP + r_lane;
          float v[W];
          if constexpr (tail) {
#pragma unroll
            for (int e = 0; e < W; e++)
              v[e] = *lds_at<float>(mine + r * 256 + ((((c + e) >> 2) ^ (r & 15)) << 4) + ((c + e) & 3) * 4);
          } else {
#pragma unroll
            for (int k = 0; k < W / 4; k++) {
              const v4f x = *lds_at<v4f>(mine + r * 256 + (((c / 4 + k) ^ (r & 15)) << 4));
#pragma unroll
              for (int e = 0; e < 4; e++) v[k * 4 + e] = x[e];
            }
          }
          if (r <= last && in) {
            const int64_t m = m_top + r;
            if constexpr (E == E_LINEAR) {
              float res[W];
#pragma unroll
              for (int e = 0; e < W; e++) res[e] = p.residual ? (float)more[u][e] : 0.f;
              finish_linear<T, W>(p, m, n, v, bias, res, w.held);
            } else if constexpr (E == E_LOSS_GRAD) {
              finish_grad<T, W>(p, m, n, v, these[u], shrink);
            } else {
              finish_store<T, W>(p, w.sheet, m, n, v);
            }
          }
        }
      }
    };
#pragma unroll
    for (int i0 = 0; i0 < FM; i0 += BLOCKS) {
      const int64_t m_top = m_wave + i0 * 16;
      if (m_top >= m_end) return;
      asm volatile("" ::: "memory");  // (a wave's LDS accesses happen in their order: the compiler is to keep it too)
#pragma unroll
      for (int i = 0; i < BLOCKS; i++)
#pragma unroll
        for (int j = 0; j < FN; j++)
          *lds_at<v4f>(mine + (i * 16 + (lane & 15)) * 256 + (((j * 4 + q) ^ (lane & 15)) << 4)) = acc[i0 + i][j];
      asm volatile("" ::: "memory");
      constexpr int W = 16 / sizeof(T);
      typedef std::integral_constant<int, 1> one;
      typedef std::integral_constant<int, 2> two;
      typedef std::integral_constant<int, 4> four;
      typedef std::integral_constant<int, W> full;
      if (cols == COLS) {
        if (E == E_STORE && W != 4 && (!p.out || p.out_f32))  // (16 bytes of fp32)
          rows_out(four(), std::integral_constant<int, 16>(), std::false_type(), m_top);
        else
          rows_out(full(), std::integral_constant<int, 64 / W>(), std::false_type(), m_top);
      } else if (E != E_LOSS_GRAD) {  // (a row of g is whole waves' parts)
        if (cols >= W)
          rows_out(full(), std::integral_constant<int, 64 / W>(), std::true_type(), m_top);
        else if (cols >= 4)
          rows_out(four(), two(), std::true_type(), m_top);
        else if (cols >= 2)
          rows_out(two(), two(), std::true_type(), m_top);
        else
          rows_out(one(), one(), std::true_type(), m_top);
      }
    }
  } else {
    // The maximum and the sum of exponentials of the tile's words for every row: over the lane's own, the four
    // lane groups, the waves side by side (through LDS).
    __syncthreads();
    DN_LDS float2* side = lds_at<float2>(room);  // [WN][BM]
    const int m_there = (int)(m_end - w.m0 < BM ? m_end - w.m0 : BM);
    const bool whole = n_wave + FN * 16 <= p.N;
    const int there = whole ? FN * 16 : (int)(p.N - n_wave < 0 ? 0 : p.N - n_wave) - q * 4;
    int labels[FM];  // (asked for together)
#pragma unroll
    for (int i = 0; i < FM; i++) {
      const int64_t m = m_wave + i * 16 + (lane & 15);
      labels[i] = p.labels[m < m_end ? m : m_end - 1];
    }
#pragma unroll
    for (int i = 0; i < FM; i++) {
      const int64_t m = m_wave + i * 16 + (lane & 15);
      // (the label's column among the lane's, or none)
      const int64_t place = m < m_end ? labels[i] - (n_wave + q * 4) : -1;
      const int mine = place >= 0 && place < 64 && labels[i] < p.N ? (int)place : -1;
      float top = -INFINITY, hit = 0.f;
      if (whole) {
#pragma unroll
        for (int j = 0; j < FN; j++)
#pragma unroll
          for (int e = 0; e < 4; e++) top = fmaxf(top, acc[i][j][e]);
      } else {
#pragma unroll
        for (int j = 0; j < FN; j++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            if (j * 16 + e >= there) acc[i][j][e] = -INFINITY;
            top = fmaxf(top, acc[i][j][e]);
          }
      }
#pragma unroll
      for (int j = 0; j < FN; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) hit = j * 16 + e == mine ? acc[i][j][e] : hit;
      if (mine >= 0 && (mine & 15) < 4) p.hit[m] = hit;
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float from = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < FN; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) sum += __expf(acc[i][j][e] - from);
      sum += __shfl_xor(sum, 16, 64);
      sum += __shfl_xor(sum, 32, 64);
      if (q == 0) {
        side[wn * BM + wm * (BM / WM) + i * 16 + lane].x = top;
        side[wn * BM + wm * (BM / WM) + i * 16 + lane].y = sum;
      }
    }
    __syncthreads();
    for (int m = tid; m < m_there; m += THREADS) {
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int v = 0; v < WN; v++) top = fmaxf(top, side[v * BM + m].x);
      const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int v = 0; v < WN; v++) {
        const float x = side[v * BM + m].x, y = side[v * BM + m].y;
        if (x != -INFINITY || y != 0.f) sum += y * __expf(x - from);
      }
      p.parts[(w.m0 + m) * p.parts_n + p.part0 + w.tn] = float2{top, sum};
    }
  }
}

// A launch's dimension holds 2^32 lanes (more are cut off without an error): workgroups past 2^22 go on in its second.  (A
// multiple of 8, for the XCDs.)
constexpr int64_t GRID_X = (int64_t)1 << 22;
inline dim3 grid_of(int64_t blocks) { return dim3((unsigned)(blocks < GRID_X ? blocks : GRID_X), (unsigned)ceil_div(blocks, GRID_X)); }
__device__ __forceinline__ unsigned block_id() { return blockIdx.y * gridDim.x + blockIdx.x; }

template <class T, int BM, int BN, int WM, int WN, bool A_ROWS, bool B_ROWS, int E>
__global__ __launch_bounds__(WM* WN * 64, 2) void k_tiles(args p) {
  typedef typename num<T>::op O;
  constexpr int THREADS = WM * WN * 64, BK = 64, TERMS = num<T>::TERMS;
  constexpr int FM = BM / WM / 16, FN = BN / WN / 16, STAGE = (BM + BN) * 128, N_LOADS = STAGE / 16 / THREADS;
  __shared__ __align__(16) char smem[2 * STAGE];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / WN, wn = wave % WN;
  const int q = lane >> 4;
  const unsigned base = (unsigned)(uintptr_t)(DN_LDS char*)smem;

  // -- which tiles --
  const int nt = (int)((p.N + BN - 1) / BN) - p.tn_first;
  const int mt = __builtin_amdgcn_readfirstlane(p.mode == BY_ROWS ? group_tiles(p.G, BM, lane) : (int)((p.M + BM - 1) / BM) - p.tm_first);
  const int plane = mt * nt, many = plane * (p.mode == BY_REDUCTION ? p.G.groups : p.splits);
  // Workgroups go to the XCDs round-robin: each XCD gets a run of tiles, in blocks of a few tiles of m by all of n, so
  // that what its workgroups read at one time is shared in its L2.
  const unsigned id = block_id();
  const int xcd = id % 8, share = many / 8, more = many % 8;
  if ((int)id >= many) return;
  const int tile = xcd * share + (xcd < more ? xcd : more) + id / 8;
  place<T> w;
  w.A = (const O*)p.A, w.B = (const O*)p.B;
  w.sheet = tile / plane;
  const int on = tile % plane;
  constexpr int HIGH = BM >= 256 ? 4 : 8;
  const int block = on / (HIGH * nt), in_block = on % (HIGH * nt);
  const int high = mt - block * HIGH < HIGH ? mt - block * HIGH : HIGH;
  const int tm = block * HIGH + in_block % high;
  w.tn = in_block / high;
  w.n0 = (int64_t)(w.tn + p.tn_first) * BN;
  w.k0 = 0, w.k_end = p.K;
  w.group = 0, w.held = true;
  if (p.mode == BY_ROWS) {
    int within;
    group_of_tile(p.G, BM, lane, tm, &w.group, &within);
    if (w.group < 0) w.group = p.G.groups;  // (not reached: there are `mt` of them)
    w.m0 = p.G.one_first(w.group) + (int64_t)within * BM;
    w.m_end = p.G.one_last(w.group);
    w.held = w.group < p.G.groups;
    if (w.held)
      w.B += w.group * p.b_group;
    else
      w.k_end = 0;
  } else {
    w.m0 = (int64_t)(tm + p.tm_first) * BM;
    w.m_end = p.M;
    if (p.mode == BY_REDUCTION) {
      w.group = w.sheet;
      w.k0 = p.G.one_first(w.group);
      w.k_end = p.G.one_last(w.group);
    } else if (p.splits > 1) {
      w.k0 = w.sheet * p.split_k;
      w.k_end = w.k0 + p.split_k < p.K ? w.k0 + p.split_k : p.K;
    }
  }

  operand<O, BM, THREADS, A_ROWS> a;
  operand<O, BN, THREADS, B_ROWS> b;
  reader<O, BM, A_ROWS> ra;
  reader<O, BN, B_ROWS> rb;
  ra.start(wm * (BM / WM), lane);
  rb.start(wn * (BN / WN), lane);
  constexpr int LA = operand<O, BM, THREADS, A_ROWS>::N, LB = operand<O, BN, THREADS, B_ROWS>::N;
  const int64_t length = uniform(w.k_end - w.k0);
  int64_t to_load = length;  // of the term that is being loaded
  int term = 0;
  auto begin = [&]() {
    const int to_go = to_load < 0 ? 0 : to_load > BK ? BK : (int)to_load;
    a.begin(to_go);
    b.begin(to_go);
  };
  auto load = [&](unsigned stage, int e) {
    if (e < LA)
      a.load(stage + wave * (LA * 1024), e);
    else if (e < LA + LB)
      b.load(stage + BM * 128 + wave * (LB * 1024), e - LA);
  };
  auto end_stage = [&]() {
    a.end_stage();
    b.end_stage();
    to_load -= BK;
    if (TERMS > 1 && to_load <= 0 && term + 1 < TERMS) {
      term++;
      to_load = length;
      a.to_plane(plane_a(term) * p.a_plane);
      b.to_plane(plane_b(term) * p.b_plane);
    }
  };
  v4f acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; i++)
#pragma unroll
    for (int j = 0; j < FN; j++) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
  // Two stages of 128 bytes of the reduction each, in two halves.  A lane's operands of one half are read while the matrix
  // cores work on the other's; once everyone has read the second half, the stage takes the one after the next, load by load
  // between products: nothing but the barrier keeps the matrix cores waiting.  (Four stages of the small tiles where a CU has
  // one: 333 x 10007 x 515 in fp32 49 us instead of 43.)
  int64_t left = length > 0 ? (length + BK - 1) / BK * TERMS : 0;  // stages
  if (left > 0) {
    a.start(w.A, p.lda, w.m0, w.k0, w.k_end, (int)(w.m_end - w.m0 < BM ? w.m_end - w.m0 : BM), tid);
    b.start(w.B, p.ldb, w.n0, w.k0, w.k_end, (int)(p.N - w.n0 < BN ? p.N - w.n0 : BN), tid);
    if (TERMS > 1) {
      a.to_plane(plane_a(0) * p.a_plane);
      b.to_plane(plane_b(0) * p.b_plane);
    }
    auto whole_stage = [&](unsigned stage) {
      begin();
      asm volatile("s_nop 4");  // (between a lane's write of an address and the loads)
#pragma unroll
      for (int e = 0; e < LA + LB; e++) load(stage, e);
      end_stage();
    };
    whole_stage(base);
    if (left > 1) {
      whole_stage(base + STAGE);
      wait_loads<N_LOADS>();
    } else {
      wait_loads<0>();
    }
    typename num<O>::piece fa[2][FM], fb[2][FN];
    auto read = [&](unsigned stage, int s, int r) {
      if (r < FN)
        fb[s][r] = rb.read(stage + BM * 128, r, s);
      else if (r < FN + FM)
        fa[s][r - FN] = ra.read(stage, r - FN, s);
    };
    // The products of half s, row by row, with the reads of the other half in the first rows' company.
    constexpr int READS = (FN + FM + FM - 3) / (FM - 2), LOADS = (LA + LB + FM - 1) / FM;
    auto products = [&](unsigned stage, int s, bool reads, bool loads, unsigned free) {
#pragma unroll
      for (int i = 0; i < FM; i++) {
        if (reads) {
#pragma unroll
          for (int r = i * READS; r < i * READS + READS; r++) read(stage, 1 - s, r);
        }
        if (loads) {
#pragma unroll
          for (int e = i * LOADS; e < i * LOADS + LOADS; e++) load(free, e);
        }
#pragma unroll
        for (int j = 0; j < FN; j++) acc[i][j] = mma(fb[s][j], fa[s][i], acc[i][j]);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    unsigned here = base, there = base + STAGE;
#pragma unroll
    for (int r = 0; r < FN + FM; r++) read(here, 0, r);
    while (left > 1) {
      products(here, 0, true, false, 0);
      // the next stage has arrived, and everyone has read this one
      wait_loads<0>();
      left--;
      begin();
      products(there, 1, true, true, here);
      end_stage();
      const unsigned x = here;
      here = there;
      there = x;
    }
    products(here, 0, true, false, 0);
    products(here, 1, false, false, 0);
    wait_loads<0>();  // (of zeros, and for everyone's reads)
  }

  finish_tile<T, BM, BN, WM, WN, E>(again(), w, acc, base, tid, wave);
}

// ---- few rows ----------------------------------------------------------------------------------------------------
// Products of at most 16 ROWS rows at a time with rows of k, bound by the one read of B: no LDS stages, every wave streams
// 16 COLS rows of B from memory straight to the matrix cores, eight loads of 1 KB ahead.  A workgroup's eight waves are `parts` of the
// reduction times 8 / parts blocks of 16 COLS columns; parts so that the chip has enough waves to keep its memory busy.  Groups
// (BY_ROWS): blockIdx.y counts those that hold rows; a group of more rows reads its B again for every 16 ROWS.
template <class T, int COLS, int ROWS, int E>
__global__ __launch_bounds__(512, 2) void k_few(args p, int parts) {
  typedef typename num<T>::piece piece;
  constexpr int CH = 16 / sizeof(T), STEP = 4 * CH, AHEAD = 8 / COLS;
  __shared__ v4f sums[COLS][8][64];
  __shared__ float2 stats[8][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int q = lane >> 4, part = wave % parts;
  const int64_t n0 = ((int64_t)blockIdx.x * (8 / parts) + wave / parts) * (16 * COLS);
  const T* B = (const T*)p.B;
  int64_t m0 = 0, m_end = p.M;
  int group = 0;
  bool held = true;
  if (p.mode == BY_ROWS) {
    int seen = 0;
    group = -1;
    for (int b = 0; b <= p.G.groups && group < 0; b += 64) {
      const int g = b + lane;
      const unsigned long long some = __ballot(g <= p.G.groups && p.G.count(g) > 0);
      const int before = __popcll(some & ((1ull << lane) - 1));
      const unsigned long long hit = __ballot(((some >> lane) & 1) && seen + before == (int)blockIdx.y);
      if (hit) group = b + __ffsll(hit) - 1;
      seen += __popcll(some);
    }
    group = __builtin_amdgcn_readfirstlane(group);
    if (group < 0) return;
    m0 = p.G.one_first(group);
    m_end = p.G.one_last(group);
    held = group < p.G.groups;
    if (held) B += group * p.b_group;
  }
  const T* b_row[COLS];
#pragma unroll
  for (int h = 0; h < COLS; h++) {
    const int64_t n = n0 + h * 16 + (lane & 15);
    b_row[h] = B + (n < p.N ? n : p.N - 1) * p.ldb + q * CH;
  }
  const int64_t steps = (p.K + STEP - 1) / STEP, each = (steps + parts - 1) / parts;
  const int64_t k_from = part * each * STEP, k_to = k_from + each * STEP < p.K ? k_from + each * STEP : p.K;
  for (; m0 < m_end; m0 += 16 * ROWS) {
    const T* a_row[ROWS];
    v4f sum[ROWS][COLS];
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
      const int64_t m = m0 + r * 16 + (lane & 15);
      a_row[r] = (const T*)p.A + (m < m_end ? m : m_end - 1) * p.lda + q * CH;
#pragma unroll
      for (int h = 0; h < COLS; h++) sum[r][h] = v4f{0.f, 0.f, 0.f, 0.f};
    }
    if (held && n0 < p.N) {
      int64_t k = k_from;
      for (; k + AHEAD * STEP <= k_to; k += AHEAD * STEP) {
        loose<T, CH> fb[AHEAD][COLS], fa[AHEAD][ROWS];
#pragma unroll
        for (int u = 0; u < AHEAD; u++)
#pragma unroll
          for (int h = 0; h < COLS; h++) fb[u][h] = *(const loose<T, CH>*)(b_row[h] + k + u * STEP);
#pragma unroll
        for (int u = 0; u < AHEAD; u++)
#pragma unroll
          for (int r = 0; r < ROWS; r++) fa[u][r] = *(const loose<T, CH>*)(a_row[r] + k + u * STEP);
#pragma unroll
        for (int u = 0; u < AHEAD; u++)
#pragma unroll
          for (int r = 0; r < ROWS; r++)
#pragma unroll
            for (int h = 0; h < COLS; h++) sum[r][h] = mma((piece)fb[u][h], (piece)fa[u][r], sum[r][h]);
      }
      for (; k < k_to; k += STEP) {
        piece fb[COLS], fa[ROWS];
        const int there = p.K - k - q * CH < CH ? (int)(p.K - k - q * CH) : CH;
        if (there == CH) {
#pragma unroll
          for (int h = 0; h < COLS; h++) fb[h] = *(const loose<T, CH>*)(b_row[h] + k);
#pragma unroll
          for (int r = 0; r < ROWS; r++) fa[r] = *(const loose<T, CH>*)(a_row[r] + k);
        } else {
#pragma unroll
          for (int e = 0; e < CH; e++) {
#pragma unroll
            for (int h = 0; h < COLS; h++) fb[h][e] = e < there ? b_row[h][k + e] : (T)0.f;
#pragma unroll
            for (int r = 0; r < ROWS; r++) fa[r][e] = e < there ? a_row[r][k + e] : (T)0.f;
          }
        }
#pragma unroll
        for (int r = 0; r < ROWS; r++)
#pragma unroll
          for (int h = 0; h < COLS; h++) sum[r][h] = mma(fb[h], fa[r], sum[r][h]);
      }
    }
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
      const int64_t m_top = m0 + r * 16;
      if (m_top >= m_end) break;
      v4f acc[COLS];
#pragma unroll
      for (int h = 0; h < COLS; h++) acc[h] = sum[r][h];
      if (parts > 1) {
        __syncthreads();  // (of the rows before)
#pragma unroll
        for (int h = 0; h < COLS; h++) sums[h][wave][lane] = acc[h];
        __syncthreads();
        if (part == 0)
          for (int w = 1; w < parts; w++)
#pragma unroll
            for (int h = 0; h < COLS; h++) acc[h] += sums[h][wave + w][lane];
      }
      const int64_t m = m_top + (lane & 15);
      if constexpr (E == E_LINEAR) {
#pragma unroll
        for (int h = 0; h < COLS; h++) {
          const int64_t n = n0 + h * 16 + q * 4;
          if (part != 0 || m >= m_end || n >= p.N) continue;
          float v[4] = {acc[h][0], acc[h][1], acc[h][2], acc[h][3]}, b[4], add[4];
          if (n + 4 <= p.N) {
            bias_of<T, 4>(p, n, group, held, b);
            residual_of<T, 4>(p, m, n, add);
            finish_linear<T, 4>(p, m, n, v, b, add, held);
          } else {
#pragma unroll
            for (int t = 0; t < 3; t++) {
              if (n + t >= p.N) break;
              bias_of<T, 1>(p, n + t, group, held, b);
              residual_of<T, 1>(p, m, n + t, add);
              finish_linear<T, 1>(p, m, n + t, v + t, b, add, held);
            }
          }
        }
      } else if constexpr (E == E_LOSS_GRAD) {
        // (at most 16 rows) out: fp32, [words][16]
        if (part == 0) {
          const int64_t label = m < m_end ? (int64_t)p.labels[m] : -1;
          const float lse = label < 0 ? 0.f : p.lse[m], w = label < 0 ? 0.f : label >= p.words ? __builtin_nanf("") : p.dloss[m];
#pragma unroll
          for (int h = 0; h < COLS; h++)
#pragma unroll
            for (int t = 0; t < 4; t++) {
              const int64_t n = n0 + h * 16 + q * 4 + t;
              const float g = label < 0 ? 0.f : (__expf(acc[h][t] - lse) - (n == label ? 1.f : 0.f)) * w;
              if (n < p.N) ((float*)p.out)[n * 16 + (lane & 15)] = g;
            }
        }
      } else {
        if (part == 0) {
          const int64_t label = m < m_end ? (int64_t)p.labels[m] : -1;
          float top = -INFINITY, sum = 0.f;
#pragma unroll
          for (int h = 0; h < COLS; h++)
#pragma unroll
            for (int t = 0; t < 4; t++) {
              const int64_t n = n0 + h * 16 + q * 4 + t;
              if (n < p.N) top = fmaxf(top, acc[h][t]);
              if (n == label && n < p.N) p.hit[m] = acc[h][t];
            }
          top = fmaxf(top, __shfl_xor(top, 16, 64));
          top = fmaxf(top, __shfl_xor(top, 32, 64));
          const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
          for (int h = 0; h < COLS; h++)
#pragma unroll
            for (int t = 0; t < 4; t++)
              if (n0 + h * 16 + q * 4 + t < p.N) sum += __expf(acc[h][t] - from);
          sum += __shfl_xor(sum, 16, 64);
          sum += __shfl_xor(sum, 32, 64);
          if (q == 0) stats[wave][lane] = float2{top, sum};
        }
        __syncthreads();
        if (threadIdx.x < 16 && m_top + threadIdx.x < m_end) {
          float top = -INFINITY, sum = 0.f;
          for (int w = 0; w < 8; w += parts) top = fmaxf(top, stats[w][threadIdx.x].x);
          const float from = top == -INFINITY ? 0.f : top;
          for (int w = 0; w < 8; w += parts) {
            const float2 s = stats[w][threadIdx.x];
            if (s.x != -INFINITY || s.y != 0.f) sum += s.y * __expf(s.x - from);
          }
          p.parts[(m_top + threadIdx.x) * p.parts_n + blockIdx.x] = float2{top, sum};
        }
        __syncthreads();
      }
    }
  }
}

// ---- host --------------------------------------------------------------------------------------------------------
// Partial sums of a split reduction, added in their order, then as the tiles' own epilogue.
template <class T, int E>
__global__ __launch_bounds__(256) void k_join(args p, const float* parts, int splits) {
  const int64_t row = (p.N + 3) / 4 * 4, per_row = row / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= p.M * per_row) return;
  const int64_t m = i / per_row, n = i % per_row * 4;
  v4f v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < splits; s++) v += *(const v4f*)(parts + ((int64_t)s * p.M + m) * row + n);
  float x[4] = {v[0], v[1], v[2], v[3]}, b[4], r[4];
  if (n + 4 <= p.N) {
    if constexpr (E == E_LINEAR) {
      bias_of<T, 4>(p, n, 0, true, b);
      residual_of<T, 4>(p, m, n, r);
      finish_linear<T, 4>(p, m, n, x, b, r, true);
    } else {
      finish_store<T, 4>(p, 0, m, n, x);
    }
  } else {
#pragma unroll
    for (int t = 0; t < 4; t++) {
      if (n + t >= p.N) break;
      if constexpr (E == E_LINEAR) {
        bias_of<T, 1>(p, n + t, 0, true, b);
        residual_of<T, 1>(p, m, n + t, r);
        finish_linear<T, 1>(p, m, n + t, x + t, b, r, true);
      } else {
        finish_store<T, 1>(p, 0, m, n + t, x + t);
      }
    }
  }
}

inline int64_t round256(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// How a product is run: with tiles of 256 x 256 (eight waves, one workgroup per CU) or of 128 x 128 (four
// waves, two per CU), and with the reduction split over workgroups where tiles are few.  What is least by these times, in us,
// measured on products of 1 to 8192 rows: a stage of a round of large tiles (256 at once) 1.6, of small ones (512 at once)
// 1.0 (with a CU each 0.7), fp32 six times that; what a round costs besides 8 and 5; a join 5 and its bytes at 4 TB/s.
// 8192 x 4096 x 16384 in bf16 is 927 us in large tiles, 1186 in small ones.
// Large tiles that leave the last round partly empty are cut: as many strips of columns (or of rows) as make whole rounds, and
// small tiles in a launch of their own for the rest.  Uncut and cut, in us: 2048 x 17880 x 4096 276 and 242, 3000 x 21976 x 768 131
// and 122, 1000 x 134360 x 512 with the loss 154 and 149.  Not after a single round of less than 32 stages, where small
// tiles alone are as fast or faster (2048 x 8920 x 1024: 52 against 56; with 4096 in place of 1024 152 and 145).
struct plan {
  bool big;
  int splits;
  int64_t split_k;
  int64_t m_cut, n_cut;  // rows or columns of the large tiles (0: all)
};
enum { NO_CUT = 0, CUT_N = 1, CUT_BOTH = 2 };
constexpr int64_t MOST_SPLITS = 32;
constexpr int64_t FEW_WAVES = 2048;  // eight on every CU
// Results of more bytes than this are stored past the caches: they would not be found there again, and push out what the
// product reads (64 experts' dW, 1 GB: 755 -> 715 us).
constexpr int64_t PAST_BYTES = (int64_t)128 << 20;
inline double rounds_of(double tiles, double at_once) { return tiles <= at_once ? 1.0 : (double)(int64_t)((tiles + at_once - 1) / at_once); }
// half_tiles: tiles of rows that groups leave half empty (BY_ROWS); sheets: products of this size in one launch.
template <class T>
inline plan plan_for(int64_t M, int64_t N, int64_t K, bool may_split, int cut, int64_t half_tiles = 0, int64_t sheets = 1) {
  constexpr int64_t BK = 64;
  plan best{false, 1, K, 0, 0};
  double least = 1e300;
  for (int big = 0; big < 2; big++) {
    const int64_t side = big ? 256 : 128;
    const double tiles = (double)(ceil_div(M, side) + half_tiles / 2) * ceil_div(N, side) * sheets, at_once = big ? 256 : 512;
    const double round = big ? 8.0 : 5.0;
    for (int64_t s = 1; s <= (may_split ? MOST_SPLITS : 1); s++) {
      const int64_t split_k = ceil_div(ceil_div(K, s), BK) * BK;
      if (s > 1 && (split_k < 2 * BK || (s - 1) * split_k >= K)) break;
      const bool one = tiles * s <= 256;  // workgroup on a CU
      const double stage = num<T>::TERMS * (big ? 1.6 : one ? 0.7 : 1.0);
      double us = rounds_of(tiles * s, at_once) * ((double)ceil_div(split_k, BK) * stage + round);
      if (s > 1) us += 5.0 + (double)s * M * N * 8.0 / 4e6;
      if (us < least) {
        least = us;
        best = plan{big != 0, (int)s, s > 1 ? split_k : K, 0, 0};
      }
    }
  }
  const int64_t tall = ceil_div(M, 256), wide = ceil_div(N, 256), rounds = tall * wide / 256;
  const double stages = (double)num<T>::TERMS * ceil_div(K, BK);
  const bool worth = rounds > 1 || (rounds == 1 && stages >= 32);
  for (int way = CUT_N; worth && way <= cut; way++) {
    const int64_t strip = way == CUT_N ? tall : wide, strips = rounds * 256 / strip;
    if (strips == 0 || strips >= (way == CUT_N ? wide : tall)) continue;
    const int64_t m_rest = way == CUT_N ? M : M - strips * 256, n_rest = way == CUT_N ? N - strips * 256 : N;
    const double rest = (double)ceil_div(m_rest, 128) * ceil_div(n_rest, 128);
    const double us = (double)ceil_div(strips * strip, 256) * (stages * 1.6 + 8.0) +
                      rounds_of(rest, 512) * (stages * (rest <= 256 ? 0.7 : 1.0) + 5.0) + 4.0;
    if (us < least) {
      least = us;
      best = plan{true, 1, K, way == CUT_N ? 0 : strips * 256, way == CUT_N ? strips * 256 : 0};
    }
  }
  return best;
}
// Floats that the partial sums of a split product take (0: it is not split).
template <class T>
inline int64_t split_floats(int64_t M, int64_t N, int64_t K) {
  const plan r = plan_for<T>(M, N, K, true, CUT_BOTH);
  return r.splits > 1 ? r.splits * M * (ceil_div(N, 4) * 4) : 0;
}

// ---- operands that tiles can be loaded from -----------------------------------------------------------------------
// A matrix of 16-bit values whose rows begin on 16 bytes and end on them is loaded as it lies; any other is first copied to rows
// that do, with zeros behind their ends (k_pack): once, where a tile's loads would come from any address again and again.  fp32
// is copied to its three planes, and a matrix whose rows do not all count to one where the others are zero (a product of zeros
// with them would not be: they may hold infinities or NaN).
struct matrix {
  const void* p;
  int64_t ld, rows, width;
  int64_t sheets, sheet;  // and so many such, so far apart
  int64_t plane;          // (packed fp32) and its planes
  const int32_t* keep;    // (NULL: all) rows of a negative word are copied as zeros, whatever they hold
};
template <class T>
inline bool lies_well(const matrix& m) {
  constexpr int64_t S = sizeof(T), NEAR = (int64_t)1 << 31;
  return S == 2 && m.keep == nullptr && (uintptr_t)m.p % 16 == 0 && m.ld * S % 16 == 0 && m.width * S % 16 == 0 && (m.sheets < 2 || m.sheet * S % 16 == 0) &&
         32 * m.ld * S < NEAR;
}
inline int64_t packed_ld(int64_t width) { return ceil_div(width, 64) * 64; }
template <class T>
inline int64_t packed_bytes(const matrix& m) {
  return lies_well<T>(m) ? 0 : round256(num<T>::PLANES * m.sheets * m.rows * packed_ld(m.width) * 2);
}
struct pack_args {
  matrix m[3];
  void* to[3];
  int64_t first[4];  // workgroups before each
};
// A lane makes eight values of a packed row.
template <class T>
__global__ __launch_bounds__(256) void k_pack(pack_args p) {
  constexpr int CH = 8;
  const int64_t id = block_id();
  const int w = id < p.first[1] ? 0 : id < p.first[2] ? 1 : 2;
  const matrix m = p.m[w];
  const int64_t ld = (m.width + 63) / 64 * 64, per_row = ld / CH;
  const int64_t at = (id - p.first[w]) * 256 + threadIdx.x, row = at / per_row;
  if (row >= m.rows * m.sheets) return;
  const int c = (int)(at - row * per_row) * CH, there = m.keep && m.keep[row] < 0 ? 0 : (int)(m.width - c);
  const T* src = (const T*)m.p + (m.sheets > 1 ? row / m.rows * m.sheet + row % m.rows * m.ld : row * m.ld) + c;
  float v[CH];
  if (there >= CH) {
    load_row<T, CH>(src, v);
  } else {
#pragma unroll
    for (int i = 0; i < CH; i++) v[i] = i < there ? (float)src[i] : 0.f;
  }
  store_op<T, CH>((typename num<T>::op*)p.to[w] + row * ld + c, m.sheets * m.rows * ld, v);
}
// Packs those of n matrices (at most 3) that do not lie well into `room`, and makes them the copies.
template <class T>
inline int pack(matrix* m, int n, char* room, hipStream_t st) {
  pack_args p{};
  int64_t blocks = 0;
  int k = 0;
  for (int i = 0; i < n; i++) {
    const int64_t bytes = packed_bytes<T>(m[i]);
    if (bytes == 0) continue;
    const int64_t ld = packed_ld(m[i].width);
    p.m[k] = m[i], p.to[k] = room, p.first[k] = blocks;
    blocks += ceil_div(m[i].sheets * m[i].rows * (ld / 8), 256);
    m[i].p = room, m[i].ld = ld, m[i].sheet = m[i].rows * ld, m[i].plane = m[i].sheets * m[i].sheet;
    room += bytes;
    k++;
  }
  if (blocks == 0) return 0;
  for (int i = k; i < 4; i++) p.first[i] = blocks;
  DN_CHECK(blocks < (int64_t)1 << 31, "operands of %lld MB that have to be copied", (long long)(blocks >> 8));
  k_pack<T><<<grid_of(blocks), 256, 0, st>>>(p);
  DN_LAUNCH_CHECK();
  return 0;
}

template <class T, int BM, int BN, int WM, int WN, bool A_ROWS, bool B_ROWS, int E>
int launch_tiles(const args& p, hipStream_t st) {
  const int64_t nt = ceil_div(p.N, BN) - p.tn_first;
  int64_t mt = ceil_div(p.M, BM) - p.tm_first, sheets = 1;
  if (p.mode == BY_ROWS)
    mt = p.G.most_tiles(BM);
  else
    sheets = p.mode == BY_REDUCTION ? p.G.groups : p.splits;
  const int64_t many = mt * nt * sheets;
  if (many == 0) return 0;
  DN_CHECK(many < (int64_t)1 << 31, "product of %lld x %lld: too many tiles for one launch", (long long)p.M, (long long)p.N);
  k_tiles<T, BM, BN, WM, WN, A_ROWS, B_ROWS, E><<<grid_of(many), WM * WN * 64, 0, st>>>(p);
  DN_LAUNCH_CHECK();
  return 0;
}

template <class T, bool A_ROWS, bool B_ROWS, int E>
int launch_size(const args& p, const plan& r, hipStream_t st) {
  if (r.big) return launch_tiles<T, 256, 256, 2, 4, A_ROWS, B_ROWS, E>(p, st);
  return launch_tiles<T, 128, 128, 2, 2, A_ROWS, B_ROWS, E>(p, st);
}

// A product whose args are complete but for splits; its operands lie well, or are packed.  ws: room for split_floats (NULL: the
// reduction is not split).  *parts_n (or NULL): the parts of a row that it leaves (E_LOSS).
template <class T, bool A_ROWS, bool B_ROWS, int E>
int launch_product(args p, float* ws, hipStream_t st, int* parts_n = nullptr) {
  p.splits = 1;
  p.split_k = p.K;
  p.c_split = 0;
  p.past = (p.mode == BY_REDUCTION ? p.G.groups : 1) * p.M * p.N * (p.out_f32 ? 4 : (int64_t)sizeof(T)) > PAST_BYTES;
  const int64_t groups = p.G.groups > 0 ? p.G.groups : 1;
  const int cut = E == E_LINEAR || E == E_STORE ? CUT_BOTH : CUT_N;
  const plan r = p.mode == BY_ROWS        ? plan_for<T>(p.M, p.N, p.K, false, NO_CUT, groups < p.M ? groups : p.M)
                 : p.mode == BY_REDUCTION ? plan_for<T>(p.M, p.N, ceil_div(p.K, groups), false, NO_CUT, 0, groups)
                                          : plan_for<T>(p.M, p.N, p.K, ws != nullptr, cut);
  const int64_t whole = r.n_cut / 256;
  p.parts_n = (int)(r.n_cut ? whole + ceil_div(p.N - r.n_cut, 128) : ceil_div(p.N, r.big ? 256 : 128));
  if (parts_n) *parts_n = p.parts_n;
  if (r.m_cut || r.n_cut) {
    args q = p;
    if (r.m_cut) q.M = r.m_cut, p.tm_first = (int)(r.m_cut / 128);
    if (r.n_cut) q.N = r.n_cut, p.tn_first = (int)(r.n_cut / 128);
    p.part0 = (int)whole;
    DN_TRY((launch_tiles<T, 256, 256, 2, 4, A_ROWS, B_ROWS, E>(q, st)));
    return launch_tiles<T, 128, 128, 2, 2, A_ROWS, B_ROWS, E>(p, st);
  }
  if constexpr (E == E_LINEAR || E == E_STORE) {
    if (r.splits > 1) {
      args q = p;
      q.splits = r.splits;
      q.split_k = r.split_k;
      q.sums = ws;
      q.out = nullptr;
      q.add_sums = 0;
      q.ldc = ceil_div(p.N, 4) * 4;
      q.c_split = p.M * q.ldc;
      DN_TRY((launch_size<T, A_ROWS, B_ROWS, E_STORE>(q, r, st)));
      const int64_t many = p.M * ceil_div(p.N, 4);
      k_join<T, E><<<(unsigned)ceil_div(many, 256), 256, 0, st>>>(p, ws, r.splits);
      DN_LAUNCH_CHECK();
      return 0;
    }
  }
  return launch_size<T, A_ROWS, B_ROWS, E>(p, r, st);
}

// (their kernels are in linear.hip)
#define DN_STORE_PRODUCTS(X, T)                                                              \
  X template int launch_product<T, true, false, E_STORE>(args, float*, hipStream_t, int*); \
  X template int launch_product<T, false, false, E_STORE>(args, float*, hipStream_t, int*);

// Few rows: how many, and a product of them (which takes its operands as they lie).  *parts_n as above.  fp32 has its packing to gain,
// and so more rows (us in tiles and here): 16384 x 4096 of 32 rows 254 and 95, of 64 262 and 147, of 96 267 and 251, 4096 x 1024 of 64 45
// and 40, of 96 45 and 67; 61 groups of 1005 x 2048 with 64 rows each 698 and 536; the loss of 64000 x 2048 of 128 rows 592 and 470.
// The loss's tiles cannot split the reduction: where they are few, more rows (3220 x 2296 of 256 rows, fp32: 152
// and 89; 48 in bf16 26 and 16, 16384 x 1024 in bf16 of 17 18 and 20).  Small layers save the launch that joins a split (1024 x 1024
// of 48 rows in bf16 13 and 9, 4096 x 1024 13 and 9, 1024 x 4096 13 and 15).  16-bit groups of two rows each: 32 of 2048 x 1024 20 and
// 23, 61 of 1005 x 2048 32 and 41.
template <class T>
inline bool is_few(int64_t rows, int64_t groups, int64_t N, int64_t K, bool loss = false) {
  if (rows <= 16) return true;
  if (groups >= 65535) return false;  // (a launch's second dimension)
  const int64_t tiles = ceil_div(rows, 128) * ceil_div(N, 128);
  if (sizeof(T) == 4) return rows <= (loss ? (tiles <= 64 ? 256 : 128) : groups > 0 ? 64 * groups : 64);
  if (loss) return rows <= 48 && tiles <= 32;
  return groups > 0 ? rows <= groups : rows <= 48 && tiles <= 32 && K <= 2048;
}
inline int few_parts(int64_t blocks) {
  int parts = 1;
  while (parts < 8 && blocks * parts < FEW_WAVES) parts *= 2;
  return parts;
}
template <class T, int E>
int launch_few(args p, hipStream_t st, int* parts_n = nullptr) {
  const int64_t slots = p.mode == BY_ROWS ? (p.G.groups + 1 < p.M ? p.G.groups + 1 : p.M) : 1;
  DN_CHECK(slots <= 65535, "product of %lld rows in %d groups: too many for one launch", (long long)p.M, p.G.groups);
  // 32 columns a wave where they are enough for three on every CU (one token of 32000 words of 4096: 43.5 us at 16, 41.1 at 32;
  // of 24576: 40.7 and 38.2), else 16 (one of 4096 of 1024: 4.6 us at 16, 6.1 at 32)
  const int wide = ceil_div(p.N, 32) * slots >= FEW_WAVES * 3 / 8 ? 32 : 16;
  const int parts = few_parts(ceil_div(p.N, wide) * slots), cols = wide * 8 / parts;
  p.parts_n = (int)ceil_div(p.N, cols);
  if (parts_n) *parts_n = p.parts_n;
  const dim3 grid((unsigned)ceil_div(p.N, cols), (unsigned)slots);
  DN_CHECK(grid.x < 1u << 23, "product of %lld columns: too many for one launch", (long long)p.N);
  // 16, 32 or 64 rows for each reading of B (fp32 products of 64000 x 2048, 16 at a time and so: 32 rows 266 and 164 us, 48 391 and
  // 233, the loss of 64 rows 449 and 253)
  const int64_t each = p.mode == BY_ROWS ? ceil_div(p.M, p.G.groups) : p.M;
  const int rows = E == E_LOSS_GRAD || each <= 16 ? 1 : each <= 32 ? 2 : 4;
  auto launch = [&](auto cols_of, auto rows_of) { k_few<T, decltype(cols_of)::value, decltype(rows_of)::value, E><<<grid, 512, 0, st>>>(p, parts); };
  auto launch_cols = [&](auto rows_of) {
    if (wide == 32)
      launch(std::integral_constant<int, 2>(), rows_of);
    else
      launch(std::integral_constant<int, 1>(), rows_of);
  };
  if constexpr (E != E_LOSS_GRAD) {
    if (rows == 4) launch_cols(std::integral_constant<int, 4>());
    if (rows == 2) launch_cols(std::integral_constant<int, 2>());
  }
  if (rows == 1) launch_cols(std::integral_constant<int, 1>());
  DN_LAUNCH_CHECK();
  return 0;
}

// ---- checks of arguments -----------------------------------------------------------------------------------------
inline int check_array(const char* what, const char* name, const void* p, int64_t ld, int64_t width, int type, bool may_lack) {
  DN_CHECK(p != nullptr || may_lack, "%s: no %s", what, name);
  if (p == nullptr) return 0;
  const int size = type == DNPEFF_F32 ? 4 : 2;
  DN_CHECK((uintptr_t)p % size == 0, "%s: %s is not aligned to its type", what, name);
  DN_CHECK(ld >= width, "%s: rows of %s are %lld elements apart and %lld wide", what, name, (long long)ld, (long long)width);
  return 0;
}

// One of the three instances of a template function, by type.
#define DN_BY_TYPE(type, call)                                          \
  ((type) == DNPEFF_F32   ? [&] { typedef float T; return call; }()     \
   : (type) == DNPEFF_F16 ? [&] { typedef _Float16 T; return call; }()  \
                          : [&] { typedef __bf16 T; return call; }())

}  // namespace tl
}  // namespace dn
