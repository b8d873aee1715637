// Matrix products on tiles of the matrix cores, for the operators of linear.hip and vocab.hip.
//
//   C(m, n) = sum over k of A(m, k) B(n, k)
//
// Each operand lies in memory either with its reduction index contiguous (rows of k) or with its own
// index contiguous (rows of m or n, one per k): a layer's forward product has two of the first kind, the
// gradient of its input one of each, the gradient of its weight two of the second.  A workgroup forms a
// tile of BM x BN, 128 bytes of the reduction at a time, from two LDS stages: while the matrix cores
// work on one, the other is filled past the registers (buffer loads to LDS), whose lanes outside the
// operand are given an offset past the buffer's end and so arrive as zeros.  Operands whose rows do not
// begin on 16 bytes go through registers instead, in 16-byte loads from any address.
//
// In LDS the 16-byte pieces of a row are permuted by its index, so that the 64 lanes of a read meet all banks:
//   rows of k:   piece c of row i sits at c ^ ((i >> 1) & 7); a lane reads its 16 bytes of k at once
//   rows of m/n: piece c of row k sits at c ^ swz(k); 16-bit values are transposed by the LDS read itself
//                (ds_read_b64_tr_b16: lane i of 16 gets element i of four rows), 32-bit ones read one by one
// The products run as B A, so that a lane ends with four consecutive n of one m: one store.
// All sums are fp32.
#pragma once

#include "dnpeff_internal.hpp"

namespace dn {
namespace tl {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef __bf16 v4b __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));

#define DN_LDS __attribute__((address_space(3)))

template <class V>
__device__ __forceinline__ DN_LDS V* lds_at(unsigned address) {
  return (DN_LDS V*)(uintptr_t)address;
}

template <class T>
struct num;
template <>
struct num<float> {
  typedef v4f piece;  // 16 bytes of the reduction index of one row, as a lane holds them
  typedef v4f four;
};
template <>
struct num<_Float16> {
  typedef v8h piece;
  typedef v4h four;
};
template <>
struct num<__bf16> {
  typedef v8b piece;
  typedef v4b four;
};

__device__ __forceinline__ v4f mma(v8b a, v8b b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ v4f mma(v8h a, v8h b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
// (any order of k serves as long as both operands have the same: element e of all four lane groups together)
__device__ __forceinline__ v4f mma(v4f a, v4f b, v4f c) {
#pragma unroll
  for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

// Four consecutive values of a row; those from `there` on are not touched (read as zero).
template <class T>
__device__ __forceinline__ v4f load4(const T* p, bool whole, int there) {
  v4f v = {0.f, 0.f, 0.f, 0.f};
  if (whole) {
    const typename num<T>::four q = *(const typename num<T>::four*)p;
#pragma unroll
    for (int t = 0; t < 4; t++) v[t] = (float)q[t];
  } else {
#pragma unroll
    for (int t = 0; t < 4; t++)
      if (t < there) v[t] = (float)p[t];
  }
  return v;
}
template <class T>
__device__ __forceinline__ void store4(T* p, v4f v, bool whole, int there) {
  if (whole) {
    typename num<T>::four q;
#pragma unroll
    for (int t = 0; t < 4; t++) q[t] = (T)v[t];
    *(typename num<T>::four*)p = q;
  } else {
#pragma unroll
    for (int t = 0; t < 4; t++)
      if (t < there) p[t] = (T)v[t];
  }
}

// ---- activations and their slopes, in fp32 -----------------------------------------------------------------------
// (16-bit results: the reciprocal and the exponential of the hardware, one ulp of fp32 off)
template <bool EXACT>
__device__ __forceinline__ float sigmoid(float z) {
  if (EXACT) return 1.f / (1.f + expf(-z));
  return __builtin_amdgcn_rcpf(1.f + __expf(-z));
}
template <bool EXACT>
__device__ __forceinline__ float gelu_tanh_t(float z) {
  // tanh(u) = 2 sigmoid(2u) - 1
  return 2.f * sigmoid<EXACT>(1.5957691216057308f * (z + 0.044715f * z * z * z)) - 1.f;
}
template <bool EXACT>
__device__ __forceinline__ float act_of(float z, int act) {
  switch (act) {
    case DNPEFF_ACT_RELU: return z > 0.f ? z : (z != z ? z : 0.f);
    case DNPEFF_ACT_SILU: return z * sigmoid<EXACT>(z);
    case DNPEFF_ACT_GELU: return 0.5f * z * erfcf(z * -0.70710678118654752f);  // (1 + erf loses what is left of it below zero)
    case DNPEFF_ACT_GELU_TANH: return 0.5f * z * (1.f + gelu_tanh_t<EXACT>(z));
  }
  return z;
}
template <bool EXACT>
__device__ __forceinline__ float slope_of(float z, int act) {
  switch (act) {
    case DNPEFF_ACT_RELU: return z > 0.f ? 1.f : 0.f;
    case DNPEFF_ACT_SILU: {
      const float p = sigmoid<EXACT>(z);
      return p * (1.f + z * (1.f - p));
    }
    case DNPEFF_ACT_GELU: {
      const float e = EXACT ? expf(-0.5f * z * z) : __expf(-0.5f * z * z);
      return 0.5f * erfcf(z * -0.70710678118654752f) + z * e * 0.39894228040143268f;
    }
    case DNPEFF_ACT_GELU_TANH: {
      const float t = gelu_tanh_t<EXACT>(z);
      return 0.5f * (1.f + t) + 0.5f * z * (1.f - t * t) * 0.79788456080286536f * (1.f + 0.134145f * z * z);
    }
  }
  return 1.f;
}

// ---- rows in groups ----------------------------------------------------------------------------------------------
// Group g holds rows ends[g] .. ends[g + 1] (the first from row 0, whatever ends[0] says); rows past the last
// end belong to none and count as group `groups`.  Ends outside the rows, or falling, are taken as the nearest
// that do not: no read or write goes by them unchecked.
struct group_rows {
  const int64_t* ends;
  int groups;
  int64_t rows;
  __device__ __forceinline__ int64_t at(int g) const {
    if (!ends) return rows;  // one group of all rows
    const int64_t e = ends[g];
    return e < 0 ? 0 : e > rows ? rows : e;
  }
  __device__ __forceinline__ int64_t first(int g) const { return g == 0 ? 0 : at(g); }
  __device__ __forceinline__ int64_t last(int g) const { return g < groups ? at(g + 1) : rows; }
  __device__ __forceinline__ int64_t count(int g) const {
    const int64_t n = last(g) - first(g);
    return n > 0 ? n : 0;
  }
};

__device__ __forceinline__ int wave_scan(int v, int lane) {  // inclusive sum over the lanes
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int u = __shfl_up(v, d, 64);
    if (lane >= d) v += u;
  }
  return v;
}
// Tiles of `tall` rows that the groups (and the rows of none) take; every wave by itself.
__device__ __forceinline__ int group_tiles(const group_rows& G, int tall, int lane) {
  int sum = 0;
  for (int b = 0; b <= G.groups; b += 64) {
    const int g = b + lane;
    const int t = g <= G.groups ? (int)((G.count(g) + tall - 1) / tall) : 0;
    sum += __shfl(wave_scan(t, lane), 63, 64);
  }
  return sum;
}
// The group of tile `tile` of them, its number within that group, and (tiles_before) the tiles of the groups before it.
__device__ __forceinline__ void group_of_tile(const group_rows& G, int tall, int lane, int tile, int* group, int* within) {
  int before = 0;
  for (int b = 0; b <= G.groups; b += 64) {
    const int g = b + lane;
    const int t = g <= G.groups ? (int)((G.count(g) + tall - 1) / tall) : 0;
    const int upto = before + wave_scan(t, lane);
    const unsigned long long hit = __ballot(tile < upto);
    if (hit) {
      const int l = __ffsll(hit) - 1;
      *group = __builtin_amdgcn_readfirstlane(b + l);
      *within = __builtin_amdgcn_readfirstlane(tile - __shfl(upto - t, l, 64));
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
  const void *A, *B;
  int64_t lda, ldb;         // elements from one row to the next
  int64_t M, N, K;          // BY_REDUCTION: K = rows of both operands
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
  int add_sums, out_f32, square, wide;  // wide: the rows of the epilogue's arrays can be accessed four values at once
  // E_LINEAR
  const void *bias, *residual;
  void* pre;
  int64_t ldp, ldr;
  int act;
  // E_LOSS, E_LOSS_GRAD: columns are words, `word0` the first of this piece
  const int32_t* labels;
  const float *lse, *dloss;
  const float* shrink;      // (dloss is multiplied by this; NULL: by 1)
  float2* parts;            // [M][tiles of words]: maximum and sum of the tile's words
  float* hit;               // [M] the label's logit
  int64_t word0, words;
};

// The result for four consecutive n of one m.
template <class T>
__device__ __forceinline__ void finish_linear(const args& p, int64_t m, int64_t n, v4f v, int group, bool held) {
  constexpr bool EXACT = sizeof(T) == 4;
  const int there = (int)(p.N - n < 4 ? p.N - n : 4);
  const bool whole = p.wide && there == 4;
  if (held) {
    if (p.bias) v += load4((const T*)p.bias + (int64_t)group * p.N + n, whole, there);
    if (p.pre) store4((T*)p.pre + m * p.ldp + n, v, whole, there);
    if (p.act != DNPEFF_ACT_NONE) {
#pragma unroll
      for (int t = 0; t < 4; t++) v[t] = act_of<EXACT>(v[t], p.act);
    }
  } else {
    v = v4f{0.f, 0.f, 0.f, 0.f};
    if (p.pre) store4((T*)p.pre + m * p.ldp + n, v, whole, there);
  }
  if (p.residual) v += load4((const T*)p.residual + m * p.ldr + n, whole, there);
  store4((T*)p.out + m * p.ldc + n, v, whole, there);
}
template <class T>
__device__ __forceinline__ void finish_store(const args& p, int64_t sheet, int64_t m, int64_t n, v4f v) {
  const int there = (int)(p.N - n < 4 ? p.N - n : 4);
  const int64_t at = sheet * p.c_split + m * p.ldc + n;
  if (p.add_sums) v += load4(p.sums + at, true, 4);
  if (!p.out) {
    store4(p.sums + at, v, true, 4);
    return;
  }
  const bool whole = p.wide && there == 4;
  const int64_t to = sheet * p.c_group + m * p.ldo + n;
  if (p.scale) v *= *p.scale;
  if (p.square) v *= v;
  if (p.out_f32)
    store4((float*)p.out + to, v, whole, there);
  else
    store4((T*)p.out + to, v, whole, there);
}

// A buffer load of 16 bytes per lane to LDS: lane l's go to lds + 16 l.
__device__ __forceinline__ void to_lds(v4i buffer, unsigned lds, int offset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(buffer) : "memory");
}
__device__ __forceinline__ v4i buffer_at(const char* p) {
  const uint64_t a = (uint64_t)p;
  return v4i{(int)(unsigned)a, (int)(unsigned)((a >> 32) & 0xffff), (int)0x80000000u, 0x00020000};
}

__device__ __forceinline__ int64_t uniform(int64_t v) {
  const unsigned lo = __builtin_amdgcn_readfirstlane((int)(unsigned)v), hi = __builtin_amdgcn_readfirstlane((int)((uint64_t)v >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}

// One operand's part of a tile: R of its own index, 128 bytes of the reduction.
template <class T, int R, int THREADS, bool ROWS_OF_K, bool DIRECT>
struct operand {
  static constexpr int S = sizeof(T), CH = 16 / S, BK = 128 / S;
  static constexpr int PER_ROW = ROWS_OF_K ? 8 : R * S / 16;  // pieces in a row
  static constexpr int N = R * 8 / THREADS;                   // pieces of a lane
  static constexpr int BYTES = R * 128;
  const char* at;   // first row's first piece of the next tile
  int64_t step;     // bytes from a tile to the next
  int64_t ld;
  int offset[DIRECT ? N : 1];
  int r0, c0;       // (not DIRECT) the lane's first row; rows come THREADS / PER_ROW apart
  int there;        // pieces' own index that exists: rows (rows of k), columns
  v4i held[DIRECT ? 1 : N];

  __device__ static __forceinline__ int swizzle(int row) {
    if (ROWS_OF_K) return (row >> 1) & 7;
    if (S == 4) return ((row >> 2) & 3) << 2;
    return (((row & 3) | ((row >> 1) & 4)) << 1) & (PER_ROW - 1);
  }
  __device__ __forceinline__ void start(const T* p, int64_t ld_, int64_t own0, int64_t k0, int there_, int tid) {
    ld = ld_ * S;
    there = there_;
    at = (const char*)uniform((int64_t)p + (ROWS_OF_K ? own0 * ld + k0 * S : k0 * ld + own0 * S));
    step = ROWS_OF_K ? 128 : BK * ld;
    if (DIRECT) {
#pragma unroll
      for (int e = 0; e < N; e++) {
        const int piece = (tid / 64 * N + e) * 64 + tid % 64, row = piece / PER_ROW, c = (piece % PER_ROW) ^ swizzle(row);
        const bool in = ROWS_OF_K ? row < there : c * CH < there;
        offset[e] = in ? (int)(row * ld) + c * 16 : (int)0x80000000u;
      }
    }
  }
  // left: what is left of the reduction.
  __device__ __forceinline__ void fill(unsigned lds, int64_t left, int tid) {
    const int k_there = left < BK ? (int)left : BK;
    if (DIRECT) {
      const v4i buffer = buffer_at(at);
#pragma unroll
      for (int e = 0; e < N; e++) {
        const int first = (tid / 64 * N + e) * 64, piece = first + tid % 64, row = piece / PER_ROW;
        const bool in = ROWS_OF_K ? (((piece % 8) ^ swizzle(row)) * CH < k_there) : row < k_there;
        to_lds(buffer, lds + __builtin_amdgcn_readfirstlane(first) * 16, in ? offset[e] : (int)0x80000000u);
      }
    } else {
#pragma unroll
      for (int e = 0; e < N; e++) {
        const int piece = e * THREADS + tid, row = piece / PER_ROW, c = (piece % PER_ROW) ^ swizzle(row);
        const int rows = ROWS_OF_K ? there : k_there, cols = ROWS_OF_K ? k_there : there;
        v4i v = {0, 0, 0, 0};
        if (row < rows && c * CH < cols) {
          const char* src = at + row * ld + c * 16;
          if ((c + 1) * CH <= cols) {
            struct __attribute__((packed, aligned(S))) loose {
              v4i v;
            };
            v = ((const loose*)src)->v;
          } else {  // the row ends within the piece
            union {
              T t[CH];
              v4i v;
            } u;
#pragma unroll
            for (int i = 0; i < CH; i++) u.t[i] = c * CH + i < cols ? ((const T*)src)[i] : (T)0.f;
            v = u.v;
          }
        }
        held[e] = v;
      }
    }
    at += step;
  }
  // (not DIRECT) what fill() left in registers to its place
  __device__ __forceinline__ void put(unsigned lds, int tid) {
    if (DIRECT) return;
#pragma unroll
    for (int e = 0; e < N; e++) *lds_at<v4i>(lds + (e * THREADS + tid) * 16) = held[e];
  }
};

// What a lane reads of 16 of an operand's index, `own` .. + 15, for 64 bytes of the reduction (s-th half).
template <class T, int R, bool ROWS_OF_K>
__device__ __forceinline__ typename num<T>::piece read_piece(unsigned lds, int own, int s, int lane) {
  typedef typename num<T>::piece piece;
  const int q = lane >> 4, i = lane & 15;
  if (ROWS_OF_K) {
    return *lds_at<piece>(lds + (own + i) * 128 + (((q + 4 * s) ^ (i >> 1)) << 4));
  } else if constexpr (sizeof(T) == 4) {
    piece v;
    const int col = own + i;
#pragma unroll
    for (int e = 0; e < 4; e++)
      v[e] = *lds_at<float>(lds + (s * 16 + q * 4 + e) * (R * 4) + (((col >> 2) ^ (q << 2)) << 4) + (col & 3) * 4);
    return v;
  } else {
    const int r = i >> 2, col = own + (i & 3) * 4;
    const int swz = ((r | ((q & 1) << 2)) << 1) & (R / 8 - 1);
    const unsigned a = lds + (s * 32 + q * 8 + r) * (R * 2) + (((col >> 3) ^ swz) << 4) + (col & 4) * 2;
    union {
      v4s h[2];
      piece p;
    } u;
    u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_at<v4s>(a));
    u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_at<v4s>(a + 4 * R * 2));
    return u.p;
  }
}

template <class T, int BM, int BN, int WM, int WN, bool A_ROWS, bool B_ROWS, bool DIRECT, int E>
__global__ __launch_bounds__(WM* WN * 64, 2) void k_tiles(args p) {
  constexpr int THREADS = WM * WN * 64, BK = 128 / sizeof(T);
  constexpr int FM = BM / WM / 16, FN = BN / WN / 16, STAGE = (BM + BN) * 128;
  __shared__ __align__(16) char smem[2 * STAGE];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / WN, wn = wave % WN;
  const int q = lane >> 4;

  // -- which tile --
  const int nt = (int)((p.N + BN - 1) / BN);
  int mt = p.mode == BY_ROWS ? group_tiles(p.G, BM, lane) : (int)((p.M + BM - 1) / BM);
  const int plane = mt * nt, many = plane * (p.mode == BY_REDUCTION ? p.G.groups : p.splits);
  if ((int)blockIdx.x >= many) return;
  // Workgroups go to the XCDs round-robin: each XCD gets a run of tiles, in blocks of a few tiles of m by all of n, so
  // that what its workgroups read at one time is shared in its L2.
  const int xcd = blockIdx.x % 8, share = many / 8, more = many % 8;
  const int t = xcd * share + (xcd < more ? xcd : more) + blockIdx.x / 8;
  const int sheet = t / plane, on = t % plane;
  constexpr int HIGH = BM >= 256 ? 4 : 8;
  const int block = on / (HIGH * nt), in_block = on % (HIGH * nt);
  const int high = mt - block * HIGH < HIGH ? mt - block * HIGH : HIGH;
  int tm = block * HIGH + in_block % high;
  const int tn = in_block / high;

  const T *A = (const T*)p.A, *B = (const T*)p.B;
  int64_t m0, m_end, k0 = 0, k_end = p.K;
  int group = 0;
  bool held = true;
  if (p.mode == BY_ROWS) {
    int within;
    group_of_tile(p.G, BM, lane, tm, &group, &within);
    if (group < 0) return;
    m0 = p.G.first(group) + (int64_t)within * BM;
    m_end = p.G.last(group);
    held = group < p.G.groups;
    if (held)
      B += group * p.b_group;
    else
      k_end = 0;
  } else {
    m0 = (int64_t)tm * BM;
    m_end = p.M;
    if (p.mode == BY_REDUCTION) {
      group = sheet;
      k0 = p.G.first(group);
      k_end = k0 + p.G.count(group);
    } else if (p.splits > 1) {
      k0 = sheet * p.split_k;
      k_end = k0 + p.split_k < p.K ? k0 + p.split_k : p.K;
    }
  }
  const int64_t n0 = (int64_t)tn * BN;
  const int m_there = (int)(m_end - m0 < BM ? m_end - m0 : BM), n_there = (int)(p.N - n0 < BN ? p.N - n0 : BN);

  // -- the product --
  v4f acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; i++)
#pragma unroll
    for (int j = 0; j < FN; j++) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
  const unsigned base = (unsigned)(uintptr_t)(DN_LDS char*)smem;
  operand<T, BM, THREADS, A_ROWS, DIRECT> a;
  operand<T, BN, THREADS, B_ROWS, DIRECT> b;
  a.start(A, p.lda, m0, k0, m_there, tid);
  b.start(B, p.ldb, n0, k0, n_there, tid);
  int64_t left = uniform(k_end - k0);
  unsigned stage = 0;
  if (left > 0) {
    a.fill(base, left, tid);
    b.fill(base + BM * 128, left, tid);
    a.put(base, tid);
    b.put(base + BM * 128, tid);
  }
  while (left > 0) {
    // the loads of this stage have arrived, and everyone has read the other one
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    left -= BK;
    const unsigned here = base + stage, next = base + (STAGE - stage);
    if (left > 0) {
      a.fill(next, left, tid);
      b.fill(next + BM * 128, left, tid);
    }
#pragma unroll
    for (int s = 0; s < 2; s++) {
      typename num<T>::piece fb[FN], fa[FM];
#pragma unroll
      for (int j = 0; j < FN; j++) fb[j] = read_piece<T, BN, B_ROWS>(here + BM * 128, wn * (BN / WN) + j * 16, s, lane);
#pragma unroll
      for (int i = 0; i < FM; i++) fa[i] = read_piece<T, BM, A_ROWS>(here, wm * (BM / WM) + i * 16, s, lane);
#pragma unroll
      for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++) acc[i][j] = mma(fb[j], fa[i], acc[i][j]);
    }
    if (left > 0) {
      a.put(next, tid);
      b.put(next + BM * 128, tid);
    }
    stage = STAGE - stage;
  }

  // -- what becomes of it --
  const int64_t mw = m0 + wm * (BM / WM) + (lane & 15), nw = n0 + wn * (BN / WN) + q * 4;
  if constexpr (E == E_LINEAR || E == E_STORE) {
#pragma unroll
    for (int i = 0; i < FM; i++) {
      const int64_t m = mw + i * 16;
      if (m >= m_end) continue;
#pragma unroll
      for (int j = 0; j < FN; j++) {
        const int64_t n = nw + j * 16;
        if (n >= p.N) continue;
        if constexpr (E == E_LINEAR)
          finish_linear<T>(p, m, n, acc[i][j], group, held);
        else
          finish_store<T>(p, sheet, m, n, acc[i][j]);
      }
    }
  } else if constexpr (E == E_LOSS) {
    // The maximum and the sum of exponentials of the tile's words for every row: over the lane's own, the four
    // lane groups, the waves side by side (through LDS).
    __syncthreads();
    float2* side = (float2*)smem;  // [WN][BM]
#pragma unroll
    for (int i = 0; i < FM; i++) {
      const int64_t m = mw + i * 16;
      const int64_t label = m < m_end ? (int64_t)p.labels[m] - p.word0 : -1;
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < FN; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int64_t n = nw + j * 16 + e;
          if (n < p.N) top = fmaxf(top, acc[i][j][e]);
          if (n == label && label >= 0 && n < p.N) p.hit[m] = acc[i][j][e];
        }
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float from = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < FN; j++)
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (nw + j * 16 + e < p.N) sum += __expf(acc[i][j][e] - from);
      sum += __shfl_xor(sum, 16, 64);
      sum += __shfl_xor(sum, 32, 64);
      if (q == 0) side[wn * BM + wm * (BM / WM) + i * 16 + lane] = float2{top, sum};
    }
    __syncthreads();
    for (int m = tid; m < m_there; m += THREADS) {
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < WN; w++) top = fmaxf(top, side[w * BM + m].x);
      const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int w = 0; w < WN; w++) {
        const float2 s = side[w * BM + m];
        if (s.x != -INFINITY || s.y != 0.f) sum += s.y * __expf(s.x - from);
      }
      p.parts[(m0 + m) * nt + tn] = float2{top, sum};
    }
  } else {
    // (softmax - label) times the token's weight; the piece's columns past the last word are zero
    const float shrink = p.shrink ? *p.shrink : 1.f;
#pragma unroll
    for (int i = 0; i < FM; i++) {
      const int64_t m = mw + i * 16;
      if (m >= m_end) continue;
      const int32_t label = p.labels[m];
      const float lse = p.lse[m];
      const float w = label < 0 ? 0.f : label >= p.words ? __builtin_nanf("") : p.dloss[m] * shrink;
#pragma unroll
      for (int j = 0; j < FN; j++) {
        const int64_t n = nw + j * 16;
        if (n >= p.ldc) continue;
        v4f g;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          float v = __expf(acc[i][j][e] - lse) - (p.word0 + n + e == label ? 1.f : 0.f);
          g[e] = n + e < p.N && label >= 0 ? v * w : 0.f;
        }
        store4((T*)p.out + m * p.ldc + n, g, true, 4);
      }
    }
  }
}

// ---- host --------------------------------------------------------------------------------------------------------
// Partial sums of a split reduction, added in their order, then as the tiles' own epilogue.
template <class T, int E>
__global__ void k_join(args p, const float* parts, int splits) {
  const int64_t n4 = (p.N + 3) / 4, i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= p.M * n4) return;
  const int64_t m = i / n4, n = i % n4 * 4, row = n4 * 4;
  v4f v = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < splits; s++) v += *(const v4f*)(parts + ((int64_t)s * p.M + m) * row + n);
  if constexpr (E == E_LINEAR)
    finish_linear<T>(p, m, n, v, 0, true);
  else
    finish_store<T>(p, 0, m, n, v);
}

// How a product is run.  Tiles of 256 x 256 (eight waves, one workgroup per CU) where they fill the chip, else of
// 128 x 128 (four waves, two per CU), the reduction of those split over workgroups where they are few.
struct plan {
  int splits;
  int64_t split_k;
};
constexpr int64_t MOST_SPLITS = 32;
template <class T>
inline plan plan_for(int64_t M, int64_t N, int64_t K, bool may_split) {
  constexpr int64_t BK = 128 / sizeof(T);
  plan r{1, K};
  const int64_t tiles = ceil_div(M, 128) * ceil_div(N, 128);
  if (!may_split || tiles == 0 || tiles >= 256 || K < 8 * BK) return r;
  int64_t s = 512 / tiles;
  if (s > K / (4 * BK)) s = K / (4 * BK);
  if (s > MOST_SPLITS) s = MOST_SPLITS;
  if (s < 2) return r;
  r.split_k = ceil_div(ceil_div(K, s), BK) * BK;
  r.splits = (int)ceil_div(K, r.split_k);
  if (r.splits < 2) r = plan{1, K};
  return r;
}
// Floats that the partial sums of a split product take (0: it is not split).
template <class T>
inline int64_t split_floats(int64_t M, int64_t N, int64_t K) {
  const plan r = plan_for<T>(M, N, K, true);
  return r.splits > 1 ? r.splits * M * (ceil_div(N, 4) * 4) : 0;
}

inline bool fits16(const void* p, int64_t ld, int64_t size) { return (uintptr_t)p % 16 == 0 && ld * size % 16 == 0; }

template <class T, int BM, int BN, int WM, int WN, bool A_ROWS, bool B_ROWS, bool DIRECT, int E>
int launch_tiles(const args& p, hipStream_t st) {
  const int64_t nt = ceil_div(p.N, BN);
  int64_t mt = ceil_div(p.M, BM), sheets = 1;
  if (p.mode == BY_ROWS)
    mt = p.G.rows / BM + (p.G.groups + 1 < p.G.rows ? p.G.groups + 1 : p.G.rows);
  else
    sheets = p.mode == BY_REDUCTION ? p.G.groups : p.splits;
  const int64_t many = mt * nt * sheets;
  if (many == 0) return 0;
  DN_CHECK(many < (int64_t)1 << 31, "product of %lld x %lld: too many tiles for one launch", (long long)p.M, (long long)p.N);
  k_tiles<T, BM, BN, WM, WN, A_ROWS, B_ROWS, DIRECT, E><<<(unsigned)many, WM * WN * 64, 0, st>>>(p);
  DN_LAUNCH_CHECK();
  return 0;
}

// A product whose args are complete but for splits.  ws: room for split_floats (NULL: the reduction is not split).  *_pad:
// the operand's rows may be read up to the next 16 bytes past their end.  *tile (or NULL): the tiles' width.
template <class T, bool A_ROWS, bool B_ROWS, int E>
int launch_product(args p, bool a_pad, bool b_pad, float* ws, hipStream_t st, int* tile = nullptr) {
  constexpr int64_t S = sizeof(T), CH = 16 / S, BK = 128 / S, NEAR = (int64_t)1 << 31;
  p.splits = 1;
  p.split_k = p.K;
  p.c_split = 0;
  const int64_t a_width = A_ROWS ? p.K : p.M, b_width = B_ROWS ? p.K : p.N;
  const bool direct = fits16(p.A, p.lda, S) && fits16(p.B, p.ldb, S) && (a_pad || a_width % CH == 0) && (b_pad || b_width % CH == 0) &&
                      (A_ROWS ? 256 : BK) * p.lda * S < NEAR && (B_ROWS ? 256 : BK) * p.ldb * S < NEAR &&
                      (p.mode != BY_ROWS || p.b_group * S % 16 == 0);
  if constexpr (E == E_LINEAR || E == E_STORE) {
    const plan r = plan_for<T>(p.M, p.N, p.K, ws != nullptr && p.mode == ONE);
    if (r.splits > 1) {
      args q = p;
      q.splits = r.splits;
      q.split_k = r.split_k;
      q.sums = ws;
      q.out = nullptr;
      q.add_sums = 0;
      q.ldc = ceil_div(p.N, 4) * 4;
      q.c_split = p.M * q.ldc;
      if (direct)
        DN_TRY((launch_tiles<T, 128, 128, 2, 2, A_ROWS, B_ROWS, true, E_STORE>(q, st)));
      else
        DN_TRY((launch_tiles<T, 128, 128, 2, 2, A_ROWS, B_ROWS, false, E_STORE>(q, st)));
      const int64_t many = p.M * ceil_div(p.N, 4);
      k_join<T, E><<<(unsigned)ceil_div(many, 256), 256, 0, st>>>(p, ws, r.splits);
      DN_LAUNCH_CHECK();
      return 0;
    }
  }
  if (tile) *tile = 128;
  if (!direct) return launch_tiles<T, 128, 128, 2, 2, A_ROWS, B_ROWS, false, E>(p, st);
  if constexpr (sizeof(T) == 2) {
    const int64_t sheets = p.mode == BY_REDUCTION ? p.G.groups : 1;
    if (ceil_div(p.M, 256) * ceil_div(p.N, 256) * sheets >= 200) {
      if (tile) *tile = 256;
      return launch_tiles<T, 256, 256, 2, 4, A_ROWS, B_ROWS, true, E>(p, st);
    }
  }
  return launch_tiles<T, 128, 128, 2, 2, A_ROWS, B_ROWS, true, E>(p, st);
}

// (their kernels are in linear.hip)
#define DN_STORE_PRODUCTS(X, T)                                                              \
  X template int launch_product<T, true, false, E_STORE>(args, bool, bool, float*, hipStream_t, int*); \
  X template int launch_product<T, false, false, E_STORE>(args, bool, bool, float*, hipStream_t, int*);

// Whether rows of `ld` elements from p on can be accessed four values at once.
template <class T>
inline bool fours(const void* p, int64_t ld) {
  return p == nullptr || ((uintptr_t)p % (4 * sizeof(T)) == 0 && ld % 4 == 0);
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

inline int64_t round256(int64_t bytes) { return (bytes + 255) / 256 * 256; }

}  // namespace tl
}  // namespace dn
