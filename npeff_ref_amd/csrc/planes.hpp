// Products of fp32 operands that were packed to three planes of bf16 (tiles.hpp): all six terms of a stage of the reduction
// together, so that a plane is loaded once for its two or three terms.
//
//   C(m, n) = sum over k of (A0 + A1 + A2)(m, k) (B0 + B1 + B2)(n, k), without A1 B2, A2 B1 and A2 B2
//
// A workgroup of four waves forms 128 x 128, 32 of the reduction at a time, a stage of 48 KB (six planes of 8 KB).  A stage's products, 96 a
// wave, are shorter than a load takes: of the stages on their way two are still loads to registers, two lie in LDS
// and one is in the registers of the waves, which read the operands of the next while the matrix cores work on this one's.  (Three
// LDS stages filled past the registers, two to three ahead: 1.6 us a stage.)
//
// What bounds it: loads of few tiles (one workgroup per CU), the matrix cores of many.
#pragma once

#include "tiles.hpp"

namespace dn {
namespace tl {

// One operand's part of a stage: 128 of its own index, 32 of the reduction, three planes.  Offsets and bounds as in `operand`.
// In LDS piece c of row i of k sits at c ^ ((i >> 2) & 3): the 16 rows that a read meets then take all banks.  Rows of m or n lie as in tiles.
template <bool ROWS_OF_K>
struct slab {
  static constexpr int PER_ROW = ROWS_OF_K ? 4 : 16, ROWS = 64 / PER_ROW, N = 2;
  int64_t at, end, step, plane;
  int offset[N];
  __device__ __forceinline__ void start(const __bf16* p, int64_t ld, int64_t plane_elements, int64_t own0, int64_t k0, int64_t k_end, int there,
                                        int tid) {
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    ld *= 2;
    const int64_t first = (int64_t)p + (ROWS_OF_K ? own0 * ld : own0 * 2);
    at = uniform(first + (ROWS_OF_K ? k0 * 2 : k0 * ld) + wave * N * ROWS * ld);
    end = uniform(first + (ROWS_OF_K ? (there - 1) * ld + (k_end + 7) / 8 * 16 : (k_end - 1) * ld + (int64_t)(there + 7) / 8 * 16));
    step = uniform(ROWS_OF_K ? 64 : 32 * ld);
    plane = uniform(plane_elements * 2);
#pragma unroll
    for (int e = 0; e < N; e++) {
      const int row = (wave * N + e) * ROWS + lane / PER_ROW;
      const int c = (lane % PER_ROW) ^ (ROWS_OF_K ? (row >> 2) & 3 : operand<__bf16, 128, 256, false>::swizzle(row));
      offset[e] = (int)((e * ROWS + lane / PER_ROW) * ld) + c * 16;
    }
  }
  // The e-th of a lane's pieces of plane h, or zeros where the reduction has ended.
  __device__ __forceinline__ v4i load(int h, int e, bool there) const {
    const int64_t r = end - at;
    const int bytes = !there || r < 0 ? 0 : r > 0x7fffffff ? 0x7fffffff : (int)r;
    return __builtin_amdgcn_raw_buffer_load_b128(__builtin_amdgcn_make_buffer_rsrc((void*)(at + h * plane), 0, bytes, 0x00020000), offset[e], 0, 0);
  }
};
template <bool ROWS_OF_K>
struct slab_reader {
  reader<__bf16, 128, false> turned;
  unsigned lane_at;
  __device__ __forceinline__ void start(int own, int lane) {
    const int q = lane >> 4, i = lane & 15;
    lane_at = (own + i) * 64 + ((q ^ (i >> 2)) << 4);
    turned.start(own, lane);
  }
  __device__ __forceinline__ v8b read(unsigned lds, int i) const {
    if (ROWS_OF_K) return *(const DN_LDS v8b*)(lds_at<const char>(lds + lane_at) + i * 1024);
    return turned.read(lds, i, 0);
  }
};

template <bool A_ROWS, bool B_ROWS, int E>
__global__ __launch_bounds__(256, 1) void k_planes(args p) {
  constexpr int PLANE = 8192, OPERAND = 3 * PLANE, STAGE = 2 * OPERAND, LOADS = 12;
  __shared__ __align__(16) char smem[2 * STAGE];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / 2, wn = wave % 2;
  const unsigned base = (unsigned)(uintptr_t)(DN_LDS char*)smem;

  // each XCD a run of tiles, by blocks of eight of m, as in k_tiles
  const int nt = (int)((p.N + 127) / 128), mt = (int)((p.M + 127) / 128), sheet = mt * nt, many = sheet * p.splits;
  const unsigned id = block_id();
  if ((int)id >= many) return;
  const int xcd = id % 8, share = many / 8, more = many % 8, tile = xcd * share + (xcd < more ? xcd : more) + id / 8;
  place<float> w;
  w.A = (const __bf16*)p.A, w.B = (const __bf16*)p.B;
  w.sheet = tile / sheet;
  const int on = tile % sheet, block = on / (8 * nt), in_block = on % (8 * nt), high = mt - block * 8 < 8 ? mt - block * 8 : 8;
  w.tn = in_block / high;
  w.m0 = (int64_t)(block * 8 + in_block % high) * 128, w.n0 = (int64_t)w.tn * 128;
  w.m_end = p.M, w.group = 0, w.held = true;
  w.k0 = p.splits > 1 ? w.sheet * p.split_k : 0;
  w.k_end = p.splits > 1 && w.k0 + p.split_k < p.K ? w.k0 + p.split_k : p.K;

  slab<A_ROWS> a;
  slab<B_ROWS> b;
  slab_reader<A_ROWS> ra;
  slab_reader<B_ROWS> rb;
  ra.start(wm * 64, lane);
  rb.start(wn * 64, lane);
  v4f acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
  const int64_t n = uniform(w.k_end > w.k0 ? (w.k_end - w.k0 + 31) / 32 : 0);  // stages
  if (n > 0) {
    a.start(w.A, p.lda, p.a_plane, w.m0, w.k0, w.k_end, (int)(p.M - w.m0 < 128 ? p.M - w.m0 : 128), tid);
    b.start(w.B, p.ldb, p.b_plane, w.n0, w.k0, w.k_end, (int)(p.N - w.n0 < 128 ? p.N - w.n0 : 128), tid);
    // Stage s passes through registers s % 2 and LDS s % 2.
    v4i way[2][LOADS];
    int64_t fetched = 0;
    auto fetch = [&](int slot, int e) { way[slot][e] = e < 6 ? a.load(e / 2, e % 2, fetched < n) : b.load(e / 2 - 3, e % 2, fetched < n); };
    auto next_fetch = [&]() {
      a.at += a.step, b.at += b.step;
      fetched++;
    };
    auto put = [&](int half, int slot, int e) {
      *lds_at<v4i>(base + half * STAGE + e / 2 * PLANE + wave * 2048 + e % 2 * 1024 + lane * 16) = way[slot][e];
    };
    v8b fa[2][3][4], fb[2][3][4];
    auto read = [&](int set, int half, int r) {
      const unsigned from = base + half * STAGE + r / 8 * PLANE;
      if (r % 8 < 4)
        fb[set][r / 8][r % 4] = rb.read(from + OPERAND, r % 4);
      else
        fa[set][r / 8][r % 4] = ra.read(from, r % 4);
    };
    // everyone's LDS accesses are done (loads may be on their way)
    auto meet = [&]() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
#pragma unroll
    for (int s = 0; s < 2; s++) {
#pragma unroll
      for (int e = 0; e < LOADS; e++) fetch(s, e);
      next_fetch();
    }
#pragma unroll
    for (int s = 0; s < 2; s++) {
#pragma unroll
      for (int e = 0; e < LOADS; e++) put(s, s, e), fetch(s, e);
      next_fetch();
    }
    meet();
#pragma unroll
    for (int r = 0; r < 24; r++) read(0, 0, r);
    // Stage s = `set` modulo 2, whose operands are in their set: the next one's are read, the one after it goes to the LDS that everyone has
    // read, and its registers take the fourth after this one.
    auto products = [&](int set) {
      const int slot = set;
      meet();
#pragma unroll
      for (int t = 0; t < 6; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int g = t * 4 + i;
          read(1 - set, 1 - set, g);
          if (g % 2 == 0) put(set, slot, g / 2), fetch(slot, g / 2);
#pragma unroll
          for (int j = 0; j < 4; j++) acc[i][j] = mma(fb[set][plane_b(t)][j], fa[set][plane_a(t)][i], acc[i][j]);
          __builtin_amdgcn_sched_barrier(0);
        }
      next_fetch();
    };
    for (int64_t s = 0;;) {
      products(0);
      if (++s >= n) break;
      products(1);
      if (++s >= n) break;
    }
    meet();  // (before the LDS is used again)
  }
  finish_tile<float, 128, 128, 2, 2, E>(again(), w, acc, base, tid, wave);
}

// How many splits of the reduction fill one round of 256 workgroups in the least time: a stage takes 1.06 us and a workgroup 12 besides, a join
// 5 and its bytes at 4 TB/s (measured: 333 x 10007 of 515 32 us, 300 x 10007 of 768 41, 300 x 768 of 10007 42 + 5).
inline plan plan_planes(int64_t M, int64_t N, int64_t K, bool may_split) {
  plan best{false, 1, K, 0, 0};
  double least = 1e300;
  const int64_t tiles = ceil_div(M, 128) * ceil_div(N, 128);
  for (int64_t s = 1; s <= (may_split ? MOST_SPLITS : 1) && (s == 1 || s * tiles <= 256); s++) {
    const int64_t split_k = ceil_div(ceil_div(K, s), 64) * 64;
    if (s > 1 && (split_k < 128 || (s - 1) * split_k >= K)) break;
    const double us = (double)ceil_div(split_k, 32) * 1.06 + 12.0 + (s > 1 ? 5.0 + (double)s * M * N * 8.0 / 4e6 : 0.0);
    if (us < least) {
      least = us;
      best = plan{false, (int)s, s > 1 ? split_k : K, 0, 0};
    }
  }
  return best;
}
// Whether a product goes this way: where its tiles, split in four at least where it can be, are one round.  With more, k_tiles, whose workgroups
// share a CU by two, is as fast (us of a trained pass, there and where this says so here: 333 tokens of 10007 words of 515 200 and 176, 300 of
// 768 241 and 207; with any number of tiles here, 1500 of 30000 words of 512 1041 and 1054, 2000 of 50001 of 1024 4320 and 4460).
inline bool better_in_planes(int64_t M, int64_t N, bool may_split) { return ceil_div(M, 128) * ceil_div(N, 128) <= (may_split ? 64 : 256); }
inline int64_t plane_split_floats(int64_t M, int64_t N, int64_t K) {
  const plan r = plan_planes(M, N, K, true);
  return r.splits > 1 ? r.splits * M * (ceil_div(N, 4) * 4) : 0;
}
// launch_product of packed planes; ws: room for plane_split_floats.
template <bool A_ROWS, bool B_ROWS, int E>
int launch_planes(args p, float* ws, hipStream_t st, int* parts_n = nullptr) {
  const plan r = plan_planes(p.M, p.N, p.K, ws != nullptr && E == E_STORE);
  p.past = p.M * p.N * 4 > PAST_BYTES;
  p.splits = 1, p.split_k = p.K, p.c_split = 0;
  p.parts_n = (int)ceil_div(p.N, 128);
  if (parts_n) *parts_n = p.parts_n;
  const int64_t many = ceil_div(p.M, 128) * ceil_div(p.N, 128) * r.splits;
  if (many == 0) return 0;
  DN_CHECK(many < (int64_t)1 << 31, "product of %lld x %lld: too many tiles for one launch", (long long)p.M, (long long)p.N);
  args q = p;
  if (r.splits > 1) {
    q.splits = r.splits;
    q.split_k = r.split_k;
    q.sums = ws;
    q.out = nullptr;
    q.add_sums = 0;
    q.ldc = ceil_div(p.N, 4) * 4;
    q.c_split = p.M * q.ldc;
  }
  k_planes<A_ROWS, B_ROWS, E><<<grid_of(many), 256, 0, st>>>(q);
  DN_LAUNCH_CHECK();
  if constexpr (E == E_STORE) {
    if (r.splits > 1) {
      k_join<float, E_STORE><<<(unsigned)ceil_div(p.M * ceil_div(p.N, 4), 256), 256, 0, st>>>(p, ws, r.splits);
      DN_LAUNCH_CHECK();
    }
  }
  return 0;
}

}  // namespace tl
}  // namespace dn
