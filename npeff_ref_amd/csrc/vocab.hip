// Softmax cross entropy of hidden states over a vocabulary, without keeping the logits, and its gradients.
//
//   z[t, v] = x_t . e_v,  lse_t = log sum_v exp z[t, v],  loss_t = lse_t - z[t, label_t]
//   g[t, v] = (exp(z[t, v] - lse_t) - [v = label_t]) dloss_t,  dX = g E,  dE = g^T X
//
// Forward: every tile of logits leaves the maximum and the sum of exponentials of its words, eight bytes per token and
// tile; a second kernel joins them.  Backward: the vocabulary goes by in pieces; the logits of a piece are formed again,
// turned into g where they are summed, and multiplied on both sides.  g is rounded to the operands' type, once: its
// products run on the matrix cores of that type, and the rounding (2^-9 of a value in bf16) is that of the results.
#include "tiles.hpp"

using namespace dn;
using namespace dn::tl;

namespace dn {
namespace tl {
DN_STORE_PRODUCTS(extern, float)
DN_STORE_PRODUCTS(extern, _Float16)
DN_STORE_PRODUCTS(extern, __bf16)
}  // namespace tl
}  // namespace dn

namespace {

// One wave per token (four a workgroup, every gridDim.x * 4th: a launch has at most 2^32 lanes).
constexpr int64_t JOIN_MOST = (int64_t)1 << 22;
__global__ __launch_bounds__(256) void k_join_loss(int64_t rows, int parts_n, const float2* parts, const float* hit, const int32_t* labels,
                                                   int64_t words, float* loss, float* lse) {
  const int lane = threadIdx.x & 63;
  for (int64_t m = (int64_t)blockIdx.x * 4 + threadIdx.x / 64; m < rows; m += (int64_t)gridDim.x * 4) {
    float top = -INFINITY;
    for (int i = lane; i < parts_n; i += 64) top = fmaxf(top, parts[m * parts_n + i].x);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d, 64));
    const float from = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    for (int i = lane; i < parts_n; i += 64) {
      const float2 s = parts[m * parts_n + i];
      if (s.x != -INFINITY || s.y != 0.f) sum += s.y * expf(s.x - from);
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d, 64);
    if (lane == 0) {
      const float l = logf(sum) + from;
      const int32_t label = labels[m];
      if (lse) lse[m] = l;
      if (loss) loss[m] = label < 0 ? 0.f : label >= words ? __builtin_nanf("") : l - hit[m];
    }
  }
}

// 16-bit types: both[0] brings the largest |dloss| of a labelled token to 1 (fp16: to 2^14, so that g stays below the
// type's largest value and probabilities down to 4e-9 above its subnormal ones), both[1] takes the results back.  With
// equal weights, as of a mean, a label's g is then -1 but for p, and its rounding not the same for every token: left as
// they come, weights of 1 / 2000 put gradients off by up to 2^-11 (fp16) or 2^-8 as a whole.
template <class T>
__global__ __launch_bounds__(1024) void k_shrink(int64_t rows, const int32_t* labels, const float* dloss, float* both) {
  __shared__ float side[16];
  float most = 0.f;
  for (int64_t i = threadIdx.x; i < rows; i += 1024) {
    const float a = fabsf(dloss[i]);
    if (labels[i] >= 0 && a < INFINITY) most = fmaxf(most, a);
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) most = fmaxf(most, __shfl_xor(most, d, 64));
  if (threadIdx.x % 64 == 0) side[threadIdx.x / 64] = most;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; i++) most = fmaxf(most, side[i]);
    const float top = std::is_same<T, _Float16>::value ? 16384.f : 1.f;
    most = most > 0.f ? fmaxf(most, top * 1e-36f) : 1.f;  // (top / most stays finite)
    both[0] = top / most;
    both[1] = most / top;
  }
}

// Both gradients of at most R <= 16 tokens from g [words][16], in one pass over E: a wave has 256 columns of a run of words, four a
// lane with the tokens' X and dX in registers, g's values lane by lane; eight words are loaded ahead.  A workgroup's eight
// waves add their dX, k_join adds the workgroups'.  What bounds it: E read and dE written, 4.3 TB/s at 65536 words of 4096 in
// fp32 (500 us, 16 tokens); in 16 bits the vector units from 8 tokens on.
constexpr int BACK_AHEAD = 8, BACK_SPLITS = 64;
struct back_args {
  int rows;
  int64_t n_in, words, run;  // words of a wave
  const void *X, *E;
  int64_t ldx, lde, ldde;
  const float* g;
  const int32_t* labels;
  void* dE;      // (or NULL)
  float* parts;  // [workgroups of words][rows][n_in, to a multiple of 4] (or NULL)
};
template <class T, int R>
__global__ __launch_bounds__(512, 2) void k_few_back(back_args p) {
  __shared__ float4 sums[4][R][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // (the last lane of a row begins as much earlier as makes its four whole: what both have is the same)
  const int64_t n = (int64_t)blockIdx.x * 256 + lane * 4, c = n + 4 <= p.n_in ? n : p.n_in - 4;
  const bool in = n < p.n_in;
  float x[R][4], acc[R][4];
#pragma unroll
  for (int m = 0; m < R; m++) {
#pragma unroll
    for (int t = 0; t < 4; t++) x[m][t] = acc[m][t] = 0.f;
    // (of a token without a label g is zero, but its x may be infinite or NaN)
    if (p.dE && m < p.rows && p.labels[m] >= 0) load_row<T, 4>((const T*)p.X + m * p.ldx + c, x[m]);
  }
  const int64_t v0 = ((int64_t)blockIdx.y * 8 + wave) * p.run, v_end = v0 + p.run < p.words ? v0 + p.run : p.words;
  const T* e_row = (const T*)p.E + c;
  T* de_row = (T*)p.dE + c;
  typedef loose<T, 4> four;
  auto word = [&](int64_t v, four e, const float* w) {
    float de[4] = {0.f, 0.f, 0.f, 0.f};
    if (p.parts) {
#pragma unroll
      for (int m = 0; m < R; m++)
#pragma unroll
        for (int t = 0; t < 4; t++) acc[m][t] = fmaf(w[m], (float)e[t], acc[m][t]);
    }
    if (p.dE) {
#pragma unroll
      for (int m = 0; m < R; m++)
#pragma unroll
        for (int t = 0; t < 4; t++) de[t] = fmaf(w[m], x[m][t], de[t]);
      if (in) store_row<T, 4>(de_row + v * p.ldde, de);
    }
  };
  // Eight words ahead, and their g: 128 values, two a lane.
  auto load = [&](int64_t v, four* e, float* g) {
    if (p.parts) {
#pragma unroll
      for (int u = 0; u < BACK_AHEAD; u++) e[u] = *(const four*)(e_row + (v + u) * p.lde);
    }
#pragma unroll
    for (int h = 0; h < BACK_AHEAD / 4; h++) g[h] = p.g[v * 16 + h * 64 + lane];
  };
  four e[BACK_AHEAD] = {}, e_next[BACK_AHEAD] = {};
  float g[BACK_AHEAD / 4] = {}, g_next[BACK_AHEAD / 4] = {};
  int64_t v = v0;
  if (v + BACK_AHEAD <= v_end) load(v, e, g);
  while (v + BACK_AHEAD <= v_end) {
    if (v + 2 * BACK_AHEAD <= v_end) load(v + BACK_AHEAD, e_next, g_next);
#pragma unroll
    for (int u = 0; u < BACK_AHEAD; u++) {
      float w[R];
#pragma unroll
      for (int m = 0; m < R; m++) w[m] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(g[u / 4]), u % 4 * 16 + m));
      word(v + u, e[u], w);
    }
#pragma unroll
    for (int u = 0; u < BACK_AHEAD; u++) e[u] = e_next[u];
#pragma unroll
    for (int h = 0; h < BACK_AHEAD / 4; h++) g[h] = g_next[h];
    v += BACK_AHEAD;
  }
  for (; v < v_end; v++) {
    float w[R];
#pragma unroll
    for (int m = 0; m < R; m++) w[m] = p.g[v * 16 + m];
    word(v, p.parts ? *(const four*)(e_row + v * p.lde) : four{}, w);
  }
  if (!p.parts) return;
#pragma unroll
  for (int half = 4; half >= 1; half /= 2) {
    __syncthreads();
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int m = 0; m < R; m++) sums[wave - half][m][lane] = float4{acc[m][0], acc[m][1], acc[m][2], acc[m][3]};
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int m = 0; m < R; m++) {
        const float4 s = sums[wave][m][lane];
        acc[m][0] += s.x, acc[m][1] += s.y, acc[m][2] += s.z, acc[m][3] += s.w;
      }
    }
  }
  if (wave == 0 && in) {
    const int64_t ld = (p.n_in + 3) / 4 * 4;
#pragma unroll
    for (int m = 0; m < R; m++)
      if (m < p.rows) store_row<float, 4>(p.parts + ((int64_t)blockIdx.y * p.rows + m) * ld + c, acc[m]);
  }
}
// Both gradients of so many tokens go through k_few_back, others through tiles (us there and here, logits included): 65536 words of 4096 in
// fp32, 16 tokens 2008 and 678; in bf16 1 token 431 and 358, 8 tokens 430 and 410, 12 tokens 431 and 502 (the products of 12 take the
// vector units longer than E takes memory); 91355 of 3683, whose rows lie anywhere, 8 tokens 774 and 891; 10007 of 515 43 and 33.
template <class T>
bool back_is_few(int64_t rows, int64_t n_in) {
  return rows >= 1 && rows <= (sizeof(T) == 4 ? 16 : 8) && n_in >= 4;
}
// Workgroups of words: eight waves on every CU, and no more than k_join should add.
int64_t back_splits(int64_t n_in, int64_t words) {
  int64_t s = ceil_div(256, ceil_div(n_in, 256));
  if (s > BACK_SPLITS) s = BACK_SPLITS;
  return s < ceil_div(words, 64) ? s : ceil_div(words, 64);
}

constexpr int64_t PIECE_BYTES = (int64_t)512 << 20;  // of g at a time
constexpr int64_t MOST_WORDS = (int64_t)1 << 24;       // (offsets within a tile are of 32 bits)
// Words per piece: even pieces, whole tiles.
int64_t piece_words(int64_t rows, int64_t words, int size) {
  int64_t most = PIECE_BYTES / (size * (rows > 0 ? rows : 1)) / 256 * 256;
  if (most < 1024) most = 1024;
  if (most > MOST_WORDS) most = MOST_WORDS;
  if (most >= words) return words;
  return ceil_div(ceil_div(words, ceil_div(words, most)), 256) * 256;
}
int64_t padded(int64_t words) { return ceil_div(words, 64) * 64; }

template <class T>
struct loss_room {  // of the forward pass
  int64_t packs = 0, parts, all;
  matrix m[2];
  loss_room(int64_t rows, int64_t n_in, int64_t words, const void* X, int64_t ldx, const void* E, int64_t lde)
      : m{{X, ldx, rows, n_in, 1, 0, 0, nullptr}, {E, lde, words, n_in, 1, 0, 0, nullptr}} {
    if (!is_few<T>(rows, 0, words, n_in, true))
      for (const matrix& q : m) packs += packed_bytes<T>(q);
    parts = round256(rows * ceil_div(words, is_few<T>(rows, 0, words, n_in, true) ? 16 : 128) * 8);
    all = packs + parts + round256(rows * 4);
  }
};
template <class T>
struct grad_room {
  int64_t packs = 0, piece, g, sums, parts, all;
  matrix m[2];
  // keep: the labels where dE is wanted (a row of X without one must not reach it, whatever it holds: X is copied, 64 MB of a pass
  // of 27 ms at 8192 tokens of 4096), else NULL
  grad_room(int64_t rows, int64_t n_in, int64_t words, const void* X, int64_t ldx, const void* E, int64_t lde, const int32_t* keep)
      : m{{X, ldx, rows, n_in, 1, 0, 0, keep}, {E, lde, words, n_in, 1, 0, 0, nullptr}} {
    if (back_is_few<T>(rows, n_in)) {
      piece = words;
      sums = 0;
      g = round256(words * 64);
      parts = round256(back_splits(n_in, words) * rows * (ceil_div(n_in, 4) * 4) * 4);
      all = 256 + g + parts;
      return;
    }
    for (const matrix& q : m) packs += packed_bytes<T>(q);
    piece = piece_words(rows, words, num<T>::PLANES * 2);
    g = round256(num<T>::PLANES * rows * padded(piece) * 2);
    sums = piece < words ? round256(rows * (ceil_div(n_in, 4) * 4) * 4) : 0;
    const int64_t last = words - (ceil_div(words, piece) - 1) * piece;
    parts = 0;
    for (int64_t n : {piece, last})
      for (int64_t f : {split_floats<T>(rows, n_in, n), split_floats<T>(n, n_in, rows)})
        if (round256(4 * f) > parts) parts = round256(4 * f);
    all = 256 + packs + g + sums + parts;
  }
};
int check_room(const char* what, int64_t need, const void* ws, int64_t bytes) {
  DN_CHECK(ws != nullptr && bytes >= need && (uintptr_t)ws % 16 == 0, "%s: a workspace of %lld bytes, aligned to 16, is needed", what,
           (long long)need);
  return 0;
}

template <class T>
int loss_forward(hipStream_t st, int64_t rows, int64_t n_in, int64_t words, const void* X, int64_t ldx, const void* E, int64_t lde,
                 const int32_t* labels, float* loss, float* lse, char* ws, int64_t ws_bytes) {
  loss_room<T> room(rows, n_in, words, X, ldx, E, lde);
  DN_TRY(check_room("dnpeff_vocab_loss", room.all, ws, ws_bytes));
  const bool few = is_few<T>(rows, 0, words, n_in, true);
  if (!few) DN_TRY(pack<T>(room.m, 2, ws, st));
  args p{};
  p.A = room.m[0].p, p.lda = room.m[0].ld, p.B = room.m[1].p, p.ldb = room.m[1].ld;
  p.a_plane = room.m[0].plane, p.b_plane = room.m[1].plane;
  p.M = rows, p.N = words, p.K = n_in;
  p.mode = ONE;
  p.labels = labels, p.words = words, p.word0 = 0;
  p.parts = (float2*)(ws + room.packs);
  p.hit = (float*)(ws + room.packs + room.parts);
  int parts_n = 0;
  if (few)
    DN_TRY((launch_few<T, E_LOSS>(p, st, &parts_n)));
  else
    DN_TRY((launch_product<T, true, true, E_LOSS>(p, nullptr, st, &parts_n)));
  const int64_t blocks = ceil_div(rows, 4);
  k_join_loss<<<(unsigned)(blocks < JOIN_MOST ? blocks : JOIN_MOST), 256, 0, st>>>(rows, parts_n, p.parts, p.hit, labels, words, loss, lse);
  DN_LAUNCH_CHECK();
  return 0;
}

// (back_is_few)
template <class T>
int few_backward(hipStream_t st, const args& logits, char* g, float* parts, void* dX, int64_t lddx, void* dE, int64_t ldde) {
  args p = logits;
  p.out = g;
  DN_TRY((launch_few<T, E_LOSS_GRAD>(p, st)));
  const int64_t splits = back_splits(p.K, p.N);
  back_args b{};
  b.rows = (int)p.M, b.n_in = p.K, b.words = p.N, b.run = ceil_div(p.N, splits * 8);
  b.X = p.A, b.ldx = p.lda, b.E = p.B, b.lde = p.ldb, b.g = (const float*)g, b.labels = p.labels, b.dE = dE, b.ldde = ldde, b.parts = dX ? parts : nullptr;
  const dim3 grid((unsigned)ceil_div(p.K, 256), (unsigned)splits);
  if (p.M <= 4)
    k_few_back<T, 4><<<grid, 512, 0, st>>>(b);
  else if (p.M <= 8)
    k_few_back<T, 8><<<grid, 512, 0, st>>>(b);
  else if constexpr (sizeof(T) == 4)
    k_few_back<T, 16><<<grid, 512, 0, st>>>(b);
  DN_LAUNCH_CHECK();
  if (!dX) return 0;
  args q{};
  q.M = p.M, q.N = p.K, q.mode = ONE, q.out = dX, q.ldo = lddx;
  k_join<T, E_STORE><<<(unsigned)ceil_div(q.M * ceil_div(q.N, 4), 256), 256, 0, st>>>(q, parts, (int)splits);
  DN_LAUNCH_CHECK();
  return 0;
}
template <class T>
int loss_backward(hipStream_t st, int64_t rows, int64_t n_in, int64_t words, const void* X, int64_t ldx, const void* E, int64_t lde,
                  const int32_t* labels, const float* lse, const float* dloss, void* dX, int64_t lddx, void* dE, int64_t ldde, char* ws,
                  int64_t ws_bytes) {
  grad_room<T> r(rows, n_in, words, X, ldx, E, lde, dE ? labels : nullptr);
  DN_TRY(check_room("dnpeff_vocab_loss_backward", r.all, ws, ws_bytes));
  if (back_is_few<T>(rows, n_in)) {
    if (!dX && !dE) return 0;
    args p{};
    p.A = X, p.lda = ldx, p.B = E, p.ldb = lde;
    p.M = rows, p.N = words, p.K = n_in;
    p.mode = ONE;
    p.labels = labels, p.lse = lse, p.dloss = dloss, p.words = words;
    return few_backward<T>(st, p, ws + 256, (float*)(ws + 256 + r.g), dX, lddx, dE, ldde);
  }
  float* both = (float*)ws;
  ws += 256;
  DN_TRY(pack<T>(r.m, 2, ws, st));
  char* g = ws + r.packs;
  float* sums = (float*)(g + r.g);
  float* parts = r.parts ? (float*)(g + r.g + r.sums) : nullptr;
  const float *shrink = nullptr, *grow = nullptr;
  if constexpr (sizeof(T) == 2) {
    k_shrink<T><<<1, 1024, 0, st>>>(rows, labels, dloss, both);
    DN_LAUNCH_CHECK();
    shrink = both, grow = both + 1;
  }
  for (int64_t w0 = 0; w0 < words; w0 += r.piece) {
    const int64_t n = words - w0 < r.piece ? words - w0 : r.piece;
    const void* Ep = (const typename num<T>::op*)r.m[1].p + w0 * r.m[1].ld;
    const bool first = w0 == 0, last = w0 + n == words;
    args p{};
    p.A = r.m[0].p, p.lda = r.m[0].ld, p.B = Ep, p.ldb = r.m[1].ld;
    p.a_plane = r.m[0].plane, p.b_plane = r.m[1].plane;
    p.M = rows, p.N = n, p.K = n_in;
    p.mode = ONE;
    p.labels = labels, p.lse = lse, p.dloss = dloss, p.shrink = shrink, p.word0 = w0, p.words = words;
    p.out = g, p.ldc = padded(n);
    DN_TRY((launch_product<T, true, true, E_LOSS_GRAD>(p, nullptr, st)));
    if (dX) {
      args q{};
      q.A = g, q.lda = padded(n), q.B = Ep, q.ldb = r.m[1].ld;
      q.a_plane = rows * padded(n), q.b_plane = r.m[1].plane;
      q.M = rows, q.N = n_in, q.K = n;
      q.mode = ONE;
      q.sums = first && last ? nullptr : sums, q.add_sums = !first;
      q.ldc = ceil_div(n_in, 4) * 4;
      if (last) q.out = dX, q.ldo = lddx, q.scale = grow;
      DN_TRY((launch_product<T, true, false, E_STORE>(q, parts, st)));
    }
    if (dE) {
      args q{};
      q.A = g, q.lda = padded(n), q.B = r.m[0].p, q.ldb = r.m[0].ld;
      q.a_plane = rows * padded(n), q.b_plane = r.m[0].plane;
      q.M = n, q.N = n_in, q.K = rows;
      q.mode = ONE;
      T* to = (T*)dE + w0 * ldde;
      q.out = to, q.ldo = ldde, q.scale = grow;
      DN_TRY((launch_product<T, false, false, E_STORE>(q, parts, st)));
    }
  }
  return 0;
}

int check_head(const char* me, int type, int64_t rows, int64_t n_in, int64_t words) {
  DN_CHECK(type == DNPEFF_F32 || type == DNPEFF_F16 || type == DNPEFF_BF16, "%s: unknown type %d", me, type);
  DN_CHECK(rows >= 0 && n_in >= 1 && words >= 1 && rows < ((int64_t)1 << 31) && n_in <= ((int64_t)1 << 24) && words < ((int64_t)1 << 31),
           "%s: rows = %lld, n_in = %lld (at most 2^24), n_words = %lld", me, (long long)rows, (long long)n_in, (long long)words);
  return 0;
}

}  // namespace

DN_API int dnpeff_vocab_loss_workspace(int type, int64_t rows, int64_t n_in, int64_t n_words, int aligned, int64_t* forward_bytes,
                                       int64_t* backward_bytes) {
  clear_error();
  DN_TRY(check_head("dnpeff_vocab_loss_workspace", type, rows, n_in, n_words));
  const void* p = (const void*)(uintptr_t)(aligned ? 16 : 1);
  if (forward_bytes) *forward_bytes = DN_BY_TYPE(type, (loss_room<T>(rows, n_in, n_words, p, n_in, p, n_in).all));
  if (backward_bytes) *backward_bytes = DN_BY_TYPE(type, (grad_room<T>(rows, n_in, n_words, p, n_in, p, n_in, (const int32_t*)p).all));
  return 0;
}

DN_API int dnpeff_vocab_loss(void* stream, int type, int64_t rows, int64_t n_in, int64_t n_words, const void* X, int64_t ldx, const void* E,
                             int64_t lde, const int32_t* labels, float* loss, float* lse, void* workspace, int64_t workspace_bytes) {
  clear_error();
  const char* me = "dnpeff_vocab_loss";
  DN_TRY(check_head(me, type, rows, n_in, n_words));
  if (rows == 0) return 0;
  DN_TRY(check_array(me, "X", X, ldx, n_in, type, false));
  DN_TRY(check_array(me, "E", E, lde, n_in, type, false));
  DN_TRY(check_array(me, "labels", labels, 1, 1, DNPEFF_F32, false));
  DN_TRY(check_array(me, "loss", loss, 1, 1, DNPEFF_F32, true));
  DN_TRY(check_array(me, "lse", lse, 1, 1, DNPEFF_F32, true));
  return DN_BY_TYPE(type, loss_forward<T>((hipStream_t)stream, rows, n_in, n_words, X, ldx, E, lde, labels, loss, lse, (char*)workspace,
                                          workspace_bytes));
}

DN_API int dnpeff_vocab_loss_backward(void* stream, int type, int64_t rows, int64_t n_in, int64_t n_words, const void* X, int64_t ldx,
                                      const void* E, int64_t lde, const int32_t* labels, const float* lse, const float* dloss, void* dX,
                                      int64_t lddx, void* dE, int64_t ldde, void* workspace, int64_t workspace_bytes) {
  clear_error();
  const char* me = "dnpeff_vocab_loss_backward";
  DN_TRY(check_head(me, type, rows, n_in, n_words));
  DN_TRY(check_array(me, "X", X, ldx, n_in, type, rows == 0));
  DN_TRY(check_array(me, "E", E, lde, n_in, type, rows == 0));
  DN_TRY(check_array(me, "labels", labels, 1, 1, DNPEFF_F32, rows == 0));
  DN_TRY(check_array(me, "lse", lse, 1, 1, DNPEFF_F32, rows == 0));
  DN_TRY(check_array(me, "dloss", dloss, 1, 1, DNPEFF_F32, rows == 0));
  DN_TRY(check_array(me, "dX", dX, lddx, n_in, type, true));
  DN_TRY(check_array(me, "dE", dE, ldde, n_in, type, true));
  return DN_BY_TYPE(type, loss_backward<T>((hipStream_t)stream, rows, n_in, n_words, X, ldx, E, lde, labels, lse, dloss, dX, lddx, dE,
                                           ldde, (char*)workspace, workspace_bytes));
}
