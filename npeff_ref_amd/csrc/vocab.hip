// Softmax cross entropy of hidden states over a vocabulary, without keeping the logits, and its gradients.
//
//   z[t, v] = x_t . e_v,  lse_t = log sum_v exp z[t, v],  loss_t = lse_t - z[t, label_t]
//   g[t, v] = (exp(z[t, v] - lse_t) - [v = label_t]) dloss_t,  dX = g E,  dE = g^T X
//
// Forward: every tile of logits leaves the maximum and the sum of exponentials of its words, eight bytes per token and
// tile; a second kernel joins them.  Backward: the vocabulary goes by in pieces; the logits of a piece are formed again,
// turned into g where they are summed, and multiplied on both sides.  g is rounded to the operands' type, once: its
// products run on the matrix cores of that type, and the rounding (2^-9 of a value in bf16) is that of the results.
//
// The same of what a model answers, at a temperature T (z = X E^T / T): log p of given words, the entropy, the likeliest
// words; and of a student that learns from a teacher's likeliest words (answers, further down).
#include "planes.hpp"

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

// Places of the logits' gradient that have values of their own (E_PROBS_GRAD): those of a row's listed words.
struct spots {
  int64_t rows;
  int many;            // of a row
  const int32_t* word; // [rows][many], negative: none
  const float* g;
};
// 16-bit types: both[0] brings the largest |dloss| of a labelled token to 1 (fp16: to 2^14, so that g stays below the
// type's largest value and probabilities down to 4e-9 above its subnormal ones), both[1] takes the results back.  With
// equal weights, as of a mean, a label's g is then -1 but for p, and its rounding not the same for every token: left as
// they come, weights of 1 / 2000 put gradients off by up to 2^-11 (fp16) or 2^-8 as a whole.
// Where the largest g are known before (`own`) the scale is less by the one of eight factors down to 2^(-7/8) with which those, or 2048 of
// them, round with the least error: a value a little above a power of two may be off by twice as much of itself as one a little below, and
// values of about one size can make up a batch (52 tokens with 44 listed words each in fp16: gradients off by 3.1e-4 of their norm
// at the largest scale and 2.8e-4 at the best, where rounding them alone is 2.1e-4).
template <class T>
__global__ __launch_bounds__(1024) void k_shrink(int64_t rows, const int32_t* labels, const float* dloss, spots own, float* both) {
  constexpr int SCALES = 8;
  __shared__ float side[16], off_of[SCALES][16];
  float most = 0.f;
  for (int64_t i = threadIdx.x; i < rows; i += 1024) {
    const float a = fabsf(dloss[i]);
    if (labels[i] >= 0 && a < INFINITY) most = fmaxf(most, a);
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) most = fmaxf(most, __shfl_xor(most, d, 64));
  if (threadIdx.x % 64 == 0) side[threadIdx.x / 64] = most;
  __syncthreads();
  for (int i = 0; i < 16; i++) most = fmaxf(most, side[i]);
  float top = std::is_same<T, _Float16>::value ? 16384.f : 1.f;
  most = most > 0.f ? fmaxf(most, top * 1e-36f) : 1.f;  // (top / most stays finite)
  const int64_t all = own.rows * own.many, step = all <= 2048 ? 1 : all / 2048 | 1;
  if (all > 0) {
    float off[SCALES];  // sums of squares
#pragma unroll
    for (int k = 0; k < SCALES; k++) off[k] = 0.f;
    for (int64_t i = threadIdx.x * step; i < all; i += 1024 * step) {
      const float g = own.g[i], a = fabsf(g) * (top / most);
      const int32_t w = own.word[i];  // (asked for together)
      if (w < 0 || !(a < INFINITY)) continue;
#pragma unroll
      for (int k = 0; k < SCALES; k++) {
        const float v = a * exp2f(-0.125f * k), d = (v - (float)(T)v) * exp2f(0.125f * k);
        off[k] = fmaf(d, d, off[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < SCALES; k++) {
#pragma unroll
      for (int d = 1; d < 64; d *= 2) off[k] += __shfl_xor(off[k], d, 64);
      if (threadIdx.x % 64 == 0) off_of[k][threadIdx.x / 64] = off[k];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    if (all > 0) {
      float least = INFINITY;
      int best = 0;
      for (int k = 0; k < SCALES; k++) {
        float sum = 0.f;
        for (int i = 0; i < 16; i++) sum += off_of[k][i];
        if (sum < least) least = sum, best = k;
      }
      top *= exp2f(-0.125f * best);
    }
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
// Below a temperature of 1/16 given words' products are always the tiles' own: another order of the same sum is off by some 2^-24 |z| / T, which
// at T = 1e-6 leaves nothing of a log p that should be 0, and of one sum the difference to itself is 0.  (Each tile then looks
// through the rows' lists.  us from rows of E and here: 2000 rows of 50001 words of 1024 with one given word 202 and 237, with 20 209 and 293, one
// row of 32000 words of 4096 48 and 46.)
constexpr float SHARP = 16.f;  // 1 / T
// The answers' fp32 products of few tiles go through planes.hpp.  (Those of the loss keep the order of their sums.)
template <class T>
constexpr bool may_be_planes(int epilogue) {
  return sizeof(T) == 4 && (is_probs(epilogue) || epilogue == E_PROBS_GRAD);
}
template <class T, int EPILOGUE>
int64_t floats_of(int64_t M, int64_t N, int64_t K) {
  return may_be_planes<T>(EPILOGUE) && better_in_planes(M, N, true) ? plane_split_floats(M, N, K) : split_floats<T>(M, N, K);
}
template <class T, int EPILOGUE>
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
      for (int64_t f : {floats_of<T, EPILOGUE>(rows, n_in, n), floats_of<T, EPILOGUE>(n, n_in, rows)})
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

// They take the place of what the tiles (or FEW: k_few, [words][16]) left there.
template <class T, bool FEW>
__global__ __launch_bounds__(256) void k_spots(spots s, int64_t word0, int64_t words, const float* shrink, void* out, int64_t ldc, int64_t plane) {
  const int64_t all = s.rows * s.many;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t n = (int64_t)s.word[i] - word0;
    if (s.word[i] < 0 || n < 0 || n >= words) continue;
    const int64_t m = i / s.many;
    const float g = s.g[i] * (shrink ? *shrink : 1.f);
    if constexpr (FEW)
      ((float*)out)[n * 16 + m] = g;
    else
      store_op<T, 1>((typename num<T>::op*)out + m * ldc + n, plane, &g);
  }
}
template <class T, bool FEW>
int put_spots(const spots& s, int64_t word0, int64_t words, const float* shrink, void* out, int64_t ldc, int64_t plane, hipStream_t st) {
  const int64_t blocks = ceil_div(s.rows * s.many, 256);
  if (blocks == 0) return 0;
  k_spots<T, FEW><<<(unsigned)(blocks < JOIN_MOST ? blocks : JOIN_MOST), 256, 0, st>>>(s, word0, words, shrink, out, ldc, plane);
  DN_LAUNCH_CHECK();
  return 0;
}

// A product of a pass whose logits end in EPILOGUE.
template <class T, bool A_ROWS, bool B_ROWS, int E, int EPILOGUE>
int launch_either(const args& p, float* parts, hipStream_t st, int* parts_n = nullptr) {
  if constexpr (may_be_planes<T>(EPILOGUE)) {
    if (better_in_planes(p.M, p.N, E == E_STORE)) return launch_planes<A_ROWS, B_ROWS, E>(p, parts, st, parts_n);
  }
  return launch_product<T, A_ROWS, B_ROWS, E>(p, parts, st, parts_n);
}

// Low temperatures (SHARP): lse as the forward pass rounded it, of products summed in another order perhaps, would put p off by the
// exponential of their difference, 2^-24 |z| / T and more.  There the backward pass sums the exponentials of its own products first
// (2000 rows of 50001 words of 1024 in bf16, forward and backward: 1104 us instead of 853; 5 rows of 32000 of 2048 147 instead of 121).
__global__ __launch_bounds__(256) void k_sums_again(int64_t rows, int parts_n, const float2* parts, float inv_heat, int first, int last, slope_row* slopes) {
  const int lane = threadIdx.x & 63;
  const float bits = inv_heat * LOG2_E;
  for (int64_t m = (int64_t)blockIdx.x * 4 + threadIdx.x / 64; m < rows; m += (int64_t)gridDim.x * 4) {
    slope_row t = slopes[m];
    if (is_dead(t)) continue;
    float top = first ? -INFINITY : t.top, sum = 0.f;
    for (int i = lane; i < parts_n; i += 64) top = fmaxf(top, parts[m * parts_n + i].x);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d, 64));
    const float from = top == -INFINITY ? 0.f : top;
    auto add = [&](float x, float s) {
      if (x != -INFINITY || s != 0.f) sum += s * __builtin_amdgcn_exp2f((x - from) * bits);
    };
    for (int i = lane; i < parts_n; i += 64) add(parts[m * parts_n + i].x, parts[m * parts_n + i].y);
    if (!first && lane == 0) add(t.top, t.rest);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d, 64);
    if (lane == 0) {
      t.top = top, t.rest = last ? logf(sum) : sum;
      if (last && !(fabsf(t.rest) < INFINITY)) t.a = __builtin_nanf("");
      slopes[m] = t;
    }
  }
}
// p: of a piece's products; room: of its g (12 bytes a row and 16 or 128 words; g takes more)
template <class T>
int sums_again(hipStream_t st, args p, bool few, char* room, bool first, bool last) {
  p.parts = (float2*)room;
  p.weighted = (float*)(room + p.M * ceil_div(p.N, few ? 16 : 128) * 8);
  int parts_n = 0;
  if (few)
    DN_TRY((launch_few<T, E_PROBS>(p, st, &parts_n)));
  else
    DN_TRY((launch_either<T, true, true, E_PROBS, E_PROBS_GRAD>(p, nullptr, st, &parts_n)));
  const int64_t blocks = ceil_div(p.M, 4);
  k_sums_again<<<(unsigned)(blocks < JOIN_MOST ? blocks : JOIN_MOST), 256, 0, st>>>(p.M, parts_n, p.parts, p.inv_heat, first, last, p.slopes);
  DN_LAUNCH_CHECK();
  return 0;
}

// (back_is_few)
template <class T, int E>
int few_backward(hipStream_t st, const args& logits, const spots& own, char* g, float* parts, void* dX, int64_t lddx, void* dE, int64_t ldde) {
  args p = logits;
  if constexpr (E == E_PROBS_GRAD) {
    if (p.inv_heat > SHARP) DN_TRY(sums_again<T>(st, p, true, g, true, true));
  }
  p.out = g;
  DN_TRY((launch_few<T, E>(p, st)));
  if constexpr (E == E_PROBS_GRAD) DN_TRY((put_spots<T, true>(own, 0, p.N, nullptr, g, 0, 0, st)));
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
// of: what the epilogue of the logits (EPILOGUE) takes of the rows; labels: rows of a negative one have no gradient; dloss: the
// rows' weights, which k_shrink brings to the range of the type.
template <class T, int EPILOGUE>
int loss_backward(hipStream_t st, int64_t rows, int64_t n_in, int64_t words, const void* X, int64_t ldx, const void* E, int64_t lde,
                  const args& of, const spots& own, void* dX, int64_t lddx, void* dE, int64_t ldde, char* ws, int64_t ws_bytes,
                  const char* me) {
  const int32_t* labels = of.labels;
  const float* dloss = of.dloss;
  grad_room<T, EPILOGUE> r(rows, n_in, words, X, ldx, E, lde, dE ? labels : nullptr);
  DN_TRY(check_room(me, r.all, ws, ws_bytes));
  if (back_is_few<T>(rows, n_in)) {
    if (!dX && !dE) return 0;
    args p = of;
    p.A = X, p.lda = ldx, p.B = E, p.ldb = lde;
    p.M = rows, p.N = words, p.K = n_in;
    p.mode = ONE;
    p.words = words;
    return few_backward<T, EPILOGUE>(st, p, own, ws + 256, (float*)(ws + 256 + r.g), dX, lddx, dE, ldde);
  }
  float* both = (float*)ws;
  ws += 256;
  DN_TRY(pack<T>(r.m, 2, ws, st));
  char* g = ws + r.packs;
  float* sums = (float*)(g + r.g);
  float* parts = r.parts ? (float*)(g + r.g + r.sums) : nullptr;
  const float *shrink = nullptr, *grow = nullptr;
  if constexpr (sizeof(T) == 2) {
    k_shrink<T><<<1, 1024, 0, st>>>(rows, labels, dloss, own, both);
    DN_LAUNCH_CHECK();
    shrink = both, grow = both + 1;
  }
  auto products_of = [&](int64_t w0) {  // of the piece that begins with this word
    args p = of;
    p.A = r.m[0].p, p.lda = r.m[0].ld, p.B = (const typename num<T>::op*)r.m[1].p + w0 * r.m[1].ld, p.ldb = r.m[1].ld;
    p.a_plane = r.m[0].plane, p.b_plane = r.m[1].plane;
    p.M = rows, p.N = words - w0 < r.piece ? words - w0 : r.piece, p.K = n_in;
    p.mode = ONE;
    return p;
  };
  if constexpr (EPILOGUE == E_PROBS_GRAD) {
    if (of.inv_heat > SHARP && rows > 0)
      for (int64_t w0 = 0; w0 < words; w0 += r.piece) DN_TRY(sums_again<T>(st, products_of(w0), false, g, w0 == 0, words - w0 <= r.piece));
  }
  for (int64_t w0 = 0; w0 < words; w0 += r.piece) {
    args p = products_of(w0);
    const int64_t n = p.N;
    const void* Ep = p.B;
    const bool first = w0 == 0, last = w0 + n == words;
    p.shrink = shrink, p.word0 = w0, p.words = words;
    p.out = g, p.ldc = padded(n);
    DN_TRY((launch_either<T, true, true, EPILOGUE, EPILOGUE>(p, nullptr, st)));
    if constexpr (EPILOGUE == E_PROBS_GRAD) DN_TRY((put_spots<T, false>(own, w0, n, shrink, g, p.ldc, p.M * p.ldc, st)));
    if (dX) {
      args q{};
      q.A = g, q.lda = padded(n), q.B = Ep, q.ldb = r.m[1].ld;
      q.a_plane = rows * padded(n), q.b_plane = r.m[1].plane;
      q.M = rows, q.N = n_in, q.K = n;
      q.mode = ONE;
      q.sums = first && last ? nullptr : sums, q.add_sums = !first;
      q.ldc = ceil_div(n_in, 4) * 4;
      if (last) q.out = dX, q.ldo = lddx, q.scale = grow;
      DN_TRY((launch_either<T, true, false, E_STORE, EPILOGUE>(q, parts, st)));
    }
    if (dE) {
      args q{};
      q.A = g, q.lda = padded(n), q.B = r.m[0].p, q.ldb = r.m[0].ld;
      q.a_plane = rows * padded(n), q.b_plane = r.m[0].plane;
      q.M = n, q.N = n_in, q.K = rows;
      q.mode = ONE;
      T* to = (T*)dE + w0 * ldde;
      q.out = to, q.ldo = ldde, q.scale = grow;
      DN_TRY((launch_either<T, false, false, E_STORE, EPILOGUE>(q, parts, st)));
    }
  }
  return 0;
}

// ---- answers -----------------------------------------------------------------------------------------------------
//   logp[t, j] = z[t, w_tj] - lse_t,  H_t = lse_t - sum_v p z = log s - W / s  with s = sum exp(z - max), W = sum exp(z - max) (z - max)
//   loss_t = sum_j q_j (log q_j - logp[t, j]),  q = softmax over the listed words of l / T
//
// Maxima are those of the products, and a word costs its difference from one, a product (by log2(e) / T), a hardware exponential and two
// additions: rounding errors are then of the differences' size, whatever |z| / T.
//
// Alternatives.  The tiles leave the largest logit of every chunk of words (64; of few rows 16 or 32) and the logits
// themselves.  The KEEP = n + 8 largest lie in the KEEP chunks of the largest maxima (in any other chunk every word is behind the KEEP
// that lead those), so what has to be read of the logits are these chunks.  The vocabulary goes by in pieces: from the first
// piece on a row has KEEP words, and a chunk that does not reach the least of them is not even stored.  The last n + 8 are then
// put in order by their products in 64 bits: the order is that of the exact logits, not of a summation's, and equal ones
// (the same embedding twice) keep the order of the words.
//
// Listed words of the gradients.  The tiles write dz = p (a + b log p) for all words, k_spots what the few listed ones have instead, from
// their log p of the forward pass: each value is still rounded once.
//
// What bounds them: E of few rows (one token of 32000 words of 4096 in bf16: 42 us at 6.3 TB/s, and 21 for the one workgroup that
// selects and orders, which waits for memory); the matrix cores of many.  8192 tokens of 131072 words of 4096 in bf16 with 64
// alternatives: products 6.4 ms (1367 TFLOP/s), selection 0.22, 4.8 GB of E's rows read again for their order 0.74 (6.5 TB/s).
constexpr int MOST_TOP = 128, SPARE = 8, MOST_KEEP = MOST_TOP + SPARE;
constexpr int MOST_LISTED = 4096;
constexpr int64_t BLOCK_ROWS = 65536;                 // rows at a time, for the workspace's sake
constexpr int64_t LOGIT_BYTES = (int64_t)2 << 30;   // of a piece's logits (512 MB: 7.89 ms where 2 GB take 7.64)
constexpr int64_t WHOLE_BYTES = (int64_t)128 << 20; // of all logits that are stored without a small first piece
// Given words' logits: rows of E read again and multiplied in fp32, or, where that would be so many bytes, taken from the tiles (us
// there and here: 20 words of 2000 rows of 1024, 82 MB, 914 and 922 with the gradients; 100 of 1999 of 1030, 412 MB, 318 and 290).
constexpr int64_t STORED_FROM = (int64_t)128 << 20;
// answer_args::stored: given words' products are among the logits of the pieces; are in logp already
enum { NOT_STORED = 0, IN_LOGITS = 1, IN_PLACE = 2 };

// Floats in the order of their values (equal zeros equal); 1: NaN, 0 is below all.
__device__ __forceinline__ unsigned key_of(float v) {
  if (v != v) return 1;
  const unsigned u = __float_as_uint(v + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned key) {
  return key <= 1 ? -INFINITY : __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// A kernel's only argument where it lies: read where it is needed.
template <class A>
__device__ __forceinline__ const __attribute__((address_space(4))) A& arguments() {
  typedef const __attribute__((address_space(4))) A kept;
  kept* p = (kept*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *p;
}
struct running {  // a row's statistics so far (top: of the products)
  float top, sum, weighted;
  int kept;
};
struct answer_args {
  int64_t rows, n_in, words;   // words: of the whole vocabulary
  int64_t word0, piece;        // this piece's
  int first, last;
  const float2* parts;         // [rows][parts_n]
  const float* weighted;
  int parts_n;
  // alternatives (n_top > 0)
  const float *tops, *logits;  // [rows][chunks], [rows][ldl]
  int64_t chunks, ldl;
  int chunk, n_top, keep;
  running* state;              // [rows]
  unsigned* kept_key;          // [rows][keep], in the order of the words
  int32_t* kept_word;
  float* floor;                // [rows]
  int32_t* top_words;
  float* top_logp;
  // given or listed words
  const void *X, *E;
  int64_t ldx, lde;
  float inv_heat;
  int n_given;
  const int32_t* given;        // [rows][n_given]
  int stored;
  float *logp, *lse, *entropy;
  const float* teacher;        // (or NULL) [rows][n_given]
  float* loss;
};

// Over the lanes of a wave, by the row shifts of its own registers: (LDS is not asked) lane l ends with the result of lanes 0 .. l; in their order.
template <int CONTROL, int ROWS, class V>
__device__ __forceinline__ V from_lane(V none, V v) {
  union {
    V v;
    int i[sizeof(V) / 4];
  } a, b;
  a.v = none, b.v = v;
#pragma unroll
  for (unsigned t = 0; t < sizeof(V) / 4; t++) a.i[t] = __builtin_amdgcn_update_dpp(a.i[t], b.i[t], CONTROL, ROWS, 0xf, false);
  return a.v;
}
template <bool WAVE = true, class V, class Op>  // (else within rows of 16 lanes)
__device__ __forceinline__ V scan_lanes(V v, V none, Op op) {
  v = op(from_lane<0x111, 0xf>(none, v), v);  // (the lane before, in rows of 16)
  v = op(from_lane<0x112, 0xf>(none, v), v);
  v = op(from_lane<0x114, 0xf>(none, v), v);
  v = op(from_lane<0x118, 0xf>(none, v), v);
  if (!WAVE) return v;
  v = op(from_lane<0x142, 0xa>(none, v), v);  // (the last of the row before, to the second and fourth)
  v = op(from_lane<0x143, 0xc>(none, v), v);  // (lane 31, to the upper half)
  return v;
}
template <class V, class Op>
__device__ __forceinline__ V over_lanes(V v, V none, Op op) {
  union {
    V v;
    int i;
  } a;
  a.v = scan_lanes(v, none, op);
  a.i = __builtin_amdgcn_readlane(a.i, 63);
  return a.v;
}
struct plus_of {
  template <class V>
  __device__ V operator()(V a, V b) const { return a + b; }
};
struct max_of {
  __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
  __device__ unsigned operator()(unsigned a, unsigned b) const { return a > b ? a : b; }
};
struct min_of {
  __device__ unsigned operator()(unsigned a, unsigned b) const { return a < b ? a : b; }
};

// The products of a row with C others in S: a lane's part of them, the lanes in this one's order `lane` of `lanes`.
template <class T, int C, class S>
__device__ __forceinline__ void dot_rows(const T* a, const T* const* b, int64_t n, int lane, int lanes, S* sum) {
  constexpr int W = 16 / sizeof(T);
  typedef loose<T, W> piece;
#pragma unroll
  for (int c = 0; c < C; c++) sum[c] = 0;
  auto add = [&](const piece& x, const piece* y, int from) {
    S d[W];
#pragma unroll
    for (int t = 0; t < W; t++) d[t] = (S)(float)x[t];
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
      for (int t = 0; t < W; t++) sum[c] = t >= from ? fma(d[t], (S)(float)y[c][t], sum[c]) : sum[c];
  };
  int64_t k = (int64_t)lane * W;
  piece x, y[C];
#pragma unroll 1
  for (; k + W <= n; k += lanes * W) {
    x = *(const piece*)(a + k);
#pragma unroll
    for (int c = 0; c < C; c++) y[c] = *(const piece*)(b[c] + k);
    add(x, y, 0);
  }
  if (k < n) {
    if (n >= W) {  // the row's last values, of which the first are another lane's
      x = *(const piece*)(a + n - W);
#pragma unroll
      for (int c = 0; c < C; c++) y[c] = *(const piece*)(b[c] + n - W);
      add(x, y, (int)(k + W - n));
    } else {
      for (int t = 0; t < n; t++)
#pragma unroll
        for (int c = 0; c < C; c++) sum[c] = fma((S)(float)a[t], (S)(float)b[c][t], sum[c]);
    }
  }
}

// Selection among n items with keys (0: not an item), which a thread keeps where n is at most THREADS HELD: by a workgroup, or
// (THREADS = 64) by one wave of it, which waits for nobody.
constexpr int MOST_HELD = 8;
template <int THREADS>
struct pick_room {
  int hist[256];
  unsigned part[3][MOST_HELD * (THREADS / 64)];  // per round and wave
  unsigned low, high;
  int left, done;
};
template <int THREADS, int HELD>
struct picker {
  static constexpr int WAVES = THREADS / 64, waves = WAVES;
  pick_room<THREADS>& r;
  const int lane = threadIdx.x & 63, tid = THREADS == 64 ? lane : threadIdx.x, wave = THREADS == 64 ? 0 : threadIdx.x >> 6;
  // (a wave's LDS accesses happen in their order)
  __device__ static __forceinline__ void sync() {
    if (THREADS == 64)
      asm volatile("" ::: "memory");
    else
      __syncthreads();
  }
  int64_t n;
  unsigned key[HELD];
  int count;          // of the items
  unsigned low, high; // the least and the largest key
  __device__ __forceinline__ picker(pick_room<THREADS>& room) : r(room) {}

  template <class Key, class F>
  __device__ __forceinline__ void each(Key key_at, F f) {
    if (n <= THREADS * HELD) {
#pragma unroll
      for (int h = 0; h < HELD; h++) f(key[h]);
    } else {
#pragma unroll 1
      for (int64_t i = tid; i < n; i += THREADS) f(key_at(i));
    }
  }
  // key_at(i) of an item; held(h): the same of the item h THREADS + tid
  template <class Key, class Held>
  __device__ __forceinline__ void look(int64_t n_items, Key key_at, Held held) {
    n = n_items;
    if (n <= THREADS * HELD) {
#pragma unroll
      for (int h = 0; h < HELD; h++) key[h] = h * THREADS + tid < n ? held(h) : 0u;
    }
    unsigned c = 0, lo = 0xffffffffu, hi = 0;
    each(key_at, [&](unsigned k) {
      c += k != 0;
      lo = k != 0 && k < lo ? k : lo;
      hi = k > hi ? k : hi;
    });
    c = over_lanes(c, 0u, plus_of());
    lo = over_lanes(lo, 0xffffffffu, min_of());
    hi = over_lanes(hi, 0u, max_of());
    if (WAVES > 1) {
      sync();
      if (lane == 0) r.part[0][wave] = c, r.part[1][wave] = lo, r.part[2][wave] = hi;
      sync();
      c = 0;
#pragma unroll
      for (int w = 0; w < WAVES; w++) {
        c += r.part[0][w];
        lo = r.part[1][w] < lo ? r.part[1][w] : lo, hi = r.part[2][w] > hi ? r.part[2][w] : hi;
      }
    }
    count = (int)c, low = lo, high = hi;
  }
  // The `need` items (of `count` or fewer) of the largest keys, of equal ones the first, to take(place, item, key) in the order of the items: the
  // range of the keys in 256 parts, how many are in each, the part in which the last of them lies, and so on within it.
  template <class Key, class Take>
  __device__ __forceinline__ void pick(int need, Key key_at, Take take) {
    unsigned lo = low, hi = high;
    int left = need;
    bool done = need >= count;
    if (done) hi = 0xffffffffu, left = count;  // (all are in the range)
    sync();
    while (!done) {
      const unsigned span = hi - lo;
      const int shift = span < 256 ? 0 : 24 - __builtin_clz(span);
      for (int i = tid; i < 256; i += THREADS) r.hist[i] = 0;
      sync();
      each(key_at, [&](unsigned k) {
        if (k >= lo && k <= hi) atomicAdd(&r.hist[(k - lo) >> shift], 1);
      });
      sync();
      if (wave == 0) {
        // lane l: the four parts from 255 - 4 l down
        int own[4], sum = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) own[e] = r.hist[255 - 4 * lane - e], sum += own[e];
        int before = scan_lanes(sum, 0, plus_of()) - sum;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          if (before < left && before + own[e] >= left) {
            const unsigned l = lo + ((unsigned)(255 - 4 * lane - e) << shift), span = (1u << shift) - 1;
            r.low = l, r.high = span < hi - l ? l + span : hi, r.left = left - before;  // (l + span may pass 32 bits)
            r.done = shift == 0 || own[e] == left - before;
          }
          before += own[e];
        }
      }
      sync();
      lo = r.low, hi = r.high, left = r.left, done = r.done != 0;
    }
    // those above the range, and the first `left` of those in it
    const unsigned long long below = (1ull << lane) - 1;
    if (WAVES == 1 && n <= THREADS * HELD) {
      int a_before = 0, b_before = 0;
#pragma unroll
      for (int h = 0; h < HELD; h++) {
        const bool up = key[h] > hi, same = key[h] != 0 && key[h] >= lo && key[h] <= hi;
        const unsigned long long above = __ballot(up), in = __ballot(same);
        const int a = a_before + __popcll(above & below), b = b_before + __popcll(in & below);
        if (up || (same && b < left)) take(a + (b < left ? b : left), (int64_t)h * THREADS + tid, key[h]);
        a_before += __popcll(above), b_before += __popcll(in);
      }
    } else if (n <= THREADS * HELD) {
      unsigned long long above[HELD], in[HELD];
#pragma unroll
      for (int h = 0; h < HELD; h++) {
        above[h] = __ballot(key[h] > hi), in[h] = __ballot(key[h] != 0 && key[h] >= lo && key[h] <= hi);
        if (lane == 0) r.part[0][h * WAVES + wave] = __popcll(above[h]), r.part[1][h * WAVES + wave] = __popcll(in[h]);
      }
      sync();
      if (wave == 0) {  // sums of what comes before
        int a_all = 0, b_all = 0;
        for (int i0 = 0; i0 < HELD * WAVES; i0 += 64) {
          const int i = i0 + lane;
          const int a = i < HELD * WAVES ? (int)r.part[0][i] : 0, b = i < HELD * WAVES ? (int)r.part[1][i] : 0;
          const int x = scan_lanes(a, 0, plus_of()), y = scan_lanes(b, 0, plus_of());
          if (i < HELD * WAVES) r.part[0][i] = a_all + x - a, r.part[1][i] = b_all + y - b;
          a_all += __builtin_amdgcn_readlane(x, 63), b_all += __builtin_amdgcn_readlane(y, 63);
        }
      }
      sync();
#pragma unroll
      for (int h = 0; h < HELD; h++) {
        const int a_before = (int)r.part[0][h * WAVES + wave], b_before = (int)r.part[1][h * WAVES + wave];
        const int a = a_before + __popcll(above[h] & below), b = b_before + __popcll(in[h] & below);
        const bool up = key[h] > hi, same = (in[h] >> lane) & 1;
        if (up || (same && b < left)) take(a + (b < left ? b : left), (int64_t)h * THREADS + tid, key[h]);
      }
    } else {
      int a_before = 0, b_before = 0;
#pragma unroll 1
      for (int64_t base = 0; base < n; base += THREADS) {
        const int64_t i = base + tid;
        const unsigned k = i < n ? key_at(i) : 0u;
        const bool up = k > hi, same = k != 0 && k >= lo && k <= hi;
        const unsigned long long above = __ballot(up), in = __ballot(same);
        int a = a_before, b = b_before, a_all = __popcll(above), b_all = __popcll(in);
        if (WAVES > 1) {
          sync();
          if (lane == 0) r.part[0][wave] = a_all, r.part[1][wave] = b_all;
          sync();
          a_all = b_all = 0;
#pragma unroll
          for (int w = 0; w < WAVES; w++) {
            if (w < wave) a += (int)r.part[0][w], b += (int)r.part[1][w];
            a_all += (int)r.part[0][w], b_all += (int)r.part[1][w];
          }
        }
        a += __popcll(above & below), b += __popcll(in & below);
        if (up || (same && b < left)) take(a + (b < left ? b : left), i, k);
        a_before += a_all, b_before += b_all;
      }
    }
    sync();
  }
};

// A workgroup has a row: joins its statistics; finds the words that lead it so far; after the last piece puts them in order and
// takes the given words' products.
// PART: all of it; or, of many rows, the selection by one wave a row, which waits for nobody, and the rest in a launch of its own with fewer
// registers (8192 rows with 72 leading words each: 1.75 ms in one launch, 0.98 in two); or the statistics and given words alone.
enum { ALL_OF_IT = 0, SELECT = 1, FINISH = 2, NO_TOPS = 3 };
template <class T, int THREADS, int PART>
__global__ __launch_bounds__(THREADS, THREADS >= 512 ? 2 : 4) void k_answers(answer_args) {
  constexpr int WAVES = THREADS / 64;
  constexpr bool TOPS = PART == ALL_OF_IT || PART == SELECT, FEW = THREADS >= 512;
  constexpr int HELD = THREADS == 64 ? 2 * MOST_HELD : MOST_HELD, AT_ONCE = FEW ? 6 : 4;  // items of a thread; rows of E that a wave multiplies at a time
  constexpr int LIST = 512, PARTS = 4;
  __shared__ pick_room<THREADS> room;
  pick_room<64>& wave_room = *(pick_room<64>*)&room;
  __shared__ int chosen;
  __shared__ unsigned list_key[LIST];
  __shared__ int32_t list_word[LIST];
  __shared__ int group_first[MOST_KEEP + 1];  // of 64 of the chunks' words
  __shared__ unsigned key_[2][MOST_KEEP];
  __shared__ int32_t word_[2][MOST_KEEP];
  __shared__ int32_t lead[MOST_KEEP];  // chunks
  __shared__ double exact_[MOST_KEEP];
  __shared__ float red[3][WAVES];
  __shared__ double part_of[FEW ? WAVES * 4 : 1][FEW ? MOST_KEEP : 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // Rows of E that are multiplied later, read ahead to the caches, and the row of X: a lane has a line.  (Each read of them from memory,
  // one after the other, would be 2 us.)
  auto touch = [&](int64_t m, int many, auto word) {
    auto& p = arguments<answer_args>();
    unsigned sum = 0;
    const int64_t bytes = p.n_in * (int64_t)sizeof(T);
    const int lines = (int)((bytes + 127) / 128);
    if ((int64_t)(many + 1) * lines > 8 * THREADS) return sum;
#pragma unroll 4
    for (int i = tid; i < (many + 1) * lines; i += THREADS) {
      const int32_t w = i < lines ? 0 : word(i / lines - 1);
      const char* row = i < lines ? (const char*)((const T*)p.X + m * p.ldx) : (const char*)((const T*)p.E + (w >= 0 && w < p.words ? w : 0) * p.lde);
      sum += *(const unsigned char*)(row + i % lines * 128);
    }
    return sum;
  };
  for (int64_t m = blockIdx.x; m < arguments<answer_args>().rows; m += gridDim.x) {
    // -- statistics --
    auto& p0 = arguments<answer_args>();
    running so_far = running{-INFINITY, 0.f, 0.f, 0};
    if (!p0.first || PART == FINISH) so_far = p0.state[m];
    const int parts_n = PART == FINISH ? 0 : p0.parts_n;
    // (what is read first is asked for together: a read takes 1 to 2 us)
    float tops_here[TOPS ? HELD : 1];
    if (TOPS && p0.n_top > 0 && p0.chunks <= THREADS * HELD) {
#pragma unroll
      for (int h = 0; h < HELD; h++) tops_here[h] = h * THREADS + tid < p0.chunks ? p0.tops[m * p0.chunks + h * THREADS + tid] : 0.f;
    }
    float2 own[PARTS];
    float own_w[PARTS];
    const bool held = parts_n <= PARTS * THREADS;
#pragma unroll
    for (int i = 0; i < PARTS; i++) {
      const bool here = held && i * THREADS + tid < parts_n;
      const int64_t at = m * parts_n + i * THREADS + tid;
      own[i] = here ? p0.parts[at] : float2{-INFINITY, 0.f};
      own_w[i] = here ? p0.weighted[at] : 0.f;
    }
    unsigned touched = 0;
    if (FEW && p0.last && !p0.stored) touched = touch(m, p0.n_given, [&](int i) { return p0.given[m * p0.n_given + i]; });
    float top = so_far.top;
#pragma unroll
    for (int i = 0; i < PARTS; i++) top = fmaxf(top, own[i].x);
    if (!held) {
      for (int i = tid; i < parts_n; i += THREADS) top = fmaxf(top, p0.parts[m * parts_n + i].x);
    }
    top = over_lanes(top, -INFINITY, max_of());
    if (WAVES > 1) {
      __syncthreads();
      if (lane == 0) red[0][wave] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WAVES; w++) top = fmaxf(top, red[0][w]);
    }
    const float from = top == -INFINITY ? 0.f : top;
    const float bits = p0.inv_heat * LOG2_E;
    float sum = 0.f, weighted = 0.f;
    auto add = [&](float x, float s, float w) {
      if (x != -INFINITY || s != 0.f) {
        const float z = (x - from) * bits, f = __builtin_amdgcn_exp2f(z);
        sum += s * f;
        weighted += f * fmaf(fmaxf(z, -200.f), s, w);
      }
    };
#pragma unroll
    for (int i = 0; i < PARTS; i++) add(own[i].x, own[i].y, own_w[i]);
    if (!held) {
#pragma unroll 1
      for (int i = tid; i < parts_n; i += THREADS) {
        const float2 s = p0.parts[m * parts_n + i];
        add(s.x, s.y, p0.weighted[m * parts_n + i]);
      }
    }
    sum = over_lanes(sum, 0.f, plus_of()), weighted = over_lanes(weighted, 0.f, plus_of());
    if (WAVES > 1) {
      if (lane == 0) red[1][wave] = sum, red[2][wave] = weighted;
      __syncthreads();
      sum = weighted = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; w++) sum += red[1][w], weighted += red[2][w];
    }
    asm volatile("" ::"v"(touched));
    add(so_far.top, so_far.sum, so_far.weighted);
    constexpr float LOG_2 = 0.69314718055994531f;
    const float log_sum = log2f(sum) * LOG_2, lse = fmaf(from, p0.inv_heat, log_sum);
    const bool sound = fabsf(lse) < INFINITY;

    // -- alternatives --
    auto& p = arguments<answer_args>();
    int kept = so_far.kept, at = 0;
    if (PART == FINISH && p.n_top > 0) {
      for (int i = tid; i < kept; i += THREADS) word_[0][i] = p.kept_word[m * p.keep + i];
      __syncthreads();
    }
    if (TOPS && p.n_top > 0) {
      for (int i = tid; i < kept; i += THREADS) key_[0][i] = p.kept_key[m * p.keep + i], word_[0][i] = p.kept_word[m * p.keep + i];
      const float* tops = p.tops + m * p.chunks;
      // (a chunk that only reaches what a full list ends with comes after it)
      unsigned least = kept == p.keep ? key_of(p.floor[m]) : 0u;
      auto chunk_key = [&](int64_t c) {
        const unsigned k = key_of(tops[c]);
        return k > least ? k : 0u;
      };
      picker<THREADS, HELD> chunks(room);
      chunks.look(p.chunks, chunk_key, [&](int h) {
        const unsigned k = key_of(tops_here[h]);
        return k > least ? k : 0u;
      });
      const int many = chunks.count < p.keep ? chunks.count : p.keep;
      if (many > 0) {
        unsigned reach = 0xffffffffu;  // the least of the chosen chunks' maxima
        chunks.pick(many, chunk_key, [&](int to, int64_t c, unsigned k) {
          lead[to] = (int32_t)c;
          reach = k < reach ? k : reach;
        });
        if (many < chunks.count) {
          reach = over_lanes(reach, 0xffffffffu, min_of());
          if (WAVES > 1) {
            if (lane == 0) room.part[0][wave] = reach;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < WAVES; w++) reach = room.part[0][w] < reach ? room.part[0][w] : reach;
          }
          least = reach - 1;
        }
        // The row's list, then the chunks' words that may join it: in the order of the words.  Of a chunk few do, so they are first
        // put together in LDS (where there is room; if not, all the chunks' words are items).
        const float* z = p.logits + m * p.ldl;
        const int bits = p.chunk == 64 ? 6 : p.chunk == 32 ? 5 : 4, in_chunks = many << bits, groups = (in_chunks + 63) >> 6;
        auto place = [&](int i) { return ((int64_t)lead[i >> bits] << bits) + (i & (p.chunk - 1)); };
        // (read whether it is a word or not, so that several reads are on their way: of each behind a branch the wave would wait)
        auto value = [&](int i) { return z[place(i < in_chunks ? i : 0)]; };
        auto key_here = [&](int i, float v) {
          const unsigned k = i < in_chunks && place(i) < p.piece ? key_of(v) : 0u;
          return k > least ? k : 0u;
        };
        auto word_key = [&](int i) { return key_here(i, value(i)); };
        int listed = kept;
        for (int i = tid; i < kept; i += THREADS) list_key[i] = key_[0][i], list_word[i] = word_[0][i];
        auto put = [&](int g, unsigned k, unsigned long long in, int from) {
          const int to = from + __popcll(in & ((1ull << lane) - 1));
          if (k != 0 && to < LIST) list_key[to] = k, list_word[to] = (int32_t)(p.word0 + place(g * 64 + lane));
        };
        if constexpr (WAVES == 1) {
          // Where no chunk could be left out nothing but the row's list bounds the words: they are looked at in 256 parts, of whose maxima the KEEP
          // largest are KEEP words, if there is no full list, or those above its end are too many.
          const bool all_of_them = many == chunks.count && kept + in_chunks > LIST;
          for (bool in_parts = all_of_them && kept < p.keep;; in_parts = true) {
            if (in_parts) {
              unsigned most[4] = {0, 0, 0, 0};
              for (int i = lane; i < kept; i += 64) most[0] = key_[0][i] > most[0] ? key_[0][i] : most[0];
#pragma unroll 1
              for (int g = 0; g < groups; g += 4) {
                float v[4];
#pragma unroll
                for (int t = 0; t < 4; t++) v[t] = value((g + t) * 64 + lane);
#pragma unroll
                for (int t = 0; t < 4; t++) {
                  const unsigned k = key_here((g + t) * 64 + lane, v[t]);
                  most[t] = k > most[t] ? k : most[t];
                }
              }
              picker<64, 4> parts(wave_room);
              parts.look(256, [&](int64_t) { return 0u; }, [&](int h) { return h == 0 ? most[0] : h == 1 ? most[1] : h == 2 ? most[2] : most[3]; });
              if (parts.count >= p.keep) {
                unsigned reach = 0xffffffffu;
                parts.pick(p.keep, [&](int64_t) { return 0u; }, [&](int, int64_t, unsigned k) { reach = k < reach ? k : reach; });
                reach = over_lanes(reach, 0xffffffffu, min_of());
                least = reach - 1 > least ? reach - 1 : least;
              }
            }
            // (eight reads on their way at a time: 72 chunks of each of 8192 rows 20 us; sixteen no less)
            constexpr int READS = 8;
            listed = kept;
#pragma unroll 1
            for (int g0 = 0; g0 < groups; g0 += READS) {
              float v[READS];
#pragma unroll
              for (int t = 0; t < READS; t++) v[t] = value((g0 + t) * 64 + lane);
#pragma unroll
              for (int t = 0; t < READS; t++) {
                const unsigned k = key_here((g0 + t) * 64 + lane, v[t]);
                const unsigned long long in = __ballot(k != 0);
                put(g0 + t, k, in, listed);
                listed += __popcll(in);
              }
            }
            if (in_parts || !all_of_them || listed <= LIST) break;
          }
        } else {
#pragma unroll 2
          for (int g = wave; g < groups; g += WAVES) {
            const int c = __popcll(__ballot(word_key(g * 64 + lane) != 0));
            if (lane == 0) group_first[g] = c;
          }
          __syncthreads();
          if (wave == 0) {
            int all = 0;
            for (int g0 = 0; g0 < groups; g0 += 64) {
              const int c = g0 + lane < groups ? group_first[g0 + lane] : 0;
              const int x = scan_lanes(c, 0, plus_of());
              if (g0 + lane < groups) group_first[g0 + lane] = kept + all + x - c;
              all += __builtin_amdgcn_readlane(x, 63);
            }
            if (lane == 0) group_first[groups] = kept + all;
          }
          __syncthreads();
          listed = group_first[groups];
          if (listed <= LIST) {
#pragma unroll 2
            for (int g = wave; g < groups; g += WAVES) {
              const unsigned k = word_key(g * 64 + lane);
              put(g, k, __ballot(k != 0), group_first[g]);
            }
          }
        }
        int found;
        if (listed <= LIST) {
          __syncthreads();
          if (FEW && listed <= THREADS) {
            // each word's rank among them, and its place among those that stay (0.5 us where a wave's selection takes 2)
            const unsigned k = tid < listed ? list_key[tid] : 0u;
            int rank = 0, to = 0;
#pragma unroll 4
            for (int j = 0; j < listed; j++) rank += list_key[j] > k || (list_key[j] == k && j < tid);
            const bool stays = tid < listed && rank < p.keep;
            const unsigned long long in = __ballot(stays);
            if (lane == 0) room.part[0][wave] = __popcll(in);
            __syncthreads();
            found = 0;
#pragma unroll
            for (int w = 0; w < WAVES; w++) {
              if (w < wave) to += (int)room.part[0][w];
              found += (int)room.part[0][w];
            }
            to += __popcll(in & ((1ull << lane) - 1));
            if (stays) key_[1][to] = k, word_[1][to] = list_word[tid];
          } else if (wave == 0) {
            picker<64, LIST / 64> items(wave_room);
            auto item_key = [&](int64_t i) { return list_key[i]; };
            items.look(listed, item_key, [&](int h) { return list_key[h * 64 + lane]; });
            found = items.count < p.keep ? items.count : p.keep;
            items.pick(found, item_key, [&](int to, int64_t i, unsigned k) { key_[1][to] = k, word_[1][to] = list_word[i]; });
            if (lane == 0) chosen = found;
          }
          if (!(FEW && listed <= THREADS)) {
            __syncthreads();
            found = chosen;
          }
        } else {
          picker<THREADS, HELD> items(room);
          auto item_key = [&](int64_t i) { return i < kept ? key_[0][i] : word_key((int)i - kept); };
          items.look(kept + in_chunks, item_key, [&](int h) { return item_key(h * THREADS + tid); });
          found = items.count < p.keep ? items.count : p.keep;
          items.pick(found, item_key, [&](int to, int64_t i, unsigned k) {
            key_[1][to] = k;
            word_[1][to] = i < kept ? word_[0][i] : (int32_t)(p.word0 + place((int)i - kept));
          });
        }
        kept = found, at = 1;
      }
      __syncthreads();
    }
    auto& p1 = p;
    if (p1.stored == IN_LOGITS && PART != FINISH) {
      for (int j = tid; j < p1.n_given; j += THREADS) {
        const int64_t w = (int64_t)p1.given[m * p1.n_given + j] - p1.word0;
        if (w >= 0 && w < p1.piece) p1.logp[m * p1.n_given + j] = p1.logits[m * p1.ldl + w];
      }
    }
    if (PART == SELECT || (PART != FINISH && !p1.last)) {
      for (int i = tid; i < kept; i += THREADS) p1.kept_key[m * p1.keep + i] = key_[at][i], p1.kept_word[m * p1.keep + i] = word_[at][i];
      if (wave == 0) {
        unsigned f = 0xffffffffu;
        for (int i = lane; i < kept; i += 64) f = key_[at][i] < f ? key_[at][i] : f;
        f = over_lanes(f, 0xffffffffu, min_of());
        if (lane == 0) {
          p1.state[m] = running{top, sum, weighted, kept};
          if (p1.n_top > 0) p1.floor[m] = kept == p1.keep ? value_of(f) : -INFINITY;
        }
      }
      __syncthreads();
      continue;
    }
    if (tid == 0) {
      if (p1.lse) p1.lse[m] = lse;
      if (p1.entropy) p1.entropy[m] = sound ? log_sum - weighted / sum * LOG_2 : __builtin_nanf("");
    }
    const T* x = (const T*)p1.X + m * p1.ldx;
    auto& p2 = arguments<answer_args>();
    // The products of `many` words' rows, each given to put(i, product) in one lane.  Few rows: `share` waves have a part each of a
    // product; else a wave has all of it.
    constexpr int W = 16 / sizeof(T);
    int share = 1;
    while (FEW && share < WAVES && share * 64 * W < p2.n_in) share *= 2;
    auto products = [&](auto zero, int many, auto word, auto put) {
      typedef decltype(zero) S;
      for (int i0 = 0; i0 < many; i0 += MOST_KEEP) {
        const int there = many - i0 < MOST_KEEP ? many - i0 : MOST_KEEP;
#pragma unroll 1
        for (int i = wave / share * AT_ONCE; i < there; i += WAVES / share * AT_ONCE) {
          const T* e[AT_ONCE];
          S s[AT_ONCE];
          bool any = false;
#pragma unroll
          for (int c = 0; c < AT_ONCE; c++) {
            const int32_t w = word(i0 + (i + c < there ? i + c : there - 1));
            any |= w >= 0;
            e[c] = (const T*)p2.E + (w >= 0 && w < p2.words ? w : 0) * p2.lde;
            s[c] = 0;
          }
          if (any) {
            dot_rows<T, AT_ONCE, S>(x, e, p2.n_in, FEW ? tid & (share * 64 - 1) : lane, share * 64, s);
#pragma unroll
            for (int c = 0; c < AT_ONCE; c++) s[c] = scan_lanes<!FEW>(s[c], zero, plus_of());
          }
          if (FEW ? lane % 16 == 15 : lane == 63) {
#pragma unroll
            for (int c = 0; c < AT_ONCE; c++)
              if (i + c < there) {
                if (FEW)
                  part_of[wave % share * 4 + lane / 16][i + c] = s[c];
                else
                  put(i0 + i + c, s[c]);
              }
          }
        }
        if (FEW) {
          __syncthreads();
          for (int i = tid; i < there; i += THREADS) {
            S s = 0;
#pragma unroll
            for (int w = 0; w < WAVES * 4; w++) s += w < share * 4 ? (S)part_of[w][i] : zero;
            put(i0 + i, s);
          }
          __syncthreads();
        }
      }
    };
    auto given_word = [&](int j) { return p2.given[m * p2.n_given + j]; };
    // log p of a word's product, from the difference to the largest (lse as it is stored is rounded, by 2^-24 |z| / T).  A given word's product
    // may be a rounding above the largest.
    auto log_p = [&](double s, double largest) {
      const float l = (float)((s - largest) * (double)p2.inv_heat - (double)log_sum);
      return l > 0.f ? 0.f : l;
    };
    auto put_given = [&](int j, double s) {
      const int32_t w = given_word(j);
      p2.logp[m * p2.n_given + j] = w < 0 ? 0.f : w >= p2.words ? __builtin_nanf("") : log_p(s, from);
    };
    // (a few given words go with the leading ones: a turn of them takes 2 us)
    const bool together = FEW && kept > 0 && p2.n_given <= AT_ONCE;
    if (TOPS || PART == FINISH) {
      auto word = [&](int i) { return i < kept ? word_[at][i] : given_word(i - kept); };
      const unsigned touched = FEW && kept > 0 ? touch(m, kept, word) : 0u;
      asm volatile("" ::"v"(touched));
      products(0.0, kept + (together && !p2.stored ? p2.n_given : 0), word, [&](int i, double s) {
        if (i < kept)
          exact_[i] = s == s ? s : -(double)INFINITY;
        else
          put_given(i - kept, s);
      });
    }
    if (!p2.stored && !together) products(0.f, p2.n_given, given_word, [&](int j, float s) { put_given(j, s); });
    if (p2.stored) {
      for (int j = tid; j < p2.n_given; j += THREADS) {  // (what this thread or an earlier launch has written)
        const int32_t w = p2.given[m * p2.n_given + j];
        float* to = p2.logp + m * p2.n_given + j;
        *to = w < 0 ? 0.f : w >= p2.words ? __builtin_nanf("") : log_p(*to, from);
      }
    }
    if (PART != NO_TOPS && p2.n_top > 0) {
      __syncthreads();
      for (int i = tid; i < p2.n_top; i += THREADS)
        if (!sound || i >= kept) p2.top_words[m * p2.n_top + i] = -1, p2.top_logp[m * p2.n_top + i] = __builtin_nanf("");
      for (int i = tid; i < kept && sound; i += THREADS) {
        const double s = exact_[i];
        double largest = s;  // (products in 64 bits against one of them: what fp32 sums are off by would be the larger part of a small log p)
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < kept; j++) rank += exact_[j] > s || (exact_[j] == s && j < i), largest = exact_[j] > largest ? exact_[j] : largest;
        if (rank < p2.n_top) {
          p2.top_words[m * p2.n_top + rank] = word_[at][i];
          p2.top_logp[m * p2.n_top + rank] = log_p(s, largest);
        }
      }
    }
    if (p2.teacher) {
      __syncthreads();  // (a workgroup's writes are there for all of it)
      if (wave == 0) {
        const float* l = p2.teacher + m * p2.n_given;
        const int32_t* w = p2.given + m * p2.n_given;
        const float *logp = p2.logp + m * p2.n_given;
        // (the first 64 are kept: asked for together, and once)
        const bool here = lane < p2.n_given;
        const int first = here ? lane : 0;
        const int32_t w_first = w[first], w0 = here ? w_first : -1;
        const float l0 = l[first], logp0 = logp[first];
        auto each = [&](auto f) {
          f(w0, l0, logp0);
          for (int j = lane + 64; j < p2.n_given; j += 64) f(w[j], l[j], logp[j]);
        };
        float most = -INFINITY, all = 0.f, loss = 0.f;
        bool odd = false;  // NaN or +infinity among them
        each([&](int32_t w, float l, float) {
          if (w >= 0 && l != -INFINITY) most = fmaxf(most, l), odd |= !(l < INFINITY) || w >= p2.words;
        });
        most = over_lanes(most, -INFINITY, max_of());
        each([&](int32_t w, float l, float) {
          if (w >= 0 && l > -INFINITY) all += expf((l - most) * p2.inv_heat);
        });
        all = over_lanes(all, 0.f, plus_of());
        const float log_all = logf(all);
        each([&](int32_t w, float l, float logp) {
          if (w >= 0 && l > -INFINITY) {
            const float log_q = (l - most) * p2.inv_heat - log_all, q = expf(log_q);
            if (q != 0.f) loss += q * (log_q - logp);
          }
        });
        loss = over_lanes(loss, 0.f, plus_of());
        const bool bad = __any(odd);
        if (lane == 0) p2.loss[m] = bad ? __builtin_nanf("") : most == -INFINITY ? 0.f : loss;
      }
    }
    __syncthreads();
  }
}

// What the backward pass takes of every row: the slopes of all words, the listed words' own values (a word that is listed twice has
// one place, its first), the size of its gradients.  A wave has a row.
//   probabilities and entropies  dz_v = (sum_j dlogp_j [v = w_j] - p_v (sum_j dlogp_j + dH (log p_v + H))) / T
//   a teacher's words            dz_v = (p_v - sum_j q_j [v = w_j]) dloss / T
struct slope_args {
  int64_t rows, words;
  int many;
  const int32_t* given;
  const float *logp, *lse, *entropy;
  const float *dlogp, *dentropy;  // (either may be NULL)
  const float *teacher, *dloss;   // (teacher NULL: probabilities)
  float inv_heat;
  slope_row* slopes;
  int32_t* alive;  // -1: no gradient
  float* size;
  int32_t* word;
  float* g;
};
__global__ __launch_bounds__(256) void k_slope_rows(slope_args p) {
  const int lane = threadIdx.x & 63;
  const float nan = __builtin_nanf("");
  for (int64_t m = (int64_t)blockIdx.x * 4 + threadIdx.x / 64; m < p.rows; m += (int64_t)gridDim.x * 4) {
    const int32_t* given = p.given + m * p.many;
    float a, b = 0.f, size, dloss = 0.f, most = -INFINITY, all = 0.f;
    bool alive = false, bad = false;
    if (p.teacher) {
      const float* l = p.teacher + m * p.many;
      bool odd = false;
      for (int j = lane; j < p.many; j += 64) {
        const int32_t w = given[j];
        if (w < 0 || l[j] == -INFINITY) continue;
        most = fmaxf(most, l[j]);
        odd |= !(l[j] < INFINITY) || w >= p.words;
        alive = true;
      }
#pragma unroll
      for (int d = 1; d < 64; d *= 2) most = fmaxf(most, __shfl_xor(most, d, 64));
      for (int j = lane; j < p.many; j += 64)
        if (given[j] >= 0 && l[j] > -INFINITY) all += expf((l[j] - most) * p.inv_heat);
#pragma unroll
      for (int d = 1; d < 64; d *= 2) all += __shfl_xor(all, d, 64);
      bad = __any(odd), alive = __any(alive);
      dloss = p.dloss[m] * p.inv_heat;
      a = dloss, size = fabsf(dloss);
    } else {
      float sum = 0.f, sizes = 0.f;
      for (int j = lane; j < p.many; j += 64) {
        const int32_t w = given[j];
        if (w < 0) continue;
        const float d = p.dlogp ? p.dlogp[m * p.many + j] : 0.f;
        sum += d, sizes += fabsf(d);
        alive |= d != 0.f || w >= p.words, bad |= w >= p.words;
      }
#pragma unroll
      for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d, 64), sizes += __shfl_xor(sizes, d, 64);
      const float dh = p.dentropy ? p.dentropy[m] : 0.f;
      bad = __any(bad), alive = __any(alive) || dh != 0.f;
      a = -sum;
      if (dh != 0.f) a = -fmaf(dh, p.entropy[m], sum), b = -dh * p.inv_heat;
      a *= p.inv_heat;
      // (p |log p + H| is at most 8 with 2^31 words: p (1 - p) log of those, and 1 / e)
      size = (sizes + 8.f * fabsf(dh)) * p.inv_heat;
    }
    if (bad || !(fabsf(p.lse[m]) < INFINITY)) a = nan;
    if (lane == 0) {
      p.slopes[m] = slope_row{alive ? 0.f : __int_as_float(DEAD), p.lse[m], a, b};
      p.alive[m] = alive ? 0 : -1;
      p.size[m] = size;
    }
    // the listed words: 64 of them against 64 at a time
    auto weight = [&](int j) {
      if (j >= p.many || given[j] < 0) return 0.f;
      if (!p.teacher) return p.dlogp ? p.dlogp[m * p.many + j] * p.inv_heat : 0.f;
      const float l = p.teacher[m * p.many + j];
      return l == -INFINITY ? 0.f : -expf((l - most) * p.inv_heat) / all * dloss;
    };
    for (int j0 = 0; j0 < p.many; j0 += 64) {
      const int j = j0 + lane;
      const int32_t w = j < p.many ? given[j] : -1;
      float sum = 0.f;
      bool first = true;
      for (int i0 = 0; i0 < p.many; i0 += 64) {
        const int i = i0 + lane;
        const int32_t wi = i < p.many ? given[i] : -1;
        const float gi = weight(i);
        const int there = p.many - i0 < 64 ? p.many - i0 : 64;
        for (int t = 0; t < there; t++) {
          const int32_t o = __builtin_amdgcn_readlane(wi, t);
          const float g = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(gi), t));
          if (o == w) sum += g, first &= i0 + t >= j;
        }
      }
      if (j < p.many) {
        p.word[m * p.many + j] = w >= 0 && w < p.words && first && alive ? w : -1;
        p.g[m * p.many + j] = slope_of(p.logp[m * p.many + j], a, b) + sum;
      }
    }
  }
}

// A bit for every chunk of 64 words that holds one of a row's given words; a wave has a row, and BITS words of it at a time.
__global__ __launch_bounds__(256) void k_wanted(int64_t rows, int many, const int32_t* given, int64_t words, unsigned* wanted, int64_t ld) {
  constexpr int BITS = 512;
  __shared__ unsigned bits[4][BITS];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int64_t m = (int64_t)blockIdx.x * 4 + wave; m < rows; m += (int64_t)gridDim.x * 4) {
    for (int64_t from = 0; from < ld; from += BITS) {
      const int there = ld - from < BITS ? (int)(ld - from) : BITS;
      for (int i = lane; i < there; i += 64) bits[wave][i] = 0;
      asm volatile("" ::: "memory");  // (a wave's LDS accesses happen in their order)
      for (int j = lane; j < many; j += 64) {
        const int32_t w = given[m * many + j];
        const int64_t at = (w >> 11) - from;
        if (w >= 0 && w < words && at >= 0 && at < there) atomicOr(&bits[wave][at], 1u << (w >> 6 & 31));
      }
      asm volatile("" ::: "memory");
      for (int i = lane; i < there; i += 64) wanted[m * ld + from + i] = bits[wave][i];
      asm volatile("" ::: "memory");
    }
  }
}

// Rows, and of them at a time, of the forward pass; its workspace.
struct answer_room {
  int64_t blocks, each;
  bool few, stored;
  int64_t first, wanted, ld_wanted;  // first: words of the first piece (0: as of the others)
  int64_t packs[2] = {0, 0};  // of a block's X, of E
  int64_t piece, parts, weighted, state, tops, logits, kept, floor, logp, all;
  int keep;
};
template <class T>
answer_room answer_room_of(int64_t rows, int64_t n_in, int64_t words, int n_given, int n_top, const matrix& X, const matrix& E) {
  answer_room r;
  r.blocks = rows > BLOCK_ROWS ? ceil_div(rows, BLOCK_ROWS) : 1;
  r.each = ceil_div(rows, r.blocks);
  r.few = is_few<T>(r.each, 0, words, n_in, true);
  if (!r.few) {
    matrix x = X;
    x.rows = r.each;
    r.packs[0] = packed_bytes<T>(x), r.packs[1] = packed_bytes<T>(E);
  }
  r.keep = n_top > 0 ? (n_top + SPARE < words ? n_top + SPARE : (int)words) : 0;
  r.stored = !r.few && r.each * n_given * n_in * (int64_t)sizeof(T) >= STORED_FROM;
  const bool logits = n_top > 0 || r.stored;
  r.piece = words, r.first = 0;
  if (logits) {
    int64_t most = LOGIT_BYTES / (4 * r.each) / 256 * 256;
    if (most < 1024) most = 1024;
    // A first piece small enough that storing all of it costs little, and large enough to know a floor for the others from (us with and without: 2000
    // rows of 50001 words with 20 alternatives 301 and 306, 8192 of 131072 with 64 7640 and 7710, 600 of 128000 of 1024 with 5 276 and 293).
    const int64_t few_words = ceil_div((int64_t)r.keep * 96, 2048) * 2048;
    if (n_top > 0 && !r.few && 4 * r.each * words > WHOLE_BYTES && 6 * few_words <= words) r.first = few_words < most ? few_words : most;
    const int64_t rest = words - r.first;
    if (most < rest) r.piece = ceil_div(ceil_div(rest, ceil_div(rest, most)), 256) * 256;
    else if (rest > 0) r.piece = rest;
  }
  r.ld_wanted = r.stored ? ceil_div(words, 2048) : 0;
  r.wanted = round256(r.each * r.ld_wanted * 4);
  r.parts = round256(r.each * ceil_div(r.piece > r.first ? r.piece : r.first, r.few ? 16 : 128) * 8);
  r.weighted = round256(r.each * ceil_div(r.piece > r.first ? r.piece : r.first, r.few ? 16 : 128) * 4);
  r.state = logits ? round256(r.each * (int64_t)sizeof(running)) : 0;
  r.tops = n_top > 0 ? round256(r.each * ceil_div(r.piece > r.first ? r.piece : r.first, r.few ? 16 : 64) * 4) : 0;
  r.logits = logits ? round256(r.each * padded(r.piece > r.first ? r.piece : r.first) * 4) : 0;
  r.kept = round256(r.each * r.keep * 4);
  r.floor = n_top > 0 ? round256(r.each * 4) : 0;
  r.logp = round256(r.each * (int64_t)n_given * 4);
  r.all = r.packs[0] + r.packs[1] + r.parts + r.weighted + r.state + r.tops + r.logits + 2 * r.kept + r.floor + r.logp + r.wanted;
  return r;
}

// Every piece of a call goes the same way, by the size of the largest: planes.hpp and tiles.hpp add an fp32 product's terms in different
// orders, and of one embedding in two pieces neither copy may lead.  (Tiles of both sizes, and k_few, keep one order.)
template <class T, int E>
int launch_answers(const args& p, bool planes, hipStream_t st, int* parts_n) {
  if constexpr (may_be_planes<T>(E)) {
    if (planes) return launch_planes<true, true, E>(p, nullptr, st, parts_n);
  }
  return launch_product<T, true, true, E>(p, nullptr, st, parts_n);
}
// to: what is wanted, of all rows.
template <class T>
int answers_forward(hipStream_t st, const char* me, const answer_args& to, char* ws, int64_t ws_bytes) {
  const int64_t words = to.words;
  matrix all_x{to.X, to.ldx, to.rows, to.n_in, 1, 0, 0, nullptr}, e{to.E, to.lde, words, to.n_in, 1, 0, 0, nullptr}, both[2];
  const answer_room r = answer_room_of<T>(to.rows, to.n_in, words, to.n_given, to.n_top, all_x, e);
  DN_TRY(check_room(me, r.all, ws, ws_bytes));
  char* x_room = ws;  // (E behind it)
  ws += r.packs[1];
  auto take = [&](int64_t bytes) {
    char* at = ws;
    ws += bytes;
    return at;
  };
  take(r.packs[0]);
  answer_args a = to;
  float2* parts = (float2*)take(r.parts);
  float* weighted = (float*)take(r.weighted);
  a.state = (running*)take(r.state);
  float *tops = (float*)take(r.tops), *logits = (float*)take(r.logits);
  a.kept_key = (unsigned*)take(r.kept);
  a.kept_word = (int32_t*)take(r.kept);
  a.floor = (float*)take(r.floor);
  float* logp_room = (float*)take(r.logp);
  unsigned* wanted = (unsigned*)take(r.wanted);
  a.stored = r.stored ? IN_LOGITS : to.n_given > 0 && to.inv_heat > SHARP ? IN_PLACE : NOT_STORED;
  const bool planes = may_be_planes<T>(E_PROBS) && better_in_planes(r.each, r.piece > r.first ? r.piece : r.first, false);
  a.parts = parts, a.weighted = weighted, a.tops = tops, a.logits = logits, a.keep = r.keep;
  for (int64_t b = 0; b < r.blocks; b++) {
    const int64_t m0 = b * r.each, rows = to.rows - m0 < r.each ? to.rows - m0 : r.each;
    matrix x = all_x;
    x.p = (const T*)to.X + m0 * to.ldx, x.rows = rows;
    a.X = x.p, a.rows = rows;
    a.given = to.given ? to.given + m0 * to.n_given : nullptr;
    a.logp = to.logp ? to.logp + m0 * to.n_given : logp_room;
    a.teacher = to.teacher ? to.teacher + m0 * to.n_given : nullptr;
    a.lse = to.lse ? to.lse + m0 : nullptr, a.entropy = to.entropy ? to.entropy + m0 : nullptr, a.loss = to.loss ? to.loss + m0 : nullptr;
    a.top_words = to.top_words ? to.top_words + m0 * to.n_top : nullptr, a.top_logp = to.top_logp ? to.top_logp + m0 * to.n_top : nullptr;
    if (!r.few) {
      both[0] = x, both[1] = e;
      DN_TRY(pack<T>(both, b == 0 ? 2 : 1, x_room, st));
      x = both[0];
      if (b == 0) e = both[1];
    }
    if (r.stored) {
      const int64_t blocks = ceil_div(rows, 4);
      k_wanted<<<(unsigned)blocks, 256, 0, st>>>(rows, to.n_given, a.given, words, wanted, r.ld_wanted);
      DN_LAUNCH_CHECK();
    }
    for (int64_t w0 = 0, n; w0 < words; w0 += n) {
      n = w0 == 0 && r.first > 0 ? r.first : r.piece;
      if (n > words - w0) n = words - w0;
      args p{};
      p.A = x.p, p.lda = x.ld, p.a_plane = x.plane, p.b_plane = e.plane, p.ldb = e.ld;
      p.M = rows, p.N = n, p.K = to.n_in;
      p.mode = ONE;
      p.inv_heat = to.inv_heat, p.word0 = w0;
      p.parts = parts, p.weighted = weighted;
      a.chunk = 64, a.chunks = ceil_div(n, 64);
      if (r.logits > 0) p.logits = logits, p.ldl = padded(n);
      if (to.n_top > 0) p.tops = tops, p.chunks = a.chunks, p.floor = w0 > 0 ? a.floor : nullptr;
      if (a.stored == IN_PLACE) p.listed = a.given, p.n_listed = to.n_given, p.listed_z = a.logp;
      if (r.stored) p.wanted = wanted, p.ld_wanted = r.ld_wanted, p.chunk0 = w0 / 64;
      if (r.few) {
        p.B = (const T*)e.p + w0 * e.ld;
        if (a.stored == IN_PLACE)
          DN_TRY((launch_few<T, E_PROBS_LISTED>(p, st, &a.parts_n, &a.chunk)));
        else
          DN_TRY((launch_few<T, E_PROBS>(p, st, &a.parts_n, &a.chunk)));
        a.chunks = ceil_div(n, a.chunk);
      } else {
        p.B = (const typename num<T>::op*)e.p + w0 * e.ld;
        if (a.stored == IN_PLACE)
          DN_TRY((launch_answers<T, E_PROBS_LISTED>(p, planes, st, &a.parts_n)));
        else
          DN_TRY((launch_answers<T, E_PROBS>(p, planes, st, &a.parts_n)));
      }
      a.first = w0 == 0, a.last = w0 + n == words, a.word0 = w0, a.piece = n, a.ldl = padded(n);
      // us of a row in 512 threads and in fewer: 64 rows of 32000 words with 20 alternatives 38 and 54 (two launches), 512 rows 75 and 77
      if (a.n_top == 0) {
        if (rows <= 256)
          k_answers<T, 512, NO_TOPS><<<(unsigned)rows, 512, 0, st>>>(a);
        else
          k_answers<T, 128, NO_TOPS><<<(unsigned)rows, 128, 0, st>>>(a);
      } else if (rows <= 512) {
        k_answers<T, 512, ALL_OF_IT><<<(unsigned)rows, 512, 0, st>>>(a);
      } else {
        k_answers<T, 64, SELECT><<<(unsigned)rows, 64, 0, st>>>(a);
        DN_LAUNCH_CHECK();
        if (a.last) k_answers<T, 256, FINISH><<<(unsigned)rows, 256, 0, st>>>(a);
      }
      DN_LAUNCH_CHECK();
    }
  }
  return 0;
}

struct slope_room {
  int64_t slopes, alive, size, word, g, all;
  slope_room(int64_t rows, int many)
      : slopes(round256(rows * (int64_t)sizeof(slope_row))), alive(round256(rows * 4)), size(round256(rows * 4)),
        word(round256(rows * many * 4)), g(round256(rows * many * 4)), all(slopes + alive + size + word + g) {}
};
template <class T>
int answers_backward(hipStream_t st, const char* me, slope_args s, int64_t n_in, const void* X, int64_t ldx, const void* E, int64_t lde,
                     void* dX, int64_t lddx, void* dE, int64_t ldde, char* ws, int64_t ws_bytes) {
  const slope_room own(s.rows, s.many);
  const grad_room<T, E_PROBS_GRAD> r(s.rows, n_in, s.words, X, ldx, E, lde, (const int32_t*)ws);
  DN_TRY(check_room(me, own.all + r.all, ws, ws_bytes));
  s.slopes = (slope_row*)ws;
  s.alive = (int32_t*)(ws + own.slopes);
  s.size = (float*)(ws + own.slopes + own.alive);
  s.word = (int32_t*)(ws + own.slopes + own.alive + own.size);
  s.g = (float*)(ws + own.slopes + own.alive + own.size + own.word);
  if (s.rows > 0) {
    const int64_t blocks = ceil_div(s.rows, 4);
    k_slope_rows<<<(unsigned)(blocks < JOIN_MOST ? blocks : JOIN_MOST), 256, 0, st>>>(s);
    DN_LAUNCH_CHECK();
  }
  args of{};
  of.labels = s.alive, of.dloss = s.size, of.slopes = s.slopes, of.inv_heat = s.inv_heat;
  return loss_backward<T, E_PROBS_GRAD>(st, s.rows, n_in, s.words, X, ldx, E, lde, of, spots{s.rows, s.many, s.word, s.g}, dX, lddx, dE,
                                        ldde, ws + own.all, ws_bytes - own.all, me);
}
int check_answers(const char* me, int64_t n_words, float temperature, int n_given, int n_top) {
  const float inv = 1.f / temperature;
  DN_CHECK(temperature > 0.f && inv > 0.f && inv * LOG2_E < INFINITY, "%s: temperature = %g", me, (double)temperature);
  DN_CHECK(n_given >= 0 && n_given <= MOST_LISTED, "%s: %d words of a row: 0 to %d", me, n_given, MOST_LISTED);
  DN_CHECK(n_top >= 0 && n_top <= MOST_TOP && n_top <= n_words, "%s: %d alternatives of %lld words: 0 to %d of them", me, n_top,
           (long long)n_words, MOST_TOP);
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
  if (backward_bytes) *backward_bytes = DN_BY_TYPE(type, (grad_room<T, E_LOSS_GRAD>(rows, n_in, n_words, p, n_in, p, n_in, (const int32_t*)p).all));
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
  args of{};
  of.labels = labels, of.lse = lse, of.dloss = dloss;
  return DN_BY_TYPE(type, (loss_backward<T, E_LOSS_GRAD>((hipStream_t)stream, rows, n_in, n_words, X, ldx, E, lde, of, spots{}, dX, lddx, dE,
                                                         ldde, (char*)workspace, workspace_bytes, me)));
}
DN_API int dnpeff_vocab_probs_workspace(int type, int64_t rows, int64_t n_in, int64_t n_words, int n_given, int n_top, int aligned,
                                        int64_t* forward_bytes, int64_t* backward_bytes) {
  clear_error();
  const char* me = "dnpeff_vocab_probs_workspace";
  DN_TRY(check_head(me, type, rows, n_in, n_words));
  DN_TRY(check_answers(me, n_words, 1.f, n_given, n_top));
  const void* p = (const void*)(uintptr_t)(aligned ? 16 : 1);
  const matrix x{p, n_in, rows, n_in, 1, 0, 0, nullptr}, e{p, n_in, n_words, n_in, 1, 0, 0, nullptr};
  if (forward_bytes) *forward_bytes = rows == 0 ? 0 : DN_BY_TYPE(type, (answer_room_of<T>(rows, n_in, n_words, n_given, n_top, x, e).all));
  if (backward_bytes)
    *backward_bytes = slope_room(rows, n_given).all + DN_BY_TYPE(type, (grad_room<T, E_PROBS_GRAD>(rows, n_in, n_words, p, n_in, p, n_in, (const int32_t*)p).all));
  return 0;
}

DN_API int dnpeff_vocab_probs(void* stream, int type, int64_t rows, int64_t n_in, int64_t n_words, const void* X, int64_t ldx, const void* E,
                              int64_t lde, float temperature, int n_given, const int32_t* words, float* logp, float* lse, float* entropy,
                              int n_top, int32_t* top_words, float* top_logp, void* workspace, int64_t workspace_bytes) {
  clear_error();
  const char* me = "dnpeff_vocab_probs";
  DN_TRY(check_head(me, type, rows, n_in, n_words));
  DN_TRY(check_answers(me, n_words, temperature, n_given, n_top));
  if (rows == 0) return 0;
  DN_TRY(check_array(me, "X", X, ldx, n_in, type, false));
  DN_TRY(check_array(me, "E", E, lde, n_in, type, false));
  DN_TRY(check_array(me, "words", words, 1, 1, DNPEFF_F32, n_given == 0));
  DN_TRY(check_array(me, "logp", logp, 1, 1, DNPEFF_F32, n_given == 0));
  DN_TRY(check_array(me, "lse", lse, 1, 1, DNPEFF_F32, true));
  DN_TRY(check_array(me, "entropy", entropy, 1, 1, DNPEFF_F32, true));
  DN_TRY(check_array(me, "top_words", top_words, 1, 1, DNPEFF_F32, n_top == 0));
  DN_TRY(check_array(me, "top_logp", top_logp, 1, 1, DNPEFF_F32, n_top == 0));
  answer_args a{};
  a.rows = rows, a.n_in = n_in, a.words = n_words, a.X = X, a.ldx = ldx, a.E = E, a.lde = lde, a.inv_heat = 1.f / temperature;
  a.n_given = n_given, a.given = words, a.logp = logp, a.lse = lse, a.entropy = entropy;
  a.n_top = n_top, a.top_words = top_words, a.top_logp = top_logp;
  return DN_BY_TYPE(type, answers_forward<T>((hipStream_t)stream, me, a, (char*)workspace, workspace_bytes));
}

DN_API int dnpeff_vocab_probs_backward(void* stream, int type, int64_t rows, int64_t n_in, int64_t n_words, const void* X, int64_t ldx,
                                       const void* E, int64_t lde, float temperature, int n_given, const int32_t* words, const float* logp,
                                       const float* lse, const float* entropy, const float* dlogp, const float* dentropy, void* dX,
                                       int64_t lddx, void* dE, int64_t ldde, void* workspace, int64_t workspace_bytes) {
  clear_error();
  const char* me = "dnpeff_vocab_probs_backward";
  const bool none = rows == 0;
  DN_TRY(check_head(me, type, rows, n_in, n_words));
  DN_TRY(check_answers(me, n_words, temperature, n_given, 0));
  DN_TRY(check_array(me, "X", X, ldx, n_in, type, none));
  DN_TRY(check_array(me, "E", E, lde, n_in, type, none));
  DN_TRY(check_array(me, "words", words, 1, 1, DNPEFF_F32, none || n_given == 0));
  DN_TRY(check_array(me, "logp", logp, 1, 1, DNPEFF_F32, none || n_given == 0));
  DN_TRY(check_array(me, "lse", lse, 1, 1, DNPEFF_F32, none));
  DN_TRY(check_array(me, "entropy", entropy, 1, 1, DNPEFF_F32, none || dentropy == nullptr));
  DN_TRY(check_array(me, "dlogp", dlogp, 1, 1, DNPEFF_F32, true));
  DN_TRY(check_array(me, "dentropy", dentropy, 1, 1, DNPEFF_F32, true));
  DN_TRY(check_array(me, "dX", dX, lddx, n_in, type, true));
  DN_TRY(check_array(me, "dE", dE, ldde, n_in, type, true));
  slope_args s{};
  s.rows = rows, s.words = n_words, s.many = n_given, s.given = words, s.logp = logp, s.lse = lse, s.entropy = entropy;
  s.dlogp = dlogp, s.dentropy = dentropy, s.inv_heat = 1.f / temperature;
  return DN_BY_TYPE(type, answers_backward<T>((hipStream_t)stream, me, s, n_in, X, ldx, E, lde, dX, lddx, dE, ldde, (char*)workspace,
                                              workspace_bytes));
}

DN_API int dnpeff_vocab_distill(void* stream, int type, int64_t rows, int64_t n_in, int64_t n_words, const void* X, int64_t ldx,
                                const void* E, int64_t lde, float temperature, int n_listed, const int32_t* words, const float* logits,
                                float* loss, float* logp, float* lse, void* workspace, int64_t workspace_bytes) {
  clear_error();
  const char* me = "dnpeff_vocab_distill";
  DN_TRY(check_head(me, type, rows, n_in, n_words));
  DN_TRY(check_answers(me, n_words, temperature, n_listed, 0));
  DN_CHECK(n_listed >= 1, "%s: no words are listed", me);
  if (rows == 0) return 0;
  DN_TRY(check_array(me, "X", X, ldx, n_in, type, false));
  DN_TRY(check_array(me, "E", E, lde, n_in, type, false));
  DN_TRY(check_array(me, "words", words, 1, 1, DNPEFF_F32, false));
  DN_TRY(check_array(me, "logits", logits, 1, 1, DNPEFF_F32, false));
  DN_TRY(check_array(me, "loss", loss, 1, 1, DNPEFF_F32, true));
  DN_TRY(check_array(me, "logp", logp, 1, 1, DNPEFF_F32, true));
  DN_TRY(check_array(me, "lse", lse, 1, 1, DNPEFF_F32, true));
  answer_args a{};
  a.rows = rows, a.n_in = n_in, a.words = n_words, a.X = X, a.ldx = ldx, a.E = E, a.lde = lde, a.inv_heat = 1.f / temperature;
  a.n_given = n_listed, a.given = words, a.logp = logp, a.lse = lse;
  if (loss) a.teacher = logits, a.loss = loss;
  if (!loss && !logp) a.n_given = 0;
  return DN_BY_TYPE(type, answers_forward<T>((hipStream_t)stream, me, a, (char*)workspace, workspace_bytes));
}

DN_API int dnpeff_vocab_distill_backward(void* stream, int type, int64_t rows, int64_t n_in, int64_t n_words, const void* X, int64_t ldx,
                                         const void* E, int64_t lde, float temperature, int n_listed, const int32_t* words,
                                         const float* logits, const float* logp, const float* lse, const float* dloss, void* dX,
                                         int64_t lddx, void* dE, int64_t ldde, void* workspace, int64_t workspace_bytes) {
  clear_error();
  const char* me = "dnpeff_vocab_distill_backward";
  const bool none = rows == 0;
  DN_TRY(check_head(me, type, rows, n_in, n_words));
  DN_TRY(check_answers(me, n_words, temperature, n_listed, 0));
  DN_CHECK(n_listed >= 1, "%s: no words are listed", me);
  DN_TRY(check_array(me, "X", X, ldx, n_in, type, none));
  DN_TRY(check_array(me, "E", E, lde, n_in, type, none));
  DN_TRY(check_array(me, "words", words, 1, 1, DNPEFF_F32, none));
  DN_TRY(check_array(me, "logits", logits, 1, 1, DNPEFF_F32, none));
  DN_TRY(check_array(me, "logp", logp, 1, 1, DNPEFF_F32, none));
  DN_TRY(check_array(me, "lse", lse, 1, 1, DNPEFF_F32, none));
  DN_TRY(check_array(me, "dloss", dloss, 1, 1, DNPEFF_F32, none));
  DN_TRY(check_array(me, "dX", dX, lddx, n_in, type, true));
  DN_TRY(check_array(me, "dE", dE, ldde, n_in, type, true));
  slope_args s{};
  s.rows = rows, s.words = n_words, s.many = n_listed, s.given = words, s.logp = logp, s.lse = lse;
  s.teacher = logits, s.dloss = dloss, s.inv_heat = 1.f / temperature;
  return DN_BY_TYPE(type, answers_backward<T>((hipStream_t)stream, me, s, n_in, X, ldx, E, lde, dX, lddx, dE, ldde, (char*)workspace,
                                              workspace_bytes));
}
