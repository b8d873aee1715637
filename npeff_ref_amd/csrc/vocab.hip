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

// One wave per token.
__global__ __launch_bounds__(256) void k_join_loss(int64_t rows, int parts_n, const float2* parts, const float* hit, const int32_t* labels,
                                                   int64_t words, float* loss, float* lse) {
  const int64_t m = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
  const int lane = threadIdx.x & 63;
  if (m >= rows) return;
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
    most = most > 0.f ? fmaxf(most, 1e-36f) : 1.f;
    both[0] = top / most;
    both[1] = most / top;
  }
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
      : m{{X, ldx, rows, n_in, 1, 0, 0}, {E, lde, words, n_in, 1, 0, 0}} {
    if (!is_few(rows, 0))
      for (const matrix& q : m) packs += packed_bytes<T>(q);
    parts = round256(rows * ceil_div(words, is_few(rows, 0) ? 16 : 128) * 8);
    all = packs + parts + round256(rows * 4);
  }
};
template <class T>
struct grad_room {
  int64_t packs = 0, piece, g, sums, parts, all;
  matrix m[2];
  grad_room(int64_t rows, int64_t n_in, int64_t words, const void* X, int64_t ldx, const void* E, int64_t lde)
      : m{{X, ldx, rows, n_in, 1, 0, 0}, {E, lde, words, n_in, 1, 0, 0}} {
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
  const bool few = is_few(rows, 0);
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
  k_join_loss<<<(unsigned)ceil_div(rows, 4), 256, 0, st>>>(rows, parts_n, p.parts, p.hit, labels, words, loss, lse);
  DN_LAUNCH_CHECK();
  return 0;
}

template <class T>
int loss_backward(hipStream_t st, int64_t rows, int64_t n_in, int64_t words, const void* X, int64_t ldx, const void* E, int64_t lde,
                  const int32_t* labels, const float* lse, const float* dloss, void* dX, int64_t lddx, void* dE, int64_t ldde, char* ws,
                  int64_t ws_bytes) {
  grad_room<T> r(rows, n_in, words, X, ldx, E, lde);
  DN_TRY(check_room("dnpeff_vocab_loss_backward", r.all, ws, ws_bytes));
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
  if (backward_bytes) *backward_bytes = DN_BY_TYPE(type, (grad_room<T>(rows, n_in, n_words, p, n_in, p, n_in).all));
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
