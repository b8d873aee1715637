// Products of a layer with their epilogues, one weight for all rows or one per group of rows, their backward pass, and
// weight gradients per example: the dense Fisher rows that dnpeff_topk_rows takes.
//
//   Z = X W^T + b,  Y = act(Z) + R
//   dZ = dY act'(Z),  dX = dZ W,  dW = dZ^T X,  db = column sums of dZ          (per group: rows and W of the group)
//   out[e] = dY_e^T X_e, squared where asked for                                 (e: the rows of an example)
#include "tiles.hpp"

using namespace dn;
using namespace dn::tl;

namespace dn {
namespace tl {
DN_STORE_PRODUCTS(, float)
DN_STORE_PRODUCTS(, _Float16)
DN_STORE_PRODUCTS(, __bf16)
}  // namespace tl
}  // namespace dn

namespace {

// Rows of a group that one workgroup of k_slopes takes (a wave every fourth of them): 64, or 16 where those would leave
// CUs without work (777 x 515 in fp32: 20 -> 8.5 us), or 256 where a launch would not hold so many workgroups.
int slope_rows(int64_t rows, int64_t n_out, int size) {
  if (rows >= (int64_t)1 << 29) return 256;
  return ceil_div(rows, 64) * ceil_div(n_out * size, 1024) >= 1024 ? 64 : 16;
}

// dZ = dY act'(Z), and the column sums of each tile of rows.  A lane has 16 bytes of each row.
template <class T>
__global__ __launch_bounds__(256) void k_slopes(group_rows G, int64_t N, const T* dY, int64_t ldy, const T* Z, int64_t ldz, int act,
                                                typename num<T>::op* dZ, int64_t ldd, float* sums, int tall) {
  constexpr bool EXACT = sizeof(T) == 4;
  constexpr int W = 16 / sizeof(T);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int group, within;
  group_of_tile(G, tall, lane, blockIdx.x, &group, &within);
  if (group < 0) return;
  const int64_t m0 = G.first(group) + (int64_t)within * tall, m_end = G.last(group);
  const bool held = group < G.groups;
  const int64_t n = (((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * 64 + lane) * W;
  const int there = n < N ? (N - n < W ? (int)(N - n) : W) : 0;
  float sum[W];
#pragma unroll
  for (int t = 0; t < W; t++) sum[t] = 0.f;
#pragma unroll 4
  for (int r = wave; r < tall; r += 4) {
    const int64_t m = m0 + r;
    if (m >= m_end) break;
    float g[W], z[W];
#pragma unroll
    for (int t = 0; t < W; t++) g[t] = z[t] = 0.f;
    if (held && there == W) {
      load_row<T, W>(dY + m * ldy + n, g);
      if (act != DNPEFF_ACT_NONE) load_row<T, W>(Z + m * ldz + n, z);
    } else if (held) {
#pragma unroll
      for (int t = 0; t < W; t++)
        if (t < there) {
          g[t] = (float)dY[m * ldy + n + t];
          if (act != DNPEFF_ACT_NONE) z[t] = (float)Z[m * ldz + n + t];
        }
    }
    slopes_of<EXACT, W>(g, z, act);
#pragma unroll
    for (int t = 0; t < W; t++) sum[t] += g[t];
    if (dZ && n < ldd) store_op<T, W>(dZ + m * ldd + n, G.rows * ldd, g);  // (past the last column: zeros)
  }
  if (!sums) return;
  __shared__ float side[4][W][64];
#pragma unroll
  for (int t = 0; t < W; t++) side[wave][t][lane] = sum[t];
  __syncthreads();
  if (wave == 0) {
#pragma unroll
    for (int t = 0; t < W; t++)
      if (t < there) sums[blockIdx.x * N + n + t] = (side[0][t][lane] + side[1][t][lane]) + (side[2][t][lane] + side[3][t][lane]);
  }
}

// db[g] = the sums of the group's tiles, in their order.
template <class T>
__global__ __launch_bounds__(256) void k_bias_sums(group_rows G, int64_t N, const float* sums, int tall, int tiles_most, T* db) {
  const int lane = threadIdx.x & 63, g = blockIdx.y;
  int before = 0;
  for (int b = 0; b < g; b += 64) {
    const int t = b + lane < g ? (int)((G.count(b + lane) + tall - 1) / tall) : 0;
    before = add_up(before, __shfl(wave_scan(t, lane), 63, 64));
  }
  int tiles = (int)((G.count(g) + tall - 1) / tall);
  if (tiles > tiles_most - before) tiles = tiles_most - before;  // (groups that overlap: no more than there were)
  const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (n >= N) return;
  float s = 0.f;
#pragma unroll 8
  for (int t = 0; t < tiles; t++) s += sums[(int64_t)(before + t) * N + n];
  db[g * N + n] = (T)s;
}

int64_t slope_tiles(int64_t rows, int groups, int tall) { return group_rows{nullptr, groups, rows}.most_tiles(tall); }

struct layer {
  int64_t rows, n_in, n_out;
  int groups;
  const int64_t* ends;
  bool grouped() const { return ends != nullptr; }
};

int check_layer(const char* what, int type, const layer& l) {
  DN_CHECK(type == DNPEFF_F32 || type == DNPEFF_F16 || type == DNPEFF_BF16, "%s: unknown type %d", what, type);
  DN_CHECK(l.rows >= 0 && l.n_in >= 1 && l.n_out >= 1, "%s: rows = %lld, n_in = %lld, n_out = %lld", what, (long long)l.rows,
           (long long)l.n_in, (long long)l.n_out);
  DN_CHECK(l.rows < ((int64_t)1 << 31) && l.n_in <= ((int64_t)1 << 24) && l.n_out <= ((int64_t)1 << 24),
           "%s: %lld rows, widths %lld and %lld: less than 2^31 rows and widths up to 2^24 are taken", what, (long long)l.rows,
           (long long)l.n_in, (long long)l.n_out);
  DN_CHECK((l.ends == nullptr) == (l.groups == 0) && l.groups >= 0 && l.groups <= 65535, "%s: %d groups, their ends %s (65535 at most)",
           what, l.groups, l.ends ? "given" : "not given");
  return 0;
}
// Matrices of groups `apart` elements from one to the next; those that are written must not share elements: each after the
// one before, or a row of each side by side.
int check_apart(const char* what, const char* name, const layer& l, const void* p, int64_t ld, int64_t apart, bool written) {
  if (p == nullptr || l.groups < 2) return 0;
  const bool after = apart >= (l.n_out - 1) * ld + l.n_in, beside = apart >= l.n_in && (l.groups - 1) * apart + l.n_in <= ld;
  DN_CHECK(written ? after || beside : apart >= 0, "%s: matrices of %s are %lld elements apart, their rows %lld", what, name, (long long)apart,
           (long long)ld);
  return 0;
}
int check_act(const char* what, int act) {
  DN_CHECK(act >= DNPEFF_ACT_NONE && act <= DNPEFF_ACT_SILU, "%s: unknown activation %d", what, act);
  return 0;
}
group_rows rows_of(const layer& l) { return group_rows{l.ends, l.grouped() ? l.groups : 1, l.rows}; }

matrix rows_matrix(const layer& l, const void* p, int64_t ld, int64_t width) { return matrix{p, ld, l.rows, width, 1, 0, 0, nullptr}; }
matrix weight_matrix(const layer& l, const void* p, int64_t ld, int64_t sheet) {
  return matrix{p, ld, l.n_out, l.n_in, l.grouped() ? l.groups : 1, sheet, 0, nullptr};
}

// Parts of a workspace: copies of operands that do not lie well, then the rest.
template <class T>
struct forward_room {
  int64_t packs = 0, parts = 0, all = 0;
  matrix m[2];
  forward_room(const layer& l, const void* X, int64_t ldx, const void* W, int64_t ldw, int64_t w_group)
      : m{rows_matrix(l, X, ldx, l.n_in), weight_matrix(l, W, ldw, w_group)} {
    if (is_few<T>(l.rows, l.groups, l.n_out, l.n_in)) return;
    for (const matrix& q : m) packs += packed_bytes<T>(q);
    parts = l.grouped() ? 0 : round256(4 * split_floats<T>(l.rows, l.n_out, l.n_in));
    all = packs + parts;
  }
};
template <class T>
struct backward_room {
  int64_t packs = 0, dz = 0, sums = 0, parts = 0, all;
  int n = 0;
  matrix m[3];
  int x = -1, w = -1, y = -1;  // which of m
  backward_room(const layer& l, const void* dY, int64_t lddy, const void* X, int64_t ldx, const void* W, int64_t ldw, int64_t w_group, int act,
                bool dX, bool dW, bool dbias) {
    if (act != DNPEFF_ACT_NONE && (dX || dW))
      dz = round256(num<T>::PLANES * l.rows * packed_ld(l.n_out) * 2);
    else if (dX || dW)
      m[y = n++] = rows_matrix(l, dY, lddy, l.n_out);
    if (dW) m[x = n++] = rows_matrix(l, X, ldx, l.n_in);
    if (dX) m[w = n++] = weight_matrix(l, W, ldw, w_group);
    for (int i = 0; i < n; i++) packs += packed_bytes<T>(m[i]);
    if (dbias) sums = round256(slope_tiles(l.rows, l.grouped() ? l.groups : 1, slope_rows(l.rows, l.n_out, sizeof(T))) * l.n_out * 4);
    if (!l.grouped()) {
      const int64_t a = dX ? split_floats<T>(l.rows, l.n_in, l.n_out) : 0, b = dW ? split_floats<T>(l.n_out, l.n_in, l.rows) : 0;
      parts = round256(4 * (a > b ? a : b));
    }
    all = packs + dz + sums + parts;
  }
};
template <class T>
struct example_room {
  int64_t packs = 0;
  matrix m[2];
  example_room(const layer& l, const void* dY, int64_t lddy, const void* X, int64_t ldx)
      : m{rows_matrix(l, dY, lddy, l.n_out), rows_matrix(l, X, ldx, l.n_in)} {
    for (const matrix& q : m) packs += packed_bytes<T>(q);
  }
};

int check_room(const char* what, int64_t need, const void* ws, int64_t bytes) {
  DN_CHECK(need == 0 || (ws != nullptr && bytes >= need && (uintptr_t)ws % 16 == 0),
           "%s: a workspace of %lld bytes, aligned to 16, is needed", what, (long long)need);
  return 0;
}

template <class T>
int forward(hipStream_t st, const layer& l, const void* X, int64_t ldx, const void* W, int64_t ldw, int64_t w_group, const void* bias, int act,
            const void* residual, int64_t ldr, void* Y, int64_t ldy, void* pre, int64_t ldp, char* ws, int64_t ws_bytes) {
  forward_room<T> room(l, X, ldx, W, ldw, w_group);
  DN_TRY(check_room("dnpeff_linear", room.all, ws, ws_bytes));
  const bool few = is_few<T>(l.rows, l.groups, l.n_out, l.n_in);
  if (!few) DN_TRY(pack<T>(room.m, 2, ws, st));
  args p{};
  p.A = room.m[0].p, p.lda = room.m[0].ld, p.B = room.m[1].p, p.ldb = room.m[1].ld, p.b_group = room.m[1].sheet;
  p.a_plane = room.m[0].plane, p.b_plane = room.m[1].plane;
  p.M = l.rows, p.N = l.n_out, p.K = l.n_in;
  p.mode = l.grouped() ? BY_ROWS : ONE;
  p.G = rows_of(l);
  p.out = Y, p.ldc = ldy, p.pre = pre, p.ldp = ldp, p.residual = residual, p.ldr = ldr, p.bias = bias, p.act = act;
  if (few) return launch_few<T, E_LINEAR>(p, st);
  return launch_product<T, true, true, E_LINEAR>(p, room.parts ? (float*)(ws + room.packs) : nullptr, st);
}

template <class T>
int backward(hipStream_t st, const layer& l, const void* dY, int64_t lddy, const void* X, int64_t ldx, const void* W, int64_t ldw,
             int64_t w_group, const void* pre, int64_t ldp, int act, void* dX, int64_t lddx, void* dW, int64_t lddw, int64_t dw_group,
             void* dbias, char* ws, int64_t ws_bytes) {
  backward_room<T> room(l, dY, lddy, X, ldx, W, ldw, w_group, act, dX, dW, dbias);
  DN_TRY(check_room("dnpeff_linear_backward", room.all, ws, ws_bytes));
  const group_rows G = rows_of(l);
  DN_TRY(pack<T>(room.m, room.n, ws, st));
  char* at = ws + room.packs;
  typedef typename num<T>::op O;
  O* dz = room.dz ? (O*)at : nullptr;
  at += room.dz;
  float* sums = dbias ? (float*)at : nullptr;
  at += room.sums;
  float* parts = room.parts ? (float*)at : nullptr;
  constexpr int PIECE = 16 / sizeof(T);
  const int tall = slope_rows(l.rows, l.n_out, sizeof(T));
  if ((dz || dbias) && l.rows > 0) {
    constexpr int64_t STRIPS = 32768;  // of columns in a launch's second dimension, the rest in its third
    const int64_t strips = ceil_div(l.n_out, 64 * PIECE);
    const dim3 grid((unsigned)slope_tiles(l.rows, G.groups, tall), (unsigned)(strips < STRIPS ? strips : STRIPS), (unsigned)ceil_div(strips, STRIPS));
    k_slopes<T><<<grid, 256, 0, st>>>(G, l.n_out, (const T*)dY, lddy, (const T*)pre, ldp, act, dz, packed_ld(l.n_out), sums, tall);
    DN_LAUNCH_CHECK();
  }
  if (dbias) {
    k_bias_sums<T><<<dim3((unsigned)ceil_div(l.n_out, 256), (unsigned)G.groups), 256, 0, st>>>(G, l.n_out, sums, tall,
                                                                                               (int)slope_tiles(l.rows, G.groups, tall), (T*)dbias);
    DN_LAUNCH_CHECK();
  }
  const void* g = dz ? dz : room.y >= 0 ? room.m[room.y].p : nullptr;
  const int64_t ldg = dz ? packed_ld(l.n_out) : room.y >= 0 ? room.m[room.y].ld : 0;
  const int64_t plane = dz ? l.rows * ldg : room.y >= 0 ? room.m[room.y].plane : 0;
  if (dX) {
    args p{};
    p.A = g, p.lda = ldg, p.B = room.m[room.w].p, p.ldb = room.m[room.w].ld, p.b_group = room.m[room.w].sheet;
    p.a_plane = plane, p.b_plane = room.m[room.w].plane;
    p.M = l.rows, p.N = l.n_in, p.K = l.n_out;
    p.mode = l.grouped() ? BY_ROWS : ONE;
    p.G = G;
    p.out = dX, p.ldo = lddx;
    DN_TRY((launch_product<T, true, false, E_STORE>(p, parts, st)));
  }
  if (dW) {
    args p{};
    p.A = g, p.lda = ldg, p.B = room.m[room.x].p, p.ldb = room.m[room.x].ld;
    p.a_plane = plane, p.b_plane = room.m[room.x].plane;
    p.M = l.n_out, p.N = l.n_in, p.K = l.rows;
    p.mode = l.grouped() ? BY_REDUCTION : ONE;
    p.G = G;
    p.out = dW, p.ldo = lddw, p.c_group = dw_group;
    DN_TRY((launch_product<T, false, false, E_STORE>(p, parts, st)));
  }
  return 0;
}

template <class T>
int example_grads(hipStream_t st, const layer& l, const void* dY, int64_t lddy, const void* X, int64_t ldx, float* out, int square, char* ws,
                  int64_t ws_bytes) {
  example_room<T> room(l, dY, lddy, X, ldx);
  DN_TRY(check_room("dnpeff_example_grads", room.packs, ws, ws_bytes));
  DN_TRY(pack<T>(room.m, 2, ws, st));
  args p{};
  p.A = room.m[0].p, p.lda = room.m[0].ld, p.B = room.m[1].p, p.ldb = room.m[1].ld;
  p.a_plane = room.m[0].plane, p.b_plane = room.m[1].plane;
  p.M = l.n_out, p.N = l.n_in, p.K = l.rows;
  p.mode = BY_REDUCTION;
  p.G = rows_of(l);
  p.out = out, p.out_f32 = 1, p.square = square, p.ldo = l.n_in, p.c_group = l.n_out * l.n_in;
  return launch_product<T, false, false, E_STORE>(p, nullptr, st);
}

// Operands as a workspace is asked for: of whole rows, on 16 bytes or (not aligned) on none.
struct as_if {
  const void* p;
  int64_t in, out;
  as_if(bool aligned, int64_t n_in, int64_t n_out) : p((const void*)(uintptr_t)(aligned ? 16 : 1)), in(n_in), out(n_out) {}
};

}  // namespace

DN_API int dnpeff_linear_workspace(int type, int64_t rows, int64_t n_in, int64_t n_out, int n_groups, int aligned, int64_t* forward_bytes,
                                   int64_t* backward_bytes, int64_t* example_bytes) {
  clear_error();
  static const int64_t some = 0;
  const layer l{rows, n_in, n_out, n_groups, n_groups > 0 ? &some : nullptr};
  DN_TRY(check_layer("dnpeff_linear_workspace", type, l));
  const as_if a(aligned, n_in, n_out);
  const int64_t sheet = n_in * n_out;
  if (forward_bytes) *forward_bytes = DN_BY_TYPE(type, (forward_room<T>(l, a.p, a.in, a.p, a.in, sheet).all));
  if (backward_bytes) {  // the larger of the two ways that dZ comes
    const int64_t y = DN_BY_TYPE(type, (backward_room<T>(l, a.p, a.out, a.p, a.in, a.p, a.in, sheet, DNPEFF_ACT_NONE, true, true, true).all));
    const int64_t z = DN_BY_TYPE(type, (backward_room<T>(l, a.p, a.out, a.p, a.in, a.p, a.in, sheet, DNPEFF_ACT_SILU, true, true, true).all));
    *backward_bytes = y > z ? y : z;
  }
  if (example_bytes) *example_bytes = DN_BY_TYPE(type, (example_room<T>(l, a.p, a.out, a.p, a.in).packs));
  return 0;
}

DN_API int dnpeff_linear(void* stream, int type, int64_t rows, int64_t n_in, int64_t n_out, const void* X, int64_t ldx, const void* W,
                         int64_t ldw, int64_t w_group, const void* bias, int act, const void* residual, int64_t ldr, void* Y, int64_t ldy,
                         void* pre, int64_t ldp, int n_groups, const int64_t* ends, void* workspace, int64_t workspace_bytes) {
  clear_error();
  const char* me = "dnpeff_linear";
  const layer l{rows, n_in, n_out, n_groups, ends};
  DN_TRY(check_layer(me, type, l));
  DN_TRY(check_act(me, act));
  if (rows == 0) return 0;
  DN_TRY(check_array(me, "X", X, ldx, n_in, type, false));
  DN_TRY(check_array(me, "W", W, ldw, n_in, type, false));
  DN_TRY(check_apart(me, "W", l, W, ldw, w_group, false));
  DN_TRY(check_array(me, "Y", Y, ldy, n_out, type, false));
  DN_TRY(check_array(me, "bias", bias, n_out, n_out, type, true));
  DN_TRY(check_array(me, "residual", residual, ldr, n_out, type, true));
  DN_TRY(check_array(me, "pre", pre, ldp, n_out, type, true));
  return DN_BY_TYPE(type, forward<T>((hipStream_t)stream, l, X, ldx, W, ldw, w_group, bias, act, residual, ldr, Y, ldy, pre, ldp,
                                     (char*)workspace, workspace_bytes));
}

DN_API int dnpeff_linear_backward(void* stream, int type, int64_t rows, int64_t n_in, int64_t n_out, const void* dY, int64_t lddy,
                                  const void* X, int64_t ldx, const void* W, int64_t ldw, int64_t w_group, const void* pre, int64_t ldp,
                                  int act, void* dX, int64_t lddx, void* dW, int64_t lddw, int64_t dw_group, void* dbias, int n_groups,
                                  const int64_t* ends, void* workspace, int64_t workspace_bytes) {
  clear_error();
  const char* me = "dnpeff_linear_backward";
  const layer l{rows, n_in, n_out, n_groups, ends};
  DN_TRY(check_layer(me, type, l));
  DN_TRY(check_act(me, act));
  DN_TRY(check_array(me, "dY", dY, lddy, n_out, type, rows == 0));
  DN_TRY(check_array(me, "X", X, ldx, n_in, type, rows == 0 || !dW));
  DN_TRY(check_array(me, "W", W, ldw, n_in, type, !dX));
  DN_TRY(check_apart(me, "W", l, W, ldw, w_group, false));
  DN_TRY(check_array(me, "pre", pre, ldp, n_out, type, rows == 0 || act == DNPEFF_ACT_NONE));
  DN_TRY(check_array(me, "dX", dX, lddx, n_in, type, true));
  DN_TRY(check_array(me, "dW", dW, lddw, n_in, type, true));
  DN_TRY(check_apart(me, "dW", l, dW, lddw, dw_group, true));
  DN_TRY(check_array(me, "dbias", dbias, n_out, n_out, type, true));
  return DN_BY_TYPE(type, backward<T>((hipStream_t)stream, l, dY, lddy, X, ldx, W, ldw, w_group, pre, ldp, act, dX, lddx, dW, lddw,
                                      dw_group, dbias, (char*)workspace, workspace_bytes));
}

DN_API int dnpeff_example_grads(void* stream, int type, int64_t rows, int64_t n_in, int64_t n_out, const void* dY, int64_t lddy,
                                const void* X, int64_t ldx, int n_examples, const int64_t* ends, float* out, int square, void* workspace,
                                int64_t workspace_bytes) {
  clear_error();
  const char* me = "dnpeff_example_grads";
  const layer l{rows, n_in, n_out, n_examples, ends};
  DN_CHECK(n_examples >= 0, "%s: %d examples", me, n_examples);
  if (n_examples == 0) return 0;
  DN_TRY(check_layer(me, type, l));
  DN_TRY(check_array(me, "dY", dY, lddy, n_out, type, rows == 0));
  DN_TRY(check_array(me, "X", X, ldx, n_in, type, rows == 0));
  DN_TRY(check_array(me, "out", out, n_in, n_in, DNPEFF_F32, false));
  return DN_BY_TYPE(type, example_grads<T>((hipStream_t)stream, l, dY, lddy, X, ldx, out, square, (char*)workspace, workspace_bytes));
}
