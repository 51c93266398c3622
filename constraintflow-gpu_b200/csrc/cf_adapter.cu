// Rows of many requests through an affine layer with per-request low-rank adapters
// (cf_adapter_matmul): checks, workspace and the choice of kernels.  With x [T, K], y [T, N]
// and, for the rows of a request with adapter e,
//   v = s_e x P_e   [T, R]      P_e: A_e^T (project) or B_e (substitute)
//   y = x M + b + v Q_e         M: W^T or W;  Q_e: B_e^T or A_e
// a shrink kernel writes v to the workspace and a product kernel adds v Q_e to its tiles.
#include "cf_adapter.cuh"
#include "cf_tc.cuh"

namespace cf {
namespace {

using namespace adapter;

int elem_bytes(int dtype) { return dtype == CF_F32 ? 4 : 2; }

cf_status check_layer(const cf_adapter_layer* L) {
  CF_REQUIRE(L, CF_ERR_NULL, "adapter_matmul: NULL layer");
  CF_REQUIRE(L->dtype == CF_F32 || L->dtype == CF_BF16 || L->dtype == CF_F16, CF_ERR_UNSUPPORTED,
             "adapter_matmul: dtype %d", L->dtype);
  CF_REQUIRE(L->n_out >= 0 && L->n_in >= 0 && L->n_adapters >= 0 && L->rank >= 0, CF_ERR_SHAPE,
             "adapter_matmul: negative size");
  CF_REQUIRE(L->n_out <= kMaxWidth && L->n_in <= kMaxWidth, CF_ERR_SHAPE, "adapter_matmul: layer too wide");
  CF_REQUIRE(L->w_rs >= L->n_in, CF_ERR_SHAPE, "adapter_matmul: rows of W overlap");
  if (L->n_adapters > 0 && L->rank > 0)
    CF_REQUIRE(L->a_rs >= L->n_in && L->b_rs >= L->rank && L->a_es >= 0 && L->b_es >= 0, CF_ERR_SHAPE,
               "adapter_matmul: rows of A or B overlap");
  return CF_OK;
}

}  // namespace
}  // namespace cf

using namespace cf;

namespace {

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

struct Operand {
  const void* p;
  int64_t entries, rows, cols, es, rs;
  int64_t pad = 0;  // zeros in place of no columns
};

// What the kernels cannot read where it lies is copied (16-bit data only): TMA wants 16-byte
// aligned rows and adapters, and adapters that do not overlap.
bool aligned(const Operand& o, int64_t size) {
  return o.cols > 0 && (uintptr_t)o.p % 16 == 0 && o.rs * size % 16 == 0 && o.rs >= o.cols &&
         (o.entries == 1 || (o.es * size % 16 == 0 && o.es >= o.rows * o.rs));
}

// (no columns of x: nothing to adapt)
bool has_adapters(const cf_adapter_layer& L, int64_t K) { return L.n_adapters > 0 && L.rank > 0 && K > 0; }

// A few rows go over the weights on the CUDA cores.  float32, against the tiles: 8 rows of 4096 x
// 4096 19 us and 38, 16 rows 36 and 38; 64 rows of 200 x 784 7 and 21, 128 of 512 x 512 23 both.
// 16-bit, rows of W along the contraction: 1 row of 4096 x 4096 5.4 and 11.2, 2 rows 7.3 and 11.0, 4
// rows 11 both; 8 rows of 512 x 512 with adapters 5.5 and 8.6.  16-bit the other way: never (1 row of
// 4096 x 4096 15 and 11).
bool few_rows(const cf_adapter_layer& L, bool substitute, int64_t T) {
  const double weights = (double)L.n_out * L.n_in;
  if (L.dtype == CF_F32) return T <= 8 || (T <= 1024 && T * weights <= 16777216.0);
  return !substitute && (T <= 2 || (T <= 8 && weights <= 1048576.0));
}

// With few rows a request, a tile of the tensor cores would be multiplied once for each of its
// requests: v row by row on the CUDA cores instead.  The mean decides for all rows, empty requests
// included: 4000 rows of one request take 127 us (4096 x 4096 bfloat16, rank 16), 241 beside 300 requests
// of one row, 202 beside 300 of none.
bool rows_alone(int64_t T, int64_t n_requests) { return T < 16 * n_requests; }

// The workspace's parts, from `base` on (NULL: only their sizes are asked for); returns its bytes.
// x, M, A and B are pointed to their copies where they have one.
size_t workspace(const cf_adapter_layer& L, bool substitute, int64_t T, int64_t n_requests, Operand& x, Operand& W, Operand& A,
                 Operand& B, char* base, Problem* p, Pack* pack) {
  if (T <= 0) return 0;
  const bool adapters = has_adapters(L, x.cols);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    char* q = base ? base + at : nullptr;
    at += align256(bytes);
    return q;
  };
  if (adapters) {
    const int64_t ld = ceil_div(L.rank, 8) * 8;
    char* v = take((size_t)T * ld * 4);
    char *hi = nullptr, *lo = nullptr;
    if (L.dtype == CF_BF16) {
      hi = take((size_t)T * ld * 2);
      lo = take((size_t)T * ld * 2);
    }
    char* tile_e = take((size_t)ceil_div(T, kBM) * 4);
    char* tile_q = take((size_t)ceil_div(T, kBM) * 4);
    if (p) {
      p->v = (float*)v, p->v_rs = ld;
      p->v_hi = (__nv_bfloat16*)hi, p->v_lo = (__nv_bfloat16*)lo;
      p->tile_e = (int32_t*)tile_e, p->tile_q = (int32_t*)tile_q;
    }
  }
  if (L.dtype == CF_F32 || few_rows(L, substitute, T)) return at;
  auto copy = [&](Operand& o, int64_t cols) {  // rows of `cols` elements, zeros behind the data's
    if (aligned(o, 2)) return;
    const int64_t rs = ceil_div(cols, 8) * 8;
    char* to = take((size_t)o.entries * o.rows * rs * 2);
    if (!pack) return;
    pack->item[pack->n++] = {o.p, to, o.entries, o.rows, o.cols, o.es, o.rs, rs};
    o.p = to, o.rs = rs, o.es = o.rows * rs;
  };
  copy(x, x.cols > 0 ? x.cols : 8);
  copy(W, W.cols > 0 ? W.cols : W.pad);
  if (adapters && !rows_alone(T, n_requests)) {
    copy(A, A.cols);
    copy(B, B.cols);
  }
  return at;
}

Operand operand_x(const void* x, int64_t T, int64_t K, int64_t x_rs) {
  return {x, 1, T, K, 0, T > 1 ? x_rs : (x_rs >= K ? x_rs : K)};
}
// A contraction over nothing is one over eight zeros.
Operand operand_W(const cf_adapter_layer& L, bool substitute) {
  if (substitute && L.n_out == 0) return {nullptr, 1, 8, 0, 0, 0, L.n_in};
  return {L.W_dev, 1, L.n_out, L.n_in, 0, L.w_rs, 8};
}
Operand operand_A(const cf_adapter_layer& L) { return {L.A_dev, L.n_adapters, L.rank, L.n_in, L.a_es, L.a_rs}; }
Operand operand_B(const cf_adapter_layer& L) { return {L.B_dev, L.n_adapters, L.n_out, L.rank, L.b_es, L.b_rs}; }

}  // namespace

extern "C" size_t cf_adapter_workspace_bytes(const cf_adapter_layer* L, int32_t substitute, int64_t T, const void* x,
                                             int64_t x_rs, int64_t n_requests) {
  if (!L || T <= 0) return 0;
  Operand ox = operand_x(x, T, substitute ? L->n_out : L->n_in, x_rs), W = operand_W(*L, substitute != 0), A = operand_A(*L),
          B = operand_B(*L);
  return workspace(*L, substitute != 0, T, n_requests, ox, W, A, B, nullptr, nullptr, nullptr);
}

extern "C" cf_status cf_adapter_matmul(const cf_adapter_layer* L, int32_t substitute, int64_t T, const void* x,
                                       int64_t x_rs, int64_t n_requests, const int64_t* offsets, const int32_t* ids,
                                       void* y, int64_t y_rs, void* ws, size_t ws_bytes, void* stream) {
  clear_error();
  CF_INJECT("adapter_matmul");
  CF_TRY(check_layer(L));
  const int64_t K = substitute ? L->n_out : L->n_in, N = substitute ? L->n_in : L->n_out;
  CF_REQUIRE(T >= 0 && n_requests >= 0, CF_ERR_SHAPE, "adapter_matmul: negative size");
  CF_REQUIRE(T < 0x7fffff00 && n_requests < 0x7fffff00, CF_ERR_SHAPE, "adapter_matmul: too many rows");
  CF_REQUIRE(T <= 1 || (x_rs >= 0 && y_rs >= N), CF_ERR_SHAPE, "adapter_matmul: rows of y overlap");
  if (T == 0 || N == 0 || n_requests == 0) return CF_OK;
  const bool adapters = has_adapters(*L, K);
  CF_REQUIRE(y && offsets && ids && (K == 0 || (x && L->W_dev)), CF_ERR_NULL, "adapter_matmul: NULL argument");
  CF_REQUIRE(!adapters || (L->A_dev && L->B_dev && L->scale_dev), CF_ERR_NULL, "adapter_matmul: NULL adapters");
  const int64_t size = elem_bytes(L->dtype);
  CF_REQUIRE(((uintptr_t)x | (uintptr_t)y | (uintptr_t)L->W_dev | (uintptr_t)L->A_dev | (uintptr_t)L->B_dev |
              (uintptr_t)L->bias_dev) % size == 0,
             CF_ERR_SHAPE, "adapter_matmul: unaligned data");
  CF_REQUIRE((uintptr_t)offsets % 8 == 0 && ((uintptr_t)ids | (uintptr_t)L->scale_dev | (uintptr_t)L->ranks_dev) % 4 == 0,
             CF_ERR_SHAPE, "adapter_matmul: unaligned offsets, ids, scales or ranks");
  CF_REQUIRE(K == 0 || !rows_overlap(x, x_rs, K, y, y_rs, N, T, size), CF_ERR_SHAPE, "adapter_matmul: x and y overlap");
  Operand ox = operand_x(x, T, K, x_rs), W = operand_W(*L, substitute != 0), A = operand_A(*L), B = operand_B(*L);
  const size_t need = workspace(*L, substitute != 0, T, n_requests, ox, W, A, B, nullptr, nullptr, nullptr);
  const bool few = few_rows(*L, substitute != 0, T), rows = rows_alone(T, n_requests);
  CF_REQUIRE(!adapters || !(few || rows) || L->rank <= kMaxRowRank, CF_ERR_SHAPE,
             "adapter_matmul: rank %d for requests of few rows", (int)L->rank);
  CF_REQUIRE(ws_bytes >= need && (need == 0 || ws), CF_ERR_WORKSPACE, "adapter_matmul: workspace of %zu bytes, needs %zu",
             ws_bytes, need);
  CF_REQUIRE((uintptr_t)ws % 256 == 0, CF_ERR_WORKSPACE, "adapter_matmul: the workspace must be 256-byte aligned");
  Problem p = {};
  Pack pack = {};
  workspace(*L, substitute != 0, T, n_requests, ox, W, A, B, (char*)ws, &p, &pack);
  p.T = T, p.K = K, p.N = N;
  p.R = adapters ? L->rank : 0, p.E = adapters ? L->n_adapters : 0, p.Q = n_requests;
  p.x = ox.p, p.x_rs = ox.rs, p.M = W.p, p.y = y, p.y_rs = y_rs;
  p.scale = L->scale_dev, p.ranks = L->ranks_dev, p.offsets = offsets, p.ids = ids;
  // CF_FAULT=adapter_withhold_stage withholds one arrival so that a wait runs out
  p.max_polls = tc::wait_polls(), p.withhold = fault_injected("adapter_withhold_stage") ? 1 : 0;
  if (substitute) {
    p.m_ks = W.rs, p.m_ns = 1;
    p.P = B.p, p.p_es = B.es, p.p_ks = B.rs, p.p_rs = 1;
    p.Qm = A.p, p.q_es = A.es, p.q_rs = A.rs, p.q_ns = 1;
  } else {
    p.bias = L->bias_dev;
    p.m_ks = 1, p.m_ns = W.rs;
    p.P = A.p, p.p_es = A.es, p.p_ks = 1, p.p_rs = A.rs;
    p.Qm = B.p, p.q_es = B.es, p.q_rs = 1, p.q_ns = B.rs;
  }
  auto vec = [&](const void* base, int64_t s0, int64_t s1) {
    return (uintptr_t)base % 16 == 0 && s0 * size % 16 == 0 && s1 * size % 16 == 0;
  };
  p.x_vec = vec(ox.p, T > 1 ? ox.rs : 0, 0);
  p.m_vec = vec(W.p, W.rs, 0);
  const bool a_vec = adapters && vec(A.p, A.rs, A.es), b_vec = adapters && vec(B.p, B.rs, B.es);
  p.p_vec = substitute ? b_vec : a_vec;
  p.q_vec = substitute ? a_vec : b_vec;
  p.y_vec = vec(y, T > 1 ? y_rs : 0, 0);
  if (few) return launch_gemv(p, L->dtype, substitute != 0, as_stream(stream));
  if (L->dtype == CF_F32) return launch_f32(p, substitute != 0, rows, as_stream(stream));
  CF_TRY(launch_pack(pack, as_stream(stream)));
  if (K == 0) p.K = 8;
  return launch_tiles(p, L->dtype, substitute != 0, rows, adapters && aligned(A, 2) && aligned(B, 2),
                      as_stream(stream));
}

extern "C" cf_status cf_adapter_check(void* stream) {
  clear_error();
  int tiles = 0, wide = 0, f32 = 0;
  CF_TRY(take_site_tiles(&tiles, as_stream(stream)));
  CF_TRY(take_site_wide(&wide, as_stream(stream)));
  CF_TRY(take_site_f32(&f32, as_stream(stream)));
  const int site = tiles ? tiles : wide ? wide : f32;
  CF_REQUIRE(site == 0, CF_ERR_TIMEOUT, "adapter_matmul: a bounded wait gave up (site %d)", site);
  return CF_OK;
}
