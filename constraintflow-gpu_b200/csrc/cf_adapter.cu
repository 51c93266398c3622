// Rows of many requests through an affine layer with per-request low-rank adapters
// (cf_adapter_matmul): checks, workspace and the choice of kernels.  With x [T, K], y [T, N]
// and, for the rows of a request with adapter e,
//   v = s_e x P_e   [T, R]      P_e: A_e^T (project) or B_e (substitute)
//   y = x M + b + v Q_e         M: W^T or W;  Q_e: B_e^T or A_e
// a shrink kernel writes v to the workspace and a product kernel adds v Q_e to its tiles.
#include "cf_adapter.cuh"

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
  CF_REQUIRE(L->n_out <= 0x7fffff00 && L->n_in <= 0x7fffff00, CF_ERR_SHAPE, "adapter_matmul: layer too wide");
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

// The workspace's parts, from `base` on; returns its bytes.
size_t workspace(const cf_adapter_layer& L, int64_t T, char* base, Problem* p) {
  if (T <= 0 || L.rank <= 0 || L.n_adapters <= 0) return 0;
  const int64_t ld = ceil_div(L.rank, 8) * 8;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    char* q = base ? base + at : nullptr;
    at += align256(bytes);
    return q;
  };
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
  return at;
}

}  // namespace

extern "C" size_t cf_adapter_workspace_bytes(const cf_adapter_layer* L, int32_t, int64_t T, int64_t) {
  return L ? workspace(*L, T, nullptr, nullptr) : 0;
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
  const bool adapters = L->n_adapters > 0 && L->rank > 0;
  CF_REQUIRE(y && offsets && ids && (K == 0 || (x && L->W_dev)), CF_ERR_NULL, "adapter_matmul: NULL argument");
  CF_REQUIRE(!adapters || (L->A_dev && L->B_dev && L->scale_dev), CF_ERR_NULL, "adapter_matmul: NULL adapters");
  const size_t need = workspace(*L, T, nullptr, nullptr);
  CF_REQUIRE(ws_bytes >= need && (need == 0 || ws), CF_ERR_WORKSPACE, "adapter_matmul: workspace of %zu bytes, needs %zu",
             ws_bytes, need);
  CF_REQUIRE((uintptr_t)ws % 256 == 0, CF_ERR_WORKSPACE, "adapter_matmul: the workspace must be 256-byte aligned");
  const int64_t size = elem_bytes(L->dtype);
  CF_REQUIRE(((uintptr_t)x | (uintptr_t)y | (uintptr_t)L->W_dev | (uintptr_t)L->A_dev | (uintptr_t)L->B_dev |
              (uintptr_t)L->bias_dev) % size == 0,
             CF_ERR_SHAPE, "adapter_matmul: unaligned data");
  Problem p = {};
  p.T = T, p.K = K, p.N = N;
  p.R = adapters ? L->rank : 0, p.E = adapters ? L->n_adapters : 0, p.Q = n_requests;
  p.x = x, p.x_rs = x_rs, p.M = L->W_dev, p.y = y, p.y_rs = y_rs;
  p.scale = L->scale_dev, p.ranks = L->ranks_dev, p.offsets = offsets, p.ids = ids;
  if (substitute) {
    p.m_ks = L->w_rs, p.m_ns = 1;
    p.P = L->B_dev, p.p_es = L->b_es, p.p_ks = L->b_rs, p.p_rs = 1;
    p.Qm = L->A_dev, p.q_es = L->a_es, p.q_rs = L->a_rs, p.q_ns = 1;
  } else {
    p.bias = L->bias_dev;
    p.m_ks = 1, p.m_ns = L->w_rs;
    p.P = L->A_dev, p.p_es = L->a_es, p.p_ks = 1, p.p_rs = L->a_rs;
    p.Qm = L->B_dev, p.q_es = L->b_es, p.q_rs = 1, p.q_ns = L->b_rs;
  }
  auto vec = [&](const void* base, int64_t s0, int64_t s1) {
    return (uintptr_t)base % 16 == 0 && s0 * size % 16 == 0 && s1 * size % 16 == 0;
  };
  p.x_vec = vec(x, T > 1 ? x_rs : 0, 0);
  p.m_vec = vec(L->W_dev, L->w_rs, 0);
  const bool a_vec = adapters && vec(L->A_dev, L->a_rs, L->a_es), b_vec = adapters && vec(L->B_dev, L->b_rs, L->b_es);
  p.p_vec = substitute ? b_vec : a_vec;
  p.q_vec = substitute ? a_vec : b_vec;
  p.y_vec = vec(y, T > 1 ? y_rs : 0, 0);
  workspace(*L, T, (char*)ws, &p);
  // Tensor maps want 16-byte strides, and adapters that do not overlap.
  const bool tma = L->dtype != CF_F32 && K > 0 && p.x_vec && p.m_vec && x_rs * size % 16 == 0 && x_rs >= K;
  const bool lowrank = a_vec && b_vec && (L->n_adapters == 1 || (L->a_es >= L->rank * L->a_rs &&
                                                                 L->b_es >= L->n_out * L->b_rs));
  // With few rows a request, a tile of the tensor cores would be multiplied once for each of
  // its requests: v row by row on the CUDA cores instead.
  const bool rows = T < 16 * n_requests;
  if (L->dtype == CF_F32) return launch_f32(p, substitute != 0, rows, as_stream(stream));
  return launch_tiles(p, L->dtype, substitute != 0, tma, rows, lowrank, as_stream(stream));
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
