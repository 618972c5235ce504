// psx_operators.cpp — entry points of the operators on parameter rows (include/psx.h): checks
// of arguments, and launches on the caller's stream.  Kernels: psx_adapter.hip,
// psx_checkpoint.hip, psx_bias.hip.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <exception>
#include <memory>
#include <utility>
#include <vector>

#include "psx_operators.hpp"

struct psx_adapters : psx::OpHandle {
  psx::DenseView a, b;
  psx::AdapterDev *d_ads = nullptr;
  int32_t *d_row_ids = nullptr;
  int32_t n = 0, max_rank = 0, rl = 0, num_rows = 0;
  ~psx_adapters() override {
    if (d_ads) (void)hipFree(d_ads);
    if (d_row_ids) (void)hipFree(d_row_ids);
  }
};

struct psx_position_bias : psx::OpHandle {
  psx::DenseView t;
  int64_t slot = 0;
  psx::BiasMap map{};
};

namespace {

using psx::op_fail;

#define OP_HIP(c, expr)                                              \
  do {                                                               \
    hipError_t _e = (expr);                                          \
    if (_e != hipSuccess) return psx::op_hip_fail((c), _e, #expr);   \
  } while (0)

size_t act_size(int32_t type) { return type == PSX_ACT_F32 ? 4 : 2; }

constexpr int64_t kMaxElements = (int64_t)1 << 46;   // products of the checks below fit 64 bits

bool overlap(const void *a, size_t na, const void *b, size_t nb) {
  return na && nb && (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}
size_t span(const psx_matrix *m) {
  return m->rows && m->cols ? (size_t)((m->rows - 1) * m->row_stride + m->cols) * act_size(m->type) : 0;
}

// rows x cols of `m`; an output has rows that do not overlap.
psx_status check_matrix(psx_ctx *c, const psx_matrix *m, int64_t rows, int64_t cols, bool output, const char *name) {
  const std::string at = std::string(name) + ": ";
  if (m->type < PSX_ACT_F32 || m->type > PSX_ACT_BF16 || m->reserved0)
    return op_fail(c, PSX_ERR_INVALID_ARG, at + "bad type");
  if (m->rows != rows || m->cols != cols)
    return op_fail(c, PSX_ERR_INVALID_ARG, at + std::to_string(m->rows) + " x " + std::to_string(m->cols) + ", expected " +
                                               std::to_string(rows) + " x " + std::to_string(cols));
  if (m->row_stride < (output ? cols : 0) || (rows && m->row_stride > kMaxElements / rows))
    return op_fail(c, PSX_ERR_INVALID_ARG, at + "bad row_stride");
  if (rows && cols && (!m->data || (uintptr_t)m->data % act_size(m->type)))
    return op_fail(c, PSX_ERR_INVALID_ARG, at + "null or misaligned data");
  return PSX_OK;
}

#define OP_TRY(expr)                        \
  do {                                      \
    psx_status _s = (expr);                 \
    if (_s != PSX_OK) return _s;            \
  } while (0)

psx_status check_requests(psx_ctx *c, const psx_requests *r) {
  if (!r || r->num_requests < 0 || r->reserved0 ||
      (r->num_requests && (!r->request_begin || !r->request_adapter)))
    return op_fail(c, PSX_ERR_INVALID_ARG, "bad psx_requests");
  if (((uintptr_t)r->request_begin | (uintptr_t)r->request_adapter) & 3)
    return op_fail(c, PSX_ERR_INVALID_ARG, "request arrays must be 4-byte aligned");
  return PSX_OK;
}

psx::BatchView batch_view(psx_adapters *s, const psx_requests *r, int64_t tokens) {
  psx::BatchView b{};
  b.begin = r->request_begin;
  b.which = r->request_adapter;
  b.ads = s->d_ads;
  b.requests = r->num_requests;
  b.adapters = s->n;
  b.tokens = (int32_t)tokens;
  b.status = psx::op_status(s->ctx);
  return b;
}

// The kernels' offsets within a block's tokens (64 at most) are 32 bits wide.
psx_status check_rows_apart(psx_ctx *c, const psx_matrix *m, const char *name) {
  if (m && m->rows > 1 && m->row_stride * (int64_t)act_size(m->type) > (int64_t)64 << 20)
    return op_fail(c, PSX_ERR_INVALID_ARG, std::string(name) + ": rows more than 64 MiB apart");
  return PSX_OK;
}
// Token indexes are 32 bits wide, and the grids of a call's kernels have to fit: shrink's (an
// item is a request, or its part of 64 tokens: 16 for the first 8192), expand's and grad's (for
// every 256 columns), join's.
psx_status check_tokens(psx_adapters *s, int64_t tokens, int64_t requests) {
  if (tokens < 0 || tokens > ((int64_t)1 << 30) || requests > ((int64_t)1 << 24))
    return op_fail(s->ctx, PSX_ERR_INVALID_ARG, "num_tokens past 2^30 or num_requests past 2^24");
  const int64_t d = std::max(s->a.cap, s->b.cap), across = (d + 255) / 256;
  const int64_t tile = psx::adapter_expand_tile(tokens, s->max_rank, 3);
  const int64_t items = psx::adapter_grad_most_chunks(tokens, d, s->max_rank) + s->n;
  if (!psx::grid_fits(tokens / 64 + requests + 512, 512) || !psx::grid_fits((tokens / tile + 1 + requests) * across, 256) ||
      !psx::grid_fits(2 * items * across, 256) || !psx::grid_fits(tokens * s->rl / 1024 + 1, 256))
    return op_fail(s->ctx, PSX_ERR_UNSUPPORTED, "too many tokens or requests for one call at these widths");
  return PSX_OK;
}

// Partial sums of one gradient: of an adapter with two items or more, so at most twice its
// tokens' chunks.  This and the sizes below serve fewer tokens, too.
int64_t grad_slots(psx_adapters *s, int64_t tokens, int64_t d) {
  const int64_t chunks = psx::adapter_grad_most_chunks(tokens, d, s->max_rank);
  return std::min(2 * chunks, chunks + s->n);
}
// Parts of v that expand adds, leaving the sum behind them.
int parts_read(int64_t tokens, int64_t d) {
  return psx::adapter_joins(tokens, d) ? 1 : psx::adapter_splits(tokens, d);
}
size_t aligned(size_t n) { return (n + 255) & ~(size_t)255; }
// v: its parts, and behind several that expand adds, their sum.
size_t part_values(psx_adapters *s, int64_t tokens) { return (size_t)tokens * (size_t)s->rl; }
size_t shrunk_size(psx_adapters *s, int64_t tokens, int64_t d) {
  size_t most = 0;
  for (int64_t t : {tokens, std::min<int64_t>(tokens, psx::kFewTokens)}) {   // fewer tokens can have more parts
    const int parts = psx::adapter_splits(t, d) + (parts_read(t, d) > 1 ? 1 : 0);
    most = std::max(most, (size_t)parts * part_values(s, t) * sizeof(float));
  }
  return aligned(most);
}
const float *whole_v(psx_adapters *s, const float *v, int64_t tokens, int64_t d) {
  const int parts = parts_read(tokens, d);
  return parts > 1 ? v + (size_t)parts * part_values(s, tokens) : v;
}
size_t partial_size(psx_adapters *s, int64_t tokens, int64_t d) {
  return aligned((size_t)grad_slots(s, tokens, d) * (size_t)s->max_rank * (size_t)d * sizeof(float));
}

// base (may be null) and out of one call: out is base, or apart from it.
psx_status check_out(psx_ctx *c, const psx_matrix *base, const psx_matrix *out, int64_t rows, int64_t cols) {
  OP_TRY(check_matrix(c, out, rows, cols, true, "out"));
  OP_TRY(check_rows_apart(c, out, "out"));
  if (!base) return PSX_OK;
  OP_TRY(check_matrix(c, base, rows, cols, false, "base"));
  OP_TRY(check_rows_apart(c, base, "base"));
  if (base->type != out->type) return op_fail(c, PSX_ERR_INVALID_ARG, "base and out differ in type");
  if (!(base->data == out->data && base->row_stride == out->row_stride) &&
      overlap(base->data, span(base), out->data, span(out)))
    return op_fail(c, PSX_ERR_INVALID_ARG, "out overlaps base without being it");
  return PSX_OK;
}

psx_status expand(psx_adapters *s, const psx::BatchView &b, float *v, int64_t v_width, bool use_b,
                  const psx_matrix *base, const psx_matrix *out, hipStream_t st) {
  psx::ExpandArgs e{};
  e.b = b;
  e.v = v;
  e.splits = parts_read(b.tokens, v_width);
  e.sum = e.splits > 1 ? const_cast<float *>(whole_v(s, v, b.tokens, v_width)) : nullptr;
  e.rl = s->rl;
  e.part = (int64_t)b.tokens * s->rl;
  e.w = use_b ? s->b.data : s->a.data;
  e.d = use_b ? s->b.cap : s->a.cap;
  e.use_b = use_b;
  e.max_rank = s->max_rank;
  e.base = base ? (const uint8_t *)base->data : nullptr;
  e.base_ld = base ? base->row_stride : 0;
  e.out = (uint8_t *)out->data;
  e.out_ld = out->row_stride;
  e.type = out->type;
  OP_HIP(s->ctx, psx::launch_adapter_expand(e, st));
  return PSX_OK;
}

// join: v's parts end in the first even where expand would add them.
psx_status shrink(psx_adapters *s, const psx::BatchView &b, const psx_matrix *x, bool use_b, float *v, bool join,
                  hipStream_t st) {
  psx::ShrinkArgs a{};
  a.b = b;
  a.x.p = (const uint8_t *)x->data;
  a.x.ld = x->row_stride;
  a.x.type = x->type;
  a.w = use_b ? s->b.data : s->a.data;
  a.d = use_b ? s->b.cap : s->a.cap;
  a.use_b = use_b;
  a.splits = psx::adapter_splits(b.tokens, a.d);
  a.rl = s->rl;
  a.max_rank = s->max_rank;
  a.part = (int64_t)b.tokens * s->rl;
  a.v = v;
  OP_HIP(s->ctx, psx::launch_adapter_shrink(a, st));
  if (join && parts_read(b.tokens, a.d) > 1) OP_HIP(s->ctx, psx::launch_adapter_join(a, st));
  return PSX_OK;
}

// n = base^power as little-endian 32-bit words, times `by`^`times`.
std::vector<uint32_t> power_product(uint32_t base, int power, uint32_t by, int times) {
  std::vector<uint32_t> w{1};
  for (int i = 0; i < power + times; ++i) {
    uint64_t carry = 0;
    for (uint32_t &x : w) {
      carry += (uint64_t)x * (i < power ? base : by);
      x = (uint32_t)carry;
      carry >>= 32;
    }
    if (carry) w.push_back((uint32_t)carry);
  }
  return w;
}
bool at_least(const std::vector<uint32_t> &a, const std::vector<uint32_t> &b) {
  if (a.size() != b.size()) return a.size() > b.size();
  for (size_t i = a.size(); i-- > 0;)
    if (a[i] != b[i]) return a[i] > b[i];
  return true;
}

// border[i - 1] = the least n with n^m >= distance^i * exact^(m - i), m = half - exact.
void bias_borders(psx::BiasMap &m, int32_t distance) {
  const int many = m.half - m.exact;
  m.nborder = many - 1;
  for (int i = 1; i < many; ++i) {
    const std::vector<uint32_t> want = power_product((uint32_t)distance, i, (uint32_t)m.exact, many - i);
    int32_t lo = m.exact, hi = distance;
    while (lo < hi) {
      const int32_t mid = lo + (hi - lo) / 2;
      if (at_least(power_product((uint32_t)mid, many, 1, 0), want)) hi = mid;
      else lo = mid + 1;
    }
    m.border[i - 1] = lo;
  }
}

psx_status check_scores(psx_position_bias *b, const psx_scores *s, bool output) {
  psx_ctx *c = b->ctx;
  if (s->type < PSX_ACT_F32 || s->type > PSX_ACT_BF16 || s->reserved0) return op_fail(c, PSX_ERR_INVALID_ARG, "scores: bad type");
  if (s->heads != b->t.cap) return op_fail(c, PSX_ERR_INVALID_ARG, "scores: heads must be the table's row_capacity");
  if (s->batch < 0 || s->q_len < 0 || s->k_len < 0 || s->batch > 65535 || s->heads > 65535 || s->q_len > ((int64_t)1 << 24) ||
      s->k_len > ((int64_t)1 << 24))
    return op_fail(c, PSX_ERR_INVALID_ARG, "scores: batch or heads past 65535, or a length past 2^24");
  if (output && s->batch != 1) return op_fail(c, PSX_ERR_INVALID_ARG, "scores: the bias has no batch");
  // what lies between the first value and the last: 2^46 elements an axis at most, so that the sum of
  // the axes fits 64 bits; an axis of one entry has no stride
  for (const auto &[n, stride] : {std::pair(s->batch, s->batch_stride), std::pair(s->heads, s->head_stride),
                                  std::pair(s->q_len, s->q_stride)})
    if (n > 1 && (stride < 0 || stride > kMaxElements / (n - 1))) return op_fail(c, PSX_ERR_INVALID_ARG, "scores: bad stride");
  if (output) {
    // heads over rows or rows over heads, no two overlapping
    const int64_t rows = s->q_len > 1 ? (s->q_len - 1) * s->q_stride + s->k_len : s->k_len;
    const int64_t cols = s->heads > 1 ? (s->heads - 1) * s->head_stride + s->k_len : s->k_len;
    const bool inner = (s->q_len <= 1 || s->q_stride >= s->k_len) && (s->heads <= 1 || s->head_stride >= rows);
    const bool outer = (s->heads <= 1 || s->head_stride >= s->k_len) && (s->q_len <= 1 || s->q_stride >= cols);
    if (!inner && !outer) return op_fail(c, PSX_ERR_INVALID_ARG, "scores: rows overlap");
  }
  if (s->batch && s->heads && s->q_len && s->k_len && (!s->data || (uintptr_t)s->data % act_size(s->type)))
    return op_fail(c, PSX_ERR_INVALID_ARG, "scores: null or misaligned data");
  return PSX_OK;
}

// The stride of an axis of n entries, as the kernels take it.
int64_t stride_of(int64_t n, int64_t stride) { return n > 1 ? stride : 0; }

psx_status check_begin(psx_position_bias *b, int64_t q_begin) {
  if (q_begin < -((int64_t)1 << 40) || q_begin > ((int64_t)1 << 40))
    return op_fail(b->ctx, PSX_ERR_INVALID_ARG, "q_begin past 2^40");
  return PSX_OK;
}

}  // namespace

extern "C" {

// ---- adapters -------------------------------------------------------------------------------

psx_status psx_adapters_create(psx_ctx *c, int32_t table_a, int32_t table_b, const psx_adapter *adapters, int32_t n,
                               psx_adapters **out) try {
  if (!c || !out) return PSX_ERR_INVALID_ARG;
  *out = nullptr;
  if (!adapters || n <= 0 || n > PSX_MAX_ADAPTERS)
    return op_fail(c, PSX_ERR_INVALID_ARG, "a set holds 1 to " + std::to_string(PSX_MAX_ADAPTERS) + " adapters");
  std::unique_ptr<psx_adapters> s(new psx_adapters);
  OP_TRY(psx::op_dense_view(c, table_a, &s->a));
  OP_TRY(psx::op_dense_view(c, table_b, &s->b));
  std::vector<psx::AdapterDev> ads((size_t)n);
  std::vector<int32_t> ids;
  for (int32_t i = 0; i < n; ++i) {
    const psx_adapter &a = adapters[i];
    const std::string at = "adapter " + std::to_string(i) + ": ";
    if (a.rank < 1 || a.rank > PSX_MAX_ADAPTER_RANK || a.reserved0 || !std::isfinite(a.scale))
      return op_fail(c, PSX_ERR_INVALID_ARG, at + "bad rank or scale");
    const int64_t sa = psx::op_slots(s->a, a.first_row, a.rank), sb = psx::op_slots(s->b, a.first_row, a.rank);
    if (s->a.cap > (int64_t)1 << 24 || s->b.cap > (int64_t)1 << 24)
      return op_fail(c, PSX_ERR_UNSUPPORTED, "rows of more than 2^24 values");
    if (sa < 0 || sb < 0) return op_fail(c, PSX_ERR_ROW_RANGE, at + "rows outside this shard");
    if (s->a.row_stride != s->b.row_stride && a.rank > 1)
      return op_fail(c, PSX_ERR_INVALID_ARG, "the two tables step their rows differently");
    ads[(size_t)i] = {(int32_t)sa, (int32_t)sb, a.rank, s->num_rows, a.scale};
    for (int32_t r = 0; r < a.rank; ++r) ids.push_back((int32_t)(a.first_row + r * s->a.row_stride));
    s->num_rows += a.rank;
    s->max_rank = std::max(s->max_rank, a.rank);
  }
  std::vector<int32_t> sorted = ids;
  std::sort(sorted.begin(), sorted.end());
  if (std::adjacent_find(sorted.begin(), sorted.end()) != sorted.end())
    return op_fail(c, PSX_ERR_INVALID_ARG, "a row belongs to two adapters of the set");
  s->n = n;
  s->rl = (s->max_rank + 15) / 16 * 16;
  psx::OpDevice dev(psx::op_device(c));
  OP_HIP(c, dev.status);
  OP_HIP(c, hipMalloc(&s->d_ads, ads.size() * sizeof(ads[0])));
  OP_HIP(c, hipMalloc(&s->d_row_ids, ids.size() * sizeof(ids[0])));
  OP_HIP(c, hipMemcpyAsync(s->d_ads, ads.data(), ads.size() * sizeof(ads[0]), hipMemcpyHostToDevice, psx::op_stream(c)));
  OP_HIP(c, hipMemcpyAsync(s->d_row_ids, ids.data(), ids.size() * sizeof(ids[0]), hipMemcpyHostToDevice, psx::op_stream(c)));
  OP_HIP(c, hipStreamSynchronize(psx::op_stream(c)));
  *out = s.get();
  psx::op_adopt(c, s.release());
  return PSX_OK;
} catch (const std::exception &) {   // the host ran out of memory
  return PSX_ERR_OOM;
}

psx_status psx_adapters_destroy(psx_adapters *s) {
  if (!s) return PSX_ERR_INVALID_ARG;
  psx::OpDevice dev(psx::op_device(s->ctx));
  psx::op_release(s);
  return PSX_OK;
}

psx_status psx_adapters_info(psx_adapters *s, int32_t *num_rows, const int32_t **row_ids) {
  if (!s) return PSX_ERR_INVALID_ARG;
  if (num_rows) *num_rows = s->num_rows;
  if (row_ids) *row_ids = s->d_row_ids;
  return PSX_OK;
}

psx_status psx_adapters_sizes(psx_adapters *s, int64_t num_tokens, size_t *shrunk_bytes, size_t *work_bytes) try {
  if (!s) return PSX_ERR_INVALID_ARG;
  OP_TRY(check_tokens(s, num_tokens, 0));
  if (shrunk_bytes) *shrunk_bytes = shrunk_size(s, num_tokens, s->a.cap);
  if (work_bytes)
    *work_bytes = shrunk_size(s, num_tokens, s->b.cap) + 2 * aligned((size_t)s->n * sizeof(int2)) +
                  partial_size(s, num_tokens, s->a.cap) + partial_size(s, num_tokens, s->b.cap);
  return PSX_OK;
} catch (const std::exception &) {   // the host ran out of memory
  return PSX_ERR_OOM;
}

psx_status psx_adapters_forward(psx_adapters *s, const psx_requests *requests, const psx_matrix *x, const psx_matrix *base,
                                const psx_matrix *out, void *shrunk, void *hip_stream) try {
  if (!s || !x || !out) return PSX_ERR_INVALID_ARG;
  psx_ctx *c = s->ctx;
  const int64_t T = x->rows;
  OP_TRY(check_requests(c, requests));
  OP_TRY(check_tokens(s, T, requests->num_requests));
  OP_TRY(check_matrix(c, x, T, s->a.cap, false, "x"));
  OP_TRY(check_out(c, base, out, T, s->b.cap));
  if (x->type != out->type) return op_fail(c, PSX_ERR_INVALID_ARG, "x and out differ in type");
  OP_TRY(check_rows_apart(c, x, "x"));
  const size_t shrunk_bytes = shrunk_size(s, T, s->a.cap);
  if (overlap(x->data, span(x), out->data, span(out))) return op_fail(c, PSX_ERR_INVALID_ARG, "out overlaps x");
  if (T && (!shrunk || (uintptr_t)shrunk % 16)) return op_fail(c, PSX_ERR_INVALID_ARG, "shrunk: null or misaligned");
  if (overlap(shrunk, shrunk_bytes, out->data, span(out)) || overlap(shrunk, shrunk_bytes, x->data, span(x)) ||
      (base && overlap(shrunk, shrunk_bytes, base->data, span(base))))
    return op_fail(c, PSX_ERR_INVALID_ARG, "shrunk overlaps a matrix");
  psx::OpDevice dev(psx::op_device(c));
  OP_HIP(c, dev.status);
  hipStream_t st = (hipStream_t)hip_stream;
  OP_TRY(psx::op_settle(c, st));
  if (T == 0 || requests->num_requests == 0) return PSX_OK;
  const psx::BatchView b = batch_view(s, requests, T);
  OP_TRY(psx::op_reads(c, st));
  OP_TRY(shrink(s, b, x, false, (float *)shrunk, false, st));
  return expand(s, b, (float *)shrunk, s->a.cap, true, base, out, st);
} catch (const std::exception &) {   // the host ran out of memory
  return PSX_ERR_OOM;
}

psx_status psx_adapters_backward(psx_adapters *s, const psx_requests *requests, const psx_matrix *x,
                                 const void *x_checkpoint, const psx_matrix *dy, const void *shrunk,
                                 const psx_matrix *base, const psx_matrix *out, float *grad_a, float *grad_b, float gain,
                                 void *work, void *hip_stream) try {
  if (!s || !dy || !grad_a || !grad_b) return PSX_ERR_INVALID_ARG;
  psx_ctx *c = s->ctx;
  const int64_t T = dy->rows;
  OP_TRY(check_requests(c, requests));
  OP_TRY(check_tokens(s, T, requests->num_requests));
  OP_TRY(check_matrix(c, dy, T, s->b.cap, false, "dy"));
  if (!x == !x_checkpoint && T) return op_fail(c, PSX_ERR_INVALID_ARG, "exactly one of x and x_checkpoint");
  if (x) {
    OP_TRY(check_matrix(c, x, T, s->a.cap, false, "x"));
    if (x->type != dy->type) return op_fail(c, PSX_ERR_INVALID_ARG, "x and dy differ in type");
  }
  OP_TRY(check_rows_apart(c, x, "x"));
  OP_TRY(check_rows_apart(c, dy, "dy"));
  if (base && !out) return op_fail(c, PSX_ERR_INVALID_ARG, "base without out");
  size_t ck = 0;
  if (x_checkpoint) {
    OP_TRY(psx_checkpoint_bytes(T, s->a.cap, &ck));
    if ((uintptr_t)x_checkpoint % 16) return op_fail(c, PSX_ERR_INVALID_ARG, "x_checkpoint: misaligned");
  }
  const size_t shrunk_bytes = shrunk_size(s, T, s->a.cap);
  size_t work_bytes = 0;
  OP_TRY(psx_adapters_sizes(s, T, nullptr, &work_bytes));
  const size_t ga = (size_t)s->num_rows * (size_t)s->a.cap * 4, gb = (size_t)s->num_rows * (size_t)s->b.cap * 4;
  if (((uintptr_t)grad_a | (uintptr_t)grad_b) & 3) return op_fail(c, PSX_ERR_INVALID_ARG, "gradients must be 4-byte aligned");
  if (T && (!shrunk || (uintptr_t)shrunk % 16 || !work || (uintptr_t)work % 16))
    return op_fail(c, PSX_ERR_INVALID_ARG, "shrunk or work: null or misaligned");
  struct Range {
    const void *p;
    size_t n;
  };
  std::vector<Range> writes{{grad_a, ga}, {grad_b, gb}, {work, T ? work_bytes : 0}};
  std::vector<Range> reads{{dy->data, span(dy)}, {shrunk, shrunk_bytes}, {x_checkpoint, ck}};
  if (x) reads.push_back({x->data, span(x)});
  if (out) {
    OP_TRY(check_out(c, base, out, T, s->a.cap));
    if (out->type != dy->type) return op_fail(c, PSX_ERR_INVALID_ARG, "dy and out differ in type");
    writes.push_back({out->data, span(out)});
  }
  for (size_t i = 0; i < writes.size(); ++i) {
    for (size_t j = 0; j < i; ++j)
      if (overlap(writes[i].p, writes[i].n, writes[j].p, writes[j].n))
        return op_fail(c, PSX_ERR_INVALID_ARG, "outputs or work overlap");
    for (const Range &r : reads)
      if (overlap(writes[i].p, writes[i].n, r.p, r.n)) return op_fail(c, PSX_ERR_INVALID_ARG, "an output or work overlaps an input");
    if (base && i < 3 && overlap(writes[i].p, writes[i].n, base->data, span(base)))
      return op_fail(c, PSX_ERR_INVALID_ARG, "a gradient or work overlaps base");
  }
  psx::OpDevice dev(psx::op_device(c));
  OP_HIP(c, dev.status);
  hipStream_t st = (hipStream_t)hip_stream;
  OP_TRY(psx::op_settle(c, st));
  OP_TRY(psx::op_reads(c, st));
  const bool any = T > 0 && requests->num_requests > 0;
  const psx::BatchView b = batch_view(s, requests, T);
  uint8_t *w = (uint8_t *)work;
  float *u = (float *)w;
  w += shrunk_size(s, T, s->b.cap);
  if (any) {
    OP_TRY(shrink(s, b, dy, true, u, !out, st));
    if (out) OP_TRY(expand(s, b, u, s->b.cap, false, base, out, st));
  }
  psx::GradArgs grads[2] = {};
  for (int k = 0; k < 2; ++k) {   // grad_a from u and x, grad_b from x A^T and dy
    psx::GradArgs &g = grads[k];
    g.b = b;
    g.v = k ? whole_v(s, (const float *)shrunk, T, s->a.cap) : out ? whole_v(s, u, T, s->b.cap) : u;
    g.rl = s->rl;
    g.d = k ? s->b.cap : s->a.cap;
    if (k || x) {
      const psx_matrix *m = k ? dy : x;
      g.x.p = (const uint8_t *)m->data;
      g.x.ld = m->row_stride;
      g.x.type = m->type;
    } else {
      const int64_t groups = (s->a.cap + psx::kCkGroup - 1) / psx::kCkGroup;
      g.x.p = (const uint8_t *)x_checkpoint;
      g.x.ld = groups * psx::kCkGroup;
      g.x.exps = g.x.p + T * g.x.ld;
      g.x.type = psx::kAct8;
    }
    g.max_rank = s->max_rank;
    g.chunk = psx::adapter_grad_chunk(T, g.d, s->max_rank);
    g.slots = (int32_t)grad_slots(s, T, g.d);
    g.gain = gain;
    g.items = (int2 *)w;
    w += aligned((size_t)s->n * sizeof(int2));
    g.partial = (float *)w;
    w += partial_size(s, T, g.d);
    g.grad = k ? grad_b : grad_a;
  }
  const bool whole = any && T <= grads[0].chunk && T <= grads[1].chunk;
  for (psx::GradArgs &g : grads) g.whole = whole;
  if (any) OP_HIP(c, psx::launch_adapter_grad(grads[0], grads[1], st));
  if (!whole) OP_HIP(c, psx::launch_adapter_grad_sum(grads[0], grads[1], st));
  return PSX_OK;
} catch (const std::exception &) {   // the host ran out of memory
  return PSX_ERR_OOM;
}

// ---- checkpoints ------------------------------------------------------------------------------

psx_status psx_checkpoint_bytes(int64_t rows, int64_t cols, size_t *bytes) {
  if (rows < 0 || cols < 0 || !bytes || (rows && cols > kMaxElements / rows)) return PSX_ERR_INVALID_ARG;
  *bytes = (size_t)rows * (size_t)((cols + psx::kCkGroup - 1) / psx::kCkGroup) * (psx::kCkGroup + 1);
  return PSX_OK;
}

static psx_status checkpoint_args(psx_ctx *c, const psx_matrix *m, const void *checkpoint, bool output, psx::CkArgs *a) {
  size_t bytes = 0;
  if (psx_checkpoint_bytes(m->rows, m->cols, &bytes) != PSX_OK) return op_fail(c, PSX_ERR_INVALID_ARG, "bad shape");
  if (m->cols > (int64_t)1 << 30) return op_fail(c, PSX_ERR_UNSUPPORTED, "rows of more than 2^30 values");
  OP_TRY(check_matrix(c, m, m->rows, m->cols, output, output ? "out" : "x"));
  if (bytes && (!checkpoint || (uintptr_t)checkpoint % 16))
    return op_fail(c, PSX_ERR_INVALID_ARG, "checkpoint: null or misaligned");
  if (overlap(checkpoint, bytes, m->data, span(m))) return op_fail(c, PSX_ERR_INVALID_ARG, "the checkpoint overlaps the matrix");
  a->p = (uint8_t *)m->data;
  a->ld = m->row_stride;
  a->type = m->type;
  a->rows = m->rows;
  a->cols = m->cols;
  a->groups = (m->cols + psx::kCkGroup - 1) / psx::kCkGroup;
  a->codes = (uint8_t *)checkpoint;
  a->exps = a->codes + m->rows * a->groups * psx::kCkGroup;
  return PSX_OK;
}

psx_status psx_checkpoint_store(psx_ctx *c, const psx_matrix *x, void *checkpoint, void *hip_stream) try {
  if (!c || !x) return PSX_ERR_INVALID_ARG;
  psx::CkArgs a{};
  OP_TRY(checkpoint_args(c, x, checkpoint, false, &a));
  psx::OpDevice dev(psx::op_device(c));
  OP_HIP(c, dev.status);
  OP_HIP(c, psx::launch_checkpoint_store(a, (hipStream_t)hip_stream));
  return PSX_OK;
} catch (const std::exception &) {   // the host ran out of memory
  return PSX_ERR_OOM;
}

psx_status psx_checkpoint_load(psx_ctx *c, const void *checkpoint, const psx_matrix *out, void *hip_stream) try {
  if (!c || !out) return PSX_ERR_INVALID_ARG;
  psx::CkArgs a{};
  OP_TRY(checkpoint_args(c, out, checkpoint, true, &a));
  psx::OpDevice dev(psx::op_device(c));
  OP_HIP(c, dev.status);
  OP_HIP(c, psx::launch_checkpoint_load(a, (hipStream_t)hip_stream));
  return PSX_OK;
} catch (const std::exception &) {   // the host ran out of memory
  return PSX_ERR_OOM;
}

// ---- position bias ------------------------------------------------------------------------------

psx_status psx_position_bias_create(psx_ctx *c, int32_t table_id, int32_t first_row, int32_t num_buckets,
                                    int32_t max_distance, int32_t bidirectional, psx_position_bias **out) try {
  if (!c || !out) return PSX_ERR_INVALID_ARG;
  *out = nullptr;
  if (bidirectional != 0 && bidirectional != 1) return op_fail(c, PSX_ERR_INVALID_ARG, "bidirectional is 0 or 1");
  const int32_t half = bidirectional ? num_buckets / 2 : num_buckets;
  if (num_buckets > psx::kMaxBuckets || half < 2 || (bidirectional && num_buckets % 2) || max_distance <= half / 2 ||
      max_distance > 1 << 20)
    return op_fail(c, PSX_ERR_INVALID_ARG, "bad num_buckets or max_distance");
  std::unique_ptr<psx_position_bias> b(new psx_position_bias);
  OP_TRY(psx::op_dense_view(c, table_id, &b->t));
  b->slot = psx::op_slots(b->t, first_row, num_buckets);
  if (b->slot < 0) return op_fail(c, PSX_ERR_ROW_RANGE, "rows outside this shard");
  b->map.buckets = num_buckets;
  b->map.both = bidirectional;
  b->map.half = half;
  b->map.exact = half / 2;
  bias_borders(b->map, max_distance);
  *out = b.get();
  psx::op_adopt(c, b.release());
  return PSX_OK;
} catch (const std::exception &) {   // the host ran out of memory
  return PSX_ERR_OOM;
}

psx_status psx_position_bias_destroy(psx_position_bias *b) {
  if (!b) return PSX_ERR_INVALID_ARG;
  psx::op_release(b);
  return PSX_OK;
}

psx_status psx_position_bias_forward(psx_position_bias *b, const psx_scores *out, int64_t q_begin, void *hip_stream) try {
  if (!b || !out) return PSX_ERR_INVALID_ARG;
  psx_ctx *c = b->ctx;
  OP_TRY(check_scores(b, out, true));
  OP_TRY(check_begin(b, q_begin));
  psx::BiasArgs a{};
  a.map = b->map;
  a.w = b->t.data + b->slot * b->t.cap;
  a.heads = (int32_t)out->heads;
  a.q = out->q_len;
  a.k = out->k_len;
  a.begin = q_begin;
  a.out = (uint8_t *)out->data;
  a.head_ld = stride_of(out->heads, out->head_stride);
  a.q_ld = stride_of(out->q_len, out->q_stride);
  a.type = out->type;
  if (!psx::grid_fits(psx::bias_blocks(a), 256)) return op_fail(c, PSX_ERR_UNSUPPORTED, "too many scores for one call");
  psx::OpDevice dev(psx::op_device(c));
  OP_HIP(c, dev.status);
  hipStream_t st = (hipStream_t)hip_stream;
  OP_TRY(psx::op_settle(c, st));
  OP_TRY(psx::op_reads(c, st));
  OP_HIP(c, psx::launch_bias(a, st));
  return PSX_OK;
} catch (const std::exception &) {   // the host ran out of memory
  return PSX_ERR_OOM;
}

psx_status psx_position_bias_work(psx_position_bias *b, int64_t batch, int64_t q_len, int64_t k_len, size_t *bytes) try {
  if (!b || !bytes) return PSX_ERR_INVALID_ARG;
  psx_scores s{};
  s.heads = b->t.cap;
  s.batch = batch;
  s.q_len = q_len;
  s.k_len = k_len;
  s.data = (void *)16;
  OP_TRY(check_scores(b, &s, false));
  size_t blocks = 0;   // of either element size: the caller names none
  for (int32_t type : {PSX_ACT_F32, PSX_ACT_F16})
    blocks = std::max(blocks, (size_t)psx::bias_grad_tiles(batch, b->t.cap, q_len, k_len, type).blocks);
  if (!psx::grid_fits((int64_t)blocks, 512)) return op_fail(b->ctx, PSX_ERR_UNSUPPORTED, "too many scores for one call");
  *bytes = (size_t)b->t.cap * (size_t)batch * blocks * (size_t)b->map.buckets * sizeof(float);
  return PSX_OK;
} catch (const std::exception &) {   // the host ran out of memory
  return PSX_ERR_OOM;
}

psx_status psx_position_bias_backward(psx_position_bias *b, const psx_scores *d, int64_t q_begin, float gain, float *grad,
                                      void *work, void *hip_stream) try {
  if (!b || !d || !grad) return PSX_ERR_INVALID_ARG;
  psx_ctx *c = b->ctx;
  OP_TRY(check_scores(b, d, false));
  OP_TRY(check_begin(b, q_begin));
  size_t bytes = 0;
  OP_TRY(psx_position_bias_work(b, d->batch, d->q_len, d->k_len, &bytes));
  if ((uintptr_t)grad & 3) return op_fail(c, PSX_ERR_INVALID_ARG, "grad must be 4-byte aligned");
  if (bytes && (!work || (uintptr_t)work % 16)) return op_fail(c, PSX_ERR_INVALID_ARG, "work: null or misaligned");
  const size_t gb = (size_t)b->map.buckets * (size_t)b->t.cap * 4;
  const size_t ds = d->batch && d->heads && d->q_len && d->k_len
                        ? (size_t)((d->batch - 1) * stride_of(d->batch, d->batch_stride) +
                                   (d->heads - 1) * stride_of(d->heads, d->head_stride) +
                                   (d->q_len - 1) * stride_of(d->q_len, d->q_stride) + d->k_len) * act_size(d->type)
                        : 0;
  if (overlap(grad, gb, work, bytes) || overlap(grad, gb, d->data, ds) || overlap(work, bytes, d->data, ds))
    return op_fail(c, PSX_ERR_INVALID_ARG, "grad, work and d overlap");
  psx::OpDevice dev(psx::op_device(c));
  OP_HIP(c, dev.status);
  psx::BiasGradArgs a{};
  a.map = b->map;
  a.d = (const uint8_t *)d->data;
  a.batch_ld = stride_of(d->batch, d->batch_stride);
  a.head_ld = stride_of(d->heads, d->head_stride);
  a.q_ld = stride_of(d->q_len, d->q_stride);
  a.batch = (int32_t)d->batch;
  a.heads = (int32_t)d->heads;
  a.q = d->q_len;
  a.k = d->k_len;
  a.begin = q_begin;
  a.type = d->type;
  a.gain = gain;
  a.tiles = psx::bias_grad_tiles(d->batch, d->heads, d->q_len, d->k_len, d->type);
  a.partial = (float *)work;
  a.grad = grad;
  OP_HIP(c, psx::launch_bias_grad(a, (hipStream_t)hip_stream));
  return PSX_OK;
} catch (const std::exception &) {   // the host ran out of memory
  return PSX_ERR_OOM;
}

}  // extern "C"
