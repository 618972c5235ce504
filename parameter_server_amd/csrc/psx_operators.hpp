// psx_operators.hpp — definitions shared by the operators on parameter rows: their kernels
// (psx_adapter.hip, psx_checkpoint.hip, psx_bias.hip), their entry points
// (psx_operators.cpp), and the part of the context they see (psx_runtime.cpp).
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>
#include <string>

#include "../../include/psx.h"

namespace psx {

// ---- what psx_runtime.cpp gives to the entry points ------------------------------------
// A dense f32 table as it lies in HBM: rows[max_rows][cap], slot = (row - row_offset) / row_stride.
struct DenseView {
  float *data;
  int64_t cap;
  int64_t row_offset, row_stride, max_rows;
};
psx_status op_fail(psx_ctx *c, psx_status s, const std::string &msg);
psx_status op_hip_fail(psx_ctx *c, hipError_t e, const char *what);
int op_device(psx_ctx *c);
hipStream_t op_stream(psx_ctx *c);   // the context's stream
// The dense f32 table `table_id`, or the error of a table that is not one.
psx_status op_dense_view(psx_ctx *c, int32_t table_id, DenseView *out);
// First slot of num_rows rows from first_row on (row ids step by the table's row_stride), or -1.
int64_t op_slots(const DenseView &t, int64_t first_row, int64_t num_rows);
// Before an operator reads rows on `st`: the calls in flight are settled, as before any row read.
psx_status op_settle(psx_ctx *c, hipStream_t st);
// After it: later writers of the tables wait for `st`, and psx_sync reports op_status.
psx_status op_reads(psx_ctx *c, hipStream_t st);
uint32_t *op_status(psx_ctx *c);      // device word of kOp* bits
// A handle that lives in a context: freed by its destroy call or with the context.
struct OpHandle {
  psx_ctx *ctx = nullptr;
  virtual ~OpHandle() {}
};
void op_adopt(psx_ctx *c, OpHandle *h);
void op_release(OpHandle *h);   // deletes h
// The caller's device, restored when the entry point returns.
struct OpDevice {
  int before = -1;
  hipError_t status;
  explicit OpDevice(int device) {
    if (hipGetDevice(&before) != hipSuccess) before = -1;
    status = before == device ? hipSuccess : hipSetDevice(device);
    if (before == device) before = -1;
  }
  ~OpDevice() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

// A grid axis takes fewer than 2^32 threads.
inline bool grid_fits(int64_t blocks, int64_t threads) { return blocks <= (((int64_t)1 << 32) - 1) / threads; }

enum : uint32_t {
  kOpRequests = 1u << 0,   // request_begin descends or leaves [0, num_tokens]
  kOpAdapter = 1u << 1,    // request_adapter outside [-1, adapters of the set)
};

// ---- adapters (psx_adapter.hip) ----------------------------------------------------------
constexpr int kAct8 = 3;         // an activation type beside psx_act: an 8-bit checkpoint
constexpr int kCkGroup = 32;     // values that share an exponent

struct AdapterDev {
  int32_t slot_a, slot_b;   // first slots in the two tables
  int32_t rank;
  int32_t out_row;          // first row of its gradients
  float scale;
};

// An activation matrix: rows of `ld` elements, or a checkpoint (exps set: codes[rows][ld], ld a
// multiple of 32, and an exponent a group).
struct ActView {
  const uint8_t *p;
  const uint8_t *exps;
  int64_t ld;
  int32_t type;             // psx_act or kAct8
};

struct BatchView {
  const int32_t *begin;     // [requests + 1]
  const int32_t *which;     // [requests]
  const AdapterDev *ads;
  int32_t requests, adapters, tokens;
  uint32_t *status;
};

// v[s][t][r] = sum over the s-th part of k of x[t][k] W[slot + r][k]
struct ShrinkArgs {
  BatchView b;
  ActView x;
  const float *w;
  int64_t d;
  int32_t use_b;            // rows of table B
  int32_t splits, rl;       // parts of k; row length of v
  int32_t max_rank;
  int64_t part;             // elements between two parts
  float *v;
};

// out[t][j] = base[t][j] + scale * sum_r v[t][r] W[slot + r][j]
struct ExpandArgs {
  BatchView b;
  const float *v;
  float *sum;               // not null: the sum of v's parts is written here
  int32_t splits, rl;
  int64_t part;
  const float *w;
  int64_t d;
  int32_t use_b;
  int32_t max_rank, tile;
  const uint8_t *base;      // null: zero
  uint8_t *out;
  int64_t base_ld, out_ld;
  int32_t type;             // psx_act
};

// grad[out_row + r][j] = gain * scale * sum_t v[t][r] x[t][j]
struct GradArgs {
  BatchView b;
  const float *v;           // one part
  int32_t rl;
  ActView x;
  int64_t d;
  int32_t max_rank;
  int32_t chunk;            // tokens of one item
  int32_t whole;            // item i is all of adapter i
  int32_t slots;            // partial results that fit `partial`
  float gain;
  float *partial;           // [slots][max_rank][d]
  int2 *items;              // [adapters] first slot, items
  float *grad;              // [rows][d]
};

constexpr int kFewTokens = 2048;   // up to here expand adds the parts of x's width
constexpr int kMostParts = 4;
int adapter_splits(int64_t tokens, int64_t d);
bool adapter_joins(int64_t tokens, int64_t d);   // v's parts are added into the first by shrink
int adapter_expand_tile(int64_t tokens, int max_rank, int parts);
int adapter_grad_chunk(int64_t tokens, int64_t d, int max_rank);
int64_t adapter_grad_most_chunks(int64_t tokens, int64_t d, int max_rank);
hipError_t launch_adapter_shrink(const ShrinkArgs &a, hipStream_t st);
hipError_t launch_adapter_join(const ShrinkArgs &a, hipStream_t st);
hipError_t launch_adapter_expand(const ExpandArgs &a, hipStream_t st);
hipError_t launch_adapter_grad(const GradArgs &a, const GradArgs &b, hipStream_t st);
hipError_t launch_adapter_grad_sum(const GradArgs &a, const GradArgs &b, hipStream_t st);

// ---- checkpoints (psx_checkpoint.hip) -----------------------------------------------------
struct CkArgs {
  uint8_t *p;               // the activation (read by store, written by load)
  int64_t ld;
  int32_t type;             // psx_act
  int64_t rows, cols, groups;
  uint8_t *codes, *exps;
};
hipError_t launch_checkpoint_store(const CkArgs &a, hipStream_t st);
hipError_t launch_checkpoint_load(const CkArgs &a, hipStream_t st);

// ---- position bias (psx_bias.hip) -----------------------------------------------------------
constexpr int kMaxBuckets = 256;
struct BiasMap {
  int32_t buckets, half, exact, both;
  int32_t nborder;
  int32_t border[kMaxBuckets];   // least distances of the buckets exact + 1, exact + 2, ...
};
// Blocks of `rows` queries and a window of `width` distances, a thread a vector of them.
struct BiasTiles {
  int32_t rows, width, windows, threads, groups;
  int64_t blocks;
};
struct BiasArgs {
  BiasMap map;
  int32_t rows, keys;        // a block's queries and keys
  const float *w;            // [buckets][heads]
  int32_t heads;
  int64_t q, k, begin;
  uint8_t *out;
  int64_t head_ld, q_ld;
  int32_t type;
};
struct BiasGradArgs {
  BiasMap map;
  const uint8_t *d;
  int64_t batch_ld, head_ld, q_ld;
  int32_t batch, heads;
  int64_t q, k, begin;
  int32_t type;
  float gain;
  BiasTiles tiles;
  float *partial;            // [heads][batch * tiles.blocks][buckets]
  float *grad;               // [buckets][heads]
};
BiasTiles bias_grad_tiles(int64_t batch, int64_t heads, int64_t q, int64_t k, int32_t type);
int64_t bias_blocks(BiasArgs &a);   // of one head; sets rows and keys
hipError_t launch_bias(const BiasArgs &a, hipStream_t st);
hipError_t launch_bias_grad(const BiasGradArgs &a, hipStream_t st);

}  // namespace psx
