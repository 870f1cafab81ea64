// Launchers of the packed-attention, rotation and distillation kernels on plain pointers. They include no PyTorch header
// (their nodes in sequence_ops.cpp check arguments, allocate, pick device and stream) and return the launch's status.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace mia {

enum SequenceType : int { kSeqBf16 = 0, kSeqF16 = 1, kSeqF32 = 2, kSeqF64 = 3 };

// Rows of heads: element (t, h, c) of a (T, H, D) tensor lies at t * row + h * head + c.
struct HeadRows {
  int64_t row, head;
};

struct PackedProblem {
  const void *q, *k, *v;
  HeadRows qs, ks, vs;
  const int2* q_bounds;  // (queries): the keys [x, y) that a query sees; both ends never fall from one row to the next
  const int2* k_bounds;  // (keys): the queries [x, y) that see a key; likewise
  int Tq, Tk;            // rows of the sequences; rows behind them are not read
  int Hq, Hk, group, D;
  int lse_stride;        // columns of lse and delta: rows rounded up to 128
  float scale;
  SequenceType type;
  void* o_low;  // like o, or null: what rounding took from o, written forward and added to o again for delta
};

// o (Tq.., Hq, D) contiguous; lse (Hq, lse_stride) fp32
cudaError_t packed_fwd_rows(const PackedProblem& P, void* o, float* lse, cudaStream_t stream);
// Few queries over many keys: pieces of a sequence's keys with all of its queries.
struct PackedFew {
  const int4* items;   // (count): first query, queries, keys [z, w)
  const int2* pieces;  // (sequences): first item, items
  int count, sequences;
  int rows;        // most queries of a sequence times the heads that share a key head
  float* partial;  // (count, Hk, rows, D + 2) fp32, or null where every sequence is one item
};
cudaError_t packed_fwd_few(const PackedProblem& P, const PackedFew& few, void* o, float* lse, cudaStream_t stream);
// dout as strided rows; delta like lse (scratch); dq (.., Hq, D), dk and dv (.., Hk, D) contiguous
cudaError_t packed_bwd_rows(const PackedProblem& P, const void* o, const void* dout, HeadRows ds, const float* lse,
                            float* delta, void* dq, void* dk, void* dv, cudaStream_t stream);

// The tensor-core kernels, where packed_tc_ok: same arguments; channels (2, Hq, lse_stride, 8) of the inputs' type is
// scratch, and for fp16 norms, (Hq, lse_stride) fp32 and behind them (Hq, lse_stride / 128).
bool packed_tc_ok(const PackedProblem& P);
cudaError_t packed_fwd_tc(const PackedProblem& P, void* o, float* lse, int* err, cudaStream_t stream);
cudaError_t packed_bwd_tc(const PackedProblem& P, const void* o, const void* dout, HeadRows ds, const float* lse,
                          float* delta, void* channels, float* norms, void* dq, void* dk, void* dv, int* err,
                          cudaStream_t stream);

struct TokenRows {
  int64_t b, t, h;  // element strides of (B, T, H, D)
};

struct RotaryParams {
  const void *q, *k;    // (B, T, H, D)
  const void *xq, *xk;  // the forward pass's inputs, for the gradient of the frequencies
  void *yq, *yk;
  TokenRows qs, ks, xqs, xks, yqs, yks;
  const void* pos;
  int pos_type;   // 0: int64, 1: int32, 2: fp32, 3: fp64
  int64_t pos_b;  // 0 where all rows of the batch share one row of positions
  const void* freq;  // (axes, P), or null: then pos holds the angles (.., P) in fp32
  int freq64;
  int axes, P, D, T, Hq, Hk;
  int64_t tokens;  // B * T
  int heads;       // of a block
  float amplitude;
  int inverse;
  float* partial;  // (blocks, axes, P)
};

struct RotaryPlan {
  bool vec;
  int heads;              // of a block
  unsigned grid, chunks;  // blocks over tokens, over heads
  size_t smem;
};
RotaryPlan rotary_plan(const RotaryParams& p, bool aligned, bool interleaved, bool learn);
cudaError_t rotary_launch(RotaryParams p, const RotaryPlan& plan, SequenceType type, bool interleaved, float* dfreq,
                          cudaStream_t stream);

constexpr int kMaxTop = 256;     // top_logits
constexpr int kMaxGiven = 1024;  // distillation

cudaError_t top_logits_rows(const void* x, int64_t stride, int R, int V, int k, double tau, void* values,
                            int64_t* indices, float* lse, SequenceType type, cudaStream_t stream);

struct DistillParams {
  const void* s;
  int64_t s_row;
  const void* values;  // (R, K)
  const void* indices;
  const void* lse;      // (R), or null
  const void* weights;  // (R), or null
  SequenceType type, value_type;
  bool index64, lse64, weights64;  // int64 indices; fp64 instead of fp32
  int R, V, K;
  double tau, teacher_tau, norm;
  double* stats;  // (R, 8)
};
cudaError_t distill_fwd(const DistillParams& p, double* row_loss, float* loss, cudaStream_t stream);
cudaError_t distill_bwd(const DistillParams& p, const float* grad, void* ds, cudaStream_t stream);

}  // namespace mia
