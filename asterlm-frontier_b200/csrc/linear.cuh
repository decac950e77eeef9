// What the two forms of linear attention share: csrc/linear_attention.cu (token by token) and
// csrc/linear_chunk.cu (chunks on the tensor cores).
#pragma once

#include "asterq_internal.h"
#include "common.cuh"

namespace asterq {
namespace lin {

struct Args {
  const void* q;
  const void* k;
  const void* v;
  const float* log_decay;
  float* state;
  const int* slots;
  const int* lengths;      // NULL: every sequence continues from its state
  const int* row_offsets;  // NULL: row s is sequence s's one token
  void* out;
  int* status;
  long long q_row, q_head, k_row, k_head, v_row, v_head, decay_row;  // strides in elements
  long long n_rows;
  int n_seqs, n_heads, n_slots;
  float scale;
};

// csrc/linear_chunk.cu: bf16 rows with row_offsets
int64_t chunk_workspace_bytes(int dk, int dv, int workers);
// ASTERQ_OK, an error, or ASTERQ_ERR_UNSUPPORTED when no tensor map describes the strides
int chunk_launch(const Args& a, int dk, int dv, int workers, int device, void* workspace, cudaStream_t s);

}  // namespace lin
}  // namespace asterq
