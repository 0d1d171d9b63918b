// Host API of the embedding kernels (embedding.hip), shared with their PyTorch bindings.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "rowvec.h"
#include "transformer_api.h"

namespace dca {
// `aligned`: all addresses and row lengths are multiples of 16 bytes.
// Token ids -> table rows: row = id - start; `shard`: ids outside [start, start + rows) belong to
// another shard (zero rows), otherwise they are mistakes (NaN rows).
struct EmbedIds {
  Index ids;
  int64_t n = 0;
  int64_t start = 0;
  int64_t rows = 0;
  bool shard = false;
};
// Learned positions: `rows` = 0 for none; without `ids` token t of a sequence of S sits at t % S.
struct EmbedPos {
  const void* table = nullptr;
  int64_t stride = 0;
  int64_t rows = 0;
  Index ids;
  int64_t S = 1;
};
void embed_fwd(TDtype dt, bool aligned, const EmbedIds& ids, const void* table, int64_t stride,
               const EmbedPos& pos, float scale, void* out, int E, hipStream_t st);
// bytes of workspace embed_grad needs for n ids and a table of `rows` rows of E
int64_t embed_grad_workspace(int64_t n, int64_t rows, int E);
// out[row] = scale * sum of dy's rows with that id, zero for rows without one; `accumulate`: added to
// what is there, rows without an id untouched. dy [n][E], out [rows][E] (16-byte aligned unless
// accumulating), both contiguous.
void embed_grad(TDtype dt, bool aligned, const EmbedIds& ids, const void* dy, void* out, int E,
                float scale, bool accumulate, void* workspace, hipStream_t st);
// out[j] (+)= sum_b dy[b][j] for dy [B][N]
void batch_sum(TDtype dt, bool aligned, const void* dy, void* out, int64_t B, int64_t N,
               bool accumulate, hipStream_t st);
}  // namespace dca
