// Host API of the query / key norm + rotary kernels (qk_norm.hip), shared with their bindings.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "rowvec.h"
#include "transformer_api.h"

namespace dca {
// One of q, k (or a gradient of theirs): [B, S, heads, D] with any strides (elements), D contiguous.
struct HeadView {
  void* p = nullptr;
  int64_t sb = 0, ss = 0, sh = 0;
};
struct QkShape {
  int64_t B = 0, S = 0;
  int heads[2] = {0, 0};  // of q, of k
  int D = 0;
  int rot = 0;            // rotated features (even; 0: norm only)
  int64_t table_rows = 0; // of cos / sin
  Index pos;              // absent: token s sits at s
  int64_t pos_sb = 0;     // of the position array [B, S] (0: one row for all sequences)
  float eps = 0.f;
};
// y = R(pos) (w x / rms(x)) for q and k in one launch; w may be absent.
void qk_norm_rope_fwd(TDtype dt, int vec_bytes, const QkShape& s, const HeadView x[2], const HeadView y[2],
                      const float* const w[2], const float* cosT, const float* sinT, hipStream_t st);
// floats of `partial` the backward needs
int64_t qk_norm_rope_partial_floats(const QkShape& s);
// dx from dy and x (dx may be dy); dw[i] (D values each, absent: not wanted) by partial rows of
// workgroups and a fixed-order sum.
void qk_norm_rope_bwd(TDtype dt, int vec_bytes, const QkShape& s, const HeadView dy[2], const HeadView x[2],
                      const HeadView dx[2], const float* const w[2], const float* cosT, const float* sinT,
                      float* partial, const ColumnOut* const dw[2], hipStream_t st);
}  // namespace dca
