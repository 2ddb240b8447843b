// RMS norm of query / key heads + rotary position embedding (kernels/qk_norm_rope.hip) and counter-based
// dropout (kernels/counter_dropout.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace bh {

// one operand of [s, b, heads, hn]; element (t, b, h, d) at p + t * st + b * sb + h * sh + d
struct HeadView {
  void* p = nullptr;
  int64_t st = 0, sb = 0, sh = 0;
};

struct QkRopeArgs {
  HeadView x[2];   // query, key
  HeadView y[2];   // forward: results; backward: gradients of the inputs
  HeadView dy[2];  // backward: gradients of the results
  int heads[2] = {0, 0};
  int s = 0, b = 0, hn = 0;
  const void* w[2] = {nullptr, nullptr};  // norm weights [hn] (both or none)
  int w_dt = 0;                           // their dtype code
  const float* cos = nullptr;             // [n_pos, rot / 2] (both or none)
  const float* sin = nullptr;
  int rot = 0;                            // rotated leading values of a head (0: no rotation)
  int64_t n_pos = 0;
  const void* pos = nullptr;              // null: position = offset + t
  int pos_i64 = 0;
  int64_t pos_st = 0, pos_sb = 0;         // strides of pos in elements
  int64_t offset = 0;
  float eps = 1e-6f;
  bool interleaved = false;
  bool vec = false;  // 4-element chunks are aligned and rot % 8 == 0: vector loads
};

void qk_rope_forward(int dt, const QkRopeArgs& a, hipStream_t st);
// rows of partial weight-gradient sums (floats: rows * 2 * hn) that the backward needs; 0 without weights
int64_t qk_rope_partial_rows(const QkRopeArgs& a);
// dwq / dwk: [hn] of the weights' dtype
void qk_rope_backward(int dt, const QkRopeArgs& a, float* partials, void* dwq, void* dwk, hipStream_t st);

// y = Philox4x32-7(counter i / 4, key seed)[i % 4] < thresh ? x * scale : 0
void counter_dropout(int dt, const void* x, void* y, int64_t n, uint32_t thresh, float scale, uint64_t seed,
                     const int64_t* seed_dev, hipStream_t st);

}  // namespace bh
