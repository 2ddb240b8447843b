// Grouped-query attention (kernels/grouped_attn.hip): fp16 / bf16, head sizes 8 .. 128 in steps of 8, np query
// heads over ng key / value heads (head j reads key head j / (np / ng)), any lengths. Masks: causal with the
// last query at the last key (query i sees keys <= i + sk - sq), a sliding window of `window` keys ending
// there, key lengths per sequence. A query that sees no key gives zeros and takes no gradient.
// Tensors are addressed as base + t * st + b * sb + h * sh + d, d contiguous.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace bh {

struct GaView {
  void* p = nullptr;
  int64_t st = 0, sb = 0, sh = 0;  // elements
};

struct GaArgs {
  GaView q, k, v, o, dout, dq, dk, dv;
  int sq = 0, sk = 0, b = 0, np = 0, ng = 0, hn = 0;
  int causal = 0;
  int window = 1 << 30;        // keys a causal query sees, its own included
  const int* lens = nullptr;  // [b] keys of each sequence (device), clamped to 0 .. sk
  float scale = 1.f;
  double p_drop = 0.;
  uint64_t seed = 0;
  const int64_t* seed_dev = nullptr;  // step seed of a captured step (utils/graph_rng.py)
  float* lse = nullptr;               // [b, np, sq] log2-sum-exp2 of the base-2 scaled scores, +inf: no key seen
  void* olo = nullptr;                // what rounding left of o, laid out like o (null: no backward follows)
  // backward scratch, written by the dQ kernel for the dK / dV kernel
  float* delta = nullptr;    // [b, np, sq] rowsum(dout * o), or its negative where the dK / dV kernel starts from it
  uint32_t* rowh = nullptr;  // [b, np, sq] dropout row hashes (with dropout)
};

// partial results of the split-key forward, in floats (0: the forward needs none)
int64_t ga_forward_workspace(const GaArgs& a);
void ga_forward(int dt, const GaArgs& a, float* ws, hipStream_t st);
// partial sums of dK / dV, in floats (0: none)
int64_t ga_backward_workspace(const GaArgs& a);
void ga_backward(int dt, const GaArgs& a, float* ws, hipStream_t st);  // dk.p null: dQ only

}  // namespace bh
