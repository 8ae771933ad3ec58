// Per-head RMS norm of queries and keys with the rotation of positions.
#pragma once

#include "attn_common.cuh"

namespace rvc {

struct RopeArgs {
  int type = 0, wtype = 0;  // of q / k and of the weights (AttnType)
  int B = 0, L = 0, Hq = 0, Hk = 0, D = 0, R = 0;
  int64_t P = 0;            // rows of the cos / sin tables
  int interleaved = 0;
  float eps = 0.f;
  const void *q = nullptr, *k = nullptr, *gq = nullptr, *gk = nullptr;  // g: gradients of the outputs
  int64_t qs[3] = {0, 0, 0}, ks[3] = {0, 0, 0}, gqs[3] = {0, 0, 0}, gks[3] = {0, 0, 0};
  const void *wq = nullptr, *wk = nullptr;     // [D]
  const float *cos = nullptr, *sin = nullptr;  // [P, R/2]
  const void* pos = nullptr;                   // [B, L] int32 / int64 with strides; nullptr = 0 .. L - 1
  int pos64 = 0;
  int64_t pos_b = 0, pos_l = 0;
  void *oq = nullptr, *ok = nullptr;           // contiguous outputs / input gradients
  void *dwq = nullptr, *dwk = nullptr;
  float* part = nullptr;                       // [blocks][D] partial weight gradients
  int head_block = 0;                          // heads of one item
  int q_blocks = 0;                            // blocks of the queries, the others take the keys
};

int64_t rope_backward_workspace(const RopeArgs& a, int sms);
void rope_forward(RopeArgs a, int sms, cudaStream_t st);
void rope_backward(RopeArgs a, void* ws, int sms, cudaStream_t st);

}  // namespace rvc
