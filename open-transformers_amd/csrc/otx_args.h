// Arguments of the masked attention and rotary kernels, as the C ABI fills them in.
#pragma once

namespace otx {

struct MaskAttnArgs {
  const void *q, *k, *v, *o, *dout;
  void *out, *dq, *dk, *dv;
  float *lse, *dsum;    // [B, H, S]; lse in units of log 2
  signed char* low;     // [B, H, S, D] or null: the next eight bits of O's significands
  float* part;          // dK/dV partial sums of each query head, [2][B, H, S, D], or null
  const float* slopes;  // [H] or null
  const int* doc;       // [B, S] or null
  const int* prefix;    // [B] or null
  void* table;          // [B, ceil(S / 64)] of int4: least and greatest document of a block, whether it holds padding
  long sq[3], sk[3], sv[3], so[3], sdo[3], sdq[3], sdk[3], sdv[3];  // strides of b, h, s in elements
  int B, H, Hkv, S, window;
  float sigma, cap;
};

struct RotaryArgs {
  const void* x;
  void* y;
  const float *cosv, *sinv;  // [P, R / 2]
  const int* positions;      // [B, T] or null: row t is position t
  long sx[3], sy[3];         // strides of b, t, h in elements
  int B, T, H, D, R, P;
  float sign;  // 1, or -1 for the gradient
};

}  // namespace otx
