// The AdamW object behind a gt_adamw handle: groups with FP32 moments (optim.hip) and with 8-bit ones (adamw8.hip).
#pragma once
#include <vector>
#include "common.h"

#define CHUNK 2048

struct Chunk { int tensor; int len; int64_t off; };
struct TensorPtrs { float *w, *g, *m, *v; };

// A run of a tensor's 256-element blocks, the tensor's buffers already advanced to it.
struct Chunk8 { float *w; const float *g; unsigned char *m, *r; signed char *e; int len; unsigned block; };
struct Tensor8 { unsigned char *m, *r; signed char *e; int64_t size; };

struct gt_adamw {
  int n = 0, nchunks = 0;
  double total_elems = 0;
  double beta1, beta2, eps, wd, clip;
  Chunk *chunks = nullptr;
  TensorPtrs *ptrs = nullptr;
  float *partial = nullptr;     // [nchunks]
  float *scale = nullptr;       // [2]: clip scale, grad norm
  bool bits8 = false;
  void *block8 = nullptr;       // the one allocation behind scale, sums8 and chunks8 of a group with 8-bit moments
  Chunk8 *chunks8 = nullptr;
  double *sums8 = nullptr;      // partial sums of squares, one per workgroup of the norm's kernel
  std::vector<Tensor8> tensors8;
};

void adamw_release(gt_adamw *o);
