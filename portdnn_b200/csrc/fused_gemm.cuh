// Interface of the tensor-core product with a fused end (fused_gemm.cu).
#pragma once

#include "common.cuh"

namespace pdnn {

// A matrix in memory: `rows` rows of `cols` elements, `pitch` elements apart.
struct Matrix {
  const void* p;
  long long pitch;
  int rows, cols;
};

// What is made of a product: forward  pre = v + bias, out = aux + scale * act(v + bias);
// gradient  out = scale * v * act'(aux).  Null tensors are left out.  rows x cols elements, pitches in elements.
struct Finish {
  const void* bias;
  const void* aux;
  void* pre;
  void* out;
  long long aux_pitch, pre_pitch, out_pitch;
  int rows, cols, act, gradient;
  float scale;
};

// op(a) [f.rows][k] times op(b) [k][f.cols] with f's finish; ta, tb: stored the other way round.  fp16 and bf16 operands
// go to the tensor cores as they are and need rows on 16-byte boundaries (fused_gemm_operand_ok); fp32 operands of any
// alignment are cut into three bf16 parts in scratch.
// beside: the kernel ahead in the stream is another product that waits for its own predecessor before it lets the
// next kernel begin, and the two have nothing to do with one another: 16-bit products then begin where the first one leaves
// room (512x512x512 bf16, both gradients' products, behind one another / beside 11.0 / 7.9 us; no difference in large ones).
bool fused_gemm_operand_ok(int dtype, const Matrix& m);
int fused_gemm(int dtype, int ta, int tb, const Matrix& a, const Matrix& b, int k, const Finish& f, bool beside, cudaStream_t s);

// The same for a few fp32 rows x (row-major) and weights w, stored [f.cols][k] (k_rows) or [k][f.cols] (fused_rows.cu).
int fused_rows(bool k_rows, const Matrix& x, const Matrix& w, int k, const Finish& f, cudaStream_t s);

}  // namespace pdnn
