// Host-side calls between the files of the chunked gated delta rule.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace tssm {
namespace delta {

// delta_prep.cu: the images of `chunks` chunks from c0 of every (batch row, head).
struct PrepCall {
  const void *B, *C;
  const float *A_log, *dt, *beta;
  uint8_t* img;
  void* gates;   // [Bt, H, nc] gates as well, or null
  int64_t Bt, L, H, G, N, c0, chunks, nc;
  float scale;
  int vec;       // N and the bases allow 16-byte pieces
};
int prep_run(const PrepCall& a, int dtype, cudaStream_t st);
int64_t prep_image_bytes();
int64_t segment_chunks(int64_t streams, int64_t nc);   // chunks whose images are made at a time

// delta_tc.cu: the scans on tcgen05 (bf16, N 64 or 128, P a multiple of 64, 16-byte aligned tensors).
struct TcCall {
  const void *u, *B, *C;
  const float *A_log, *dt, *beta, *h0;
  void* y;
  float *h_last, *states, *errs;
  uint8_t* img;
  float* carry;   // the state between segments
  int64_t Bt, L, H, G, P, N;
  float scale;
};
struct TcBackCall {   // the backward's chain: dE, dS1 and gates of every chunk, dh0
  const void *B, *C, *dy;
  const float *A_log, *dt, *beta, *dh_last;
  float *dh0, *dstates, *derrs;
  void* gates;
  uint8_t* img;
  int64_t Bt, L, H, G, P, N;
  float scale;
};
bool tc_takes(int64_t P, int64_t N, int dtype);
int tc_run(const TcCall& a, cudaStream_t st);
int tc_back_run(const TcBackCall& a, cudaStream_t st);

// delta_grad_tc.cu: the gradients of every (chunk, head) on tcgen05 (what tc_takes, with N = 128 and
// at most 8 value heads a key head).
struct TcGradCall {
  const void *B, *C, *dy;
  const float *A_log, *dt, *states, *errs, *dstates, *derrs;
  const void* gates;
  void *du, *dB, *dC;
  float *ddt, *dbeta, *da_part;
  int64_t Bt, L, H, G, P, nc;
  float scale;
  int* status;   // set by tc_grad_run
};
bool tc_grad_takes(int64_t H, int64_t G, int64_t N, bool tc);
int tc_grad_run(TcGradCall a, cudaStream_t st);

}  // namespace delta
}  // namespace tssm
