// The tcgen05 form of the chunked gated delta rule (delta_tc.cu), as the entry point calls it.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace tssm {
namespace delta {

struct TcCall {
  const void *u, *B, *C;
  const float *A_log, *dt, *beta, *h0;
  void* y;
  float *h_last, *states, *errs;
  void* ws;
  int64_t Bt, L, H, G, P, N;
  float scale;
};
struct TcBackCall {   // the backward's chain: dE, du, dS1 of every chunk, dh0
  const void *B, *C, *dy;
  const float *A_log, *dt, *beta, *dh_last;
  void* du;
  float *dh0, *dstates, *derrs;
  void* gates;   // one per (batch row, head, chunk)
  void* ws;
  int64_t Bt, L, H, G, P, N;
  float scale;
};
bool tc_takes(int64_t P, int64_t N, int dtype);   // shapes; the tensors must be 16-byte aligned as well
int64_t tc_workspace(int64_t Bt, int64_t L, int64_t H, int64_t P, int64_t N);
int tc_run(const TcCall& a, cudaStream_t st);
int64_t tc_back_workspace(int64_t Bt, int64_t L, int64_t H);
int tc_back_run(const TcBackCall& a, cudaStream_t st);

}  // namespace delta
}  // namespace tssm
