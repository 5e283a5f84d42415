// The chunk matrices of the gated delta rule, for every (chunk, head) of a segment at
// once: T and Aq diag(beta) depend on no state (formulas: delta.cuh).  A block builds one
// chunk's image (planes and gates, as the scans copy them to shared memory) and leaves it in
// HBM; a segment's images take about SEGMENT_BYTES, so that a long sequence needs no more.
//
// Bound by issue slots and latency (about 1900 instructions a warp; 128 threads, six blocks an
// SM for bf16): 17 ns per chunk and head with N = 128 on a full GPU.  Inside the scans, one
// group of four warps took 4 to 6 us a chunk, more than the scan itself.
#include "delta.cuh"
#include "delta_tc.h"

namespace tssm {
namespace delta {
namespace {

template <int XS, int KN>
struct PrepSmem {
  static constexpr int PLANE = Q * KN * 2, MB = Q * AM * 4;   // the work matrix lies over the Q tile
  static constexpr int K = 0, QQ = XS * PLANE, M = QQ, G = QQ + (MB > XS * PLANE ? MB : XS * PLANE),
                       BYTES = G + (int)sizeof(Gates) + 128;
};

template <int XS, int KN>
__global__ void __launch_bounds__(128, XS == 1 ? 6 : 2) delta_prep_kernel(const PrepCall a) {
  let_next_start();
  using T = typename std::conditional<XS == 1, __nv_bfloat16, float>::type;
  using SM = PrepSmem<XS, KN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((128u - (smem_addr(smem_raw) & 127u)) & 127u);
  const uint32_t s = smem_addr(smem);
  const int t = threadIdx.x;
  const int64_t bh = blockIdx.x / a.chunks, ci = blockIdx.x - bh * a.chunks, b = bh / a.H;
  const int h = (int)(bh - b * a.H), g = h / (int)(a.H / a.G);
  const int64_t t0 = (a.c0 + ci) * Q, sk = a.G * a.N;
  const int rows = (int)min((int64_t)Q, a.L - t0);
  const int64_t at = (b * a.L + t0) * sk + (int64_t)g * a.N;
  load_planes<XS, KN, 128>(s + SM::K, SM::PLANE, (const T*)a.B + at, sk, rows, (int)a.N, a.vec, t);
  load_planes<XS, KN, 128>(s + SM::QQ, SM::PLANE, (const T*)a.C + at, sk, rows, (int)a.N, a.vec, t);
  Gates& gt = *reinterpret_cast<Gates*>(smem + SM::G);
  if (t < 32) gates_warp(gt, a.dt + b * a.L * a.H + h, a.beta + b * a.L * a.H + h, a.H, a.A_log[h], t0, a.L, t);
  cp_async_wait_all();
  __syncthreads();
  uint8_t* img = a.img + (bh * a.chunks + ci) * IMG_BYTES;
  copy_gates(reinterpret_cast<Gates*>(img + IMG_GATES), gt, t);
  if (a.gates) copy_gates((Gates*)a.gates + bh * a.nc + a.c0 + ci, gt, t);
  chunk_matrices<XS, KN>(s + SM::K, s + SM::QQ, gt, a.scale, reinterpret_cast<float*>(smem + SM::M),
                                img + IMG_AQ, img + IMG_T, t, 1);
}

template <int XS, int KN>
int launch(const PrepCall& a, cudaStream_t st) {
  auto kern = delta_prep_kernel<XS, KN>;
  constexpr int bytes = PrepSmem<XS, KN>::BYTES;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return check_launch("gated_delta_rule: set smem attribute");
  kern<<<(unsigned)(a.Bt * a.H * a.chunks), 128, bytes, st>>>(a);
  return check_launch("gated_delta_rule: chunk matrices");
}

}  // namespace

int64_t prep_image_bytes() { return IMG_BYTES; }

int prep_run(const PrepCall& a, int dtype, cudaStream_t st) {
  TSSM_REQUIRE(a.Bt * a.H * a.chunks < (int64_t(1) << 31), "gated_delta_rule: size out of range");
  if (dtype == TSSM_F32) return a.N <= 64 ? launch<3, 64>(a, st) : launch<3, 128>(a, st);
  return a.N <= 64 ? launch<1, 64>(a, st) : launch<1, 128>(a, st);
}

int64_t segment_chunks(int64_t streams, int64_t nc) {
  constexpr int64_t SEGMENT_BYTES = 320ll << 20;   // in L2 (126 MB) or not makes little difference; fewer segments do
  return std::max<int64_t>(1, std::min(nc, SEGMENT_BYTES / (streams * IMG_BYTES)));
}

}  // namespace delta
}  // namespace tssm
