// Single-token gated delta rule on an f32 state resident in HBM.
//
// Per (stream, head), with the state row h_p [N] of value channel p:
//     hd = exp(-exp(A_log) dt) h_p ;  e = beta (x_p - hd . B)
//     h_p <- hd + e B ;  y_p = scale * (h_p . C)
// A pure HBM stream over the state (4 N bytes read and written per row, all
// other operands are shared by the P rows of a head).  Eight lanes own a row
// and hold it in registers between the two dot products, so each row is read
// and written once; lane l takes the 16-byte pieces l, l+8, ... so that eight
// lanes cover 128 contiguous bytes per load.  One row a thread and many resident
// blocks: at 192 streams x 32 heads of 128 x 128 the states (805 MB moved) take 120 us,
// as long as a copy of them; two and four rows a thread took 125 to 170.
#include "common.cuh"

namespace tssm {
namespace {

constexpr int LANES = 8;              // lanes per state row
constexpr int GROUPS = 256 / LANES;   // rows per pass of a block

template <typename T, bool VEC>
__device__ __forceinline__ void load4(const T* p, int n, int N, float (&f)[4]) {
  if constexpr (VEC) {
    if constexpr (std::is_same<T, float>::value) {
      const float4 v = n < N ? *reinterpret_cast<const float4*>(p + n) : make_float4(0.f, 0.f, 0.f, 0.f);
      f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
    } else {
      const uint2 v = n < N ? *reinterpret_cast<const uint2*>(p + n) : make_uint2(0u, 0u);
      const __nv_bfloat162 a = *reinterpret_cast<const __nv_bfloat162*>(&v.x);
      const __nv_bfloat162 b = *reinterpret_cast<const __nv_bfloat162*>(&v.y);
      f[0] = __low2float(a); f[1] = __high2float(a); f[2] = __low2float(b); f[3] = __high2float(b);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = n + i < N ? ldf(p + n + i) : 0.f;
  }
}

__device__ __forceinline__ float sum8(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// NV: 4-wide pieces of a row per lane (N <= 32 NV); VEC: 16-byte state and aligned B, C pieces.
template <typename IO, int NV, bool VEC>
__global__ void __launch_bounds__(256) delta_step_kernel(
    const IO* __restrict__ x, const float* __restrict__ dt, float* __restrict__ h, const float* __restrict__ A_log,
    const IO* __restrict__ B, const IO* __restrict__ C, const float* __restrict__ beta, IO* __restrict__ y, int H,
    int G, int P, int N, int ptiles, float scale) {
  const int64_t sh = blockIdx.x / ptiles;   // (stream, head)
  const int p = (int)(blockIdx.x - sh * ptiles) * GROUPS + threadIdx.x / LANES;
  const bool ok = p < P;
  const int l = threadIdx.x % LANES;
  const int64_t s = sh / H;
  const int hh = (int)(sh - s * H);
  float* hp = h + (sh * P + p) * N;
  float st[NV][4];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int n = 4 * (l + LANES * j);
    if constexpr (VEC) {
      const float4 v = ok && n < N ? __ldcs(reinterpret_cast<const float4*>(hp + n)) : make_float4(0.f, 0.f, 0.f, 0.f);
      st[j][0] = v.x; st[j][1] = v.y; st[j][2] = v.z; st[j][3] = v.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) st[j][i] = ok && n + i < N ? hp[n + i] : 0.f;
    }
  }
  const int64_t kv = (s * G + hh / (H / G)) * N;
  float k[NV][4], q[NV][4];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    load4<IO, VEC>(B + kv, 4 * (l + LANES * j), N, k[j]);
    load4<IO, VEC>(C + kv, 4 * (l + LANES * j), N, q[j]);
  }
  const float a = expf(-expf(__ldg(A_log + hh)) * __ldg(dt + sh));
  const float xv = ok ? ldf(x + sh * P + p) : 0.f;
  float pred = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      st[j][i] *= a;
      pred += st[j][i] * k[j][i];
    }
  const float e = __ldg(beta + sh) * (xv - sum8(pred));
  float out = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int n = 4 * (l + LANES * j);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      st[j][i] += e * k[j][i];
      out += st[j][i] * q[j][i];
    }
    if constexpr (VEC) {
      if (ok && n < N) __stcs(reinterpret_cast<float4*>(hp + n), make_float4(st[j][0], st[j][1], st[j][2], st[j][3]));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (ok && n + i < N) hp[n + i] = st[j][i];
    }
  }
  out = sum8(out);
  if (ok && l == 0) stf(y + sh * P + p, scale * out);
}

struct StepArgs {
  const void *x, *dt, *A_log, *B, *C, *beta;
  void *h, *y;
  int64_t S;
  int H, G, P, N;
  float scale;
};

template <typename IO, int NV, bool VEC>
void launch(const StepArgs& a, cudaStream_t st) {
  const int ptiles = (int)cdiv(a.P, GROUPS);
  delta_step_kernel<IO, NV, VEC><<<(unsigned)(a.S * a.H * ptiles), 256, 0, st>>>(
      (const IO*)a.x, (const float*)a.dt, (float*)a.h, (const float*)a.A_log, (const IO*)a.B, (const IO*)a.C,
      (const float*)a.beta, (IO*)a.y, a.H, a.G, a.P, a.N, ptiles, a.scale);
}

template <typename IO, int NV>
void pick(const StepArgs& a, bool vec, cudaStream_t st) {
  vec ? launch<IO, NV, true>(a, st) : launch<IO, NV, false>(a, st);
}

template <typename IO>
void by_width(const StepArgs& a, bool vec, cudaStream_t st) {
  if (a.N <= 32) pick<IO, 1>(a, vec, st);
  else if (a.N <= 64) pick<IO, 2>(a, vec, st);
  else if (a.N <= 128) pick<IO, 4>(a, vec, st);
  else pick<IO, 8>(a, vec, st);
}

}  // namespace
}  // namespace tssm

extern "C" int tssm_gated_delta_step(const void* x, const void* dt, void* h, const void* A_log, const void* B,
                                     const void* C, const void* beta, void* y, int64_t S, int64_t H, int64_t G,
                                     int64_t P, int64_t N, double scale, int dtype, tssm_stream_t stream) {
  using namespace tssm;
  TSSM_REQUIRE(S >= 0 && H >= 0 && G >= 0 && P >= 0 && N >= 0, "gated_delta_step: negative size");
  if (S * H * P == 0) return TSSM_OK;
  TSSM_REQUIRE(N >= 1 && N <= 256, "gated_delta_step: state size N must be 1 to 256 (got %lld)", (long long)N);
  TSSM_REQUIRE(G >= 1 && H % G == 0, "gated_delta_step: H (%lld) must be a multiple of the key heads G (%lld)",
               (long long)H, (long long)G);
  TSSM_REQUIRE(x && dt && h && A_log && B && C && beta && y, "gated_delta_step: null pointer");
  TSSM_REQUIRE(dtype == TSSM_F32 || dtype == TSSM_BF16, "gated_delta_step: dtype must be f32 or bf16 (got %d)", dtype);
  TSSM_REQUIRE(H <= 1 << 20 && P <= 1 << 20 && S * H * cdiv(P, GROUPS) < (int64_t(1) << 31),
               "gated_delta_step: size out of range");
  const StepArgs a{x, dt, A_log, B, C, beta, h, y, S, (int)H, (int)G, (int)P, (int)N, (float)scale};
  const uintptr_t kq = reinterpret_cast<uintptr_t>(B) | reinterpret_cast<uintptr_t>(C);
  const bool vec = N % 4 == 0 && aligned16(h) && (kq & (dtype == TSSM_F32 ? 15u : 7u)) == 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == TSSM_F32) by_width<float>(a, vec, st);
  else by_width<__nv_bfloat16>(a, vec, st);
  return check_launch("gated_delta_step");
}
