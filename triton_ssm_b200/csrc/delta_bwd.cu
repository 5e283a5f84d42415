// Chunked gated delta rule, backward (forward formulas: delta.cuh).
//
// With dO, the gradient dS1 of the state behind a chunk, and E, S0 as the
// forward saved them (w = exp(l_last - l), A strictly lower, both without beta):
//     R   = diag(beta) (Aq^T dO + w K dS1)             dE = T^T R  (= du)
//     dS0 = exp(l_last) dS1 + (scale exp(l) Q)^T dO - (exp(l) K)^T dE
//     M1  = scale D (dO E^T) diag(beta)                M2 = D (dE E^T) diag(beta), strictly lower
//     dQ  = scale exp(l) dO S0^T + M1 K
//     dK  = w beta E dS1^T - exp(l) dE S0^T + M1^T Q - M2 K - M2^T K
//     Y   = scale D (q.k) (dO E^T) - D (k.k) (dE E^T)  (the second strictly lower)
//     dbeta_j = sum_i Y_ij + w_j (E dS1^T)_j . k_j
//     dl_t, the gradient of token t's log-decay, sums every path that crosses it, so that
//     nothing cancels:  sum_{i >= t > j} Y_ij beta_j + sum_{i >= t} a_i + sum_{j < t} b_j
//     + exp(l_last) <S0, dS1>,  a_i = (state parts of dQ, dK)_i . (q, k)_i,
//     b_j = w_j beta_j (E dS1^T)_j . k_j.
//
// The chain runs the chunks of a (batch row, head) backwards as the forward runs them
// forwards, over the images of delta_prep.cu, and leaves dE and the dS1 of every chunk in
// HBM (du, which is dE, is written by the gradient kernel: in the serial chain its narrow stores
// took 20 us more than there).  bf16 shapes that delta_tc.cu takes run there; the kernel here (16 value channels
// and a state gradient per warp, in registers) is for f32 and the others.  The gradient
// kernel then takes all (chunk, head) pairs at once: delta_grad_tc.cu for the chain's bf16
// shapes with N = 128, the one here (mma.sync) for the rest.  Shared key heads and dA_log are
// summed last, in a fixed order, so results repeat bit for bit.
//
// Measured at 4 x 2048 tokens x 16 heads on 8 key heads, N = P = 128, bf16 (with the
// forward 0.64 ms): images 40 us, chain 153, gradients with du and the key heads' sums 270,
// dA_log 3.  The gradient kernel here took 384 for them and 38 for the key heads (M1, M2 in two
// planes then): it has 11 products of 64-wide tiles in up to three planes, its mma.sync pipe is
// busy 38 % of the time, and the loads of its one block an SM are exposed.
#include "delta.cuh"
#include "delta_tc.h"

namespace tssm {
namespace delta {
namespace {

struct BwdArgs {
  const void *u, *B, *C, *dy;
  const float *A_log, *dt, *beta, *states, *errs, *dh_last;
  void *du, *dB, *dC;
  float *dA_log, *ddt, *dbeta, *dh0;
  float *dstates, *derrs, *dk_part, *dq_part, *da_part;   // workspace
  Gates* gates;   // of every chunk
  uint8_t* img;   // of a segment
  const float* ds_in;      // the chain's segment: its state gradient, first chunk, chunks
  int64_t c0, nseg;
  int64_t Bt, L, nc;
  int H, G, P, N, npb;
  float scale;
  int vec_kq, vec_v;
};

// ------------------------------------------------------------------ the chain
template <int XS, int KN, int NCW>
struct ChainSmem {
  static constexpr int BUFS = XS == 1 ? 2 : 1;
  static constexpr int PB = 16 * NCW, PLANE = Q * KN * 2, DO_PLANE = Q * PB * 2;
  static constexpr int K = 0, QQ = K + XS * PLANE, DO = QQ + XS * PLANE, T = DO + XS * DO_PLANE, AQ = T + 3 * SQ_BYTES,
                       G = AQ + 3 * SQ_BYTES, BUF = (G + (int)sizeof(Gates) + 127) / 128 * 128;   // T, AQ, G: an image
  static constexpr int BYTES = BUFS * BUF + 128;
};

template <int XS, int KN, int NCW>
__global__ void __launch_bounds__((NCW + 4) * 32, 1) delta_bwd_chain_kernel(const BwdArgs a) {
  let_next_start();
  wait_for_previous();
  using T = typename std::conditional<XS == 1, __nv_bfloat16, float>::type;
  using SM = ChainSmem<XS, KN, NCW>;
  constexpr int PB = SM::PB, RB = KN * 2, NT = KN / 8, NS = 3, RV = PB * 2;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((128u - (smem_addr(smem_raw) & 127u)) & 127u);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t bh = blockIdx.x / a.npb;
  const int pb = (int)(blockIdx.x - bh * a.npb) * PB;
  const int64_t b = bh / a.H;
  const int h = (int)(bh - b * a.H), g = h / (a.H / a.G);
  const int64_t su = (int64_t)a.H * a.P, sk = (int64_t)a.G * a.N;
  const T* kp = (const T*)a.B + (b * a.L) * sk + (int64_t)g * a.N;
  const T* qp = (const T*)a.C + (b * a.L) * sk + (int64_t)g * a.N;
  const T* op = (const T*)a.dy + (b * a.L) * su + (int64_t)h * a.P + pb;
  const int pvalid = min(PB, a.P - pb);

  // Chunk c of the segment to shared memory: by the four loading warps, or (one buffer) by all.
  constexpr int LT = SM::BUFS == 2 ? 128 : (NCW + 4) * 32;
  auto load = [&](int64_t c) {
    const int t = threadIdx.x - (SM::BUFS == 2 ? NCW * 32 : 0);
    uint8_t* buf = smem + (SM::BUFS == 2 ? (int)(c & 1) * SM::BUF : 0);
    const uint32_t s = smem_addr(buf);
    const int64_t t0 = (a.c0 + c) * Q;
    const int rows = (int)min((int64_t)Q, a.L - t0);
    load_image<LT>(s + SM::T, a.img + (bh * a.nseg + c) * IMG_BYTES, t);
    load_planes<XS, KN, LT>(s + SM::K, SM::PLANE, kp + t0 * sk, sk, rows, a.N, a.vec_kq, t);
    load_planes<XS, KN, LT>(s + SM::QQ, SM::PLANE, qp + t0 * sk, sk, rows, a.N, a.vec_kq, t);
    load_planes<XS, PB, LT>(s + SM::DO, SM::DO_PLANE, op + t0 * su, su, rows, pvalid, a.vec_v, t);
    cp_async_wait_all();
  };

  const int p0 = 16 * warp;
  const int pr = lane / 4, q2 = 2 * (lane % 4);
  float S[NT][4];   // dS^T: 16 channels x N
  const int64_t srow = (bh * a.P + pb + p0 + pr) * (int64_t)a.N;
  auto state_io = [&](float* dst, const float* src) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = 8 * j + q2 + (e & 1), p = pb + p0 + pr + (e >> 1) * 8;
        const bool in = n < a.N && p < a.P;
        const int64_t at = (int64_t)(e >> 1) * 8 * a.N + n;
        if (dst) {
          if (in) dst[at] = S[j][e];
        } else {
          S[j][e] = src && in ? src[at] : 0.f;
        }
      }
  };

  auto chain = [&](int64_t c) {
    uint8_t* buf = smem + (SM::BUFS == 2 ? (int)(c & 1) * SM::BUF : 0);
    const uint32_t s = smem_addr(buf);
    const Gates& gt = *reinterpret_cast<const Gates*>(buf + SM::G);
    const int64_t t0 = (a.c0 + c) * Q;
    const int rows = (int)min((int64_t)Q, a.L - t0);
    {
      float* dst = a.dstates + (bh * a.nc + a.c0 + c) * saved_floats(a.P, a.N);
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int r = 0; r < 2; ++r)
          if (8 * j + q2 < (a.N + 3) / 4 * 4 && pb + p0 + pr + 8 * r < a.P)
            *saved_pair(dst, a.P, pb + p0 + pr + 8 * r, 8 * j + q2) = make_float2(S[j][2 * r], S[j][2 * r + 1]);
    }
    // dO^T fragments of 16 tokens from 16 t
    auto load_do = [&](int t, uint32_t (&f)[XS][4]) {
#pragma unroll
      for (int z = 0; z < XS; ++z)
        ldsm4t(f[z], s + SM::DO + z * SM::DO_PLANE +
                         tile_off<RV>(16 * t + ((lane >> 4) << 3) + (lane & 7), p0 / 8 + ((lane >> 3) & 1)));
    };
    // R^T = (dS^T K^T) diag(w beta) + dO^T (Aq diag(beta))
    float x[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[i][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < KN / 16; ++kk) {
      uint32_t f[NS][4];
      split_a<NS>(S[2 * kk], S[2 * kk + 1], f);
#pragma unroll
      for (int np = 0; np < 4; ++np) {
        uint32_t w[XS][4];
#pragma unroll
        for (int z = 0; z < XS; ++z) ldsm4(w[z], at_b<RB>(s + SM::K + z * SM::PLANE, 16 * np, 2 * kk, lane));
        mma_planes<NS, XS, NS, XS == 3>(x[2 * np], x[2 * np + 1], f, w);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 wb = *reinterpret_cast<const float2*>(gt.wb + 8 * i + q2);
      x[i][0] *= wb.x;
      x[i][1] *= wb.y;
      x[i][2] *= wb.x;
      x[i][3] *= wb.y;
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      uint32_t f[XS][4];
      load_do(t, f);
#pragma unroll
      for (int np = 0; np <= t; ++np) {
        uint32_t w[3][4];
#pragma unroll
        for (int z = 0; z < 3; ++z) ldsm4t(w[z], at_a<SQ_RB>(s + SM::AQ + z * SQ_BYTES, 16 * t, 2 * np, lane));
        mma_planes<XS, 3, 3>(x[2 * np], x[2 * np + 1], f, w);
      }
    }
    // dE^T = R^T T
    float er[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) er[i][e] = 0.f;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      uint32_t f[NS][4];
      split_a<NS>(x[2 * t], x[2 * t + 1], f);
#pragma unroll
      for (int np = 0; np <= t; ++np) {
        uint32_t w[3][4];
#pragma unroll
        for (int z = 0; z < 3; ++z) ldsm4t(w[z], at_a<SQ_RB>(s + SM::T + z * SQ_BYTES, 16 * t, 2 * np, lane));
        mma_planes<NS, 3, 3>(er[2 * np], er[2 * np + 1], f, w);
      }
    }
    // dS^T = exp(l_last) dS^T + (scale dO exp(l))^T Q - (dE exp(l))^T K
    const float el = gt.eg[Q - 1];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) S[j][e] *= el;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      float d[2][4], k2[2][4];
      {
        uint32_t f[XS][4];
        load_do(t, f);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const float2 eg = *reinterpret_cast<const float2*>(gt.eg + 16 * t + 8 * m + q2);
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float lo = 0.f, hi = 0.f;
#pragma unroll
            for (int z = XS - 1; z >= 0; --z) {
              lo += lo2(f[z][2 * m + r]);
              hi += hi2(f[z][2 * m + r]);
            }
            d[m][2 * r] = a.scale * eg.x * lo;
            d[m][2 * r + 1] = a.scale * eg.y * hi;
            k2[m][2 * r] = -eg.x * er[2 * t + m][2 * r];
            k2[m][2 * r + 1] = -eg.y * er[2 * t + m][2 * r + 1];
          }
        }
      }
      uint32_t fd[NS][4], fk[NS][4];
      split_a<NS>(d[0], d[1], fd);
      split_a<NS>(k2[0], k2[1], fk);
#pragma unroll
      for (int nn = 0; nn < KN / 16; ++nn) {
        uint32_t w[XS][4];
#pragma unroll
        for (int z = 0; z < XS; ++z) ldsm4t(w[z], at_a<RB>(s + SM::QQ + z * SM::PLANE, 16 * t, 2 * nn, lane));
        mma_planes<NS, XS, NS, true>(S[2 * nn], S[2 * nn + 1], fd, w);
#pragma unroll
        for (int z = 0; z < XS; ++z) ldsm4t(w[z], at_a<RB>(s + SM::K + z * SM::PLANE, 16 * t, 2 * nn, lane));
        mma_planes<NS, XS, NS, true>(S[2 * nn], S[2 * nn + 1], fk, w);
      }
    }
    // dE for the gradient kernel
    float* ep = a.derrs + bh * saved_floats(a.P, a.L);
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int tk = 8 * i + q2, p = 8 * r;
        if (p0 + pr + p >= pvalid) continue;
        if ((tk & ~3) < rows)
          *saved_pair(ep, a.P, pb + p0 + pr + p, t0 + tk) = make_float2(er[i][2 * r], er[i][2 * r + 1]);
      }
  };

  if (warp < NCW) state_io(nullptr, a.ds_in ? a.ds_in + srow : nullptr);
  if constexpr (SM::BUFS == 2) {
    if (warp >= NCW) load(a.nseg - 1);
    __syncthreads();
    for (int64_t c = a.nseg - 1; c >= 0; --c) {
      if (warp < NCW) chain(c);
      else if (c > 0) load(c - 1);
      __syncthreads();
    }
  } else {
    for (int64_t c = a.nseg - 1; c >= 0; --c) {
      load(c);
      __syncthreads();
      if (warp < NCW) chain(c);
      __syncthreads();
    }
  }
  if (warp < NCW) state_io(a.dh0 + srow, nullptr);
}

// ------------------------------------------------------------------ the gradients of one (chunk, head)
template <int XS, int KN>
struct GradSmem {
  static constexpr int PLANE = Q * KN * 2;        // of K, Q, and of 64 state rows
  static constexpr int K = 0, QQ = K + XS * PLANE, DO = QQ + XS * PLANE, E = DO + XS * SQ_BYTES, DE = E + 3 * SQ_BYTES,
                       S = DE + 3 * SQ_BYTES, G = S + 3 * PLANE, VEC = G + (int)sizeof(Gates);
  static constexpr int M1 = E, M2 = DE;           // after the channel loop
  static constexpr int Y = S;                     // 64 x 65 floats, after it too
  static constexpr int BYTES = VEC + (4 * Q * 3 + Q * 8 + 16) * 4 + 128;
  static_assert(3 * PLANE >= Q * 65 * 4, "Y fits the state region");
};
constexpr int GT = 512;   // threads: warp = (16 tokens, a quarter of N)

template <int XS, int KN>
__global__ void __launch_bounds__(GT, 1) delta_bwd_grad_kernel(const BwdArgs a) {
  let_next_start();
  wait_for_previous();
  using T = typename std::conditional<XS == 1, __nv_bfloat16, float>::type;
  using SM = GradSmem<XS, KN>;
  constexpr int RB = KN * 2, NTQ = KN / 32;   // 8-wide tiles of a warp's quarter of N
  constexpr int SP = KN / 64;                 // pieces of a 64 x KN state tile per thread
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((128u - (smem_addr(smem_raw) & 127u)) & 127u);
  const uint32_t s = smem_addr(smem);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int mt = warp % 4, qt = warp / 4, pr = lane / 4, q2 = 2 * (lane % 4);
  const int64_t bh = blockIdx.x / a.nc, c = blockIdx.x - bh * a.nc, b = bh / a.H;
  const int h = (int)(bh - b * a.H), g = h / (a.H / a.G);
  const int64_t t0 = c * Q, su = (int64_t)a.H * a.P, sk = (int64_t)a.G * a.N;
  const int rows = (int)min((int64_t)Q, a.L - t0);
  const Gates& gt = *reinterpret_cast<const Gates*>(smem + SM::G);
  float* vec = reinterpret_cast<float*>(smem + SM::VEC);
  float *va = vec, *vb = vec + 4 * Q, *vw = vec + 8 * Q;   // [4][Q] row dots of a, b, and w e.(K dS1), by quarter
  float* seg = vec + 12 * Q;                               // [8][Q] column sums of Y by row eighth
  float* red = seg + 8 * Q;                                // [16] <S0, dS1> by warp

  const float* S0 = a.states + (bh * a.nc + c) * saved_floats(a.P, a.N);
  const float* dS = a.dstates + (bh * a.nc + c) * saved_floats(a.P, a.N);
  const int64_t tok = (b * a.L + t0) * su + (int64_t)h * a.P;
  // A thread's state pieces: row sr, pieces sc, sc + 8.
  const int sr = tid % 64, sc = tid / 64;   // lanes on neighbouring rows
  float fs[SP][8];   // the next pieces of S0 and dS1, in flight during the products
  auto fetch_state = [&](const float* src, int p0, float (&fs)[SP][8]) {
#pragma unroll
    for (int i = 0; i < SP; ++i)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int n4 = 2 * (sc + 8 * i) + q;
        const float4 v = p0 + sr < a.P && 4 * n4 < a.N
                             ? *reinterpret_cast<const float4*>(src + ((int64_t)n4 * a.P + p0 + sr) * 4)
                             : make_float4(0.f, 0.f, 0.f, 0.f);
        fs[i][4 * q] = v.x; fs[i][4 * q + 1] = v.y; fs[i][4 * q + 2] = v.z; fs[i][4 * q + 3] = v.w;
      }
  };
  float fd[SP][8];
  fetch_state(S0, 0, fs);
  fetch_state(dS, 0, fd);
  if (tid < (int)(sizeof(Gates) / 16))
    cp_async16(s + SM::G + 16 * tid, reinterpret_cast<const uint4*>(a.gates + bh * a.nc + c) + tid, true);
  load_planes<XS, KN, GT>(s + SM::K, SM::PLANE, (const T*)a.B + (b * a.L + t0) * sk + (int64_t)g * a.N, sk, rows, a.N,
                          a.vec_kq, tid);
  load_planes<XS, KN, GT>(s + SM::QQ, SM::PLANE, (const T*)a.C + (b * a.L + t0) * sk + (int64_t)g * a.N, sk, rows, a.N,
                          a.vec_kq, tid);

  float dq0[NTQ][4], dk0[NTQ][4], dk1[NTQ][4], m1[2][4], m2[2][4];
  auto zero = [](auto& m) {
    for (auto& r : m)
      for (float& v : r) v = 0.f;
  };
  zero(dq0);
  zero(dk0);
  zero(dk1);
  zero(m1);
  zero(m2);
  float dot = 0.f;
  for (int p0 = 0; p0 < a.P; p0 += 64) {
    const int pv = min(64, a.P - p0);
    if (p0) __syncthreads();
    {
      float4 fe[2], fr[2];   // four tokens from 4 warp of channels 2 lane, 2 lane + 1
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const bool in = 4 * warp < rows && 2 * lane + q < pv;
        const int64_t at = bh * saved_floats(a.P, a.L) + ((t0 / 4 + warp) * a.P + p0 + 2 * lane + q) * 4;
        fe[q] = in ? *reinterpret_cast<const float4*>(a.errs + at) : make_float4(0.f, 0.f, 0.f, 0.f);
        fr[q] = in ? *reinterpret_cast<const float4*>(a.derrs + at) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      load_planes<XS, 64, GT>(s + SM::DO, SQ_BYTES, (const T*)a.dy + tok + p0, su, rows, pv, a.vec_v, tid);
#pragma unroll
      for (int i = 0; i < SP; ++i) {
#pragma unroll
        for (int e = 0; e < 8; ++e) dot += fs[i][e] * fd[i][e];
        put8(smem + SM::S + tile_off<RB>(sr, sc + 8 * i), SM::PLANE, fs[i]);
      }
      put4x2(smem + SM::E, 4 * warp, lane, fe);
      put4x2(smem + SM::DE, 4 * warp, lane, fr);
#pragma unroll
      for (int q = 0; q < 2; ++q) {   // du = dE
        const float d[4] = {fr[q].x, fr[q].y, fr[q].z, fr[q].w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (4 * warp + i < rows && 2 * lane + q < pv) stf((T*)a.du + tok + (4 * warp + i) * su + p0 + 2 * lane + q, d[i]);
      }
    }
    cp_async_wait_all();
    __syncthreads();
#pragma unroll 1
    for (int kk = 0; kk < 4; ++kk) {
      uint32_t fo[XS][4], fe[3][4], w[3][4];
#pragma unroll
      for (int z = 0; z < XS; ++z) ldsm4(fo[z], at_a<SQ_RB>(s + SM::DO + z * SQ_BYTES, 16 * mt, 2 * kk, lane));
#pragma unroll
      for (int z = 0; z < 3; ++z) ldsm4(fe[z], at_a<SQ_RB>(s + SM::DE + z * SQ_BYTES, 16 * mt, 2 * kk, lane));
      if (qt <= mt) {
#pragma unroll
        for (int z = 0; z < 3; ++z) ldsm4(w[z], at_b<SQ_RB>(s + SM::E + z * SQ_BYTES, 16 * qt, 2 * kk, lane));
        mma_planes<XS, 3, 3, XS == 3>(m1[0], m1[1], fo, w);
        mma_planes<3, 3, 3, XS == 3>(m2[0], m2[1], fe, w);
      }
#pragma unroll
      for (int nn = 0; nn < NTQ / 2; ++nn) {
#pragma unroll
        for (int z = 0; z < 3; ++z) ldsm4t(w[z], at_a<RB>(s + SM::S + z * SM::PLANE, 16 * kk, qt * NTQ + 2 * nn, lane));
        mma_planes<XS, 3, 3, XS == 3>(dq0[2 * nn], dq0[2 * nn + 1], fo, w);
        mma_planes<3, 3, 3, XS == 3>(dk0[2 * nn], dk0[2 * nn + 1], fe, w);
      }
    }
    __syncthreads();
    // dS1 takes S0's place
#pragma unroll
    for (int i = 0; i < SP; ++i) put8(smem + SM::S + tile_off<RB>(sr, sc + 8 * i), SM::PLANE, fd[i]);
    __syncthreads();
    if (p0 + 64 < a.P) {
      fetch_state(S0, p0 + 64, fs);
      fetch_state(dS, p0 + 64, fd);
    }
#pragma unroll 1
    for (int kk = 0; kk < 4; ++kk) {
      uint32_t fe[3][4], w[3][4];
#pragma unroll
      for (int z = 0; z < 3; ++z) ldsm4(fe[z], at_a<SQ_RB>(s + SM::E + z * SQ_BYTES, 16 * mt, 2 * kk, lane));
#pragma unroll
      for (int nn = 0; nn < NTQ / 2; ++nn) {
#pragma unroll
        for (int z = 0; z < 3; ++z) ldsm4t(w[z], at_a<RB>(s + SM::S + z * SM::PLANE, 16 * kk, qt * NTQ + 2 * nn, lane));
        mma_planes<3, 3, 3, XS == 3>(dk1[2 * nn], dk1[2 * nn + 1], fe, w);
      }
    }
  }
  __syncthreads();   // the regions of E, dE and the state are free; the gates were written long ago

  // row dots over this warp's quarter of N, and the state parts of dQ, dK (in dq0, dk0)
  {
    float ra[2] = {0.f, 0.f}, rb[2] = {0.f, 0.f};
    const int i0 = 16 * mt + pr;
#pragma unroll
    for (int j = 0; j < NTQ; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int i = i0 + 8 * r;
        const float eg = gt.eg[i], wb = gt.wb[i];
        const uint32_t off = tile_off<RB>(i, qt * NTQ + j) + 2 * q2;
        float kl = 0.f, kh = 0.f, ql = 0.f, qh = 0.f;
#pragma unroll
        for (int z = XS - 1; z >= 0; --z) {
          const uint32_t kv = *reinterpret_cast<const uint32_t*>(smem + SM::K + z * SM::PLANE + off);
          const uint32_t qv = *reinterpret_cast<const uint32_t*>(smem + SM::QQ + z * SM::PLANE + off);
          kl += lo2(kv); kh += hi2(kv); ql += lo2(qv); qh += hi2(qv);
        }
        const float q0 = a.scale * eg * dq0[j][2 * r], q1 = a.scale * eg * dq0[j][2 * r + 1];
        const float k0 = -eg * dk0[j][2 * r], k1 = -eg * dk0[j][2 * r + 1];
        ra[r] += q0 * ql + q1 * qh + k0 * kl + k1 * kh;
        rb[r] += dk1[j][2 * r] * kl + dk1[j][2 * r + 1] * kh;
        dq0[j][2 * r] = q0;
        dq0[j][2 * r + 1] = q1;
        dk0[j][2 * r] = k0 + wb * dk1[j][2 * r];
        dk0[j][2 * r + 1] = k1 + wb * dk1[j][2 * r + 1];
      }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        ra[r] += __shfl_xor_sync(0xffffffffu, ra[r], o);
        rb[r] += __shfl_xor_sync(0xffffffffu, rb[r], o);
      }
      if (lane % 4 == 0) {
        const int i = i0 + 8 * r;
        va[qt * Q + i] = ra[r];
        vb[qt * Q + i] = gt.wb[i] * rb[r];
        vw[qt * Q + i] = gt.w[i] * rb[r];
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if (lane == 0) red[warp] = dot;
  }
  // q.k and k.k of this warp's 16 x 16 block, then M1, M2 (planes) and Y
  {
    float gk[2][4], gq[2][4];
    zero(gk);
    zero(gq);
    if (qt <= mt) {
#pragma unroll 4
      for (int kk = 0; kk < KN / 16; ++kk) {
        uint32_t fk[XS][4], fq[XS][4], w[XS][4];
#pragma unroll
        for (int z = 0; z < XS; ++z) {
          ldsm4(fk[z], at_a<RB>(s + SM::K + z * SM::PLANE, 16 * mt, 2 * kk, lane));
          ldsm4(fq[z], at_a<RB>(s + SM::QQ + z * SM::PLANE, 16 * mt, 2 * kk, lane));
          ldsm4(w[z], at_b<RB>(s + SM::K + z * SM::PLANE, 16 * qt, 2 * kk, lane));
        }
        mma_planes<XS, XS, XS, XS == 3>(gk[0], gk[1], fk, w);
        mma_planes<XS, XS, XS, XS == 3>(gq[0], gq[1], fq, w);
      }
    }
    float* Y = reinterpret_cast<float*>(smem + SM::Y);
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      const int j = 16 * qt + 8 * nt + q2;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int i = 16 * mt + pr + 8 * r;
        float u1[2], u2[2], yy[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int jj = j + e;
          const float D = jj <= i ? exp2f((gt.lh[i] - gt.lh[jj]) + (gt.ll[i] - gt.ll[jj])) : 0.f;
          const float f1 = jj <= i ? a.scale * D * m1[nt][2 * r + e] : 0.f;
          const float f2 = jj < i ? D * m2[nt][2 * r + e] : 0.f;
          yy[e] = f1 * gq[nt][2 * r + e] - f2 * gk[nt][2 * r + e];
          u1[e] = f1 * gt.beta[jj];
          u2[e] = f2 * gt.beta[jj];
          Y[i * 65 + jj] = yy[e];
        }
        uint32_t p1[3], p2[3];
        split2<3>(u1[0], u1[1], p1);
        split2<3>(u2[0], u2[1], p2);
        const uint32_t off = tile_off<SQ_RB>(i, 2 * qt + nt) + 2 * q2;
#pragma unroll
        for (int z = 0; z < 3; ++z) {
          *reinterpret_cast<uint32_t*>(smem + SM::M1 + z * SQ_BYTES + off) = p1[z];
          *reinterpret_cast<uint32_t*>(smem + SM::M2 + z * SQ_BYTES + off) = p2[z];
        }
      }
    }
  }
  __syncthreads();
  // dQ += M1 K;  dK += M1^T Q - M2 K - M2^T K   (lower triangles: 16-blocks i >= j)
  zero(dk1);
#pragma unroll 1
  for (int t = 0; t < 4; ++t) {
    uint32_t f[3][4], w[XS][4], w2[XS][4];
#pragma unroll
    for (int nn = 0; nn < NTQ / 2; ++nn) {
#pragma unroll
      for (int z = 0; z < XS; ++z) {
        ldsm4t(w[z], at_a<RB>(s + SM::K + z * SM::PLANE, 16 * t, qt * NTQ + 2 * nn, lane));
        ldsm4t(w2[z], at_a<RB>(s + SM::QQ + z * SM::PLANE, 16 * t, qt * NTQ + 2 * nn, lane));
      }
      if (t <= mt) {   // rows i = 16 mt, k = j = 16 t
#pragma unroll
        for (int z = 0; z < 3; ++z) ldsm4(f[z], at_a<SQ_RB>(s + SM::M1 + z * SQ_BYTES, 16 * mt, 2 * t, lane));
        mma_planes<3, XS, 3>(dq0[2 * nn], dq0[2 * nn + 1], f, w);
#pragma unroll
        for (int z = 0; z < 3; ++z) ldsm4(f[z], at_a<SQ_RB>(s + SM::M2 + z * SQ_BYTES, 16 * mt, 2 * t, lane));
        mma_planes<3, XS, 3>(dk1[2 * nn], dk1[2 * nn + 1], f, w);
      }
      if (t >= mt) {   // rows j = 16 mt, k = i = 16 t: the transposes
        const uint32_t off = tile_off<SQ_RB>(16 * t + ((lane >> 4) << 3) + (lane & 7), 2 * mt + ((lane >> 3) & 1));
#pragma unroll
        for (int z = 0; z < 3; ++z) ldsm4t(f[z], s + SM::M1 + z * SQ_BYTES + off);
        mma_planes<3, XS, 3>(dk0[2 * nn], dk0[2 * nn + 1], f, w2);
#pragma unroll
        for (int z = 0; z < 3; ++z) ldsm4t(f[z], s + SM::M2 + z * SQ_BYTES + off);
        mma_planes<3, XS, 3>(dk1[2 * nn], dk1[2 * nn + 1], f, w);
      }
    }
  }
  // column sums of Y, then its row prefixes with beta (in place, a row per warp and step)
  float* Y = reinterpret_cast<float*>(smem + SM::Y);
  {
    const int j = tid % 64, o = tid / 64;
    float v = 0.f;
#pragma unroll
    for (int i = 8 * o; i < 8 * o + 8; ++i) v += Y[i * 65 + j];
    seg[o * Q + j] = v;
  }
  __syncthreads();
  {
    const float b0 = gt.beta[2 * lane], b1 = gt.beta[2 * lane + 1];
    float y0[4], y1[4], v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float* row = Y + (warp + 16 * k) * 65 + 2 * lane;
      y0[k] = row[0] * b0;
      y1[k] = row[1] * b1;
      v[k] = y0[k] + y1[k];
    }
#pragma unroll
    for (int x = 1; x < 32; x <<= 1)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float u = __shfl_up_sync(0xffffffffu, v[k], x);
        if (lane >= x) v[k] += u;
      }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float before = __shfl_up_sync(0xffffffffu, v[k], 1);
      float* row = Y + (warp + 16 * k) * 65 + 2 * lane;
      row[0] = (lane ? before : 0.f) + y0[k];
      row[1] = v[k];
    }
  }
  // dQ, dK: two adjacent columns a store
#pragma unroll
  for (int j = 0; j < NTQ; ++j)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int i = 16 * mt + pr + 8 * r, n = 8 * (qt * NTQ + j) + q2;
      if (i >= rows || n >= a.N) continue;
      const float vq[2] = {dq0[j][2 * r], dq0[j][2 * r + 1]};
      const float vk[2] = {dk0[j][2 * r] - dk1[j][2 * r], dk0[j][2 * r + 1] - dk1[j][2 * r + 1]};
      const bool two = n + 1 < a.N;
      if (a.dk_part) {
        const int64_t at = ((b * a.L + t0 + i) * a.H + h) * (int64_t)a.N + n;
        if (a.N % 2 == 0) {
          *reinterpret_cast<float2*>(a.dq_part + at) = make_float2(vq[0], vq[1]);
          *reinterpret_cast<float2*>(a.dk_part + at) = make_float2(vk[0], vk[1]);
        } else {
          for (int e = 0; e <= (int)two; ++e) {
            a.dq_part[at + e] = vq[e];
            a.dk_part[at + e] = vk[e];
          }
        }
      } else {   // one value head a key head
        const int64_t at = (b * a.L + t0 + i) * sk + (int64_t)g * a.N + n;
        for (int e = 0; e <= (int)two; ++e) {
          stf((T*)a.dC + at + e, vq[e]);
          stf((T*)a.dB + at + e, vk[e]);
        }
      }
    }
  __syncthreads();
  {
    const int t = tid / 8, o = tid % 8;   // eight threads a token
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int i = 8 * o + k;
      if (i >= t) v += (va[i] + va[Q + i]) + (va[2 * Q + i] + va[3 * Q + i]) + (t > 0 ? Y[i * 65 + t - 1] : 0.f);
      else v += (vb[i] + vb[Q + i]) + (vb[2 * Q + i] + vb[3 * Q + i]);
    }
#pragma unroll
    for (int x = 1; x < 8; x <<= 1) v += __shfl_xor_sync(0xffffffffu, v, x);
    float da = 0.f;
    if (o == 0) {
      float d = 0.f;
      for (int k = 0; k < GT / 32; ++k) d += red[k];
      const float dl = t < rows ? v + gt.eg[Q - 1] * d : 0.f;
      const float ea = expf(a.A_log[h]);
      if (t < rows) {
        const int64_t at = (b * a.L + t0 + t) * a.H + h;
        float db = (vw[t] + vw[Q + t]) + (vw[2 * Q + t] + vw[3 * Q + t]);
        for (int k = 0; k < 8; ++k) db += seg[k * Q + t];
        a.ddt[at] = -ea * dl;
        a.dbeta[at] = db;
        // dA_log: dl times the log-decay, which is bounded as the forward bounds it
        da = dl * fmaxf(-ea * a.dt[at], -139.f);
      }
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) da += __shfl_xor_sync(0xffffffffu, da, x);
    __syncthreads();
    if (lane == 0) red[warp] = da;
  }
  __syncthreads();
  if (tid == 0) {
    float d = 0.f;
    for (int k = 0; k < GT / 32; ++k) d += red[k];
    a.da_part[bh * a.nc + c] = d;
  }
}

// dB, dC [rows, G, N] io: the sums over a key head's H / G value heads.
template <typename T>
__global__ void __launch_bounds__(256) delta_head_sum_kernel(const float* __restrict__ pk, const float* __restrict__ pq,
                                                             T* __restrict__ dB, T* __restrict__ dC, int64_t n, int G,
                                                             int rep, int N) {
  let_next_start();
  wait_for_previous();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const int64_t row = i / N;   // (token, key head)
  const int64_t at = row * rep * N + (i - row * N);
  float k = 0.f, q = 0.f;
  for (int r = 0; r < rep; ++r) {
    k += pk[at + (int64_t)r * N];
    q += pq[at + (int64_t)r * N];
  }
  stf(dB + i, k);
  stf(dC + i, q);
}

// dA_log [H]: a block per head sums its batch rows' chunks in a fixed order, in 64 bits
// (the terms are of either sign).
__global__ void __launch_bounds__(256) delta_da_kernel(const float* __restrict__ part, float* __restrict__ out,
                                                       int64_t Bt, int H, int64_t nc) {
  let_next_start();
  wait_for_previous();
  __shared__ double sm[256];
  double v = 0.0;
  for (int64_t i = threadIdx.x; i < Bt * nc; i += 256) {
    const int64_t b = i / nc;
    v += (double)part[(b * H + blockIdx.x) * nc + (i - b * nc)];
  }
  sm[threadIdx.x] = v;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if (threadIdx.x < o) sm[threadIdx.x] += sm[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) out[blockIdx.x] = (float)sm[0];
}

// ------------------------------------------------------------------ host side
template <int XS, int KN, int NCW>
int launch_chain(BwdArgs a, cudaStream_t st) {
  constexpr int bytes = ChainSmem<XS, KN, NCW>::BYTES;
  static_assert(bytes <= 232448, "shared-memory layout exceeds the per-block limit");
  auto kern = delta_bwd_chain_kernel<XS, KN, NCW>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return check_launch("gated_delta_rule_bwd: set smem attribute");
  a.npb = (int)cdiv(a.P, 16 * NCW);
  TSSM_REQUIRE(a.Bt * a.H * a.npb < (int64_t(1) << 31), "gated_delta_rule_bwd: size out of range");
  launch_next(kern, (unsigned)(a.Bt * a.H * a.npb), (NCW + 4) * 32, bytes, st, a);
  return check_launch("gated_delta_rule_bwd: chain");
}

template <int XS, int KN>
int launch_grad(const BwdArgs& a, cudaStream_t st) {
  constexpr int bytes = GradSmem<XS, KN>::BYTES;
  static_assert(bytes <= 232448, "shared-memory layout exceeds the per-block limit");
  auto kern = delta_bwd_grad_kernel<XS, KN>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return check_launch("gated_delta_rule_bwd: set smem attribute");
  TSSM_REQUIRE(a.Bt * a.H * a.nc < (int64_t(1) << 31), "gated_delta_rule_bwd: size out of range");
  launch_next(kern, (unsigned)(a.Bt * a.H * a.nc), GT, bytes, st, a);
  return check_launch("gated_delta_rule_bwd: gradients");
}

template <int XS, int KN>
int launch_all(BwdArgs a, bool tc, cudaStream_t st) {
  using T = typename std::conditional<XS == 1, __nv_bfloat16, float>::type;
  if (a.nc == 0) {   // no tokens: the state's gradient passes through
    const size_t n = (size_t)(a.Bt * a.H * a.P) * a.N * 4;
    if ((a.dh_last ? cudaMemcpyAsync(a.dh0, a.dh_last, n, cudaMemcpyDeviceToDevice, st) : cudaMemsetAsync(a.dh0, 0, n, st)) !=
        cudaSuccess)
      return check_launch("gated_delta_rule_bwd: pass the state's gradient");
  } else if (tc) {
    const TcBackCall t{a.B, a.C, a.dy, a.A_log, a.dt, a.beta, a.dh_last, a.dh0, a.dstates, a.derrs, a.gates,
                       a.img, a.Bt, a.L, a.H, a.G, a.P, a.N, a.scale};
    if (int e = tc_back_run(t, st)) return e;
  } else {
    const bool wide = a.P > 64 && a.Bt * a.H * cdiv(a.P, 128) >= num_sms();
    const int64_t seg = segment_chunks(a.Bt * a.H, a.nc);
    for (int64_t end = a.nc; end > 0; end -= seg) {   // segments from the last; dh0 carries the state's gradient
      a.c0 = std::max<int64_t>(0, end - seg);
      a.nseg = end - a.c0;
      a.ds_in = end == a.nc ? a.dh_last : a.dh0;
      const PrepCall p{a.B, a.C, a.A_log, a.dt, a.beta, a.img, a.gates, a.Bt, a.L, a.H, a.G, a.N, a.c0, a.nseg, a.nc,
                       a.scale, a.vec_kq};
      if (int e = prep_run(p, XS == 1 ? TSSM_BF16 : TSSM_F32, st)) return e;
      if (int e = wide ? launch_chain<XS, KN, 8>(a, st) : launch_chain<XS, KN, 4>(a, st)) return e;
    }
  }
  if (a.nc > 0) {
    if (tc_grad_takes(a.H, a.G, a.N, tc)) {   // key heads summed as well
      const TcGradCall t{a.B, a.C, a.dy, a.A_log, a.dt, a.states, a.errs, a.dstates, a.derrs, a.gates, a.du, a.dB, a.dC, a.ddt,
                         a.dbeta, a.da_part, a.Bt, a.L, a.H, a.G, a.P, a.nc, a.scale, nullptr};
      if (int e = tc_grad_run(t, st)) return e;
    } else {
      if (int e = launch_grad<XS, KN>(a, st)) return e;
      if (a.dk_part) {
        const int64_t n = a.Bt * a.L * a.G * a.N;
        TSSM_REQUIRE(cdiv(n, 256) < (int64_t(1) << 31), "gated_delta_rule_bwd: size out of range");
        launch_next(delta_head_sum_kernel<T>, (unsigned)cdiv(n, 256), 256, 0, st, (const float*)a.dk_part,
                    (const float*)a.dq_part, (T*)a.dB, (T*)a.dC, n, a.G, a.H / a.G, a.N);
      }
    }
  }
  launch_next(delta_da_kernel, (unsigned)a.H, 256, 0, st, (const float*)a.da_part, a.dA_log, a.Bt, a.H, a.nc);
  return check_launch("gated_delta_rule_bwd");
}

// Workspace in floats: dS1 of every chunk, dE, per-head dK and dQ (shared key heads that the gradient
// kernel does not sum itself), dA parts, gates, a segment's images.
struct BwdSpace {
  int64_t dstates, derrs, part, da, gates, img, total;
};
BwdSpace space(int64_t Bt, int64_t L, int64_t H, int64_t G, int64_t P, int64_t N, bool tc) {   // tc: the chain is delta_tc.cu's
  auto up = [](int64_t n) { return (n + 3) / 4 * 4; };
  const int64_t nc = cdiv(L, delta::Q);
  BwdSpace s;
  s.dstates = Bt * H * nc * saved_floats(P, N);
  s.derrs = Bt * H * saved_floats(P, L);
  s.part = H == G || tc_grad_takes(H, G, N, tc) ? 0 : up(Bt * L * H * N);
  s.da = up(Bt * H * nc);
  s.img = Bt * nc ? Bt * H * segment_chunks(Bt * H, nc) * prep_image_bytes() / 4 : 0;
  s.gates = Bt * H * nc * (int64_t)(sizeof(Gates) / 4);
  s.total = s.dstates + s.derrs + 2 * s.part + s.da + s.gates + s.img;
  return s;
}

}  // namespace
}  // namespace delta
}  // namespace tssm

extern "C" int64_t tssm_gated_delta_rule_bwd_workspace_size(int64_t Bt, int64_t L, int64_t H, int64_t G, int64_t P,
                                                            int64_t N) {
  if (Bt <= 0 || L <= 0 || H <= 0 || G <= 0 || P <= 0 || N <= 0) return 0;
  return tssm::delta::space(Bt, L, H, G, P, N, false).total * 4;
}

extern "C" int64_t tssm_gated_delta_rule_bwd_workspace_size_dtype(int64_t Bt, int64_t L, int64_t H, int64_t G, int64_t P,
                                                                  int64_t N, int dtype) {
  if (Bt <= 0 || L <= 0 || H <= 0 || G <= 0 || P <= 0 || N <= 0) return 0;
  return tssm::delta::space(Bt, L, H, G, P, N, tssm::delta::tc_takes(P, N, dtype)).total * 4;
}

extern "C" int tssm_gated_delta_rule_bwd(const void* u, const void* A_log, const void* B, const void* C, const void* dt,
                                         const void* beta, const void* dy, const void* states, const void* errors,
                                         const void* dh_last, void* du, void* dA_log, void* dB, void* dC, void* ddt,
                                         void* dbeta, void* dh0, void* workspace, int64_t workspace_bytes, int64_t Bt,
                                         int64_t L, int64_t H, int64_t G, int64_t P, int64_t N, double scale,
                                         int dtype, tssm_stream_t stream) {
  using namespace tssm;
  using namespace tssm::delta;
  TSSM_REQUIRE(Bt >= 0 && L >= 0 && H >= 0 && G >= 0 && P >= 0 && N >= 0, "gated_delta_rule_bwd: negative size");
  TSSM_REQUIRE(N >= 1 && N <= 128, "gated_delta_rule_bwd: state size N must be 1 to 128 (got %lld)", (long long)N);
  TSSM_REQUIRE(H >= 1 && P >= 1 && G >= 1 && H % G == 0,
               "gated_delta_rule_bwd: H (%lld) must be a positive multiple of the key heads G (%lld)", (long long)H,
               (long long)G);
  TSSM_REQUIRE(dtype == TSSM_F32 || dtype == TSSM_BF16, "gated_delta_rule_bwd: dtype must be f32 or bf16 (got %d)", dtype);
  TSSM_REQUIRE(L < (int64_t(1) << 31) && Bt < (int64_t(1) << 31) && H <= 1 << 20 && P <= 1 << 20 &&
                   Bt * H * std::max(cdiv(L, delta::Q), cdiv(P, 16)) < (int64_t(1) << 31),
               "gated_delta_rule_bwd: size out of range");
  TSSM_REQUIRE(A_log && dA_log && (Bt == 0 || dh0), "gated_delta_rule_bwd: null pointer");
  TSSM_REQUIRE(Bt * L == 0 || (u && B && C && dt && beta && dy && states && errors && du && dB && dC && ddt && dbeta),
               "gated_delta_rule_bwd: null pointer");
  const uintptr_t bases = reinterpret_cast<uintptr_t>(B) | reinterpret_cast<uintptr_t>(C) | reinterpret_cast<uintptr_t>(dy) |
                          reinterpret_cast<uintptr_t>(dh_last) | reinterpret_cast<uintptr_t>(dh0) |
                          reinterpret_cast<uintptr_t>(du) | reinterpret_cast<uintptr_t>(dB) | reinterpret_cast<uintptr_t>(dC);
  const bool tc = tc_takes(P, N, dtype) && (bases & 15u) == 0;
  const BwdSpace sp = space(Bt, L, H, G, P, N, tc);
  const int64_t need = sp.total * 4;
  TSSM_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned16(workspace)),
               "gated_delta_rule_bwd: workspace of %lld bytes (16-byte aligned) needed, %lld given", (long long)need,
               (long long)workspace_bytes);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (Bt == 0) {
    if (cudaMemsetAsync(dA_log, 0, H * 4, st) != cudaSuccess) return check_launch("gated_delta_rule_bwd: clear");
    return TSSM_OK;
  }
  TSSM_REQUIRE(Bt * L == 0 || (aligned16(states) && aligned16(errors)),
               "gated_delta_rule_bwd: states and errors must be 16-byte aligned");
  BwdArgs a{};
  a.u = u; a.B = B; a.C = C; a.dy = dy;
  a.A_log = (const float*)A_log; a.dt = (const float*)dt; a.beta = (const float*)beta;
  a.states = (const float*)states; a.errs = (const float*)errors; a.dh_last = (const float*)dh_last;
  a.du = du; a.dB = dB; a.dC = dC;
  a.dA_log = (float*)dA_log; a.ddt = (float*)ddt; a.dbeta = (float*)dbeta; a.dh0 = (float*)dh0;
  a.dstates = (float*)workspace;
  a.derrs = a.dstates + sp.dstates;
  a.dk_part = sp.part ? a.derrs + sp.derrs : nullptr;
  a.dq_part = sp.part ? a.dk_part + sp.part : nullptr;
  a.da_part = a.derrs + sp.derrs + 2 * sp.part;
  a.gates = (Gates*)(a.da_part + sp.da);
  a.img = (uint8_t*)(a.da_part + sp.da + sp.gates);
  a.Bt = Bt; a.L = L; a.H = (int)H; a.G = (int)G; a.P = (int)P; a.N = (int)N;
  a.nc = cdiv(L, delta::Q);
  a.scale = (float)scale;
  const int per = dtype == TSSM_F32 ? 4 : 8;
  a.vec_kq = N % per == 0 && aligned16(B) && aligned16(C);
  a.vec_v = P % per == 0 && aligned16(dy);
  if (dtype == TSSM_F32) return N <= 64 ? launch_all<3, 64>(a, tc, st) : launch_all<3, 128>(a, tc, st);
  return N <= 64 ? launch_all<1, 64>(a, tc, st) : launch_all<1, 128>(a, tc, st);
}
