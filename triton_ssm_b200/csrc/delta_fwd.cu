// Chunked gated delta rule, forward (formulas and precision: delta.cuh).
//
// A block walks one (batch row, head) and 16 NCW value channels through the
// sequence, 64 tokens at a time.  Value channels never mix, so each of the NCW
// chain warps owns 16 of them and carries its state S^T [16 x N] in registers:
//     KS^T = S^T K^T,  X^T = V^T - exp(l) KS^T,  E^T = X^T T^T,
//     O^T  = scale exp(l) S^T Q^T + E^T (Aq diag(beta))^T,
//     S^T  = exp(l_last) S^T + (E diag(w beta))^T K
// Transposed, every product's result has the register layout of the next one's
// left operand, so the chain needs no shared memory and no barrier; K, Q, T and
// Aq are shared by the warps as right operands.  T and Aq come from delta_prep.cu;
// four more warps load the next chunk meanwhile (bf16; f32 tiles fill the shared
// memory, so there all warps load between chunks).  mma.sync gives a quarter of
// tcgen05's rate here (1024 of 4096 multiply-adds a cycle and SM): this kernel is
// for f32 and for shapes and addresses that delta_tc.cu does not take.
#include "delta.cuh"
#include "delta_tc.h"

namespace tssm {
namespace delta {
namespace {

// XS: planes of an io value (1: bf16, 3: f32).  KN: N padded to 64 or 128.  NCW: chain warps.
template <int XS, int KN, int NCW>
struct FwdSmem {
  static constexpr int BUFS = XS == 1 ? 2 : 1;
  static constexpr int PB = 16 * NCW;                    // value channels of the block
  static constexpr int PLANE = Q * KN * 2;
  static constexpr int VROW = XS == 1 ? PB * 2 : (PB + 4) * 4;   // f32 values: padded rows
  static constexpr int K = 0, QQ = K + XS * PLANE, V = QQ + XS * PLANE, T = V + Q * VROW, AQ = T + 3 * SQ_BYTES,
                       G = AQ + 3 * SQ_BYTES, BUF = (G + (int)sizeof(Gates) + 127) / 128 * 128;   // T, AQ, G: an image
  static constexpr int BYTES = BUFS * BUF + 128;
};

struct FwdArgs {
  const void *u, *B, *C;
  const uint8_t* img;
  const float* h_in;
  void* y;
  float *h_out, *states, *errs;
  int64_t L, c0, nseg, nc;   // first chunk and chunks of the segment; all chunks
  int H, G, P, N, npb;
  float scale;
  int vec_kq, vec_v;
};

template <int XS, int KN, int NCW>
__global__ void __launch_bounds__((NCW + 4) * 32, 1) delta_fwd_kernel(const FwdArgs a) {
  let_next_start();
  wait_for_previous();
  using T = typename std::conditional<XS == 1, __nv_bfloat16, float>::type;
  using SM = FwdSmem<XS, KN, NCW>;
  constexpr int PB = SM::PB, RB = KN * 2, NT = KN / 8, NS = 3;
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
  const T* vp = (const T*)a.u + (b * a.L) * su + (int64_t)h * a.P + pb;
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
    if constexpr (XS == 1) {
      load_planes<1, PB, LT>(s + SM::V, 0, vp + t0 * su, su, rows, pvalid, a.vec_v, t);
    } else {
      float* vs = reinterpret_cast<float*>(buf + SM::V);
      if (a.vec_v) {
#pragma unroll 4
        for (int i = t; i < Q * PB / 4; i += LT) {
          const int r = i / (PB / 4), p = i % (PB / 4) * 4;
          const bool in = r < rows && p < pvalid;
          cp_async16(s + SM::V + (r * (PB + 4) + p) * 4, in ? vp + (t0 + r) * su + p : vp, in);
        }
      } else {
#pragma unroll 4
        for (int i = t; i < Q * PB; i += LT) {
          const int r = i / PB, p = i % PB;
          vs[r * (PB + 4) + p] = r < rows && p < pvalid ? ldf(vp + (t0 + r) * su + p) : 0.f;
        }
      }
    }
    cp_async_wait_all();
  };

  // ---- chain state
  const int p0 = 16 * warp;   // of the block's channels
  const int pr = lane / 4, q2 = 2 * (lane % 4);
  float S[NT][4];
  const int64_t srow = (bh * a.P + pb + p0 + pr) * (int64_t)a.N;   // of h_in, h_out
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
    if (a.states) {
      float* dst = a.states + (bh * a.nc + a.c0 + c) * saved_floats(a.P, a.N);
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int r = 0; r < 2; ++r)   // columns beyond N are 0
          if (8 * j + q2 < (a.N + 3) / 4 * 4 && pb + p0 + pr + 8 * r < a.P)
            *saved_pair(dst, a.P, pb + p0 + pr + 8 * r, 8 * j + q2) = make_float2(S[j][2 * r], S[j][2 * r + 1]);
    }
    // KS^T, then X^T
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
    for (int np = 0; np < 4; ++np) {
      float v[2][4];
      if constexpr (XS == 1) {
        uint32_t w[4];
        ldsm4t(w, s + SM::V + tile_off<PB * 2>(16 * np + ((lane >> 4) << 3) + (lane & 7), p0 / 8 + ((lane >> 3) & 1)));
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          v[m >> 1][(m & 1) * 2] = lo2(w[m]);
          v[m >> 1][(m & 1) * 2 + 1] = hi2(w[m]);
        }
      } else {
        const float* vs = reinterpret_cast<const float*>(buf + SM::V) + p0 + pr;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[m][e] = vs[(16 * np + 8 * m + q2 + (e & 1)) * (PB + 4) + (e >> 1) * 8];
      }
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const float2 eg = *reinterpret_cast<const float2*>(gt.eg + 16 * np + 8 * m + q2);
        float(&xx)[4] = x[2 * np + m];
        xx[0] = v[m][0] - eg.x * xx[0];
        xx[1] = v[m][1] - eg.y * xx[1];
        xx[2] = v[m][2] - eg.x * xx[2];
        xx[3] = v[m][3] - eg.y * xx[3];
      }
    }
    // E^T = X^T T^T (T lower triangular: 16-blocks i >= j)
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
      for (int np = t; np < 4; ++np) {
        uint32_t w[NS][4];
#pragma unroll
        for (int z = 0; z < NS; ++z) ldsm4(w[z], at_b<SQ_RB>(s + SM::T + z * SQ_BYTES, 16 * np, 2 * t, lane));
        mma_planes<NS, NS, NS>(er[2 * np], er[2 * np + 1], f, w);
      }
    }
    if (a.errs) {
      float* ep = a.errs + bh * saved_floats(a.P, a.L);
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int r = 0; r < 2; ++r) {   // groups of four tokens that reach the end; behind it e = 0
          const int tk = 8 * i + q2, p = p0 + pr + 8 * r;
          if ((tk & ~3) < rows && p < pvalid)
            *saved_pair(ep, a.P, pb + p, t0 + tk) = make_float2(er[i][2 * r], er[i][2 * r + 1]);
        }
    }
    // O^T: the state's part (x is free now), then the chunk's own
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
        for (int z = 0; z < XS; ++z) ldsm4(w[z], at_b<RB>(s + SM::QQ + z * SM::PLANE, 16 * np, 2 * kk, lane));
        mma_planes<NS, XS, NS, XS == 3>(x[2 * np], x[2 * np + 1], f, w);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 eg = *reinterpret_cast<const float2*>(gt.eg + 8 * i + q2);
      x[i][0] *= a.scale * eg.x;
      x[i][1] *= a.scale * eg.y;
      x[i][2] *= a.scale * eg.x;
      x[i][3] *= a.scale * eg.y;
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      uint32_t f[NS][4];
      split_a<NS>(er[2 * t], er[2 * t + 1], f);
#pragma unroll
      for (int np = t; np < 4; ++np) {
        uint32_t w[NS][4];
#pragma unroll
        for (int z = 0; z < NS; ++z) ldsm4(w[z], at_b<SQ_RB>(s + SM::AQ + z * SQ_BYTES, 16 * np, 2 * t, lane));
        mma_planes<NS, NS, NS>(x[2 * np], x[2 * np + 1], f, w);
      }
    }
    // y: through this warp's own columns of the value tile (bf16), one 16-byte piece a lane
    T* yp = (T*)a.y + (b * a.L + t0) * su + (int64_t)h * a.P + pb;
    if constexpr (XS == 1) {
      __syncwarp();
#pragma unroll
      for (int np = 0; np < 4; ++np) {
        const uint32_t w[4] = {pack2(x[2 * np][0], x[2 * np][1]), pack2(x[2 * np][2], x[2 * np][3]),
                               pack2(x[2 * np + 1][0], x[2 * np + 1][1]), pack2(x[2 * np + 1][2], x[2 * np + 1][3])};
        stsm4t(s + SM::V + tile_off<PB * 2>(16 * np + ((lane >> 4) << 3) + (lane & 7), p0 / 8 + ((lane >> 3) & 1)), w);
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = i * 16 + lane / 2, c8 = lane % 2;
        const uint4 v = *reinterpret_cast<const uint4*>(buf + SM::V + tile_off<PB * 2>(r, p0 / 8 + c8));
        const int p = p0 + 8 * c8;
        if (r >= rows || p >= pvalid) continue;
        if (a.vec_v) {
          *reinterpret_cast<uint4*>(yp + (int64_t)r * su + p) = v;
        } else {
          const uint32_t vv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (p + e < pvalid) stf(yp + (int64_t)r * su + p + e, e & 1 ? hi2(vv[e / 2]) : lo2(vv[e / 2]));
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int tk = 8 * i + q2 + (e & 1), p = p0 + pr + (e >> 1) * 8;
          if (tk < rows && p < pvalid) stf(yp + (int64_t)tk * su + p, x[i][e]);
        }
    }
    // S^T = exp(l_last) S^T + (E diag(w beta))^T K
    const float el = gt.eg[Q - 1];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) S[j][e] *= el;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const float2 wb = *reinterpret_cast<const float2*>(gt.wb + 16 * t + 8 * m + q2);
        float(&ee)[4] = er[2 * t + m];
        ee[0] *= wb.x;
        ee[1] *= wb.y;
        ee[2] *= wb.x;
        ee[3] *= wb.y;
      }
      uint32_t f[NS][4];
      split_a<NS>(er[2 * t], er[2 * t + 1], f);
#pragma unroll
      for (int nn = 0; nn < KN / 16; ++nn) {
        uint32_t w[XS][4];
#pragma unroll
        for (int z = 0; z < XS; ++z) ldsm4t(w[z], at_a<RB>(s + SM::K + z * SM::PLANE, 16 * t, 2 * nn, lane));
        mma_planes<NS, XS, NS, true>(S[2 * nn], S[2 * nn + 1], f, w);
      }
    }
  };

  if (warp < NCW) state_io(nullptr, a.h_in ? a.h_in + srow : nullptr);
  if constexpr (SM::BUFS == 2) {
    if (warp >= NCW) load(0);
    __syncthreads();
    for (int64_t c = 0; c < a.nseg; ++c) {
      if (warp < NCW) chain(c);
      else if (c + 1 < a.nseg) load(c + 1);
      __syncthreads();
    }
  } else {
    for (int64_t c = 0; c < a.nseg; ++c) {
      load(c);
      __syncthreads();
      if (warp < NCW) chain(c);
      __syncthreads();
    }
  }
  if (warp < NCW && a.h_out) state_io(a.h_out + srow, nullptr);
}

template <int XS, int KN, int NCW>
int launch(FwdArgs a, int64_t Bt, cudaStream_t st) {
  constexpr int bytes = FwdSmem<XS, KN, NCW>::BYTES;
  static_assert(bytes <= 232448, "shared-memory layout exceeds the per-block limit");
  auto kern = delta_fwd_kernel<XS, KN, NCW>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return check_launch("gated_delta_rule: set smem attribute");
  a.npb = (int)cdiv(a.P, 16 * NCW);
  const int64_t blocks = Bt * a.H * a.npb;
  TSSM_REQUIRE(blocks < (int64_t(1) << 31), "gated_delta_rule: size out of range");
  launch_next(kern, (unsigned)blocks, (NCW + 4) * 32, bytes, st, a);
  return check_launch("gated_delta_rule");
}

template <int XS, int KN>
int by_block(const FwdArgs& a, int64_t Bt, cudaStream_t st) {
  // 128 channels a block when that still fills the SMs, else 64
  if (a.P > 64 && Bt * a.H * cdiv(a.P, 128) >= num_sms()) return launch<XS, KN, 8>(a, Bt, st);
  return launch<XS, KN, 4>(a, Bt, st);
}

}  // namespace
}  // namespace delta
}  // namespace tssm

extern "C" int64_t tssm_gated_delta_rule_workspace_size(int64_t Bt, int64_t L, int64_t H, int64_t G, int64_t P,
                                                        int64_t N, int dtype) {
  using namespace tssm;
  using namespace tssm::delta;
  if (Bt <= 0 || L <= 0 || H <= 0 || G <= 0 || P <= 0 || N <= 0) return 0;
  const int64_t streams = Bt * H, nc = cdiv(L, delta::Q), seg = segment_chunks(streams, nc);
  return streams * seg * prep_image_bytes() + (seg < nc ? streams * P * N * 4 : 0);
}

extern "C" int tssm_gated_delta_rule(const void* u, const void* A_log, const void* B, const void* C, const void* dt,
                                     const void* beta, const void* h0, void* y, void* h_last, void* states,
                                     void* errors, void* workspace, int64_t workspace_bytes, int64_t Bt, int64_t L,
                                     int64_t H, int64_t G, int64_t P, int64_t N, double scale, int dtype,
                                     tssm_stream_t stream) {
  using namespace tssm;
  using namespace tssm::delta;
  TSSM_REQUIRE(Bt >= 0 && L >= 0 && H >= 0 && G >= 0 && P >= 0 && N >= 0, "gated_delta_rule: negative size");
  if (Bt * H * P == 0) return TSSM_OK;
  TSSM_REQUIRE(N >= 1 && N <= 128, "gated_delta_rule: state size N must be 1 to 128 (got %lld)", (long long)N);
  TSSM_REQUIRE(G >= 1 && H % G == 0, "gated_delta_rule: H (%lld) must be a multiple of the key heads G (%lld)",
               (long long)H, (long long)G);
  TSSM_REQUIRE(A_log && (L == 0 || (u && B && C && dt && beta && y)), "gated_delta_rule: null pointer");
  TSSM_REQUIRE((states != nullptr) == (errors != nullptr), "gated_delta_rule: states and errors go together");
  TSSM_REQUIRE(dtype == TSSM_F32 || dtype == TSSM_BF16, "gated_delta_rule: dtype must be f32 or bf16 (got %d)", dtype);
  TSSM_REQUIRE(L < (int64_t(1) << 31) && Bt < (int64_t(1) << 31) && H <= 1 << 20 && P <= 1 << 20 &&
                   Bt * H * std::max(cdiv(L, delta::Q), cdiv(P, 16)) < (int64_t(1) << 31),
               "gated_delta_rule: size out of range");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const uintptr_t bases = reinterpret_cast<uintptr_t>(u) | reinterpret_cast<uintptr_t>(B) |
                          reinterpret_cast<uintptr_t>(C) | reinterpret_cast<uintptr_t>(y) |
                          reinterpret_cast<uintptr_t>(h0) | reinterpret_cast<uintptr_t>(h_last) |
                          reinterpret_cast<uintptr_t>(states) | reinterpret_cast<uintptr_t>(errors);
  const int64_t need = tssm_gated_delta_rule_workspace_size(Bt, L, H, G, P, N, dtype);
  TSSM_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned16(workspace)),
               "gated_delta_rule: workspace of %lld bytes (16-byte aligned) needed, %lld given", (long long)need,
               (long long)workspace_bytes);
  const int64_t streams = Bt * H, nc = cdiv(L, delta::Q);
  if (nc == 0) {   // no tokens: the state passes through
    if (!h_last || h_last == h0) return TSSM_OK;
    const size_t bytes = (size_t)(streams * P * N) * 4;
    if ((h0 ? cudaMemcpyAsync(h_last, h0, bytes, cudaMemcpyDeviceToDevice, st) : cudaMemsetAsync(h_last, 0, bytes, st)) !=
        cudaSuccess)
      return check_launch("gated_delta_rule: pass the state");
    return TSSM_OK;
  }
  const int64_t seg = segment_chunks(streams, nc);
  uint8_t* img = (uint8_t*)workspace;
  float* carry = h_last ? (float*)h_last : (float*)(img + streams * seg * prep_image_bytes());
  if (tc_takes(P, N, dtype) && (bases & 15u) == 0) {
    const TcCall t{u, B, C, (const float*)A_log, (const float*)dt, (const float*)beta, (const float*)h0, y,
                   (float*)h_last, (float*)states, (float*)errors, img, carry, Bt, L, H, G, P, N, (float)scale};
    return tc_run(t, st);
  }
  const int per = dtype == TSSM_F32 ? 4 : 8;   // elements of 16 bytes
  FwdArgs a{};
  a.u = u; a.B = B; a.C = C; a.img = img;
  a.y = y; a.states = (float*)states; a.errs = (float*)errors;
  a.L = L; a.H = (int)H; a.G = (int)G; a.P = (int)P; a.N = (int)N;
  a.nc = nc;
  a.scale = (float)scale;
  a.vec_kq = N % per == 0 && aligned16(B) && aligned16(C);
  a.vec_v = P % per == 0 && aligned16(u) && aligned16(y);
  for (int64_t c0 = 0; c0 < nc; c0 += seg) {
    const int64_t m = std::min(seg, nc - c0);
    const PrepCall p{B, C, (const float*)A_log, (const float*)dt, (const float*)beta, img, nullptr, Bt, L, H, G, N, c0,
                     m, nc, (float)scale, a.vec_kq};
    if (int e = prep_run(p, dtype, st)) return e;
    a.c0 = c0; a.nseg = m;
    a.h_in = c0 ? carry : (const float*)h0;
    a.h_out = c0 + m == nc && !h_last ? nullptr : carry;
    int e;
    if (dtype == TSSM_F32) e = N <= 64 ? by_block<3, 64>(a, Bt, st) : by_block<3, 128>(a, Bt, st);
    else e = N <= 64 ? by_block<1, 64>(a, Bt, st) : by_block<1, 128>(a, Bt, st);
    if (e) return e;
  }
  return TSSM_OK;
}
