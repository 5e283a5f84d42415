// The gradients of one (chunk, head) of the gated delta rule on tcgen05 (bf16, N = 128, P a
// multiple of 64; formulas: delta_bwd.cu, where the kernel for the other shapes is).
//
// Transposed, so that the state operands have the 128 rows of a full-rate product and lie as
// they were saved ([p][n]); TMEM lane = n, column = token, f32:
//   dQ0^T = S0^T dO^T        dK0^T = S0^T dE^T       dK1^T = dS1^T E^T       (64 value channels a step)
//   dQ^T  = scale exp(l) dQ0^T + K^T M1^T
//   dK^T  = w beta dK1^T - exp(l) dK0^T + Q^T M1 - K^T M2^T - K^T M2
// with S0, dS1, E, dE, M1 and M2 in three bf16 planes (products of planes i + j < 3).  The
// state parts are scaled in place, so that the last line's products add onto them.  dO E^T and
// dE E^T (triangles of 64 x 64, in registers), q.k and k.k stay on mma.sync, which runs meanwhile.
//
// 256 threads, 111 KB and half of TMEM: two blocks an SM, each waiting for its loads while the
// other works (in registers, the three 64 x 128 accumulators leave room for one block only).
// Blocks of one key head are a cluster: each leaves its dQ, dK in shared memory and sums a share
// of the rows over all of them, in the heads' order (parts in HBM and a kernel for their sums took
// 65 us more at 64 heads x 2048 tokens).
// Measured there (2048 chunks and heads, P = 128, 16 value on 8 key heads): 270 us, 18 us for one on
// its SM, against 27 on mma.sync.  Bound by shared memory: a 128 x 64 x 16 product reads 6 KB for
// its 32 cycles, and planes, fragments and sums take about as many cycles again.  Fetching the next
// blocks' states to L2 ahead made it slower (311): their own loads queued behind that.
// K and Q come last, where dE and dO were.
//
// Every wait on an mbarrier is bounded.  A block that gives up sets the status word and goes on
// without waiting; it writes no ddt, dbeta and dA_log behind that, and no block of its cluster writes
// dB and dC, which would hold its part.
#include "delta.cuh"
#include "delta_tc.h"
#include "tcgen05.cuh"

namespace tssm {
namespace delta {
namespace {
using namespace sm100;

constexpr int NT = 256, N = 128, TILE = SQ_BYTES, PLANE = 2 * TILE;   // a plane of 64 rows x 128: two tiles
constexpr int S = 0, E = S + 3 * PLANE, DE = E + 3 * TILE, DO = DE + 3 * TILE, G = DO + TILE,
              VEC = G + (int)sizeof(Gates), BAR = VEC + (3 * 4 * Q + 4 * Q + 8) * 4, BYTES = BAR + 64 + 1024;
constexpr int K = DE, QQ = K + PLANE;                            // when the last channels' dE, dO have been read
constexpr int M1 = S, M2 = S + 3 * TILE, Y = S + 6 * TILE;       // after the products over p; Y: 64 x 65 floats
constexpr int OUT = S;                                           // last: dQ, dK [64][128] f32
static_assert(QQ + PLANE == G && Y + Q * 65 * 4 <= K && OUT + 2 * Q * N * 4 <= G && BAR % 8 == 0, "regions");
static_assert(2 * (BYTES + 1024) <= 233472, "two blocks an SM");
constexpr uint32_t C_Q = 0, C_K = 64, C_K1 = 128, COLS = 256;

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ld_peer(uint32_t addr, uint32_t rank) {   // from a block of the cluster
  float4 v;
  asm volatile(
      "{\n\t.reg .b32 p;\n\tmapa.shared::cluster.u32 p, %4, %5;\n\t"
      "ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [p];\n\t}"
      : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr), "r"(rank) : "memory");
  return v;
}
__device__ __forceinline__ int ld_peer_int(uint32_t addr, uint32_t rank) {
  int v;
  asm volatile(
      "{\n\t.reg .b32 p;\n\tmapa.shared::cluster.u32 p, %1, %2;\n\tld.shared::cluster.s32 %0, [p];\n\t}"
      : "=r"(v) : "r"(addr), "r"(rank) : "memory");
  return v;
}

// Sums over a warp's lanes of 16 values each: lanes 2 i, 2 i + 1 get the sum of v[i] (v is used up).
__device__ __forceinline__ float lanes_sum16(float (&v)[16], int lane) {
#pragma unroll
  for (int o = 16, n = 8; n >= 1; o >>= 1, n >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float keep = up ? v[i + n] : v[i], send = up ? v[i] : v[i + n];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
  return v[0] + __shfl_xor_sync(0xffffffffu, v[0], 1);
}

__global__ void __launch_bounds__(NT, 2) delta_grad_tc_kernel(const TcGradCall a) {
  let_next_start();
  using T = __nv_bfloat16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t s = smem_u32(smem);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int mt = warp % 4, qh = warp / 4, pr = lane / 4, q2 = 2 * (lane % 4);   // 16 tokens, a half of the others
  const int rep = (int)(a.H / a.G), P = (int)a.P;
  const uint32_t rank = blockIdx.x % rep;   // of the key head's cluster
  const uint32_t bgc = blockIdx.x / rep, bg = bgc / (uint32_t)a.nc, c = bgc - bg * (uint32_t)a.nc, bi = bg / (uint32_t)a.G;
  const int g = (int)(bg - bi * (uint32_t)a.G), h = g * rep + (int)rank;
  const int64_t b = bi;
  const uint32_t bhc = (bi * (uint32_t)a.H + h) * (uint32_t)a.nc + c;   // (batch row, head, chunk): below 2^31
  const int t0 = (int)(c * Q), rows = (int)min((int64_t)Q, a.L - t0);
  const int64_t su = a.H * a.P, sk = a.G * N;
  const Gates& gt = *reinterpret_cast<const Gates*>(smem + G);
  float* vec = reinterpret_cast<float*>(smem + VEC);
  float *va = vec, *vb = vec + 4 * Q, *vw = vec + 8 * Q;   // [4][Q] row dots of a, b, and w e.(K dS1), by quarter of N
  float* seg = vec + 12 * Q;                               // [4][Q] column sums of Y by row quarter
  float* red = seg + 4 * Q;                                // [8] <S0, dS1> by warp

  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + BAR);
  uint64_t *adone = bar, *bdone = bar + 1, *mdone = bar + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bar + 5);
  if (tid == 0) {
    mbar_init(adone, 1);
    mbar_init(bdone, 1);
    mbar_init(mdone, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  __syncwarp();
  if (warp == 0) {
    tmem_alloc(tmem_slot, COLS);
    tmem_relinquish();
  }
  if (tid < (int)(sizeof(Gates) / 16))
    cp_async16(s + G + 16 * tid, reinterpret_cast<const uint4*>((const Gates*)a.gates + bhc) + tid, true);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto wait = [&](uint64_t* m, int phase, int code) {
    const bool ok = mbar_wait(m, phase & 1, abort_flag);
    tc_fence_after();
    if (!ok && !*abort_flag) {
      *abort_flag = 1;
      atomicExch(a.status, code);
    }
    __syncwarp();
  };

  const int64_t tok = (b * a.L + t0) * su + (int64_t)h * a.P;
  const int sr = tid % 64, sc = tid / 64;   // a thread's state pieces (8 n of a row): row sr, pieces sc, sc + 4, ...
  auto fetch = [&](const float* states, int p0, int i, float (&f)[8]) {
    const float* src = states + ((int64_t)bhc * (N / 4) * P + p0 + sr) * 4;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const float4 v = *reinterpret_cast<const float4*>(src + (2 * (sc + 4 * i) + q) * 4 * P);
      f[4 * q] = v.x; f[4 * q + 1] = v.y; f[4 * q + 2] = v.z; f[4 * q + 3] = v.w;
    }
  };
  auto put = [&](int i, const float (&f)[8]) {
    const int pc = sc + 4 * i;
    put8(smem + S + (pc / 8) * TILE + tile_off<SQ_RB>(sr, pc % 8), PLANE, f);
  };
  // TMEM (columns d) (+)= the state's transpose times X^T, over 64 value channels
  auto state_product = [&](uint32_t d, int x, int planes, bool add) {
    constexpr uint32_t ID = make_idesc_bf16(N, Q, true, false);
#pragma unroll 1
    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
      for (int o = 2; o >= 0; --o)
#pragma unroll
        for (int z = 0; z <= o; ++z)
          if (z < planes) {
            umma_bf16(tmem + d, make_desc_sw128(s + S + (o - z) * PLANE, TILE) + 128 * kk,
                      make_desc_sw128(s + x + z * TILE, 16) + 2 * kk, ID, add);
            add = true;
          }
  };

  float m1[4][4], m2[4][4];   // dO E^T, dE E^T: rows 16 mt, columns 32 qh
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) m1[i][e] = m2[i][e] = 0.f;
  float dot = 0.f;
  const int steps = P / 64;
  for (int it = 0; it < steps; ++it) {
    const int p0 = 64 * it;
    float fs[4][8], fd[4][8];
    float4 fe[2][2], fr[2][2];   // four tokens (warp, warp + 8) of channels 2 lane, 2 lane + 1
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int quad = warp + 8 * r;
        const bool in = 4 * quad < rows;
        const int64_t at = (((b * a.H + h) * cdiv(a.L, 4) + t0 / 4 + quad) * P + p0 + 2 * lane + q) * 4;
        fe[r][q] = in ? *reinterpret_cast<const float4*>(a.errs + at) : make_float4(0.f, 0.f, 0.f, 0.f);
        fr[r][q] = in ? *reinterpret_cast<const float4*>(a.derrs + at) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
    for (int i = 0; i < 4; ++i) fetch(a.states, p0, i, fs[i]);
    if (it) wait(bdone, it - 1, 3201);
    load_planes<1, 64, NT>(s + DO, 0, (const T*)a.dy + tok + p0, su, rows, 64, true, tid);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      put4x2(smem + E, 4 * (warp + 8 * r), lane, fe[r]);
      put4x2(smem + DE, 4 * (warp + 8 * r), lane, fr[r]);
      const float d0[4] = {fr[r][0].x, fr[r][0].y, fr[r][0].z, fr[r][0].w};
      const float d1[4] = {fr[r][1].x, fr[r][1].y, fr[r][1].z, fr[r][1].w};
#pragma unroll
      for (int i = 0; i < 4; ++i)   // du = dE
        if (4 * (warp + 8 * r) + i < rows)
          *reinterpret_cast<uint32_t*>((T*)a.du + tok + (4 * (warp + 8 * r) + i) * su + p0 + 2 * lane) = pack2(d0[i], d1[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) fetch(a.dstates, p0, i, fd[i]);   // arrives during the first products
#pragma unroll
    for (int i = 0; i < 4; ++i) put(i, fs[i]);
    cp_async_wait_all();
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
      tc_fence_after();
      if (elect_one()) {
        state_product(C_Q, DO, 1, it > 0);
        state_product(C_K, DE, 3, it > 0);
        umma_commit(adone);
      }
      __syncwarp();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) dot += fs[i][e] * fd[i][e];
#pragma unroll 1
    for (int kk = 0; kk < 4; ++kk) {
      uint32_t fo[1][4], fe[3][4], w[3][4];
      ldsm4(fo[0], at_a<SQ_RB>(s + DO, 16 * mt, 2 * kk, lane));
#pragma unroll
      for (int z = 0; z < 3; ++z) ldsm4(fe[z], at_a<SQ_RB>(s + DE + z * TILE, 16 * mt, 2 * kk, lane));
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (2 * qh + x > mt) continue;
#pragma unroll
        for (int z = 0; z < 3; ++z) ldsm4(w[z], at_b<SQ_RB>(s + E + z * TILE, 32 * qh + 16 * x, 2 * kk, lane));
        mma_planes<1, 3, 3>(m1[2 * x], m1[2 * x + 1], fo, w);
        mma_planes<3, 3, 3>(m2[2 * x], m2[2 * x + 1], fe, w);
      }
    }
    wait(adone, it, 3202);
#pragma unroll
    for (int i = 0; i < 4; ++i) put(i, fd[i]);   // dS1 takes S0's place
    fence_proxy_async_smem();
    __syncthreads();
    if (warp == 0) {
      if (elect_one()) {
        state_product(C_K1, E, 3, it > 0);
        umma_commit(bdone);
      }
      __syncwarp();
    }
  }
  {   // K, Q while the last products run
    const int64_t at = (b * a.L + t0) * sk + (int64_t)g * N;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      load_planes<1, 64, NT>(s + K + x * TILE, 0, (const T*)a.B + at + 64 * x, sk, rows, 64, true, tid);
      load_planes<1, 64, NT>(s + QQ + x * TILE, 0, (const T*)a.C + at + 64 * x, sk, rows, 64, true, tid);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
  if (lane == 0) red[warp] = dot;
  wait(bdone, steps - 1, 3203);
  cp_async_wait_all();
  __syncthreads();
  // q.k and k.k of this warp's 16 x 32 block, then M1, -M2 (planes) and Y
  float* Yf = reinterpret_cast<float*>(smem + Y);
  float gk[4][4], gq[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) gk[i][e] = gq[i][e] = 0.f;
  if (2 * qh <= mt) {
#pragma unroll 2
    for (int kk = 0; kk < N / 16; ++kk) {
      uint32_t fk[1][4], fq[1][4], w[1][4];
      const uint32_t tile = s + K + (kk / 4) * TILE;
      ldsm4(fk[0], at_a<SQ_RB>(tile, 16 * mt, 2 * (kk % 4), lane));
      ldsm4(fq[0], at_a<SQ_RB>(tile + (QQ - K), 16 * mt, 2 * (kk % 4), lane));
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (2 * qh + x > mt) continue;
        ldsm4(w[0], at_b<SQ_RB>(tile, 32 * qh + 16 * x, 2 * (kk % 4), lane));
        mma_planes<1, 1, 1>(gk[2 * x], gk[2 * x + 1], fk, w);
        mma_planes<1, 1, 1>(gq[2 * x], gq[2 * x + 1], fq, w);
      }
    }
  }
#pragma unroll
  for (int x = 0; x < 2; ++x) {
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      const int j = 32 * qh + 16 * x + 8 * nt + q2;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int i = 16 * mt + pr + 8 * r;
        float u1[2], u2[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int jj = j + e;
          const float D = jj <= i ? exp2f((gt.lh[i] - gt.lh[jj]) + (gt.ll[i] - gt.ll[jj])) : 0.f;
          const float f1 = jj <= i ? a.scale * D * m1[2 * x + nt][2 * r + e] : 0.f;
          const float f2 = jj < i ? D * m2[2 * x + nt][2 * r + e] : 0.f;
          Yf[i * 65 + jj] = f1 * gq[2 * x + nt][2 * r + e] - f2 * gk[2 * x + nt][2 * r + e];
          u1[e] = f1 * gt.beta[jj];
          u2[e] = -f2 * gt.beta[jj];
        }
        uint32_t p1[3], p2[3];
        split2<3>(u1[0], u1[1], p1);
        split2<3>(u2[0], u2[1], p2);
        const uint32_t off = tile_off<SQ_RB>(i, 4 * qh + 2 * x + nt) + 2 * q2;
#pragma unroll
        for (int z = 0; z < 3; ++z) {
          *reinterpret_cast<uint32_t*>(smem + M1 + z * TILE + off) = p1[z];
          *reinterpret_cast<uint32_t*>(smem + M2 + z * TILE + off) = p2[z];
        }
      }
    }
  }
  // the state parts of dQ, dK (n = 32 mt + lane, 32 tokens from 32 qh), in place, and their dots with
  // the rows of Q, K over this warp's quarter of N
  const uint32_t tl = tmem + ((uint32_t)(32 * mt) << 16);
  {
    const int n = 32 * mt + lane;
    const uint8_t* kn = smem + K + (n / 64) * TILE;
#pragma unroll 1
    for (int i0 = 32 * qh; i0 < 32 * qh + 32; i0 += 16) {
      float x[16], y[16], av[16];
      auto at = [&](const uint8_t* base, int i) {
        return __bfloat162float(
            *reinterpret_cast<const T*>(base + tile_off<SQ_RB>(i0 + i, (n % 64) / 8) + 2 * (n % 8)));
      };
      tmem_get16(tl + C_Q + i0, x);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x[i] *= a.scale * gt.eg[i0 + i];
        av[i] = x[i] * at(kn + (QQ - K), i);
      }
      tmem_st16(tl + C_Q + i0, x);
      tmem_get16(tl + C_K + i0, x);
      tmem_get16(tl + C_K1 + i0, y);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float k = at(kn, i), k0 = -gt.eg[i0 + i] * x[i];
        av[i] += k0 * k;
        x[i] = k0 + gt.wb[i0 + i] * y[i];
        y[i] *= k;
      }
      tmem_st16(tl + C_K + i0, x);
      const float ra = lanes_sum16(av, lane), rb = lanes_sum16(y, lane);
      if (lane % 2 == 0) {
        const int i = i0 + lane / 2;
        va[mt * Q + i] = ra;
        vb[mt * Q + i] = gt.wb[i] * rb;
        vw[mt * Q + i] = gt.w[i] * rb;
      }
    }
    tmem_wait_st();
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    if (elect_one()) {
      constexpr uint32_t ID = make_idesc_bf16(N, Q, true, false), IDT = make_idesc_bf16(N, Q, true, true);
#pragma unroll 1
      for (int kk = 0; kk < 4; ++kk) {
        const uint64_t k = make_desc_sw128(s + K, TILE) + 128 * kk, q = make_desc_sw128(s + QQ, TILE) + 128 * kk;
#pragma unroll
        for (int z = 2; z >= 0; --z) {
          const uint64_t p1 = make_desc_sw128(s + M1 + z * TILE, 16), p2 = make_desc_sw128(s + M2 + z * TILE, 16);
          umma_bf16(tmem + C_Q, k, p1 + 2 * kk, ID, true);
          umma_bf16(tmem + C_K, q, p1 + 128 * kk, IDT, true);
          umma_bf16(tmem + C_K, k, p2 + 2 * kk, ID, true);
          umma_bf16(tmem + C_K, k, p2 + 128 * kk, IDT, true);
        }
      }
      umma_commit(mdone);
    }
    __syncwarp();
  }
  // column sums of Y, then its row prefixes with beta (in place, a row per warp and step)
  {
    const int j = tid % 64, o = tid / 64;
    float v = 0.f;
#pragma unroll
    for (int i = 16 * o; i < 16 * o + 16; ++i) v += Yf[i * 65 + j];
    seg[o * Q + j] = v;
    if (o < 3) {   // and the quarters of va, vb, vw
      float* q = vec + 4 * Q * o;
      q[j] = (q[j] + q[Q + j]) + (q[2 * Q + j] + q[3 * Q + j]);
    }
  }
  __syncthreads();
  {
    const float b0 = gt.beta[2 * lane], b1 = gt.beta[2 * lane + 1];
#pragma unroll
    for (int k0 = 0; k0 < 8; k0 += 4) {
      float y0[4], y1[4], v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float* row = Yf + (warp + 8 * (k0 + k)) * 65 + 2 * lane;
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
        float* row = Yf + (warp + 8 * (k0 + k)) * 65 + 2 * lane;
        row[0] = (lane ? before : 0.f) + y0[k];
        row[1] = v[k];
      }
    }
  }
  __syncthreads();
  {
    const int t = tid / 4, o = tid % 4;   // four threads a token
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int i = k % 8 + 8 * o + 32 * (k / 8);   // a warp's rows of Y in different banks
      v += i >= t ? va[i] + (t > 0 ? Yf[i * 65 + t - 1] : 0.f) : vb[i];
    }
#pragma unroll
    for (int x = 1; x < 4; x <<= 1) v += __shfl_xor_sync(0xffffffffu, v, x);
    float da = 0.f;
    if (o == 0) {
      float d = 0.f;
#pragma unroll
      for (int k = 0; k < NT / 32; ++k) d += red[k];
      const float dl = t < rows ? v + gt.eg[Q - 1] * d : 0.f;
      const float ea = expf(a.A_log[h]);
      if (t < rows) {
        const int64_t at = (b * a.L + t0 + t) * a.H + h;
        if (!*abort_flag) {
          a.ddt[at] = -ea * dl;
          a.dbeta[at] = vw[t] + ((seg[t] + seg[Q + t]) + (seg[2 * Q + t] + seg[3 * Q + t]));
        }
        // dA_log: dl times the log-decay, which is bounded as the forward bounds it
        da = dl * fmaxf(-ea * a.dt[at], -139.f);
      }
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) da += __shfl_xor_sync(0xffffffffu, da, x);
    __syncthreads();
    if (lane == 0) red[warp] = da;
  }
  wait(mdone, 0, 3204);
  __syncthreads();   // Y has been read, M1 and M2 by the products
  // dQ, dK in f32, then the sums over the key head's value heads, in their order: this block's share of the rows
  float* out = reinterpret_cast<float*>(smem + OUT);
#pragma unroll 1
  for (int i0 = 32 * qh; i0 < 32 * qh + 32; i0 += 16) {
    float x[16];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      tmem_get16(tl + (m ? C_K : C_Q) + i0, x);
#pragma unroll
      for (int i = 0; i < 16; ++i) out[(m * Q + i0 + i) * N + 32 * mt + lane] = x[i];
    }
  }
  tc_fence_before();
  if (rep > 1) cluster_sync();
  else __syncthreads();
  bool ok = !*abort_flag;
  if (rep > 1)
    for (int x = 0; x < rep; ++x) ok &= !ld_peer_int(s + BAR + 5 * 8, x);
  for (int i = (int)rank + rep * warp; i < rows && ok; i += rep * (NT / 32)) {
    const int64_t at = (b * a.L + t0 + i) * sk + (int64_t)g * N + 4 * lane;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const uint32_t src = s + OUT + ((m * Q + i) * N + 4 * lane) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int x = 0; x < rep; ++x) {
        const float4 p = rep > 1 ? ld_peer(src, x) : *reinterpret_cast<const float4*>(out + (m * Q + i) * N + 4 * lane);
        v.x += p.x; v.y += p.y; v.z += p.z; v.w += p.w;
      }
      *reinterpret_cast<uint2*>((T*)(m ? a.dB : a.dC) + at) = make_uint2(pack2(v.x, v.y), pack2(v.z, v.w));
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0) {
    float d = 0.f;
    for (int k = 0; k < NT / 32; ++k) d += red[k];
    if (!*abort_flag) a.da_part[bhc] = d;
  }
  if (warp == 0) {
    if (*abort_flag) {   // products that were issued end before their memory is given back
      mbar_wait(mdone, 0, nullptr, 100000000ull);
      __syncwarp();
    }
    tc_fence_after();
    tmem_dealloc(tmem, COLS);
  }
  __syncwarp();
  if (rep > 1) cluster_sync();   // the peers have read this block's sums
}

}  // namespace

bool tc_grad_takes(int64_t H, int64_t G, int64_t N_, bool tc) { return tc && N_ == N && H / G <= 8; }   // 8: a cluster

int tc_grad_run(TcGradCall a, cudaStream_t st) {
  const int64_t blocks = a.Bt * a.H * a.nc;
  TSSM_REQUIRE(blocks < (int64_t(1) << 31), "gated_delta_rule_bwd: size out of range");
  a.status = device_status_ptr();
  if (!a.status) {
    set_error("gated_delta_rule_bwd: device status word unavailable");
    return TSSM_ERR_CUDA;
  }
  if (cudaFuncSetAttribute(delta_grad_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, BYTES) != cudaSuccess)
    return check_launch("gated_delta_rule_bwd: set smem attribute");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = BYTES;
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = (unsigned)(a.H / a.G);
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, delta_grad_tc_kernel, a);
  return check_launch("gated_delta_rule_bwd: gradients");
}

}  // namespace delta
}  // namespace tssm
