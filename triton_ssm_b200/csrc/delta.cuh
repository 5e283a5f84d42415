// Pieces shared by the chunked gated delta rule's kernels.
//
// One chunk of Q = 64 tokens of one (batch row, head), with l_i the inclusive
// sum of log-decays within the chunk, D_ij = exp(l_i - l_j) for j <= i, S0 the
// state before the chunk (rows n, columns p):
//     A_ij  = D_ij (k_i . k_j)            j < i       Aq_ij = scale D_ij (q_i . k_j)   j <= i
//     T     = (I + A diag(beta))^-1
//     E     = T (V - exp(l) K S0)                     prediction errors  [Q x P]
//     O     = scale exp(l) Q S0 + Aq diag(beta) E
//     S1    = exp(l_last) S0 + K^T diag(exp(l_last - l) beta) E
// beta multiplies columns only, so that nothing is ever divided by it.
//
// Precision: a matrix product on the tensor cores takes bf16 operands.  An f32
// operand is split into 2 or 3 bf16 planes (8 bits each, 3 planes are exact to
// f32) and the products of planes i + j < planes are summed in f32: the state,
// the errors and every f32 result keep f32 accuracy; bf16 inputs are one plane.
#pragma once
#include "common.cuh"

namespace tssm {
namespace delta {

constexpr int Q = 64;   // tokens per chunk
constexpr float LOG2E = 1.4426950408889634f;

// ------------------------------------------------------------------ tensor-core fragments
__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void stsm4t(uint32_t a, const uint32_t (&r)[4]) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]) : "memory");
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float lo2(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float hi2(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// (x, y) as NS bf16 pairs whose sum is exact to 8 NS bits.
template <int NS>
__device__ __forceinline__ void split2(float x, float y, uint32_t (&r)[NS]) {
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    r[s] = pack2(x, y);
    if (s + 1 < NS) {
      x -= lo2(r[s]);
      y -= hi2(r[s]);
    }
  }
}
// The A operand (16 rows x 16 k) of two adjacent 16 x 8 result tiles: results feed the
// next product without leaving the registers.
template <int NS>
__device__ __forceinline__ void split_a(const float (&t0)[4], const float (&t1)[4], uint32_t (&a)[NS][4]) {
  uint32_t r[4][NS];
  split2<NS>(t0[0], t0[1], r[0]);
  split2<NS>(t0[2], t0[3], r[1]);
  split2<NS>(t1[0], t1[1], r[2]);
  split2<NS>(t1[2], t1[3], r[3]);
#pragma unroll
  for (int s = 0; s < NS; ++s)
#pragma unroll
    for (int i = 0; i < 4; ++i) a[s][i] = r[i][s];
}

// Tiles in shared memory: rows of RB bytes, 16-byte pieces XOR-swizzled by the row so that
// the eight rows of a matrix load fall in different banks.
template <int RB>
__device__ __forceinline__ uint32_t tile_off(int row, int piece) {
  return (uint32_t)(row * RB + ((piece ^ (row & 7)) << 4));
}
// Lane addresses of the matrix loads, for 16 rows from r0 and two 16-byte pieces from c0.
template <int RB>
__device__ __forceinline__ uint32_t at_b(uint32_t base, int r0, int c0, int lane) {   // B from [n][k]; two n tiles
  return base + tile_off<RB>(r0 + ((lane >> 4) << 3) + (lane & 7), c0 + ((lane >> 3) & 1));
}
template <int RB>
__device__ __forceinline__ uint32_t at_a(uint32_t base, int r0, int c0, int lane) {   // A from [m][k]; B (trans) from [k][n]
  return base + tile_off<RB>(r0 + (lane & 15), c0 + (lane >> 4));
}

// d0, d1 += sum over planes s + x < NM of a[s] b[x], smallest terms first.
template <int NA, int NB, int NM>
__device__ __forceinline__ void mma_planes(float (&d0)[4], float (&d1)[4], const uint32_t (&a)[NA][4],
                                           const uint32_t (&b)[NB][4]) {
#pragma unroll
  for (int t = NM - 1; t >= 0; --t)
#pragma unroll
    for (int s = 0; s < NA; ++s) {
      const int x = t - s;
      if (x < 0 || x >= NB) continue;
      mma(d0, a[s], b[x][0], b[x][1]);
      mma(d1, a[s], b[x][2], b[x][3]);
    }
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
  const int n = live ? 16 : 0;   // 0 bytes read: the 16 bytes are zero-filled
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void bar_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }

// ------------------------------------------------------------------ one chunk's gates
struct Gates {        // in shared memory
  float lh[Q], ll[Q];   // l_i in log2 units as a sum of two floats (differences of long sums stay exact)
  float eg[Q];          // exp(l_i)
  float w[Q];           // exp(l_last - l_i)
  float wb[Q];          // w_i beta_i
  float beta[Q];
};

__device__ __forceinline__ float exp2_pair(float h, float l) {
  const float e = exp2f(h);
  return e + e * (l * 0.6931471805599453f);
}

// One warp: gates of tokens t0.. of a row with `stride` floats between tokens.  Tokens behind
// the end get decay 1 and beta 0.  A step's log2-decay is held above -200 (its factor is 0 in
// f32 there), so that an infinite dt forgets the state instead of making inf - inf.
__device__ __forceinline__ void gates_warp(Gates& g, const float* dt, const float* beta, int64_t stride, float a_log,
                                           int64_t t0, int64_t L, int lane) {
  const double a2 = -(double)expf(a_log) * 1.4426950408889634074;
  double l[2];
  float b[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int64_t t = t0 + 2 * lane + e;
    const bool in = t < L;
    const double v = in ? a2 * (double)dt[t * stride] : 0.0;
    l[e] = v > -200.0 ? v : -200.0;
    if (v != v) l[e] = v;
    b[e] = in ? beta[t * stride] : 0.f;
  }
  double s = l[0] + l[1];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double v = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += v;
  }
  const double last = __shfl_sync(0xffffffffu, s, 31);
  const double li[2] = {s - l[1], s};
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = 2 * lane + e;
    const float h = (float)li[e], lo = (float)(li[e] - (double)h);
    g.lh[i] = h;
    g.ll[i] = lo;
    g.eg[i] = exp2_pair(h, lo);
    const double d = last - li[e];
    const float dh = (float)d;
    g.w[i] = exp2_pair(dh, (float)(d - (double)dh));
    g.wb[i] = g.w[i] * b[e];
    g.beta[i] = b[e];
  }
}

// ------------------------------------------------------------------ loading tiles
// A [64 x W] tile of an io tensor (rows `stride` elements apart, `valid` columns, zero beyond)
// into XS bf16 planes of RB-byte rows (XS = 1: bf16, copied asynchronously; XS = 3: f32, split).
template <int XS, int W, int NTH, typename T>
__device__ __forceinline__ void load_planes(uint32_t dst, int plane_bytes, const T* src, int64_t stride, int rows,
                                            int valid, bool vec, int t) {
  constexpr int RB = W * 2, PIECES = W / 8;
  for (int i = t; i < Q * PIECES; i += NTH) {
    const int r = i / PIECES, c = i % PIECES;
    const uint32_t off = tile_off<RB>(r, c);
    if constexpr (XS == 1) {
      if (vec) {
        const bool in = r < rows && c * 8 < valid;
        cp_async16(dst + off, src + (in ? (int64_t)r * stride + c * 8 : 0), in);
        continue;
      }
    }
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = 0.f;
    if (r < rows) {
      const T* p = src + (int64_t)r * stride + c * 8;
      if (XS == 3 && vec) {
#pragma unroll
        for (int q = 0; q < 2; ++q)
          if (c * 8 + 4 * q < valid) {
            const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + 4 * q);
            f[4 * q] = v.x; f[4 * q + 1] = v.y; f[4 * q + 2] = v.z; f[4 * q + 3] = v.w;
          }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c * 8 + e < valid) f[e] = ldf(p + e);
      }
    }
    uint32_t w[4][XS];
#pragma unroll
    for (int q = 0; q < 4; ++q) split2<XS>(f[2 * q], f[2 * q + 1], w[q]);
#pragma unroll
    for (int x = 0; x < XS; ++x)
      asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst + x * plane_bytes + off), "r"(w[0][x]),
                   "r"(w[1][x]), "r"(w[2][x]), "r"(w[3][x]) : "memory");
  }
}

// ------------------------------------------------------------------ A, Aq and T of one chunk
constexpr int AM = Q + 4;   // floats per row of the f32 work matrix

// Lower triangle of X K^T for the 16 rows from 16 w of X (one warp): g[nt] holds columns
// 8 nt .., tiles behind the diagonal block are not computed.
template <int XS, int KN>
__device__ __forceinline__ void gram_rows(float (&g)[8][4], uint32_t x, uint32_t k, int w, int lane) {
  constexpr int RB = KN * 2, PB = Q * RB;
#pragma unroll
  for (int nt = 0; nt < 8; ++nt)
#pragma unroll
    for (int i = 0; i < 4; ++i) g[nt][i] = 0.f;
#pragma unroll 2
  for (int kk = 0; kk < KN / 16; ++kk) {
    uint32_t a[XS][4];
#pragma unroll
    for (int s = 0; s < XS; ++s) ldsm4(a[s], at_a<RB>(x + s * PB, 16 * w, 2 * kk, lane));
#pragma unroll
    for (int np = 0; np < 4; ++np) {
      if (np > w) break;
      uint32_t b[XS][4];
#pragma unroll
      for (int s = 0; s < XS; ++s) ldsm4(b[s], at_b<RB>(k + s * PB, 16 * np, 2 * kk, lane));
      mma_planes<XS, XS, XS>(g[2 * np], g[2 * np + 1], a, b);
    }
  }
}

// c[2 rows x 4 columns] (+)= X[r.., k] Y[k, c..] over k in [0, KD): X, Y, out rows of AM floats.
template <int KD>
__device__ __forceinline__ void block_2x4(const float* X, const float* Y, float (&c)[2][4]) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) c[i][j] = 0.f;
#pragma unroll 8
  for (int k = 0; k < KD; ++k) {
    const float4 y = *reinterpret_cast<const float4*>(Y + k * AM);
    const float x0 = X[k], x1 = X[AM + k];
    c[0][0] += x0 * y.x; c[0][1] += x0 * y.y; c[0][2] += x0 * y.z; c[0][3] += x0 * y.w;
    c[1][0] += x1 * y.x; c[1][1] += x1 * y.y; c[1][2] += x1 * y.z; c[1][3] += x1 * y.w;
  }
}

// In place: the strictly lower M (row-major, AM floats a row) becomes (I + M)^-1.  128 threads
// (t), named barrier `bar`.  16 x 16 diagonal blocks by forward substitution (a column per
// thread), then 16 -> 32 -> 64 by T21 = -T22 (M21 T11); the unused upper blocks hold M21 T11.
__device__ __forceinline__ void invert_unit_lower(float* M, int t, int bar) {
  if (t < 64) {
    const int o = (t / 16) * 16, col = t % 16;
    const float* B = M + o * AM + o;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = i == col ? 1.f : 0.f;
#pragma unroll
      for (int k = 0; k < 16; k += 4) {
        if (k >= i) break;
        const float4 m = *reinterpret_cast<const float4*>(B + i * AM + k);
        const float mm[4] = {m.x, m.y, m.z, m.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (k + e < i) v -= mm[e] * x[k + e];
      }
      x[i] = v;
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; ++i) M[(o + i) * AM + o + col] = x[i];
  }
  bar_sync(bar, 128);
  {   // two pairs of 16-blocks, 32 threads each (2 x 4 outputs a thread)
    float c[2][4];
    const int o = (t / 32 & 1) * 32, r = (t % 32) / 4 * 2, cc = t % 4 * 4;
    if (t < 64) {
      block_2x4<16>(M + (o + 16 + r) * AM + o, M + o * AM + o + cc, c);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        *reinterpret_cast<float4*>(M + (o + r + i) * AM + o + 16 + cc) = make_float4(c[i][0], c[i][1], c[i][2], c[i][3]);
      __syncwarp();
      block_2x4<16>(M + (o + 16 + r) * AM + o + 16, M + o * AM + o + 16 + cc, c);
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 2; ++i)
        *reinterpret_cast<float4*>(M + (o + 16 + r + i) * AM + o + cc) = make_float4(-c[i][0], -c[i][1], -c[i][2], -c[i][3]);
    }
  }
  bar_sync(bar, 128);
  {
    // The 16-blocks above the diagonal inside the 32-blocks held scratch: they are zero in T.
    if (t >= 64) {
      const int o = (t / 32 & 1) * 32, r = (t % 32) / 2, h = (t % 2) * 8;
#pragma unroll
      for (int e = 0; e < 8; e += 4)
        *reinterpret_cast<float4*>(M + (o + r) * AM + o + 16 + h + e) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
  bar_sync(bar, 128);
  {
    float c[2][4];
    const int r = t / 8 * 2, cc = t % 8 * 4;
    block_2x4<32>(M + (32 + r) * AM, M + cc, c);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      *reinterpret_cast<float4*>(M + (r + i) * AM + 32 + cc) = make_float4(c[i][0], c[i][1], c[i][2], c[i][3]);
    bar_sync(bar, 128);
    block_2x4<32>(M + (32 + r) * AM + 32, M + 32 + cc, c);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      *reinterpret_cast<float4*>(M + (32 + r + i) * AM + cc) = make_float4(-c[i][0], -c[i][1], -c[i][2], -c[i][3]);
  }
  bar_sync(bar, 128);
}

// A 64 x 64 tile of planes: 128-byte rows.
constexpr int SQ_RB = 128, SQ_BYTES = Q * SQ_RB;

// 128 threads (t = 0..127): from the loaded K, Q planes and the gates, the planes of
// Aq diag(beta) (NA of them) and of T (NTP).  M is the f32 work matrix.  Entries of 16-blocks
// above the diagonal are not written: nobody reads them.
template <int XS, int KN, int NA, int NTP>
__device__ __forceinline__ void chunk_matrices(uint32_t k, uint32_t q, const Gates& g, float scale, float* M,
                                               uint32_t aq, uint32_t tp, int t, int bar) {
  const int w = t / 32, lane = t % 32;
  const int r0 = 16 * w + lane / 4;
  float acc[8][4];
#pragma unroll
  for (int pass = 0; pass < 2; ++pass) {   // K K^T, then Q K^T
    gram_rows<XS, KN>(acc, pass ? q : k, k, w, lane);
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) {
      if (nt > 2 * w + 1) break;
      const int j = 8 * nt + 2 * (lane % 4);
      const float2 bj = *reinterpret_cast<const float2*>(g.beta + j);
      const float2 hj = *reinterpret_cast<const float2*>(g.lh + j);
      const float2 lj = *reinterpret_cast<const float2*>(g.ll + j);
#pragma unroll
      for (int hrow = 0; hrow < 2; ++hrow) {
        const int i = r0 + 8 * hrow;
        const float hi = g.lh[i], li = g.ll[i];
        const bool in0 = pass ? j <= i : j < i, in1 = pass ? j + 1 <= i : j + 1 < i;
        const float v0 = in0 ? acc[nt][2 * hrow] * exp2f((hi - hj.x) + (li - lj.x)) * bj.x : 0.f;
        const float v1 = in1 ? acc[nt][2 * hrow + 1] * exp2f((hi - hj.y) + (li - lj.y)) * bj.y : 0.f;
        if (pass == 0) {
          *reinterpret_cast<float2*>(M + i * AM + j) = make_float2(v0, v1);
        } else {
          uint32_t p[NA];
          split2<NA>(scale * v0, scale * v1, p);
#pragma unroll
          for (int s = 0; s < NA; ++s)
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(aq + s * SQ_BYTES + tile_off<SQ_RB>(i, nt) + 4 * (lane % 4)),
                         "r"(p[s]) : "memory");
        }
      }
    }
  }
  bar_sync(bar, 128);
  invert_unit_lower(M, t, bar);
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int idx = t + it * 128, i = idx / 8, c = idx % 8;
    if (c / 2 > i / 16) continue;
    const float4 x = *reinterpret_cast<const float4*>(M + i * AM + 8 * c);
    const float4 y = *reinterpret_cast<const float4*>(M + i * AM + 8 * c + 4);
    uint32_t r[4][NTP];
    split2<NTP>(x.x, x.y, r[0]);
    split2<NTP>(x.z, x.w, r[1]);
    split2<NTP>(y.x, y.y, r[2]);
    split2<NTP>(y.z, y.w, r[3]);
#pragma unroll
    for (int s = 0; s < NTP; ++s)
      asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(tp + s * SQ_BYTES + tile_off<SQ_RB>(i, c)),
                   "r"(r[0][s]), "r"(r[1][s]), "r"(r[2][s]), "r"(r[3][s]) : "memory");
  }
}

}  // namespace delta
}  // namespace tssm
