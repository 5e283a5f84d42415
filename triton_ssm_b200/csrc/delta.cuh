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
// operand is split into three bf16 planes (8 bits each: exact to f32) and the
// products of planes i + j < 3 are summed in f32: every result has f32 accuracy,
// a bf16 one is then rounded once; bf16 inputs are one plane.
#pragma once
#include "common.cuh"

namespace tssm {
namespace delta {

constexpr int Q = 64;   // tokens per chunk
constexpr float LOG2E = 1.4426950408889634f;

// A dependent kernel of a call: started early when it is small (its latency counts then);
// larger grids gained nothing from it and lost 2 % behind the scans.
template <typename... P, typename... A>
inline void launch_next(void (*kern)(P...), unsigned blocks, int threads, size_t smem, cudaStream_t st, A&&... args) {
  if ((int)blocks <= num_sms()) launch_after(kern, dim3(blocks), dim3(threads), smem, st, static_cast<A&&>(args)...);
  else kern<<<blocks, threads, smem, st>>>(static_cast<P>(args)...);
}

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
// d = a b
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float lo2(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float hi2(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// x, y -= the bf16 pair h (exactly: the mixed-precision FMA reads bf16 operands, which saves
// the shifts and masks; 13 instead of 16 cycles per pair split into three planes).
__device__ __forceinline__ void sub2(float& x, float& y, uint32_t h) {
  asm("{\n\t.reg .b16 l, u, m;\n\tmov.b32 {l, u}, %2;\n\tmov.b16 m, 0xBF80;\n\t"
      "fma.rn.f32.bf16 %0, l, m, %0;\n\tfma.rn.f32.bf16 %1, u, m, %1;\n\t}"
      : "+f"(x), "+f"(y) : "r"(h));
}

// (x, y) as NS bf16 pairs whose sum is exact to 8 NS bits.
template <int NS>
__device__ __forceinline__ void split2(float x, float y, uint32_t (&r)[NS]) {
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    r[s] = pack2(x, y);
    if (s + 1 < NS) sub2(x, y, r[s]);
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

// d0, d1 += sum over planes s + x < NM of a[s] b[x], smallest terms first.  APART: they are summed
// by themselves and then added, rounded, as the tensor core cuts a sum at every step.  So done where
// a value is added to a state that lasts (a cut is a whole step of the state, always towards 0), and
// in f32 for sums over the state's width and over value channels: 48 cuts of one growing sum (N = 128)
// made f32 results five times less exact than plain f32 arithmetic.  The triangular sums over 64
// tokens stay as they are: f32 results are off by 2 to 4e-7, with those apart too by 2e-7, but f32
// calls take 2 to 8 % longer as it is and another 4 to 6 % then.
template <int NA, int NB, int NM, bool APART = false>
__device__ __forceinline__ void mma_planes(float (&d0)[4], float (&d1)[4], const uint32_t (&a)[NA][4],
                                           const uint32_t (&b)[NB][4]) {
  float p0[4], p1[4];
  bool first = true;
#pragma unroll
  for (int t = NM - 1; t >= 0; --t)
#pragma unroll
    for (int s = 0; s < NA; ++s) {
      const int x = t - s;
      if (x < 0 || x >= NB) continue;
      if (APART && first) {
        mma_first(p0, a[s], b[x][0], b[x][1]);
        mma_first(p1, a[s], b[x][2], b[x][3]);
        first = false;
        continue;
      }
      mma(APART ? p0 : d0, a[s], b[x][0], b[x][1]);
      mma(APART ? p1 : d1, a[s], b[x][2], b[x][3]);
    }
  if constexpr (APART)
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      const float2 u = fadd2(make_float2(d0[e], d0[e + 1]), make_float2(p0[e], p0[e + 1]));
      const float2 v = fadd2(make_float2(d1[e], d1[e + 1]), make_float2(p1[e], p1[e + 1]));
      d0[e] = u.x; d0[e + 1] = u.y; d1[e] = v.x; d1[e + 1] = v.y;
    }
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
  const int n = live ? 16 : 0;   // 0 bytes read: the 16 bytes are zero-filled
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void bar_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }

// What the forward saves, and the backward's chain leaves for its gradients, has a value
// channel's rows four beside each other: the states of a chunk [ceil(N / 4)][P][4], the errors of
// a (batch row, head) [ceil(L / 4)][P][4], so that lanes on neighbouring channels move neighbouring
// 16 bytes.  Two adjacent n (or tokens; n even) of channel p:
__device__ __forceinline__ float2* saved_pair(float* base, int P, int p, int64_t n) {
  return reinterpret_cast<float2*>(base + ((n >> 2) * P + p) * 4 + (n & 2));
}
__host__ __device__ constexpr inline int64_t saved_floats(int64_t P, int64_t N) { return (N + 3) / 4 * 4 * P; }

// ------------------------------------------------------------------ one chunk's gates
// D_ij of tokens in different 16-token blocks I > J is a_i c_IJ b_j, every factor at most 1
// and from the 64-bit sums: a_i = exp(l_i - l_{16 I - 1}), b_j = exp(l_{16 J + 15} - l_j),
// c_IJ = exp(l_{16 I - 1} - l_{16 J + 15}).
struct Gates {        // in shared memory
  float lh[Q], ll[Q];   // l_i in log2 units as a sum of two floats (differences of long sums stay exact)
  float a[Q];           // a_i (blocks 1 to 3)
  float bb[Q];          // b_i beta_i
  float b[Q];           // b_i
  float c[16];          // c_IJ at 4 I + J
  float eg[Q];          // exp(l_i)
  float w[Q];           // exp(l_last - l_i)
  float wb[Q];          // w_i beta_i
  float beta[Q];
};

static_assert(sizeof(Gates) % 16 == 0, "copied in 16-byte pieces");
// 128 threads (t): the gates of a chunk to HBM.
__device__ __forceinline__ void copy_gates(Gates* dst, const Gates& g, int t) {
  for (int i = t; i < (int)(sizeof(Gates) / 16); i += 128)
    reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(&g)[i];
}

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
  const double blk = __shfl_sync(0xffffffffu, s, lane | 7);               // l at the end of this token's block
  const double prv = __shfl_sync(0xffffffffu, s, ((lane & 24) - 1) & 31);   // and of the block before
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = 2 * lane + e;
    g.a[i] = lane >= 8 ? exp2f((float)(li[e] - prv)) : 1.f;
    g.b[i] = exp2f((float)(blk - li[e]));
    g.bb[i] = g.b[i] * b[e];
  }
  const int I = (lane >> 2) & 3, J = lane & 3;
  const double lI = __shfl_sync(0xffffffffu, s, (8 * I - 1) & 31), lJ = __shfl_sync(0xffffffffu, s, 8 * J + 7);
  if (lane < 16) g.c[lane] = J < I ? exp2f((float)(lI - lJ)) : 1.f;
}

// ------------------------------------------------------------------ loading tiles
// A [64 x W] tile of an io tensor (rows `stride` elements apart, `valid` columns, zero beyond)
// into XS bf16 planes of RB-byte rows (XS = 1: bf16, copied asynchronously; XS = 3: f32, split).
template <int XS, int W, int NTH, typename T>
__device__ __forceinline__ void load_planes(uint32_t dst, int plane_bytes, const T* src, int64_t stride, int rows,
                                            int valid, bool vec, int t) {
  constexpr int RB = W * 2, PIECES = W / 8;
  static_assert(NTH % PIECES == 0, "a thread keeps its column");
  if constexpr (XS == 1) {
    if (vec) {
      constexpr int STEP = NTH / PIECES;   // rows per pass
      const int c = t % PIECES, r0 = t / PIECES;
      const bool col = c * 8 < valid;
      const T* p = src + (col ? (int64_t)r0 * stride + c * 8 : 0);
#pragma unroll 2
      for (int r = r0; r < Q; r += STEP, p += STEP * stride)
        cp_async16(dst + tile_off<RB>(r, c), r < rows && col ? p : src, r < rows && col);
      return;
    }
  }
#pragma unroll 2
  for (int i = t; i < Q * PIECES; i += NTH) {
    const int r = i / PIECES, c = i % PIECES;
    const uint32_t off = tile_off<RB>(r, c);
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

__device__ __forceinline__ void mma_tf32(float (&d)[4], const float (&a)[4], float b0, float b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(__float_as_uint(a[0])), "r"(__float_as_uint(a[1])), "r"(__float_as_uint(a[2])), "r"(__float_as_uint(a[3])),
        "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)));
}
// x = hi + lo: hi the 11 leading bits, lo the rest (of which the tensor core takes 11).
__device__ __forceinline__ void tf32_split(float x, float& hi, float& lo) {
  hi = __uint_as_float(__float_as_uint(x) & 0xffffe000u);
  lo = x - hi;
}

// One warp: out [16 x 8 NT] = sign * X [16 x 8 KS] Y [8 KS x 8 NT], rows of AM floats, f32
// accuracy from three products of tf32 halves.
template <int KS, int NT>
__device__ __forceinline__ void block_mma(const float* X, const float* Y, float* out, float sign, int lane) {
  const int g = lane >> 2, t = lane & 3;
  float d[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) d[n][e] = 0.f;
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    float ah[4], al[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) tf32_split(X[(g + 8 * (e & 1)) * AM + 8 * k + t + 4 * (e >> 1)], ah[e], al[e]);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float bh[2], bl[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) tf32_split(Y[(8 * k + t + 4 * e) * AM + 8 * n + g], bh[e], bl[e]);
      mma_tf32(d[n], al, bh[0], bh[1]);
      mma_tf32(d[n], ah, bl[0], bl[1]);
      mma_tf32(d[n], ah, bh[0], bh[1]);
    }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      *reinterpret_cast<float2*>(out + (g + 8 * e) * AM + 8 * n + 2 * t) =
          make_float2(sign * d[n][2 * e], sign * d[n][2 * e + 1]);
}

// In place: the strictly lower M (row-major, AM floats a row) becomes (I + M)^-1, on and below
// the diagonal 16 x 16 blocks; the blocks above hold scratch.  128 threads (t), named barrier
// `bar`.  Diagonal blocks by forward substitution (a column per thread), then 16 -> 32 -> 64 by
// T21 = -T22 (M21 T11) on the tensor cores.
__device__ __forceinline__ void invert_unit_lower(float* M, int t, int bar) {
  const int w = t / 32, lane = t % 32;
  if (t < 64) {
    const int o = (t / 16) * 16, col = t % 16;
    const float* B = M + o * AM + o;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = i == col ? 1.f : 0.f, v2 = 0.f;
#pragma unroll
      for (int k = 0; k < 16; k += 4) {
        if (k >= i) break;
        const float4 m = *reinterpret_cast<const float4*>(B + i * AM + k);
        const float mm[4] = {m.x, m.y, m.z, m.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (k + e < i) (e & 1 ? v2 : v) -= mm[e] * x[k + e];
      }
      x[i] = v + v2;
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; ++i) M[(o + i) * AM + o + col] = x[i];
  }
  bar_sync(bar, 128);
  {   // two pairs of 16-blocks, two warps each
    const int o = (w / 2) * 32, n = (w % 2) * 8;
    block_mma<2, 1>(M + (o + 16) * AM + o, M + o * AM + o + n, M + o * AM + o + 16 + n, 1.f, lane);
    bar_sync(bar, 128);
    block_mma<2, 1>(M + (o + 16) * AM + o + 16, M + o * AM + o + 16 + n, M + (o + 16) * AM + o + n, -1.f, lane);
  }
  bar_sync(bar, 128);
  {   // the pair of 32-blocks, a 16 x 16 quarter per warp; blocks above T's diagonal are skipped
    const int m = (w / 2) * 16, n = (w % 2) * 16;
    const float *A21 = M + (32 + m) * AM, *T22 = M + (32 + m) * AM + 32;
    float *Y = M + 32, *T21 = M + (32 + m) * AM + n;
    if (n == 0) block_mma<4, 2>(A21, M, Y + m * AM, 1.f, lane);
    else block_mma<2, 2>(A21 + 16, M + 16 * AM + 16, Y + m * AM + 16, 1.f, lane);
    bar_sync(bar, 128);
    if (m == 0) block_mma<2, 2>(T22, Y + n, T21, -1.f, lane);
    else block_mma<4, 2>(T22, Y + n, T21, -1.f, lane);
  }
  bar_sync(bar, 128);
}

// A 64 x 64 tile of planes: 128-byte rows.
constexpr int SQ_RB = 128, SQ_BYTES = Q * SQ_RB;

// Eight values, as three planes of 16-byte pieces.
__device__ __forceinline__ void put8(uint8_t* dst, int plane, const float (&f)[8]) {
  uint32_t w[4][3];
#pragma unroll
  for (int q = 0; q < 4; ++q) split2<3>(f[2 * q], f[2 * q + 1], w[q]);
#pragma unroll
  for (int z = 0; z < 3; ++z)
    *reinterpret_cast<uint4*>(dst + z * plane) = make_uint4(w[0][z], w[1][z], w[2][z], w[3][z]);
}

// Four tokens (rows from r) of channels 2 lane, 2 lane + 1 into three planes of a 64 x 64 tile.
__device__ __forceinline__ void put4x2(uint8_t* tile, int r, int lane, const float4 (&f)[2]) {
  const float a[4] = {f[0].x, f[0].y, f[0].z, f[0].w}, b[4] = {f[1].x, f[1].y, f[1].z, f[1].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t w[3];
    split2<3>(a[i], b[i], w);
#pragma unroll
    for (int z = 0; z < 3; ++z)
      *reinterpret_cast<uint32_t*>(tile + z * SQ_BYTES + tile_off<SQ_RB>(r + i, lane / 4) + 4 * (lane % 4)) = w[z];
  }
}

// A chunk's image, as it lies in shared memory: planes of T and of Aq diag(beta), gates.
constexpr int IMG_T = 0, IMG_AQ = 3 * SQ_BYTES, IMG_GATES = 6 * SQ_BYTES, IMG_BYTES = IMG_GATES + (int)sizeof(Gates);
// NTH threads: an image to shared memory.
template <int NTH>
__device__ __forceinline__ void load_image(uint32_t dst, const uint8_t* src, int t) {
#pragma unroll 4
  for (int i = t; i < IMG_BYTES / 16; i += NTH) cp_async16(dst + 16 * i, src + 16 * i, true);
}

// 128 threads (t = 0..127): from the loaded K, Q planes and the gates, the three planes of
// Aq diag(beta) and of T.  M is the f32 work matrix; it may lie over the Q
// planes (their product comes first).  Entries of 16-blocks
// above the diagonal are not written: nobody reads them.
template <int XS, int KN>
__device__ __forceinline__ void chunk_matrices(uint32_t k, uint32_t q, const Gates& g, float scale, float* M,
                                               uint8_t* aq, uint8_t* tp, int t, int bar) {
  constexpr int RB = KN * 2, PB = Q * RB, KK = KN / 16;
  const int w = t / 32, lane = t % 32, gr = lane / 4, q2 = 2 * (lane % 4);
#pragma unroll
  for (int pass = 1; pass >= 0; --pass) {   // Q K^T, then K K^T with the rows dealt the other way round
    if (pass == 0) bar_sync(bar, 128);
    const int I = pass ? 3 - w : w, r0 = 16 * I + gr;
    uint32_t a[XS == 1 ? KK : 1][XS][4];   // this row block's operand (bf16: kept for all column blocks)
    if constexpr (XS == 1)
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) ldsm4(a[kk][0], at_a<RB>(pass ? q : k, 16 * I, 2 * kk, lane));
    const float ra[2] = {g.a[r0], g.a[r0 + 8]};
    const float sc = pass ? scale : 1.f;
#pragma unroll 1
    for (int J = 0; J <= I; ++J) {
      float d[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) d[i][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        uint32_t b[XS][4];
#pragma unroll
        for (int s = 0; s < XS; ++s) ldsm4(b[s], at_b<RB>(k + s * PB, 16 * J, 2 * kk, lane));
        if constexpr (XS > 1)
#pragma unroll
          for (int s = 0; s < XS; ++s) ldsm4(a[0][s], at_a<RB>((pass ? q : k) + s * PB, 16 * I, 2 * kk, lane));
        mma_planes<XS, XS, XS, XS == 3>(d[0], d[1], a[XS == 1 ? kk : 0], b);
      }
      const float cIJ = g.c[4 * I + J] * sc;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int j = 16 * J + 8 * n + q2;
        float v[4];
        if (J < I) {
          const float2 bb = *reinterpret_cast<const float2*>(g.bb + j);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = d[n][e] * (ra[e >> 1] * cIJ) * (e & 1 ? bb.y : bb.x);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = r0 + 8 * (e >> 1), jj = j + (e & 1);
            const float D = exp2f((g.lh[i] - g.lh[jj]) + (g.ll[i] - g.ll[jj])) * g.beta[jj];
            v[e] = (pass ? jj <= i : jj < i) ? d[n][e] * D * sc : 0.f;
          }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int i = r0 + 8 * r;
          if (pass == 0) {
            *reinterpret_cast<float2*>(M + i * AM + j) = make_float2(v[2 * r], v[2 * r + 1]);
          } else {
            uint32_t p[3];
            split2<3>(v[2 * r], v[2 * r + 1], p);
#pragma unroll
            for (int s = 0; s < 3; ++s)
              *reinterpret_cast<uint32_t*>(aq + s * SQ_BYTES + tile_off<SQ_RB>(i, 2 * J + n) + 2 * q2) = p[s];
          }
        }
      }
    }
  }
  bar_sync(bar, 128);
  invert_unit_lower(M, t, bar);
#pragma unroll 1
  for (int idx = t; idx < 320; idx += 128) {   // 10 blocks x 16 rows x two 8-wide pieces
    const int blk = idx / 32, bi = blk < 1 ? 0 : blk < 3 ? 1 : blk < 6 ? 2 : 3, bj = blk - bi * (bi + 1) / 2;
    const int i = 16 * bi + (idx % 32) / 2, c = 2 * bj + idx % 2;
    const float4 x = *reinterpret_cast<const float4*>(M + i * AM + 8 * c);
    const float4 y = *reinterpret_cast<const float4*>(M + i * AM + 8 * c + 4);
    uint32_t r[4][3];
    split2<3>(x.x, x.y, r[0]);
    split2<3>(x.z, x.w, r[1]);
    split2<3>(y.x, y.y, r[2]);
    split2<3>(y.z, y.w, r[3]);
#pragma unroll
    for (int s = 0; s < 3; ++s)
      *reinterpret_cast<uint4*>(tp + s * SQ_BYTES + tile_off<SQ_RB>(i, c)) =
          make_uint4(r[0][s], r[1][s], r[2][s], r[3][s]);
  }
}

}  // namespace delta
}  // namespace tssm
