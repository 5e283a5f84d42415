// Group norm with an activation, channels last, forward and backward.
//
// x [Bt, L, C]: for each batch row b and group g of Cg = C / groups channels,
//     mean, var over the L * Cg values;  r = 1 / sqrt(var + eps)
//     n = (x - mean) r ;  z = n w_c + b_c ;  y = act(z)
// and with dz = dy act'(z), gr = dz w:
//     dx = r (gr - mean(gr) - n mean(gr n)),  dw_c = sum dz n,  db_c = sum dz.
// All of it is bound by HBM: x in and y out (backward: x, dy in, dx out).
//
// L = 1 (one token's head groups): 1 to 32 lanes hold a group in registers, so
// x is read once.  A thread keeps the same channels from row to row, so its
// weights (and the backward's dw, db sums) stay in registers.
// L > 1: a statistics pass and an apply pass.  The batch goes through them in
// pieces of about L2_BYTES, so that the second pass finds most of its inputs in L2
// (it reads 13 of 61 MB from HBM at 4 x 5000 x 768 f32, and 25 of 134 MB in the
// backward at 8 x 4096 x 1024 bf16).
// Variances are merged from per-batch means and squared deviations (Chan's
// pairwise update), never as E[x^2] - E[x]^2.
// Measured: 32768 tokens x 4096 bf16 with SiLU take 107 us (5.0 TB/s of x and y);
// 6000 x 1536 f32 with the backward 57 us (22 forward, 30 backward, 5 the sums of dw and db).  L > 1: 39 us at 4 x 5000 x 768 f32 (3.2 TB/s:
// 14 us statistics, 6 merge, 19 apply), 140 us with the backward at 8 x 4096 x 1024 bf16.
#include "common.cuh"

namespace tssm {
namespace {

constexpr int NT = 256;
constexpr int64_t L2_BYTES = 64ll << 20;   // of 126 MB: room for the outputs written meanwhile

// V elements moved as one access: R as they lie in memory, cvt to f32.
template <typename T, int V> struct vec;
template <> struct vec<float, 4> {
  using R = float4;
  __device__ static void cvt(const R& v, float (&f)[4]) {
    f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
  }
  __device__ static R pack(const float (&f)[4]) { return make_float4(f[0], f[1], f[2], f[3]); }
};
template <> struct vec<__nv_bfloat16, 8> {
  using R = uint4;
  __device__ static void cvt(const R& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ static R pack(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct vec<__nv_bfloat16, 4> {
  using R = uint2;
  __device__ static void cvt(const R& v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x << 16); f[1] = __uint_as_float(v.x & 0xffff0000u);
    f[2] = __uint_as_float(v.y << 16); f[3] = __uint_as_float(v.y & 0xffff0000u);
  }
  __device__ static R pack(const float (&f)[4]) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
    return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  }
};
template <> struct vec<float, 1> {
  using R = float;
  __device__ static void cvt(const R& v, float (&f)[1]) { f[0] = v; }
  __device__ static R pack(const float (&f)[1]) { return f[0]; }
};
template <> struct vec<__nv_bfloat16, 1> {
  using R = uint16_t;
  __device__ static void cvt(const R& v, float (&f)[1]) { f[0] = __uint_as_float((uint32_t)v << 16); }
  __device__ static R pack(const float (&f)[1]) { return __bfloat16_as_ushort(__float2bfloat16_rn(f[0])); }
};
template <typename T, int V> using raw = typename vec<T, V>::R;
template <typename T, int V>
__device__ __forceinline__ raw<T, V> ldr(const T* p) { return *reinterpret_cast<const raw<T, V>*>(p); }
template <typename T, int V>
__device__ __forceinline__ void stv(T* p, const float (&f)[V]) { *reinterpret_cast<raw<T, V>*>(p) = vec<T, V>::pack(f); }

// sigmoid(z).  A bf16 result takes the hardware exponential and reciprocal (relative
// error near 2^-21, far below bf16's 2^-9); f32 takes the accurate ones.  z far below 0
// gives 1 / inf = 0.
template <typename T>
__device__ __forceinline__ float sigmoid(float z) {
  if constexpr (std::is_same<T, float>::value) {
    return 1.f / (1.f + expf(-z));
  } else {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-1.4426950408889634f * z));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
    return r;
  }
}
template <typename T, bool SILU>
__device__ __forceinline__ float act(float z) {
  return SILU ? z * sigmoid<T>(z) : z;
}
template <typename T, bool SILU>
__device__ __forceinline__ float dact(float z) {
  if (!SILU) return 1.f;
  const float s = sigmoid<T>(z);
  return s * (1.f + z * (1.f - s));
}

// Element-wise arithmetic on V values, two lanes an instruction where V is even: a bf16
// pass at the HBM rate leaves about 20 instructions per value.
template <int V>
__device__ __forceinline__ float vsum(const float (&v)[V]) {
  if constexpr (V % 2 == 0) {
    float2 s = make_float2(v[0], v[1]);
#pragma unroll
    for (int i = 2; i < V; i += 2) s = fadd2(s, make_float2(v[i], v[i + 1]));
    return s.x + s.y;
  } else {
    float s = v[0];
#pragma unroll
    for (int i = 1; i < V; ++i) s += v[i];
    return s;
  }
}
// v += c
template <int V>
__device__ __forceinline__ void vadd(float (&v)[V], float c) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float2 r = fadd2(make_float2(v[i], v[i + 1]), make_float2(c, c));
      v[i] = r.x;
      v[i + 1] = r.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] += c;
  }
}
// d = a * b + c (any of b, c broadcast by the caller's arrays)
template <int V>
__device__ __forceinline__ void vfma(float (&d)[V], const float (&a)[V], const float (&b)[V], const float (&c)[V]) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float2 r = ffma2(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]), make_float2(c[i], c[i + 1]));
      d[i] = r.x;
      d[i + 1] = r.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] = a[i] * b[i] + c[i];
  }
}
template <int V>
__device__ __forceinline__ void vscale(float (&d)[V], const float (&a)[V], float c) {   // d = a * c
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float2 r = fmul2(make_float2(a[i], a[i + 1]), make_float2(c, c));
      d[i] = r.x;
      d[i + 1] = r.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] = a[i] * c;
  }
}
template <int V>
__device__ __forceinline__ float vdot(const float (&a)[V], const float (&b)[V]) {
  if constexpr (V % 2 == 0) {
    float2 s = fmul2(make_float2(a[0], a[1]), make_float2(b[0], b[1]));
#pragma unroll
    for (int i = 2; i < V; i += 2) s = ffma2(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]), s);
    return s.x + s.y;
  } else {
    float s = a[0] * b[0];
#pragma unroll
    for (int i = 1; i < V; ++i) s += a[i] * b[i];
    return s;
  }
}
// What the backward needs of V values x with their dy: n = (x - mean) rstd into x, and
// dz = dy act'(n w + b) into d.  sh = -mean rstd.
template <typename T, int V, bool SILU>
__device__ __forceinline__ void to_dz(float (&x)[V], float (&d)[V], const float (&w)[V], const float (&b)[V], float r,
                                      float sh) {
  float rr[V], ss[V], z[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    rr[i] = r;
    ss[i] = sh;
  }
  vfma<V>(x, x, rr, ss);
  if (SILU) {
    vfma<V>(z, x, w, b);
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] *= dact<T, true>(z[i]);
  }
}

__device__ __forceinline__ float lane_sum(float v, int w) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < w) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// ------------------------------------------------------------------ L = 1
// A slot of TL lanes owns one group; gpb groups x rpb rows per block and pass.
struct TokenGeom {
  int tl, gpb, rpb, cblocks;
};

template <typename T, int V, int NV, bool SILU>
__global__ void __launch_bounds__(NT, NV == 1 ? 4 : NV == 2 ? 3 : 2) gn_token_kernel(const T* __restrict__ x, const float* __restrict__ w,
                                                      const float* __restrict__ b, T* __restrict__ y,
                                                      float* __restrict__ mean_o, float* __restrict__ rstd_o,
                                                      int64_t rows, int groups, int Cg, float eps, TokenGeom ge) {
  constexpr int U = NV == 1 ? 2 : 1;   // rows in flight per thread (more resident warps beat more rows)
  const int slot = threadIdx.x / ge.tl, lane = threadIdx.x % ge.tl;
  const int g = blockIdx.y * ge.gpb + slot % ge.gpb, rr = slot / ge.gpb;
  const bool live = rr < ge.rpb && g < groups;
  const int64_t C = (int64_t)groups * Cg;
  const int nvec = Cg / V;
  const float inv = 1.f / (float)Cg;
  float wr[NV][V], br[NV][V];
  bool has[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    has[j] = live && lane + j * ge.tl < nvec;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = g * Cg + (lane + j * ge.tl) * V + i;
      wr[j][i] = has[j] ? w[c] : 0.f;
      br[j][i] = has[j] ? b[c] : 0.f;
    }
  }
  const int64_t step = (int64_t)gridDim.x * ge.rpb;
  const int64_t off = (int64_t)g * Cg + lane * V;
  // The next rows' loads go out before this row's arithmetic (as they lie in memory: half
  // the registers of f32).  The loop bound is the block's, so that every lane of a warp
  // takes part in the shuffles.
  raw<T, V> nx[U][NV];
  auto fetch = [&](int64_t r0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + rr + u * step;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        nx[u][j] = has[j] && r < rows ? ldr<T, V>(x + r * C + off + j * ge.tl * V) : raw<T, V>{};
    }
  };
  int64_t r0 = (int64_t)blockIdx.x * ge.rpb;
  fetch(r0);
  for (; r0 < rows; r0 += step * U) {
    raw<T, V> cur[U][NV];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < NV; ++j) cur[u][j] = nx[u][j];
    fetch(r0 + step * U);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + rr + u * step;
      float v[NV][V];
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        vec<T, V>::cvt(cur[u][j], v[j]);
        s += vsum<V>(v[j]);
      }
      const float mean = lane_sum(s, ge.tl) * inv;
      float m2 = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        vadd<V>(v[j], -mean);
        const float q = vdot<V>(v[j], v[j]);
        m2 += has[j] ? q : 0.f;
      }
      const float rstd = rsqrtf(lane_sum(m2, ge.tl) * inv + eps);
      if (r >= rows) continue;   // after the shuffles
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (!has[j]) continue;
        float o[V];
        vscale<V>(o, v[j], rstd);
        vfma<V>(o, o, wr[j], br[j]);
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = act<T, SILU>(o[i]);
        stv<T, V>(y + r * C + off + j * ge.tl * V, o);
      }
      if (mean_o && live && lane == 0) {
        mean_o[r * groups + g] = mean;
        rstd_o[r * groups + g] = rstd;
      }
    }
  }
}

// Backward: dx, and per (block, row slot) partial sums of dw and db: part [2][parts][C].
template <typename T, int V, int NV, bool SILU>
__global__ void __launch_bounds__(NT, NV == 1 ? 3 : NV == 2 ? 2 : 1) gn_token_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                          const float* __restrict__ w, const float* __restrict__ b,
                                                          const float* __restrict__ mean_i,
                                                          const float* __restrict__ rstd_i, T* __restrict__ dx,
                                                          float* __restrict__ part, int64_t rows, int groups, int Cg,
                                                          TokenGeom ge) {
  let_next_start();
  wait_for_previous();
  const int slot = threadIdx.x / ge.tl, lane = threadIdx.x % ge.tl;
  const int g = blockIdx.y * ge.gpb + slot % ge.gpb, rr = slot / ge.gpb;
  const bool live = rr < ge.rpb && g < groups;
  const int64_t C = (int64_t)groups * Cg;
  const int nvec = Cg / V;
  const float inv = 1.f / (float)Cg;
  float wr[NV][V], br[NV][V], aw[NV][V], ab[NV][V];
  bool has[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    has[j] = live && lane + j * ge.tl < nvec;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = g * Cg + (lane + j * ge.tl) * V + i;
      wr[j][i] = has[j] ? w[c] : 0.f;
      br[j][i] = has[j] ? b[c] : 0.f;
      aw[j][i] = ab[j][i] = 0.f;
    }
  }
  const int64_t step = (int64_t)gridDim.x * ge.rpb;
  const int64_t off = (int64_t)g * Cg + lane * V;
  raw<T, V> nx[NV], nd[NV];
  float nm, nr;
  auto fetch = [&](int64_t r0) {   // the next row, before this one's arithmetic
    const int64_t r = r0 + rr;
    const bool in = live && r < rows;
    nm = in ? mean_i[r * groups + g] : 0.f;
    nr = in ? rstd_i[r * groups + g] : 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const bool ok = has[j] && in;
      const int64_t at = r * C + off + j * ge.tl * V;
      nx[j] = ok ? ldr<T, V>(x + at) : raw<T, V>{};
      nd[j] = ok ? ldr<T, V>(dy + at) : raw<T, V>{};
    }
  };
  int64_t r0 = (int64_t)blockIdx.x * ge.rpb;
  fetch(r0);
  for (; r0 < rows; r0 += step) {
    float v[NV][V], d[NV][V];
    const float mean = nm, rstd = nr;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      vec<T, V>::cvt(nx[j], v[j]);
      vec<T, V>::cvt(nd[j], d[j]);
    }
    fetch(r0 + step);
    const int64_t r = r0 + rr;
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {   // lanes without values have w = dy = 0
      to_dz<T, V, SILU>(v[j], d[j], wr[j], br[j], rstd, -mean * rstd);
      vfma<V>(aw[j], d[j], v[j], aw[j]);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        ab[j][i] += d[j][i];
        d[j][i] *= wr[j][i];
      }
      s0 += vsum<V>(d[j]);
      s1 += vdot<V>(d[j], v[j]);
    }
    s0 = lane_sum(s0, ge.tl) * inv;
    s1 = lane_sum(s1, ge.tl) * inv;
    if (r >= rows) continue;   // after the shuffles
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!has[j]) continue;
      float o[V];
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = rstd * (d[j][i] - s0 - v[j][i] * s1);
      stv<T, V>(dx + r * C + off + j * ge.tl * V, o);
    }
  }
  const int64_t parts = (int64_t)gridDim.x * ge.rpb;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (!has[j]) continue;
    const int64_t at = ((int64_t)blockIdx.x * ge.rpb + rr) * C + (int64_t)g * Cg + (lane + j * ge.tl) * V;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      part[at + i] = aw[j][i];
      part[parts * C + at + i] = ab[j][i];
    }
  }
}

// out0[c] = sum_p part[0][p][c], out1[c] = sum_p part[1][p][c], in a fixed order.
__global__ void __launch_bounds__(NT) gn_column_sum_kernel(const float* __restrict__ part, float* __restrict__ out0,
                                                           float* __restrict__ out1, int64_t parts, int64_t C) {
  let_next_start();
  wait_for_previous();
  __shared__ float sm[8][33];
  const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x % 32;
  const int ty = threadIdx.x / 32;
  const float* src = part + (int64_t)blockIdx.y * parts * C;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < C) {
    int64_t p = ty;
    for (; p + 24 < parts; p += 32)
#pragma unroll
      for (int k = 0; k < 4; ++k) s[k] += src[(p + 8 * k) * C + c];
    for (; p < parts; p += 8) s[0] += src[p * C + c];
  }
  sm[ty][threadIdx.x % 32] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  if (ty == 0 && c < C) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) t += sm[k][threadIdx.x];
    (blockIdx.y ? out1 : out0)[c] = t;
  }
}

// ------------------------------------------------------------------ L > 1
// A thread owns V adjacent channels (one group) of rows l0 + ty, l0 + ty + TY, ...
// cols threads across the channels, rows_y of them deep; blockIdx = (row chunk, column block, b).
struct MapGeom {
  int cols, rows_y, cblocks;
  int64_t chunk, nchunks;   // rows per chunk
};
constexpr int UR = 4;   // rows in flight per thread

// (n, m, q) += (n2, m2, q2): counts, means, sums of squared deviations.
__device__ __forceinline__ void chan(float& n, float& m, float& q, float n2, float m2, float q2) {
  if (n2 == 0.f) return;
  const float t = n + n2, d = m2 - m, f = __fdividef(n2, t);
  m += d * f;
  q += q2 + d * d * n * f;
  n = t;
}

// st [b][chunk][C / V] x (mean, squared deviations) of each thread column.
template <typename T, int V>
__global__ void __launch_bounds__(NT, 4) gn_stats_kernel(const T* __restrict__ x, float2* __restrict__ st, int64_t L,
                                                      int64_t C, MapGeom ge) {
  let_next_start();
  wait_for_previous();
  __shared__ float sn[NT], sm[NT], sq[NT];
  const int tx = threadIdx.x % ge.cols, ty = threadIdx.x / ge.cols;
  const int64_t cv = (int64_t)blockIdx.y * ge.cols + tx, ncv = C / V;
  const int64_t l0 = (int64_t)blockIdx.x * ge.chunk, l1 = min(L, l0 + ge.chunk);
  float n = 0.f, m = 0.f, q = 0.f;
  if (ty < ge.rows_y && cv < ncv) {
    const T* p = x + ((int64_t)blockIdx.z * L) * C + cv * V;
    raw<T, V> nx[UR];
    auto fetch = [&](int64_t l) {
#pragma unroll
      for (int u = 0; u < UR; ++u) {
        const int64_t lu = l + (int64_t)u * ge.rows_y;
        nx[u] = lu < l1 ? ldr<T, V>(p + lu * C) : raw<T, V>{};
      }
    };
    fetch(l0 + ty);
    for (int64_t l = l0 + ty; l < l1; l += (int64_t)ge.rows_y * UR) {
      float v[UR][V];
      float cnt = 0.f, s = 0.f;
#pragma unroll
      for (int u = 0; u < UR; ++u) vec<T, V>::cvt(nx[u], v[u]);
      fetch(l + (int64_t)ge.rows_y * UR);
#pragma unroll
      for (int u = 0; u < UR; ++u)
        if (l + (int64_t)u * ge.rows_y < l1) {
          cnt += V;
          s += vsum<V>(v[u]);
        }
      const float mu = __fdividef(s, cnt);
      float d2 = 0.f;
#pragma unroll
      for (int u = 0; u < UR; ++u)
        if (l + (int64_t)u * ge.rows_y < l1) {
          vadd<V>(v[u], -mu);
          d2 += vdot<V>(v[u], v[u]);
        }
      chan(n, m, q, cnt, mu, d2);
    }
  }
  sn[threadIdx.x] = n;
  sm[threadIdx.x] = m;
  sq[threadIdx.x] = q;
  __syncthreads();
  if (ty == 0 && cv < ncv) {
    for (int k = 1; k < ge.rows_y; ++k)
      chan(n, m, q, sn[k * ge.cols + tx], sm[k * ge.cols + tx], sq[k * ge.cols + tx]);
    st[((int64_t)blockIdx.z * ge.nchunks + blockIdx.x) * ncv + cv] = make_float2(m, q);
  }
}

__device__ __forceinline__ float block_sum(float v, float* sm) {   // every thread gets the sum
  v = lane_sum(v, 32);
  if (threadIdx.x % 32 == 0) sm[threadIdx.x / 32] = v;
  __syncthreads();
  float t = 0.f;
  for (int k = 0; k < (int)blockDim.x / 32; ++k) t += sm[k];
  __syncthreads();
  return t;
}

// mean, rstd of one (b, g) per block, from the partial statistics: their weighted mean,
// then the squared deviations about it (two passes over values that stay in L1).
__global__ void __launch_bounds__(NT) gn_merge_kernel(const float2* __restrict__ st, float* __restrict__ mean_o,
                                                      float* __restrict__ rstd_o, int64_t L, int64_t ncv, int per,
                                                      int V, int groups, int64_t chunk, int64_t nchunks, float eps) {
  let_next_start();
  wait_for_previous();
  __shared__ float sm[NT / 32];
  const int64_t b = blockIdx.y;
  const int g = blockIdx.x;
  const float2* p = st + b * nchunks * ncv + (int64_t)g * per;
  const int n = (int)(nchunks * per);
  const float inv = 1.f / ((float)L * (float)(per * V)), last = (float)(L - (nchunks - 1) * chunk) * V;
  float s = 0.f;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += NT) {
    const int ck = i / per;
    s += (ck == nchunks - 1 ? last : (float)chunk * V) * p[(int64_t)ck * ncv + (i - ck * per)].x;
  }
  const float mean = block_sum(s, sm) * inv;
  float q = 0.f;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += NT) {
    const int ck = i / per;
    const float2 e = p[(int64_t)ck * ncv + (i - ck * per)];
    q += e.y + (ck == nchunks - 1 ? last : (float)chunk * V) * (e.x - mean) * (e.x - mean);
  }
  q = block_sum(q, sm);
  if (threadIdx.x == 0) {
    mean_o[b * groups + g] = mean;
    rstd_o[b * groups + g] = rsqrtf(q * inv + eps);
  }
}

template <typename T, int V, bool SILU>
__global__ void __launch_bounds__(NT, 4) gn_apply_kernel(const T* __restrict__ x, const float* __restrict__ w,
                                                      const float* __restrict__ b, const float* __restrict__ mean,
                                                      const float* __restrict__ rstd, T* __restrict__ y, int64_t L,
                                                      int64_t C, int groups, int Cg, MapGeom ge) {
  let_next_start();
  wait_for_previous();
  const int tx = threadIdx.x % ge.cols, ty = threadIdx.x / ge.cols;
  const int64_t cv = (int64_t)blockIdx.y * ge.cols + tx;
  if (ty >= ge.rows_y || cv >= C / V) return;
  const int64_t c = cv * V, bz = blockIdx.z;
  const float m = mean[bz * groups + c / Cg], r = rstd[bz * groups + c / Cg];
  float a[V], o[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    a[i] = r * w[c + i];
    o[i] = b[c + i];
  }
  const int64_t l0 = (int64_t)blockIdx.x * ge.chunk, l1 = min(L, l0 + ge.chunk);
  const T* px = x + bz * L * C + c;
  T* py = y + bz * L * C + c;
  raw<T, V> nx[UR];
  auto fetch = [&](int64_t l) {
#pragma unroll
    for (int u = 0; u < UR; ++u) {
      const int64_t lu = l + (int64_t)u * ge.rows_y;
      nx[u] = lu < l1 ? ldr<T, V>(px + lu * C) : raw<T, V>{};
    }
  };
  fetch(l0 + ty);
  for (int64_t l = l0 + ty; l < l1; l += (int64_t)ge.rows_y * UR) {
    raw<T, V> cur[UR];
#pragma unroll
    for (int u = 0; u < UR; ++u) cur[u] = nx[u];
    fetch(l + (int64_t)ge.rows_y * UR);
#pragma unroll
    for (int u = 0; u < UR; ++u) {
      const int64_t lu = l + (int64_t)u * ge.rows_y;
      if (lu >= l1) break;
      float v[V];
      vec<T, V>::cvt(cur[u], v);
      vadd<V>(v, -m);
      vfma<V>(v, v, a, o);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = act<T, SILU>(v[i]);
      stv<T, V>(py + lu * C, v);
    }
  }
}

// part [b][chunk][2][C]: sums of dz n and dz over the chunk's rows.
template <typename T, int V, bool SILU>
__global__ void __launch_bounds__(NT, 2) gn_bwd_sums_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                         const float* __restrict__ w, const float* __restrict__ b,
                                                         const float* __restrict__ mean,
                                                         const float* __restrict__ rstd, float* __restrict__ part,
                                                         int64_t L, int64_t C, int groups, int Cg, MapGeom ge) {
  let_next_start();
  wait_for_previous();
  __shared__ float s0[NT][V], s1[NT][V];
  const int tx = threadIdx.x % ge.cols, ty = threadIdx.x / ge.cols;
  const int64_t cv = (int64_t)blockIdx.y * ge.cols + tx, c = cv * V, bz = blockIdx.z;
  const bool live = ty < ge.rows_y && cv < C / V;
  float aw[V], ab[V];
#pragma unroll
  for (int i = 0; i < V; ++i) aw[i] = ab[i] = 0.f;
  if (live) {
    const float m = mean[bz * groups + c / Cg], r = rstd[bz * groups + c / Cg];
    float wr[V], br[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      wr[i] = w[c + i];
      br[i] = b[c + i];
    }
    const int64_t l0 = (int64_t)blockIdx.x * ge.chunk, l1 = min(L, l0 + ge.chunk);
    const int64_t base = bz * L * C + c;
    raw<T, V> nx[UR], nd[UR];
    auto fetch = [&](int64_t l) {
#pragma unroll
      for (int u = 0; u < UR; ++u) {
        const int64_t lu = l + (int64_t)u * ge.rows_y;
        nx[u] = lu < l1 ? ldr<T, V>(x + base + lu * C) : raw<T, V>{};
        nd[u] = lu < l1 ? ldr<T, V>(dy + base + lu * C) : raw<T, V>{};
      }
    };
    fetch(l0 + ty);
    for (int64_t l = l0 + ty; l < l1; l += (int64_t)ge.rows_y * UR) {
      raw<T, V> cx[UR], cd[UR];
#pragma unroll
      for (int u = 0; u < UR; ++u) {
        cx[u] = nx[u];
        cd[u] = nd[u];
      }
      fetch(l + (int64_t)ge.rows_y * UR);
#pragma unroll
      for (int u = 0; u < UR; ++u) {   // rows behind the chunk have dy = 0
        float v[V], d[V];
        vec<T, V>::cvt(cx[u], v);
        vec<T, V>::cvt(cd[u], d);
        to_dz<T, V, SILU>(v, d, wr, br, r, -m * r);
        vfma<V>(aw, d, v, aw);
#pragma unroll
        for (int i = 0; i < V; ++i) ab[i] += d[i];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    s0[threadIdx.x][i] = aw[i];
    s1[threadIdx.x][i] = ab[i];
  }
  __syncthreads();
  if (ty == 0 && live) {
    for (int k = 1; k < ge.rows_y; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        aw[i] += s0[k * ge.cols + tx][i];
        ab[i] += s1[k * ge.cols + tx][i];
      }
    float* o = part + ((bz * ge.nchunks + blockIdx.x) * 2) * C + c;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      o[i] = aw[i];
      o[C + i] = ab[i];
    }
  }
}

// One (b, g) per block of 1024: per-channel sums over the chunks into chan_sum [2][Bt][C], and
// the group means of gr and gr n into gm [Bt][groups] (x: mean gr, y: mean gr n).  A warp per
// 32 channels and every 32nd chunk.
__global__ void __launch_bounds__(1024) gn_bwd_merge_kernel(const float* __restrict__ part, const float* __restrict__ w,
                                                            float* __restrict__ chan_sum, float2* __restrict__ gm,
                                                            int64_t L, int64_t C, int groups, int Cg, int64_t nchunks,
                                                            int64_t Bt, int64_t b0) {
  let_next_start();
  wait_for_previous();
  __shared__ float sa[32][33], sb[32][33];
  const int64_t b = blockIdx.y;
  const int g = blockIdx.x, tx = threadIdx.x % 32, ty = threadIdx.x / 32;
  float ga = 0.f, gb = 0.f;
  for (int i0 = 0; i0 < Cg; i0 += 32) {
    const int64_t c = (int64_t)g * Cg + i0 + tx;
    const bool in = i0 + tx < Cg;
    float a = 0.f, d = 0.f;
    if (in) {
#pragma unroll 4
      for (int64_t k = ty; k < nchunks; k += 32) {
        const float* p = part + (b * nchunks + k) * 2 * C + c;
        a += p[0];
        d += p[C];
      }
    }
    sa[ty][tx] = a;
    sb[ty][tx] = d;
    __syncthreads();
    // the 32 partial sums of a channel: a warp per channel, chunks across its lanes
    a = lane_sum(sa[tx][ty], 32);
    d = lane_sum(sb[tx][ty], 32);
    if (tx == 0 && i0 + ty < Cg) {
      const int64_t cc = (int64_t)g * Cg + i0 + ty;
      chan_sum[(b0 + b) * C + cc] = a;
      chan_sum[(Bt + b0 + b) * C + cc] = d;
      ga += a * w[cc];
      gb += d * w[cc];
    }
    __syncthreads();
  }
  if (tx == 0) {
    sa[0][ty] = ga;
    sb[0][ty] = gb;
  }
  __syncthreads();
  if (ty == 0) {
    ga = lane_sum(sa[0][tx], 32);
    gb = lane_sum(sb[0][tx], 32);
    const float inv = 1.f / ((float)L * (float)Cg);
    if (tx == 0) gm[b * groups + g] = make_float2(gb * inv, ga * inv);
  }
}

template <typename T, int V, bool SILU>
__global__ void __launch_bounds__(NT, 2) gn_bwd_apply_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                          const float* __restrict__ w, const float* __restrict__ b,
                                                          const float* __restrict__ mean,
                                                          const float* __restrict__ rstd,
                                                          const float2* __restrict__ gm, T* __restrict__ dx,
                                                          int64_t L, int64_t C, int groups, int Cg, MapGeom ge) {
  let_next_start();
  wait_for_previous();
  const int tx = threadIdx.x % ge.cols, ty = threadIdx.x / ge.cols;
  const int64_t cv = (int64_t)blockIdx.y * ge.cols + tx;
  if (ty >= ge.rows_y || cv >= C / V) return;
  const int64_t c = cv * V, bz = blockIdx.z, gi = bz * groups + c / Cg;
  const float m = mean[gi], r = rstd[gi];
  const float2 mm = gm[gi];
  float wr[V], br[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    wr[i] = w[c + i];
    br[i] = b[c + i];
  }
  const int64_t l0 = (int64_t)blockIdx.x * ge.chunk, l1 = min(L, l0 + ge.chunk);
  const int64_t base = bz * L * C + c;
  raw<T, V> nx[UR], nd[UR];
  auto fetch = [&](int64_t l) {
#pragma unroll
    for (int u = 0; u < UR; ++u) {
      const int64_t lu = l + (int64_t)u * ge.rows_y;
      nx[u] = lu < l1 ? ldr<T, V>(x + base + lu * C) : raw<T, V>{};
      nd[u] = lu < l1 ? ldr<T, V>(dy + base + lu * C) : raw<T, V>{};
    }
  };
  fetch(l0 + ty);
  for (int64_t l = l0 + ty; l < l1; l += (int64_t)ge.rows_y * UR) {
    raw<T, V> cx[UR], cd[UR];
#pragma unroll
    for (int u = 0; u < UR; ++u) {
      cx[u] = nx[u];
      cd[u] = nd[u];
    }
    fetch(l + (int64_t)ge.rows_y * UR);
#pragma unroll
    for (int u = 0; u < UR; ++u) {
      const int64_t lu = l + (int64_t)u * ge.rows_y;
      if (lu >= l1) break;
      float v[V], d[V];
      vec<T, V>::cvt(cx[u], v);
      vec<T, V>::cvt(cd[u], d);
      to_dz<T, V, SILU>(v, d, wr, br, r, -m * r);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = r * (d[i] * wr[i] - mm.x - v[i] * mm.y);
      stv<T, V>(dx + base + lu * C, v);
    }
  }
}

// ------------------------------------------------------------------ host side
struct Norm {
  const void *x, *w, *b, *dy;
  void *y, *mean, *rstd;   // y: dx in the backward
  void *dw, *db, *ws;
  int64_t Bt, L, C;
  int groups, Cg;
  float eps;
  bool silu;
  cudaStream_t st;
};

// Elements per access: the widest that divides a group and that every base allows.
int width(int dtype, int Cg, uintptr_t bases) {
  const int es = dtype == TSSM_F32 ? 4 : 2;
  for (int v = 16 / es; v >= 4; v /= 2)
    if (Cg % v == 0 && (bases & (uintptr_t)(v * es - 1)) == 0) return v;
  return 1;
}

// Lanes and rows of the L = 1 kernels; nv = 0 when a group is too wide for 32 lanes x 4 accesses.
TokenGeom token_geom(int Cg, int groups, int V, int* nv) {
  const int nvec = Cg / V;
  *nv = nvec <= 32 ? 1 : nvec <= 64 ? 2 : nvec <= 128 ? 4 : 0;
  TokenGeom ge{1, 1, 1, 1};
  if (!*nv) return ge;
  while (ge.tl * *nv < nvec) ge.tl *= 2;
  const int slots = NT / ge.tl;
  ge.cblocks = (int)cdiv(groups, slots);
  ge.gpb = (int)cdiv(groups, ge.cblocks);
  ge.rpb = slots / ge.gpb;
  return ge;
}

// Row blocks of the L = 1 kernels: enough for `waves` resident sets, at most one pass each.
int64_t token_blocks(const TokenGeom& ge, int64_t rows, int per_sm) {
  const int64_t want = cdiv((int64_t)num_sms() * per_sm, ge.cblocks);
  return std::max<int64_t>(1, std::min(want, cdiv(rows, ge.rpb)));
}
constexpr int TOKEN_BWD_PER_SM = 3;

MapGeom map_geom(int64_t Bt, int64_t L, int64_t C, int V, bool bwd) {
  MapGeom ge;
  const int64_t ncv = C / V;
  ge.cblocks = (int)cdiv(ncv, NT);
  ge.cols = (int)cdiv(ncv, ge.cblocks);
  ge.rows_y = NT / ge.cols;
  // one set of resident blocks over the batch (launch bounds: 4 per SM forward, 2 backward),
  // and no chunk below one unrolled pass
  const int64_t want = std::max<int64_t>(1, (int64_t)num_sms() * (bwd ? 2 : 4) / (Bt * ge.cblocks));
  ge.chunk = std::max<int64_t>(cdiv(L, want), (int64_t)ge.rows_y * UR);
  ge.nchunks = cdiv(L, ge.chunk);
  return ge;
}

int64_t batch_piece(int64_t Bt, int64_t bytes_per_row) {
  // at most 32768 batch rows: they are a grid's y or z extent
  return std::max<int64_t>(1, std::min(std::min<int64_t>(Bt, 32768), L2_BYTES / std::max<int64_t>(1, bytes_per_row)));
}

// Workspace of the L > 1 passes: partial sums of one piece, group means, per-row channel sums.
int64_t map_part_floats(int64_t piece, int64_t L, int64_t C, int V, bool train) {
  const MapGeom ge = map_geom(piece, L, C, V, train);
  return piece * ge.nchunks * 2 * (train ? C : C / V);
}

template <typename T, int V, bool SILU>
void token_fwd(const Norm& a, const TokenGeom& ge, int nv) {
  dim3 grid((unsigned)token_blocks(ge, a.Bt, 8), (unsigned)ge.cblocks);
  auto go = [&](auto kern) {
    kern<<<grid, NT, 0, a.st>>>((const T*)a.x, (const float*)a.w, (const float*)a.b, (T*)a.y, (float*)a.mean,
                                (float*)a.rstd, a.Bt, a.groups, a.Cg, a.eps, ge);
  };
  if (nv == 1) go(gn_token_kernel<T, V, 1, SILU>);
  else if (nv == 2) go(gn_token_kernel<T, V, 2, SILU>);
  else go(gn_token_kernel<T, V, 4, SILU>);
}

template <typename T, int V, bool SILU>
void token_bwd(const Norm& a, const TokenGeom& ge, int nv) {
  dim3 grid((unsigned)token_blocks(ge, a.Bt, TOKEN_BWD_PER_SM), (unsigned)ge.cblocks);
  auto go = [&](auto kern) {
    kern<<<grid, NT, 0, a.st>>>((const T*)a.dy, (const T*)a.x, (const float*)a.w, (const float*)a.b,
                                (const float*)a.mean, (const float*)a.rstd, (T*)a.y, (float*)a.ws, a.Bt, a.groups,
                                a.Cg, ge);
  };
  if (nv == 1) go(gn_token_bwd_kernel<T, V, 1, SILU>);
  else if (nv == 2) go(gn_token_bwd_kernel<T, V, 2, SILU>);
  else go(gn_token_bwd_kernel<T, V, 4, SILU>);
  launch_after(gn_column_sum_kernel, dim3((unsigned)cdiv(a.C, 32), 2), NT, 0, a.st, (const float*)a.ws, (float*)a.dw,
               (float*)a.db, (int64_t)grid.x * ge.rpb, a.C);
}

template <typename T, int V, bool SILU>
void map_fwd(const Norm& a) {
  const int64_t row = a.L * a.C, piece = batch_piece(a.Bt, row * sizeof(T));
  const MapGeom ge = map_geom(piece, a.L, a.C, V, false);
  float2* st = (float2*)a.ws;
  for (int64_t b0 = 0; b0 < a.Bt; b0 += piece) {
    const int64_t nb = std::min(piece, a.Bt - b0);
    dim3 grid((unsigned)ge.nchunks, (unsigned)ge.cblocks, (unsigned)nb);
    const T* x = (const T*)a.x + b0 * row;
    float *mean = (float*)a.mean + b0 * a.groups, *rstd = (float*)a.rstd + b0 * a.groups;
    if (b0) launch_after(gn_stats_kernel<T, V>, grid, NT, 0, a.st, x, st, a.L, a.C, ge);
    else gn_stats_kernel<T, V><<<grid, NT, 0, a.st>>>(x, st, a.L, a.C, ge);
    launch_after(gn_merge_kernel, dim3((unsigned)a.groups, (unsigned)nb), NT, 0, a.st, (const float2*)st, mean, rstd,
                 a.L, a.C / V, a.Cg / V, V, a.groups, ge.chunk, ge.nchunks, a.eps);
    launch_after(gn_apply_kernel<T, V, SILU>, grid, NT, 0, a.st, x, (const float*)a.w, (const float*)a.b,
                 (const float*)mean, (const float*)rstd, (T*)a.y + b0 * row, a.L, a.C, a.groups, a.Cg, ge);
  }
}

template <typename T, int V, bool SILU>
void map_bwd(const Norm& a) {
  const int64_t row = a.L * a.C, piece = batch_piece(a.Bt, 2 * row * sizeof(T));
  const MapGeom ge = map_geom(piece, a.L, a.C, V, true);
  float* part = (float*)a.ws;
  float* chan_sum = part + map_part_floats(piece, a.L, a.C, V, true);
  float2* gm = (float2*)(chan_sum + 2 * a.Bt * a.C);
  for (int64_t b0 = 0; b0 < a.Bt; b0 += piece) {
    const int64_t nb = std::min(piece, a.Bt - b0);
    dim3 grid((unsigned)ge.nchunks, (unsigned)ge.cblocks, (unsigned)nb);
    const T *x = (const T*)a.x + b0 * row, *dy = (const T*)a.dy + b0 * row;
    const float *mean = (const float*)a.mean + b0 * a.groups, *rstd = (const float*)a.rstd + b0 * a.groups;
    if (b0)
      launch_after(gn_bwd_sums_kernel<T, V, SILU>, grid, NT, 0, a.st, dy, x, (const float*)a.w, (const float*)a.b, mean,
                   rstd, part, a.L, a.C, a.groups, a.Cg, ge);
    else
      gn_bwd_sums_kernel<T, V, SILU><<<grid, NT, 0, a.st>>>(dy, x, (const float*)a.w, (const float*)a.b, mean, rstd,
                                                            part, a.L, a.C, a.groups, a.Cg, ge);
    launch_after(gn_bwd_merge_kernel, dim3((unsigned)a.groups, (unsigned)nb), 1024, 0, a.st, (const float*)part,
                 (const float*)a.w, chan_sum, gm, a.L, a.C, a.groups, a.Cg, ge.nchunks, a.Bt, b0);
    launch_after(gn_bwd_apply_kernel<T, V, SILU>, grid, NT, 0, a.st, dy, x, (const float*)a.w, (const float*)a.b, mean,
                 rstd, (const float2*)gm, (T*)a.y + b0 * row, a.L, a.C, a.groups, a.Cg, ge);
  }
  launch_after(gn_column_sum_kernel, dim3((unsigned)cdiv(a.C, 32), 2), NT, 0, a.st, (const float*)chan_sum,
               (float*)a.dw, (float*)a.db, a.Bt, a.C);
}

template <typename T, int V, bool SILU>
void run(const Norm& a, bool bwd) {
  int nv = 0;
  const TokenGeom ge = token_geom(a.Cg, a.groups, V, &nv);
  const bool token = a.L == 1 && nv;
  if (bwd) token ? token_bwd<T, V, SILU>(a, ge, nv) : map_bwd<T, V, SILU>(a);
  else token ? token_fwd<T, V, SILU>(a, ge, nv) : map_fwd<T, V, SILU>(a);
}

template <typename T, int V>
void by_act(const Norm& a, bool bwd) {
  a.silu ? run<T, V, true>(a, bwd) : run<T, V, false>(a, bwd);
}

int width(const Norm& a, int dtype) {
  return width(dtype, a.Cg, reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y) |
                                reinterpret_cast<uintptr_t>(a.dy));
}

void dispatch(const Norm& a, int dtype, bool bwd) {
  const int V = width(a, dtype);
  if (dtype == TSSM_F32) V == 4 ? by_act<float, 4>(a, bwd) : by_act<float, 1>(a, bwd);
  else if (V == 8) by_act<__nv_bfloat16, 8>(a, bwd);
  else V == 4 ? by_act<__nv_bfloat16, 4>(a, bwd) : by_act<__nv_bfloat16, 1>(a, bwd);
}

int check_sizes(const char* name, int64_t Bt, int64_t L, int64_t C, int64_t groups, int act, int dtype) {
  TSSM_REQUIRE(Bt >= 0 && L >= 0 && C >= 0, "%s: negative size", name);
  TSSM_REQUIRE(groups >= 1 && C % groups == 0, "%s: C (%lld) must be a multiple of groups (%lld)", name, (long long)C,
               (long long)groups);
  TSSM_REQUIRE(act == 0 || act == 1, "%s: act must be 0 (none) or 1 (silu)", name);
  TSSM_REQUIRE(dtype == TSSM_F32 || dtype == TSSM_BF16, "%s: dtype must be f32 or bf16 (got %d)", name, dtype);
  TSSM_REQUIRE(C <= (int64_t(1) << 23) && L < (int64_t(1) << 31) && Bt < (int64_t(1) << 40), "%s: size out of range",
               name);
  return TSSM_OK;
}

}  // namespace
}  // namespace tssm

extern "C" int64_t tssm_group_norm_workspace_size(int64_t Bt, int64_t L, int64_t C, int64_t groups, int dtype,
                                                  int backward) {
  using namespace tssm;
  if (Bt <= 0 || L <= 0 || C <= 0 || groups <= 0 || C % groups) return 0;
  const int64_t es = dtype == TSSM_F32 ? 4 : 2;
  const int Cg = (int)(C / groups);
  int64_t need = 0;
  // over every access width the launch may settle on (alignment is not known here)
  for (int V : {8, 4, 1}) {
    if (Cg % V || V * es > 16) continue;
    int nv = 0;
    const TokenGeom ge = token_geom(Cg, (int)groups, V, &nv);
    int64_t f;
    if (L == 1 && nv) {
      f = backward ? 2 * token_blocks(ge, Bt, TOKEN_BWD_PER_SM) * ge.rpb * C : 0;
    } else {
      const int64_t piece = batch_piece(Bt, (backward ? 2 : 1) * L * C * es);
      f = map_part_floats(piece, L, C, V, backward);
      if (backward) f += 2 * Bt * C + 2 * piece * groups;
    }
    need = std::max(need, f * 4);
  }
  return need;
}

extern "C" int tssm_group_norm_act(const void* x, const void* weight, const void* bias, void* y, void* mean,
                                   void* rstd, void* workspace, int64_t workspace_bytes, int64_t Bt, int64_t L,
                                   int64_t C, int64_t groups, double eps, int act, int dtype, tssm_stream_t stream) {
  using namespace tssm;
  if (int e = check_sizes("group_norm_act", Bt, L, C, groups, act, dtype)) return e;
  TSSM_REQUIRE(eps >= 0, "group_norm_act: eps must not be negative (got %g)", eps);
  if (Bt * L * C == 0) return TSSM_OK;
  TSSM_REQUIRE(x && weight && bias && y, "group_norm_act: null pointer");
  TSSM_REQUIRE((mean != nullptr) == (rstd != nullptr), "group_norm_act: mean and rstd go together");
  // with L = 1 and groups of up to 128 channels every access width takes the kernel that needs none
  TSSM_REQUIRE(mean || (L == 1 && C / groups <= 128), "group_norm_act: mean and rstd are needed");
  const int64_t need = tssm_group_norm_workspace_size(Bt, L, C, groups, dtype, 0);
  TSSM_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned16(workspace)),
               "group_norm_act: workspace of %lld bytes (16-byte aligned) needed, %lld given", (long long)need,
               (long long)workspace_bytes);
  const Norm a{x, weight, bias, nullptr, y, mean, rstd, nullptr, nullptr, workspace, Bt, L, C, (int)groups,
               (int)(C / groups), (float)eps, act == 1, reinterpret_cast<cudaStream_t>(stream)};
  dispatch(a, dtype, false);
  return check_launch("group_norm_act");
}

extern "C" int tssm_group_norm_act_bwd(const void* dy, const void* x, const void* weight, const void* bias,
                                       const void* mean, const void* rstd, void* dx, void* dweight, void* dbias,
                                       void* workspace, int64_t workspace_bytes, int64_t Bt, int64_t L, int64_t C,
                                       int64_t groups, int act, int dtype, tssm_stream_t stream) {
  using namespace tssm;
  if (int e = check_sizes("group_norm_act_bwd", Bt, L, C, groups, act, dtype)) return e;
  if (C == 0) return TSSM_OK;
  TSSM_REQUIRE(dweight && dbias, "group_norm_act_bwd: null pointer");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (Bt * L == 0) {
    if (cudaMemsetAsync(dweight, 0, C * 4, st) != cudaSuccess || cudaMemsetAsync(dbias, 0, C * 4, st) != cudaSuccess)
      return check_launch("group_norm_act_bwd: clear");
    return TSSM_OK;
  }
  TSSM_REQUIRE(dy && x && weight && bias && mean && rstd && dx, "group_norm_act_bwd: null pointer");
  const int64_t need = tssm_group_norm_workspace_size(Bt, L, C, groups, dtype, 1);
  TSSM_REQUIRE(workspace && workspace_bytes >= need && aligned16(workspace),
               "group_norm_act_bwd: workspace of %lld bytes (16-byte aligned) needed, %lld given", (long long)need,
               (long long)workspace_bytes);
  const Norm a{x, weight, bias, dy, dx, const_cast<void*>(mean), const_cast<void*>(rstd), dweight, dbias, workspace,
               Bt, L, C, (int)groups, (int)(C / groups), 0.f, act == 1, st};
  dispatch(a, dtype, true);
  return check_launch("group_norm_act_bwd");
}
