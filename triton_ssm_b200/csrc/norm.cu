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
// pieces of about L2_BYTES, so that the second pass finds its inputs in L2.
// Variances are merged from per-batch means and squared deviations (Chan's
// pairwise update), never as E[x^2] - E[x]^2.
#include "common.cuh"

namespace tssm {
namespace {

constexpr int NT = 256;
constexpr int64_t L2_BYTES = 64ll << 20;   // of 126 MB: room for the outputs written meanwhile

template <typename T, int V> struct vec;   // V elements moved as one access
template <> struct vec<float, 4> {
  __device__ static void ld(const float* p, float (&f)[4]) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
  }
  __device__ static void st(float* p, const float (&f)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  }
};
template <> struct vec<__nv_bfloat16, 8> {
  __device__ static void ld(const __nv_bfloat16* p, float (&f)[8]) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ static void st(__nv_bfloat16* p, const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct vec<__nv_bfloat16, 4> {
  __device__ static void ld(const __nv_bfloat16* p, float (&f)[4]) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    f[0] = __uint_as_float(v.x << 16); f[1] = __uint_as_float(v.x & 0xffff0000u);
    f[2] = __uint_as_float(v.y << 16); f[3] = __uint_as_float(v.y & 0xffff0000u);
  }
  __device__ static void st(__nv_bfloat16* p, const float (&f)[4]) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  }
};
template <typename T> struct vec<T, 1> {
  __device__ static void ld(const T* p, float (&f)[1]) { f[0] = ldf(p); }
  __device__ static void st(T* p, const float (&f)[1]) { stf(p, f[0]); }
};

// sigmoid(z).  A bf16 result takes the hardware exponential and division (relative
// error near 2^-21, far below bf16's 2^-9); f32 takes the accurate ones.
template <typename T>
__device__ __forceinline__ float sigmoid(float z) {
  if constexpr (std::is_same<T, float>::value) return 1.f / (1.f + expf(-z));
  else return __fdividef(1.f, 1.f + __expf(fminf(-z, 80.f)));
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

__device__ __forceinline__ float lane_sum(float v, int w) {
  for (int o = w >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// ------------------------------------------------------------------ L = 1
// A slot of TL lanes owns one group; gpb groups x rpb rows per block and pass.
struct TokenGeom {
  int tl, gpb, rpb, cblocks;
};

template <typename T, int V, int NV, bool SILU>
__global__ void __launch_bounds__(NT) gn_token_kernel(const T* __restrict__ x, const float* __restrict__ w,
                                                      const float* __restrict__ b, T* __restrict__ y,
                                                      float* __restrict__ mean_o, float* __restrict__ rstd_o,
                                                      int64_t rows, int groups, int Cg, float eps, TokenGeom ge) {
  constexpr int U = NV == 1 ? 4 : NV == 2 ? 2 : 1;   // rows in flight per thread
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
  // the loop bound is the block's, so that every lane of a warp takes part in the shuffles
  for (int64_t r0 = (int64_t)blockIdx.x * ge.rpb; r0 < rows; r0 += step * U) {
    float v[U][NV][V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + rr + u * step;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (has[j] && r < rows) vec<T, V>::ld(x + r * C + (int64_t)g * Cg + (lane + j * ge.tl) * V, v[u][j]);
        else
#pragma unroll
          for (int i = 0; i < V; ++i) v[u][j][i] = 0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + rr + u * step;
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) s += v[u][j][i];
      const float mean = lane_sum(s, ge.tl) * inv;
      float m2 = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          v[u][j][i] -= mean;
          m2 += has[j] ? v[u][j][i] * v[u][j][i] : 0.f;
        }
      const float rstd = 1.f / sqrtf(lane_sum(m2, ge.tl) * inv + eps);
      if (r >= rows) continue;   // after the shuffles
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (!has[j]) continue;
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = act<T, SILU>(v[u][j][i] * rstd * wr[j][i] + br[j][i]);
        vec<T, V>::st(y + r * C + (int64_t)g * Cg + (lane + j * ge.tl) * V, o);
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
__global__ void __launch_bounds__(NT) gn_token_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                          const float* __restrict__ w, const float* __restrict__ b,
                                                          const float* __restrict__ mean_i,
                                                          const float* __restrict__ rstd_i, T* __restrict__ dx,
                                                          float* __restrict__ part, int64_t rows, int groups, int Cg,
                                                          TokenGeom ge) {
  constexpr int U = NV == 1 ? 2 : 1;
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
  for (int64_t r0 = (int64_t)blockIdx.x * ge.rpb; r0 < rows; r0 += step * U) {
    float v[U][NV][V], d[U][NV][V], mean[U], rstd[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + rr + u * step;
      const bool in = live && r < rows;
      mean[u] = in ? mean_i[r * groups + g] : 0.f;
      rstd[u] = in ? rstd_i[r * groups + g] : 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int64_t at = r * C + (int64_t)g * Cg + (lane + j * ge.tl) * V;
        if (has[j] && in) {
          vec<T, V>::ld(x + at, v[u][j]);
          vec<T, V>::ld(dy + at, d[u][j]);
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) v[u][j][i] = d[u][j][i] = 0.f;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + rr + u * step;
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float n = (v[u][j][i] - mean[u]) * rstd[u];
          const float dz = d[u][j][i] * dact<T, SILU>(n * wr[j][i] + br[j][i]);
          aw[j][i] += dz * n;
          ab[j][i] += dz;
          v[u][j][i] = n;
          d[u][j][i] = dz * wr[j][i];
          s0 += d[u][j][i];
          s1 += d[u][j][i] * n;
        }
      s0 = lane_sum(s0, ge.tl) * inv;
      s1 = lane_sum(s1, ge.tl) * inv;
      if (r >= rows) continue;   // after the shuffles
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (!has[j]) continue;
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = rstd[u] * (d[u][j][i] - s0 - v[u][j][i] * s1);
        vec<T, V>::st(dx + r * C + (int64_t)g * Cg + (lane + j * ge.tl) * V, o);
      }
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
  const float t = n + n2, d = m2 - m, f = n2 / t;
  m += d * f;
  q += q2 + d * d * n * f;
  n = t;
}

// st [b][chunk][C / V] x (mean, squared deviations) of each thread column.
template <typename T, int V>
__global__ void __launch_bounds__(NT) gn_stats_kernel(const T* __restrict__ x, float2* __restrict__ st, int64_t L,
                                                      int64_t C, MapGeom ge) {
  __shared__ float sn[NT], sm[NT], sq[NT];
  const int tx = threadIdx.x % ge.cols, ty = threadIdx.x / ge.cols;
  const int64_t cv = (int64_t)blockIdx.y * ge.cols + tx, ncv = C / V;
  const int64_t l0 = (int64_t)blockIdx.x * ge.chunk, l1 = min(L, l0 + ge.chunk);
  float n = 0.f, m = 0.f, q = 0.f;
  if (ty < ge.rows_y && cv < ncv) {
    const T* p = x + ((int64_t)blockIdx.z * L) * C + cv * V;
    for (int64_t l = l0 + ty; l < l1; l += (int64_t)ge.rows_y * UR) {
      float v[UR][V];
      float cnt = 0.f, s = 0.f;
#pragma unroll
      for (int u = 0; u < UR; ++u) {
        const int64_t lu = l + (int64_t)u * ge.rows_y;
        if (lu < l1) vec<T, V>::ld(p + lu * C, v[u]);
      }
#pragma unroll
      for (int u = 0; u < UR; ++u)
        if (l + (int64_t)u * ge.rows_y < l1) {
          cnt += V;
#pragma unroll
          for (int i = 0; i < V; ++i) s += v[u][i];
        }
      const float mu = s / cnt;
      float d2 = 0.f;
#pragma unroll
      for (int u = 0; u < UR; ++u)
        if (l + (int64_t)u * ge.rows_y < l1)
#pragma unroll
          for (int i = 0; i < V; ++i) d2 += (v[u][i] - mu) * (v[u][i] - mu);
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

// mean, rstd of one (b, g) per block, from the partial statistics.
__global__ void __launch_bounds__(NT) gn_merge_kernel(const float2* __restrict__ st, float* __restrict__ mean_o,
                                                      float* __restrict__ rstd_o, int64_t L, int64_t ncv, int per,
                                                      int V, int groups, int64_t chunk, int64_t nchunks, float eps) {
  __shared__ float sn[NT], sm[NT], sq[NT];
  const int64_t b = blockIdx.y;
  const int g = blockIdx.x;
  float n = 0.f, m = 0.f, q = 0.f;
  for (int64_t i = threadIdx.x; i < nchunks * per; i += NT) {
    const int64_t ck = i / per, c = (int64_t)g * per + (i - ck * per);
    const float2 e = st[(b * nchunks + ck) * ncv + c];
    chan(n, m, q, (float)(min(L, (ck + 1) * chunk) - ck * chunk) * V, e.x, e.y);
  }
  sn[threadIdx.x] = n;
  sm[threadIdx.x] = m;
  sq[threadIdx.x] = q;
  __syncthreads();
  for (int o = NT / 2; o > 0; o >>= 1) {
    if (threadIdx.x < o) {
      const int k = threadIdx.x + o;
      chan(sn[threadIdx.x], sm[threadIdx.x], sq[threadIdx.x], sn[k], sm[k], sq[k]);
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    mean_o[b * groups + g] = sm[0];
    rstd_o[b * groups + g] = 1.f / sqrtf(sq[0] / sn[0] + eps);
  }
}

template <typename T, int V, bool SILU>
__global__ void __launch_bounds__(NT) gn_apply_kernel(const T* __restrict__ x, const float* __restrict__ w,
                                                      const float* __restrict__ b, const float* __restrict__ mean,
                                                      const float* __restrict__ rstd, T* __restrict__ y, int64_t L,
                                                      int64_t C, int groups, int Cg, MapGeom ge) {
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
  for (int64_t l = l0 + ty; l < l1; l += (int64_t)ge.rows_y * UR) {
    float v[UR][V];
#pragma unroll
    for (int u = 0; u < UR; ++u) {
      const int64_t lu = l + (int64_t)u * ge.rows_y;
      if (lu < l1) vec<T, V>::ld(px + lu * C, v[u]);
    }
#pragma unroll
    for (int u = 0; u < UR; ++u) {
      const int64_t lu = l + (int64_t)u * ge.rows_y;
      if (lu >= l1) break;
#pragma unroll
      for (int i = 0; i < V; ++i) v[u][i] = act<T, SILU>((v[u][i] - m) * a[i] + o[i]);
      vec<T, V>::st(py + lu * C, v[u]);
    }
  }
}

// part [b][chunk][2][C]: sums of dz n and dz over the chunk's rows.
template <typename T, int V, bool SILU>
__global__ void __launch_bounds__(NT) gn_bwd_sums_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                         const float* __restrict__ w, const float* __restrict__ b,
                                                         const float* __restrict__ mean,
                                                         const float* __restrict__ rstd, float* __restrict__ part,
                                                         int64_t L, int64_t C, int groups, int Cg, MapGeom ge) {
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
    for (int64_t l = l0 + ty; l < l1; l += (int64_t)ge.rows_y * UR) {
      float v[UR][V], d[UR][V];
#pragma unroll
      for (int u = 0; u < UR; ++u) {
        const int64_t lu = l + (int64_t)u * ge.rows_y;
        if (lu < l1) {
          vec<T, V>::ld(x + base + lu * C, v[u]);
          vec<T, V>::ld(dy + base + lu * C, d[u]);
        }
      }
#pragma unroll
      for (int u = 0; u < UR; ++u) {
        if (l + (int64_t)u * ge.rows_y >= l1) break;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float n = (v[u][i] - m) * r;
          const float dz = d[u][i] * dact<T, SILU>(n * wr[i] + br[i]);
          aw[i] += dz * n;
          ab[i] += dz;
        }
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

// One (b, g) per block: per-channel sums over the chunks into chan_sum [2][Bt][C], and the
// group means of gr and gr n into gm [Bt][groups] (x: mean gr, y: mean gr n).
__global__ void __launch_bounds__(NT) gn_bwd_merge_kernel(const float* __restrict__ part, const float* __restrict__ w,
                                                          float* __restrict__ chan_sum, float2* __restrict__ gm,
                                                          int64_t L, int64_t C, int groups, int Cg, int64_t nchunks,
                                                          int64_t Bt, int64_t b0) {
  __shared__ float sa[NT / 32], sb[NT / 32];
  const int64_t b = blockIdx.y;
  const int g = blockIdx.x;
  float ga = 0.f, gb = 0.f;
  for (int i = threadIdx.x; i < Cg; i += NT) {
    const int64_t c = (int64_t)g * Cg + i;
    float a = 0.f, d = 0.f;
#pragma unroll 4
    for (int64_t k = 0; k < nchunks; ++k) {
      const float* p = part + (b * nchunks + k) * 2 * C + c;
      a += p[0];
      d += p[C];
    }
    chan_sum[(b0 + b) * C + c] = a;
    chan_sum[(Bt + b0 + b) * C + c] = d;
    ga += a * w[c];
    gb += d * w[c];
  }
  ga = lane_sum(ga, 32);
  gb = lane_sum(gb, 32);
  if (threadIdx.x % 32 == 0) {
    sa[threadIdx.x / 32] = ga;
    sb[threadIdx.x / 32] = gb;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < NT / 32; ++k) {
      sa[0] += sa[k];
      sb[0] += sb[k];
    }
    const float inv = 1.f / ((float)L * (float)Cg);
    gm[b * groups + g] = make_float2(sb[0] * inv, sa[0] * inv);
  }
}

template <typename T, int V, bool SILU>
__global__ void __launch_bounds__(NT) gn_bwd_apply_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                          const float* __restrict__ w, const float* __restrict__ b,
                                                          const float* __restrict__ mean,
                                                          const float* __restrict__ rstd,
                                                          const float2* __restrict__ gm, T* __restrict__ dx,
                                                          int64_t L, int64_t C, int groups, int Cg, MapGeom ge) {
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
  for (int64_t l = l0 + ty; l < l1; l += (int64_t)ge.rows_y * UR) {
    float v[UR][V], d[UR][V];
#pragma unroll
    for (int u = 0; u < UR; ++u) {
      const int64_t lu = l + (int64_t)u * ge.rows_y;
      if (lu < l1) {
        vec<T, V>::ld(x + base + lu * C, v[u]);
        vec<T, V>::ld(dy + base + lu * C, d[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < UR; ++u) {
      const int64_t lu = l + (int64_t)u * ge.rows_y;
      if (lu >= l1) break;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float n = (v[u][i] - m) * r;
        const float gr = d[u][i] * dact<T, SILU>(n * wr[i] + br[i]) * wr[i];
        v[u][i] = r * (gr - mm.x - n * mm.y);
      }
      vec<T, V>::st(dx + base + lu * C, v[u]);
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
constexpr int TOKEN_BWD_PER_SM = 4;

MapGeom map_geom(int64_t Bt, int64_t L, int64_t C, int V) {
  MapGeom ge;
  const int64_t ncv = C / V;
  ge.cblocks = (int)cdiv(ncv, NT);
  ge.cols = (int)cdiv(ncv, ge.cblocks);
  ge.rows_y = NT / ge.cols;
  // about eight blocks per SM over the batch, and no chunk below one unrolled pass
  const int64_t want = std::max<int64_t>(1, cdiv((int64_t)num_sms() * 8, Bt * ge.cblocks));
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
  const MapGeom ge = map_geom(piece, L, C, V);
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
  gn_column_sum_kernel<<<dim3((unsigned)cdiv(a.C, 32), 2), NT, 0, a.st>>>((const float*)a.ws, (float*)a.dw,
                                                                         (float*)a.db, (int64_t)grid.x * ge.rpb, a.C);
}

template <typename T, int V, bool SILU>
void map_fwd(const Norm& a) {
  const int64_t row = a.L * a.C, piece = batch_piece(a.Bt, row * sizeof(T));
  const MapGeom ge = map_geom(piece, a.L, a.C, V);
  float2* st = (float2*)a.ws;
  for (int64_t b0 = 0; b0 < a.Bt; b0 += piece) {
    const int64_t nb = std::min(piece, a.Bt - b0);
    dim3 grid((unsigned)ge.nchunks, (unsigned)ge.cblocks, (unsigned)nb);
    const T* x = (const T*)a.x + b0 * row;
    float *mean = (float*)a.mean + b0 * a.groups, *rstd = (float*)a.rstd + b0 * a.groups;
    gn_stats_kernel<T, V><<<grid, NT, 0, a.st>>>(x, st, a.L, a.C, ge);
    gn_merge_kernel<<<dim3((unsigned)a.groups, (unsigned)nb), NT, 0, a.st>>>(
        st, mean, rstd, a.L, a.C / V, a.Cg / V, V, a.groups, ge.chunk, ge.nchunks, a.eps);
    gn_apply_kernel<T, V, SILU><<<grid, NT, 0, a.st>>>(x, (const float*)a.w, (const float*)a.b, mean, rstd,
                                                       (T*)a.y + b0 * row, a.L, a.C, a.groups, a.Cg, ge);
  }
}

template <typename T, int V, bool SILU>
void map_bwd(const Norm& a) {
  const int64_t row = a.L * a.C, piece = batch_piece(a.Bt, 2 * row * sizeof(T));
  const MapGeom ge = map_geom(piece, a.L, a.C, V);
  float* part = (float*)a.ws;
  float* chan_sum = part + map_part_floats(piece, a.L, a.C, V, true);
  float2* gm = (float2*)(chan_sum + 2 * a.Bt * a.C);
  for (int64_t b0 = 0; b0 < a.Bt; b0 += piece) {
    const int64_t nb = std::min(piece, a.Bt - b0);
    dim3 grid((unsigned)ge.nchunks, (unsigned)ge.cblocks, (unsigned)nb);
    const T *x = (const T*)a.x + b0 * row, *dy = (const T*)a.dy + b0 * row;
    const float *mean = (const float*)a.mean + b0 * a.groups, *rstd = (const float*)a.rstd + b0 * a.groups;
    gn_bwd_sums_kernel<T, V, SILU><<<grid, NT, 0, a.st>>>(dy, x, (const float*)a.w, (const float*)a.b, mean, rstd,
                                                          part, a.L, a.C, a.groups, a.Cg, ge);
    gn_bwd_merge_kernel<<<dim3((unsigned)a.groups, (unsigned)nb), NT, 0, a.st>>>(
        part, (const float*)a.w, chan_sum, gm, a.L, a.C, a.groups, a.Cg, ge.nchunks, a.Bt, b0);
    gn_bwd_apply_kernel<T, V, SILU><<<grid, NT, 0, a.st>>>(dy, x, (const float*)a.w, (const float*)a.b, mean, rstd,
                                                           gm, (T*)a.y + b0 * row, a.L, a.C, a.groups, a.Cg, ge);
  }
  gn_column_sum_kernel<<<dim3((unsigned)cdiv(a.C, 32), 2), NT, 0, a.st>>>(chan_sum, (float*)a.dw, (float*)a.db, a.Bt,
                                                                         a.C);
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
