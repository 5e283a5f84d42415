// Chunked gated delta rule, forward, on tcgen05 (bf16, N = 64 or 128, P a
// multiple of 64; formulas and precision: delta.cuh).
//
// Per segment of the sequence delta_prep.cu makes the chunks' images, then
// delta_scan_kernel: a block carries one (batch row, head) and 128 value channels,
// transposed: TMEM lane = value channel p, so every step of the chain stays in its
// thread.  Per chunk
//   KS^T = S^T K^T              A: S planes (TMEM), B: K (shared memory)
//   X^T  = V^T - exp(l) KS^T    threads: TMEM -> registers -> X planes (TMEM)
//   E^T  = X^T T^T              A: X planes, B: T planes, 16-column steps of the triangle
//   S^T  = exp(l_last) S^T + (E diag(w beta))^T K   (S in f32 registers, the sum from TMEM)
//   O^T  = scale exp(l) S^T Q^T + E^T (Aq diag(beta))^T
// Warps: 0 issues the chain's products, 2 those of O, 1 copies, 4-11 are the chain (two
// per 32 lanes, each half of the columns: S 64 f32 a thread), 12-15 the outputs.  The
// chain is serial, so its latency counts: pieces of its operands are handed over as
// they are written, by named barriers (a hand-over through an mbarrier measured 136
// cycles, through a barrier 25), and a product runs while the next piece is split.
// tcgen05 takes 32 cycles per 128 x 64 x 16 and 190 from issue to a thread that waits.
// Measured: 3.7 us a chunk (N = P = 128; 118 us for 2 x 2048 tokens x 16 heads).  With two
// planes for O it is 3.5, but one y in 450 then misses the nearest bf16 value (one in 5000
// with three).  Holding the third plane's QS back until X is made gained nothing.  Four chain
// warps per 32 lanes, a quarter of the columns each, were a fifth slower than two: they slow
// the issuing warps down.
// States and errors for a backward, stored a quarter at a time between the steps: 4.4 us a chunk
// (4.6 in one go).  Those sequences took 317 us in all on the register chain, 136 here.
//
// TMEM columns: [0, 192) S planes (planes 0, 1 of a half side by side, then both plane
// 2s), later the state update's sum over planes 0, 1.  [192, 256) KS.  [256, 352) X
// planes, then E diag(w beta) planes, 48 per half.  [352, 416) E, then its planes 0, 1
// for O; [480, 512) plane 2.  [416, 480) QS, then O.  A thread overwrites columns of
// its own lane and half only, so only products are waited for.
//
// Loops are left rolled where registers allow: unrolled (130 KB of code) the warps
// waited for instructions, the more so with both SMs of a pair at work.
//
// Every wait on an mbarrier is bounded.  A warp that gives up sets the abort flag and
// goes on without waiting, storing nothing: the named barriers' counts stay whole.
#include <cudaTypedefs.h>

#include <cstddef>

#include "delta.cuh"
#include "delta_tc.h"
#include "tcgen05.cuh"
#include "tmap.cuh"

namespace tssm {
namespace delta {
namespace {
using namespace sm100;

constexpr int TILE = 8192;                       // [64 x 64] bf16
constexpr int IMG = IMG_BYTES, IMG_EG = IMG_GATES + (int)offsetof(Gates, eg);
constexpr int EG_TO_WB = (int)(offsetof(Gates, wb) - offsetof(Gates, eg)) / 4;
static_assert(IMG % 16 == 0 && IMG_EG % 16 == 0, "bulk copies, 16-byte reads");

// ------------------------------------------------------------------ the scan
struct ScanArgs {
  const uint8_t* img;
  const float* h_in;
  float *h_out, *states, *errs;
  int* status;
  int64_t L, c0, nseg, nc;
  int H, G, P, N, npb;
  float scale;
};

template <int KN>
struct ScanSmem {
  static constexpr int NB = KN / 64;   // 64-wide blocks of K, Q
  static constexpr int K = 0, QQ = K + NB * TILE, V = QQ + NB * TILE, IM = V + 2 * TILE, STAGE = (IM + IMG + 1023) / 1024 * 1024;
  static constexpr int Y = 2 * STAGE, BAR = Y + 2 * TILE, BYTES = BAR + 256 + 1024;
  static_assert(BYTES <= 232448, "shared-memory layout exceeds the per-block limit");
};

constexpr uint32_t C_KS = 192, C_XP = 256, C_E = 352, C_O = 416, C_E2 = 480;
// named barriers (0: __syncthreads): outputs; pieces of S, X, E diag(w beta), E for their issuers
constexpr uint32_t B_OUT = 1, B_S = 2, B_X = 6, B_W = 8, B_E = 10, B_ISSUE = 256 + 32;

// D (+)= A B with A in TMEM: row m in lane m, 16 bf16 of k in 8 columns.
__device__ __forceinline__ void umma_bf16_ta(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc),
      "r"((uint32_t)acc)
      : "memory");
}
// A wait on the chain's path: a few short hardware-timed waits (a round trip through a
// test_wait loop measured 272 cycles, through try_wait 237, and a waiting warp takes no
// issue slots from the working ones), then as mbar_wait.
__device__ __forceinline__ bool mbar_wait_hot(uint64_t* m, uint32_t parity, const volatile int* abort_flag) {
#pragma unroll 1
  for (int i = 0; i < 64; ++i)
    if (mbar_try_wait(m, parity, 20000u)) return true;
  if (*abort_flag) return false;
  return mbar_wait_slow(m, parity, abort_flag, 2000000000ull);
}
__device__ __forceinline__ void tmem_st8u(uint32_t taddr, const uint32_t (&u)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(u[0]),
               "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
               : "memory");
}
// 16 values as NS planes of 8 columns, plane s at taddr[s] (r is used up).
template <int NS>
__device__ __forceinline__ void store_planes(const uint32_t (&taddr)[NS], float (&r)[16]) {
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      u[i] = pack2(r[2 * i], r[2 * i + 1]);
      if (s + 1 < NS) sub2(r[2 * i], r[2 * i + 1], u[i]);
    }
    tmem_st8u(taddr[s], u);
  }
}
template <int NS>
__device__ __forceinline__ void store_planes(uint32_t taddr, uint32_t step, float (&r)[16]) {
  uint32_t at[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) at[s] = taddr + s * step;
  store_planes<NS>(at, r);
}

template <int KN>
__global__ void __launch_bounds__(512, 1) delta_scan_kernel(const __grid_constant__ CUtensorMap tm_k,
                                                            const __grid_constant__ CUtensorMap tm_q,
                                                            const __grid_constant__ CUtensorMap tm_u,
                                                            const __grid_constant__ CUtensorMap tm_y, const ScanArgs a) {
  using SM = ScanSmem<KN>;
  constexpr int NB = SM::NB, HN = KN / 2, NS = 3;   // HN: state columns of a thread; NS: planes of the state, X and E
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t bh = blockIdx.x / a.npb;
  const int pb = (int)(blockIdx.x - bh * a.npb) * 128;
  const int b = (int)(bh / a.H), h = (int)(bh - (int64_t)b * a.H), g = h / (a.H / a.G);
  const int boxes = min(2, (a.P - pb) / 64);   // 64-channel boxes of this block
  const int n = (int)a.nseg;

  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + SM::BAR);
  uint64_t *full = bar, *empty = bar + 2;      // [2] stage loaded / released
  uint64_t *ksdone = bar + 4, *edone = bar + 5, *dsdone = bar + 6, *qdone = bar + 7, *odone = bar + 8, *qread = bar + 9,
           *oread = bar + 10, *drain = bar + 11;   // drain [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + SM::BAR + 192);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + SM::BAR + 196);
  int* issued = reinterpret_cast<int*>(smem + SM::BAR + 200);
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 2 + 8 + 4);   // two issuers' commits, chain and output warps
      mbar_init(&drain[i], 1);
    }
    mbar_init(qread, 4);
    mbar_init(oread, 4);
    mbar_init(ksdone, 1);
    mbar_init(edone, 1);
    mbar_init(dsdone, 1);
    mbar_init(qdone, 1);
    mbar_init(odone, 1);
    *abort_flag = 0;
    *issued = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  auto stage = [&](int c) { return smem + (c & 1) * SM::STAGE; };
  auto fail = [&](int code) {
    *abort_flag = 1;
    atomicExch(a.status, code);
  };
  // A wait by a whole warp: every lane takes the same decision; false: give up.
  auto waitw = [&](uint64_t* m, int phase, int code) {
    const bool ok = mbar_wait_hot(m, phase & 1, abort_flag);
    tc_fence_after();
    if (__all_sync(0xffffffffu, ok)) return true;
    if (lane == 0 && !*abort_flag) fail(code);
    return false;
  };
  auto arrive_warp = [&](uint64_t* m) {   // this warp's TMEM accesses before it are ordered before the arrival
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(m);
  };
  auto hand_over = [&](uint32_t b) {      // TMEM stores of a piece -> its issuer
    tmem_wait_st();
    tc_fence_before();
    named_bar_arrive(b, B_ISSUE);
  };
  auto take = [&](uint32_t b) {
    named_bar_sync(b, B_ISSUE);
    tc_fence_after();
  };
  // first column of plane s of a half of the state
  auto plane = [](int s, int hf) { return (uint32_t)(s < 2 ? HN * hf + (HN / 2) * s : KN + (HN / 2) * hf); };

  if (warp >= 4 && warp < 12) {
    // ================================================================ the chain
    const int half = (warp >> 2) - 1, p = (warp & 3) * 32 + lane;   // value channel = TMEM lane
    const uint32_t tl = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const bool live = p < boxes * 64;
    const int64_t row = (bh * a.P + pb + p) * (int64_t)a.N + half * HN;   // of h_in, h_out
    float S[HN];
#pragma unroll
    for (int j = 0; j < HN; j += 4) {
      const float4 v = live && a.h_in ? *reinterpret_cast<const float4*>(a.h_in + row + j) : make_float4(0.f, 0.f, 0.f, 0.f);
      S[j] = v.x; S[j + 1] = v.y; S[j + 2] = v.z; S[j + 3] = v.w;
    }
    bool ok = true;
    for (int c = 0; c < n; ++c) {
      // S planes, 16 columns of the half at a time
#pragma unroll
      for (int i = 0; i < HN / 16; ++i) {
        float r[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) r[j] = S[16 * i + j];
        uint32_t at[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) at[s] = tl + plane(s, half) + 8 * i;
        store_planes<NS>(at, r);
        hand_over(B_S + i);
      }
      auto save = [&](int q) {   // a quarter of the state, [N / 4][P][4]: 512 bytes a warp and store
        if (!(a.states && live && ok)) return;
        float4* dst = reinterpret_cast<float4*>(a.states) +
                      ((bh * a.nc + a.c0 + c) * (a.N / 4) + half * (HN / 4)) * (int64_t)a.P + pb + p;
#pragma unroll
        for (int j = q * HN / 4; j < (q + 1) * HN / 4; j += 4)
          dst[(int64_t)(j / 4) * a.P] = make_float4(S[j], S[j + 1], S[j + 2], S[j + 3]);
      };
      save(0);
      // X^T = V^T - exp(l) KS^T, 32 tokens of this half
      const uint8_t* st = stage(c);
      ok = ok && waitw(&full[c & 1], c >> 1, 3002);
      const float* eg = reinterpret_cast<const float*>(st + SM::IM + IMG_EG) + 32 * half;
      const float* wb = eg + EG_TO_WB;
      const float el = (eg - 32 * half)[Q - 1];
      const uint16_t* vs = reinterpret_cast<const uint16_t*>(st + SM::V + (p >> 6) * TILE) + (p & 63) + half * 32 * 64;
      ok = ok && waitw(ksdone, c, 3003);
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        float x[16];
        uint32_t v[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = vs[(16 * i + j) * 64];
        tmem_get16(tl + C_KS + 32 * half + 16 * i, x);
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const float4 e4 = *reinterpret_cast<const float4*>(eg + 16 * i + j);
          x[j] = lo2(v[j]) - e4.x * x[j];
          x[j + 1] = lo2(v[j + 1]) - e4.y * x[j + 1];
          x[j + 2] = lo2(v[j + 2]) - e4.z * x[j + 2];
          x[j + 3] = lo2(v[j + 3]) - e4.w * x[j + 3];
        }
        store_planes<NS>(tl + C_XP + 48 * half + 8 * i, 16, x);
        hand_over(B_X + i);
      }
      save(1);
      // E^T: planes of E diag(w beta) for the state
      ok = ok && waitw(edone, c, 3004);
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        float x[16];
        tmem_get16(tl + C_E + 32 * half + 16 * i, x);
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const float4 w4 = *reinterpret_cast<const float4*>(wb + 16 * i + j);
          x[j] *= w4.x;
          x[j + 1] *= w4.y;
          x[j + 2] *= w4.z;
          x[j + 3] *= w4.w;
        }
        store_planes<NS>(tl + C_XP + 48 * half + 8 * i, 16, x);
        hand_over(B_W + i);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[c & 1]);   // V and the gates are read
      save(2);
      // E's planes for O, over E (both pieces are read before either is written)
      {
        float x[2][16];
        tmem_get16(tl + C_E + 32 * half, x[0]);
        tmem_get16(tl + C_E + 32 * half + 16, x[1]);
        if (a.errs && live && ok) {
          const int64_t tk = (a.c0 + c) * Q + 32 * half;
          float4* ep = reinterpret_cast<float4*>(a.errs + bh * saved_floats(a.P, a.L)) + tk / 4 * a.P + pb + p;
          const int left = (int)min((int64_t)32, a.L - tk);
#pragma unroll
          for (int j = 0; j < 32; j += 4)   // tokens behind the end have e = 0
            if (j < left)
              ep[j / 4 * a.P] = make_float4(x[j >> 4][j & 15], x[j >> 4][(j + 1) & 15], x[j >> 4][(j + 2) & 15],
                                            x[j >> 4][(j + 3) & 15]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t at[NS] = {tl + C_E + 32 * half + 8 * i, tl + C_E + 32 * half + 16 + 8 * i,
                                   tl + C_E2 + 16 * half + 8 * i};
          store_planes<NS>(at, x[i]);
        }
      }
      hand_over(B_E);
      save(3);
      // S^T
      ok = ok && waitw(dsdone, c, 3005);
#pragma unroll
      for (int i = 0; i < HN / 16; ++i) {
        float d[16];
        tmem_get16(tl + HN * half + 16 * i, d);
#pragma unroll
        for (int j = 0; j < 16; ++j) S[16 * i + j] = el * S[16 * i + j] + d[j];
      }
    }
    if (ok && a.h_out && live) {
#pragma unroll
      for (int j = 0; j < HN; j += 4)
        *reinterpret_cast<float4*>(a.h_out + row + j) = make_float4(S[j], S[j + 1], S[j + 2], S[j + 3]);
    }
  } else if (warp >= 12) {
    // ================================================================ outputs
    const int w = warp - 12, p = w * 32 + lane;
    const uint32_t tl = tmem + ((uint32_t)(w * 32) << 16);
    for (int c = 0; c < n; ++c) {
      const uint8_t* st = stage(c);
      // scale exp(l) QS^T goes back to its columns, where Aq diag(beta) E is added
      bool bad = !waitw(&full[c & 1], c >> 1, 3006) || !waitw(qdone, c, 3007);
      const float* eg = reinterpret_cast<const float*>(st + SM::IM + IMG_EG);
      if (!bad) {
#pragma unroll 1
        for (int i = 0; i < Q; i += 16) {
          float t[16];
          tmem_get16(tl + C_O + i, t);
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            const float4 e4 = *reinterpret_cast<const float4*>(eg + i + j);
            t[j] *= a.scale * e4.x;
            t[j + 1] *= a.scale * e4.y;
            t[j + 2] *= a.scale * e4.z;
            t[j + 3] *= a.scale * e4.w;
          }
          tmem_st16(tl + C_O + i, t);
        }
        tmem_wait_st();
        arrive_warp(qread);
        bad = !waitw(odone, c, 3008);
      }
      if (tid == 384 && c > 0) bulk_wait_read<0>();   // the last chunk's store has left the tile
      if (named_bar_or(B_OUT, 128, bad)) break;
      __nv_bfloat16* ys = reinterpret_cast<__nv_bfloat16*>(smem + SM::Y + (p >> 6) * TILE) + (p & 63);
#pragma unroll 1
      for (int i = 0; i < Q; i += 16) {
        float t[16];
        tmem_get16(tl + C_O + i, t);
#pragma unroll
        for (int j = 0; j < 16; ++j) ys[(i + j) * 64] = __float2bfloat16_rn(t[j]);
      }
      arrive_warp(oread);
      if (lane == 0) mbar_arrive(&empty[c & 1]);
      fence_proxy_async_smem();
      named_bar_sync(B_OUT, 128);
      if (tid == 384) {
        for (int x = 0; x < boxes; ++x)   // rows past L are clipped by the map
          tma_store_3d(&tm_y, smem + SM::Y + x * TILE, h * a.P + pb + 64 * x, (int)(a.c0 + c) * Q, b);
        bulk_commit();
      }
    }
    if (tid == 384) bulk_wait<0>();
  } else if (warp == 1) {
    // ================================================================ copies
    if (lane == 0) {
      const uint32_t bytes = 2 * NB * TILE + boxes * TILE + IMG;
      for (int c = 0; c < n; ++c) {
        if (c >= 2 && !mbar_wait(&empty[c & 1], ((c >> 1) - 1) & 1, abort_flag)) {
          if (!*abort_flag) fail(3009);
          break;
        }
        uint8_t* st = stage(c);
        uint64_t* f = &full[c & 1];
        const int t0 = (int)(a.c0 + c) * Q;
        mbar_arrive_expect_tx(f, bytes);
        for (int x = 0; x < NB; ++x) {
          tma_load_3d(st + SM::K + x * TILE, &tm_k, g * a.N + 64 * x, t0, b, f);
          tma_load_3d(st + SM::QQ + x * TILE, &tm_q, g * a.N + 64 * x, t0, b, f);
        }
        for (int x = 0; x < boxes; ++x) tma_load_3d(st + SM::V + x * TILE, &tm_u, h * a.P + pb + 64 * x, t0, b, f);
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                         smem_u32(st + SM::IM)),
                     "l"(a.img + (bh * a.nseg + c) * IMG), "r"(IMG), "r"(smem_u32(f))
                     : "memory");
        *issued = c + 1;
      }
    }
  } else if (warp == 0) {
    // ================================================================ the chain's products
    bool ok = true;
    for (int c = 0; c < n; ++c) {
      const uint32_t st = smem_u32(stage(c));
      ok = ok && waitw(&full[c & 1], c >> 1, 3010);
      // KS
#pragma unroll 1
      for (int i = 0; i < HN / 16; ++i) {
        take(B_S + i);
        if (ok && elect_one())
#pragma unroll
          for (int hf = 0; hf < 2; ++hf)
#pragma unroll
            for (int s = NS - 1; s >= 0; --s) {
              const int kk = hf * (HN / 16) + i;
              umma_bf16_ta(tmem + C_KS, tmem + plane(s, hf) + 8 * i,
                           make_desc_sw128(st + SM::K + (kk / 4) * TILE, 16) + 2 * (kk & 3),
                           make_idesc_bf16(128, 64, false, false), i || hf || s != NS - 1);
            }
      }
      umma_commit_warp(ksdone);
      // E, where O's product of the chunk before has read its planes
      ok = ok && (c == 0 || waitw(odone, c - 1, 3018));
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        take(B_X + i);
        if (ok && elect_one())
#pragma unroll
          for (int hf = 0; hf < 2; ++hf)
#pragma unroll
            for (int o = NS - 1; o >= 0; --o)
#pragma unroll
              for (int s = 0; s <= o; ++s) {
                const int t = 2 * hf + i;   // tokens 16 t .. reach the columns from 16 t
                umma_bf16_ta(tmem + C_E + 16 * t, tmem + C_XP + 48 * hf + 16 * s + 8 * i,
                             make_desc_sw128(st + SM::IM + IMG_T + (o - s) * SQ_BYTES, 16) + 130 * t,
                             make_idesc_bf16(128, 64 - 16 * t, false, false), t || o != NS - 1 || s);
              }
      }
      umma_commit_warp(edone);
      // state update, over S planes 0 and 1, which QS has read by now
      ok = ok && waitw(qdone, c, 3011);
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        take(B_W + i);
        if (ok && elect_one())
#pragma unroll
          for (int hf = 0; hf < 2; ++hf)
#pragma unroll
            for (int s = NS - 1; s >= 0; --s)
              umma_bf16_ta(tmem, tmem + C_XP + 48 * hf + 16 * s + 8 * i,
                           make_desc_sw128(st + SM::K, TILE) + 128 * (2 * hf + i),
                           make_idesc_bf16(128, KN, false, true), i || hf || s != NS - 1);
      }
      umma_commit_warp(dsdone);
      umma_commit_warp(&empty[c & 1]);
    }
    umma_commit_warp(&drain[0]);
    mbar_wait(&drain[0], 0, nullptr, 100000000ull);
  } else if (warp == 2) {
    // ================================================================ O's products
    bool ok = true;
    for (int c = 0; c < n; ++c) {
      const uint32_t st = smem_u32(stage(c));
      // QS behind KS (it runs while X is made), once the columns of the last output are read
      ok = ok && waitw(&full[c & 1], c >> 1, 3012) && waitw(ksdone, c, 3013) && (c == 0 || waitw(oread, c - 1, 3014));
      if (ok && elect_one())
#pragma unroll 1
        for (int kk = 0; kk < KN / 16; ++kk)
#pragma unroll
          for (int s = NS - 1; s >= 0; --s)
            umma_bf16_ta(tmem + C_O, tmem + plane(s, kk / (HN / 16)) + 8 * (kk % (HN / 16)),
                         make_desc_sw128(st + SM::QQ + (kk / 4) * TILE, 16) + 2 * (kk & 3),
                         make_idesc_bf16(128, 64, false, false), s != NS - 1 || kk);
      umma_commit_warp(qdone);
      take(B_E);
      ok = ok && waitw(qread, c, 3015);
      if (ok && elect_one())
#pragma unroll 1
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int o = NS - 1; o >= 0; --o)
#pragma unroll
            for (int s = 0; s <= o; ++s)
              umma_bf16_ta(tmem + C_O + 16 * t, tmem + (s < 2 ? C_E + 32 * (t >> 1) + 16 * s : C_E2 + 16 * (t >> 1)) + 8 * (t & 1),
                           make_desc_sw128(st + SM::IM + IMG_AQ + (o - s) * SQ_BYTES, 16) + 130 * t,
                           make_idesc_bf16(128, 64 - 16 * t, false, false), true);   // onto scale exp(l) QS
      umma_commit_warp(odone);
      umma_commit_warp(&empty[c & 1]);
    }
    umma_commit_warp(&drain[1]);
    mbar_wait(&drain[1], 0, nullptr, 100000000ull);
  }
  // ================================================================ teardown
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *abort_flag)   // copies that were started land before the block leaves
    for (int c = max(0, *issued - 2); c < *issued; ++c) mbar_wait(&full[c & 1], (c >> 1) & 1, nullptr, 100000000ull);
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}


// ------------------------------------------------------------------ the backward's chain
// The same walk in reverse (formulas: delta_bwd.cu), transposed as above; dS^T is the state:
//   R^T   = (dS^T K^T) diag(w beta) + dO^T (Aq diag(beta))
//   dE^T  = R^T T
//   dS^T <- exp(l_last) dS^T + (scale exp(l) dO)^T Q - (exp(l) dE)^T K
// TMEM columns: [0, 192) dS planes, later the update's sum over planes 0, 1 and two planes of
// scale exp(l) dO over plane 2 (the third: [480, 512)).  [192, 256) dS K.  [256, 352) dO^T in its
// first 32, then R planes, then -exp(l) dE planes.  [352, 416) dE.  [416, 480) dO^T Aq.
struct BackArgs {
  const uint8_t* img;
  const float* ds_in;
  float *ds_out, *dstates, *derrs;
  int* status;
  int64_t L, c0, nseg, nc;
  int H, G, P, N, npb;
  float scale;
};

template <int KN>
struct BackSmem {
  static constexpr int NB = KN / 64;
  static constexpr int K = 0, QQ = K + NB * TILE, DO = QQ + NB * TILE, IM = DO + 2 * TILE,
                       STAGE = (IM + IMG + 1023) / 1024 * 1024;
  static constexpr int BAR = 2 * STAGE, BYTES = BAR + 256 + 1024;
  static_assert(BYTES <= 232448, "shared-memory layout exceeds the per-block limit");
};

constexpr uint32_t C_AO = 416, C_D2 = 480;
constexpr uint32_t B_A = 1, B_D = 11;   // named barriers: dO^T, planes of scale exp(l) dO (B_S, B_X, B_W as above)

template <int KN>
__global__ void __launch_bounds__(384, 1) delta_back_scan_kernel(const __grid_constant__ CUtensorMap tm_k,
                                                                 const __grid_constant__ CUtensorMap tm_q,
                                                                 const __grid_constant__ CUtensorMap tm_o,
                                                                 const BackArgs a) {
  using SM = BackSmem<KN>;
  constexpr int NB = SM::NB, HN = KN / 2, NS = 3;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t bh = blockIdx.x / a.npb;
  const int pb = (int)(blockIdx.x - bh * a.npb) * 128;
  const int b = (int)(bh / a.H), h = (int)(bh - (int64_t)b * a.H), g = h / (a.H / a.G);
  const int boxes = min(2, (a.P - pb) / 64);
  const int n = (int)a.nseg;

  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + SM::BAR);
  uint64_t *full = bar, *empty = bar + 2, *ksdone = bar + 4, *edone = bar + 5, *dsdone = bar + 6, *drain = bar + 7;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + SM::BAR + 192);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + SM::BAR + 196);
  int* issued = reinterpret_cast<int*>(smem + SM::BAR + 200);
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1 + 8);   // the issuer's commit, chain warps
    }
    mbar_init(ksdone, 1);
    mbar_init(edone, 1);
    mbar_init(dsdone, 1);
    mbar_init(drain, 1);
    *abort_flag = 0;
    *issued = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // step k works on chunk n - 1 - k of the segment
  auto stage = [&](int k) { return smem + (k & 1) * SM::STAGE; };
  auto fail = [&](int code) {
    *abort_flag = 1;
    atomicExch(a.status, code);
  };
  auto waitw = [&](uint64_t* m, int phase, int code) {
    const bool ok = mbar_wait_hot(m, phase & 1, abort_flag);
    tc_fence_after();
    if (__all_sync(0xffffffffu, ok)) return true;
    if (lane == 0 && !*abort_flag) fail(code);
    return false;
  };
  auto hand_over = [&](uint32_t x) {
    tmem_wait_st();
    tc_fence_before();
    named_bar_arrive(x, B_ISSUE);
  };
  auto take = [&](uint32_t x) {
    named_bar_sync(x, B_ISSUE);
    tc_fence_after();
  };
  auto plane = [](int s, int hf) { return (uint32_t)(s < 2 ? HN * hf + (HN / 2) * s : KN + (HN / 2) * hf); };
  auto dplane = [](int s) { return s < 2 ? 128u + 32u * s : C_D2; };   // of scale exp(l) dO

  if (warp >= 4) {
    // ================================================================ the chain
    const int half = (warp >> 2) - 1, p = (warp & 3) * 32 + lane;
    const uint32_t tl = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const bool live = p < boxes * 64;
    const int64_t row = (bh * a.P + pb + p) * (int64_t)a.N + half * HN;
    float S[HN];
#pragma unroll
    for (int j = 0; j < HN; j += 4) {
      const float4 v = live && a.ds_in ? *reinterpret_cast<const float4*>(a.ds_in + row + j) : make_float4(0.f, 0.f, 0.f, 0.f);
      S[j] = v.x; S[j + 1] = v.y; S[j + 2] = v.z; S[j + 3] = v.w;
    }
    bool ok = true;
    for (int k = 0; k < n; ++k) {
      const int64_t cc = a.c0 + n - 1 - k;
      const uint8_t* st = stage(k);
      ok = ok && waitw(&full[k & 1], k >> 1, 3102);
      const float* eg = reinterpret_cast<const float*>(st + SM::IM + IMG_EG) + 32 * half;
      const float* wb = eg + EG_TO_WB;
      const float el = (eg - 32 * half)[Q - 1];
      const uint16_t* os = reinterpret_cast<const uint16_t*>(st + SM::DO + (p >> 6) * TILE) + (p & 63) + half * 32 * 64;
      // dO^T, 32 tokens of this half
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        uint32_t u[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          u[j] = __byte_perm(os[(16 * i + 2 * j) * 64], os[(16 * i + 2 * j + 1) * 64], 0x5410);
        tmem_st8u(tl + C_XP + 16 * half + 8 * i, u);
      }
      hand_over(B_A);
      // dS planes
#pragma unroll
      for (int i = 0; i < HN / 16; ++i) {
        float r[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) r[j] = S[16 * i + j];
        uint32_t at[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) at[s] = tl + plane(s, half) + 8 * i;
        store_planes<NS>(at, r);
        hand_over(B_S + i);
      }
      auto save = [&](int q) {   // a quarter of the state's gradient
        if (!(live && ok)) return;
        float4* dst = reinterpret_cast<float4*>(a.dstates) +
                      ((bh * a.nc + cc) * (a.N / 4) + half * (HN / 4)) * (int64_t)a.P + pb + p;
#pragma unroll
        for (int j = q * HN / 4; j < (q + 1) * HN / 4; j += 4)
          dst[(int64_t)(j / 4) * a.P] = make_float4(S[j], S[j + 1], S[j + 2], S[j + 3]);
      };
      save(0);
      // R^T; the last tokens' products reach all columns and go first
      ok = ok && waitw(ksdone, k, 3103);
#pragma unroll 1
      for (int i = 1; i >= 0; --i) {
        float x[16], y[16];
        tmem_get16(tl + C_KS + 32 * half + 16 * i, x);
        tmem_get16(tl + C_AO + 32 * half + 16 * i, y);
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const float4 w4 = *reinterpret_cast<const float4*>(wb + 16 * i + j);
          x[j] = w4.x * x[j] + y[j];
          x[j + 1] = w4.y * x[j + 1] + y[j + 1];
          x[j + 2] = w4.z * x[j + 2] + y[j + 2];
          x[j + 3] = w4.w * x[j + 3] + y[j + 3];
        }
        store_planes<NS>(tl + C_XP + 48 * half + 8 * i, 16, x);
        hand_over(B_X + i);
      }
      save(1);
      // scale exp(l) dO, while dE is made
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        float x[16];
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const float4 e4 = *reinterpret_cast<const float4*>(eg + 16 * i + j);
          const uint16_t* o = os + (16 * i + j) * 64;
          x[j] = a.scale * e4.x * lo2(o[0]);
          x[j + 1] = a.scale * e4.y * lo2(o[64]);
          x[j + 2] = a.scale * e4.z * lo2(o[128]);
          x[j + 3] = a.scale * e4.w * lo2(o[192]);
        }
        const uint32_t at[NS] = {tl + dplane(0) + 16 * half + 8 * i, tl + dplane(1) + 16 * half + 8 * i,
                                 tl + dplane(2) + 16 * half + 8 * i};
        store_planes<NS>(at, x);
      }
      hand_over(B_D);
      save(2);
      // -exp(l) dE
      ok = ok && waitw(edone, k, 3104);
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        float x[16];
        tmem_get16(tl + C_E + 32 * half + 16 * i, x);
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const float4 e4 = *reinterpret_cast<const float4*>(eg + 16 * i + j);
          x[j] *= -e4.x;
          x[j + 1] *= -e4.y;
          x[j + 2] *= -e4.z;
          x[j + 3] *= -e4.w;
        }
        store_planes<NS>(tl + C_XP + 48 * half + 8 * i, 16, x);
        hand_over(B_W + i);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[k & 1]);   // dO and the gates are read
      save(3);
      // dE for the gradient kernel
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        float x[16];
        tmem_get16(tl + C_E + 32 * half + 16 * i, x);
        const int64_t tk = cc * Q + 32 * half + 16 * i;
        const int left = live && ok ? (int)max((int64_t)0, min((int64_t)16, a.L - tk)) : 0;
        float4* ep = reinterpret_cast<float4*>(a.derrs + bh * saved_floats(a.P, a.L)) + tk / 4 * a.P + pb + p;
#pragma unroll
        for (int j = 0; j < 16; j += 4)
          if (j < left) ep[j / 4 * a.P] = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
      }
      // dS^T
      ok = ok && waitw(dsdone, k, 3105);
#pragma unroll
      for (int i = 0; i < HN / 16; ++i) {
        float d[16];
        tmem_get16(tl + HN * half + 16 * i, d);
#pragma unroll
        for (int j = 0; j < 16; ++j) S[16 * i + j] = el * S[16 * i + j] + d[j];
      }
    }
    if (ok && live) {
#pragma unroll
      for (int j = 0; j < HN; j += 4)
        *reinterpret_cast<float4*>(a.ds_out + row + j) = make_float4(S[j], S[j + 1], S[j + 2], S[j + 3]);
    }
  } else if (warp == 1) {
    // ================================================================ copies
    if (lane == 0) {
      const uint32_t bytes = 2 * NB * TILE + boxes * TILE + IMG;
      for (int k = 0; k < n; ++k) {
        if (k >= 2 && !mbar_wait(&empty[k & 1], ((k >> 1) - 1) & 1, abort_flag)) {
          if (!*abort_flag) fail(3109);
          break;
        }
        uint8_t* st = stage(k);
        uint64_t* f = &full[k & 1];
        const int c = n - 1 - k, t0 = (int)(a.c0 + c) * Q;
        mbar_arrive_expect_tx(f, bytes);
        for (int x = 0; x < NB; ++x) {
          tma_load_3d(st + SM::K + x * TILE, &tm_k, g * a.N + 64 * x, t0, b, f);
          tma_load_3d(st + SM::QQ + x * TILE, &tm_q, g * a.N + 64 * x, t0, b, f);
        }
        for (int x = 0; x < boxes; ++x) tma_load_3d(st + SM::DO + x * TILE, &tm_o, h * a.P + pb + 64 * x, t0, b, f);
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                         smem_u32(st + SM::IM)),
                     "l"(a.img + (bh * a.nseg + c) * IMG), "r"(IMG), "r"(smem_u32(f))
                     : "memory");
        *issued = k + 1;
      }
    }
  } else if (warp == 0) {
    // ================================================================ products
    bool ok = true;
    for (int k = 0; k < n; ++k) {
      const uint32_t st = smem_u32(stage(k));
      ok = ok && waitw(&full[k & 1], k >> 1, 3110);
      // dO^T Aq: tokens 16 t .. reach the columns up to 16 t + 15
      take(B_A);
      if (ok && elect_one())
#pragma unroll 1
        for (int t = 3; t >= 0; --t)
#pragma unroll
          for (int z = 2; z >= 0; --z)
            umma_bf16_ta(tmem + C_AO, tmem + C_XP + 8 * t,
                         make_desc_sw128(st + SM::IM + IMG_AQ + z * SQ_BYTES, TILE) + 128 * t,
                         make_idesc_bf16(128, 16 * (t + 1), false, true), t != 3 || z != 2);
      // dS K
#pragma unroll 1
      for (int i = 0; i < HN / 16; ++i) {
        take(B_S + i);
        if (ok && elect_one())
#pragma unroll
          for (int hf = 0; hf < 2; ++hf)
#pragma unroll
            for (int s = NS - 1; s >= 0; --s) {
              const int kk = hf * (HN / 16) + i;
              umma_bf16_ta(tmem + C_KS, tmem + plane(s, hf) + 8 * i,
                           make_desc_sw128(st + SM::K + (kk / 4) * TILE, 16) + 2 * (kk & 3),
                           make_idesc_bf16(128, 64, false, false), i || hf || s != NS - 1);
            }
      }
      umma_commit_warp(ksdone);   // both products
      // dE
#pragma unroll 1
      for (int i = 1; i >= 0; --i) {
        take(B_X + i);
        if (ok && elect_one())
#pragma unroll
          for (int hf = 1; hf >= 0; --hf)
#pragma unroll
            for (int o = NS - 1; o >= 0; --o)
#pragma unroll
              for (int s = 0; s <= o; ++s) {
                const int t = 2 * hf + i;
                umma_bf16_ta(tmem + C_E, tmem + C_XP + 48 * hf + 16 * s + 8 * i,
                             make_desc_sw128(st + SM::IM + IMG_T + (o - s) * SQ_BYTES, TILE) + 128 * t,
                             make_idesc_bf16(128, 16 * (t + 1), false, true), t != 3 || o != NS - 1 || s);
              }
      }
      umma_commit_warp(edone);
      // the update, over the dS planes that dS K has read: Q's part, then K's
      take(B_D);
      if (ok && elect_one())
#pragma unroll 1
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int s = NS - 1; s >= 0; --s)
            umma_bf16_ta(tmem, tmem + dplane(s) + 8 * t, make_desc_sw128(st + SM::QQ, TILE) + 128 * t,
                         make_idesc_bf16(128, KN, false, true), t || s != NS - 1);
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        take(B_W + i);
        if (ok && elect_one())
#pragma unroll
          for (int hf = 0; hf < 2; ++hf)
#pragma unroll
            for (int s = NS - 1; s >= 0; --s)
              umma_bf16_ta(tmem, tmem + C_XP + 48 * hf + 16 * s + 8 * i,
                           make_desc_sw128(st + SM::K, TILE) + 128 * (2 * hf + i),
                           make_idesc_bf16(128, KN, false, true), true);
      }
      umma_commit_warp(dsdone);
      umma_commit_warp(&empty[k & 1]);
    }
    umma_commit_warp(drain);
    mbar_wait(drain, 0, nullptr, 100000000ull);
  }
  // ================================================================ teardown
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *abort_flag)   // copies that were started land before the block leaves
    for (int k = max(0, *issued - 2); k < *issued; ++k) mbar_wait(&full[k & 1], (k >> 1) & 1, nullptr, 100000000ull);
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

bool map_bf16(CUtensorMap* m, const void* base, uint64_t d0, uint64_t d1, uint64_t d2, bool swizzle) {
  auto fn = tmap_encode_fn();
  if (!fn) return false;
  cuuint64_t dims[3] = {d0, d1, d2};
  cuuint64_t strides[2] = {d0 * 2, d0 * d1 * 2};
  cuuint32_t box[3] = {64, 64, 1};
  cuuint32_t es[3] = {1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int KN>
int run(const TcCall& a, cudaStream_t st) {
  const int64_t streams = a.Bt * a.H, nc = cdiv(a.L, Q), seg = segment_chunks(streams, nc);
  CUtensorMap mk, mq, mu, my;
  if (!map_bf16(&mk, a.B, a.G * a.N, a.L, a.Bt, true) || !map_bf16(&mq, a.C, a.G * a.N, a.L, a.Bt, true) ||
      !map_bf16(&mu, a.u, a.H * a.P, a.L, a.Bt, false) || !map_bf16(&my, a.y, a.H * a.P, a.L, a.Bt, false)) {
    set_error("gated_delta_rule: cuTensorMapEncodeTiled failed");
    return TSSM_ERR_CUDA;
  }
  int* status = device_status_ptr();
  if (!status) {
    set_error("gated_delta_rule: device status word unavailable");
    return TSSM_ERR_CUDA;
  }
  auto scan = delta_scan_kernel<KN>;
  if (cudaFuncSetAttribute(scan, cudaFuncAttributeMaxDynamicSharedMemorySize, ScanSmem<KN>::BYTES) != cudaSuccess)
    return check_launch("gated_delta_rule: set smem attribute");
  for (int64_t c0 = 0; c0 < nc; c0 += seg) {
    const int64_t m = std::min(seg, nc - c0);
    const PrepCall p{a.B, a.C, a.A_log, a.dt, a.beta, a.img, nullptr, a.Bt, a.L, a.H, a.G, a.N, c0, m, nc, a.scale, 1};
    if (int e = prep_run(p, TSSM_BF16, st)) return e;
    const bool last = c0 + m == nc;
    const ScanArgs s{a.img, c0 ? a.carry : a.h0, last && !a.h_last ? nullptr : a.carry, a.states, a.errs, status, a.L,
                     c0, m, nc, (int)a.H, (int)a.G, (int)a.P, (int)a.N, (int)cdiv(a.P, 128), a.scale};
    scan<<<(unsigned)(streams * s.npb), 512, ScanSmem<KN>::BYTES, st>>>(mk, mq, mu, my, s);
  }
  return check_launch("gated_delta_rule");
}

template <int KN>
int run_back(const TcBackCall& a, cudaStream_t st) {
  const int64_t streams = a.Bt * a.H, nc = cdiv(a.L, Q), seg = segment_chunks(streams, nc);
  CUtensorMap mk, mq, mo;
  if (!map_bf16(&mk, a.B, a.G * a.N, a.L, a.Bt, true) || !map_bf16(&mq, a.C, a.G * a.N, a.L, a.Bt, true) ||
      !map_bf16(&mo, a.dy, a.H * a.P, a.L, a.Bt, false)) {
    set_error("gated_delta_rule_bwd: cuTensorMapEncodeTiled failed");
    return TSSM_ERR_CUDA;
  }
  int* status = device_status_ptr();
  if (!status) {
    set_error("gated_delta_rule_bwd: device status word unavailable");
    return TSSM_ERR_CUDA;
  }
  auto scan = delta_back_scan_kernel<KN>;
  if (cudaFuncSetAttribute(scan, cudaFuncAttributeMaxDynamicSharedMemorySize, BackSmem<KN>::BYTES) != cudaSuccess)
    return check_launch("gated_delta_rule_bwd: set smem attribute");
  for (int64_t end = nc; end > 0; end -= seg) {   // segments from the last; dh0 carries the state's gradient
    const int64_t c0 = std::max<int64_t>(0, end - seg), m = end - c0;
    const PrepCall p{a.B, a.C, a.A_log, a.dt, a.beta, a.img, a.gates, a.Bt, a.L, a.H, a.G, a.N, c0, m, nc, a.scale, 1};
    if (int e = prep_run(p, TSSM_BF16, st)) return e;
    const BackArgs s{a.img, end == nc ? a.dh_last : a.dh0, a.dh0, a.dstates, a.derrs, status, a.L,
                     c0, m, nc, (int)a.H, (int)a.G, (int)a.P, (int)a.N, (int)cdiv(a.P, 128), a.scale};
    scan<<<(unsigned)(streams * s.npb), 384, BackSmem<KN>::BYTES, st>>>(mk, mq, mo, s);
  }
  return check_launch("gated_delta_rule_bwd: chain");
}

}  // namespace

bool tc_takes(int64_t P, int64_t N, int dtype) {
  return dtype == TSSM_BF16 && (N == 64 || N == 128) && P % 64 == 0;
}

int tc_back_run(const TcBackCall& a, cudaStream_t st) {
  TSSM_REQUIRE(a.Bt * a.H * cdiv(a.P, 128) < (int64_t(1) << 31) && a.H * a.P < (int64_t(1) << 31) && a.G * a.N < (int64_t(1) << 31),
               "gated_delta_rule_bwd: size out of range");
  return a.N == 64 ? run_back<64>(a, st) : run_back<128>(a, st);
}

int tc_run(const TcCall& a, cudaStream_t st) {
  TSSM_REQUIRE(a.Bt * a.H * cdiv(a.P, 128) < (int64_t(1) << 31) && a.H * a.P < (int64_t(1) << 31) && a.G * a.N < (int64_t(1) << 31),
               "gated_delta_rule: size out of range");
  return a.N == 64 ? run<64>(a, st) : run<128>(a, st);
}

}  // namespace delta
}  // namespace tssm
