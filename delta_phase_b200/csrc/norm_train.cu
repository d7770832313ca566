// Layer norm for training, forward and backward (norm1, norm_retrieved and norm2 of
// DeltaPhaseHolographicBlock, delta_phase/layers.py:177-244, under autograd):
//   dp_layernorm_fwd : s = x (+ residual), m = mean(s), r = 1 / sqrt(mean((s - m)^2) + eps),
//                      y = (s - m) r w + b; m and r are kept for the backward pass
//   dp_layernorm_bwd : n = (s - m) r, g = w dy,
//                      ds = r (g - mean(g) - n mean(g n)) (+ the gradient that reaches s),
//                      dw = sum_rows dy n, db = sum_rows dy
// All statistics, products and sums are float32.  HBM bounds both passes: a row is held in
// registers between its read and its write, so each pass moves every tensor once.
//   forward : a warp a row up to d = 1024 (no barrier), a block of 256 up to 8192; parameters in
//             pieces from L1, so that 24 warps an SM (32 without a
//             residual) fit their rows into registers.
//   backward: eight columns a thread, so that dw and db of a thread's columns stay in registers
//             while its block walks over the rows; the next rows are loaded meanwhile.  Two
//             resident blocks of 256 threads without spills beat three with (183 against 222 us
//             below); 16-bit rows, half as large, go two at a time (90 against 132 us).  Spills are
//             left where single 16-bit values are loaded (12 to 40 bytes a thread up to d = 1024) and
//             from d = 4097 on, where a block of 1024 has 64 registers a thread (32 to 128 bytes).
// Measured (B200, copy rate 6540 GB/s), forward and backward: 65536 x 1024 bf16 with the float32
// residual 132 us (94% of the copy rate) and 183 us (90%), without 70 us (59%) and 89 us (69%);
// 16384 x 2048 float32 with residual 88 us (93%) and 109 us (94%); 8192 x 4096 bf16 44 us (47%) and
// 56 us (55%); 4096 x 8192 bf16 with residual 82 us (75%) and 122 us (67%); 32768 x 1000 bf16 with
// residual 78 us (77%) and 99 us (81%).  Above d = 8192, single values and several passes over a row:
// 2048 x 16384 bf16 475 us for both.
#include <algorithm>
#include <string>
#include <type_traits>

#include "dp_common.cuh"

namespace dp {
namespace {

constexpr int kLnSms = 148;
constexpr float kNoWeight = 1.0f;

__device__ __forceinline__ float ln_warp_sum(float v) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

template <typename T>
__device__ __forceinline__ void ln_load8(const T *p, float (&v)[8]) {
  const uint4 a = *reinterpret_cast<const uint4 *>(p);
  const T *e = reinterpret_cast<const T *>(&a);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = to_f32(e[i]);
}
template <>
__device__ __forceinline__ void ln_load8<float>(const float *p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <typename T>
__device__ __forceinline__ void ln_store8(T *p, const float (&v)[8]) {
  uint4 a;
  T *e = reinterpret_cast<T *>(&a);
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(v[i]);
  *reinterpret_cast<uint4 *>(p) = a;
}
template <>
__device__ __forceinline__ void ln_store8<float>(float *p, const float (&v)[8]) {
  reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// The columns a thread owns: VEC: groups of eight consecutive ones, 8 (g + G i) + j
// (d a multiple of 8, 16-byte aligned rows); otherwise single ones, g + G (8 i + j).
// Columns past d read 0 and are not written.
template <int G, int NV, bool VEC, typename T>
__device__ __forceinline__ void ln_load_row(const T *row, int g, int d, float (&v)[NV][8]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (VEC) {
      const int c = 8 * (g + G * i);
      if (c < d) {
        ln_load8(row + c, v[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = g + G * (8 * i + j);
        v[i][j] = c < d ? to_f32(row[c]) : 0.f;
      }
    }
  }
}
template <int G, int NV, bool VEC, typename T>
__device__ __forceinline__ void ln_store_row(T *row, int g, int d, const float (&v)[NV][8]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (VEC) {
      const int c = 8 * (g + G * i);
      if (c < d) ln_store8(row + c, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = g + G * (8 * i + j);
        if (c < d) row[c] = from_f32<T>(v[i][j]);
      }
    }
  }
}
// The same by dtype code: the branch is uniform over the grid, the loads of a row stay
// together inside it, and one kernel serves every combination of types.
template <int G, int NV, bool VEC>
__device__ __forceinline__ void ln_load_row(const void *p, int dt, int64_t off, int g, int d, float (&v)[NV][8]) {
  if (dt == DP_F32)
    ln_load_row<G, NV, VEC>(static_cast<const float *>(p) + off, g, d, v);
  else if (dt == DP_BF16)
    ln_load_row<G, NV, VEC>(static_cast<const __nv_bfloat16 *>(p) + off, g, d, v);
  else
    ln_load_row<G, NV, VEC>(static_cast<const __half *>(p) + off, g, d, v);
}
template <int G, int NV, bool VEC>
__device__ __forceinline__ void ln_store_row(void *p, int dt, int64_t off, int g, int d, const float (&v)[NV][8]) {
  if (dt == DP_F32)
    ln_store_row<G, NV, VEC>(static_cast<float *>(p) + off, g, d, v);
  else if (dt == DP_BF16)
    ln_store_row<G, NV, VEC>(static_cast<__nv_bfloat16 *>(p) + off, g, d, v);
  else
    ln_store_row<G, NV, VEC>(static_cast<__half *>(p) + off, g, d, v);
}
__device__ __forceinline__ float ln_load1(const void *p, int dt, int64_t i) {
  if (dt == DP_F32) return static_cast<const float *>(p)[i];
  if (dt == DP_BF16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
  return __half2float(static_cast<const __half *>(p)[i]);
}
__device__ __forceinline__ void ln_store1(void *p, int dt, int64_t i, float v) {
  if (dt == DP_F32)
    static_cast<float *>(p)[i] = v;
  else if (dt == DP_BF16)
    static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
  else
    static_cast<__half *>(p)[i] = __float2half_rn(v);
}

// ---------------------------------------------------------------- forward
struct LnFwdArgs {
  const void *x;
  const float *res, *w, *b;
  float *sum, *mean, *rstd;
  void *y;
  int x_dt, y_dt, d;
  int64_t rows;
  float eps;
};

// Sum over the G threads of a row: a warp, or the whole block through `slot`.
template <int G>
__device__ __forceinline__ float ln_group_sum(float v, float *slot) {
  v = ln_warp_sum(v);
  if (G == 32) return v;
  if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < G / 32; ++i) t += slot[i];
  return t;
}

// G threads per row, 8 NV columns per thread.  RES: there may be a residual; without its registers a
// third to twice as many warps fit on an SM (65536 x 1024 bf16 80 -> 70 us, 8192 x 8192 83 -> 71).
template <int G, int NV, bool VEC, bool RES>
__global__ void __launch_bounds__(G == 32 ? 128 : G, G == 32 ? (RES ? 6 : 8) : RES ? 2 : 4) ln_fwd_kernel(LnFwdArgs a) {
  __shared__ float slot[2][G / 32];
  const int g = threadIdx.x % G;
  const int64_t r = (int64_t)blockIdx.x * (blockDim.x / G) + threadIdx.x / G;
  if (r >= a.rows) return;  // a whole warp (G = 32) or never (one row per block)
  const int64_t off = r * a.d;
  float v[NV][8], t[NV][8];
  // the residual first: x is converted, and waited for, where it is loaded (132 against 138 us)
  if (RES && a.res) ln_load_row<G, NV, VEC>(a.res + off, g, a.d, t);
  ln_load_row<G, NV, VEC>(a.x, a.x_dt, off, g, a.d, v);
  if (RES && a.res) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] += t[i][j];
    ln_store_row<G, NV, VEC>(a.sum + off, g, a.d, v);
  }
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) s += v[i][j];
  const float mean = ln_group_sum<G>(s, slot[0]) / (float)a.d;
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = VEC ? 8 * (g + G * i) : g + G * (8 * i + j);
      const float t = v[i][j] - mean;
      if (c < a.d) q = fmaf(t, t, q);
      v[i][j] = t;
    }
  const float rstd = rsqrtf(ln_group_sum<G>(q, slot[1]) / (float)a.d + a.eps);
  if (g == 0) {
    a.mean[r] = mean;
    a.rstd[r] = rstd;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    // the parameters eight columns at a time (L1), not all of them in registers
    float w[1][8], b[1][8];
    const int gi = VEC ? g + G * i : g + 8 * G * i;
    if (a.w) ln_load_row<G, 1, VEC>(a.w, gi, a.d, w);
    if (a.b) ln_load_row<G, 1, VEC>(a.b, gi, a.d, b);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      v[i][j] = fmaf(v[i][j] * rstd, a.w ? w[0][j] : kNoWeight, a.b ? b[0][j] : 0.f);
  }
  ln_store_row<G, NV, VEC>(a.y, a.y_dt, off, g, a.d, v);
}

__device__ __forceinline__ float ln_block_sum(float v, float *slot) {  // 1024 threads
  v = ln_warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
  __syncthreads();
  return ln_warp_sum(slot[threadIdx.x & 31]);
}

// Rows too wide for the registers of a block: the row is read again from L2 in each pass.
__global__ void __launch_bounds__(1024) ln_fwd_wide_kernel(LnFwdArgs a) {
  __shared__ float slot[32];
  const int64_t off = (int64_t)blockIdx.x * a.d;
  // s: written first, then read back by the thread that wrote it (sum may be the residual)
  auto value = [&](int c) { return a.res ? a.sum[off + c] : ln_load1(a.x, a.x_dt, off + c); };
  float s = 0.f;
  for (int c = threadIdx.x; c < a.d; c += 1024) {
    float v = ln_load1(a.x, a.x_dt, off + c);
    if (a.res) {
      v += a.res[off + c];
      a.sum[off + c] = v;
    }
    s += v;
  }
  const float mean = ln_block_sum(s, slot) / (float)a.d;
  float q = 0.f;
  for (int c = threadIdx.x; c < a.d; c += 1024) {
    const float t = value(c) - mean;
    q = fmaf(t, t, q);
  }
  const float rstd = rsqrtf(ln_block_sum(q, slot) / (float)a.d + a.eps);
  if (threadIdx.x == 0) {
    a.mean[blockIdx.x] = mean;
    a.rstd[blockIdx.x] = rstd;
  }
  for (int c = threadIdx.x; c < a.d; c += 1024)
    ln_store1(a.y, a.y_dt, off + c,
              fmaf((value(c) - mean) * rstd, a.w ? a.w[c] : kNoWeight, a.b ? a.b[c] : 0.f));
}

// ---------------------------------------------------------------- backward
struct LnBwdArgs {
  const void *s, *dy;
  const float *w, *mean, *rstd, *dsum;
  void *dx;
  float *dres, *part;  // part: (blocks, 2, d) partial dw, db; null when neither is wanted
  int s_dt, dy_dt, dx_dt, d;
  int64_t rows;
};

// Resident blocks of the backward kernel: all of them run at once and walk over the rows.
constexpr int ln_bwd_per_sm(int G) { return G <= 256 ? 2 : 1; }

// Eight columns of a row as they lie in memory (vectors, or single values), loaded a row ahead
// and converted when their turn comes.  WIDE: float32; otherwise a 16-bit type by its code.
template <int G, bool VEC, bool WIDE>
struct LnRaw {
  static constexpr int N = VEC && !WIDE ? 4 : 8;
  uint32_t r[N];
  __device__ __forceinline__ void load(const void *p, int64_t off, int g, int d) {
    if constexpr (VEC) {
#pragma unroll
      for (int j = 0; j < N; ++j) r[j] = 0;
      if (8 * g < d) {
        const uint4 *q = reinterpret_cast<const uint4 *>(static_cast<const char *>(p) + (off + 8 * g) * (WIDE ? 4 : 2));
#pragma unroll
        for (int j = 0; j < N / 4; ++j) {
          const uint4 a = q[j];
          r[4 * j] = a.x, r[4 * j + 1] = a.y, r[4 * j + 2] = a.z, r[4 * j + 3] = a.w;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int64_t i = off + g + G * j;
        r[j] = g + G * j >= d ? 0u
               : WIDE         ? static_cast<const uint32_t *>(p)[i]
                              : (uint32_t)static_cast<const unsigned short *>(p)[i];
      }
    }
  }
  __device__ __forceinline__ float get(int dt, int j) const {
    if constexpr (WIDE)
      return __uint_as_float(r[j]);
    else if constexpr (VEC)
      return raw_scalar_to_f32(j & 1 ? r[j / 2] >> 16 : r[j / 2] & 0xffffu, dt);
    else
      return raw_scalar_to_f32(r[j], dt);
  }
};

// G threads per row, eight columns per thread; a block is max(G, 256) threads.  The block
// walks over the rows (grid-stride), each thread adding up dw and db of its own columns in
// registers; at the end the block writes one partial row, and ln_bwd_reduce_kernel adds
// the blocks' rows in a fixed order (the result does not depend on timing).  The two sums
// of a row cross the block through shared memory, R rows a barrier; the next rows' s and dy are
// on their way meanwhile.
template <int G, bool VEC, bool S32, bool D32>
__global__ void __launch_bounds__(G < 256 ? 256 : G, ln_bwd_per_sm(G)) ln_bwd_kernel(LnBwdArgs a) {
  constexpr int BT = G < 256 ? 256 : G, NG = BT / G, W = G / 32;
  constexpr int R = S32 || D32 || G == 1024 ? 1 : 2;  // rows a group handles between two barriers
  constexpr bool KEEP_W = G < 1024;  // 64 registers a thread: the weight is read again for every row (L1)
  __shared__ float2 red[2][NG][R][W];
  __shared__ float comb[NG > 1 ? NG : 1][NG > 1 ? G * 8 : 1];
  const int g = threadIdx.x % G, grp = threadIdx.x / G;
  float w[1][8], aw[8], ab[8];
  auto weight = [&] {
    if (a.w) {
      ln_load_row<G, 1, VEC>(a.w, g, a.d, w);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[0][j] = kNoWeight;
    }
  };
  if (KEEP_W) weight();
#pragma unroll
  for (int j = 0; j < 8; ++j) aw[j] = ab[j] = 0.f;
  const float inv_d = 1.f / (float)a.d;
  const int64_t step = (int64_t)gridDim.x * NG * R;
  int64_t r = ((int64_t)blockIdx.x * NG + grp) * R;
  LnRaw<G, VEC, S32> rs[R];
  LnRaw<G, VEC, D32> rd[R];
  float mean[R], rstd[R];
  auto fetch = [&](int64_t row0) {  // a row past the end reads zeros
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const int64_t row = row0 + k;
      const bool on = row < a.rows;
      rs[k].load(a.s, row * a.d, g, on ? a.d : 0);
      rd[k].load(a.dy, row * a.d, g, on ? a.d : 0);
      mean[k] = on ? a.mean[row] : 0.f;
      rstd[k] = on ? a.rstd[row] : 0.f;
    }
  };
  fetch(r);
  int buf = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * NG * R; r0 < a.rows; r0 += step, r += step, buf ^= 1) {
    if (!KEEP_W) weight();
    float n[R][8], gv[R][1][8], rr[R], s1[R], s2[R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      s1[k] = s2[k] = 0.f;
      rr[k] = rstd[k];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        n[k][j] = (rs[k].get(a.s_dt, j) - mean[k]) * rr[k];
        const float t = rd[k].get(a.dy_dt, j);
        aw[j] = fmaf(t, n[k][j], aw[j]);
        ab[j] += t;
        gv[k][0][j] = t * w[0][j];
        s1[k] += gv[k][0][j];
        s2[k] = fmaf(gv[k][0][j], n[k][j], s2[k]);
      }
    }
    float ds[1][8];  // with R = 1 (a residual comes with a float32 s); read in its place otherwise
    if (R == 1 && a.dsum) ln_load_row<G, 1, VEC>(a.dsum + r * a.d, g, r < a.rows ? a.d : 0, ds);
    fetch(r + step);
#pragma unroll
    for (int k = 0; k < R; ++k) {
      s1[k] = ln_warp_sum(s1[k]);
      s2[k] = ln_warp_sum(s2[k]);
    }
    if (W > 1) {
      if ((threadIdx.x & 31) == 0) {
#pragma unroll
        for (int k = 0; k < R; ++k) red[buf][grp][k][g >> 5] = make_float2(s1[k], s2[k]);
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < R; ++k) {
        s1[k] = s2[k] = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const float2 t = red[buf][grp][k][i];
          s1[k] += t.x;
          s2[k] += t.y;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < R; ++k) {
      if (r + k >= a.rows) continue;
      const int64_t off = (r + k) * a.d;
      const float c1 = s1[k] * inv_d, c2 = s2[k] * inv_d;
      if (R > 1 && a.dsum) ln_load_row<G, 1, VEC>(a.dsum + off, g, a.d, ds);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float t = rr[k] * (gv[k][0][j] - c1 - n[k][j] * c2);
        if (a.dsum) t += ds[0][j];
        gv[k][0][j] = t;
      }
      if (a.dx) ln_store_row<G, 1, VEC>(a.dx, a.dx_dt, off, g, a.d, gv[k]);
      if (a.dres) ln_store_row<G, 1, VEC>(a.dres + off, g, a.d, gv[k]);
    }
  }
  if (!a.part) return;
  float *pw = a.part + (int64_t)blockIdx.x * 2 * a.d;
#pragma unroll
  for (int pass = 0; pass < 2; ++pass) {
    float v[1][8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[0][j] = pass ? ab[j] : aw[j];
    if (NG > 1) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) comb[grp][g + G * j] = v[0][j];
      __syncthreads();
      if (grp == 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          for (int i = 1; i < NG; ++i) v[0][j] += comb[i][g + G * j];
      }
    }
    if (grp == 0) ln_store_row<G, 1, VEC>(pw + pass * a.d, g, a.d, v);
  }
}

// Rows wider than the registers of a block: two passes over the row, the second from L2;
// dw and db are added up in the block's partial row itself (L2), one owner per column.
__global__ void __launch_bounds__(1024) ln_bwd_wide_kernel(LnBwdArgs a) {
  __shared__ float slot[32];
  float *pw = a.part ? a.part + (int64_t)blockIdx.x * 2 * a.d : nullptr;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const int64_t off = r * a.d;
    const float mean = a.mean[r], rs = a.rstd[r];
    const bool first = r == blockIdx.x;
    float s1 = 0.f, s2 = 0.f;
    for (int c = threadIdx.x; c < a.d; c += 1024) {
      const float n = (ln_load1(a.s, a.s_dt, off + c) - mean) * rs, t = ln_load1(a.dy, a.dy_dt, off + c);
      const float gv = t * (a.w ? a.w[c] : kNoWeight);
      s1 += gv;
      s2 = fmaf(gv, n, s2);
      if (pw) {
        pw[c] = first ? t * n : fmaf(t, n, pw[c]);
        pw[a.d + c] = first ? t : t + pw[a.d + c];
      }
    }
    const float c1 = ln_block_sum(s1, slot) / (float)a.d, c2 = ln_block_sum(s2, slot) / (float)a.d;
    for (int c = threadIdx.x; c < a.d; c += 1024) {
      const float n = (ln_load1(a.s, a.s_dt, off + c) - mean) * rs, t = ln_load1(a.dy, a.dy_dt, off + c);
      float v = rs * (t * (a.w ? a.w[c] : kNoWeight) - c1 - n * c2);
      if (a.dsum) v += a.dsum[off + c];
      if (a.dx) ln_store1(a.dx, a.dx_dt, off + c, v);
      if (a.dres) a.dres[off + c] = v;
    }
  }
}

// Column sums of the partial rows: block (32, 32), 32 columns of dw (blockIdx.y = 0) or
// db (1); thread (x, y) adds the partial rows y, y + 32, ..., then a warp adds the 32.
__global__ void __launch_bounds__(1024) ln_bwd_reduce_kernel(const float *part, int np, int d, float *dw, float *db) {
  __shared__ float t[32][33];
  pdl_wait();
  float *out = blockIdx.y ? db : dw;
  if (!out) return;
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + x;
  float s = 0.f;
  if (c < d)
    for (int p = y; p < np; p += 32) s += part[((int64_t)p * 2 + blockIdx.y) * d + c];
  t[y][x] = s;
  __syncthreads();
  const float v = ln_warp_sum(t[x][y]);
  if (x == 0 && blockIdx.x * 32 + y < d) out[blockIdx.x * 32 + y] = v;
}

// Threads per row of the backward kernel: eight columns each; 0: the wide kernel.
int ln_bwd_group(int d) {
  for (int g = 32; g <= 1024; g *= 2)
    if (d <= 8 * g) return g;
  return 0;
}

// Blocks of the backward kernel (and partial rows in its workspace): those that are resident at
// once, fewer when there are fewer rows.
int ln_bwd_blocks(int64_t rows, int d) {
  const int G = ln_bwd_group(d);
  if (G == 0) return (int)std::min<int64_t>(rows, kLnSms);
  const int ng = G < 256 ? 256 / G : 1;
  return (int)std::min<int64_t>((rows + ng - 1) / ng, (int64_t)kLnSms * ln_bwd_per_sm(G));
}

bool ln_al16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace dp

extern "C" int dp_layernorm_fwd(const void *x, int x_dtype, const float *residual, const float *ln_w,
                                const float *ln_b, float eps, float *sum_out, void *y, int y_dtype, float *mean,
                                float *rstd, int64_t rows, int d, void *stream) {
  using namespace dp;
  DP_REQUIRE(rows >= 0 && d >= 1, DP_ERR_INVALID_ARGUMENT, "dp_layernorm_fwd: bad sizes");
  DP_REQUIRE(valid_dtype(x_dtype) && valid_dtype(y_dtype), DP_ERR_INVALID_ARGUMENT,
             "dp_layernorm_fwd: unknown dtype code");
  if (rows == 0) return DP_OK;
  DP_REQUIRE(x && y && mean && rstd, DP_ERR_INVALID_ARGUMENT, "dp_layernorm_fwd: null pointer");
  DP_REQUIRE(!residual == !sum_out, DP_ERR_INVALID_ARGUMENT,
             "dp_layernorm_fwd: residual and sum_out come together");
  DP_REQUIRE(rows < (1ll << 31), DP_ERR_UNSUPPORTED, "dp_layernorm_fwd: too many rows");
  DP_REQUIRE(d <= 1 << 30, DP_ERR_UNSUPPORTED, "dp_layernorm_fwd: d must be <= 2^30");
  LnFwdArgs a{x, residual, ln_w, ln_b, sum_out, mean, rstd, y, x_dtype, y_dtype, d, rows, eps};
  cudaStream_t st = as_stream(stream);
  const bool vec = d % 8 == 0 && ln_al16(x) && ln_al16(residual) && ln_al16(ln_w) && ln_al16(ln_b) &&
                   ln_al16(sum_out) && ln_al16(y);
  // a warp per row up to d = 1024 (no barrier), a block of 256 up to 8192, then the wide kernel
  auto run = [&](auto v, auto res) {
    constexpr bool V = decltype(v)::value, R = decltype(res)::value;
    auto launch = [&](auto kern, int G) {
      const int threads = G == 32 ? 128 : G;
      const int per = threads / G;
      kern<<<(unsigned)((rows + per - 1) / per), threads, 0, st>>>(a);
    };
    if (d <= 256)
      launch(ln_fwd_kernel<32, 1, V, R>, 32);
    else if (d <= 512)
      launch(ln_fwd_kernel<32, 2, V, R>, 32);
    else if (d <= 1024)
      launch(ln_fwd_kernel<32, 4, V, R>, 32);
    else if (d <= 2048)
      launch(ln_fwd_kernel<256, 1, V, R>, 256);
    else if (d <= 4096)
      launch(ln_fwd_kernel<256, 2, V, R>, 256);
    else
      launch(ln_fwd_kernel<256, 4, V, R>, 256);
  };
  if (d > 8192)
    ln_fwd_wide_kernel<<<(unsigned)rows, 1024, 0, st>>>(a);
  else if (vec)
    residual ? run(std::true_type{}, std::true_type{}) : run(std::true_type{}, std::false_type{});
  else  // single values: bound by their many loads, not by warps (20000 x 1001 f16: 36 us, without RES 39)
    run(std::false_type{}, std::true_type{});
  return check_launch("dp_layernorm_fwd");
}

extern "C" size_t dp_layernorm_bwd_workspace_size(int64_t rows, int d) {
  if (rows <= 0 || d <= 0) return 0;
  return (size_t)dp::ln_bwd_blocks(rows, d) * 2 * (size_t)d * sizeof(float);
}

extern "C" int dp_layernorm_bwd(const void *s, int s_dtype, const void *dy, int dy_dtype, const float *ln_w,
                                const float *mean, const float *rstd, const float *grad_sum, void *dx, int dx_dtype,
                                float *grad_residual, float *grad_w, float *grad_b, int64_t rows, int d,
                                void *workspace, size_t workspace_bytes, void *stream) {
  using namespace dp;
  DP_REQUIRE(rows >= 0 && d >= 1, DP_ERR_INVALID_ARGUMENT, "dp_layernorm_bwd: bad sizes");
  DP_REQUIRE(valid_dtype(s_dtype) && valid_dtype(dy_dtype) && valid_dtype(dx_dtype), DP_ERR_INVALID_ARGUMENT,
             "dp_layernorm_bwd: unknown dtype code");
  DP_REQUIRE(rows < (1ll << 31), DP_ERR_UNSUPPORTED, "dp_layernorm_bwd: too many rows");
  DP_REQUIRE(d <= 1 << 30, DP_ERR_UNSUPPORTED, "dp_layernorm_bwd: d must be <= 2^30");
  cudaStream_t st = as_stream(stream);
  if (rows == 0) {  // the sums over no rows
    cudaError_t e = cudaSuccess;
    if (grad_w) e = cudaMemsetAsync(grad_w, 0, (size_t)d * sizeof(float), st);
    if (e == cudaSuccess && grad_b) e = cudaMemsetAsync(grad_b, 0, (size_t)d * sizeof(float), st);
    if (e != cudaSuccess)
      return set_error(DP_ERR_CUDA, std::string("dp_layernorm_bwd: ") + cudaGetErrorString(e));
    return DP_OK;
  }
  DP_REQUIRE(s && dy && mean && rstd, DP_ERR_INVALID_ARGUMENT, "dp_layernorm_bwd: null pointer");
  const int np = ln_bwd_blocks(rows, d);
  const bool sums = grad_w || grad_b;
  DP_REQUIRE(!sums || (workspace && workspace_bytes >= dp_layernorm_bwd_workspace_size(rows, d)), DP_ERR_WORKSPACE,
             "dp_layernorm_bwd: workspace too small");
  float *part = sums ? static_cast<float *>(workspace) : nullptr;
  LnBwdArgs a{s, dy, ln_w, mean, rstd, grad_sum, dx, grad_residual, part, s_dtype, dy_dtype, dx_dtype, d, rows};
  DP_REQUIRE(!sums || (reinterpret_cast<uintptr_t>(workspace) & 15) == 0, DP_ERR_MISALIGNED,
             "dp_layernorm_bwd: the workspace must be 16-byte aligned");
  const bool vec = d % 8 == 0 && ln_al16(s) && ln_al16(dy) && ln_al16(ln_w) && ln_al16(grad_sum) && ln_al16(dx) &&
                   ln_al16(grad_residual);
  auto run = [&](auto s32, auto d32) {
    constexpr bool S = decltype(s32)::value, D = decltype(d32)::value;
    auto launch = [&](auto kern, int G) { kern<<<np, G < 256 ? 256 : G, 0, st>>>(a); };
    switch (ln_bwd_group(d)) {
      case 32: vec ? launch(ln_bwd_kernel<32, true, S, D>, 32) : launch(ln_bwd_kernel<32, false, S, D>, 32); break;
      case 64: vec ? launch(ln_bwd_kernel<64, true, S, D>, 64) : launch(ln_bwd_kernel<64, false, S, D>, 64); break;
      case 128: vec ? launch(ln_bwd_kernel<128, true, S, D>, 128) : launch(ln_bwd_kernel<128, false, S, D>, 128); break;
      case 256: vec ? launch(ln_bwd_kernel<256, true, S, D>, 256) : launch(ln_bwd_kernel<256, false, S, D>, 256); break;
      case 512: vec ? launch(ln_bwd_kernel<512, true, S, D>, 512) : launch(ln_bwd_kernel<512, false, S, D>, 512); break;
      case 1024:
        vec ? launch(ln_bwd_kernel<1024, true, S, D>, 1024) : launch(ln_bwd_kernel<1024, false, S, D>, 1024);
        break;
      default: ln_bwd_wide_kernel<<<np, 1024, 0, st>>>(a);
    }
  };
  const bool s32 = s_dtype == DP_F32, d32 = dy_dtype == DP_F32;
  if (s32)
    d32 ? run(std::true_type{}, std::true_type{}) : run(std::true_type{}, std::false_type{});
  else
    d32 ? run(std::false_type{}, std::true_type{}) : run(std::false_type{}, std::false_type{});
  const int rc = check_launch("dp_layernorm_bwd");
  if (rc != DP_OK || !sums) return rc;
  return pdl_status(launch_pdl(ln_bwd_reduce_kernel, dim3((d + 31) / 32, 2), dim3(1024), 0, st, a.part, np, d, grad_w,
                               grad_b),
                    "ln_bwd_reduce_kernel");
}
