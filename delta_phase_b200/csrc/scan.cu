// Gated linear recurrence over long sequences, forward and backward: the vector-state
// counterpart of LaplacePhaseCore's per-row decay (delta_phase/layers.py:481-561).
//   h_t = a_t h_{t-1} + u_t per channel, out_t = h_t;  with d_t = 1 - a_t:
//   DP_SCAN_DECAY   a = exp(gate),     u = x
//   DP_SCAN_SIGMOID a = sigmoid(gate), u = d x
// Backward: p_t = dout_t + q_{t+1}, q_t = a_t p_t (q_L = dL/dh_{L-1} from outside):
//   decay: dx = p, dgate = q h_{t-1};  sigmoid: dx = d p, dgate = q d (h_{t-1} - x)
//   and dL/dh_{-1} = q_0.
//
// Everything is kept in terms of the drop d, not of a: a close to 1 has lost the digits of
// 1 - a, which is what a long memory consists of.  h - d h is one fused multiply-add, exact
// in d, and a gate that drops the state (d = 1) leaves exactly nothing of it.
//
// Layout: a lane owns the channels of one 4-byte word (two 16-bit values or one float), a
// warp kTok consecutive tokens of its 32 words, a block kWarps warps (kTile tokens), and a
// thread-block cluster up to 16 consecutive tiles of one sequence.  Each warp reduces its
// tokens to an affine map h -> (1 - d) h + H, the maps are combined through shared memory
// inside the block and through distributed shared memory inside the cluster (one cluster
// barrier per 16 tiles), and each warp then runs the recurrence over its tokens again from
// the exact state that reaches it: every input is read from HBM once, the order of all sums
// is fixed.  A cluster walks over a long sequence in steps of its span.
#include <cooperative_groups.h>

#include <algorithm>
#include <string>

#include "dp_common.cuh"

namespace cg = cooperative_groups;

namespace dp {
namespace {

constexpr int kTok = 16;               // tokens per warp
constexpr int kWarps = 8;              // warps per block
constexpr int kTile = kTok * kWarps;   // tokens per block; one saved state per tile
constexpr int kMaxCluster = 16;
constexpr int kThreads = kWarps * 32;

// ---------------------------------------------------------------- gates
// 1 - exp(g).  float32: the library's accurate form.  16-bit inputs: a Taylor polynomial
// near 0 (|g| < 1/4: the first term left out is below 5e-8 of the value) and the hardware
// exponential elsewhere (relative error below 1e-6), far below the rounding of g itself.
template <typename T>
__device__ __forceinline__ float drop_of_log(float g) {
  float p = fmaf(g, 1.f / 720.f, 1.f / 120.f);
  p = fmaf(g, p, 1.f / 24.f);
  p = fmaf(g, p, 1.f / 6.f);
  p = fmaf(g, p, 0.5f);
  p = fmaf(g, p, 1.f);
  return fabsf(g) < 0.25f ? -g * p : 1.f - __expf(g);
}
template <>
__device__ __forceinline__ float drop_of_log<float>(float g) { return -expm1f(g); }

// 1 - sigmoid(f) = 1 / (1 + exp(f))
template <typename T>
__device__ __forceinline__ float drop_of_logit(float f) { return __fdividef(1.f, 1.f + __expf(f)); }
template <>
__device__ __forceinline__ float drop_of_logit<float>(float f) { return 1.f / (1.f + expf(f)); }

template <typename T, int MODE>
__device__ __forceinline__ float drop_of(float g) {
  return MODE == DP_SCAN_SIGMOID ? drop_of_logit<T>(g) : drop_of_log<T>(g);
}

// The affine map of some tokens: h -> (1 - d) h + H.
struct Map {
  float d, H;
};
__device__ __forceinline__ float apply(const Map &m, float h) { return fmaf(-m.d, h, h) + m.H; }

// ---------------------------------------------------------------- words of channels
// V channels of type T in a word (V = 2: a 16-bit pair, 4-byte aligned; V = 1: one value).
template <typename T, int V>
struct Word;
template <typename T>
struct Word<T, 1> {
  T v;
  __device__ __forceinline__ float get(int) const { return to_f32(v); }
  __device__ __forceinline__ void set(int, float x) { v = from_f32<T>(x); }
};
template <typename T>
struct __align__(4) Word<T, 2> {
  T v[2];
  __device__ __forceinline__ float get(int i) const { return to_f32(v[i]); }
  __device__ __forceinline__ void set(int i, float x) { v[i] = from_f32<T>(x); }
};
template <typename T, int V>
__device__ __forceinline__ Word<T, V> word_zero() {
  Word<T, V> w;
#pragma unroll
  for (int i = 0; i < V; ++i) w.set(i, 0.f);
  return w;
}

struct ScanArgs {
  const void *x, *gate, *dout;  // (B, L, D), strides {sb, st}
  const float *h0;              // (B, D) or null
  float *hL;                    // (B, D) final state
  float *saved;                 // (B, ceil(L / kTile), D) state before each tile (forward: or null)
  void *out, *dx, *dgate;
  const float *dhL;             // (B, D) or null
  float *dh0;                   // (B, D) or null
  int64_t xs[2], gs[2], os[2];  // strides of x, gate and of out (forward) or dout (backward)
  int B, L, D, tiles_c, cs;
};

// Shared memory of another block may be written only once that block runs.
__device__ __forceinline__ void scan_start(int cs) {
  if (cs > 1) cg::this_cluster().sync();
}
// Every block's map has reached every block of the cluster.  The buffers alternate, so one
// barrier per span is enough: a block that writes a buffer again has passed the barrier of
// the span between, which every thread that read the buffer has reached.
__device__ __forceinline__ void scan_sync(int cs) {
  if (cs > 1)
    cg::this_cluster().sync();
  else
    __syncthreads();
}

// ---------------------------------------------------------------- forward
template <typename T, int V, int MODE>
__global__ void __launch_bounds__(kThreads) scan_fwd_kernel(ScanArgs a) {
  constexpr int C = 32 * V;
  __shared__ Map wmap[2][kWarps][C];
  __shared__ Map bmap[2][kMaxCluster][C];
  const int rank = blockIdx.x % a.cs, chain = blockIdx.x / a.cs;
  const int b = chain / a.tiles_c, c0 = (chain % a.tiles_c) * C;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c = c0 + lane * V;
  const bool on = c < a.D;  // D is a multiple of V
  const T *x = static_cast<const T *>(a.x) + b * a.xs[0] + c;
  const T *gate = static_cast<const T *>(a.gate) + b * a.gs[0] + c;
  T *out = static_cast<T *>(a.out) + b * a.os[0] + c;
  float h[V];
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = on && a.h0 ? a.h0[(int64_t)b * a.D + c + v] : 0.f;
  const int span = a.cs * kTile, tiles = (a.L + kTile - 1) / kTile;
  scan_start(a.cs);
  int buf = 0;
  for (int64_t base = 0; base < a.L; base += span, buf ^= 1) {
    const int64_t tile0 = base + rank * kTile, t0 = tile0 + warp * kTok;
    const int n = (int)min((int64_t)kTok, max((int64_t)0, (int64_t)a.L - t0));
    Word<T, V> xw[kTok], gw[kTok];
#pragma unroll
    for (int i = 0; i < kTok; ++i) {
      if (on && i < n) {
        xw[i] = *reinterpret_cast<const Word<T, V> *>(x + (t0 + i) * a.xs[1]);
        gw[i] = *reinterpret_cast<const Word<T, V> *>(gate + (t0 + i) * a.gs[1]);
      }
    }
    float d[kTok][V];
    Map m[V];
#pragma unroll
    for (int v = 0; v < V; ++v) m[v] = {0.f, 0.f};
    float dmax[V];
#pragma unroll
    for (int v = 0; v < V; ++v) dmax[v] = 0.f;
#pragma unroll
    for (int i = 0; i < kTok; ++i) {
      if (!(on && i < n)) xw[i] = word_zero<T, V>();
#pragma unroll
      for (int v = 0; v < V; ++v) {
        d[i][v] = on && i < n ? drop_of<T, MODE>(gw[i].get(v)) : 0.f;
        const float xv = xw[i].get(v), u = MODE == DP_SCAN_SIGMOID ? d[i][v] * xv : xv;
        m[v].H = fmaf(-d[i][v], m[v].H, m[v].H) + u;
        m[v].d = fmaf(-d[i][v], m[v].d, m[v].d) + d[i][v];
        dmax[v] = fmaxf(dmax[v], d[i][v]);
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (dmax[v] == 1.f) m[v].d = 1.f;  // a dropped state stays dropped: no rounding brings it back
      wmap[buf][warp][lane * V + v] = m[v];
    }
    __syncthreads();
    // the block's map, by its last warp, to every block of the cluster
    if (warp == kWarps - 1) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        Map r = wmap[buf][0][lane * V + v];
        bool drop = r.d == 1.f;
#pragma unroll
        for (int j = 1; j < kWarps; ++j) {
          const Map w = wmap[buf][j][lane * V + v];
          r.H = apply(w, r.H);
          r.d = fmaf(-w.d, r.d, r.d) + w.d;
          drop |= w.d == 1.f;
        }
        if (drop) r.d = 1.f;
        if (a.cs > 1) {
          for (int k = 0; k < a.cs; ++k) cg::this_cluster().map_shared_rank(&bmap[buf][rank][lane * V + v], k)[0] = r;
        } else {
          bmap[buf][0][lane * V + v] = r;
        }
      }
    }
    scan_sync(a.cs);
    // the state that reaches this block, this warp, and the next span
    float in[V];
#pragma unroll
    for (int v = 0; v < V; ++v) in[v] = h[v];
    for (int k = 0; k < a.cs; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (k == rank) in[v] = h[v];
        h[v] = apply(bmap[buf][k][lane * V + v], h[v]);
      }
    if (warp == 0 && a.saved && on && tile0 < a.L)
#pragma unroll
      for (int v = 0; v < V; ++v) a.saved[((int64_t)b * tiles + tile0 / kTile) * a.D + c + v] = in[v];
    for (int j = 0; j < warp; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) in[v] = apply(wmap[buf][j][lane * V + v], in[v]);
#pragma unroll
    for (int i = 0; i < kTok; ++i) {
      Word<T, V> o;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float xv = xw[i].get(v), u = MODE == DP_SCAN_SIGMOID ? d[i][v] * xv : xv;
        in[v] = fmaf(-d[i][v], in[v], in[v]) + u;
        o.set(v, in[v]);
      }
      if (on && i < n) *reinterpret_cast<Word<T, V> *>(out + (t0 + i) * a.os[1]) = o;
    }
  }
  if (on && rank == 0 && warp == 0)
#pragma unroll
    for (int v = 0; v < V; ++v) a.hL[(int64_t)b * a.D + c + v] = h[v];
}

// ---------------------------------------------------------------- backward
// The same walk from the end of the sequence.  The states before each token come from the
// saved state of the tile and the forward maps of the warps before; the gradient q that
// flows to earlier tokens is an affine map too (h -> (1 - d) h + Q with the same d).
struct Map3 {
  float d, H, Q;
};

template <typename T, int V, int MODE>
__global__ void __launch_bounds__(kThreads) scan_bwd_kernel(ScanArgs a) {
  constexpr int C = 32 * V;
  __shared__ Map3 wmap[2][kWarps][C];
  __shared__ Map bmap[2][kMaxCluster][C];
  const int rank = blockIdx.x % a.cs, chain = blockIdx.x / a.cs;
  const int b = chain / a.tiles_c, c0 = (chain % a.tiles_c) * C;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c = c0 + lane * V;
  const bool on = c < a.D;
  const T *x = static_cast<const T *>(a.x) + b * a.xs[0] + c;
  const T *gate = static_cast<const T *>(a.gate) + b * a.gs[0] + c;
  const T *dout = static_cast<const T *>(a.dout) + b * a.os[0] + c;
  T *dx = static_cast<T *>(a.dx) + (int64_t)b * a.L * a.D + c;
  T *dg = static_cast<T *>(a.dgate) + (int64_t)b * a.L * a.D + c;
  float q[V];
#pragma unroll
  for (int v = 0; v < V; ++v) q[v] = on && a.dhL ? a.dhL[(int64_t)b * a.D + c + v] : 0.f;
  const int span = a.cs * kTile, tiles = (a.L + kTile - 1) / kTile;
  scan_start(a.cs);
  int buf = 0;
  for (int64_t base = ((int64_t)(a.L - 1) / span) * span; base >= 0; base -= span, buf ^= 1) {
    const int64_t tile0 = base + rank * kTile, t0 = tile0 + warp * kTok;
    const int n = (int)min((int64_t)kTok, max((int64_t)0, (int64_t)a.L - t0));
    Word<T, V> xw[kTok], gw[kTok], yw[kTok];
#pragma unroll
    for (int i = 0; i < kTok; ++i) {
      if (on && i < n) {
        xw[i] = *reinterpret_cast<const Word<T, V> *>(x + (t0 + i) * a.xs[1]);
        gw[i] = *reinterpret_cast<const Word<T, V> *>(gate + (t0 + i) * a.gs[1]);
        yw[i] = *reinterpret_cast<const Word<T, V> *>(dout + (t0 + i) * a.os[1]);
      }
    }
    float in[V];
#pragma unroll
    for (int v = 0; v < V; ++v)
      in[v] = on && tile0 < a.L ? a.saved[((int64_t)b * tiles + tile0 / kTile) * a.D + c + v] : 0.f;
    float d[kTok][V];
    Map3 m[V];
    float dmax[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      m[v] = {0.f, 0.f, 0.f};
      dmax[v] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < kTok; ++i) {
      if (!(on && i < n)) {
        xw[i] = word_zero<T, V>();
        yw[i] = word_zero<T, V>();
      }
#pragma unroll
      for (int v = 0; v < V; ++v) {
        d[i][v] = on && i < n ? drop_of<T, MODE>(gw[i].get(v)) : 0.f;
        const float xv = xw[i].get(v), u = MODE == DP_SCAN_SIGMOID ? d[i][v] * xv : xv;
        m[v].H = fmaf(-d[i][v], m[v].H, m[v].H) + u;
        m[v].d = fmaf(-d[i][v], m[v].d, m[v].d) + d[i][v];
        dmax[v] = fmaxf(dmax[v], d[i][v]);
      }
    }
#pragma unroll
    for (int i = kTok - 1; i >= 0; --i)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float p = yw[i].get(v) + m[v].Q;
        m[v].Q = fmaf(-d[i][v], p, p);
      }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (dmax[v] == 1.f) m[v].d = 1.f;
      wmap[buf][warp][lane * V + v] = m[v];
    }
    __syncthreads();
    if (warp == 0) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        Map r = {0.f, 0.f};
        bool drop = false;
#pragma unroll
        for (int j = kWarps - 1; j >= 0; --j) {
          const Map3 w = wmap[buf][j][lane * V + v];
          r.H = apply({w.d, w.Q}, r.H);
          r.d = fmaf(-w.d, r.d, r.d) + w.d;
          drop |= w.d == 1.f;
        }
        if (drop) r.d = 1.f;
        if (a.cs > 1) {
          for (int k = 0; k < a.cs; ++k) cg::this_cluster().map_shared_rank(&bmap[buf][rank][lane * V + v], k)[0] = r;
        } else {
          bmap[buf][0][lane * V + v] = r;
        }
      }
    }
    scan_sync(a.cs);
    float qi[V];
#pragma unroll
    for (int v = 0; v < V; ++v) qi[v] = q[v];
    for (int k = a.cs - 1; k >= 0; --k)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (k == rank) qi[v] = q[v];
        q[v] = apply(bmap[buf][k][lane * V + v], q[v]);
      }
    for (int j = kWarps - 1; j > warp; --j)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const Map3 w = wmap[buf][j][lane * V + v];
        qi[v] = apply({w.d, w.Q}, qi[v]);
      }
    for (int j = 0; j < warp; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const Map3 w = wmap[buf][j][lane * V + v];
        in[v] = apply({w.d, w.H}, in[v]);
      }
    float hb[kTok][V];  // the state before each token
#pragma unroll
    for (int i = 0; i < kTok; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        hb[i][v] = in[v];
        const float xv = xw[i].get(v), u = MODE == DP_SCAN_SIGMOID ? d[i][v] * xv : xv;
        in[v] = fmaf(-d[i][v], in[v], in[v]) + u;
      }
#pragma unroll
    for (int i = kTok - 1; i >= 0; --i) {
      Word<T, V> ox, og;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float p = yw[i].get(v) + qi[v];
        qi[v] = fmaf(-d[i][v], p, p);
        if (MODE == DP_SCAN_SIGMOID) {
          ox.set(v, p * d[i][v]);
          og.set(v, qi[v] * d[i][v] * (hb[i][v] - xw[i].get(v)));
        } else {
          ox.set(v, p);
          og.set(v, qi[v] * hb[i][v]);
        }
      }
      if (on && i < n) {
        *reinterpret_cast<Word<T, V> *>(dx + (t0 + i) * a.D) = ox;
        *reinterpret_cast<Word<T, V> *>(dg + (t0 + i) * a.D) = og;
      }
    }
  }
  if (on && rank == 0 && warp == 0 && a.dh0)
#pragma unroll
    for (int v = 0; v < V; ++v) a.dh0[(int64_t)b * a.D + c + v] = q[v];
}

// ---------------------------------------------------------------- one token
template <typename T, int MODE>
__global__ void __launch_bounds__(256)
scan_step_kernel(const float *state, float *state_out, const T *x, const T *gate, T *out, int64_t xs, int64_t gs,
                 int64_t os, int64_t n, int D) {
  pdl_wait();
  pdl_trigger();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const int64_t b = i / D;
  const int c = (int)(i - b * D);
  const float d = drop_of<float, MODE>(to_f32(gate[b * gs + c])), xv = to_f32(x[b * xs + c]);
  const float h = state[i];
  const float r = fmaf(-d, h, h) + (MODE == DP_SCAN_SIGMOID ? d * xv : xv);
  state_out[i] = r;
  out[b * os + c] = from_f32<T>(r);
}

// Blocks of a cluster: as many tiles as the sequence has, up to 16.
int scan_cluster(int L) {
  int cs = 1;
  while (cs < kMaxCluster && cs * kTile < L) cs *= 2;
  return cs;
}

template <typename Kern>
int scan_launch(Kern kern, const ScanArgs &a, cudaStream_t st, const char *what) {
  if (a.cs > 8) {  // a non-portable size: opt in
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return set_error(DP_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((int64_t)a.B * a.tiles_c * a.cs));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.cs;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(DP_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
  }
  return check_launch(what);
}

// Channel pairs of 16-bit values can be moved as 4-byte words.
template <typename... P>
bool scan_pairs(int D, const int64_t *s, int ns, P... ptrs) {
  if (D % 2) return false;
  for (int i = 0; i < ns; ++i)
    if (s[i] % 2) return false;
  const void *ps[] = {ptrs...};
  for (const void *p : ps)
    if (reinterpret_cast<uintptr_t>(p) & 3) return false;
  return true;
}

template <bool BWD, typename T, int V>
int scan_run(ScanArgs a, int mode, cudaStream_t st, const char *what) {
  a.tiles_c = (a.D + 32 * V - 1) / (32 * V);
  a.cs = scan_cluster(a.L);
  DP_REQUIRE((int64_t)a.B * a.tiles_c * a.cs < (1ll << 31), DP_ERR_UNSUPPORTED,
             std::string(what) + ": too many channels");
  if constexpr (BWD)
    return mode == DP_SCAN_SIGMOID ? scan_launch(scan_bwd_kernel<T, V, DP_SCAN_SIGMOID>, a, st, what)
                                   : scan_launch(scan_bwd_kernel<T, V, DP_SCAN_DECAY>, a, st, what);
  else
    return mode == DP_SCAN_SIGMOID ? scan_launch(scan_fwd_kernel<T, V, DP_SCAN_SIGMOID>, a, st, what)
                                   : scan_launch(scan_fwd_kernel<T, V, DP_SCAN_DECAY>, a, st, what);
}

template <bool BWD>
int scan_dispatch(const ScanArgs &a, int dtype, int mode, bool pairs, cudaStream_t st, const char *what) {
  if (dtype == DP_F32) return scan_run<BWD, float, 1>(a, mode, st, what);
  if (dtype == DP_BF16)
    return pairs ? scan_run<BWD, __nv_bfloat16, 2>(a, mode, st, what) : scan_run<BWD, __nv_bfloat16, 1>(a, mode, st, what);
  return pairs ? scan_run<BWD, __half, 2>(a, mode, st, what) : scan_run<BWD, __half, 1>(a, mode, st, what);
}

}  // namespace
}  // namespace dp

extern "C" int dp_scan_tile(void) { return dp::kTile; }

extern "C" int dp_scan_fwd(const void *x, const void *gate, int dtype, int mode, const float *state_in, void *out,
                           float *state_out, float *saved, int B, int L, int D, const int64_t *strides, void *stream) {
  using namespace dp;
  DP_REQUIRE(B >= 0 && L >= 0 && D >= 1, DP_ERR_INVALID_ARGUMENT, "dp_scan_fwd: bad sizes");
  DP_REQUIRE(valid_dtype(dtype), DP_ERR_INVALID_ARGUMENT, "dp_scan_fwd: unknown dtype code");
  DP_REQUIRE(mode == DP_SCAN_DECAY || mode == DP_SCAN_SIGMOID, DP_ERR_INVALID_ARGUMENT, "dp_scan_fwd: unknown mode");
  if (B == 0) return DP_OK;
  DP_REQUIRE(state_out && strides && (L == 0 || (x && gate && out)), DP_ERR_INVALID_ARGUMENT,
             "dp_scan_fwd: null pointer");
  DP_REQUIRE(state_in != state_out, DP_ERR_INVALID_ARGUMENT, "dp_scan_fwd: state_out must not be state_in");
  cudaStream_t st = as_stream(stream);
  if (L == 0) {
    const size_t bytes = (size_t)B * D * sizeof(float);
    const cudaError_t e = state_in ? cudaMemcpyAsync(state_out, state_in, bytes, cudaMemcpyDeviceToDevice, st)
                                   : cudaMemsetAsync(state_out, 0, bytes, st);
    return e == cudaSuccess ? (int)DP_OK : set_error(DP_ERR_CUDA, std::string("dp_scan_fwd: ") + cudaGetErrorString(e));
  }
  ScanArgs a = {};
  a.x = x, a.gate = gate, a.h0 = state_in, a.hL = state_out, a.saved = saved, a.out = out;
  for (int i = 0; i < 2; ++i) a.xs[i] = strides[i], a.gs[i] = strides[2 + i], a.os[i] = strides[4 + i];
  a.B = B, a.L = L, a.D = D;
  return scan_dispatch<false>(a, dtype, mode, scan_pairs(D, strides, 6, x, gate, (const void *)out), st, "dp_scan_fwd");
}

extern "C" int dp_scan_bwd(const void *x, const void *gate, const void *grad_out, int dtype, int mode,
                           const float *saved, const float *grad_state_out, void *grad_x, void *grad_gate,
                           float *grad_state_in, int B, int L, int D, const int64_t *strides, void *stream) {
  using namespace dp;
  DP_REQUIRE(B >= 0 && L >= 0 && D >= 1, DP_ERR_INVALID_ARGUMENT, "dp_scan_bwd: bad sizes");
  DP_REQUIRE(valid_dtype(dtype), DP_ERR_INVALID_ARGUMENT, "dp_scan_bwd: unknown dtype code");
  DP_REQUIRE(mode == DP_SCAN_DECAY || mode == DP_SCAN_SIGMOID, DP_ERR_INVALID_ARGUMENT, "dp_scan_bwd: unknown mode");
  if (B == 0) return DP_OK;
  cudaStream_t st = as_stream(stream);
  if (L == 0) {
    if (!grad_state_in) return DP_OK;
    const size_t bytes = (size_t)B * D * sizeof(float);
    const cudaError_t e = grad_state_out
                              ? cudaMemcpyAsync(grad_state_in, grad_state_out, bytes, cudaMemcpyDeviceToDevice, st)
                              : cudaMemsetAsync(grad_state_in, 0, bytes, st);
    return e == cudaSuccess ? (int)DP_OK : set_error(DP_ERR_CUDA, std::string("dp_scan_bwd: ") + cudaGetErrorString(e));
  }
  DP_REQUIRE(x && gate && grad_out && saved && grad_x && grad_gate && strides, DP_ERR_INVALID_ARGUMENT,
             "dp_scan_bwd: null pointer");
  ScanArgs a = {};
  a.x = x, a.gate = gate, a.dout = grad_out, a.saved = const_cast<float *>(saved), a.dhL = grad_state_out;
  a.dx = grad_x, a.dgate = grad_gate, a.dh0 = grad_state_in;
  for (int i = 0; i < 2; ++i) a.xs[i] = strides[i], a.gs[i] = strides[2 + i], a.os[i] = strides[4 + i];
  a.B = B, a.L = L, a.D = D;
  return scan_dispatch<true>(a, dtype, mode,
                             scan_pairs(D, strides, 6, x, gate, grad_out, (const void *)grad_x, (const void *)grad_gate),
                             st, "dp_scan_bwd");
}

extern "C" int dp_scan_step(const float *state_in, float *state_out, const void *x, const void *gate, int dtype,
                            int mode, void *out, int B, int D, const int64_t *strides, void *stream) {
  using namespace dp;
  DP_REQUIRE(B >= 0 && D >= 1, DP_ERR_INVALID_ARGUMENT, "dp_scan_step: bad sizes");
  DP_REQUIRE(valid_dtype(dtype), DP_ERR_INVALID_ARGUMENT, "dp_scan_step: unknown dtype code");
  DP_REQUIRE(mode == DP_SCAN_DECAY || mode == DP_SCAN_SIGMOID, DP_ERR_INVALID_ARGUMENT, "dp_scan_step: unknown mode");
  if (B == 0) return DP_OK;
  DP_REQUIRE(state_in && state_out && x && gate && out && strides, DP_ERR_INVALID_ARGUMENT,
             "dp_scan_step: null pointer");
  const int64_t n = (int64_t)B * D, blocks = (n + 255) / 256;
  DP_REQUIRE(blocks < (1ll << 31), DP_ERR_UNSUPPORTED, "dp_scan_step: too many channels");
  return dispatch_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    auto kern = mode == DP_SCAN_SIGMOID ? scan_step_kernel<T, DP_SCAN_SIGMOID> : scan_step_kernel<T, DP_SCAN_DECAY>;
    return pdl_status(launch_pdl(kern, dim3((unsigned)blocks), dim3(256), 0, as_stream(stream), state_in, state_out,
                                 static_cast<const T *>(x), static_cast<const T *>(gate), static_cast<T *>(out),
                                 strides[0], strides[1], strides[2], n, D),
                      "scan_step_kernel");
  });
}
