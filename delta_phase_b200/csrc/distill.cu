// Distillation from a teacher's top logits: per row, with p = softmax(teacher / tau) over
// the K entries and q = softmax(z / tau) over the V logits of the student,
//   loss = weight tau^2 sum_k p_k (log p_k - log q_{i_k})
//   dz_v = grad weight tau (q_v - sum_{k: i_k = v} p_k)
// for the head of DeltaPhaseModel (delta_phase/model.py:60-66, 101).
//
// The logits are by far the largest tensors of a training step and HBM bounds the pass:
// a row is read once into the registers of a block (or of a cluster of blocks, for wide
// rows and for few rows), its maximum and sum of exponentials are reduced there, and the
// gradient is written from the same registers, so loss and gradient together move 2 V
// values a row.  Statistics and products are float32; the gradient is rounded once.
#include <cooperative_groups.h>

#include <algorithm>
#include <string>

#include "dp_common.cuh"

namespace cg = cooperative_groups;

namespace dp {
namespace {

constexpr int kDiMaxVec = 8;      // 16-byte vectors of a row per thread, at most
constexpr int kDiMaxThreads = 512;
constexpr int kDiMaxK = 1024;
constexpr int kDiMaxCluster = 16;
constexpr int kDiSms = 148;
constexpr int kDiWarpRows = 4;    // rows of a block where a warp holds a row

struct DistillArgs {
  const void *z, *index, *teacher;
  const float *weight, *grad;
  float *loss;
  void *dz;
  int64_t rows, sb, st;
  int index64, teacher_dt, L, V, K, cs;
  int group_smem;  // bytes of shared memory of a group
  float tau, inv_tau, c;  // c = log2(e) / tau
};

__device__ __forceinline__ float di_warp_sum(float v) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}
__device__ __forceinline__ float di_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float di_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float di_warp_redux_max(float v) {  // NaN is passed over
  float m;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;\n" : "=f"(m) : "f"(v));
  return m;
}

// What a warp knows of its part of the row: the maximum m of its logits, s = sum 2^((z - m) c)
// with c = log2(e) / tau; the maximum tm of its teacher entries, ts = sum 2^((t - tm) c), and
// d = sum 2^((t - tm) c) ((t - tm) - (z_index - m)), from which the loss follows.
struct Part {
  float m, s, tm, ts, d;
};

// A 16-byte vector of the row as pairs of float32, and back.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int E = 4;
  static __device__ __forceinline__ float2 pair(const uint4 &v, int i) {
    return i == 0 ? make_float2(__uint_as_float(v.x), __uint_as_float(v.y))
                  : make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
  }
  static __device__ __forceinline__ void set(uint4 &v, int i, float2 f) {
    (i == 0 ? v.x : v.z) = __float_as_uint(f.x);
    (i == 0 ? v.y : v.w) = __float_as_uint(f.y);
  }
  static __device__ __forceinline__ float max(const uint4 &v, float m) {
    return fmaxf(fmaxf(m, fmaxf(__uint_as_float(v.x), __uint_as_float(v.y))),
                 fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
};
__device__ __forceinline__ uint32_t &di_word(uint4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
__device__ __forceinline__ uint32_t di_word(const uint4 &v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int E = 8;
  static __device__ __forceinline__ float2 pair(const uint4 &v, int i) {
    const uint32_t w = di_word(v, i);
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ void set(uint4 &v, int i, float2 f) {
    const __nv_bfloat162 h = __float22bfloat162_rn(f);
    di_word(v, i) = *reinterpret_cast<const uint32_t *>(&h);
  }
  static __device__ __forceinline__ float max(const uint4 &v, float m) {
    const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&v);
    const float2 f = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(m, fmaxf(f.x, f.y));
  }
};
template <>
struct Vec<__half> {
  static constexpr int E = 8;
  static __device__ __forceinline__ float2 pair(const uint4 &v, int i) {
    const uint32_t w = di_word(v, i);
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
  }
  static __device__ __forceinline__ void set(uint4 &v, int i, float2 f) {
    const __half2 h = __float22half2_rn(f);
    di_word(v, i) = *reinterpret_cast<const uint32_t *>(&h);
  }
  static __device__ __forceinline__ float max(const uint4 &v, float m) {
    const __half2 *h = reinterpret_cast<const __half2 *>(&v);
    const float2 f = __half22float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(m, fmaxf(f.x, f.y));
  }
};

// Shared memory of one group: the teacher's entries (index, logit, the student's logit there)
// and two bit maps over hashed indices: an entry is there; more than one is (or two indices
// meet, which costs time only).  32 K bits and more: few indices meet.
__host__ __device__ inline int di_map_words(int K) {
  int w = 8;
  while (w < K) w *= 2;
  return w;
}
inline int di_smem(int K) { return 12 * K + 8 * di_map_words(K); }

// NV vectors per thread; WARP: a warp holds a row, kDiWarpRows rows a block; else a block (or
// a cluster of a.cs blocks) holds a row.
template <typename T, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? 32 * kDiWarpRows : kDiMaxThreads, WARP ? 6 : 2)
distill_kernel(const DistillArgs a) {
  using W = Vec<T>;
  constexpr int E = W::E;
  __shared__ Part parts[kDiMaxThreads / 32];
  __shared__ float2 cpart[kDiMaxCluster];
  extern __shared__ __align__(16) unsigned char dyn[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tid = WARP ? lane : (int)threadIdx.x, n = WARP ? 32 : (int)blockDim.x;
  const int cs = WARP ? 1 : a.cs, rank = WARP ? 0 : blockIdx.x % cs;
  const unsigned row = WARP ? blockIdx.x * kDiWarpRows + warp : blockIdx.x / cs;
  if (WARP && row >= a.rows) return;  // whole warps
  const float weight = a.weight ? a.weight[row] : 1.f, grad = a.grad ? a.grad[row] : 1.f;
  const unsigned batch = row / a.L;
  const T *z = static_cast<const T *>(a.z) + batch * a.sb + (row - batch * a.L) * a.st;
  T *dz = a.dz ? static_cast<T *>(a.dz) + (int64_t)row * a.V : nullptr;
  // The row: 16-byte aligned vectors from element `head` on, split over the cluster, and fewer
  // than 2 E single elements before and behind them, one each for the first block's threads.
  const int phase = (int)((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(T));
  const int head = min(phase ? E - phase : 0, a.V), nvec = (a.V - head) / E, tail = head + nvec * E;
  const int per = (nvec + cs - 1) / cs, v0 = min(rank * per, nvec), cnt = min(per, nvec - v0);
  const int edge = rank ? a.V : tid < head ? tid : tail + tid - head;  // this thread's; none: V and on
  const uint4 *zv = reinterpret_cast<const uint4 *>(z + head) + v0;
  // dz may lie differently against the 16-byte grid than z
  const bool vec = (reinterpret_cast<uintptr_t>(dz) & 15) == (reinterpret_cast<uintptr_t>(z) & 15);
  auto write_zeros = [&] {
    for (int j = tid; j < cnt; j += n) {
      T *p = dz + head + (v0 + j) * E;
      if (vec)
        *reinterpret_cast<uint4 *>(p) = make_uint4(0, 0, 0, 0);
      else
        for (int k = 0; k < E; ++k) p[k] = from_f32<T>(0.f);
    }
    if (edge < a.V) dz[edge] = from_f32<T>(0.f);
  };
  if (weight == 0.f) {  // a padding row: z is not looked at (the same for the whole cluster)
    if (a.loss && rank == 0 && tid == 0) a.loss[row] = 0.f;
    if (dz) write_zeros();
    return;
  }
  if (cs > 1) cg::this_cluster().sync();  // every block of the cluster runs
  uint4 raw[NV];
  if (cnt == NV * n) {
#pragma unroll
    for (int i = 0; i < NV; ++i) raw[i] = zv[tid + i * n];
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int k = 0; k < E / 2; ++k) W::set(raw[i], k, make_float2(-INFINITY, -INFINITY));
      if (tid + i * n < cnt) raw[i] = zv[tid + i * n];
    }
  }
  const float ze = edge < a.V ? to_f32(z[edge]) : -INFINITY;
  // the teacher's entries, and the student's logits there
  int *si = reinterpret_cast<int *>(dyn + (WARP ? warp * a.group_smem : 0));
  float *st = reinterpret_cast<float *>(si + a.K), *sz = st + a.K;
  const int words = di_map_words(a.K);
  uint32_t *once = reinterpret_cast<uint32_t *>(sz + a.K), *again = once + words;
  float tm = -INFINITY;
  for (int k = tid; k < a.K; k += n) {
    const int64_t o = (int64_t)row * a.K + k;
    const int64_t i = a.index64 ? static_cast<const int64_t *>(a.index)[o] : static_cast<const int32_t *>(a.index)[o];
    const bool ok = i >= 0 && i < a.V;
    const float t = ok ? raw_scalar_to_f32(load_raw_scalar(a.teacher, a.teacher_dt, o), a.teacher_dt) : -INFINITY;
    si[k] = ok ? (int)i : -1;
    st[k] = t;
    sz[k] = ok ? to_f32(z[i]) : 0.f;
    tm = fmaxf(tm, t);
  }
  if (dz)
    for (int k = tid; k < 2 * words; k += n) once[k] = 0;
  // Exponents: the maximum is taken off before the factor is applied, so masked logits of the
  // type's lowest value do not overflow; what is masked throughout has the sum 0, not NaN.
  const float c = a.c;
  const float2 c2 = make_float2(c, c);
  Part w;
  w.m = ze;
#pragma unroll
  for (int i = 0; i < NV; ++i) w.m = W::max(raw[i], w.m);
  w.m = di_warp_redux_max(w.m);
  const float m0 = w.m == -INFINITY ? 0.f : w.m;
  {
    float2 acc[2] = {make_float2(di_ex2((ze - m0) * c), 0.f), make_float2(0.f, 0.f)};
    const float2 off = make_float2(-m0, -m0);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < E / 2; ++k) {
        const float2 x = __fmul2_rn(__fadd2_rn(W::pair(raw[i], k), off), c2);
        acc[k & 1] = __fadd2_rn(acc[k & 1], make_float2(di_ex2(x.x), di_ex2(x.y)));
      }
    acc[0] = __fadd2_rn(acc[0], acc[1]);
    w.s = di_warp_sum(acc[0].x + acc[0].y);
  }
  w.tm = -INFINITY, w.ts = w.d = 0.f;
  if (tid - lane < a.K) {  // a warp that has entries
    w.tm = di_warp_redux_max(tm);
    const float t0 = w.tm == -INFINITY ? 0.f : w.tm;
    for (int k = tid; k < a.K; k += n) {
      const float t = st[k] - t0, e = di_ex2(t * c);
      w.ts += e;
      if (e != 0.f && si[k] >= 0) w.d = fmaf(e, t - (sz[k] - m0), w.d);
    }
    w.ts = di_warp_sum(w.ts);
    w.d = di_warp_sum(w.d);
  }
  // the parts of all warps: maxima, then sums relative to them
  float M = w.m, S = w.s, TM = w.tm, TS = w.ts, D = w.d;
  const int warps = blockDim.x >> 5;
  if (WARP) {
    __syncwarp();  // the entries and the cleared maps are seen by all lanes
  } else {
    if (lane == 0) parts[warp] = w;
    __syncthreads();
    Part q = {-INFINITY, 0.f, -INFINITY, 0.f, 0.f};
    if (lane < warps) q = parts[lane];
    M = di_warp_redux_max(q.m);
    TM = di_warp_redux_max(q.tm);
    S = di_warp_sum(q.m == -INFINITY ? q.s : q.s * di_ex2((q.m - M) * c));
    const float f = q.tm == -INFINITY ? 1.f : di_ex2((q.tm - TM) * c);
    TS = di_warp_sum(q.ts * f);
    // d against the common maxima (a part without entries has ts = d = 0)
    if (q.ts != 0.f) q.d = f * fmaf(q.ts, (q.tm - TM) - ((q.m == -INFINITY ? 0.f : q.m) - (M == -INFINITY ? 0.f : M)), q.d);
    D = di_warp_sum(q.d);
  }
  // the entries' bits (their maps were cleared before the barrier)
  if (dz)
    for (int k = tid; k < a.K; k += n)
      if (si[k] >= 0) {
        const uint32_t bit = 1u << (si[k] & 31);
        uint32_t *word = &once[si[k] >> 5 & (words - 1)];
        if (atomicOr(word, bit) & bit) atomicOr(word + words, bit);
      }
  const float M0 = M;
  if (cs > 1) {
    cg::cluster_group cl = cg::this_cluster();
    if (tid < cs) cl.map_shared_rank(cpart, tid)[rank] = make_float2(M, S);
    cl.sync();
    for (int r = 0; r < cs; ++r) M = fmaxf(M, cpart[r].x);
    S = 0.f;
    for (int r = 0; r < cs; ++r)
      S += cpart[r].x == -INFINITY ? cpart[r].y : cpart[r].y * di_ex2((cpart[r].x - M) * c);
  }
  // masked throughout (or NaN throughout): 0 / 0
  if (M == -INFINITY) S = NAN;
  const bool empty = TS == 0.f;
  if (a.loss && rank == 0 && tid == 0) {
    // sum p (log p - log q) = sum p ((t - TM) - (z - M)) / tau - log TS + log S
    const float d = D / TS - ((M0 == -INFINITY ? 0.f : M0) - M);
    a.loss[row] = empty ? 0.f : weight * a.tau * a.tau * (d * a.inv_tau + (logf(S) - logf(TS)));
  }
  if (!dz) return;
  if (empty || grad == 0.f) {
    write_zeros();
    return;
  }
  const float cw = weight * a.tau * grad, inv_S = di_rcp(S), scale = cw * inv_S;
  const float2 off = make_float2(-M, -M), scale2 = make_float2(scale, scale);
  T *pd = dz + head + (v0 + tid) * E;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    uint4 o;
#pragma unroll
    for (int k = 0; k < E / 2; ++k) {
      const float2 x = __fmul2_rn(__fadd2_rn(W::pair(raw[i], k), off), c2);
      W::set(o, k, __fmul2_rn(make_float2(di_ex2(x.x), di_ex2(x.y)), scale2));
    }
    if (tid + i * n < cnt) {
      T *p = pd + i * n * E;
      if (vec) {
        *reinterpret_cast<uint4 *>(p) = o;
      } else {
        const T *e = reinterpret_cast<const T *>(&o);
#pragma unroll
        for (int k = 0; k < E; ++k) p[k] = e[k];
      }
    }
  }
  if (edge < a.V) dz[edge] = from_f32<T>(di_ex2((ze - M) * c) * scale);
  if (WARP)
    __syncwarp();
  else
    __syncthreads();  // the dense values are written and the maps complete: now the teacher's entries
  const float inv_TS = di_rcp(TS);
  for (int k0 = tid - lane; k0 < a.K; k0 += n) {  // whole warps
    const int k = k0 + lane, i = k < a.K ? si[k] : -1;
    // this block's elements (vectors, and the single ones for the first)
    const bool here = i >= 0 && (i < head || i >= tail ? rank == 0 : i >= head + v0 * E && i < head + (v0 + cnt) * E);
    float p = here ? di_ex2((st[k] - TM) * c) * inv_TS : 0.f;
    // an index that occurs more than once: the warp adds up all its entries, in a fixed order,
    // so each of them writes the same value
    uint32_t more = __ballot_sync(0xffffffffu, here && (again[i >> 5 & (words - 1)] >> (i & 31) & 1));
    while (more) {
      const int src = __ffs(more) - 1, at = __shfl_sync(0xffffffffu, i, src);
      more &= more - 1;
      float t = 0.f;
      for (int q = lane; q < a.K; q += 32)
        if (si[q] == at) t += di_ex2((st[q] - TM) * c) * inv_TS;
      t = di_warp_sum(t);
      if (lane == src) p = t;
    }
    if (here) dz[i] = from_f32<T>(cw * (di_ex2((sz[k] - M) * c) * inv_S - p));
  }
}

template <typename T, int NV, bool WARP>
int distill_run(const DistillArgs &a, int64_t blocks, int threads, size_t smem, cudaStream_t st) {
  auto kern = distill_kernel<T, NV, WARP>;
  cudaError_t e = cudaSuccess;
  if (smem > 40 * 1024)  // beside the static part
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e == cudaSuccess && a.cs > 8)  // a non-portable size: opt in
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = a.cs;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.cs > 1 ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, kern, a);
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(DP_ERR_CUDA, std::string("dp_distill: ") + cudaGetErrorString(e));
  }
  return check_launch("distill_kernel");
}

template <typename T>
int distill_launch(DistillArgs a, cudaStream_t st) {
  constexpr int E = Vec<T>::E;
  const int nvec = a.V / E;  // at most: fewer where a row does not start on 16 bytes
  a.cs = 1;
  if (nvec <= 32 * kDiMaxVec) {
    const int64_t blocks = (a.rows + kDiWarpRows - 1) / kDiWarpRows;
    a.group_smem = di_smem(a.K);
    const size_t smem = (size_t)a.group_smem * kDiWarpRows;
    if (nvec <= 64) return distill_run<T, 2, true>(a, blocks, 32 * kDiWarpRows, smem, st);
    return distill_run<T, kDiMaxVec, true>(a, blocks, 32 * kDiWarpRows, smem, st);
  }
  const int most = kDiMaxThreads * kDiMaxVec;
  while (a.cs < kDiMaxCluster && (int64_t)a.cs * most < nvec) a.cs *= 2;
  DP_REQUIRE((int64_t)a.cs * most >= nvec, DP_ERR_UNSUPPORTED, "dp_distill: V too large");
  // few rows: split each over more blocks, down to a vector per thread
  while (a.cs < kDiMaxCluster && a.rows * a.cs < kDiSms && nvec / a.cs >= 2 * kDiMaxThreads) a.cs *= 2;
  const int per = (nvec + a.cs - 1) / a.cs;
  const int64_t blocks = a.rows * a.cs;
  const int nv = blocks >= 2 * kDiSms ? kDiMaxVec : per > 4 * kDiMaxThreads ? kDiMaxVec : per > kDiMaxThreads ? 4 : 1;
  const int threads = std::max(64, ((per + nv - 1) / nv + 31) / 32 * 32);
  const size_t smem = a.group_smem = di_smem(a.K);
  if (nv == 1) return distill_run<T, 1, false>(a, blocks, threads, smem, st);
  if (nv == 4) return distill_run<T, 4, false>(a, blocks, threads, smem, st);
  return distill_run<T, kDiMaxVec, false>(a, blocks, threads, smem, st);
}

}  // namespace
}  // namespace dp

extern "C" int dp_distill(const void *z, int z_dtype, const void *index, int index_bytes, const void *teacher,
                          int teacher_dtype, const float *weight, const float *grad, float tau, float *loss, void *dz,
                          int B, int L, int V, int K, const int64_t *strides, void *stream) {
  using namespace dp;
  DP_REQUIRE(B >= 0 && L >= 0 && V >= 1 && K >= 1, DP_ERR_INVALID_ARGUMENT, "dp_distill: bad sizes");
  DP_REQUIRE(valid_dtype(z_dtype) && valid_dtype(teacher_dtype), DP_ERR_INVALID_ARGUMENT,
             "dp_distill: unknown dtype code");
  DP_REQUIRE(index_bytes == 4 || index_bytes == 8, DP_ERR_INVALID_ARGUMENT, "dp_distill: index must be int32 or int64");
  DP_REQUIRE(tau > 1e-30f && tau < 1e30f, DP_ERR_INVALID_ARGUMENT, "dp_distill: tau must be positive and finite");
  DP_REQUIRE(K <= kDiMaxK, DP_ERR_UNSUPPORTED, "dp_distill: K must be <= 1024");
  DP_REQUIRE((int64_t)V * (int64_t)dtype_size(z_dtype) <= (1 << 20) - 32, DP_ERR_UNSUPPORTED,
             "dp_distill: a row of z must be smaller than 1 MiB");
  if (B == 0 || L == 0) return DP_OK;
  DP_REQUIRE(z && index && teacher && strides && (loss || dz), DP_ERR_INVALID_ARGUMENT, "dp_distill: null pointer");
  DP_REQUIRE(z != dz, DP_ERR_INVALID_ARGUMENT, "dp_distill: dz must not be z");
  const int64_t rows = (int64_t)B * L;
  DP_REQUIRE(rows * kDiMaxCluster < (1ll << 31), DP_ERR_UNSUPPORTED, "dp_distill: too many rows");
  DistillArgs a = {};
  a.z = z, a.sb = strides[0], a.st = strides[1], a.index = index, a.index64 = index_bytes == 8, a.teacher = teacher;
  a.teacher_dt = teacher_dtype, a.weight = weight, a.grad = grad, a.tau = tau, a.inv_tau = 1.f / tau, a.c = 1.4426950408889634f / tau, a.loss = loss, a.dz = dz;
  a.rows = rows, a.L = L, a.V = V, a.K = K;
  cudaStream_t st = as_stream(stream);
  return dispatch_dtype(z_dtype, [&](auto t) { return distill_launch<decltype(t)>(a, st); });
}
