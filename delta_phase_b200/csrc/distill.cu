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

constexpr int kDiVec = 8;            // 16-byte vectors of the row per thread
constexpr int kDiMaxThreads = 512;
constexpr int kDiMaxK = 1024;
constexpr int kDiMaxCluster = 16;
constexpr int kDiSms = 148;

struct DistillArgs {
  const void *z, *index, *teacher;
  const float *weight, *grad;
  float *loss;
  void *dz;
  int64_t sb, st;
  int index64, teacher_dt, L, V, K, cs;
  float tau;
};

__device__ __forceinline__ float di_warp_sum(float v) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}
__device__ __forceinline__ float di_warp_max(float v) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, m));
  return v;
}

// Two values reduced over the block at once (maxima or sums), through `slot`, which is used
// once per kernel.
template <bool MAX>
__device__ __forceinline__ float2 di_block_reduce(float2 v, float2 *slot) {
  v.x = MAX ? di_warp_max(v.x) : di_warp_sum(v.x);
  v.y = MAX ? di_warp_max(v.y) : di_warp_sum(v.y);
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (lane == 0) slot[threadIdx.x >> 5] = v;
  __syncthreads();
  const float none = MAX ? -INFINITY : 0.f;
  float2 t = lane < warps ? slot[lane] : make_float2(none, none);
  t.x = MAX ? di_warp_max(t.x) : di_warp_sum(t.x);
  t.y = MAX ? di_warp_max(t.y) : di_warp_sum(t.y);
  return t;
}

template <typename T>
__global__ void __launch_bounds__(kDiMaxThreads) distill_kernel(DistillArgs a) {
  constexpr int E = 16 / (int)sizeof(T);
  __shared__ float2 slot_max[kDiMaxThreads / 32], slot_sum[kDiMaxThreads / 32], slot_loss[kDiMaxThreads / 32];
  __shared__ float2 part[kDiMaxCluster];
  __shared__ float sp[kDiMaxK];
  __shared__ int si[kDiMaxK];
  const int tid = threadIdx.x, rank = blockIdx.x % a.cs;
  const int64_t row = blockIdx.x / a.cs;
  const float weight = a.weight ? a.weight[row] : 1.f, grad = a.grad ? a.grad[row] : 1.f;
  const T *z = static_cast<const T *>(a.z) + row / a.L * a.sb + row % a.L * a.st;
  T *dz = a.dz ? static_cast<T *>(a.dz) + row * a.V : nullptr;
  if (weight == 0.f) {  // a padding row: z is not looked at (the same for the whole cluster)
    if (a.loss && rank == 0 && tid == 0) a.loss[row] = 0.f;
    if (dz)
      for (int i = rank * blockDim.x + tid; i < a.V; i += a.cs * blockDim.x) dz[i] = from_f32<T>(0.f);
    return;
  }
  // The row as 16-byte aligned vectors: vector j holds elements j E - phase .. + E - 1.
  const int phase = (int)((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(T));
  const int nvec = (a.V + phase + E - 1) / E, per = (nvec + a.cs - 1) / a.cs;
  const int v0 = min(rank * per, nvec), v1 = min(v0 + per, nvec);
  if (a.cs > 1) cg::this_cluster().sync();  // every block of the cluster runs
  uint4 raw[kDiVec];
#pragma unroll
  for (int i = 0; i < kDiVec; ++i) {
    const int j = v0 + tid + i * blockDim.x, e0 = j * E - phase;
    T *r = reinterpret_cast<T *>(&raw[i]);
    if (j < v1 && e0 >= 0 && e0 + E <= a.V) {
      raw[i] = *reinterpret_cast<const uint4 *>(z + e0);
    } else {
#pragma unroll
      for (int k = 0; k < E; ++k)
        r[k] = j < v1 && e0 + k >= 0 && e0 + k < a.V ? z[e0 + k] : from_f32<T>(-INFINITY);
    }
  }
  // the teacher's entries: 1 / tau is applied after the maximum is taken off, so a masked
  // logit of the type's lowest value does not overflow
  const float inv_tau = 1.f / a.tau;
  float tmax = -INFINITY;
  for (int k = tid; k < a.K; k += blockDim.x) {
    const int64_t o = row * a.K + k;
    const int64_t i = a.index64 ? static_cast<const int64_t *>(a.index)[o] : static_cast<const int32_t *>(a.index)[o];
    const bool ok = i >= 0 && i < a.V;
    const float t = ok ? raw_scalar_to_f32(load_raw_scalar(a.teacher, a.teacher_dt, o), a.teacher_dt) : -INFINITY;
    si[k] = ok ? (int)i : -1;
    sp[k] = t;
    tmax = fmaxf(tmax, t);
  }
  float zmax = -INFINITY;
#pragma unroll
  for (int i = 0; i < kDiVec; ++i)
#pragma unroll
    for (int k = 0; k < E; ++k) zmax = fmaxf(zmax, to_f32(reinterpret_cast<const T *>(&raw[i])[k]));
  float2 m = di_block_reduce<true>(make_float2(zmax, tmax), slot_max);
  // a block (or a row's teacher) that is masked throughout: its sum is 0, not NaN
  const float m0 = m.x == -INFINITY ? 0.f : m.x, t0 = m.y == -INFINITY ? 0.f : m.y;
  float zsum = 0.f, tsum = 0.f;
#pragma unroll
  for (int i = 0; i < kDiVec; ++i)
#pragma unroll
    for (int k = 0; k < E; ++k)
      zsum += __expf((to_f32(reinterpret_cast<const T *>(&raw[i])[k]) - m0) * inv_tau);
  for (int k = tid; k < a.K; k += blockDim.x) {
    const float e = __expf((sp[k] - t0) * inv_tau);
    tsum += e;
  }
  const float2 s = di_block_reduce<false>(make_float2(zsum, tsum), slot_sum);
  float zm = m.x, S = s.x;
  if (a.cs > 1) {
    cg::cluster_group cl = cg::this_cluster();
    if (tid < a.cs) cl.map_shared_rank(part, tid)[rank] = make_float2(m.x, s.x);
    cl.sync();
    zm = -INFINITY;
    for (int r = 0; r < a.cs; ++r) zm = fmaxf(zm, part[r].x);
    S = 0.f;
    for (int r = 0; r < a.cs; ++r) S += part[r].y * __expf((part[r].x - zm) * inv_tau);
  }
  const bool empty = s.y == 0.f;
  // p_k, and the row's loss by the cluster's first block
  const float log_tsum = logf(s.y), log_S = logf(S);
  float l = 0.f;
  for (int k = tid; k < a.K; k += blockDim.x) {
    const float t = (sp[k] - t0) * inv_tau, p = __expf(t) / s.y;
    sp[k] = p;
    if (a.loss && rank == 0 && !empty && si[k] >= 0 && p != 0.f) {
      const float lq = (to_f32(z[si[k]]) - zm) * inv_tau - log_S;
      l = fmaf(p, t - log_tsum - lq, l);
    }
  }
  if (a.loss && rank == 0) {
    const float2 r = di_block_reduce<false>(make_float2(l, 0.f), slot_loss);
    if (tid == 0) a.loss[row] = empty ? 0.f : weight * a.tau * a.tau * r.x;
  }
  if (!dz) return;
  const bool zero = empty || grad == 0.f;
  const float cw = weight * a.tau * grad, scale = cw / S;
  // dz may lie differently against the 16-byte grid than z
  const bool vec = (reinterpret_cast<uintptr_t>(dz) & 15) == (reinterpret_cast<uintptr_t>(z) & 15);
#pragma unroll
  for (int i = 0; i < kDiVec; ++i) {
    const int j = v0 + tid + i * blockDim.x, e0 = j * E - phase;
    if (j >= v1) continue;
    uint4 o;
    T *w = reinterpret_cast<T *>(&o);
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const float q = __expf((to_f32(reinterpret_cast<const T *>(&raw[i])[k]) - zm) * inv_tau);
      w[k] = from_f32<T>(zero ? 0.f : q * scale);
    }
    if (vec && e0 >= 0 && e0 + E <= a.V) {
      *reinterpret_cast<uint4 *>(dz + e0) = o;
    } else {
#pragma unroll
      for (int k = 0; k < E; ++k)
        if (e0 + k >= 0 && e0 + k < a.V) dz[e0 + k] = w[k];
    }
  }
  if (zero) return;
  __syncthreads();  // p complete, the dense values written: now the teacher's entries
  for (int k = tid; k < a.K; k += blockDim.x) {
    const int i = si[k], j = (i + phase) / E;
    if (i < 0 || j < v0 || j >= v1) continue;
    // all entries of the same index, in their order: every one of them writes the same value
    float p = 0.f;
    for (int n = 0; n < a.K; ++n)
      if (si[n] == i) p += sp[n];
    const float q = __expf((to_f32(z[i]) - zm) * inv_tau) / S;
    dz[i] = from_f32<T>(cw * (q - p));
  }
}

template <typename T>
int distill_launch(DistillArgs a, int N, cudaStream_t st) {
  constexpr int E = 16 / (int)sizeof(T);
  const int nvec = (a.V + 2 * (E - 1)) / E;  // at the worst alignment
  const int most = kDiMaxThreads * kDiVec;
  int cs = 1;
  while (cs < kDiMaxCluster && (int64_t)cs * most < nvec) cs *= 2;
  DP_REQUIRE((int64_t)cs * most >= nvec, DP_ERR_UNSUPPORTED, "dp_distill: V too large");
  // few rows: split each over more blocks, down to a vector per thread
  while (cs < kDiMaxCluster && (int64_t)N * cs < 2 * kDiSms && nvec / cs >= 2 * kDiMaxThreads) cs *= 2;
  const int per = (nvec + cs - 1) / cs;
  int threads = 64;
  while (threads < kDiMaxThreads && threads * kDiVec < per) threads *= 2;
  while (threads < kDiMaxThreads && (int64_t)N * cs < 2 * kDiSms && threads < per) threads *= 2;
  a.cs = cs;
  if (cs > 8) {  // a non-portable size: opt in
    const cudaError_t e =
        cudaFuncSetAttribute(distill_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return set_error(DP_ERR_CUDA, std::string("dp_distill: ") + cudaGetErrorString(e));
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((int64_t)N * cs));
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cs;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, distill_kernel<T>, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(DP_ERR_CUDA, std::string("dp_distill: ") + cudaGetErrorString(e));
  }
  return check_launch("distill_kernel");
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
  a.teacher_dt = teacher_dtype, a.weight = weight, a.grad = grad, a.tau = tau, a.loss = loss, a.dz = dz;
  a.L = L, a.V = V, a.K = K;
  cudaStream_t st = as_stream(stream);
  return dispatch_dtype(z_dtype, [&](auto t) { return distill_launch<decltype(t)>(a, (int)rows, st); });
}
