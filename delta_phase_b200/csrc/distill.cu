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
__device__ __forceinline__ float di_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

// The threads that hold a row (or a block's slice of it): a warp, or the block.
template <bool WARP>
struct Group {
  static __device__ __forceinline__ int size() { return WARP ? 32 : (int)blockDim.x; }
  static __device__ __forceinline__ int rank() { return WARP ? threadIdx.x & 31 : (int)threadIdx.x; }
  static __device__ __forceinline__ void sync() {
    if (WARP)
      __syncwarp();
    else
      __syncthreads();
  }
  // Two values reduced at once (maxima or sums); `slot` is used once per kernel.
  template <bool MAX>
  static __device__ __forceinline__ float2 reduce(float2 v, float2 *slot) {
    v.x = MAX ? di_warp_max(v.x) : di_warp_sum(v.x);
    v.y = MAX ? di_warp_max(v.y) : di_warp_sum(v.y);
    if (WARP) {
      __syncwarp();  // like the block's barriers: what was written to shared memory before is seen after
      return v;
    }
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) slot[threadIdx.x >> 5] = v;
    __syncthreads();
    const float none = MAX ? -INFINITY : 0.f;
    v = lane < warps ? slot[lane] : make_float2(none, none);
    v.x = MAX ? di_warp_max(v.x) : di_warp_sum(v.x);
    v.y = MAX ? di_warp_max(v.y) : di_warp_sum(v.y);
    return v;
  }
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

// Shared memory of one group: the teacher's entries (index, p, the student's logit there) and
// two bits per element of the group's slice (an entry names it; more than one does).
__host__ __device__ inline int di_bits_words(int slice_elems) { return (slice_elems + 31) / 32; }
inline int di_smem(int K, int slice_elems) { return 12 * K + 8 * di_bits_words(slice_elems); }

// NV vectors per thread; WARP: a warp holds a row, kDiWarpRows rows a block; else a block (or
// a cluster of a.cs blocks) holds a row.
template <typename T, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? 32 * kDiWarpRows : kDiMaxThreads, WARP ? 6 : 2)
distill_kernel(const DistillArgs a) {
  using G = Group<WARP>;
  using W = Vec<T>;
  constexpr int E = W::E;
  __shared__ float2 slots[3][kDiMaxThreads / 32];
  __shared__ float2 part[kDiMaxCluster];
  extern __shared__ __align__(16) unsigned char dyn[];
  const int tid = G::rank(), n = G::size(), cs = WARP ? 1 : a.cs, rank = WARP ? 0 : blockIdx.x % cs;
  const int64_t row = WARP ? (int64_t)blockIdx.x * kDiWarpRows + (threadIdx.x >> 5) : blockIdx.x / cs;
  if (WARP && row >= a.rows) return;  // whole warps
  const float weight = a.weight ? a.weight[row] : 1.f, grad = a.grad ? a.grad[row] : 1.f;
  const T *z = static_cast<const T *>(a.z) + row / a.L * a.sb + row % a.L * a.st;
  T *dz = a.dz ? static_cast<T *>(a.dz) + row * a.V : nullptr;
  // The row as 16-byte aligned vectors: vector j holds elements j E - phase .. + E - 1.
  const int phase = (int)((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(T));
  const int nvec = (a.V + phase + E - 1) / E, per = (nvec + cs - 1) / cs;
  const int v0 = min(rank * per, nvec), v1 = min(v0 + per, nvec);
  if (weight == 0.f) {  // a padding row: z is not looked at (the same for the whole cluster)
    if (a.loss && rank == 0 && tid == 0) a.loss[row] = 0.f;
    if (dz) {
      const bool vec = (reinterpret_cast<uintptr_t>(dz) & 15) == (reinterpret_cast<uintptr_t>(z) & 15);
      for (int j = v0 + tid; j < v1; j += n) {
        const int e0 = j * E - phase;
        if (vec && e0 >= 0 && e0 + E <= a.V) {
          *reinterpret_cast<uint4 *>(dz + e0) = make_uint4(0, 0, 0, 0);
        } else {
          for (int k = max(e0, 0); k < min(e0 + E, a.V); ++k) dz[k] = from_f32<T>(0.f);
        }
      }
    }
    return;
  }
  if (cs > 1) cg::this_cluster().sync();  // every block of the cluster runs
  uint4 raw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = v0 + tid + i * n, e0 = j * E - phase;
    if (j < v1 && e0 >= 0 && e0 + E <= a.V) {
      raw[i] = *reinterpret_cast<const uint4 *>(z + e0);
    } else {
#pragma unroll
      for (int k = 0; k < E / 2; ++k) {
        const int e = e0 + 2 * k;
        const bool lo = j < v1 && e >= 0 && e < a.V, hi = j < v1 && e + 1 >= 0 && e + 1 < a.V;
        W::set(raw[i], k, make_float2(lo ? to_f32(z[e]) : -INFINITY, hi ? to_f32(z[e + 1]) : -INFINITY));
      }
    }
  }
  // the teacher's entries, and the student's logits there
  const int slice = per * E, words = di_bits_words(slice);
  unsigned char *mine = dyn + (WARP ? (threadIdx.x >> 5) * a.group_smem : 0);
  int *si = reinterpret_cast<int *>(mine);
  float *sp = reinterpret_cast<float *>(si + a.K), *sz = sp + a.K;
  uint32_t *once = reinterpret_cast<uint32_t *>(sz + a.K), *again = once + words;
  float tmax = -INFINITY;
  for (int k = tid; k < a.K; k += n) {
    const int64_t o = row * a.K + k;
    const int64_t i = a.index64 ? static_cast<const int64_t *>(a.index)[o] : static_cast<const int32_t *>(a.index)[o];
    const bool ok = i >= 0 && i < a.V;
    const float t = ok ? raw_scalar_to_f32(load_raw_scalar(a.teacher, a.teacher_dt, o), a.teacher_dt) : -INFINITY;
    si[k] = ok ? (int)i : -1;
    sp[k] = t;
    sz[k] = ok ? to_f32(z[i]) : 0.f;
    tmax = fmaxf(tmax, t);
  }
  if (dz)
    for (int k = tid; k < 2 * words; k += n) once[k] = 0;
  float zmax = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i) zmax = W::max(raw[i], zmax);
  const float2 m = G::template reduce<true>(make_float2(zmax, tmax), slots[0]);
  // Exponents: the maximum is taken off before the factor log2(e) / tau is applied, so masked
  // logits of the type's lowest value do not overflow; a slice (or a row's teacher) that is
  // masked throughout has the sum 0, not NaN.
  const float c = 1.4426950408889634f / a.tau, inv_tau = 1.f / a.tau;
  const float m0 = m.x == -INFINITY ? 0.f : m.x, t0 = m.y == -INFINITY ? 0.f : m.y;
  const float2 c2 = make_float2(c, c);
  float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
  {
    const float2 off = make_float2(-m0, -m0);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < E / 2; ++k) {
        const float2 x = __fmul2_rn(__fadd2_rn(W::pair(raw[i], k), off), c2);
        acc[k & 1] = __fadd2_rn(acc[k & 1], make_float2(di_ex2(x.x), di_ex2(x.y)));
      }
  }
  float tsum = 0.f;
  for (int k = tid; k < a.K; k += n) {
    tsum += di_ex2((sp[k] - t0) * c);
    if (dz && si[k] >= 0) {
      const int e = si[k] + phase - v0 * E;
      if (e >= 0 && e < slice) {
        const uint32_t bit = 1u << (e & 31);
        if (atomicOr(&once[e >> 5], bit) & bit) atomicOr(&again[e >> 5], bit);
      }
    }
  }
  const float2 s = G::template reduce<false>(make_float2((acc[0].x + acc[0].y) + (acc[1].x + acc[1].y), tsum), slots[1]);
  float zm = m.x, S = s.x;
  if (cs > 1) {
    cg::cluster_group cl = cg::this_cluster();
    if (tid < cs) cl.map_shared_rank(part, tid)[rank] = make_float2(m.x, s.x);
    cl.sync();
    zm = -INFINITY;
    for (int r = 0; r < cs; ++r) zm = fmaxf(zm, part[r].x);
    S = 0.f;
    for (int r = 0; r < cs; ++r) S += part[r].y * di_ex2((part[r].x - zm) * c);
  }
  const bool empty = s.y == 0.f;
  // p_k, and the row's loss by the cluster's first block
  const bool loss = a.loss && rank == 0;
  const float log_tsum = logf(s.y), log_S = logf(S), inv_tsum = 1.f / s.y;
  float l = 0.f;
  for (int k = tid; k < a.K; k += n) {
    const float t = sp[k] - t0, p = di_ex2(t * c) * inv_tsum;
    sp[k] = p;
    if (loss && p != 0.f && si[k] >= 0)
      l = fmaf(p, t * inv_tau - log_tsum - ((sz[k] - zm) * inv_tau - log_S), l);
  }
  if (loss) {
    const float2 r = G::template reduce<false>(make_float2(l, 0.f), slots[2]);
    if (tid == 0) a.loss[row] = empty ? 0.f : weight * a.tau * a.tau * r.x;
  }
  if (!dz) return;
  const bool zero = empty || grad == 0.f;
  const float cw = weight * a.tau * grad, scale = zero ? 0.f : cw / S;
  // dz may lie differently against the 16-byte grid than z
  const bool vec = (reinterpret_cast<uintptr_t>(dz) & 15) == (reinterpret_cast<uintptr_t>(z) & 15);
  const float2 off = make_float2(-zm, -zm), scale2 = make_float2(scale, scale);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = v0 + tid + i * n, e0 = j * E - phase;
    if (j >= v1) continue;
    uint4 o;
#pragma unroll
    for (int k = 0; k < E / 2; ++k) {
      const float2 x = __fmul2_rn(__fadd2_rn(W::pair(raw[i], k), off), c2);
      W::set(o, k, __fmul2_rn(make_float2(di_ex2(x.x), di_ex2(x.y)), scale2));
    }
    if (zero) o = make_uint4(0, 0, 0, 0);
    if (vec && e0 >= 0 && e0 + E <= a.V) {
      *reinterpret_cast<uint4 *>(dz + e0) = o;
    } else {
      const T *w = reinterpret_cast<const T *>(&o);
#pragma unroll
      for (int k = 0; k < E; ++k)
        if (e0 + k >= 0 && e0 + k < a.V) dz[e0 + k] = w[k];
    }
  }
  if (zero) return;
  G::sync();  // every p is there and the dense values are written: now the teacher's entries
  const float inv_S = 1.f / S;
  const int lane = threadIdx.x & 31;
  for (int k0 = tid - lane; k0 < a.K; k0 += n) {  // whole warps
    const int k = k0 + lane, i = k < a.K ? si[k] : -1, e = i + phase - v0 * E;
    const bool here = i >= 0 && e >= 0 && e < slice;
    float p = here ? sp[k] : 0.f;
    // an index that occurs more than once: the warp adds up all its entries, in a fixed order,
    // so each of them writes the same value
    uint32_t more = __ballot_sync(0xffffffffu, here && (again[e >> 5] >> (e & 31) & 1));
    while (more) {
      const int src = __ffs(more) - 1, at = __shfl_sync(0xffffffffu, i, src);
      more &= more - 1;
      float t = 0.f;
      for (int q = lane; q < a.K; q += 32)
        if (si[q] == at) t += sp[q];
      t = di_warp_sum(t);
      if (lane == src) p = t;
    }
    if (here) dz[i] = from_f32<T>(cw * (di_ex2((sz[k] - zm) * c) * inv_S - p));
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
  const int64_t size = sizeof(T);
  // vectors of a row, with up to one more where rows do not start on 16 bytes
  const bool aligned = reinterpret_cast<uintptr_t>(a.z) % 16 == 0 && a.sb * size % 16 == 0 && a.st * size % 16 == 0;
  const int nvec = aligned ? (a.V + E - 1) / E : (a.V + 2 * (E - 1)) / E;
  a.cs = 1;
  if (nvec <= 32 * kDiMaxVec) {
    const int64_t blocks = (a.rows + kDiWarpRows - 1) / kDiWarpRows;
    a.group_smem = di_smem(a.K, nvec * E);
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
  const size_t smem = a.group_smem = di_smem(a.K, per * E);
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
  a.teacher_dt = teacher_dtype, a.weight = weight, a.grad = grad, a.tau = tau, a.loss = loss, a.dz = dz;
  a.rows = rows, a.L = L, a.V = V, a.K = K;
  cudaStream_t st = as_stream(stream);
  return dispatch_dtype(z_dtype, [&](auto t) { return distill_launch<decltype(t)>(a, st); });
}
