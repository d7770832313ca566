// Distillation from a teacher's top logits: per row, with p = softmax(teacher / tau) over
// the K entries and q = softmax(z / tau) over the V logits of the student,
//   loss = weight tau^2 sum_k p_k (log p_k - log q_{i_k})
//   dz_v = grad weight tau (q_v - sum_{k: i_k = v} p_k)
// for the head of DeltaPhaseModel (delta_phase/model.py:60-66, 101).
//
// The logits are by far the largest tensors of a training step, and HBM bounds every pass.
//   loss and gradient at once: a row (a block's slice of it, for rows above 64 KB and for few
//     rows; the slices meet in one exchange over distributed shared memory) is read once, into
//     shared memory; its maximum, its sum of exponentials and the gradient come from there, so
//     2 V values a row move.  The exponentials are taken twice, not kept: kept in float32 they
//     fill the registers, one block an SM remains, and its phases (load, reduce, write) follow one
//     another instead of overlapping with those of two others (582 against 406 us).  What a
//     block does per row besides its 64 elements a thread is kept short: one exchange of maxima
//     and sums, teacher entries by the warps that have some.
//   loss alone: the row is read once, against running maxima, and its sums are kept for
//   the backward pass: with them every value of the gradient is a function of its logit.
// Statistics and products are float32; the gradient is rounded once.
//
// Measured (B200, K = 64, copy rate 6540 GB/s):
//                          loss and gradient      loss alone      gradient from the sums
//   16384 x 32768 bf16     383 us (86% of rate)   176 us (93%)    347 us (95%)
//   2048 x 32768 bf16      58 us (71%)            33 us (62%)     50 us (83%)
//   4096 x 32768 float32   203 us (81%)           88 us (93%)     164 us (100%)
//   4096 x 32767 bf16 (rows off the 16-byte grid)
//                          113 us (73%)           56 us (74%)     95 us (87%)
//   20000 x 8192 bf16      144 us (70%)           66 us (76%)     116 us (87%)
//   65536 x 1000 bf16, K = 16
//                          82 us (49%)            50 us (40%)     60 us (67%)
// The loss alone through the staged rows was 235 us (70%) and 140 us (59%) for the first and third,
// their backward pass without sums 405 and 213 us; with the running sum rescaled for every new
// maximum the loss was 192 and 98 us (versions before this one).  What the loss sums over the
// entries goes against the row's own maxima, after the exchange (1 to 3% of the loss alone).
#include <cooperative_groups.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "dp_common.cuh"
#include "tc_ptx.cuh"

namespace cg = cooperative_groups;

namespace dp {
namespace {

using namespace ptx;

constexpr int kDiMaxVec = 8;  // 16-byte vectors of a row per thread, at most
constexpr int kDiMaxThreads = 512;
constexpr int kDiMaxK = 1024;
constexpr float kDiShrink = 1.f / kDiMaxK;
constexpr int kDiMaxCluster = 16;
constexpr int64_t kDiMaxRows = 1 << 26;  // of a call, below this
constexpr int kDiSms = 148;
constexpr int kDiWarpRows = 4;    // rows of a block where a warp holds a row
constexpr int kDiLossThreads = 256;
constexpr int kDiStream = 4;      // vectors a thread adds to its running sum at a time
constexpr int kDiGradThreads = 512;  // gradient from the sums, at most

struct DistillArgs {
  const void *z, *index, *teacher;
  const float *weight, *grad;
  float *loss;
  float4 *stats;  // per row M, S, TM, TS: written by the loss (or null), read by the backward pass
  void *dz;
  int64_t rows, sb, st;
  int index64, teacher_dt, L, V, K, cs;
  int group_smem;   // bytes of shared memory of a group
  int stage_bytes;  // the part of it that holds the group's vectors
  int regular;      // one row stride, rows (dz's too) of whole vectors on 16 bytes
  float tau, c;     // c = log2(e) / tau
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
// with c = log2(e) / tau; the maximum tm of its teacher entries and ts = sum 2^((t - tm) c).
struct Part {
  float m, s, tm, ts;
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
  struct Max {
    float m;
    __device__ __forceinline__ void start() { m = -INFINITY; }
    __device__ __forceinline__ void add(const uint4 &v) {
      m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)),
                         fmaxf(__uint_as_float(v.z), __uint_as_float(v.w))));
    }
    __device__ __forceinline__ float get(float x) const { return fmaxf(x, m); }
  };
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
  struct Max {  // in pairs until the end
    __nv_bfloat162 m;
    __device__ __forceinline__ void start() { m = __float2bfloat162_rn(-INFINITY); }
    __device__ __forceinline__ void add(const uint4 &v) {
      const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&v);
      m = __hmax2(m, __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    }
    __device__ __forceinline__ float get(float x) const {
      const float2 f = __bfloat1622float2(m);
      return fmaxf(x, fmaxf(f.x, f.y));
    }
  };
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
  struct Max {  // in pairs until the end
    __half2 m;
    __device__ __forceinline__ void start() { m = __float2half2_rn(-INFINITY); }
    __device__ __forceinline__ void add(const uint4 &v) {
      const __half2 *h = reinterpret_cast<const __half2 *>(&v);
      m = __hmax2(m, __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    }
    __device__ __forceinline__ float get(float x) const {
      const float2 f = __half22float2(m);
      return fmaxf(x, fmaxf(f.x, f.y));
    }
  };
};

// v 2^((m - M) c), for a sum v against the maximum m; against -inf (nothing there) v is 0 or NaN.
__device__ __forceinline__ float di_scaled(float v, float m, float M, float c) {
  return m == -INFINITY ? v : v * di_ex2((m - M) * c);
}
// The (maximum, sum) of the cluster out of its blocks'.
__device__ __forceinline__ void di_join(const float2 *part, int cs, float c, float &M, float &S) {
  for (int r = 0; r < cs; ++r) M = fmaxf(M, part[r].x);
  S = 0.f;
  for (int r = 0; r < cs; ++r) S += di_scaled(part[r].y, part[r].x, M, c);
}

// Shared memory of one group: the teacher's entries (index, logit, the student's logit there)
// and two bit maps over hashed indices: an entry is there; more than one is (or two indices
// meet, which costs time only).  32 K bits and more: few indices meet.
__host__ __device__ inline int di_map_words(int K) {
  int w = 8;
  while (w < K) w *= 2;
  return w;
}
inline int di_smem(int K) { return 12 * K + 8 * di_map_words(K); }

struct Entries {
  int *index;       // -1: padding
  float *t, *z;     // teacher's and student's logit there
  uint32_t *once, *again;
  int words;
  __device__ __forceinline__ void clear(int tid, int n) const;                       // the bit maps
  __device__ __forceinline__ void mark(const DistillArgs &a, int tid, int n) const;  // the entries' bits
};
__device__ __forceinline__ Entries di_entries(unsigned char *mem, int K) {
  Entries e;
  e.index = reinterpret_cast<int *>(mem);
  e.t = reinterpret_cast<float *>(e.index + K), e.z = e.t + K;
  e.words = di_map_words(K);
  e.once = reinterpret_cast<uint32_t *>(e.z + K), e.again = e.once + e.words;
  return e;
}
__device__ __forceinline__ void Entries::clear(int tid, int n) const {
  for (int k = tid; k < 2 * words; k += n) once[k] = 0;
}
__device__ __forceinline__ void Entries::mark(const DistillArgs &a, int tid, int n) const {
  for (int k = tid; k < a.K; k += n)
    if (index[k] >= 0) {
      const uint32_t bit = 1u << (index[k] & 31);
      uint32_t *word = &once[index[k] >> 5 & (words - 1)];
      if (atomicOr(word, bit) & bit) atomicOr(word + words, bit);
    }
}

// One teacher entry as it is read ahead of its row.
struct Entry {
  int64_t index;
  uint32_t t;
  __device__ __forceinline__ void read(const DistillArgs &a, unsigned row, int k) {
    const int64_t o = (int64_t)row * a.K + k;
    index = a.index64 ? static_cast<const int64_t *>(a.index)[o] : static_cast<const int32_t *>(a.index)[o];
    t = load_raw_scalar(a.teacher, a.teacher_dt, o);
  }
  __device__ __forceinline__ bool ok(const DistillArgs &a) const { return index >= 0 && index < a.V; }
};
// The same with the student's logit there; index -1: padding.
struct Seen {
  int index;
  float t, z;
  template <typename T>
  __device__ __forceinline__ Seen(const DistillArgs &a, const T *row, const Entry &x) {
    const bool ok = x.ok(a);
    index = ok ? (int)x.index : -1;
    t = ok ? raw_scalar_to_f32(x.t, a.teacher_dt) : -INFINITY;
    z = ok ? to_f32(row[x.index]) : 0.f;
  }
};

// A row as its group sees it: 16-byte aligned vectors from element `head` on, split over the
// cluster (this block's: v0 .. v0 + cnt - 1), and fewer than 2 E single elements before and
// behind them, one each for the threads of the first block (edge; none: V and on).
template <typename T>
struct Row {
  const T *z;
  T *dz;
  unsigned row;
  int head, tail, v0, cnt, edge;
  bool vec;  // dz lies like z against the 16-byte grid
  __device__ __forceinline__ Row(const DistillArgs &a, unsigned row_, int rank, int cs, int tid) : row(row_) {
    constexpr int E = Vec<T>::E;
    dz = a.dz ? static_cast<T *>(a.dz) + (int64_t)row * a.V : nullptr;
    int nvec;
    if (a.regular) {  // every row is vectors from its first element to its last
      z = static_cast<const T *>(a.z) + row * a.st;
      head = 0, tail = edge = a.V, nvec = a.V / E;
      vec = true;
    } else {
      const unsigned batch = row / a.L;
      z = static_cast<const T *>(a.z) + batch * a.sb + (row - batch * a.L) * a.st;
      const int phase = (int)((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(T));
      head = min(phase ? E - phase : 0, a.V);
      nvec = (a.V - head) / E;
      tail = head + nvec * E;
      edge = rank ? a.V : tid < head ? tid : tail + tid - head;
      vec = (reinterpret_cast<uintptr_t>(dz) & 15) == (reinterpret_cast<uintptr_t>(z) & 15);
    }
    const int per = cs == 1 ? nvec : (nvec + cs - 1) / cs;
    v0 = min(rank * per, nvec), cnt = min(per, nvec - v0);
  }
  __device__ __forceinline__ const uint4 *vectors() const { return reinterpret_cast<const uint4 *>(z + head) + v0; }
  // Element i lies in this block's part: its vectors, and the single elements for the first.
  __device__ __forceinline__ bool has(int i, int rank) const {
    constexpr int E = Vec<T>::E;
    return i < head || i >= tail ? rank == 0 : i >= head + v0 * E && i < head + (v0 + cnt) * E;
  }
  // A row that does not count: loss 0 (by the caller), gradient 0, z not looked at.
  __device__ __forceinline__ void zeros(const DistillArgs &a, int tid, int n) const {
    constexpr int E = Vec<T>::E;
    for (int j = tid; j < cnt; j += n) {
      T *p = dz + head + (v0 + j) * E;
      if (vec)
        *reinterpret_cast<uint4 *>(p) = make_uint4(0, 0, 0, 0);
      else
        for (int k = 0; k < E; ++k) p[k] = from_f32<T>(0.f);
    }
    if (edge < a.V) dz[edge] = from_f32<T>(0.f);
  }
};

// The threads that hold a row (or a block's slice of it): tid of n, whole warps.
struct WarpGroup {
  int tid, n = 32;
  Part *parts;
  __device__ __forceinline__ void sync() const { __syncwarp(); }
};
struct BlockGroup {
  int tid, n;
  Part *parts;
  __device__ __forceinline__ void sync() const { __syncthreads(); }
};

template <typename T>
__device__ __forceinline__ uint4 di_nothing() {  // a vector of -inf
  uint4 v;
#pragma unroll
  for (int k = 0; k < Vec<T>::E / 2; ++k) Vec<T>::set(v, k, make_float2(-INFINITY, -INFINITY));
  return v;
}
// The i-th vector of a thread, -inf past the end: out of the row's copy in shared memory, or
// out of the registers it was read into.
struct FromShared {
  uint32_t v;  // of this thread
  int n;
  // volatile: read again in each pass, not kept in registers between them
  __device__ __forceinline__ uint4 operator()(int i) const {
    uint4 x;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n"
                 : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                 : "r"(v + i * n * 16));
    return x;
  }
};
template <int NV>
struct FromRegisters {
  uint4 v[NV];
  __device__ __forceinline__ uint4 operator()(int i) const { return v[i]; }
};

__device__ __forceinline__ void di_no_loss(const DistillArgs &a, unsigned row) {
  a.loss[row] = 0.f;
  if (a.stats) a.stats[row] = make_float4(0.f, 1.f, 0.f, 0.f);
}

// Exponentials of logits against a maximum m: z c - m c in one rounding; what the rounding of m c
// did to all of them alike is taken back from their sums (corr).  From |m c| = 2^31 on -- a small
// tau, or a row that is masked throughout by the type's lowest value -- that rounding would
// leave the exponents' range (m c might overflow), but there the float32 next to m is 2^-24 |m c|
// = 128 or more away in the exponent: 1 for m, 0 for all others (far).
struct Exps {
  float m0, c, mc, corr;  // m0: what is masked throughout has the sum 0, not NaN
  bool far;
  __device__ __forceinline__ Exps(float m, float c_) : c(c_) {
    m0 = m == -INFINITY ? 0.f : m;
    far = fabsf(m0) * c >= 2147483648.f && fabsf(m0) < INFINITY;
    mc = m0 * c, corr = far ? 1.f : di_ex2(-fmaf(m0, c, -mc));
  }
  __device__ __forceinline__ float near1(float z) const { return di_ex2(fmaf(z, c, -mc)); }
  __device__ __forceinline__ float2 near2(float2 z) const {
    const float2 x = __ffma2_rn(z, make_float2(c, c), make_float2(-mc, -mc));
    return make_float2(di_ex2(x.x), di_ex2(x.y));
  }
  __device__ __forceinline__ float far1(float z) const { return z == m0 ? 1.f : z == -INFINITY ? 0.f : z * 0.f; }
  __device__ __forceinline__ float2 far2(float2 z) const { return make_float2(far1(z.x), far1(z.y)); }
  __device__ __forceinline__ float one(float z) const { return far ? far1(z) : near1(z); }
};

// The maximum and the sum of exponentials of a thread's logits as they come by (from `one` on, a
// single one or -inf).  The sum s is against m, which follows the maximum where that is 2^32 ahead:
// until then the terms are larger, and as exact, as against the maximum itself.
template <typename T>
struct Running {
  typename Vec<T>::Max vm;
  float one, m, s;
  Exps x;
  __device__ __forceinline__ Running(float one_, float c) : one(one_), m(one_), x(one_, c) {
    vm.start();
    s = one == -INFINITY ? 0.f : one - one + 1.f;  // NaN and +inf: NaN
  }
  template <int N>
  __device__ __forceinline__ void add(const uint4 (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) vm.add(v[i]);
    const float m1 = vm.get(m);
    if ((m1 - m) * x.c > 32.f) {
      s = di_scaled(s, m, m1, x.c);
      m = m1;
      x = Exps(m, x.c);
    }
    float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
    auto sum = [&](auto exp_of) {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int k = 0; k < Vec<T>::E / 2; ++k) acc[k & 1] = __fadd2_rn(acc[k & 1], exp_of(Vec<T>::pair(v[i], k)));
    };
    if (!x.far)
      sum([&](float2 z) { return x.near2(z); });
    else
      sum([&](float2 z) { return x.far2(z); });
    acc[0] = __fadd2_rn(acc[0], acc[1]);
    s = fmaf(acc[0].x + acc[0].y, x.corr, s);
  }
  // the warp's
  __device__ __forceinline__ void finish(Part &w) const {
    w.m = di_warp_redux_max(vm.get(one));
    w.s = di_warp_sum(di_scaled(s, m, w.m, x.c));
  }
};

// What a row's sums are: the maximum and the sum of its logits' exponentials, those of the
// teacher's, and whether it has no teacher entries.
struct Sums {
  float M, S, TM, TS;
  bool empty;
};

// The group's entries into shared memory, their sums, the sums of the row out of the warps' (w.m
// and w.s are there), and its loss.  TM and TS are valid in the warps that handle entries.
// first: entry `tid`, read ahead.  `join` makes the (maximum, sum)
// of the cluster out of this block's.
template <typename T, class G, class Join>
__device__ __forceinline__ Sums di_sums(const DistillArgs &a, const G &g, const Row<T> &r, const Entries &e, int rank,
                                        float weight, Part w, const Seen &first, Join join) {
  const int tid = g.tid, n = g.n, lane = threadIdx.x & 31, warps = n >> 5;
  const float c = a.c;
  const bool entries = tid - lane < a.K;  // a warp that has some
  constexpr bool kWhole = std::is_same_v<G, WarpGroup>;  // the warp has the whole row
  float d = 0.f;
  w.tm = -INFINITY, w.ts = 0.f;
  if (entries) {
    float tm = -INFINITY;
    auto put = [&](int k, const Seen &x) {
      e.index[k] = x.index, e.t[k] = x.t, e.z[k] = x.z;
      tm = fmaxf(tm, x.t);
    };
    if (tid < a.K) put(tid, first);
    for (int k = tid + n; k < a.K; k += n) {
      Entry x;
      x.read(a, r.row, k);
      put(k, Seen(a, r.z, x));
    }
    w.tm = di_warp_redux_max(tm);
    const float t0 = w.tm == -INFINITY ? 0.f : w.tm;
    for (int k = tid; k < a.K; k += n) {
      const float t = e.t[k] - t0, x = di_ex2(t * c);
      w.ts += x;
      if (kWhole && x != 0.f) d = fmaf(x * kDiShrink, t - (e.z[k] - w.m), d);
    }
    w.ts = di_warp_sum(w.ts);
  }
  if (a.dz) e.clear(tid, n);
  // the parts of all warps: maxima, then sums relative to them; what the teacher's side gives
  // is needed where entries are handled and by the thread that writes the loss
  Sums q = {w.m, w.s, w.tm, w.ts, w.ts == 0.f};
  if (warps > 1) {
    if (lane == 0) g.parts[tid >> 5] = w;
    g.sync();
    Part o = {-INFINITY, 0.f, -INFINITY, 0.f};
    if (lane < warps) o = g.parts[lane];
    q.M = di_warp_redux_max(o.m);
    const float os = di_scaled(o.s, o.m, q.M, c);
    q.S = di_warp_sum(os);
    q.empty = !__any_sync(0xffffffffu, o.ts != 0.f);
    if (entries) {
      q.TM = di_warp_redux_max(o.tm);
      const float f = o.tm == -INFINITY ? 1.f : di_ex2((o.tm - q.TM) * c);
      q.TS = di_warp_sum(o.ts * f);
    }
  } else {
    g.sync();
  }
  if (a.dz && entries) e.mark(a, tid, n);  // the maps were cleared before the barrier
  join(q.M, q.S);
  // masked throughout (or NaN throughout): 0 / 0
  if (q.M == -INFINITY) q.S = NAN;
  if (rank == 0 && tid < 32) {
    // sum p (log p - log q) = sum p ((t - TM) - (z - M)) / tau - log TS + log S; times tau^2
    // without tau^2 or 1 / tau, which may leave the float32 range.  One warp forms it from the
    // row's own maxima: a part's maximum may be that of masked logits or entries only, and
    // differences from it keep no digits of z.  p, or its multiple made small, so that the sum of
    // masked logits stays in range; a p that is 0 counts nothing, whatever z is.
    const float inv_TS = di_rcp(q.TS);
    if (!kWhole)
      for (int k = tid; k < a.K; k += 32) {
        const float t = e.t[k] - q.TM, p = di_ex2(t * c) * inv_TS;
        if (p != 0.f) d = fmaf(p, t - (e.z[k] - q.M), d);
      }
    d = di_warp_sum(d);
    if (kWhole) d = d * inv_TS / kDiShrink;
    if (tid == 0) {
      a.loss[r.row] = q.empty ? 0.f : weight * (a.tau * (d + a.tau * (logf(q.S) - logf(q.TS))));
      if (a.stats) a.stats[r.row] = make_float4(q.M, q.S, q.TM, q.TS);
    }
  }
  return q;
}

// The gradients at the teacher's entries, over the dense values written there (a barrier and the
// completed bit maps before).  cw = weight tau grad.
template <typename T, class G>
__device__ __forceinline__ void di_entry_grads(const DistillArgs &a, const G &g, const Row<T> &r, const Entries &e,
                                               int rank, const Sums &q, float cw) {
  const int tid = g.tid, n = g.n, lane = threadIdx.x & 31;
  const float c = a.c, inv_S = di_rcp(q.S), inv_TS = di_rcp(q.TS);
  for (int k0 = tid - lane; k0 < a.K; k0 += n) {  // whole warps
    const int k = k0 + lane, i = k < a.K ? e.index[k] : -1;
    const bool here = i >= 0 && r.has(i, rank);
    float p = here ? di_ex2((e.t[k] - q.TM) * c) * inv_TS : 0.f;
    // an index that occurs more than once: the warp adds up all its entries, in a fixed
    // order, so each of them writes the same value
    uint32_t more = __ballot_sync(0xffffffffu, here && (e.again[i >> 5 & (e.words - 1)] >> (i & 31) & 1));
    while (more) {
      const int from = __ffs(more) - 1, at = __shfl_sync(0xffffffffu, i, from);
      more &= more - 1;
      float t = 0.f;
      for (int j = lane; j < a.K; j += 32)
        if (e.index[j] == at) t += di_ex2((e.t[j] - q.TM) * c) * inv_TS;
      t = di_warp_sum(t);
      if (lane == from) p = t;
    }
    if (here) r.dz[i] = from_f32<T>(cw * (di_ex2((e.z[k] - q.M) * c) * inv_S - p));
  }
}

// A vector of a row's gradient at p.
template <typename T>
__device__ __forceinline__ void di_store(const Row<T> &r, T *p, const uint4 &o) {
  constexpr int E = Vec<T>::E;
  if (r.vec) {
    *reinterpret_cast<uint4 *>(p) = o;
  } else {
    const T *x = reinterpret_cast<const T *>(&o);
#pragma unroll
    for (int k = 0; k < E; ++k) p[k] = x[k];
  }
}

// Loss and gradient of a row (ze: the thread's single element, -inf if none).
// KEEP: the exponentials, against the warp's maximum, are kept in float32 registers and the
// gradient is their multiple; otherwise a running sum takes kDiStream vectors at a time (16384 x
// 32768 bf16: 387 us; 2: 422, 8: 465 with spilled registers) and the gradient's pass computes the
// exponentials again, against the row's maximum.
template <typename T, int NV, bool KEEP, class G, class Src, class Join>
__device__ __forceinline__ void di_row(const DistillArgs &a, const G &g, const Row<T> &r, const Entries &e, int rank,
                                       float weight, const Src &src, float ze, const Seen &first,
                                       Join join) {
  using W = Vec<T>;
  constexpr int E = W::E;
  const int tid = g.tid, n = g.n, lane = threadIdx.x & 31;
  Part w;
  float2 ev[KEEP ? NV * E / 2 : 1];
  if constexpr (KEEP) {
    typename W::Max vm;
    vm.start();
#pragma unroll
    for (int i = 0; i < NV; ++i) vm.add(src(i));
    w.m = di_warp_redux_max(vm.get(ze));
    const Exps x(w.m, a.c);
    float2 acc[2] = {make_float2(x.one(ze), 0.f), make_float2(0.f, 0.f)};
    auto sum = [&](auto exp_of) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < E / 2; ++k) {
          ev[i * (E / 2) + k] = exp_of(W::pair(src(i), k));
          acc[k & 1] = __fadd2_rn(acc[k & 1], ev[i * (E / 2) + k]);
        }
    };
    if (!x.far)
      sum([&](float2 z) { return x.near2(z); });
    else
      sum([&](float2 z) { return x.far2(z); });
    acc[0] = __fadd2_rn(acc[0], acc[1]);
    w.s = di_warp_sum(acc[0].x + acc[0].y) * x.corr;
  } else {
    constexpr int H = NV < kDiStream ? NV : kDiStream;
    Running<T> sum(ze, a.c);
#pragma unroll
    for (int i = 0; i < NV; i += H) {
      uint4 v[H];
#pragma unroll
      for (int k = 0; k < H; ++k) v[k] = src(i + k);
      sum.add(v);
    }
    sum.finish(w);
  }
  const Sums q = di_sums(a, g, r, e, rank, weight, w, first, join);
  if (!a.dz) return;
  if (q.empty) {
    r.zeros(a, tid, n);
    return;
  }
  const bool entries = tid - lane < a.K;
  const float cw = weight * a.tau;
  // KEEP: from the warp's maximum to the row's (a warp that is masked throughout has only zeros)
  const Exps y(KEEP ? w.m : q.M, a.c);
  const float scale = (KEEP ? di_scaled(cw * di_rcp(q.S), w.m, q.M, a.c) : cw * di_rcp(q.S)) * y.corr;
  const float2 scale2 = make_float2(scale, scale);
  T *pd = r.dz + r.head + (r.v0 + tid) * E;
  auto write = [&](auto exp_of) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      uint4 o, v;
      if (!KEEP) v = src(i);
#pragma unroll
      for (int k = 0; k < E / 2; ++k)
        W::set(o, k, __fmul2_rn(KEEP ? ev[i * (E / 2) + k] : exp_of(W::pair(v, k)), scale2));
      if (tid + i * n < r.cnt) di_store(r, pd + i * n * E, o);
    }
  };
  if (!KEEP && y.far)
    write([&](float2 z) { return y.far2(z); });
  else
    write([&](float2 z) { return y.near2(z); });
  if (r.edge < a.V) r.dz[r.edge] = from_f32<T>(y.one(ze) * scale);
  g.sync();  // the dense values are written and the maps complete: now the teacher's entries
  if (entries) di_entry_grads(a, g, r, e, rank, q, cw);
}

// Loss and gradient, and the loss alone of short or few rows.
// A block (or a cluster of a.cs blocks) holds a row, or with WARP a warp, kDiWarpRows rows a
// block; NV vectors per thread.  STAGE: the vectors wait in shared memory, each copied there
// (cp.async) by the thread that reads it, twice, so that three times as many threads fit on an
// SM as hold their exponentials in registers: many rows, HBM counts.  Otherwise they are read
// into registers: few rows, latency counts (16 x 32768 bf16, loss: 4 blocks a row, 15 us a call
// with 12 us of it on the host).
template <typename T, int NV, bool WARP, bool STAGE>
__global__ void __launch_bounds__(WARP ? 32 * kDiWarpRows : kDiMaxThreads, WARP ? 8 : STAGE ? 3 : 2)
distill_kernel(const DistillArgs a) {
  __shared__ Part parts[kDiMaxThreads / 32];
  __shared__ float2 cpart[kDiMaxCluster];
  extern __shared__ __align__(16) unsigned char dyn[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int cs = WARP ? 1 : a.cs, rank = WARP ? 0 : blockIdx.x % cs;
  const unsigned row = WARP ? blockIdx.x * kDiWarpRows + warp : blockIdx.x / cs;
  if (WARP && row >= a.rows) return;  // whole warps
  std::conditional_t<WARP, WarpGroup, BlockGroup> g;
  g.tid = WARP ? lane : (int)threadIdx.x, g.n = WARP ? 32 : (int)blockDim.x, g.parts = parts;
  const float weight = a.weight ? a.weight[row] : 1.f;
  Entry first = {-1, 0};
  if (g.tid < a.K) first.read(a, row, g.tid);
  const Row<T> r(a, row, rank, cs, g.tid);
  if (weight == 0.f) {  // the same for the whole cluster
    if (rank == 0 && g.tid == 0) di_no_loss(a, row);
    if (a.dz) r.zeros(a, g.tid, g.n);
    return;
  }
  unsigned char *mem = dyn + (WARP ? warp * a.group_smem : 0);
  std::conditional_t<STAGE, FromShared, FromRegisters<NV>> src;
  if constexpr (STAGE) {
    uint4 *slot = reinterpret_cast<uint4 *>(mem) + g.tid;
    const uint32_t s = smem_u32(slot);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (g.tid + i * g.n < r.cnt)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(s + i * g.n * 16),
                     "l"(r.vectors() + g.tid + i * g.n)
                     : "memory");
      else
        slot[i * g.n] = di_nothing<T>();
    }
    mem += a.stage_bytes;
    src.v = s, src.n = g.n;
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      src.v[i] = g.tid + i * g.n < r.cnt ? r.vectors()[g.tid + i * g.n] : di_nothing<T>();
  }
  if (cs > 1) cg::this_cluster().sync();  // every block of the cluster runs
  const float ze = r.edge < a.V ? to_f32(r.z[r.edge]) : -INFINITY;
  const Seen seen(a, r.z, first);
  if constexpr (STAGE) asm volatile("cp.async.wait_all;\n" ::: "memory");
  di_row<T, NV, !STAGE>(a, g, r, di_entries(mem, a.K), rank, weight, src, ze, seen, [&](float &M, float &S) {
    if (cs == 1) return;
    cg::cluster_group cl = cg::this_cluster();
    if (g.tid < cs) cl.map_shared_rank(cpart, g.tid)[rank] = make_float2(M, S);
    cl.sync();
    di_join(cpart, cs, a.c, M, S);
  });
}

// The loss alone, many rows: a block a row, which each thread reads once, kDiStream vectors at a
// time; 48 warps an SM are what hides the loads (2 vectors and 64 warps: 189 against 174 us for
// 16384 x 32768 bf16, 8 and 32: 193).
template <typename T>
__global__ void __launch_bounds__(kDiLossThreads, 6) distill_loss_kernel(const DistillArgs a) {
  using W = Vec<T>;
  __shared__ Part parts[kDiMaxThreads / 32];
  extern __shared__ __align__(16) unsigned char dyn[];
  const unsigned row = blockIdx.x;
  BlockGroup g;
  g.tid = threadIdx.x, g.n = blockDim.x, g.parts = parts;
  const float weight = a.weight ? a.weight[row] : 1.f;
  Entry first = {-1, 0};
  if (g.tid < a.K) first.read(a, row, g.tid);
  const Row<T> r(a, row, 0, 1, g.tid);
  if (weight == 0.f) {
    if (g.tid == 0) di_no_loss(a, row);
    return;
  }
  const uint4 *vec = r.vectors() + g.tid;
  const int step = kDiStream * g.n, full = r.cnt / step;
  uint4 v[kDiStream];
  auto fetch = [&](int j) {
#pragma unroll
    for (int i = 0; i < kDiStream; ++i) v[i] = vec[j + i * g.n];
  };
  auto fetch_end = [&] {
#pragma unroll
    for (int i = 0; i < kDiStream; ++i)
      v[i] = g.tid + full * step + i * g.n < r.cnt ? vec[full * step + i * g.n] : di_nothing<T>();
  };
  const float ze = r.edge < a.V ? to_f32(r.z[r.edge]) : -INFINITY;
  Running<T> sum(ze, a.c);
  for (int j = 0; j < full; ++j) {
    fetch(j * step);
    sum.add(v);
  }
  if (full * step < r.cnt) {
    fetch_end();
    sum.add(v);
  }
  const Seen seen(a, r.z, first);
  Part w;
  sum.finish(w);
  di_sums(a, g, r, di_entries(dyn, a.K), 0, weight, w, seen, [](float &, float &) {});
}

// The gradient from the row's sums, as the loss left them: every value by itself.  A block
// (WARP: a warp) takes one of the a.cs slices of a row.  64 registers a thread, of which eight
// vectors spill 8 to 48 bytes.
template <typename T, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? 32 * kDiWarpRows : kDiGradThreads, WARP ? 8 : 2)
distill_grad_kernel(const DistillArgs a) {
  using W = Vec<T>;
  constexpr int E = W::E;
  extern __shared__ __align__(16) unsigned char dyn[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = WARP ? 0 : blockIdx.x % a.cs;
  const unsigned row = WARP ? blockIdx.x * kDiWarpRows + warp : blockIdx.x / a.cs;
  if (WARP && row >= a.rows) return;  // whole warps
  std::conditional_t<WARP, WarpGroup, BlockGroup> g;
  g.tid = WARP ? lane : (int)threadIdx.x, g.n = WARP ? 32 : (int)blockDim.x, g.parts = nullptr;
  const Row<T> r(a, row, rank, WARP ? 1 : a.cs, g.tid);
  Entry first = {-1, 0};
  if (g.tid < a.K) first.read(a, row, g.tid);
  uint4 v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i)
    v[i] = g.tid + i * g.n < r.cnt ? r.vectors()[g.tid + i * g.n] : di_nothing<T>();
  const float grad = a.grad ? a.grad[row] : 1.f, cw = (a.weight ? a.weight[row] : 1.f) * a.tau * grad;
  const float4 st = a.stats[row];
  if (st.w == 0.f || grad == 0.f) {  // no entries, weight 0; or the loss does not count
    r.zeros(a, g.tid, g.n);
    return;
  }
  const float ze = r.edge < a.V ? to_f32(r.z[r.edge]) : -INFINITY;
  const Sums q = {st.x, st.y, st.z, st.w, false};
  const Entries e = di_entries(dyn + (WARP ? warp * a.group_smem : 0), a.K);
  const bool entries = g.tid - lane < a.K;
  e.clear(g.tid, g.n);
  for (int k = g.tid; k < a.K; k += g.n) {
    Entry x = first;
    if (k != g.tid) x.read(a, row, k);
    const bool ok = x.ok(a);
    e.index[k] = ok ? (int)x.index : -1;
    e.t[k] = ok ? raw_scalar_to_f32(x.t, a.teacher_dt) : -INFINITY;
    e.z[k] = ok && r.has((int)x.index, rank) ? to_f32(r.z[x.index]) : 0.f;
  }
  g.sync();
  if (entries) e.mark(a, g.tid, g.n);
  const Exps x(q.M, a.c);
  const float scale = cw * di_rcp(q.S) * x.corr;
  const float2 scale2 = make_float2(scale, scale);
  T *pd = r.dz + r.head + (r.v0 + g.tid) * E;
  auto write = [&](auto exp_of) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      uint4 o;
#pragma unroll
      for (int k = 0; k < E / 2; ++k) W::set(o, k, __fmul2_rn(exp_of(W::pair(v[i], k)), scale2));
      if (g.tid + i * g.n < r.cnt) di_store(r, pd + i * g.n * E, o);
    }
  };
  if (x.far)
    write([&](float2 z) { return x.far2(z); });
  else
    write([&](float2 z) { return x.near2(z); });
  if (r.edge < a.V) r.dz[r.edge] = from_f32<T>(x.one(ze) * scale);
  g.sync();
  if (entries) di_entry_grads(a, g, r, e, rank, q, cw);
}

// Launches KERN with clusters of `cluster` blocks; `most`: bytes of shared memory it may ask for.
template <void (*KERN)(const DistillArgs)>
int distill_run(const DistillArgs &a, int64_t blocks, int threads, size_t smem, size_t most, int cluster,
                cudaStream_t st) {
  DP_REQUIRE(blocks < (1ll << 31), DP_ERR_UNSUPPORTED, "dp_distill: too many rows of this width");
  // more than 48 KB of shared memory and 16-block clusters (a non-portable size): opt in once
  static thread_local bool opted[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !opted[dev])) {
    e = cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(KERN, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess && dev < 64) opted[dev] = true;
  }
  if (e == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, KERN, a);
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(DP_ERR_CUDA, std::string("dp_distill: ") + cudaGetErrorString(e));
  }
  return check_launch("distill kernel");
}
template <typename T, int NV, bool WARP, bool STAGE>
int distill_run_row(const DistillArgs &a, int64_t blocks, int threads, size_t smem, cudaStream_t st) {
  constexpr int groups = WARP ? kDiWarpRows : 1, n = WARP ? 32 : kDiMaxThreads;
  return distill_run<distill_kernel<T, NV, WARP, STAGE>>(
      a, blocks, threads, smem, groups * ((STAGE ? n * NV * 16 : 0) + di_smem(kDiMaxK)), a.cs, st);
}

template <typename T>
int distill_launch(DistillArgs a, cudaStream_t st) {
  constexpr int E = Vec<T>::E;
  const int64_t size = sizeof(T);
  const int nvec = a.V / E;  // at most: fewer where a row does not start on 16 bytes
  a.regular = a.V % E == 0 && (a.rows == a.L || a.sb == a.L * a.st) && a.st * size % 16 == 0 &&
              ((reinterpret_cast<uintptr_t>(a.z) | reinterpret_cast<uintptr_t>(a.dz)) & 15) == 0;
  const int entries = (di_smem(a.K) + 15) / 16 * 16;
  const size_t most_entries = di_smem(kDiMaxK);
  a.cs = 1;
  if (nvec <= 32 * kDiMaxVec) {
    const int64_t blocks = (a.rows + kDiWarpRows - 1) / kDiWarpRows;
    const int threads = 32 * kDiWarpRows;
    const size_t most = most_entries * kDiWarpRows;
    // no more vectors a thread than the row has (65536 x 1000 bf16, 4 instead of 8: loss and gradient
    // 82 against 101 us, loss 50 against 60, gradient from the sums 60 against 68)
    auto run = [&](auto vectors) {
      constexpr int NV = decltype(vectors)::value;
      a.stage_bytes = a.loss ? 32 * NV * 16 : 0;
      a.group_smem = a.stage_bytes + entries;
      const size_t smem = (size_t)a.group_smem * kDiWarpRows;
      return a.loss ? distill_run_row<T, NV, true, true>(a, blocks, threads, smem, st)
                    : distill_run<distill_grad_kernel<T, NV, true>>(a, blocks, threads, smem, most, 1, st);
    };
    return nvec <= 64    ? run(std::integral_constant<int, 2>{})
           : nvec <= 128 ? run(std::integral_constant<int, 4>{})
                         : run(std::integral_constant<int, kDiMaxVec>{});
  }
  if (!a.loss) {
    // the gradient from the sums: slices that need nothing of one another.  Small blocks overlap
    // best (16384 x 32768 bf16, K = 64: 128 threads 348 us, 512 threads 365), but each slice goes
    // through all K entries (1000 x 131072 float32, K = 1024: 339 against 228 us).
    const int slice = (a.K <= 128 ? 128 : kDiGradThreads) * kDiMaxVec;
    a.cs = (nvec + slice - 1) / slice;
    const int per = (nvec + a.cs - 1) / a.cs;
    const int threads = std::max(64, ((per + kDiMaxVec - 1) / kDiMaxVec + 31) / 32 * 32);
    return distill_run<distill_grad_kernel<T, kDiMaxVec, false>>(a, a.rows * a.cs, threads, entries, most_entries, 1,
                                                                 st);
  }
  if (!a.dz && a.rows >= 2 * kDiSms) {
    // 16 vectors a thread in small blocks (20000 x 8192 bf16: 64 us, with 8 vectors 72; 509 x 50021
    // float32 in blocks of 512: 29 us against 25)
    const int threads = std::min(kDiLossThreads, std::max(64, (nvec / 16 + 31) / 32 * 32));
    return distill_run<distill_loss_kernel<T>>(a, a.rows, threads, entries, most_entries, 1, st);
  }
  const int most = kDiMaxThreads * kDiMaxVec;
  while (a.cs < kDiMaxCluster && (int64_t)a.cs * most < nvec) a.cs *= 2;
  DP_REQUIRE((int64_t)a.cs * most >= nvec, DP_ERR_UNSUPPORTED, "dp_distill: V too large");
  // few rows: split each over more blocks, down to a vector per thread (one row of 131072
  // float32 logits: 16 blocks); enough rows to fill the GPU are split only as far as they must
  // (loss and gradient at 1 / 2 / 4 / 8 blocks a row: 16384 x 32768 bf16 383 / 439 / 547 / 917 us, 2048
  // rows 58 / 66 / 78 / 121; 16 or 200 rows, from the host, 18 to 22 us with any of them)
  while (a.cs < kDiMaxCluster && a.rows * a.cs < kDiSms && nvec / a.cs >= 2 * kDiMaxThreads) a.cs *= 2;
  const int per = (nvec + a.cs - 1) / a.cs;
  const int64_t blocks = a.rows * a.cs;
  const int nv = blocks >= 2 * kDiSms || per > 4 * kDiMaxThreads ? kDiMaxVec : per > kDiMaxThreads ? 4 : 1;
  const int threads = std::max(64, ((per + nv - 1) / nv + 31) / 32 * 32);
  a.stage_bytes = nv == kDiMaxVec ? threads * nv * 16 : 0;
  a.group_smem = a.stage_bytes + entries;
  if (nv == 1) return distill_run_row<T, 1, false, false>(a, blocks, threads, a.group_smem, st);
  if (nv == 4) return distill_run_row<T, 4, false, false>(a, blocks, threads, a.group_smem, st);
  return distill_run_row<T, kDiMaxVec, false, true>(a, blocks, threads, a.group_smem, st);
}

}  // namespace
}  // namespace dp

namespace {

// What both entry points check of their arguments; DP_OK: go on (with B L rows).
int distill_args(dp::DistillArgs &a, const char *what, const void *z, int z_dtype, const void *index, int index_bytes,
                 const void *teacher, int teacher_dtype, const float *weight, float tau, void *dz, int B, int L, int V,
                 int K, const int64_t *strides) {
  using namespace dp;
  const std::string w = std::string(what) + ": ";
  DP_REQUIRE(B >= 0 && L >= 0 && V >= 1 && K >= 1, DP_ERR_INVALID_ARGUMENT, w + "bad sizes");
  DP_REQUIRE(valid_dtype(z_dtype) && valid_dtype(teacher_dtype), DP_ERR_INVALID_ARGUMENT, w + "unknown dtype code");
  DP_REQUIRE(index_bytes == 4 || index_bytes == 8, DP_ERR_INVALID_ARGUMENT, w + "index must be int32 or int64");
  DP_REQUIRE(tau > 1e-30f && tau < 1e30f, DP_ERR_INVALID_ARGUMENT, w + "tau must be positive and finite");
  DP_REQUIRE(K <= kDiMaxK, DP_ERR_UNSUPPORTED, w + "K must be <= 1024");
  DP_REQUIRE((int64_t)V * (int64_t)dtype_size(z_dtype) <= (1 << 20) - 32, DP_ERR_UNSUPPORTED,
             w + "a row of z must be smaller than 1 MiB");
  a.rows = (int64_t)B * L;
  if (a.rows == 0) return DP_OK;
  DP_REQUIRE(z && index && teacher && strides, DP_ERR_INVALID_ARGUMENT, w + "null pointer");
  DP_REQUIRE(z != dz, DP_ERR_INVALID_ARGUMENT, w + "dz must not be z");
  DP_REQUIRE(a.rows < kDiMaxRows, DP_ERR_UNSUPPORTED, w + "too many rows");
  a.z = z, a.sb = strides[0], a.st = strides[1], a.index = index, a.index64 = index_bytes == 8, a.teacher = teacher;
  a.teacher_dt = teacher_dtype, a.weight = weight, a.dz = dz;
  a.tau = tau, a.c = 1.4426950408889634f / tau;
  a.L = L, a.V = V, a.K = K;
  return DP_OK;
}

}  // namespace

extern "C" int dp_distill(const void *z, int z_dtype, const void *index, int index_bytes, const void *teacher,
                          int teacher_dtype, const float *weight, float tau, float *loss, float *stats, void *dz,
                          int B, int L, int V, int K, const int64_t *strides, void *stream) {
  using namespace dp;
  DistillArgs a = {};
  const int rc = distill_args(a, "dp_distill", z, z_dtype, index, index_bytes, teacher, teacher_dtype, weight, tau, dz,
                              B, L, V, K, strides);
  if (rc != DP_OK || a.rows == 0) return rc;
  DP_REQUIRE(loss, DP_ERR_INVALID_ARGUMENT, "dp_distill: null pointer");
  DP_REQUIRE((reinterpret_cast<uintptr_t>(stats) & 15) == 0, DP_ERR_MISALIGNED,
             "dp_distill: stats must be 16-byte aligned");
  a.loss = loss, a.stats = reinterpret_cast<float4 *>(stats);
  cudaStream_t st = as_stream(stream);
  return dispatch_dtype(z_dtype, [&](auto t) { return distill_launch<decltype(t)>(a, st); });
}

extern "C" int dp_distill_bwd(const void *z, int z_dtype, const void *index, int index_bytes, const void *teacher,
                              int teacher_dtype, const float *weight, const float *stats, const float *grad, float tau,
                              void *dz, int B, int L, int V, int K, const int64_t *strides, void *stream) {
  using namespace dp;
  DistillArgs a = {};
  const int rc = distill_args(a, "dp_distill_bwd", z, z_dtype, index, index_bytes, teacher, teacher_dtype, weight, tau,
                              dz, B, L, V, K, strides);
  if (rc != DP_OK || a.rows == 0) return rc;
  DP_REQUIRE(stats && dz, DP_ERR_INVALID_ARGUMENT, "dp_distill_bwd: null pointer");
  DP_REQUIRE((reinterpret_cast<uintptr_t>(stats) & 15) == 0, DP_ERR_MISALIGNED,
             "dp_distill_bwd: stats must be 16-byte aligned");
  a.grad = grad, a.stats = reinterpret_cast<float4 *>(const_cast<float *>(stats));
  cudaStream_t st = as_stream(stream);
  return dispatch_dtype(z_dtype, [&](auto t) { return distill_launch<decltype(t)>(a, st); });
}
