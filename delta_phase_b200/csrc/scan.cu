// Gated linear recurrence over long sequences, forward and backward: the vector-state
// counterpart of LaplacePhaseCore's per-row decay (delta_phase/layers.py:481-561).
//   h_t = a_t h_{t-1} + u_t per channel, out_t = h_t;  with d_t = 1 - a_t:
//   DP_SCAN_DECAY   a = exp(gate),     u = x
//   DP_SCAN_SIGMOID a = sigmoid(gate), u = d x
// Backward: p_t = dout_t + q_{t+1}, q_t = a_t p_t (q_L = dL/dh_{L-1} from outside):
//   decay: dx = p, dgate = q h_{t-1};  sigmoid: dx = d p, dgate = q d (h_{t-1} - x)
//   and dL/dh_{-1} = q_0.
//
// No float32 holds both ends of a gate: an a close to 1 has lost the digits of 1 - a, which is
// what a long memory consists of, and a d close to 1 those of a, which is all that the old state
// and the gate's gradient see.  Tokens use a (and in sigmoid mode d beside it), each exact to its
// own digits: the few of a block lose nothing that shows.  What goes on from block to block is a
// map whose factor is a - 1 where the product of the a is close to 1 and the product elsewhere.  A
// gate that drops the state (a = 0) leaves exactly nothing of it.
//
// Layout: a lane owns the channels of one 4-byte word (two 16-bit values, packed two-wide
// float32 arithmetic, or one float), a warp kTok consecutive tokens of its 32 words, a block
// kWarps warps (kTile tokens), and a thread-block cluster up to 16 consecutive tiles of one
// sequence.  Each warp reduces its tokens to an affine map of the state, the maps are combined
// through shared memory inside the block and by messages inside the cluster, and each warp then
// runs the recurrence over its tokens again from the exact state that reaches it: every input
// is read from HBM once and the order of all sums is fixed.  A cluster walks over a long
// sequence in steps of its span; the next span is on its way to shared memory while one is
// computed, and the outputs leave from the slots of the inputs they replace: by bulk tensor
// copies of a warp's box (kTok tokens of 32 words) where the tensors' alignment allows them,
// else by cp.async of single words and plain stores.  No warp waits for another one's copies.
//
// HBM bounds it where enough channels and tokens run at once (about 1.7 blocks an SM), the chain
// of spans (2.3 to 2.9 us each) where there are few.  Measured (B200, copy rate 6540 GB/s), forward
// and backward: 2 x 32768 x 1024 bf16 84 us (73% of the copy rate) and 121 us (85%), 8 x 8192 x
// 1024 bf16 78 us (79%) and 116 us (88%), in sigmoid mode 86 us (71%) and 132 us (78%), 4 x 8192 x
// 512 float32 39 us (78%) and 62 us (83%), 1 x 65536 x 256 bf16 (4 chains) 74 us (21%) and 92 us
// (28%).  The first was 148 and 190 us with a marked factor, and the selection that goes with it,
// for every token, and 93 and 125 us with one for every warp.  The backward pass fetches the next
// span's x and gradient after the second barrier: before the first, loads and stores meet (8 x
// 8192 x 1024 134 us, the first 117).  Older versions: every warp combining the maps 97 and 130 us
// against 88 and 123 by one; single words instead of boxes 144 and 216 us (address arithmetic), and
// with a cluster barrier instead of messages 179 and 321 us (its fence).
#include <cooperative_groups.h>

#include <algorithm>
#include <cstdlib>
#include <string>
#include <type_traits>

#include "cluster_msg.cuh"
#include "dp_common.cuh"
#include "tmap.cuh"

namespace cg = cooperative_groups;

namespace dp {

int *device_error_ptr();

namespace {

using namespace ptx;

constexpr int kTok = 16;              // tokens per warp
constexpr int kWarps = 8;             // warps per block
constexpr int kTile = kTok * kWarps;  // tokens per block; one saved state per tile
constexpr int kMaxCluster = 16;
constexpr int kThreads = kWarps * 32;

// ---------------------------------------------------------------- words of channels
__device__ __forceinline__ float fma_(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float add_(float a, float b) { return a + b; }
__device__ __forceinline__ float mul_(float a, float b) { return a * b; }
__device__ __forceinline__ float2 fma_(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 add_(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 mul_(float2 a, float2 b) { return __fmul2_rn(a, b); }
template <typename F>
__device__ __forceinline__ F all_(float v);
template <>
__device__ __forceinline__ float all_<float>(float v) { return v; }
template <>
__device__ __forceinline__ float2 all_<float2>(float v) { return make_float2(v, v); }

// V channels of type T in a 4-byte word: V = 2 for 16-bit pairs, V = 1 for a float or, where
// pairs cannot be loaded, for one 16-bit value.
template <typename T, int V>
struct Lane;
template <>
struct Lane<float, 1> {
  using F = float;
  static __device__ __forceinline__ F get(uint32_t w) { return __uint_as_float(w); }
  static __device__ __forceinline__ void store(float *p, F v) { *p = v; }
};
template <typename T>
struct Lane<T, 1> {
  using F = float;
  static __device__ __forceinline__ F get(uint32_t w) {
    const unsigned short h = (unsigned short)w;
    return to_f32(*reinterpret_cast<const T *>(&h));
  }
  static __device__ __forceinline__ void store(T *p, F v) { *p = from_f32<T>(v); }
};
template <>
struct Lane<__nv_bfloat16, 2> {
  using F = float2;
  static __device__ __forceinline__ F get(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ void store(__nv_bfloat16 *p, F v) {
    *reinterpret_cast<__nv_bfloat162 *>(p) = __float22bfloat162_rn(v);
  }
};
template <>
struct Lane<__half, 2> {
  using F = float2;
  static __device__ __forceinline__ F get(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
  static __device__ __forceinline__ void store(__half *p, F v) {
    *reinterpret_cast<__half2 *>(p) = __float22half2_rn(v);
  }
};

// ---------------------------------------------------------------- gates
__device__ __forceinline__ float ex2_(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 ex2_(float2 x) { return make_float2(ex2_(x.x), ex2_(x.y)); }
__device__ __forceinline__ float rcp_(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 rcp_(float2 x) { return make_float2(rcp_(x.x), rcp_(x.y)); }
__device__ __forceinline__ float min_nan(float a, float b) {  // NaN stays
  float m;
  asm("min.NaN.f32 %0, %1, %2;\n" : "=f"(m) : "f"(a), "f"(b));
  return m;
}
__device__ __forceinline__ float2 min_nan(float2 a, float b) { return make_float2(min_nan(a.x, b), min_nan(a.y, b)); }

// a of a gate, and in sigmoid mode d, each within a few steps of its own value.  16-bit gates: the
// hardware exponential and reciprocal (2^-22, and |gate| 2^-24 from the exponent's rounding):
// f = exp(gate), d = 1 / (1 + f), a = f d; f ends at 2^125, where a is 1, and the 2^-125 that is d
// there is taken from every d.  float32: the library's functions.
template <typename T, int MODE, typename F>
__device__ __forceinline__ void gate_(F g, F &a, F &d) {
  d = all_<F>(0.f);  // not used in decay mode
  if constexpr (sizeof(T) == 4) {
    if constexpr (MODE == DP_SCAN_SIGMOID) {
      const float v = 1.f / (1.f + expf(fabsf(g))), w = 1.f - v;
      a = g < 0.f ? v : w, d = g < 0.f ? w : v;
    } else {
      a = expf(g);
    }
  } else {
    a = ex2_(mul_(g, all_<F>(1.4426950408889634f)));
    if constexpr (MODE == DP_SCAN_SIGMOID) {
      a = min_nan(a, 4.2535296e37f);
      d = rcp_(add_(a, all_<F>(1.f)));
      a = mul_(a, d);
      d = add_(d, all_<F>(-2.3509887e-38f));
    }
  }
}

// ---------------------------------------------------------------- affine maps of the state
// What some tokens do to the state: h -> a h + H.  Inside a block a is enough, like it is for tokens.
// What the chain of blocks applies to the state, block after block, keeps a and n = a - 1, each to
// its own digits, in one word m: n where a lies in [1/2, 2], else a.  Its lowest bit tells which
// (1: n), for which it is cut to 23 bits; n = 0 becomes 2^-149, which no state sees.
template <typename F>
struct __align__(2 * sizeof(F)) Map {
  F a, H;  // of a block: m, H
};
__device__ __forceinline__ bool near_one(float n) { return fabsf(n - 0.25f) <= 0.75f; }
__device__ __forceinline__ float marked(float a, float n) {
  return __uint_as_float(near_one(n) ? __float_as_uint(n) | 1u : __float_as_uint(a) & ~1u);
}
__device__ __forceinline__ float2 marked(float2 a, float2 n) { return make_float2(marked(a.x, n.x), marked(a.y, n.y)); }
__device__ __forceinline__ float if_near(float m, float h) { return __float_as_uint(m) & 1u ? h : 0.f; }
__device__ __forceinline__ float2 if_near(float2 m, float2 h) { return make_float2(if_near(m.x, h.x), if_near(m.y, h.y)); }
// a h + H from m; the small part first, so that a state at its fixed point stays there
template <typename F>
__device__ __forceinline__ F apply_marked(const Map<F> &m, F h) {
  return add_(if_near(m.a, h), fma_(m.a, h, m.H));
}
template <typename F>
__device__ __forceinline__ F apply(const Map<F> &m, F h) {
  return fma_(m.a, h, m.H);
}
// The map of r and then w, and the n of both.
template <typename F>
__device__ __forceinline__ void follow(Map<F> &r, F &n, const Map<F> &w, F wn) {
  r.H = apply(w, r.H);
  r.a = mul_(r.a, w.a);
  n = add_(fma_(wn, n, n), wn);
}

// exp(s) - 1 beside a = exp(s): by its Taylor series where |s| < ln 2 (the first term left out is
// below 2^-26 of the value).
__device__ __forceinline__ float in_ln2(float s, float series, float other) { return fabsf(s) < 0.6931472f ? series : other; }
__device__ __forceinline__ float2 in_ln2(float2 s, float2 series, float2 other) {
  return make_float2(in_ln2(s.x, series.x, other.x), in_ln2(s.y, series.y, other.y));
}
template <typename F>
__device__ __forceinline__ F exp_less1(F s, F a) {
  F p = fma_(s, all_<F>(1.f / 362880.f), all_<F>(1.f / 40320.f));
  p = fma_(p, s, all_<F>(1.f / 5040.f));
  p = fma_(p, s, all_<F>(1.f / 720.f));
  p = fma_(p, s, all_<F>(1.f / 120.f));
  p = fma_(p, s, all_<F>(1.f / 24.f));
  p = fma_(p, s, all_<F>(1.f / 6.f));
  p = fma_(p, s, all_<F>(0.5f));
  p = fma_(p, s, all_<F>(1.f));
  return in_ln2(s, mul_(p, s), add_(a, all_<F>(-1.f)));
}

// a, and from n where that has more digits
__device__ __forceinline__ float best_a(float a, float n) { return near_one(n) ? n + 1.f : a; }
__device__ __forceinline__ float2 best_a(float2 a, float2 n) { return make_float2(best_a(a.x, n.x), best_a(a.y, n.y)); }

// The factor of a warp's tokens, as their gates come by.  Decay: from the gates' sum, whose exponential
// is the product (float32: the product itself where that is small, as the sum's roundings would show).
// Sigmoid: 1 - a follows a recurrence of its own, of positive terms: d + a D.
template <typename T, int MODE, typename F>
struct Product {
  F a = all_<F>(1.f), s = all_<F>(0.f);
  __device__ __forceinline__ void add(F gate, F ta, F td) {
    s = MODE == DP_SCAN_SIGMOID ? fma_(ta, s, td) : add_(s, gate);
    if (MODE == DP_SCAN_SIGMOID || sizeof(T) == 4) a = mul_(a, ta);
  }
  __device__ __forceinline__ void get(F &pa, F &pn) const {
    if constexpr (MODE == DP_SCAN_SIGMOID) {
      pa = a, pn = mul_(s, all_<F>(-1.f));
    } else {
      if constexpr (sizeof(T) == 4)
        pa = a;
      else
        pa = ex2_(mul_(s, all_<F>(1.4426950408889634f)));
      pn = exp_less1(s, pa);
    }
    pa = best_a(pa, pn);
  }
};

struct ScanArgs {
  const void *x, *gate, *dout;  // (B, L, D), strides {sb, st}
  const float *h0;              // (B, D) or null
  float *hL;                    // (B, D) final state
  float *saved;                 // (B, ceil(L / kTile), D) state before each tile (forward: or null)
  void *out, *dx, *dgate;
  const float *dhL;             // (B, D) or null
  float *dh0;                   // (B, D) or null
  int64_t xb, gb, ob;  // batch strides of x, gate and of out (forward) or dout (backward), elements
  int xt, gt, ot;      // their token strides, bytes
  int B, L, D, tiles_c, cs;
  int *err;  // device error word
};

// (B, D) and saved states: V consecutive floats
__device__ __forceinline__ void load_state(const float *p, float &v) { v = *p; }
__device__ __forceinline__ void load_state(const float *p, float2 &v) { v = make_float2(p[0], p[1]); }
__device__ __forceinline__ void store_state(float *p, float v) { *p = v; }
__device__ __forceinline__ void store_state(float *p, float2 v) { p[0] = v.x, p[1] = v.y; }

// p + t tokens of st bytes
template <typename T>
__device__ __forceinline__ T *at(T *p, int64_t t, int st) {
  using C = std::conditional_t<std::is_const_v<T>, const char, char>;
  return reinterpret_cast<T *>(reinterpret_cast<C *>(p) + t * st);
}
// The same for a small i: one 32 x 32 -> 64 bit multiply-add.
template <typename T>
__device__ __forceinline__ T *token(T *p, int i, int st) {
  using C = std::conditional_t<std::is_const_v<T>, const char, char>;
  return reinterpret_cast<T *>(reinterpret_cast<C *>(p) + (int64_t)i * st);
}

template <int BYTES>
__device__ __forceinline__ void copy_word(uint32_t dst, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}

// Copies the words of kTok tokens, st bytes apart, into the thread's own slots; tokens from n
// on are zero.  p points at the first token where n > 0, else at any valid element.
template <typename T, int V>
__device__ __forceinline__ void stage(uint32_t *slot, const T *p, int st, int n) {
  if constexpr (sizeof(T) * V == 4) {
    const uint32_t s = (uint32_t)__cvta_generic_to_shared(slot);
    if (n == kTok) {
#pragma unroll
      for (int i = 0; i < kTok; ++i) copy_word<4>(s + i * 128, token(p, i, st));
    } else {
#pragma unroll 1
      for (int i = 0; i < kTok; ++i) {
        if (i < n)
          copy_word<4>(s + i * 128, token(p, i, st));
        else
          copy_word<0>(s + i * 128, p);
      }
    }
  } else {
    unsigned short w[kTok];
#pragma unroll
    for (int i = 0; i < kTok; ++i) w[i] = i < n ? *reinterpret_cast<const unsigned short *>(token(p, i, st)) : 0;
#pragma unroll
    for (int i = 0; i < kTok; ++i) slot[i * 32] = w[i];
  }
}
__device__ __forceinline__ void stage_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
__device__ __forceinline__ void stage_wait() { asm volatile("cp.async.wait_group 0;\n" ::: "memory"); }

// Bulk tensor copies of a warp's box (kTok tokens of 32 words) where the tensors allow them:
// one instruction a box for one lane instead of a copy, its address and its bounds a word for
// every lane.  Tokens past L and channels past D arrive as zeros and are not stored.
struct ScanMaps {
  CUtensorMap x, gate, out;  // out: out, or dout
  CUtensorMap dx, dgate;
};
__device__ __forceinline__ void box_load(void *dst, const CUtensorMap *m, int c, int t, int b, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
      "[%5];\n" ::"r"(smem_u32(dst)),
      "l"(m), "r"(c), "r"(t), "r"(b), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void box_store(const CUtensorMap *m, const void *src, int c, int t, int b) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];\n" ::"l"(m), "r"(c),
               "r"(t), "r"(b), "r"(smem_u32(src))
               : "memory");
}

// The combination of the maps is the work of one warp of a block, between two barriers: it
// composes the warps' maps, leaving in each one's place the map of the warps before it, sends
// the block's map to every block of the cluster (st.async, counted in bytes on the receiver's
// mbarrier), waits for the maps of all, and leaves the state that reaches the block.  There is
// no cluster-wide barrier.  The buffers of the blocks' maps alternate: a block sends a span's map
// after it has used those of the span before, so whoever has received the maps of span s may
// send those of span s + 1 into the buffer of span s - 1.  No message is left when a block
// ends: it has received all that is sent to it.
//
// Every wait has a limit (kWaitNs; a GPU that answers is far below it).  A thread whose wait ran out
// arms no barrier, starts no copy, sends and stores nothing more: it goes through the remaining
// spans without waits, so that the others pass their barriers; threads that wait for its messages
// follow.  At the end (scan_end) it waits once more, with the same limit, for what it has in flight,
// and the block until no block of the cluster can send to it any more; the error word is set.
template <typename Shared>
__device__ __forceinline__ void scan_start(Shared &sh, int cs) {
  if (threadIdx.x == 0) {
    sh.expired = 0;
    mbar_init(&sh.bar[0], 1);
    mbar_init(&sh.bar[1], 1);
    for (int w = 0; w < kWarps; ++w) {
      mbar_init(&sh.gate_bar[w], 1);
      mbar_init(&sh.x_bar[w], 1);
    }
    fence_mbar_init();
  }
  if (cs > 1)
    cg::this_cluster().sync();  // the barriers exist in every block before the first message
  else
    __syncthreads();
}
// After the loop, by all threads.
template <bool TMA, typename Shared>
__device__ __forceinline__ void scan_end(Shared &sh, bool alive, int cs, int *err) {
  if (!alive) {
    sh.expired = 1;
    atomicCAS(err, 0, DP_ERR_TIMEOUT);
    if (TMA)  // the phase in flight, if any, is one of the two; the other one's wait passes or runs out
      for (int k = 0; k < 4; ++k)
        mbar_wait_loop(k & 1 ? &sh.x_bar[threadIdx.x >> 5] : &sh.gate_bar[threadIdx.x >> 5], k >> 1, kWaitNs);
  }
  __syncthreads();
  if (sh.expired && cs > 1) {
    // blocks that ended well have left and do not count; the others come here, too, and what they
    // sent before arrives within the time below
    cg::this_cluster().sync();
    const uint64_t t0 = globaltimer();
    while (globaltimer() - t0 < 1000000) __nanosleep(1000);
  }
}

// a and d of a thread's tokens from the staged gates, and the factor of them all.  Tokens past the
// end keep the state: their gates and x are staged as 0, which in decay mode is a = 1 already.
template <typename T, int V, int MODE, typename F>
__device__ __forceinline__ Product<T, MODE, F> load_gates(const uint32_t *slot, int n, F (&a)[kTok], F (&d)[kTok]) {
  Product<T, MODE, F> p;
  auto load = [&](auto whole) {
#pragma unroll
    for (int i = 0; i < kTok; ++i) {
      const F g = Lane<T, V>::get(slot[i * 32]);
      gate_<T, MODE>(g, a[i], d[i]);
      if (!decltype(whole)::value && i >= n) a[i] = all_<F>(1.f), d[i] = all_<F>(0.f);
      p.add(g, a[i], d[i]);
    }
  };
  if (MODE == DP_SCAN_DECAY || n == kTok)
    load(std::true_type{});
  else
    load(std::false_type{});
  return p;
}

// h' of a token
template <int MODE, typename F>
__device__ __forceinline__ F step_(F a, F d, F h, F x) {
  return fma_(a, h, MODE == DP_SCAN_SIGMOID ? mul_(d, x) : x);
}

// The H of a thread's tokens.  KEEP: their u stay in registers (d's) for the second pass.
template <typename T, int V, int MODE, bool KEEP, typename F>
__device__ __forceinline__ F reduce_tokens(const uint32_t *xw, const F (&a)[kTok], F (&d)[kTok]) {
  F H = all_<F>(0.f);
#pragma unroll
  for (int i = 0; i < kTok; ++i) {
    const F x = Lane<T, V>::get(xw[i * 32]), u = MODE == DP_SCAN_SIGMOID ? mul_(d[i], x) : x;
    if constexpr (KEEP) d[i] = u;
    H = fma_(a[i], H, u);
  }
  return H;
}

template <typename F, int NX>
struct ScanShared {
  uint32_t gate[kWarps][kTok][32];
  uint32_t x[NX][2][kWarps][kTok][32];      // x, and dout in the backward pass
  Map<F> wmap[kWarps][32];                  // the warps' maps, then those of the warps before each
  F wn[kWarps][32];                         // their n
  Map<F> bmap[2][kMaxCluster][32];          // the blocks' maps
  F carry[32];                              // the state (gradient) that reaches the block
  uint64_t bar[2];                          // one per buffer of bmap
  uint64_t gate_bar[kWarps], x_bar[kWarps];  // the warps' bulk copies
  int expired;                               // a wait of the block ran out
};
template <typename F>
struct ScanSharedBwd : ScanShared<F, 2> {
  F wq[kWarps][32];  // H of the warps' gradient maps
};

// ---------------------------------------------------------------- forward
// u in registers between the two passes: single values, and pairs in sigmoid mode, where it is d x
// (two blocks an SM instead of three: 8 x 8192 x 1024 bf16 84 us against 96 with a and d in one
// marked word; 11 x 8192 x 512, 352 blocks, 75 against 68, as they no longer all run at once).  Pairs
// in decay mode read x again: three blocks an SM have no registers left for it.
template <int V, int MODE>
constexpr bool kKeepU = V == 1 || MODE == DP_SCAN_SIGMOID;
template <typename T, int V, int MODE, bool TMA>
__global__ void __launch_bounds__(kThreads, V == 2 && kKeepU<V, MODE> ? 2 : 3)
scan_fwd_kernel(const ScanArgs a, const __grid_constant__ ScanMaps maps) {
  using F = typename Lane<T, V>::F;
  constexpr bool kKeep = kKeepU<V, MODE>;
  extern __shared__ __align__(128) unsigned char smem[];
  auto &sh = *reinterpret_cast<ScanShared<F, 1> *>(smem);
  const int rank = blockIdx.x % a.cs, chain = blockIdx.x / a.cs;
  const int b = chain / a.tiles_c, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c0 = (chain % a.tiles_c) * 32 * V, c = c0 + lane * V, cc = min(c, a.D - V);
  const bool on = c < a.D;  // D is a multiple of V
  const T *x = static_cast<const T *>(a.x) + b * a.xb + cc;
  const T *gate = static_cast<const T *>(a.gate) + b * a.gb + cc;
  T *out = static_cast<T *>(a.out) + b * a.ob + cc;
  const int span = a.cs * kTile, tiles = (a.L + kTile - 1) / kTile;
  const int off = rank * kTile + warp * kTok;
  uint32_t *gw = &sh.gate[warp][0][lane];
  constexpr uint32_t kBox = sizeof(sh.gate[0]);
  auto fetch_gate = [&](int64_t base) {
    const int64_t t0 = min(base + off, (int64_t)a.L - 1);
    if constexpr (TMA) {
      if (lane == 0) {
        mbar_arrive_expect_tx(&sh.gate_bar[warp], kBox);
        box_load(gw, &maps.gate, c0, (int)min(base + off, (int64_t)a.L), b, &sh.gate_bar[warp]);
      }
    } else {
      stage<T, V>(gw, at(gate, t0, a.gt), a.gt, (int)max((int64_t)0, min((int64_t)kTok, a.L - (base + off))));
    }
  };
  auto fetch_x = [&](int64_t base, int buf) {
    const int64_t t0 = min(base + off, (int64_t)a.L - 1);
    if constexpr (TMA) {
      if (lane == 0) {
        bulk_wait_read_all();  // the outputs staged in these slots have been read
        mbar_arrive_expect_tx(&sh.x_bar[warp], kBox);
        box_load(&sh.x[0][buf][warp][0][0], &maps.x, c0, (int)min(base + off, (int64_t)a.L), b, &sh.x_bar[warp]);
      }
    } else {
      stage<T, V>(&sh.x[0][buf][warp][0][lane], at(x, t0, a.xt), a.xt,
                  (int)max((int64_t)0, min((int64_t)kTok, a.L - (base + off))));
      stage_commit();
    }
  };
  F h = all_<F>(0.f);
  if (on && a.h0) load_state(a.h0 + (int64_t)b * a.D + c, h);
  scan_start(sh, a.cs);
  fetch_gate(0);
  fetch_x(0, 0);
  int buf = 0, phase = 0;
  bool alive = true;
  for (int64_t base = 0; base < a.L; base += span, buf ^= 1, ++phase) {
    const int64_t t0 = base + off;
    const int n = (int)max((int64_t)0, min((int64_t)kTok, a.L - t0));
    uint32_t *xw = &sh.x[0][buf][warp][0][lane];
    F ta[kTok], td[kTok];
    const bool more = base + span < a.L;
    if constexpr (TMA) {
      if (alive) alive = mbar_wait(&sh.gate_bar[warp], phase & 1, kWaitNs);
    } else {
      stage_wait();
    }
    const Product<T, MODE, F> product = load_gates<T, V, MODE>(gw, n, ta, td);
    if constexpr (TMA) {
      __syncwarp();  // every lane has its gates
      if (more && alive) fetch_gate(base + span);
      if (alive) alive = mbar_wait(&sh.x_bar[warp], phase & 1, kWaitNs);
    } else if (more) {
      fetch_gate(base + span);
      fetch_x(base + span, buf ^ 1);
    }
    Map<F> own;
    product.get(own.a, sh.wn[warp][lane]);
    own.H = reduce_tokens<T, V, MODE, kKeep>(xw, ta, td);
    sh.wmap[warp][lane] = own;
    if (TMA && more && alive) fetch_x(base + span, buf ^ 1);
    __syncthreads();
    if (warp == kWarps - 1) {
      Map<F> r = {all_<F>(1.f), all_<F>(0.f)};
      F rn = all_<F>(0.f);
#pragma unroll
      for (int j = 0; j < kWarps; ++j) {
        const Map<F> w = sh.wmap[j][lane];
        sh.wmap[j][lane] = r;
        follow(r, rn, w, sh.wn[j][lane]);
      }
      r.a = marked(r.a, rn);
      F in = h;
      if (a.cs > 1) {
        if (alive) {
          if (lane == 0) mbar_arrive_expect_tx(&sh.bar[buf], (uint32_t)(a.cs * sizeof(sh.bmap[0][0])));
          for (int k = 0; k < a.cs; ++k)
            cluster_send(peer_addr(&sh.bmap[buf][rank][lane], k), peer_addr(&sh.bar[buf], k), r.a, r.H);
          alive = cluster_wait(&sh.bar[buf], phase >> 1 & 1);
        }
#pragma unroll 4
        for (int k = 0; k < a.cs; ++k) {
          if (k == rank) in = h;
          h = apply_marked(sh.bmap[buf][k][lane], h);
        }
      } else {
        h = apply_marked(r, h);
      }
      sh.carry[lane] = in;
      const int64_t tile = base / kTile + rank;
      if (a.saved && on && tile < tiles) store_state(a.saved + ((int64_t)b * tiles + tile) * a.D + c, in);
    }
    __syncthreads();
    F in = apply(sh.wmap[warp][lane], sh.carry[lane]);
    const int lim = on ? n : 0;
    T *o = at(out, t0, a.ot);
#pragma unroll
    for (int i = 0; i < kTok; ++i) {
      in = kKeep ? fma_(ta[i], in, td[i]) : step_<MODE>(ta[i], td[i], in, Lane<T, V>::get(xw[i * 32]));
      if constexpr (TMA)
        Lane<T, V>::store(reinterpret_cast<T *>(xw + i * 32), in);  // over the x that it took
      else if (i < lim)
        Lane<T, V>::store(token(o, i, a.ot), in);
    }
    if constexpr (TMA) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0 && n > 0 && alive) {
        box_store(&maps.out, &sh.x[0][buf][warp][0][0], c0, (int)t0, b);
        bulk_commit_group();
      }
    }
  }
  if (TMA && lane == 0) bulk_wait_all();
  scan_end<TMA>(sh, alive, a.cs, a.err);
  if (on && rank == 0 && warp == kWarps - 1) store_state(a.hL + (int64_t)b * a.D + c, h);
}

// ---------------------------------------------------------------- backward
// The same walk from the end of the sequence.  The states before each token come from the
// saved state of the tile and the maps of the warps before; the gradient q that flows to
// earlier tokens follows an affine map too, q -> a q + Q with the same a.
template <typename T, int V, int MODE, bool TMA>
__global__ void __launch_bounds__(kThreads, 2)
scan_bwd_kernel(const ScanArgs a, const __grid_constant__ ScanMaps maps) {
  using F = typename Lane<T, V>::F;
  extern __shared__ __align__(128) unsigned char smem[];
  auto &sh = *reinterpret_cast<ScanSharedBwd<F> *>(smem);
  const int rank = blockIdx.x % a.cs, chain = blockIdx.x / a.cs;
  const int b = chain / a.tiles_c, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c0 = (chain % a.tiles_c) * 32 * V, c = c0 + lane * V, cc = min(c, a.D - V);
  const bool on = c < a.D;
  const T *x = static_cast<const T *>(a.x) + b * a.xb + cc;
  const T *gate = static_cast<const T *>(a.gate) + b * a.gb + cc;
  const T *dout = static_cast<const T *>(a.dout) + b * a.ob + cc;
  T *dx = static_cast<T *>(a.dx) + (int64_t)b * a.L * a.D + cc;
  T *dg = static_cast<T *>(a.dgate) + (int64_t)b * a.L * a.D + cc;
  const int span = a.cs * kTile, tiles = (a.L + kTile - 1) / kTile;
  const int off = rank * kTile + warp * kTok;
  uint32_t *gw = &sh.gate[warp][0][lane];
  constexpr uint32_t kBox = sizeof(sh.gate[0]);
  auto fetch_gate = [&](int64_t base) {
    const int64_t t0 = min(base + off, (int64_t)a.L - 1);
    if constexpr (TMA) {
      if (lane == 0) {
        mbar_arrive_expect_tx(&sh.gate_bar[warp], kBox);
        box_load(gw, &maps.gate, c0, (int)min(base + off, (int64_t)a.L), b, &sh.gate_bar[warp]);
      }
    } else {
      stage<T, V>(gw, at(gate, t0, a.gt), a.gt, (int)max((int64_t)0, min((int64_t)kTok, a.L - (base + off))));
    }
  };
  auto fetch_x = [&](int64_t base, int buf) {
    const int64_t t0 = min(base + off, (int64_t)a.L - 1);
    if constexpr (TMA) {
      if (lane == 0) {
        const int t = (int)min(base + off, (int64_t)a.L);
        bulk_wait_read_all();  // the gradients staged in these slots have been read
        mbar_arrive_expect_tx(&sh.x_bar[warp], 2 * kBox);
        box_load(&sh.x[0][buf][warp][0][0], &maps.x, c0, t, b, &sh.x_bar[warp]);
        box_load(&sh.x[1][buf][warp][0][0], &maps.out, c0, t, b, &sh.x_bar[warp]);
      }
    } else {
      const int n = (int)max((int64_t)0, min((int64_t)kTok, a.L - (base + off)));
      stage<T, V>(&sh.x[0][buf][warp][0][lane], at(x, t0, a.xt), a.xt, n);
      stage<T, V>(&sh.x[1][buf][warp][0][lane], at(dout, t0, a.ot), a.ot, n);
      stage_commit();
    }
  };
  const int64_t last = (int64_t)(a.L - 1) / span * span;
  F q = all_<F>(0.f);
  if (on && a.dhL) load_state(a.dhL + (int64_t)b * a.D + c, q);
  scan_start(sh, a.cs);
  fetch_gate(last);
  fetch_x(last, 0);
  int buf = 0, phase = 0;
  bool alive = true;
  for (int64_t base = last; base >= 0; base -= span, buf ^= 1, ++phase) {
    const int64_t t0 = base + off;
    const int n = (int)max((int64_t)0, min((int64_t)kTok, a.L - t0));
    uint32_t *xw = &sh.x[0][buf][warp][0][lane], *yw = &sh.x[1][buf][warp][0][lane];
    F in = all_<F>(0.f);  // the state before the tile
    if (warp == 0 && on && base + rank * kTile < a.L)
      load_state(a.saved + ((int64_t)b * tiles + base / kTile + rank) * a.D + c, in);
    F ta[kTok], td[kTok];
    const bool more = base > 0;
    if constexpr (TMA) {
      if (alive) alive = mbar_wait(&sh.gate_bar[warp], phase & 1, kWaitNs);
    } else {
      stage_wait();
    }
    const Product<T, MODE, F> product = load_gates<T, V, MODE>(gw, n, ta, td);
    if constexpr (TMA) {
      __syncwarp();  // every lane has its gates
      if (more && alive) fetch_gate(base - span);
      if (alive) alive = mbar_wait(&sh.x_bar[warp], phase & 1, kWaitNs);
    } else if (more) {
      fetch_gate(base - span);
      fetch_x(base - span, buf ^ 1);
    }
    Map<F> own;
    product.get(own.a, sh.wn[warp][lane]);
    own.H = reduce_tokens<T, V, MODE, false>(xw, ta, td);
    sh.wmap[warp][lane] = own;
    F Q = all_<F>(0.f);
#pragma unroll
    for (int i = kTok - 1; i >= 0; --i) {
      Q = mul_(ta[i], add_(Q, Lane<T, V>::get(yw[i * 32])));
    }
    sh.wq[warp][lane] = Q;
    __syncthreads();
    if (warp == 0) {
      // in the place of each warp's maps the state before it and the map of the warps behind it
#pragma unroll
      for (int j = 0; j < kWarps; ++j) {
        const Map<F> w = sh.wmap[j][lane];
        sh.wmap[j][lane].H = in;
        in = apply(w, in);
      }
      Map<F> r = {all_<F>(1.f), all_<F>(0.f)};
      F rn = all_<F>(0.f);
#pragma unroll
      for (int j = kWarps - 1; j >= 0; --j) {
        const Map<F> w = {sh.wmap[j][lane].a, sh.wq[j][lane]};
        sh.wmap[j][lane].a = r.a;
        sh.wq[j][lane] = r.H;
        follow(r, rn, w, sh.wn[j][lane]);
      }
      r.a = marked(r.a, rn);
      F qin = q;
      if (a.cs > 1) {
        if (alive) {
          if (lane == 0) mbar_arrive_expect_tx(&sh.bar[buf], (uint32_t)(a.cs * sizeof(sh.bmap[0][0])));
          for (int k = 0; k < a.cs; ++k)
            cluster_send(peer_addr(&sh.bmap[buf][rank][lane], k), peer_addr(&sh.bar[buf], k), r.a, r.H);
          alive = cluster_wait(&sh.bar[buf], phase >> 1 & 1);
        }
#pragma unroll 4
        for (int k = a.cs - 1; k >= 0; --k) {
          if (k == rank) qin = q;
          q = apply_marked(sh.bmap[buf][k][lane], q);
        }
      } else {
        q = apply_marked(r, q);
      }
      sh.carry[lane] = qin;
    }
    __syncthreads();
    if (TMA && more && alive) fetch_x(base - span, buf ^ 1);
    F qi = apply(Map<F>{sh.wmap[warp][lane].a, sh.wq[warp][lane]}, sh.carry[lane]);
    in = sh.wmap[warp][lane].H;
    // backwards over the tokens; the states before them are run forwards again, half of the
    // tokens at a time (registers)
    constexpr int kHalf = kTok / 2;
    const int lim = on ? n : 0, st = a.D * (int)sizeof(T);
    T *px = at(dx, t0, st), *pg = at(dg, t0, st);
    F mid = in;
#pragma unroll
    for (int i = 0; i < kHalf; ++i) mid = step_<MODE>(ta[i], td[i], mid, Lane<T, V>::get(xw[i * 32]));
#pragma unroll
    for (int half = 1; half >= 0; --half) {
      // what q times is the gate's gradient: the state before the token, in sigmoid mode d (h - x),
      // which single values form at the end (registers: 3 x 4000 x 777 bf16 99 -> 91 us)
      constexpr bool kDiff = MODE == DP_SCAN_SIGMOID && V == 2;
      F hb[kHalf], h = half ? mid : in;
#pragma unroll
      for (int k = 0; k < kHalf; ++k) {
        const int i = half * kHalf + k;
        const F xv = kDiff || k + 1 < kHalf ? Lane<T, V>::get(xw[i * 32]) : h;
        hb[k] = kDiff ? mul_(td[i], fma_(xv, all_<F>(-1.f), h)) : h;
        if (k + 1 < kHalf) h = step_<MODE>(ta[i], td[i], h, xv);
      }
#pragma unroll
      for (int k = kHalf - 1; k >= 0; --k) {
        const int i = half * kHalf + k;
        const F p = add_(qi, Lane<T, V>::get(yw[i * 32]));
        qi = mul_(ta[i], p);
        F ox = p, og = mul_(qi, hb[k]);
        if constexpr (MODE == DP_SCAN_SIGMOID) {
          ox = mul_(p, td[i]);
          if (!kDiff) og = mul_(qi, mul_(td[i], fma_(Lane<T, V>::get(xw[i * 32]), all_<F>(-1.f), hb[k])));
        }
        if constexpr (TMA) {  // over the dout and the x that they took
          Lane<T, V>::store(reinterpret_cast<T *>(yw + i * 32), ox);
          Lane<T, V>::store(reinterpret_cast<T *>(xw + i * 32), og);
        } else if (i < lim) {
          Lane<T, V>::store(token(px, i, st), ox);
          Lane<T, V>::store(token(pg, i, st), og);
        }
      }
    }
    if constexpr (TMA) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0 && n > 0 && alive) {
        box_store(&maps.dx, &sh.x[1][buf][warp][0][0], c0, (int)t0, b);
        box_store(&maps.dgate, &sh.x[0][buf][warp][0][0], c0, (int)t0, b);
        bulk_commit_group();
      }
    }
  }
  if (TMA && lane == 0) bulk_wait_all();
  scan_end<TMA>(sh, alive, a.cs, a.err);
  if (on && rank == 0 && warp == 0 && a.dh0) store_state(a.dh0 + (int64_t)b * a.D + c, q);
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
  const float g = to_f32(gate[b * gs + c]), xv = to_f32(x[b * xs + c]), h = state[i];
  // the state goes on from call to call, so an open gate's 1 - a counts here
  float r, ta, td;
  gate_<float, MODE>(g, ta, td);
  if (MODE == DP_SCAN_SIGMOID)
    r = ta < 0.5f ? fmaf(ta, h, td * xv) : fmaf(td, xv - h, h);
  else
    r = fabsf(g) < 0.6931472f ? h + fmaf(expm1f(g), h, xv) : fmaf(ta, h, xv);
  state_out[i] = r;
  out[b * os + c] = from_f32<T>(r);
}

// Blocks of a cluster.  Smaller clusters wait less for one another, but a sequence's chain of
// spans has to be split until about 1.7 blocks an SM run; sizes that are no power of two pack
// badly into the GPU's processor clusters.  Measured (us forward, backward at 2 / 4 / 8 / 9 / 16
// blocks): 32 chains x 32768 tokens bf16 226, 289 / 119, 162 / 84, 121 / 93, 180 / 99, 170;
// 128 chains x 8192 tokens bf16 78, 116 / 94, 123 / 83, 132 / 87, 146 / 103, 172, in sigmoid mode
// 86, 132 / 91, 136 / 102, 148 / 113, 162 / 138, 191; 4 chains x 65536 tokens bf16 439, 557 / 228,
// 292 / 125, 158 / 115, 144 / 74, 93.
int scan_cluster(int L, int64_t chains) {
  int cs = 1;
  while (cs < kMaxCluster && cs * kTile < L && chains * cs < 256) cs *= 2;
  return cs;
}

template <void (*KERN)(const ScanArgs, const ScanMaps), size_t SMEM>
int scan_launch(const ScanArgs &a, const ScanMaps &maps, cudaStream_t st, const char *what) {
  static thread_local bool opted[64] = {};  // shared memory and 16-block clusters: opt in once
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !opted[dev])) {
    e = cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(KERN, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess && dev < 64) opted[dev] = true;
  }
  if (e == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((int64_t)a.B * a.tiles_c * a.cs));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = a.cs;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, KERN, a, maps);
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(DP_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
  }
  return check_launch(what);
}

// Fills in the strides ({sb, st} of x, gate and out or dout); false where a token stride does
// not fit the kernels' 32 bits of bytes.
bool scan_strides(ScanArgs &a, const int64_t *s, int size) {
  int64_t t[3];
  for (int i = 0; i < 3; ++i) {
    t[i] = s[2 * i + 1] * size;
    if (s[2 * i + 1] > (1 << 28) || s[2 * i + 1] < -(1 << 28)) return false;
  }
  a.xb = s[0], a.gb = s[2], a.ob = s[4], a.xt = (int)t[0], a.gt = (int)t[1], a.ot = (int)t[2];
  return a.D <= 1 << 28;
}

// Channel pairs of 16-bit values can be moved as 4-byte words.
template <typename... P>
bool scan_pairs(int D, const int64_t *s, P... ptrs) {
  if (D % 2) return false;
  for (int i = 0; i < 6; ++i)
    if (s[i] % 2) return false;
  const void *ps[] = {ptrs...};
  for (const void *p : ps)
    if (reinterpret_cast<uintptr_t>(p) & 3) return false;
  return true;
}

// The map of a (B, L, D) tensor with byte strides sb, st and unit channel stride: boxes of kTok
// tokens by 32 words.  False where its alignment does not allow bulk tensor copies.
template <typename T>
bool scan_map(CUtensorMap *m, const void *p, const ScanArgs &a, int64_t sb, int64_t st) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (a.B == 1) sb = st * a.L;
  if (!enc || reinterpret_cast<uintptr_t>(p) % 16 || sb % 16 || st % 16 || st < a.D * (int64_t)sizeof(T) || sb < st ||
      sb >= (1ll << 40))
    return false;
  const cuuint64_t dims[3] = {(cuuint64_t)a.D, (cuuint64_t)a.L, (cuuint64_t)a.B};
  const cuuint64_t strides[2] = {(cuuint64_t)st, (cuuint64_t)sb};
  const cuuint32_t box[3] = {128 / sizeof(T), kTok, 1}, one[3] = {1, 1, 1};
  const CUtensorMapDataType type = std::is_same_v<T, float>            ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : std::is_same_v<T, __nv_bfloat16> ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                      : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return enc(m, type, 3, const_cast<void *>(p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool BWD, typename T, int V, bool TMA>
int scan_run_mode(const ScanArgs &a, const ScanMaps &maps, int mode, cudaStream_t st, const char *what) {
  using F = typename Lane<T, V>::F;
  if constexpr (BWD) {
    constexpr size_t kSmem = sizeof(ScanSharedBwd<F>);
    return mode == DP_SCAN_SIGMOID ? scan_launch<scan_bwd_kernel<T, V, DP_SCAN_SIGMOID, TMA>, kSmem>(a, maps, st, what)
                                   : scan_launch<scan_bwd_kernel<T, V, DP_SCAN_DECAY, TMA>, kSmem>(a, maps, st, what);
  } else {
    constexpr size_t kSmem = sizeof(ScanShared<F, 1>);
    return mode == DP_SCAN_SIGMOID ? scan_launch<scan_fwd_kernel<T, V, DP_SCAN_SIGMOID, TMA>, kSmem>(a, maps, st, what)
                                   : scan_launch<scan_fwd_kernel<T, V, DP_SCAN_DECAY, TMA>, kSmem>(a, maps, st, what);
  }
}

template <bool BWD, typename T, int V>
int scan_run(ScanArgs a, int mode, cudaStream_t st, const char *what) {
  a.tiles_c = (a.D + 32 * V - 1) / (32 * V);
  a.cs = scan_cluster(a.L, (int64_t)a.B * a.tiles_c);
  a.err = device_error_ptr();
  DP_REQUIRE(a.err, DP_ERR_CUDA, std::string(what) + ": device error word unavailable");
  DP_REQUIRE((int64_t)a.B * a.tiles_c * a.cs < (1ll << 31), DP_ERR_UNSUPPORTED,
             std::string(what) + ": too many channels");
  ScanMaps maps = {};
  if constexpr (sizeof(T) * V == 4) {
    const int64_t e = sizeof(T), dense = a.D * e;
    bool tma = scan_map<T>(&maps.x, a.x, a, a.xb * e, a.xt) && scan_map<T>(&maps.gate, a.gate, a, a.gb * e, a.gt) &&
               scan_map<T>(&maps.out, BWD ? a.dout : a.out, a, a.ob * e, a.ot);
    if (BWD) tma = tma && scan_map<T>(&maps.dx, a.dx, a, dense * a.L, dense) &&
                   scan_map<T>(&maps.dgate, a.dgate, a, dense * a.L, dense);
    if (tma) return scan_run_mode<BWD, T, V, true>(a, maps, mode, st, what);
  }
  return scan_run_mode<BWD, T, V, false>(a, maps, mode, st, what);
}

template <bool BWD>
int scan_dispatch(const ScanArgs &a, int dtype, int mode, bool pairs, cudaStream_t st, const char *what) {
  if (dtype == DP_F32) return scan_run<BWD, float, 1>(a, mode, st, what);
  if (dtype == DP_BF16)
    return pairs ? scan_run<BWD, __nv_bfloat16, 2>(a, mode, st, what) : scan_run<BWD, __nv_bfloat16, 1>(a, mode, st, what);
  return pairs ? scan_run<BWD, __half, 2>(a, mode, st, what) : scan_run<BWD, __half, 1>(a, mode, st, what);
}

// (B, D) values of `size` bytes, rows `row` bytes apart.
struct Rows {
  const void *p;
  int64_t row, size;
};
// An output may lie on another tensor element for element (a thread reads its channel of all inputs
// before it writes it), but share no memory with it otherwise.
bool scan_clash(const Rows &o, const Rows &t, int B, int D) {
  const int64_t p = (int64_t)reinterpret_cast<uintptr_t>(o.p), q = (int64_t)reinterpret_cast<uintptr_t>(t.p);
  const int64_t pw = o.size * D, qw = t.size * D, pr = (B - 1) * o.row, qr = (B - 1) * t.row;
  if (p == q && o.size == t.size && pr == qr) return false;
  if (p + std::max<int64_t>(pr, 0) + pw <= q + std::min<int64_t>(qr, 0) ||
      q + std::max<int64_t>(qr, 0) + qw <= p + std::min<int64_t>(pr, 0))
    return false;
  if (B == 1 || o.row != t.row || o.row == 0) return true;
  // slices of one buffer's rows lie between one another
  const int64_t row = std::abs(o.row), off = ((q - p) % row + row) % row;
  return off < pw || off + qw > row;
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
  DP_REQUIRE(L <= 1 << 30, DP_ERR_UNSUPPORTED, "dp_scan_fwd: L must be <= 2^30");
  ScanArgs a = {};
  a.x = x, a.gate = gate, a.h0 = state_in, a.hL = state_out, a.saved = saved, a.out = out;
  a.B = B, a.L = L, a.D = D;
  DP_REQUIRE(scan_strides(a, strides, (int)dtype_size(dtype)), DP_ERR_UNSUPPORTED,
             "dp_scan_fwd: token stride too large");
  return scan_dispatch<false>(a, dtype, mode, scan_pairs(D, strides, x, gate, (const void *)out), st, "dp_scan_fwd");
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
  DP_REQUIRE(L <= 1 << 30, DP_ERR_UNSUPPORTED, "dp_scan_bwd: L must be <= 2^30");
  ScanArgs a = {};
  a.x = x, a.gate = gate, a.dout = grad_out, a.saved = const_cast<float *>(saved), a.dhL = grad_state_out;
  a.dx = grad_x, a.dgate = grad_gate, a.dh0 = grad_state_in;
  a.B = B, a.L = L, a.D = D;
  DP_REQUIRE(scan_strides(a, strides, (int)dtype_size(dtype)), DP_ERR_UNSUPPORTED,
             "dp_scan_bwd: token stride too large");
  return scan_dispatch<true>(a, dtype, mode,
                             scan_pairs(D, strides, x, gate, grad_out, (const void *)grad_x, (const void *)grad_gate),
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
  const int64_t e = (int64_t)dtype_size(dtype);
  const Rows outs[] = {{state_out, 4ll * D, 4}, {out, strides[2] * e, e}};
  const Rows ins[] = {outs[1], {state_in, 4ll * D, 4}, {x, strides[0] * e, e}, {gate, strides[1] * e, e}};
  for (int k = 0; k < 2; ++k)
    for (int j = k; j < 4; ++j)
      DP_REQUIRE(!scan_clash(outs[k], ins[j], B, D), DP_ERR_INVALID_ARGUMENT,
                 "dp_scan_step: state_out or out overlaps another tensor");
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
