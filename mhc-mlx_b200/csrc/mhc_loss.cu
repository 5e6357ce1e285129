// Losses on logits for preference and policy tuning, with their gradients.
//
//   m_t = max_v x[t, v],  e_t = exp(x[t, y_t] - m_t),
//   R_t = sum_{v != y_t} exp(x[t, v] - m_t),  S_t = R_t + e_t
//   logp_t = ln(e_t / S_t)                              (0 where y_t is ignored)
//   dx[t, v] = -c_t exp(x[t, v] - m_t) / S_t,  dx[t, y_t] = c_t R_t / S_t
// The target stays out of the sum: 1 - p of a token that the model is sure of
// is R / S to full precision, and its logp is -ln(1 + R).
//
// c_t = d loss / d logp_t comes from the loss:
//   preference  R_s = sum_{t in s} (logp_t - ref_t),  z_b = beta (R_2b - R_2b+1),
//               loss = 1/D sum_b (1 - e) softplus(-z_b) + e softplus(z_b)
//   policy      r = exp(logp - old),  k = expm1(ref - logp) - (ref - logp),
//               loss = 1/D sum_t kl k - min(r A, clip(r, 1 - lo, 1 + hi) A)
// Everything between the logits and their gradient is fp32 (sums over tokens
// fp64); the gradient is rounded once, to the logits' type.
//
// What bounds them is the logits' traffic: T V values in and, for a gradient,
// T V out.  A policy token's c_t depends on its own row alone, so its row
// stays in registers between the reduction and the gradient (k_rows with
// POLICY: one read, one write).  A preference pair's c_t needs every token of
// both sequences, so its logits are read twice (k_rows for the sums,
// k_preference, k_logits_grad), the second time from the last row to the first:
// what the first pass left in L2 is read again before it is evicted.
//
// Differences (x - m) are formed before the scaling by log2(e): a row of the
// type's lowest values is a uniform distribution, and a masked (-inf) logit
// contributes exactly 0.  A row without a finite logit, or with a NaN or
// +inf, gives NaN; a target outside [0, V) too.
#include <math_constants.h>

#include "mhc_common.cuh"
#include "mhc_internal.h"

namespace mhc {
namespace {

constexpr int kNT = 256;        // threads of a block
constexpr int kMaxCluster = 8;  // blocks that share a row: the portable cluster size
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLog2eLow = (float)(1.4426950408889634 - (double)kLog2e);

// ---------------------------------------------------------------- pieces --
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The hardware's 2^x is low by 5.0e-8 on average over 4 M points of (-20, 0]
// (largest error 1.4e-7).  A sum over a vocabulary keeps that mean, and a
// sequence's summed log probabilities would collect it token by token, so the
// exponents that go into a sum are raised, before their rounding.  A term meets
// it up to three times (its own exponential, its thread's and its warp's
// rescaling, the last two exact for those that hold the maximum), so what is best
// depends on the row: 4.1e-8 each was fitted to normal logits of deviation 2, 4000
// rows of 32000 (5.0e-8 left their sums 2.6e-8 high, none 9e-8 low).  Mean error
// of ln S with it, at 512 to 131072 logits in fp32, bf16 and fp16: deviation 2
// 7e-9 at most, 1 2e-8 high, 5 up to 4.5e-8 low, even over (-20, 0) up to 6.3e-8
// high, one logit 12 above the rest 5e-9, flat rows 0.
constexpr float kExp2Mean = 4.1e-8f * kLog2e;
// exp of a difference a - b <= 0 of finite values, or 0 for a = -inf.
__device__ __forceinline__ float exp_diff(float a, float b) {
  const float d = a - b;
  return ex2(fmaf(d, kLog2e, fmaf(d, kLog2eLow, kExp2Mean)));
}

// (a - m) log2(e), (b - m) log2(e) as packed two-lane operations, then 2^.
template <bool Fine = false>
__device__ __forceinline__ float2 exp2_diff(float a, float b, float neg_m) {
  float x, y;
  if constexpr (Fine)
    asm("{\n .reg .b64 p, q, r, s;\n mov.b64 p, {%2, %3};\n mov.b64 q, {%4, %4};\n"
        " add.rn.f32x2 p, p, q;\n mov.b64 r, {%5, %5};\n mov.b64 s, {%6, %6};\n"
        " mov.b64 q, {%7, %7};\n fma.rn.f32x2 q, p, s, q;\n fma.rn.f32x2 p, p, r, q;\n"
        " mov.b64 {%0, %1}, p;\n}"
        : "=f"(x), "=f"(y)
        : "f"(a), "f"(b), "f"(neg_m), "f"(kLog2e), "f"(kLog2eLow), "f"(kExp2Mean));
  else
    asm("{\n .reg .b64 p, q, r;\n mov.b64 p, {%2, %3};\n mov.b64 q, {%4, %4};\n"
        " add.rn.f32x2 p, p, q;\n mov.b64 r, {%5, %5};\n mul.rn.f32x2 p, p, r;\n"
        " mov.b64 {%0, %1}, p;\n}"
        : "=f"(x), "=f"(y)
        : "f"(a), "f"(b), "f"(neg_m), "f"(kLog2e));
  return make_float2(ex2(x), ex2(y));
}

__device__ __forceinline__ float2 unpack2(unsigned w, bf16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 unpack2(unsigned w, f16) {
  return __half22float2(*reinterpret_cast<__half2*>(&w));
}

// A 16-byte vector of T: VE values, visited as pairs.
template <typename T> struct Vec {
  static constexpr int VE = 16 / (int)sizeof(T);
  uint4 u;
  __device__ __forceinline__ void fill_neg_inf() {
    const unsigned w = sizeof(T) == 4 ? 0xff800000u
                                      : (std::is_same<T, bf16>::value ? 0xff80ff80u : 0xfc00fc00u);
    u = make_uint4(w, w, w, w);
  }
  __device__ __forceinline__ float2 pair(int i) const {  // i in [0, VE / 2)
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
    if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    else return unpack2(w[i], T());
  }
};

// Largest of NV vectors (NaN is passed over: the sum keeps it).
template <typename T, int NV>
__device__ __forceinline__ float max_of(const Vec<T> (&r)[NV]) {
  if constexpr (sizeof(T) == 4) {
    float m = -CUDART_INF_F;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      m = fmaxf(m, fmaxf(fmaxf(r[i].pair(0).x, r[i].pair(0).y), fmaxf(r[i].pair(1).x, r[i].pair(1).y)));
    return m;
  } else {
    using P = typename std::conditional<std::is_same<T, bf16>::value, __nv_bfloat162, __half2>::type;
    P m = *reinterpret_cast<const P*>(&r[0].u.x);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const unsigned w[4] = {r[i].u.x, r[i].u.y, r[i].u.z, r[i].u.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) m = __hmax2(m, *reinterpret_cast<const P*>(&w[k]));
    }
    const float2 f = unpack2(*reinterpret_cast<unsigned*>(&m), T());
    return fmaxf(f.x, f.y);
  }
}

// sum exp(x - m) over the first n of NV vectors, m finite.  log2(e) to 48 bits here: with 24
// every term is off the same way (1e-8 of the difference), and a sequence's
// summed log probabilities keep what their errors have in common.
template <typename T, int NV>
__device__ __forceinline__ float sum_of(const Vec<T> (&r)[NV], float m, int n) {
  float s0 = 0.f, s1 = 0.f;  // added in pairs
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (i >= NV / 2 && i >= n) break;  // a branch for each of the first half costs more than it saves
#pragma unroll
    for (int k = 0; k < Vec<T>::VE / 2; ++k) {
      const float2 f = r[i].pair(k);
      const float2 e = exp2_diff<true>(f.x, f.y, -m);
      asm("{\n .reg .b64 p, q;\n mov.b64 p, {%0, %1};\n mov.b64 q, {%2, %3};\n"
          " add.rn.f32x2 p, p, q;\n mov.b64 {%0, %1}, p;\n}"
          : "+f"(s0), "+f"(s1)
          : "f"(e.x), "f"(e.y));
    }
  }
  return s0 + s1;
}

// A running (max, sum): sum = sum exp(x - max) over what it has seen; max is
// -inf and sum 0 before any value above -inf.
struct MaxSum {
  float m, s;
};
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b) {
  const float m = fmaxf(a.m, b.m);
  if (m == -CUDART_INF_F) return {m, a.s + b.s};  // 0, or NaN kept
  return {m, (a.m == -CUDART_INF_F ? a.s : a.s * exp_diff(a.m, m)) +
                 (b.m == -CUDART_INF_F ? b.s : b.s * exp_diff(b.m, m))};
}
// The largest of a warp's values, by the integers that order as they do.
__device__ __forceinline__ float warp_max(float m) {
  const int i = __float_as_int(m), k = i ^ ((i >> 31) & 0x7fffffff);
  const int t = __reduce_max_sync(0xffffffffu, k);
  return __int_as_float(t ^ ((t >> 31) & 0x7fffffff));
}
// All of a warp's (max, sum), on every lane: one exponential a lane.
__device__ __forceinline__ MaxSum warp_join(MaxSum v) {
  const float m = warp_max(v.m);
  return {m, warp_sum(v.m == m ? v.s : v.s * exp_diff(v.m, m))};
}

// ------------------------------------------------------------- clusters --
__device__ __forceinline__ unsigned cluster_rank() {
  unsigned r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ float2 peer_float2(const float2* own, unsigned rank) {
  unsigned a;
  float2 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(own)), "r"(rank));
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
}

// Writes v to `own`'s place in another block of the cluster and counts its 8 bytes
// on `bar` there.
__device__ __forceinline__ void send_float2(const float2* own, uint64_t* bar, unsigned rank, float2 v) {
  unsigned a, b;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(own)), "r"(rank));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"(smem_u32(bar)), "r"(rank));
  const uint64_t u = (uint64_t)__float_as_uint(v.x) | (uint64_t)__float_as_uint(v.y) << 32;
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(a), "l"(u),
               "r"(b)
               : "memory");
}
// As mbar_wait, for what other blocks of the cluster have sent.
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, unsigned parity) {
  for (unsigned k = 0; k < (1u << 22); ++k) {
    unsigned ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (ok) return true;
  }
  return false;
}

// (max, sum) of the whole row, on the first warp of every block that shares it:
// each warp's, then the warps' by the first, then the blocks' by the first warp
// of each; the order is fixed.  `k` counts the rows that the block has joined:
// the slots alternate, so that a slot is written again only after a later
// row's barrier.  The blocks of a cluster send their values into each other's
// slots, counted on an mbarrier there: a cluster barrier would first wait for
// the gradient's stores of the row before (8 % of 1000 rows of 50001 fp16 values,
// two blocks each).  A block sends for row k + 2 only after it has everyone's
// values of k + 1, and so after everyone has read those of row k.
template <int NT>
struct RowShared {
  float2 warp[2][NT / 32];
  float2 block[2][kMaxCluster];
  uint64_t got[2];
};
// Before the first join, by all threads of all blocks of the cluster; they end
// with cluster_arrive(); cluster_wait().
template <int NT>
__device__ __forceinline__ void row_shared_init(RowShared<NT>& sh, int cs) {
  if (cs == 1) return;
  if (threadIdx.x == 0) {
    mbar_init(&sh.got[0], 1);
    mbar_init(&sh.got[1], 1);
    mbar_init_fence();
  }
  cluster_arrive();
  cluster_wait();
}
template <int NT>
__device__ __forceinline__ MaxSum row_join(MaxSum v, RowShared<NT>& sh, int cs, unsigned k) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b = k & 1;
  v = warp_join(v);
  if (lane == 0) sh.warp[b][warp] = make_float2(v.m, v.s);
  __syncthreads();
  if (warp == 0) {
    const float2 f = lane < NT / 32 ? sh.warp[b][lane] : make_float2(-CUDART_INF_F, 0.f);
    v = warp_join({f.x, f.y});
    if (cs > 1) {
      if (lane == 0) mbar_arrive_expect_tx(&sh.got[b], 8u * (unsigned)cs);
      if (lane < cs) send_float2(&sh.block[b][cluster_rank()], &sh.got[b], lane, make_float2(v.m, v.s));
      const bool got = mbar_wait_cluster(&sh.got[b], (k >> 1) & 1u);
      const float2 g = lane < cs ? sh.block[b][lane] : make_float2(-CUDART_INF_F, 0.f);
      v = warp_join({g.x, got ? g.y : CUDART_NAN_F});
    }
  }
  return v;
}

// ------------------------------------------------------------------ rows --
// The slice [lo, hi) of a row that one block works on: up to VE - 1 values
// before the first 16-byte boundary, whole vectors, and what is left.
template <typename T>
struct Slice {
  const T* x;  // the row
  int64_t lo;  // first element of the slice
  int head, tail;
  int64_t vecs, body, end;  // elements [body, body + vecs VE) are whole vectors
  __device__ Slice(const T* row, int64_t lo_, int64_t hi) : x(row), lo(lo_) {
    constexpr int VE = Vec<T>::VE;
    const int off = (int)((reinterpret_cast<uintptr_t>(row + lo) / sizeof(T)) % VE);
    int64_t h = (VE - off) % VE;
    if (h > hi - lo) h = hi > lo ? hi - lo : 0;
    head = (int)h;
    body = lo + h;
    vecs = hi > body ? (hi - body) / VE : 0;
    end = body + vecs * VE;
    tail = hi > end ? (int)(hi - end) : 0;
  }
};

// One value as a (max, sum): NaN and +inf leave NaN in the sum.
__device__ __forceinline__ MaxSum one_of(float v) {
  if (v == -CUDART_INF_F) return {v, 0.f};
  return {v == v ? v : -CUDART_INF_F, 1.f + (v - v)};
}
// Values of the unaligned ends, the target's left out: thread i < head has
// one, thread i < tail one.
template <typename T>
__device__ __forceinline__ MaxSum ends_of(const Slice<T>& s, int64_t y) {
  MaxSum a = {-CUDART_INF_F, 0.f};
  const int t = threadIdx.x;
  if (t < s.head && s.lo + t != y) a = one_of(to_f(s.x[s.lo + t]));
  if (t < s.tail && s.end + t != y) a = join(a, one_of(to_f(s.x[s.end + t])));
  return a;
}
// Where the target lies among the slice's vectors: `vec` (-1: not there) and
// the bits of it that it fills.
template <typename T>
struct Hidden {
  int64_t vec;
  uint4 mask;
  __device__ Hidden(const Slice<T>& s, int64_t y) : vec(-1), mask(make_uint4(0, 0, 0, 0)) {
    if (y < s.body || y >= s.end) return;
    const int64_t at = y - s.body;
    vec = at / Vec<T>::VE;
    const int byte = (int)(at - vec * Vec<T>::VE) * (int)sizeof(T);
    const unsigned m = (sizeof(T) == 4 ? 0xffffffffu : 0xffffu) << (8 * (byte & 3));
    mask = make_uint4(byte / 4 == 0 ? m : 0u, byte / 4 == 1 ? m : 0u, byte / 4 == 2 ? m : 0u,
                      byte / 4 == 3 ? m : 0u);
  }
  __device__ __forceinline__ void apply(Vec<T>& v) const {  // the target becomes -inf
    Vec<T> n;
    n.fill_neg_inf();
    v.u = make_uint4((v.u.x & ~mask.x) | (n.u.x & mask.x), (v.u.y & ~mask.y) | (n.u.y & mask.y),
                     (v.u.z & ~mask.z) | (n.u.z & mask.z), (v.u.w & ~mask.w) | (n.u.w & mask.w));
  }
};

// (max, sum) of one thread's NV vectors, those from n on -inf throughout.
template <typename T, int NV>
__device__ __forceinline__ MaxSum vecs_of(const Vec<T> (&r)[NV], int n = NV) {
  const float m = max_of(r);
  // all -inf (or NaN): sum against 0, which gives 0 (or NaN)
  return {m, sum_of(r, m == -CUDART_INF_F ? 0.f : m, n)};
}

// --------------------------------------------------------------- the grids --
struct Rows {  // logits: row t at base + (t / per_batch) batch_stride + (t % per_batch) row_stride
  const void* base;
  int rows, per_batch;  // < 2^28
  int64_t batch_stride, row_stride;
  int V;
  const int64_t* targets;
  int64_t ignore;
};
template <typename T>
__device__ __forceinline__ const T* row_ptr(const Rows& a, int t) {
  const int b = (int)((unsigned)t / (unsigned)a.per_batch);
  return static_cast<const T*>(a.base) + b * a.batch_stride + (t - b * a.per_batch) * a.row_stride;
}
// A target as a class, or what it is instead.
constexpr int kIgnored = -1, kBad = -2;
__device__ __forceinline__ int class_of(const Rows& a, int64_t y) {
  return y == a.ignore ? kIgnored : (y >= 0 && y < a.V) ? (int)y : kBad;
}
template <typename T>
__device__ __forceinline__ float target_logit(const T* x, int64_t y, int64_t V) {
  return (y >= 0 && y < V) ? to_f(x[y]) : CUDART_NAN_F;
}
// A row's record: m, 1 / S, R / S, and logp's low part.  Where rows are worked on in
// order (k_order) the fourth word is instead the i-th row to be worked on, which
// has nothing to do with row i itself, and is left alone.
__device__ __forceinline__ void put_stats(float4* p, float m, float inv_s, float miss) {
  *reinterpret_cast<float2*>(p) = make_float2(m, inv_s);
  reinterpret_cast<float*>(p)[2] = miss;
}
// What a row comes to, from the (max, sum) of all but its target and the
// target's logit.  Without a finite logit, or with a NaN, +inf or a bad
// target, all is NaN.
struct RowEnd {
  float logp, low, m, inv_s, miss;  // logp + low in more digits; miss: 1 - p of the target
};
__device__ __forceinline__ RowEnd row_end(float xt, MaxSum a) {
  const float m = fmaxf(xt, a.m);
  const float r = a.m == m ? a.s : a.s * exp_diff(a.m, m);
  const float e = xt == m ? 1.0f + (m - m) : exp_diff(xt, m);  // NaN where m is not finite
  const float s = r + e, inv = 1.0f / s, bad = s - s;
  // What is summed over a sequence or subtracted from another log probability
  // should not lose logp's last digits to its rounding.
  const double l = xt == m ? -log1p((double)r) : ((double)xt - (double)m) - log((double)s);
  const float logp = (float)l + bad;
  return {logp, isfinite(logp) ? (float)(l - (double)logp) : 0.f, m, inv, r * inv + bad};
}

__device__ __forceinline__ double block_sum_f64(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) s += red[w];
  return s;
}

// ---------------------------------------------------------- values and ends --
// f exp(x - m) of a vector, in T.  log2(e) in 24 bits and no correction here, since
// nothing adds the values up: each is off by |x - m| 1.4e-7 and the hardware's 1.4e-7 of
// itself, which comes to 1.4e-7 of f at most.
template <typename T>
__device__ __forceinline__ uint4 scaled(const Vec<T>& v, float m, float f) {
  unsigned w[4];
#pragma unroll
  for (int k = 0; k < Vec<T>::VE / 2; ++k) {
    const float2 x = v.pair(k);
    const float2 e = exp2_diff(x.x, x.y, -m);
    float a, b;
    asm("{\n .reg .b64 p, q;\n mov.b64 p, {%2, %3};\n mov.b64 q, {%4, %4};\n"
        " mul.rn.f32x2 p, p, q;\n mov.b64 {%0, %1}, p;\n}"
        : "=f"(a), "=f"(b)
        : "f"(e.x), "f"(e.y), "f"(f));
    if constexpr (sizeof(T) == 4) {
      w[2 * k] = __float_as_uint(a);
      w[2 * k + 1] = __float_as_uint(b);
    } else {
      w[k] = pack2_16<T>(a, b);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// Values [from, to) of a vector, one by one (any alignment).
template <typename T>
__device__ __forceinline__ void store_values(T* dst, const uint4& v, int from, int to) {
  const T* h = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int e = 0; e < 16 / (int)sizeof(T); ++e)
    if (e >= from && e < to) dst[e] = h[e];
}
template <typename T, int NT>
__device__ __forceinline__ void zero_slice(T* out, int64_t lo, int64_t hi) {
  const Slice<T> o(out, lo, hi);
  if (threadIdx.x < o.head) out[lo + threadIdx.x] = from_f<T>(0.f);
  uint4* q = reinterpret_cast<uint4*>(out + o.body);
  for (int64_t i = threadIdx.x; i < o.vecs; i += NT) __stcs(q + i, make_uint4(0, 0, 0, 0));
  if (threadIdx.x < o.tail) out[o.end + threadIdx.x] = from_f<T>(0.f);
}

// ------------------------------------------------------------ policy terms --
struct Policy {
  const float* old;
  const float* adv;
  const float* ref;  // null: no KL term
  float clip_lo, clip_hi, kl_coef;
};
struct Token {
  float loss, kl, slope;
};
__device__ __forceinline__ Token policy_token(float logp, float low, float old, float adv, float ref,
                                              const Policy& p) {
  const float r = expf((logp - old) + low);
  const float free = r * adv, held = fminf(fmaxf(r, p.clip_lo), p.clip_hi) * adv;
  Token k;
  // where the two agree (inside the clip) the gradient is the free one's
  k.loss = free <= held ? -free : -held;
  k.slope = free <= held ? -free : 0.f;
  if (free != free) k.loss = k.slope = free;  // comparisons and fminf drop a NaN
  k.kl = 0.f;
  if (p.ref) {
    const float d = (ref - logp) - low, em = expm1f(d);
    k.kl = em - d;
    if (p.kl_coef != 0.f) {
      k.loss += p.kl_coef * k.kl;
      k.slope -= p.kl_coef * em;
    }
  }
  return k;
}

// -------------------------------------------------------- the row pipeline --
// A row's slice as 16-byte granules of memory: the first and the last may hold
// values of its neighbours, which are passed over.
template <typename T>
struct Grains {
  static constexpr int VE = 16 / (int)sizeof(T);
  const uint4* at;   // first granule
  int count;         // granules
  int skip, last;    // values before the slice in the first, of the slice in the last granule
  int bulk0, bulk1;  // granules [bulk0, bulk1) may be copied whole
  int head, tail;    // granules that have others' values too, or -1
  __device__ void set(const T* x, int lo, int hi, uintptr_t span0, uintptr_t span1) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(x + lo), b = reinterpret_cast<uintptr_t>(x + hi);
    const uintptr_t a0 = a & ~(uintptr_t)15, b1 = (b + 15) & ~(uintptr_t)15;
    at = reinterpret_cast<const uint4*>(a0);
    count = hi > lo ? (int)((b1 - a0) >> 4) : 0;
    skip = (int)(a - a0) / (int)sizeof(T);
    last = VE - (int)(b1 - b) / (int)sizeof(T);
    // a granule that reaches past the tensor itself is read value by value
    bulk0 = a0 < span0 ? 1 : 0;
    bulk1 = b1 > span1 ? count - 1 : count;
    if (bulk1 < bulk0) bulk1 = bulk0;
    head = count > 0 && skip != 0 ? 0 : -1;
    tail = count > 0 && last != VE ? count - 1 : -1;
  }
  // The slice's values in granule j are [from(j), to(j)).
  __device__ __forceinline__ int from(int j) const { return j == 0 ? skip : 0; }
  __device__ __forceinline__ int to(int j) const { return j == count - 1 ? last : VE; }
};
template <typename T>
__device__ __forceinline__ unsigned neg_inf_bits() {
  return sizeof(T) == 4 ? 0xff800000u : (std::is_same<T, bf16>::value ? 0xff80u : 0xfc00u);
}
// Value e of a vector <- bits.
template <typename T>
__device__ __forceinline__ void put(uint4& u, int e, unsigned bits) {
  const int byte = e * (int)sizeof(T), w = byte >> 2, sh = 8 * (byte & 3);
  const unsigned m = (sizeof(T) == 4 ? 0xffffffffu : 0xffffu) << sh, v = bits << sh;
  if (w == 0) u.x = (u.x & ~m) | v;
  if (w == 1) u.y = (u.y & ~m) | v;
  if (w == 2) u.z = (u.z & ~m) | v;
  if (w == 3) u.w = (u.w & ~m) | v;
}
// The first n values (Below), or those from n on, become -inf.
template <typename T, bool Below>
__device__ __forceinline__ void trim(uint4& u, int n) {
  Vec<T> inf;
  inf.fill_neg_inf();
  const auto word = [&](unsigned w, int i) {
    const int bits = 8 * (int)sizeof(T) * n - 32 * i;  // of this word, below n
    const unsigned m = bits <= 0 ? 0u : bits >= 32 ? 0xffffffffu : (1u << bits) - 1u;
    return Below ? (w & ~m) | (inf.u.x & m) : (w & m) | (inf.u.x & ~m);
  };
  u = make_uint4(word(u.x, 0), word(u.y, 1), word(u.z, 2), word(u.w, 3));
}
template <typename T>
__device__ __forceinline__ unsigned bits_of(float v) {
  const T t = from_f<T>(v);
  if constexpr (sizeof(T) == 4) return __float_as_uint(t);
  else return (unsigned)*reinterpret_cast<const unsigned short*>(&t);
}

// The order in which rows are worked on (stats[i].w): those that count first,
// then the ignored ones, so that blocks that walk it at a stride have equal
// work (masked prompts come in runs: by row number the busiest block of 8192
// rows, a fifth of them masked, had a quarter more than the mean).  With it 1 / D,
// D the rows that count (0 without any) where inv_d_in is 0, and a cleared ticket.
__global__ void __launch_bounds__(1024)
k_order(const int64_t* __restrict__ targets, int rows, int64_t ignore, float4* __restrict__ stats,
        float inv_d_in, float* __restrict__ inv_d, unsigned* __restrict__ ticket) {
  __shared__ int red[2][32];
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int total = 0;  // rows that count so far
  for (int base = 0, k = 0; base < rows; base += 1024, k ^= 1) {
    const int t = base + threadIdx.x;
    const bool counts = t < rows && targets[t] != ignore;
    const unsigned who = __ballot_sync(0xffffffffu, counts);
    if (lane == 0) red[k][warp] = __popc(who);
    __syncthreads();
    // counts of the warps before this one, and of all
    int v = red[k][lane], before = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += u;
    }
    const int all = __shfl_sync(0xffffffffu, before, 31);
    before = __shfl_sync(0xffffffffu, before - v, warp);
    const int at = total + before + __popc(who & ((1u << lane) - 1u));
    // an ignored row goes to the end, the first of them last
    if (stats && t < rows) stats[counts ? at : rows - 1 - (t - at)].w = __int_as_float(t);
    total += all;
  }
  if (threadIdx.x == 0 && inv_d) {
    *ticket = 0u;
    *inv_d = inv_d_in > 0.f ? inv_d_in : total > 0 ? (float)(1.0 / (double)total) : 0.f;
  }
}

// Rows' statistics, and with POLICY the loss and the gradient, by blocks that
// stay and walk the rows in k_order's order (`ordered`; else by number, where a
// cluster has one row at most), `first + i * stride` for cluster `first`.  A row is
// shared by the cs blocks of a cluster; a block's slice of it is at most
// NT * kNV granules.  The slice of the next row is on its way into shared
// memory (one thread's bulk copy, completing on an mbarrier) while the present
// one is worked on: it moves from shared memory to registers at once (kNV
// vectors a thread), where it stays from the sum to the gradient, and the next
// row's copy starts then.  With POLICY an SM holds 1024 threads at 64 registers
// and 128 KB of slots whatever NT is (512, 256 or 128, by the slice's length),
// about three times what 44 GB/s an SM needs in flight.
//
// Measured, 8192 rows of 32000 bf16 logits (524 MB): loss and gradient with 30 %
// of the rows ignored 181 us (136 us at the copy rate for the other rows in and all
// out; memory and a row's chain from sum to gradient), the sums alone with a fifth
// ignored 88 us (64 us at the copy rate for the others; the exponential unit is 62 %
// busy and the rest of the issue slots' work waits between rows).  A block a row
// that loads its row itself: loss and gradient 224 us.
constexpr int64_t kGrainsMax = 4096;  // 64 KB
template <typename T, int NT>
struct RowSmem {
  RowShared<NT> sh;
  Grains<T> grains[2];
  double red[NT / 32];
  double loss, kl;  // this cluster's sums
  float4 end;       // of the row: m, and -c / S, c R / S, c (with the gradient's scale)
  uint64_t full;
  unsigned last;
};

struct PolicyRun {
  Policy pol;
  float inv_d_in;  // 0: one over the rows that count
  float* inv_d;
  float grad_scale;
  double2* partial;  // a pair of sums a cluster
  float *loss, *kl;
  unsigned* ticket;
};

// Vectors a thread: 8 where they wait for the gradient, 16 in two halves where
// only the sums are wanted (half the threads, so half of what each thread does
// once a row).
template <bool POLICY>
struct RowShape {
  static constexpr int kNV = POLICY ? 8 : 16;
  static constexpr int kThreadsSM = POLICY ? 128 * kPolicyClustersSM : 768;
};
template <typename T, int NT, bool POLICY>
__global__ void __launch_bounds__(NT, RowShape<POLICY>::kThreadsSM / NT)
k_rows(const Rows a, int slice, int cs, int ordered, float* __restrict__ logp, float4* stats,
       float* __restrict__ coef, const PolicyRun run, T* __restrict__ dx) {
  extern __shared__ uint4 slot[];
  __shared__ RowSmem<T, NT> sm;
  constexpr int VE = 16 / (int)sizeof(T);
  constexpr int kNV = RowShape<POLICY>::kNV;
  constexpr int kHold = 8;  // vectors a thread holds at a time
  const int tid = threadIdx.x;
  const int rank = cs > 1 ? (int)cluster_rank() : 0;
  const bool first = rank == 0 && tid == 0;
  const int c0 = blockIdx.x / cs, step = gridDim.x / cs;
  const int lo = min((int64_t)rank * slice, (int64_t)a.V), hi = min((int64_t)lo + slice, (int64_t)a.V);
  if (tid == 0) {
    mbar_init(&sm.full, 1);
    mbar_init_fence();
    sm.loss = sm.kl = 0.0;
  }
  row_shared_init(sm.sh, cs);
  __syncthreads();
  if constexpr (!POLICY) pdl_trigger();

  // Thread 0: the row's slice as granules, for all threads, and its copy.
  const auto fetch = [&](int t, unsigned k) {
    Grains<T>& g = sm.grains[k & 1];
    g.set(row_ptr<T>(a, t), lo, hi, reinterpret_cast<uintptr_t>(row_ptr<T>(a, 0)),
          reinterpret_cast<uintptr_t>(row_ptr<T>(a, a.rows - 1) + a.V));
    const unsigned bytes = (unsigned)(g.bulk1 - g.bulk0) * 16u;
    mbar_arrive_expect_tx(&sm.full, bytes);
    if (bytes) bulk_g2s(slot + g.bulk0, g.at + g.bulk0, bytes, &sm.full);
  };

  bool counted = false;
  if (ordered) {
    pdl_wait();
    counted = true;
  }
  // the i-th row to be worked on; the two after the present one are known ahead,
  // and the next one's target
  const auto row_at = [&](int64_t i) -> int {
    if (i >= a.rows) return -1;
    return ordered ? __float_as_int(reinterpret_cast<const volatile float*>(stats + i)[3]) : (int)i;
  };
  const auto target_of = [&](int t) { return t < 0 ? a.ignore : a.targets[t]; };
  int64_t at = c0;
  int t = row_at(at), tn = row_at(at + step);
  int y = class_of(a, target_of(t));
  int64_t yn = target_of(tn);
  if (tid == 0 && y != kIgnored) fetch(t, 0);
  unsigned joined = 0;
  for (; t >= 0; at += step) {
    const int tnn = row_at(at + 2 * (int64_t)step);
    T* out = dx ? dx + (int64_t)t * a.V : nullptr;
    if (y == kIgnored) {  // the same for the whole cluster
      if (POLICY && !counted) {
        pdl_wait();
        counted = true;
      }
      if (out) zero_slice<T, NT>(out, lo, hi);
      if (first) {
        logp[t] = 0.f;
        put_stats(stats + t, 0.f, 0.f, 0.f);
        if (coef) coef[t] = 0.f;
      }
      if (tid == 0 && yn != a.ignore) {
        fence_proxy_async_smem();
        fetch(tn, joined);
      }
      y = class_of(a, yn);
      t = tn;
      tn = tnn;
      yn = target_of(tn);
      continue;
    }
    float old = 0.f, adv = 0.f, ref = 0.f;  // asked for now, used after the sum
    if (POLICY && tid < 32) {
      old = run.pol.old[t];
      adv = run.pol.adv[t];
      if (run.pol.ref) ref = run.pol.ref[t];
    }
    const bool landed = mbar_wait(&sm.full, joined & 1u);
    const Grains<T>& g = sm.grains[joined & 1];  // set again two rows on
    const int count = g.count, skip = g.skip;
    // the target's granule and its place there
    const int ye = y >= lo && y < hi ? y - lo + skip : -1;
    const int yj = ye >= 0 ? ye / VE : -1;
    float xt;
    if (y == kBad || !landed) xt = CUDART_NAN_F;
    else if (yj >= g.bulk0 && yj < g.bulk1) xt = to_f(reinterpret_cast<const T*>(slot)[ye]);
    else xt = to_f(row_ptr<T>(a, t)[y]);
    const bool mine = yj >= 0 && yj % NT == tid;  // this thread has the target
    Vec<T> r[kHold];
    MaxSum acc = {-CUDART_INF_F, 0.f};
    // unrolled: a loop over the halves is 10 % slower (8192 x 32000 bf16 sums 99 us, 89)
#pragma unroll
    for (int i0 = 0; i0 < kNV; i0 += kHold) {
#pragma unroll
      for (int i = 0; i < kHold; ++i) {
        r[i].fill_neg_inf();
        if (tid + (i0 + i) * NT < count) r[i].u = slot[tid + (i0 + i) * NT];
      }
      if (g.bulk0 != 0 || g.bulk1 != count) {  // value by value, what the copy left out
#pragma unroll
        for (int i = 0; i < kHold; ++i) {
          const int j = tid + (i0 + i) * NT;
          if (j < count && (j < g.bulk0 || j >= g.bulk1)) {
#pragma unroll 1
            for (int e = 0; e < VE; ++e) {
              const bool ours = e >= g.from(j) && e < g.to(j);
              put<T>(r[i].u, e, ours ? bits_of<T>(to_f(reinterpret_cast<const T*>(g.at + j)[e])) : neg_inf_bits<T>());
            }
          }
        }
      }
      // other rows' values at the ends
      if (g.head == 0 && tid == 0 && i0 == 0) trim<T, true>(r[0].u, skip);
      if (g.tail >= 0 && g.tail % NT == tid) {
#pragma unroll
        for (int i = 0; i < kHold; ++i)
          if (g.tail == tid + (i0 + i) * NT) trim<T, false>(r[i].u, g.last);
      }
      if (i0 + kHold >= kNV) {
        __syncthreads();
        // every thread has its part of the slot: the next row may come
        if (tid == 0 && yn != a.ignore) {
          fence_proxy_async_smem();
          fetch(tn, joined + 1);
        }
      }
      if (mine) {
#pragma unroll
        for (int i = 0; i < kHold; ++i)
          if (yj == tid + (i0 + i) * NT) put<T>(r[i].u, ye % VE, neg_inf_bits<T>());
      }
      const int own = (count - tid - i0 * NT + NT - 1) / NT;  // vectors from here on
      acc = kHold == kNV ? vecs_of(r, own) : i0 == 0 ? vecs_of(r) : join(acc, vecs_of(r, own));
    }
    acc = row_join<NT>(acc, sm.sh, cs, joined);
    ++joined;
    if (POLICY && !counted) {
      pdl_wait();  // the count is complete
      counted = true;
    }
    if (tid < 32) {
      const RowEnd e = row_end(xt, acc);
      float c = 0.f;
      if constexpr (POLICY) {
        const Token k = policy_token(e.logp, e.low, old, adv, ref, run.pol);
        c = k.slope * *run.inv_d;
        if (tid == 0) {
          const float cg = c * run.grad_scale;
          sm.end = make_float4(e.m, -cg * e.inv_s, cg * e.miss, cg);
          if (first) {
            sm.loss += (double)k.loss;
            sm.kl += (double)k.kl;
          }
        }
      }
      if (first) {
        logp[t] = e.logp;
        put_stats(stats + t, e.m, e.inv_s, e.miss);
        if (!POLICY) stats[t].w = e.low;
        if (coef) coef[t] = c;
      }
    }
    if constexpr (POLICY) {
      __syncthreads();
      // the values wait as 16 bits: without this the compiler keeps what pass one
      // unpacked, and spills
#pragma unroll
      for (int i = 0; i < kHold; ++i)
        asm volatile("" : "+r"(r[i].u.x), "+r"(r[i].u.y), "+r"(r[i].u.z), "+r"(r[i].u.w));
      const float4 e = sm.end;  // written again only after the next row's first barrier
      if (out && e.w == 0.f) {
        zero_slice<T, NT>(out, lo, hi);
      } else if (out) {
        const int count = g.count, skip = g.skip, head = g.head, tail = g.tail;
        T* o = out + (lo - skip) + tid * VE;  // granule j begins at (j - tid) VE from here
        const auto gradient = [&](const Vec<T>& x, int j) {
          uint4 v = scaled<T>(x, e.x, e.y);
          if (mine && j == yj) put<T>(v, ye % VE, bits_of<T>(e.z));
          return v;
        };
        if ((reinterpret_cast<uintptr_t>(o) & 15u) == 0) {
#pragma unroll
          for (int i = 0; i < kHold; ++i) {
            const int j = tid + i * NT;
            if (j < count && j != head && j != tail) __stcs(reinterpret_cast<uint4*>(o) + i * NT, gradient(r[i], j));
          }
          if (head == 0 && tid == 0) store_values(o, gradient(r[0], 0), skip, g.to(0));
          if (tail != head && tail % NT == tid) {
            Vec<T> x = r[0];
#pragma unroll
            for (int i = 1; i < kHold; ++i)
              if (tail == tid + i * NT) x = r[i];
            store_values(o + (tail - tid) * VE, gradient(x, tail), 0, g.last);
          }
        } else {
#pragma unroll
          for (int i = 0; i < kHold; ++i) {
            const int j = tid + i * NT;
            if (j < count) store_values(o + i * NT * VE, gradient(r[i], j), g.from(j), g.to(j));
          }
        }
      }
    }
    y = class_of(a, yn);
    t = tn;
    tn = tnn;
    yn = target_of(tn);
  }
  if (cs > 1) {
    cluster_arrive();
    cluster_wait();
  }
  if constexpr (POLICY) {
    if (rank != 0) return;
    if (tid == 0) {
      run.partial[c0] = make_double2(sm.loss, sm.kl);
      __threadfence();
      sm.last = atomicAdd(run.ticket, 1u) == (unsigned)(step - 1) ? 1u : 0u;
    }
    __syncthreads();
    if (!sm.last) return;
    __threadfence();
    double u = 0.0, v = 0.0;
    for (int i = tid; i < step; i += NT) {
      u += __ldcg(&run.partial[i].x);
      v += __ldcg(&run.partial[i].y);
    }
    u = block_sum_f64(u, sm.red);
    v = block_sum_f64(v, sm.red);
    if (tid == 0) {
      const double d = (double)*run.inv_d;
      *run.loss = (float)(u * d);
      *run.kl = (float)(v * d);
    }
  }
}

// Rows past what a cluster's registers hold (more than 8 x 64 KB): statistics
// by a loop over the row, kBatch vectors a thread at a time.
constexpr int kBatch = 8;
template <typename T>
__global__ void __launch_bounds__(kNT, 3)
k_long_rows(Rows a, int slice, int cs, float* __restrict__ logp, float4* __restrict__ stats,
            float* __restrict__ coef) {
  __shared__ RowShared<kNT> sh;
  const int t = blockIdx.x / cs;
  const int rank = (int)cluster_rank();
  const bool first = rank == 0 && threadIdx.x == 0;
  if (first && coef) coef[t] = 0.f;
  const int64_t y = a.targets[t];
  if (y == a.ignore) {  // the same for the whole cluster
    if (first) {
      logp[t] = 0.f;
      put_stats(stats + t, 0.f, 0.f, 0.f);
    }
    return;
  }
  row_shared_init(sh, cs);
  const T* x = row_ptr<T>(a, t);
  const float xt = first ? target_logit(x, y, a.V) : 0.f;
  const int64_t lo = (int64_t)rank * slice < a.V ? (int64_t)rank * slice : a.V;
  const int64_t hi = lo + slice < a.V ? lo + slice : a.V;
  const Slice<T> s(x, lo, hi);
  const uint4* p = reinterpret_cast<const uint4*>(x + s.body);
  const Hidden<T> hide(s, y);
  MaxSum acc = ends_of(s, y);
  for (int64_t i0 = threadIdx.x; i0 < s.vecs; i0 += kBatch * kNT) {
    Vec<T> r[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int64_t j = i0 + i * kNT;
      if (j < s.vecs) r[i].u = __ldg(p + j);
      else r[i].fill_neg_inf();
      if (j == hide.vec) hide.apply(r[i]);
    }
    acc = join(acc, vecs_of(r));
  }
  acc = row_join<kNT>(acc, sh, cs, 0);
  if (first) {
    const RowEnd e = row_end(xt, acc);
    logp[t] = e.logp;
    put_stats(stats + t, e.m, e.inv_s, e.miss);
    stats[t].w = e.low;
  }
  cluster_arrive();
  cluster_wait();
}

// ------------------------------------------------------------- preference --
// The sequences' sums in fp64 (a fixed tree), each pair's margin and loss, and c_t
// for its tokens: a cluster of up to 8 blocks takes the pairs in turn, half a
// block to a sequence, and its first block adds the blocks' losses in order.
// (One block for all pairs took 13 us for 8192 tokens, on one SM's loads.)
struct Preference {
  const void* cu;  // 2 * pairs + 1 offsets (int32 or int64), or null: `uniform` rows a sequence
  int cu64;
  int64_t uniform;
  int64_t pairs, rows;
  const float* logp;
  const float4* stats;
  const float* ref;
  const int64_t* targets;
  int64_t ignore;
  float beta, smoothing, inv_d;
};
__device__ __forceinline__ int64_t seq_offset(const Preference& a, int64_t i) {
  int64_t v = a.cu ? (a.cu64 ? static_cast<const int64_t*>(a.cu)[i]
                             : (int64_t)static_cast<const int*>(a.cu)[i])
                   : i * a.uniform;
  return v < 0 ? 0 : v > a.rows ? a.rows : v;
}
// ln(1 + exp(z))
__device__ __forceinline__ float softplus(float z) { return fmaxf(z, 0.f) + log1pf(expf(-fabsf(z))); }

constexpr int kSeqThreads = 256;
__global__ void __launch_bounds__(2 * kSeqThreads)
k_preference(Preference a, int cs, float* __restrict__ margins, float* __restrict__ coef,
             float* __restrict__ loss) {
  constexpr int kWarps = kSeqThreads / 32, kU = 4;
  __shared__ double part[2][2 * kWarps];
  __shared__ float2 mine;  // this block's loss, in two parts
  pdl_wait();
  pdl_trigger();
  const int rank = cs > 1 ? (int)cluster_rank() : 0;
  const int me = threadIdx.x / kSeqThreads, tid = threadIdx.x % kSeqThreads;
  double sum_loss = 0.0;
  int k = 0;
  for (int64_t b = rank; b < a.pairs; b += cs, k ^= 1) {
    const int64_t lo = seq_offset(a, 2 * b + me), hi = seq_offset(a, 2 * b + me + 1);
    double v = 0.0;
    for (int64_t t = lo + tid; t < hi; t += kU * kSeqThreads) {
      float d[kU], low[kU], r[kU];
      int64_t y[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) {  // all asked for before the first is used
        const int64_t at = t + u * kSeqThreads < hi ? t + u * kSeqThreads : t;
        y[u] = a.targets[at];
        d[u] = a.logp[at];
        low[u] = a.stats[at].w;
        r[u] = a.ref[at];
      }
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (t + u * kSeqThreads < hi && y[u] != a.ignore) v += ((double)d[u] - (double)r[u]) + (double)low[u];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) part[k][threadIdx.x >> 5] = v;  // written again two pairs on
    __syncthreads();
    double r[2] = {0.0, 0.0};
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      r[0] += part[k][w];
      r[1] += part[k][kWarps + w];
    }
    const float z = (float)((double)a.beta * (r[0] - r[1]));
    const float e = a.smoothing;
    // d loss / d z = sigmoid(z) - (1 - e) = e sigmoid(z) - (1 - e) sigmoid(-z):
    // the second form loses nothing where one of the two is near 1
    const float dn = 1.0f / (1.0f + expf(z)), up = 1.0f / (1.0f + expf(-z));
    const float c = (me ? -1.0f : 1.0f) * a.beta * a.inv_d * (e * up - (1.0f - e) * dn);
    for (int64_t t = lo + tid; t < hi; t += kSeqThreads)
      if (a.targets[t] != a.ignore) coef[t] = c;
    if (threadIdx.x == 0) {
      margins[b] = z;
      sum_loss += (double)((1.0f - e) * softplus(-z) + (e > 0.f ? e * softplus(z) : 0.f));
    }
  }
  if (threadIdx.x == 0) {
    const float big = (float)sum_loss;
    mine = make_float2(big, isfinite(big) ? (float)(sum_loss - (double)big) : 0.f);
  }
  if (cs > 1) {
    cluster_arrive();
    cluster_wait();
  }
  if (rank == 0 && threadIdx.x == 0) {
    double v = 0.0;
    for (int r = 0; r < cs; ++r) {
      const float2 f = cs > 1 ? peer_float2(&mine, r) : mine;
      v += (double)f.x + (double)f.y;
    }
    *loss = (float)(v * (double)a.inv_d);
  }
  if (cs > 1) {
    cluster_arrive();
    cluster_wait();
  }
}

// --------------------------------------------------------------- gradient --
// dx from the logits, the rows' (m, 1/S, R/S) and c_t: elementwise, one read and
// one write.  Rows run from the last to the first (see the head of the file)
// and c_t = 0 writes zeros without a read.  With `unless_one`, nothing is
// done when *scale_ptr is 1: dx already holds the gradient.
template <typename T>
__global__ void __launch_bounds__(kNT)
k_logits_grad(Rows a, int64_t slice, int parts, const float4* __restrict__ stats,
              const float* __restrict__ coef, float scale, const float* __restrict__ scale_ptr,
              int unless_one, T* __restrict__ dx) {
  constexpr int kB = 4;
  pdl_wait();
  float g = scale;
  if (scale_ptr) {
    const float up = *scale_ptr;
    if (unless_one && up == 1.0f) return;
    g *= up;
  }
  const int t = a.rows - 1 - (int)(blockIdx.x / parts);
  const int64_t lo = (int64_t)(blockIdx.x % parts) * slice;
  if (lo >= a.V) return;
  const int64_t hi = lo + slice < a.V ? lo + slice : a.V;
  T* out = dx + (int64_t)t * a.V;
  const int64_t y = a.targets[t];
  const float c = y == a.ignore ? 0.f : g * coef[t];
  if (c == 0.f) {
    zero_slice<T, kNT>(out, lo, hi);
    return;
  }
  const T* x = row_ptr<T>(a, t);
  const float4 st = stats[t];
  const float m = st.x, f = -c * st.y;
  const Slice<T> s(x, lo, hi);
  const uint4* p = reinterpret_cast<const uint4*>(x + s.body);
  const bool same = (reinterpret_cast<uintptr_t>(out + s.body) & 15u) == 0;
  for (int64_t i0 = threadIdx.x; i0 < s.vecs; i0 += kB * kNT) {
    Vec<T> r[kB];
#pragma unroll
    for (int i = 0; i < kB; ++i)
      if (i0 + i * kNT < s.vecs) r[i].u = __ldcs(p + i0 + i * kNT);
#pragma unroll
    for (int i = 0; i < kB; ++i) {
      const int64_t j = i0 + i * kNT;
      if (j >= s.vecs) break;
      const uint4 v = scaled<T>(r[i], m, f);
      if (same) __stcs(reinterpret_cast<uint4*>(out + s.body) + j, v);
      else store_values(out + s.body + j * Vec<T>::VE, v, 0, Vec<T>::VE);
    }
  }
  const int u = threadIdx.x;
  if (u < s.head) out[s.lo + u] = from_f<T>(f * exp_diff(to_f(x[s.lo + u]), m));
  if (u < s.tail) out[s.end + u] = from_f<T>(f * exp_diff(to_f(x[s.end + u]), m));
  if (y >= lo && y < hi) {
    __syncthreads();  // over what the loop wrote there
    if (u == 0) out[y] = from_f<T>(c * st.z);
  }
}

// ----------------------------------------------------------------- policy --
// Rows too long for registers: the tokens' c_t and the totals, from their log
// probabilities, by one block (k_long_rows before, k_logits_grad after).
__global__ void __launch_bounds__(1024)
k_policy_tokens(const int64_t* __restrict__ targets, int64_t ignore, int64_t rows, Policy pol,
                const float* __restrict__ logp, const float4* __restrict__ stats,
                const float* __restrict__ inv_d_ptr,
                float* __restrict__ coef, float* __restrict__ loss, float* __restrict__ kl) {
  __shared__ double red[32];
  const float inv_d = *inv_d_ptr;
  double u = 0.0, v = 0.0;
  for (int64_t t = threadIdx.x; t < rows; t += 1024) {
    Token k = {0.f, 0.f, 0.f};
    if (targets[t] != ignore)
      k = policy_token(logp[t], stats[t].w, pol.old[t], pol.adv[t], pol.ref ? pol.ref[t] : 0.f, pol);
    coef[t] = k.slope * inv_d;
    u += (double)k.loss;
    v += (double)k.kl;
  }
  u = block_sum_f64(u, red);
  v = block_sum_f64(v, red);
  if (threadIdx.x == 0) {
    *loss = (float)(u * (double)inv_d);
    *kl = (float)(v * (double)inv_d);
  }
}

// ------------------------------------------------------------------- host --
// How the rows are cut.  cs blocks share a row: as many as bring a slice down to
// kGrainsMax granules, and with few rows more, until there are two blocks an SM
// or a slice would fall under 16 KB.
struct Split {
  int cs, slice;
  int quarter;  // a slice is at most 1, 2 or 4 quarters of kGrainsMax; 0: too long
};
Split split_rows(const LogitsArg& l) {
  const int64_t rows = l.rows, V = l.vocab, elem = dtype_size(l.dtype);
  // rows that begin on a 16-byte boundary need no granule more than their values do
  const int off = ((reinterpret_cast<uintptr_t>(l.logits) | (uintptr_t)(l.row_stride * elem) |
                    (uintptr_t)(l.batch_stride * elem)) & 15) != 0;
  const int64_t ve = 16 / elem;
  const auto slice_of = [&](int cs) {
    return ((V + cs - 1) / cs + ve - 1) / ve * ve;  // whole granules of an aligned row
  };
  const auto grains_of = [&](int cs) { return slice_of(cs) / ve + off; };
  int cs = 1;
  while (cs < kMaxCluster && grains_of(cs) > kGrainsMax) cs *= 2;
  while (cs < kMaxCluster && rows * cs < 2 * (int64_t)sm_count() && V / (2 * cs) * elem >= 16 * 1024)
    cs *= 2;
  const int64_t n = grains_of(cs);
  const int quarter = n <= kGrainsMax / 4 ? 1 : n <= kGrainsMax / 2 ? 2 : n <= kGrainsMax ? 4 : 0;
  return {cs, (int)slice_of(cs), quarter};
}

template <typename... KArgs, typename... Args>
cudaError_t launch_rows(void (*kernel)(KArgs...), int64_t blocks, int threads, size_t smem,
                        int cs, bool pdl, cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (cs > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = cs;
    at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl && pdl_enabled()) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Args&&>(args)...);
}
int launched(const char* what, cudaError_t e) {
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return set_error(MHC_ERR_CUDA, "%s: launch failed: %s", what, cudaGetErrorString(e));
  }
  return MHC_OK;
}

Rows rows_of(const LogitsArg& l) {
  const int64_t per = l.per_batch < l.rows ? l.per_batch : l.rows;
  return {l.logits, (int)l.rows, (int)(per > 0 ? per : 1), l.batch_stride, l.row_stride, (int)l.vocab,
          l.targets, l.ignore};
}

template <typename T, int NT, bool POLICY>
int run_rows_nt(const char* what, const LogitsArg& l, const Split& sp, float* logp, float4* stats,
                float* coef, const PolicyRun& run, void* dx, cudaStream_t st) {
  const auto kern = k_rows<T, NT, POLICY>;
  const size_t smem = (size_t)(sp.slice / (16 / (int64_t)sizeof(T)) + 1) * 16;
  const cudaError_t e = allow_dyn_smem(kern, smem);
  if (e != cudaSuccess) return launched(what, e);
  // as many clusters as are resident at once: blocks walk the rows
  int64_t clusters = (int64_t)sm_count() * blocks_per_sm(kern, NT, smem) / sp.cs;
  if (clusters < 1) clusters = 1;
  if (clusters > l.rows) clusters = l.rows;
  // each has its pair of sums in the workspace, whatever number of blocks fits
  if (POLICY && clusters > (int64_t)sm_count() * kPolicyClustersSM)
    clusters = (int64_t)sm_count() * kPolicyClustersSM;
  // the order pays where the rows' work is what counts: 8192 rows of 32000 bf16,
  // 30 % ignored, 187 us by number and 172 in order; reading alone gains 7 us of
  // 98 and would pay a launch for it
  const int ordered = POLICY && clusters < l.rows;
  if (POLICY) {
    k_order<<<1, 1024, 0, st>>>(l.targets, (int)l.rows, l.ignore, ordered ? stats : nullptr, run.inv_d_in,
                                run.inv_d, run.ticket);
    const int r = check_launch(what);
    if (r != MHC_OK) return r;
  }
  return launched(what, launch_rows(kern, clusters * sp.cs, NT, smem, sp.cs, POLICY, st, rows_of(l),
                                    sp.slice, sp.cs, ordered, logp, stats, coef, run, static_cast<T*>(dx)));
}
template <typename T, bool POLICY>
int run_rows(const char* what, const LogitsArg& l, const Split& sp, float* logp, float4* stats,
             float* coef, const PolicyRun& run, void* dx, cudaStream_t st) {
  constexpr int q = (int)(kGrainsMax / 4) / RowShape<POLICY>::kNV;  // threads for a quarter
  if (sp.quarter == 1) return run_rows_nt<T, q, POLICY>(what, l, sp, logp, stats, coef, run, dx, st);
  if (sp.quarter == 2) return run_rows_nt<T, 2 * q, POLICY>(what, l, sp, logp, stats, coef, run, dx, st);
  return run_rows_nt<T, 4 * q, POLICY>(what, l, sp, logp, stats, coef, run, dx, st);
}

template <typename T>
int run_stats(const LogitsArg& l, float* logp, float4* stats, float* coef, cudaStream_t st) {
  const Split sp = split_rows(l);
  if (sp.quarter)
    return run_rows<T, false>("token_logprobs", l, sp, logp, stats, coef, PolicyRun{}, nullptr, st);
  return launched("token_logprobs",
                  launch_rows(k_long_rows<T>, l.rows * sp.cs, kNT, 0, sp.cs, false, st, rows_of(l),
                              sp.slice, sp.cs, logp, stats, coef));
}

template <typename T>
int run_grad(const LogitsArg& l, const float4* stats, const float* coef, float scale,
             const float* scale_ptr, int unless_one, void* dx, bool pdl, cudaStream_t st) {
  // slices of 64 KB or less; few rows are cut finer, to 8 KB, to fill the SMs
  const int64_t ve = 16 / (int64_t)sizeof(T);
  int64_t parts = (l.vocab * (int64_t)sizeof(T) + (64 << 10) - 1) / (64 << 10);
  while (l.rows * parts < 4 * (int64_t)sm_count() &&
         l.vocab / (2 * parts) * (int64_t)sizeof(T) >= 8 * 1024)
    parts *= 2;
  int64_t slice = (l.vocab + parts - 1) / parts;
  slice = (slice + ve - 1) / ve * ve;
  if (l.rows > (int64_t)0x7fffffff / parts)
    return set_error(MHC_ERR_UNSUPPORTED, "logits_grad: %lld rows of %lld logits are too many",
                     (long long)l.rows, (long long)l.vocab);
  return launched("logits_grad",
                  launch_rows(k_logits_grad<T>, l.rows * parts, kNT, 0, 1, pdl, st, rows_of(l), slice,
                              (int)parts, stats, coef, scale, scale_ptr, unless_one,
                              static_cast<T*>(dx)));
}

template <typename T>
int run_policy(const LogitsArg& l, const Policy& p, float inv_d, float scale, const PolicyOut& o,
               cudaStream_t st) {
  float4* stats = reinterpret_cast<float4*>(o.stats);
  const Split sp = split_rows(l);
  if (sp.quarter) {
    const PolicyRun run = {p, inv_d, o.inv_d, scale, reinterpret_cast<double2*>(o.partial), o.loss, o.kl, o.ticket};
    return run_rows<T, true>("policy_loss", l, sp, o.logp, stats, o.coef, run, o.dlogits, st);
  }
  int r = run_stats<T>(l, o.logp, stats, nullptr, st);
  if (r != MHC_OK) return r;
  k_order<<<1, 1024, 0, st>>>(l.targets, (int)l.rows, l.ignore, nullptr, inv_d, o.inv_d, o.ticket);
  r = check_launch("policy_loss");
  if (r != MHC_OK) return r;
  k_policy_tokens<<<1, 1024, 0, st>>>(l.targets, l.ignore, l.rows, p, o.logp, stats, o.inv_d, o.coef,
                                      o.loss, o.kl);
  r = check_launch("policy_loss");
  if (r != MHC_OK || !o.dlogits) return r;
  return run_grad<T>(l, stats, o.coef, scale, nullptr, 0, o.dlogits, false, st);
}

}  // namespace

#define MHC_BY_DTYPE(dt, CALL)              \
  switch (dt) {                             \
    case MHC_F32: return CALL(float);       \
    case MHC_F16: return CALL(f16);         \
    default: return CALL(bf16);             \
  }

int launch_token_logprobs(const LogitsArg& l, float* logp, float* stats, cudaStream_t st) {
  if (l.rows == 0) return MHC_OK;
#define CALL(T) run_stats<T>(l, logp, reinterpret_cast<float4*>(stats), nullptr, st)
  MHC_BY_DTYPE(l.dtype, CALL)
#undef CALL
}

int launch_logits_grad(const LogitsArg& l, const float* stats, const float* coef, float scale,
                       const float* scale_ptr, int unless_one, void* dlogits, cudaStream_t st) {
  if (l.rows == 0) return MHC_OK;
#define CALL(T)                                                                                  \
  run_grad<T>(l, reinterpret_cast<const float4*>(stats), coef, scale, scale_ptr, unless_one,     \
              dlogits, false, st)
  MHC_BY_DTYPE(l.dtype, CALL)
#undef CALL
}

template <typename T>
static int run_preference(const LogitsArg& l, const PreferenceArg& a, const PreferenceOut& o,
                          cudaStream_t st) {
  if (l.rows > 0) {
    const int r = run_stats<T>(l, o.logp, reinterpret_cast<float4*>(o.stats), o.coef, st);
    if (r != MHC_OK) return r;
  }
  const Preference p = {a.cu_seqlens, a.cu_is64, a.uniform, a.pairs,  l.rows,  o.logp, reinterpret_cast<const float4*>(o.stats), a.ref,
                        l.targets,    l.ignore,  a.beta,    a.smoothing, a.inv_d};
  int cs = 1;
  while (cs < kMaxCluster && cs < a.pairs) cs *= 2;
  const int r = launched("preference_loss", launch_rows(k_preference, cs, 2 * kSeqThreads, 0, cs, true, st,
                                                        p, cs, o.margins, o.coef, o.loss));
  if (r != MHC_OK || !o.dlogits || l.rows == 0) return r;
  return run_grad<T>(l, reinterpret_cast<float4*>(o.stats), o.coef, a.grad_scale, nullptr, 0,
                     o.dlogits, true, st);
}

int launch_preference(const LogitsArg& l, const PreferenceArg& a, const PreferenceOut& o,
                      cudaStream_t st) {
#define CALL(T) run_preference<T>(l, a, o, st)
  MHC_BY_DTYPE(l.dtype, CALL)
#undef CALL
}

int launch_policy(const LogitsArg& l, const PolicyArg& a, const PolicyOut& o, cudaStream_t st) {
  const Policy p = {a.old, a.adv, a.ref, 1.0f - a.clip_low, 1.0f + a.clip_high, a.kl_coef};
  if (l.rows == 0) {
    const cudaError_t e = cudaMemsetAsync(o.loss, 0, sizeof(float), st);
    const cudaError_t f = cudaMemsetAsync(o.kl, 0, sizeof(float), st);
    if (e != cudaSuccess || f != cudaSuccess)
      return set_error(MHC_ERR_CUDA, "policy_loss: %s", cudaGetErrorString(e != cudaSuccess ? e : f));
    return MHC_OK;
  }
#define CALL(T) run_policy<T>(l, p, a.inv_d, a.grad_scale, o, st)
  MHC_BY_DTYPE(l.dtype, CALL)
#undef CALL
}

}  // namespace mhc
