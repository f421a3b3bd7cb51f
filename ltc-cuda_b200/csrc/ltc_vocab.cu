// Row-wise softmax operators over a vocabulary: z (rows, V), q = softmax(z / tau).
//   distillation   p = softmax(teacher / tau) over the K given entries of a row,
//                  loss = tau^2 sum_k p_k (log p_k - log q_{id_k})
//   token scores   log q[token], entropy -sum q log q, the k largest log q with their ids
// and their gradients, both of the form  dz_j = q_j (alpha + beta log q_j) + a few entries:
//   distillation   alpha = g tau, beta = 0;  -g tau p_k at id_k
//   token scores   alpha = -(g_lp + g_H H) / tau, beta = -g_H / tau;  +g_lp / tau at the token
//
// Forward: one pass over the row.  A thread keeps the running maximum m and, relative to
// it, s = sum 2^y and u = sum 2^y y with y = (z - m) log2(e) / tau; two such triples merge
// by moving the smaller maximum's sums to the larger.  z - m is taken before the scaling,
// so the type's lowest value (a mask) neither overflows nor costs accuracy.  A row is one
// block, or a cluster of up to 8 blocks where there are few rows: the blocks' triples meet
// in shared memory over DSMEM, in rank order.  Bound by the one read of the logits.
//
// The k best ride in the same pass: every thread notes the maximum of each window of values it
// reads.  Behind the pass a threshold that at least k thread maxima reach (the k-th largest of
// the ceil(k / warps) + 1 largest of every warp) leaves a few windows, whose values are read
// again; the few that reach the threshold are ranked by counting.  Where too many reach it (a
// row of equal values, say) the row is searched k times instead: slow and right.  Ties go
// to the lowest index.
//
// Backward: elementwise over (row, chunk of columns), then the block that wrote a listed
// entry's chunk writes that entry again with its extra term, rounded once.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "ltc_common.cuh"
#include "ltc_internal.h"

namespace cg = cooperative_groups;

namespace ltc {

namespace {

constexpr int kThreads = 256;  // of the gradient's blocks
constexpr int kUnroll = 4;     // 16-byte loads in flight per thread
constexpr int kCap = 1024;     // candidates for the k best
constexpr int kSlots = 16;     // noted maxima per thread; longer rows note several windows as one
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// Stands for everything below it where 2^y multiplies it: 2^y is 0 from y = -127 on (ex2 flushes), and
// small enough that a factor of up to 3e35 (a large loss scale over a small temperature) leaves the product
// finite.
constexpr float kFar = -1024.f;

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// ---- element types ---------------------------------------------------------------
template <typename T> struct Elem;
template <> struct Elem<float> {
  static constexpr int N = 4;  // per 16 bytes
  static constexpr unsigned kNegInf = 0xff800000u;
  __device__ static void unpack(const uint4& r, float* v) {
    v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y);
    v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
  }
  __device__ static uint4 pack(const float (&v)[4]) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
  template <int U>
  __device__ static float top(const uint4 (&r)[U]) {  // largest value, NaN if there is one
    float m = max3_nan(__uint_as_float(r[0].x), __uint_as_float(r[0].y), __uint_as_float(r[0].z));
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (k > 0) {
        m = max3_nan(m, __uint_as_float(r[k].x), __uint_as_float(r[k].y));
        m = max3_nan(m, __uint_as_float(r[k].z), __uint_as_float(r[k].w));
      } else {
        m = max_nan(m, __uint_as_float(r[k].w));
      }
    }
    return m;
  }
  __device__ static float one(const float* p) { return __ldg(p); }
  __device__ static float down(float x) { return x; }
};
template <> struct Elem<__nv_bfloat16> {
  static constexpr int N = 8;
  static constexpr unsigned kNegInf = 0xff80ff80u;
  __device__ static void two(unsigned r, float& a, float& b) {
    a = __uint_as_float(r << 16);
    b = __uint_as_float(r & 0xffff0000u);
  }
  __device__ static void unpack(const uint4& r, float* v) {
    two(r.x, v[0], v[1]); two(r.y, v[2], v[3]); two(r.z, v[4], v[5]); two(r.w, v[6], v[7]);
  }
  __device__ static unsigned p2(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<unsigned*>(&h);
  }
  __device__ static uint4 pack(const float (&v)[8]) {
    return make_uint4(p2(v[0], v[1]), p2(v[2], v[3]), p2(v[4], v[5]), p2(v[6], v[7]));
  }
  template <int U>
  __device__ static float top(const uint4 (&r)[U]) {
    unsigned m = r[0].x;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (k > 0) m = max2(m, r[k].x);
      m = max2(max2(max2(m, r[k].y), r[k].z), r[k].w);
    }
    float a, b;
    two(m, a, b);
    return max_nan(a, b);
  }
  __device__ static unsigned max2(unsigned a, unsigned b) {
    unsigned y;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
    return y;
  }
  __device__ static float one(const __nv_bfloat16* p) {
    return __uint_as_float((unsigned)__ldg(reinterpret_cast<const unsigned short*>(p)) << 16);
  }
  __device__ static __nv_bfloat16 down(float x) { return __float2bfloat16_rn(x); }
};
template <> struct Elem<__half> {
  static constexpr int N = 8;
  static constexpr unsigned kNegInf = 0xfc00fc00u;
  __device__ static void two(unsigned r, float& a, float& b) {
    const float2 f = __half22float2(*reinterpret_cast<__half2*>(&r));
    a = f.x;
    b = f.y;
  }
  __device__ static void unpack(const uint4& r, float* v) {
    two(r.x, v[0], v[1]); two(r.y, v[2], v[3]); two(r.z, v[4], v[5]); two(r.w, v[6], v[7]);
  }
  __device__ static unsigned p2(float a, float b) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<unsigned*>(&h);
  }
  __device__ static uint4 pack(const float (&v)[8]) {
    return make_uint4(p2(v[0], v[1]), p2(v[2], v[3]), p2(v[4], v[5]), p2(v[6], v[7]));
  }
  template <int U>
  __device__ static float top(const uint4 (&r)[U]) {
    unsigned m = r[0].x;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (k > 0) m = max2(m, r[k].x);
      m = max2(max2(max2(m, r[k].y), r[k].z), r[k].w);
    }
    float a, b;
    two(m, a, b);
    return max_nan(a, b);
  }
  __device__ static unsigned max2(unsigned a, unsigned b) {
    unsigned y;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
    return y;
  }
  __device__ static float one(const __half* p) { return __half2float(*p); }
  __device__ static __half down(float x) { return __float2half_rn(x); }
};

__device__ __forceinline__ float teacher_at(const void* p, int dtype, long long i) {
  if (dtype == 0) return Elem<float>::one(static_cast<const float*>(p) + i);
  if (dtype == 1) return Elem<__nv_bfloat16>::one(static_cast<const __nv_bfloat16*>(p) + i);
  return Elem<__half>::one(static_cast<const __half*>(p) + i);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }
__device__ __forceinline__ float quiet_nan() { return __int_as_float(0x7fffffff); }

// running maximum and sums of a set of logits; s = u = 0 while m is -inf
struct Sums {
  float m, s, u;
};
// moves the sums to the maximum mn >= a.m (mn not -inf)
__device__ __forceinline__ void move_to(Sums& a, float mn, float c2) {
  if (a.m != neg_inf()) {
    const float d = (a.m - mn) * c2;
    const float f = ex2(d);
    a.u = f * fmaf(fmaxf(d, kFar), a.s, a.u);
    a.s *= f;
  }
  a.m = mn;
}
__device__ __forceinline__ Sums merge(Sums a, Sums b, float c2) {
  const float mn = max_nan(a.m, b.m);
  if (mn == neg_inf()) return a;
  move_to(a, mn, c2);
  move_to(b, mn, c2);
  a.s += b.s;
  a.u += b.u;
  return a;
}

__device__ __forceinline__ bool better(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

template <typename T>
__device__ __forceinline__ const T* row_ptr(const VocabArgs& g, long long row) {
  const long long outer = row < g.n1 ? 0 : row / g.n1;  // no division where one stride walks all rows
  return static_cast<const T*>(g.z) + outer * g.s0 + (row - outer * g.n1) * g.s1;
}

// elements before the first 16-byte boundary of p (at most len)
template <typename T>
__device__ __forceinline__ int head_of(const T* p, int len) {
  const int mis = (int)(reinterpret_cast<uintptr_t>(p) & 15);
  const int h = mis ? (16 - mis) / (int)sizeof(T) : 0;
  return h < len ? h : len;
}

// k best of n candidates, best first, (-inf, -1) where there are fewer; all threads call it
template <int NT>
__device__ void select_best(const float* cv, const int* ci, int n, int k, float* ov, int* oi) {
  for (int j = threadIdx.x; j < k; j += NT) {
    ov[j] = neg_inf();
    oi[j] = -1;
  }
  __syncthreads();
  for (int c = threadIdx.x; c < n; c += NT) {
    const float v = cv[c];
    const int i = ci[c];
    int rank = 0;
    for (int d = 0; d < n && rank < k; ++d) rank += better(cv[d], ci[d], v, i) ? 1 : 0;
    if (rank < k) {
      ov[rank] = v;
      oi[rank] = i;
    }
  }
  __syncthreads();
}

template <int NT>
struct TopShared {
  float cv[kCap];
  int ci[kCap];
  float noted[kSlots][NT];
  float ov[kVocabMaxTop];
  int oi[kVocabMaxTop];
  float thread_v[NT];
  float best_v[kVocabMaxTop + 2 * (NT / 32)];
  float warp_v[NT / 32];
  int warp_i[NT / 32];
  int count;
  float pv, thr, thr_all;
  int pi;
};
struct NoShared {};

// a block's part of a row: values before the first 16-byte boundary, aligned vectors, the rest
template <typename T>
struct Part {
  const T* p;
  int len, head, nvec;
  __device__ __forceinline__ Part(const VocabArgs& g, long long row, int lo, int hi) {
    p = row_ptr<T>(g, row) + lo;
    len = hi - lo;
    head = head_of(p, len);
    nvec = (len - head) / Elem<T>::N;
  }
};
template <int NT, typename T>
__device__ __forceinline__ void load_window(uint4 (&r)[kUnroll], const Part<T>& part, int base) {
  const uint4* pv = reinterpret_cast<const uint4*>(part.p + part.head) + base + threadIdx.x;
  const int left = part.nvec - base - (int)threadIdx.x;
#pragma unroll
  for (int k = 0; k < kUnroll; ++k)
    r[k] = k * NT < left ? __ldg(pv + k * NT)
                         : make_uint4(Elem<T>::kNegInf, Elem<T>::kNegInf, Elem<T>::kNegInf, Elem<T>::kNegInf);
}

// ---- forward -----------------------------------------------------------------------
// A block or cluster per row; reads of one block run while others compute.  (Persistent blocks
// whose next windows are on their way, in registers or a cp.async ring, were slower: 87 and 75
// against 72 us at 4096 x 32768 bf16, before the reductions became cheaper: 64 now.)
template <typename T, bool DISTILL, bool TOPK, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) vocab_fwd_kernel(VocabArgs g) {
  constexpr int N = Elem<T>::N, NW = NT / 32, EPT = kVocabMaxTeacher / NT;  // teacher entries of a thread
  constexpr int kWindow = NT * kUnroll;  // vectors read at a time
  __shared__ float warp_m[NW], warp_em[NW], warp_loss[NW];
  __shared__ float2 warp_sums[NW];
  __shared__ Sums block_sums;
  __shared__ typename std::conditional<TOPK, TopShared<NT>, NoShared>::type top;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cs = g.cluster, rank = cs > 1 ? (int)(blockIdx.x % cs) : 0;
  const int lo = min(rank * g.chunk, g.V), hi = min(lo + g.chunk, g.V);
  const float c2 = g.inv_tau * kLog2e;
  const long long row = blockIdx.x / cs;
  const Part<T> part(g, row, lo, hi);
  const T* p = part.p;
  const int len = part.len, head = part.head, nvec = part.nvec;
  const int tail = head + nvec * N;  // fewer than N values
  uint4 r[kUnroll];
  load_window<NT>(r, part, 0);
  // read now, looked at behind the pass: this thread's teacher entries, or the row's token, and the edges
  constexpr int E = DISTILL ? EPT : 1;
  const int entries = rank != 0 ? 0 : DISTILL ? g.K : 1;
  long long id[E];
  float z_id[E], t_id[E], z_head = 0.f, z_tail = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int k = e * NT + tid;
    id[e] = -1;
    z_id[e] = t_id[e] = 0.f;
    if (k < entries) {
      id[e] = DISTILL ? g.ids[row * g.K + k] : g.tokens[row];
      if (DISTILL) t_id[e] = teacher_at(g.teacher, g.teacher_dtype, row * g.K + k);
    }
  }
  if (tid < head) z_head = Elem<T>::one(p + tid);
  if (tid < len - tail) z_tail = Elem<T>::one(p + tail + tid);
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (id[e] >= 0 && id[e] < g.V) z_id[e] = Elem<T>::one(p - lo + id[e]);

  Sums a{neg_inf(), 0.f, 0.f};
  const int windows = (nvec + kWindow - 1) / kWindow, per_slot = (windows + kSlots - 1) / kSlots;
  float best = neg_inf(), slot_v = neg_inf();  // this thread's maximum, and that of the slot at hand
  int in_slot = 0, slot = 0;
  int base = 0;
  do {
    const bool last = base + kWindow >= nvec;
    const float top_v = Elem<T>::template top<kUnroll>(r);
    float v[kUnroll * N];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) Elem<T>::unpack(r[k], v + k * N);
    if (!last) load_window<NT>(r, part, base + kWindow);
    const float mn = max_nan(a.m, top_v);
    if (mn != neg_inf()) {
      if (mn != a.m) move_to(a, mn, c2);
      float2 s2 = make_float2(0.f, 0.f), u2 = s2;
#pragma unroll
      for (int j = 0; j < kUnroll * N; j += 2) {
        const float2 y = mul2(add2(make_float2(v[j], v[j + 1]), make_float2(-mn, -mn)), make_float2(c2, c2));
        const float2 e = make_float2(ex2(y.x), ex2(y.y));
        s2 = add2(s2, e);
        if (!DISTILL) u2 = fma2(e, make_float2(fmaxf(y.x, kFar), fmaxf(y.y, kFar)), u2);
      }
      a.s += s2.x + s2.y;
      if (!DISTILL) a.u += u2.x + u2.y;
    }
    if constexpr (TOPK) {
      slot_v = fmaxf(slot_v, top_v);  // NaN is left out
      if (++in_slot == per_slot || last) {
        if (nvec > 0) top.noted[slot++][tid] = slot_v;
        best = fmaxf(best, slot_v);
        slot_v = neg_inf();
        in_slot = 0;
      }
    }
    base += kWindow;
  } while (base < nvec);
  auto single = [&](float v) {  // a value outside the aligned body
    const float mn = max_nan(a.m, v);
    if (mn == neg_inf()) return;
    if (mn != a.m) move_to(a, mn, c2);
    const float y = (v - a.m) * c2, e = ex2(y);
    a.s += e;
    a.u = fmaf(e, fmaxf(y, kFar), a.u);
  };
  if (tid < head) single(z_head);
  if (tid < len - tail) single(z_tail);

  // block sums: the maximum first, then every thread's sums moved to it, in lane and warp order
  float wm = a.m, em = neg_inf();
  if (DISTILL) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (id[e] >= 0) em = max_nan(em, t_id[e]);
  }
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) {
    wm = max_nan(wm, __shfl_xor_sync(0xffffffffu, wm, d));
    if (DISTILL) em = max_nan(em, __shfl_xor_sync(0xffffffffu, em, d));
  }
  if (lane == 0) {
    warp_m[warp] = wm;
    if (DISTILL) warp_em[warp] = em;
  }
  if constexpr (TOPK) {
    // the largest maxima of each warp's threads, at least k in all
    const int need = (g.k + NW - 1) / NW + 1;
    float x = best;
    for (int q = 0; q < need; ++q) {
      float w = x;
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, d));
      const unsigned who = __ballot_sync(0xffffffffu, x == w);
      if (lane == __ffs(who) - 1) x = neg_inf();
      if (lane == 0) top.best_v[warp * need + q] = w;
    }
    top.thread_v[tid] = best;
    if (tid == 0) {
      top.count = 0;
      top.thr = neg_inf();
    }
  }
  __syncthreads();
  Sums t{warp_m[0], 0.f, 0.f};
#pragma unroll
  for (int w = 1; w < NW; ++w) t.m = max_nan(t.m, warp_m[w]);
  if constexpr (TOPK) {  // the k-th largest of them: k values reach it
    const int m = ((g.k + NW - 1) / NW + 1) * NW;
    if (tid < m) {
      const float v = top.best_v[tid];
      int above = 0;
      for (int d = 0; d < m; ++d) above += better(top.best_v[d], d, v, tid) ? 1 : 0;
      if (above == g.k - 1) top.thr = v;
    }
  }
  float te[E], es = 0.f;  // this thread's entries up to their sum
  if constexpr (DISTILL) {
    em = warp_em[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) em = max_nan(em, warp_em[w]);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      te[e] = id[e] >= 0 && em != neg_inf() ? ex2((t_id[e] - em) * c2) : 0.f;
      es += te[e];
    }
  }
  if (t.m != neg_inf()) move_to(a, t.m, c2);
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, d);
    if (!DISTILL) a.u += __shfl_xor_sync(0xffffffffu, a.u, d);
    if (DISTILL) es += __shfl_xor_sync(0xffffffffu, es, d);
  }
  if (lane == 0) warp_sums[warp] = make_float2(a.s, DISTILL ? es : a.u);
  __syncthreads();
  // from here on the warps that hold results go on
  const bool busy = cs > 1 || TOPK || warp * 32 < entries;
  es = 0.f;
  if (busy) {
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float2 v = warp_sums[w];
      t.s += v.x;
      (DISTILL ? es : t.u) += v.y;
    }
  }

  if constexpr (TOPK) {
    float thr = top.thr;  // every warp branches on it below, so nothing writes it any more
    if (thr == neg_inf() && t.m != neg_inf()) {
      // short or masked rows leave warps without values: the k-th largest of all thread maxima instead
      int above = 0;
      for (int d = 0; d < NT; ++d) above += better(top.thread_v[d], d, best, tid) ? 1 : 0;
      if (above == g.k - 1) top.thr_all = best;
      __syncthreads();
      thr = top.thr_all;
    }
    auto reaches = [&](float v) { return v >= thr && v > neg_inf(); };
    auto keep = [&](float v, int i) {
      const int at = atomicAdd(&top.count, 1);  // the order in the list does not matter
      LTC_CHECK(i >= 0 && i < g.V, 911);
      if (at < kCap) {
        top.cv[at] = v;
        top.ci[at] = i;
      }
    };
    if (tid < head && reaches(z_head)) keep(z_head, lo + tid);
    if (tid < len - tail && reaches(z_tail)) keep(z_tail, lo + tail + tid);
    for (int sl = 0; sl < slot; ++sl) {
      // a warp takes its threads' windows that reach the threshold one after the other, a lane per value
      unsigned who = __ballot_sync(0xffffffffu, reaches(top.noted[sl][tid]));
      while (who) {
        const int th = warp * 32 + __ffs(who) - 1;
        who &= who - 1;
        for (int e = lane; e < per_slot * kUnroll * N; e += 32) {
          const int vec = sl * per_slot * kWindow + (e / N) * NT + th;
          if (vec >= nvec) break;
          const int i = head + vec * N + e % N;
          const float v = Elem<T>::one(p + i);
          if (reaches(v)) keep(v, lo + i);
        }
        __syncwarp();
      }
    }
    __syncthreads();
    const int n = top.count;
    if (n <= kCap) {
      select_best<NT>(top.cv, top.ci, n, g.k, top.ov, top.oi);
    } else {
      float pbest = __int_as_float(0x7f800000);
      int ibest = -1;
      for (int q = 0; q < g.k; ++q) {
        float bv = neg_inf();
        int bi = 0x7fffffff;
        for (int i = tid; i < len; i += NT) {
          const float x = Elem<T>::one(p + i);
          if (x > neg_inf() && better(pbest, ibest, x, lo + i) && better(x, lo + i, bv, bi)) {
            bv = x;
            bi = lo + i;
          }
        }
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) {
          const float ov = __shfl_xor_sync(0xffffffffu, bv, d);
          const int oi = __shfl_xor_sync(0xffffffffu, bi, d);
          if (better(ov, oi, bv, bi)) {
            bv = ov;
            bi = oi;
          }
        }
        if (lane == 0) {
          top.warp_v[warp] = bv;
          top.warp_i[warp] = bi;
        }
        __syncthreads();
        if (tid == 0) {
          for (int w = 1; w < NW; ++w)
            if (better(top.warp_v[w], top.warp_i[w], bv, bi)) {
              bv = top.warp_v[w];
              bi = top.warp_i[w];
            }
          top.pv = top.ov[q] = bv;
          top.pi = bi;
          top.oi[q] = bv > neg_inf() ? bi : -1;
        }
        __syncthreads();
        pbest = top.pv;
        ibest = top.pi;
      }
    }
  }

  if (cs > 1) {
    cg::cluster_group cl = cg::this_cluster();
    if (tid == 0) block_sums = t;
    cl.sync();
    if (rank == 0) {
      if constexpr (TOPK) {
        for (int c = tid; c < cs * g.k; c += NT) {
          const int q = c / g.k, j = c - q * g.k;
          top.cv[c] = cl.map_shared_rank(&top.ov[0], q)[j];
          top.ci[c] = cl.map_shared_rank(&top.oi[0], q)[j];
        }
      }
      Sums o{neg_inf(), 0.f, 0.f};  // lane q: block q's
      if (lane < cs) o = *cl.map_shared_rank(&block_sums, lane);
      t = o;
#pragma unroll
      for (int d = 4; d >= 1; d >>= 1) t.m = max_nan(t.m, __shfl_xor_sync(0xffffffffu, t.m, d));
      t.m = __shfl_sync(0xffffffffu, t.m, 0);
      if (t.m != neg_inf()) move_to(o, t.m, c2);
#pragma unroll
      for (int d = 4; d >= 1; d >>= 1) {
        o.s += __shfl_xor_sync(0xffffffffu, o.s, d);
        o.u += __shfl_xor_sync(0xffffffffu, o.u, d);
      }
      t.s = __shfl_sync(0xffffffffu, o.s, 0);
      t.u = __shfl_sync(0xffffffffu, o.u, 0);
    }
    cl.sync();  // the others' shared memory has been read
    if (rank != 0) return;
    if constexpr (TOPK) select_best<NT>(top.cv, top.ci, cs * g.k, g.k, top.ov, top.oi);
  }
  if (!DISTILL && warp * 32 >= max(entries, TOPK ? g.k : 0)) return;  // no barrier follows
  const bool empty = t.m == neg_inf();
  const float l2 = empty ? 0.f : log2f(t.s);

  if constexpr (DISTILL) {
    const bool any = em != neg_inf();  // no entries, or all of them -inf: no distribution
    float loss = 0.f;
    bool bad = false;
    if (busy) {
      // tau (log p - log q) in the logits' own units: a masked entry at the type's lowest value stays
      // finite as long as the loss does.  The other tau comes before the sum where it is small and
      // after it where it is large, so that no term leaves the range before the sum does.
      const float le = log2f(es), tl = g.tau * kLn2;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float pk = 0.f;
        bad = bad || id[e] >= g.V;
        if (id[e] >= 0 && any) {
          pk = te[e] / es;
          if (pk != 0.f && id[e] < g.V)
            loss = fmaf(pk * fminf(g.tau, 1.f),
                        empty ? -neg_inf() : fmaf(tl, l2 - le, (t_id[e] - em) - (z_id[e] - t.m)), loss);
        }
        if (e * NT + tid < entries && g.probs) g.probs[row * g.K + e * NT + tid] = pk;
      }
      if (bad) loss = quiet_nan();
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) loss += __shfl_xor_sync(0xffffffffu, loss, d);
      bad = __any_sync(0xffffffffu, bad);
    }
    if (g.K > 32) {
      if (lane == 0) warp_loss[warp] = loss;
      bad = __syncthreads_or(bad);
      loss = 0.f;
      if (tid == 0)
        for (int w = 0; w < NW; ++w) loss += warp_loss[w];
    }
    if (tid == 0) {
      g.loss[row] = loss * fmaxf(g.tau, 1.f);
      if (g.stats)
        reinterpret_cast<float4*>(g.stats)[row] = make_float4(t.m, l2, bad ? quiet_nan() : any ? 1.f : 0.f, 0.f);
    }
  } else {
    const float ent = empty ? 0.f : (l2 - t.u / t.s) * kLn2;
    if (tid == 0) {
      float lp = 0.f;
      if (id[0] >= g.V) lp = quiet_nan();
      else if (id[0] >= 0) lp = empty ? neg_inf() : (z_id[0] - t.m) * g.inv_tau - l2 * kLn2;
      g.logprob[row] = lp;
      g.entropy[row] = ent;
      if (g.stats) reinterpret_cast<float4*>(g.stats)[row] = make_float4(t.m, l2, ent, 0.f);
    }
    if constexpr (TOPK) {
      if (tid < g.k) {
        const float v = top.ov[tid];
        const int i = top.oi[tid];
        g.top_ids[row * g.k + tid] = i;
        g.top_logprob[row * g.k + tid] = i < 0 ? neg_inf() : (v - t.m) * g.inv_tau - l2 * kLn2;
      }
    }
  }
}

// ---- backward ------------------------------------------------------------------------
template <typename T, bool DISTILL>
__global__ void __launch_bounds__(kThreads) vocab_bwd_kernel(VocabArgs g) {
  constexpr int N = Elem<T>::N;
  __shared__ int sid[DISTILL ? kVocabMaxTeacher : 1];
  __shared__ float sp[DISTILL ? kVocabMaxTeacher : 1];
  const int tid = threadIdx.x;
  // the last rows first: a forward just before has left them in L2 (83 -> 78 us at 4096 x 32768 bf16)
  const long long row = g.rows - 1 - blockIdx.x / g.chunks;
  const int part = (int)(blockIdx.x % g.chunks);
  const int lo = part * g.chunk, hi = min(lo + g.chunk, g.V), len = hi - lo;
  const T* p = row_ptr<T>(g, row) + lo;
  T* d = static_cast<T*>(g.dz) + row * g.V + lo;
  const float4 st = reinterpret_cast<const float4*>(g.stats)[row];
  const float m = st.x, l2 = st.y, c2 = g.inv_tau * kLog2e;
  float alpha, beta = 0.f, extra = 0.f;  // beta per unit of log2 q
  long long tok = -1;
  if (DISTILL) {
    const float gl = g.g0 ? g.g0[row * g.g0_stride] : 0.f;
    alpha = gl != 0.f && st.z != 0.f ? gl * g.tau * st.z : 0.f;  // st.z: 1, or NaN for an id past the vocabulary
    extra = -alpha;
  } else {
    tok = g.tokens[row];
    float glp = !g.g0 || tok < 0 ? 0.f : g.g0[row * g.g0_stride];
    if (glp != 0.f && tok >= g.V) glp = quiet_nan();
    const float gh = g.g1 ? g.g1[row * g.g1_stride] : 0.f;
    alpha = -(gh != 0.f ? fmaf(gh, st.z, glp) : glp) * g.inv_tau;
    beta = -gh * g.inv_tau * kLn2;
    extra = glp * g.inv_tau;
  }
  // no gradient comes in, or the row has no distribution: zeros, without a read
  const bool zero = m == neg_inf() || (alpha == 0.f && beta == 0.f && extra == 0.f);
  auto grad = [&](float z) {
    const float y = (z - m) * c2 - l2;
    const float q = ex2(y);
    return DISTILL ? q * alpha : q * fmaf(beta, fmaxf(y, kFar), alpha);
  };
  const bool phase = ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(d)) & 15) == 0;
  const int head = head_of(d, len);
  const int nvec = phase || zero ? (len - head) / N : 0;
  uint4* dv = reinterpret_cast<uint4*>(d + head);
  if (zero) {
    for (int i = tid; i < nvec; i += kThreads) dv[i] = make_uint4(0, 0, 0, 0);
  } else {
    const uint4* pv = reinterpret_cast<const uint4*>(p + head);
    for (int base = 0; base < nvec; base += kThreads * kUnroll) {
      uint4 r[kUnroll];
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        const int i = base + k * kThreads + tid;
        if (i < nvec) r[k] = __ldg(pv + i);
      }
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        const int i = base + k * kThreads + tid;
        if (i < nvec) {
          float v[N];
          Elem<T>::unpack(r[k], v);
#pragma unroll
          for (int j = 0; j < N; ++j) v[j] = grad(v[j]);
          dv[i] = Elem<T>::pack(v);
        }
      }
    }
  }
  auto edge = [&](int i) { d[i] = Elem<T>::down(zero ? 0.f : grad(Elem<T>::one(p + i))); };
  if (tid < head) edge(tid);
  for (int i = head + nvec * N + tid; i < len; i += kThreads) edge(i);
  if (zero) return;
  if (DISTILL) {
    for (int k = tid; k < g.K; k += kThreads) {
      const long long id = g.ids[row * g.K + k];
      sid[k] = id >= lo && id < hi ? (int)(id - lo) : -1;
      sp[k] = g.probs[row * g.K + k];
    }
    __syncthreads();  // also: the body's stores of this block come first
    for (int k = tid; k < g.K; k += kThreads) {
      const int id = sid[k];
      if (id < 0) continue;
      float sum = 0.f;
      bool first = true;
      for (int j = 0; j < g.K; ++j)
        if (sid[j] == id) {
          first = first && j >= k;
          sum += sp[j];
        }
      if (first) d[id] = Elem<T>::down(fmaf(extra, sum, grad(Elem<T>::one(p + id))));
    }
  } else {
    __syncthreads();
    if (tid == 0 && tok >= lo && tok < hi) {
      const int id = (int)(tok - lo);
      d[id] = Elem<T>::down(extra + grad(Elem<T>::one(p + id)));
    }
  }
}

template <typename T, bool DISTILL, bool TOPK, int NT>
cudaError_t launch_fwd_one(const VocabArgs& a, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.rows * a.cluster));
  cfg.blockDim = dim3(NT);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)a.cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = a.cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, vocab_fwd_kernel<T, DISTILL, TOPK, NT>, a);
}

template <typename T, int NT>
cudaError_t launch_fwd_sized(const VocabArgs& a, bool distill, cudaStream_t st) {
  if (distill) return launch_fwd_one<T, true, false, NT>(a, st);
  return a.k > 0 ? launch_fwd_one<T, false, true, NT>(a, st) : launch_fwd_one<T, false, false, NT>(a, st);
}
// Many rows: blocks of 128 threads, whose reductions cost half as much (176 -> 134 us at 8192 x 32003
// fp16 with 5 alternatives); below 8 rows an SM 256 threads, for the reads in flight (62 -> 55 us
// forward and backward at 517 x 50001 fp32).
template <typename T>
cudaError_t launch_fwd_typed(const VocabArgs& a, bool distill, int num_sms, cudaStream_t st) {
  return a.rows < 8LL * num_sms ? launch_fwd_sized<T, 256>(a, distill, st) : launch_fwd_sized<T, 128>(a, distill, st);
}

template <typename T>
cudaError_t launch_bwd_typed(const VocabArgs& a, bool distill, cudaStream_t st) {
  const unsigned blocks = (unsigned)(a.rows * a.chunks);
  if (distill) vocab_bwd_kernel<T, true><<<blocks, kThreads, 0, st>>>(a);
  else vocab_bwd_kernel<T, false><<<blocks, kThreads, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_vocab_fwd(VocabArgs a, int dtype, bool distill, int num_sms, cudaStream_t st) {
  // blocks per row: up to 8 while the GPU has room for them and each keeps 4096 values
  a.cluster = 1;
  while (a.cluster < 8 && a.rows * a.cluster * 2 <= 4LL * num_sms && a.V / (a.cluster * 2) >= 4096) a.cluster *= 2;
  a.chunk = round_up((a.V + a.cluster - 1) / a.cluster, 64);
  if (a.rows * a.cluster > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  switch (dtype) {
    case 0: return launch_fwd_typed<float>(a, distill, num_sms, st);
    case 1: return launch_fwd_typed<__nv_bfloat16>(a, distill, num_sms, st);
    default: return launch_fwd_typed<__half>(a, distill, num_sms, st);
  }
}

cudaError_t launch_vocab_bwd(VocabArgs a, int dtype, bool distill, cudaStream_t st) {
  a.chunk = dtype == 0 ? 8192 : 16384;  // 32 KB: two rounds of loads a thread
  a.chunks = (a.V + a.chunk - 1) / a.chunk;
  if (a.rows * a.chunks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  switch (dtype) {
    case 0: return launch_bwd_typed<float>(a, distill, st);
    case 1: return launch_bwd_typed<__nv_bfloat16>(a, distill, st);
    default: return launch_bwd_typed<__half>(a, distill, st);
  }
}

}  // namespace ltc
