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
// The k best ride in the same pass: the first window with a finite value gives a threshold
// that at least k of its values reach (the ceil(k/8)-th largest lane maximum, least over
// the 8 warps); later values are kept where they beat it, and the list is cut to its k
// best whenever half full, which raises the threshold.  A row that overruns the list (a
// long rising run, a row of equal values) is searched k times instead: slow and right.
// Ties go to the lowest index.
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

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kUnroll = 4;     // 16-byte loads in flight per thread
constexpr int kCap = 2048;     // candidate list; one vector per thread of a 16-bit type fits
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kFar = -1e30f; // stands for -inf where a zero weight multiplies it

// ---- element types ---------------------------------------------------------------
template <typename T> struct Elem;
template <> struct Elem<float> {
  static constexpr int N = 4;  // per 16 bytes
  static constexpr unsigned kNegInf = 0xff800000u;
  __device__ static void unpack(const uint4& r, float (&v)[4]) {
    v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y);
    v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
  }
  __device__ static uint4 pack(const float (&v)[4]) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
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
  __device__ static void unpack(const uint4& r, float (&v)[8]) {
    two(r.x, v[0], v[1]); two(r.y, v[2], v[3]); two(r.z, v[4], v[5]); two(r.w, v[6], v[7]);
  }
  __device__ static unsigned p2(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<unsigned*>(&h);
  }
  __device__ static uint4 pack(const float (&v)[8]) {
    return make_uint4(p2(v[0], v[1]), p2(v[2], v[3]), p2(v[4], v[5]), p2(v[6], v[7]));
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
  __device__ static void unpack(const uint4& r, float (&v)[8]) {
    two(r.x, v[0], v[1]); two(r.y, v[2], v[3]); two(r.z, v[4], v[5]); two(r.w, v[6], v[7]);
  }
  __device__ static unsigned p2(float a, float b) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<unsigned*>(&h);
  }
  __device__ static uint4 pack(const float (&v)[8]) {
    return make_uint4(p2(v[0], v[1]), p2(v[2], v[3]), p2(v[4], v[5]), p2(v[6], v[7]));
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
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
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
  return static_cast<const T*>(g.z) + (row / g.n1) * g.s0 + (row % g.n1) * g.s1;
}

// elements before the first 16-byte boundary of p (at most len)
template <typename T>
__device__ __forceinline__ int head_of(const T* p, int len) {
  const int mis = (int)(reinterpret_cast<uintptr_t>(p) & 15);
  const int h = mis ? (16 - mis) / (int)sizeof(T) : 0;
  return h < len ? h : len;
}

// k best of n candidates, best first, (-inf, -1) where there are fewer; all threads call it
__device__ void select_best(const float* cv, const int* ci, int n, int k, float* ov, int* oi) {
  for (int j = threadIdx.x; j < k; j += kThreads) {
    ov[j] = neg_inf();
    oi[j] = -1;
  }
  __syncthreads();
  for (int c = threadIdx.x; c < n; c += kThreads) {
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

struct TopShared {
  float cv[kCap];
  int ci[kCap];
  float ov[kVocabMaxTop];
  int oi[kVocabMaxTop];
  float warp_v[kWarps];
  int warp_i[kWarps];
  int count;
  float pv;
  int pi;
};
struct NoShared {};

// ---- forward -----------------------------------------------------------------------
template <typename T, bool DISTILL, bool TOPK>
__global__ void __launch_bounds__(kThreads) vocab_fwd_kernel(VocabArgs g) {
  constexpr int N = Elem<T>::N;
  __shared__ Sums warp_sums[kWarps];
  __shared__ Sums block_sums;
  __shared__ typename std::conditional<TOPK, TopShared, NoShared>::type top;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cs = g.cluster, rank = cs > 1 ? (int)(blockIdx.x % cs) : 0;
  const long long row = blockIdx.x / cs;
  const T* zr = row_ptr<T>(g, row);
  const int lo = min(rank * g.chunk, g.V), hi = min(lo + g.chunk, g.V);
  const T* p = zr + lo;
  const int len = hi - lo;
  const int head = head_of(p, len);
  const int nvec = (len - head) / N;
  const uint4* pv = reinterpret_cast<const uint4*>(p + head);
  const float c2 = g.inv_tau * kLog2e;

  Sums a{neg_inf(), 0.f, 0.f};
  float thr = neg_inf();  // a value has to beat it (equal counts in the window that set it)
  bool slow = false;
  int mine = 0;  // length of the list behind this thread's latest entry
  if constexpr (TOPK) {
    if (tid == 0) top.count = 0;
    __syncthreads();
  }
  auto keep = [&](float v, int i) {
    if constexpr (TOPK) {
      const int at = atomicAdd(&top.count, 1);
      if (at < kCap) {
        top.cv[at] = v;
        top.ci[at] = i;
      }
      mine = at + 1;
    }
  };
  auto single = [&](float v, int i) {  // a value outside the aligned body
    const float mn = max_nan(a.m, v);
    if (mn == neg_inf()) return;
    if (mn != a.m) move_to(a, mn, c2);
    const float y = (v - a.m) * c2, e = ex2(y);
    a.s += e;
    a.u = fmaf(e, fmaxf(y, kFar), a.u);
    if (TOPK && !slow && v > thr) keep(v, i);
  };

  if (tid < head) single(Elem<T>::one(p + tid), lo + tid);

  for (int base = 0; base < nvec; base += kThreads * kUnroll) {
    uint4 r[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      const int i = base + k * kThreads + tid;
      r[k] = i < nvec ? __ldg(pv + i) : make_uint4(Elem<T>::kNegInf, Elem<T>::kNegInf, Elem<T>::kNegInf, Elem<T>::kNegInf);
    }
    float v[kUnroll][N];
    float top_v = neg_inf();
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      Elem<T>::unpack(r[k], v[k]);
#pragma unroll
      for (int j = 0; j < N; ++j) top_v = max_nan(top_v, v[k][j]);
    }
    const float mn = max_nan(a.m, top_v);
    if (mn != neg_inf()) {
      if (mn != a.m) move_to(a, mn, c2);
#pragma unroll
      for (int k = 0; k < kUnroll; ++k)
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float y = (v[k][j] - mn) * c2, e = ex2(y);
          a.s += e;
          if (!DISTILL) a.u = fmaf(e, fmaxf(y, kFar), a.u);
        }
    }
    if constexpr (TOPK) {
      if (!slow) {
        bool equal = false;
        if (thr == neg_inf()) {  // the same for all threads
          // the need-th largest lane maximum of this warp, then the least of the warps
          const int need = (g.k + kWarps - 1) / kWarps;
          float x = top_v == top_v ? top_v : neg_inf(), w = neg_inf();
          for (int q = 0; q < need; ++q) {
            w = x;
#pragma unroll
            for (int d = 16; d >= 1; d >>= 1) w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, d));
            const unsigned who = __ballot_sync(0xffffffffu, x == w);
            if (lane == __ffs(who) - 1) x = neg_inf();
          }
          if (lane == 0) top.warp_v[warp] = w;
          __syncthreads();
          thr = top.warp_v[0];
#pragma unroll
          for (int q = 1; q < kWarps; ++q) thr = fminf(thr, top.warp_v[q]);
          equal = true;
        }
        if (top_v > thr || equal || top_v != top_v) {
#pragma unroll
          for (int k = 0; k < kUnroll; ++k)
#pragma unroll
            for (int j = 0; j < N; ++j) {
              const float x = v[k][j];
              if (x > thr || (equal && x == thr && x > neg_inf()))
                keep(x, lo + head + (base + k * kThreads + tid) * N + j);
            }
        }
        if (__syncthreads_or(mine > kCap / 2)) {
          const int n = top.count;
          if (n > kCap) {
            slow = true;
          } else {
            select_best(top.cv, top.ci, n, g.k, top.ov, top.oi);
            if (tid < g.k) {
              top.cv[tid] = top.ov[tid];
              top.ci[tid] = top.oi[tid];
            }
            thr = top.ov[g.k - 1];
            __syncthreads();
            if (tid == 0) top.count = g.k;
          }
          mine = 0;
          __syncthreads();
        }
      }
    }
  }
  for (int i = head + nvec * N + tid; i < len; i += kThreads) single(Elem<T>::one(p + i), lo + i);

  // block sums, in lane and warp order
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) {
    Sums b;
    b.m = __shfl_xor_sync(0xffffffffu, a.m, d);
    b.s = __shfl_xor_sync(0xffffffffu, a.s, d);
    b.u = __shfl_xor_sync(0xffffffffu, a.u, d);
    a = merge(a, b, c2);
  }
  if (lane == 0) warp_sums[warp] = a;
  __syncthreads();
  if (tid == 0) {
    Sums b = warp_sums[0];
    for (int w = 1; w < kWarps; ++w) b = merge(b, warp_sums[w], c2);
    block_sums = b;
  }

  if constexpr (TOPK) {
    // the tail's entries came after the last look at the list's length
    const int n = top.count;
    slow = slow || n > kCap;
    __syncthreads();
    if (!slow) {
      select_best(top.cv, top.ci, n, g.k, top.ov, top.oi);
    } else {
      float pbest = __int_as_float(0x7f800000);
      int ibest = -1;
      for (int q = 0; q < g.k; ++q) {
        float bv = neg_inf();
        int bi = 0x7fffffff;
        for (int i = tid; i < len; i += kThreads) {
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
          for (int w = 1; w < kWarps; ++w)
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
    cl.sync();
    if (rank == 0) {
      if (tid == 0) {
        Sums b = block_sums;
        for (int r = 1; r < cs; ++r) b = merge(b, *cl.map_shared_rank(&block_sums, r), c2);
        warp_sums[0] = b;
      }
      if constexpr (TOPK) {
        for (int c = tid; c < cs * g.k; c += kThreads) {
          const int r = c / g.k, j = c - r * g.k;
          top.cv[c] = cl.map_shared_rank(&top.ov[0], r)[j];
          top.ci[c] = cl.map_shared_rank(&top.oi[0], r)[j];
        }
      }
    }
    cl.sync();  // the others' shared memory has been read
    if (rank != 0) return;
    if (tid == 0) block_sums = warp_sums[0];
    if constexpr (TOPK) select_best(top.cv, top.ci, cs * g.k, g.k, top.ov, top.oi);
  }
  __syncthreads();
  const Sums t = block_sums;
  const bool empty = t.m == neg_inf();
  const float l2 = empty ? 0.f : log2f(t.s);

  if constexpr (DISTILL) {
    if (warp != 0) return;
    const long long* ids = g.ids + row * g.K;
    bool any = false, bad = false;
    float tm = neg_inf();
    for (int k = lane; k < g.K; k += 32) {
      if (ids[k] < 0) continue;
      any = true;
      bad = bad || ids[k] >= g.V;
      tm = max_nan(tm, teacher_at(g.teacher, g.teacher_dtype, row * g.K + k));
    }
    any = __any_sync(0xffffffffu, any);
    bad = __any_sync(0xffffffffu, bad);
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) tm = max_nan(tm, __shfl_xor_sync(0xffffffffu, tm, d));
    any = any && tm != neg_inf();  // entries that are all -inf leave no distribution either
    float ts = 0.f;
    for (int k = lane; k < g.K && any; k += 32)
      if (ids[k] >= 0) ts += ex2((teacher_at(g.teacher, g.teacher_dtype, row * g.K + k) - tm) * c2);
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) ts += __shfl_xor_sync(0xffffffffu, ts, d);
    const float lt = any ? log2f(ts) : 0.f;
    float loss = 0.f;
    for (int k = lane; k < g.K; k += 32) {
      float pk = 0.f;
      if (any && ids[k] >= 0) {
        const float lp = (teacher_at(g.teacher, g.teacher_dtype, row * g.K + k) - tm) * c2 - lt;
        pk = ex2(lp);
        if (pk != 0.f && ids[k] < g.V) {
          const float lq = empty ? neg_inf() : (Elem<T>::one(zr + ids[k]) - t.m) * c2 - l2;
          loss = fmaf(pk, lp - lq, loss);
        }
      }
      if (g.probs) g.probs[row * g.K + k] = pk;
    }
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) loss += __shfl_xor_sync(0xffffffffu, loss, d);
    if (lane == 0) {
      g.loss[row] = bad ? quiet_nan() : loss * (g.tau * g.tau * kLn2);
      if (g.stats) reinterpret_cast<float4*>(g.stats)[row] = make_float4(t.m, l2, bad ? quiet_nan() : any ? 1.f : 0.f, 0.f);
    }
  } else {
    const float ent = empty ? 0.f : (l2 - t.u / t.s) * kLn2;
    if (tid == 0) {
      const long long tok = g.tokens[row];
      float lp = 0.f;
      if (tok >= g.V) lp = quiet_nan();
      else if (tok >= 0) lp = empty ? neg_inf() : (Elem<T>::one(zr + tok) - t.m) * g.inv_tau - l2 * kLn2;
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
  const long long row = blockIdx.x / g.chunks;
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
    alpha = st.z != 0.f ? gl * g.tau * st.z : 0.f;  // st.z: 1, or NaN for an id past the vocabulary
    extra = -alpha;
  } else {
    tok = g.tokens[row];
    const float glp = !g.g0 || tok < 0 ? 0.f : tok < g.V ? g.g0[row * g.g0_stride] : quiet_nan();
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

template <typename T, bool DISTILL, bool TOPK>
cudaError_t launch_fwd_one(const VocabArgs& a, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.rows * a.cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)a.cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = a.cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, vocab_fwd_kernel<T, DISTILL, TOPK>, a);
}

template <typename T>
cudaError_t launch_fwd_typed(const VocabArgs& a, bool distill, cudaStream_t st) {
  if (distill) return launch_fwd_one<T, true, false>(a, st);
  return a.k > 0 ? launch_fwd_one<T, false, true>(a, st) : launch_fwd_one<T, false, false>(a, st);
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
    case 0: return launch_fwd_typed<float>(a, distill, st);
    case 1: return launch_fwd_typed<__nv_bfloat16>(a, distill, st);
    default: return launch_fwd_typed<__half>(a, distill, st);
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
