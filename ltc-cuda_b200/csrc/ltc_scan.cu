// Linear recurrences over time, one independent chain per (sequence, channel):
//   linear scan   h_t = a_t h_{t-1} + b_t                     (a, b given)
//   gated scan    L_t = -scale softplus(decay) sigmoid(rate_t),  a_t = exp(L_t),
//                 b_t = sqrt(1 - a_t^2) sigmoid(gate_t) x_t   (gates computed here)
// and their backward pass, in fp32 whatever the type of the inputs.
//
// Mathematics.  A run of tokens maps the state before it to the state behind it,
// h -> A h + B, and two runs compose as (A2 A1, A2 B1 + B2).  With c_t = a_t lambda_t the
// adjoint lambda_t = dh_t + a_{t+1} lambda_{t+1} runs backwards by the same kind of map,
// c -> A c + B with B folded from the far end, over the SAME product A.
//
// Work split.  A tile is TY x R tokens by LX x VEC channels: a thread keeps R consecutive
// tokens of VEC channels in registers, folds them to one (A, B), the fold is combined
// over the tile's TY threads (shuffles inside a warp, shared memory across warps, one
// barrier per tile), and the thread then runs its tokens again from its own first state.
// A group of threads marches over its tiles with the state in registers, so every input
// is read once.  Where there are too few (sequence, channel) chains to fill the GPU, time
// is cut into segments: a first launch folds each segment to (A, B), the second starts
// each segment from the fold of the earlier ones (fixed order: results do not depend on
// scheduling; nothing waits inside a kernel).
//
// Backward.  The forward leaves the state before each tile (fp32, one row in 16 or 64
// tokens); the backward rebuilds the states of a tile from it in registers instead of
// reading h, which is both one tensor less and exact where h was rounded to 16 bits.
//
// Packed sequences: token t that starts sequence n is a cut, h_t = a_t h0[n] + b_t whatever came
// before, and a run that holds one is a constant map; tokens outside every sequence give h = 0 and zero gradients.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ltc_common.cuh"
#include "ltc_internal.h"

namespace ltc {

namespace {

constexpr int kThreads = 128;

// ---- element types -------------------------------------------------------------
template <typename T, int VEC> struct Raw;  // VEC elements as loaded
template <> struct Raw<float, 4> { using type = float4; };
template <> struct Raw<float, 1> { using type = float; };
template <> struct Raw<__nv_bfloat16, 4> { using type = uint2; };
template <> struct Raw<__nv_bfloat16, 1> { using type = unsigned short; };
template <> struct Raw<__half, 4> { using type = uint2; };
template <> struct Raw<__half, 1> { using type = unsigned short; };

__device__ __forceinline__ float2 up2(unsigned v, __nv_bfloat16) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
__device__ __forceinline__ float2 up2(unsigned v, __half) {
  return __half22float2(*reinterpret_cast<__half2*>(&v));
}
__device__ __forceinline__ unsigned down2(float x, float y, __nv_bfloat16) {
  __nv_bfloat162 p = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<unsigned*>(&p);
}
__device__ __forceinline__ unsigned down2(float x, float y, __half) {
  __half2 p = __floats2half2_rn(x, y);
  return *reinterpret_cast<unsigned*>(&p);
}

__device__ __forceinline__ void unpack(const float4& r, float (&v)[4], float) {
  v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w;
}
template <typename T>
__device__ __forceinline__ void unpack(const uint2& r, float (&v)[4], T) {
  const float2 lo = up2(r.x, T()), hi = up2(r.y, T());
  v[0] = lo.x; v[1] = lo.y; v[2] = hi.x; v[3] = hi.y;
}
__device__ __forceinline__ void unpack(const float& r, float (&v)[1], float) { v[0] = r; }
template <typename T>
__device__ __forceinline__ void unpack(const unsigned short& r, float (&v)[1], T) {
  v[0] = up2(r, T()).x;
}

__device__ __forceinline__ void store(float* p, const float (&v)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store(float* p, const float (&v)[1]) { *p = v[0]; }
template <typename T>
__device__ __forceinline__ void store(T* p, const float (&v)[4]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(down2(v[0], v[1], T()), down2(v[2], v[3], T()));
}
template <typename T>
__device__ __forceinline__ void store(T* p, const float (&v)[1]) {
  *reinterpret_cast<unsigned short*>(p) = (unsigned short)(down2(v[0], 0.f, T()) & 0xffffu);
}
__device__ __forceinline__ void load_f32(const float* p, float (&v)[4]) {
  const float4 r = *reinterpret_cast<const float4*>(p);
  v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w;
}
__device__ __forceinline__ void load_f32(const float* p, float (&v)[1]) { v[0] = *p; }

template <typename T, int VEC>
__device__ __forceinline__ typename Raw<T, VEC>::type load_raw(const void* base, long long off, bool ok) {
  using V = typename Raw<T, VEC>::type;
  V r{};
  if (ok) r = __ldg(reinterpret_cast<const V*>(static_cast<const T*>(base) + off));
  return r;
}

// ---- gates ---------------------------------------------------------------------
// fp32 inputs take the library's expf; 16-bit inputs __expf (2 ulp plus the rounding of
// its argument, far below the inputs' own 2^-9)
template <typename T> __device__ __forceinline__ float exp_of(float x) { return __expf(x); }
template <> __device__ __forceinline__ float exp_of<float>(float x) { return expf(x); }

template <typename T>
__device__ __forceinline__ float sigmoid_of(float x) { return rcp_approx(1.f + exp_of<T>(-x)); }

// 1 - exp(y), y <= 0.  Near 0, where 1 - exp(y) cancels, the Taylor series of
// -(exp(y) - 1), whose first left-out term is below 2^-24 of the sum for y > -1/4; past
// it 1 - e is at least 0.22.
__device__ __forceinline__ float one_minus_exp(float y, float e) {
  float p = fmaf(y, 1.f / 720.f, 1.f / 120.f);
  p = fmaf(y, p, 1.f / 24.f);
  p = fmaf(y, p, 1.f / 6.f);
  p = fmaf(y, p, 0.5f);
  p = fmaf(y, p, 1.f);
  return y > -0.25f ? -y * p : 1.f - e;
}

__device__ __forceinline__ float sqrt_approx(float x) {
  float y;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float softplus_of(float x) { return x > 20.f ? x : log1pf(expf(x)); }

struct Gate {
  float sr, sg, a, beta;
};
// cs = -scale * softplus(decay)
template <typename T>
__device__ __forceinline__ Gate gate_of(float rate, float gate, float cs) {
  Gate g;
  g.sr = sigmoid_of<T>(rate);
  g.sg = sigmoid_of<T>(gate);
  const float L = cs * g.sr;
  g.a = exp_of<T>(L);
  g.beta = sqrt_approx(one_minus_exp(2.f * L, g.a * g.a));
  return g;
}

// h -> a h + b, or b behind a cut: where a packed sequence starts, whatever the earlier one
// holds stops there, infinities and NaN too, which a zero factor would let through.  (An
// underflown product is no cut: a NaN goes on through it as in the definition.)
template <bool PACKED>
__device__ __forceinline__ float flow(bool cut, float a, float h, float b) {
  return PACKED && cut ? b : fmaf(a, h, b);
}

// ---- packed sequences ------------------------------------------------------------
// largest n < S with starts[n] <= t (0 if there is none); in bounds for any contents
__device__ __forceinline__ int seq_of(const int* starts, int S, int t) {
  int lo = 0, hi = S;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(starts + mid) <= t) lo = mid; else hi = mid;
  }
  return lo;
}

struct Marks {         // of a thread's R tokens, one bit each
  unsigned first = 0;  // starts its sequence
  unsigned last = 0;   // ends it
  unsigned out = 0;    // belongs to none
  int n0 = 0;          // sequence of the first token
};
template <int R>
__device__ __forceinline__ Marks marks_of(const int* starts, int S, int t0, int T) {
  Marks m;
  m.n0 = seq_of(starts, S, t0);
  const int end = min(__ldg(starts + S), T), begin = __ldg(starts);
  int n = m.n0, s0 = __ldg(starts + n), s1 = __ldg(starts + n + 1);
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int t = t0 + j;
    while (t >= s1 && n + 1 < S) {
      ++n;
      s0 = s1;
      s1 = __ldg(starts + n + 1);
    }
    const bool in = t >= begin && t < end;
    m.out |= (in ? 0u : 1u) << j;
    m.first |= (in && t == s0 ? 1u : 0u) << j;
    m.last |= (in && t + 1 == s1 ? 1u : 0u) << j;
  }
  return m;
}

// ---- one tile's fold over the threads of a group -----------------------------------
// NF forward folds and NR reverse folds share the product A.  LX lanes hold different
// channels; the TY threads with the same channels hold consecutive tokens.
template <int LX, int TY>
struct Geo {
  static constexpr int GPW = 32 / LX;       // time groups inside a warp
  static constexpr int NW = TY / GPW > 0 ? TY / GPW : 1;  // warps along time
  static_assert(TY % GPW == 0, "a warp's time groups belong to one tile");
};

// ---- forward -----------------------------------------------------------------------
template <int P, typename T, int VEC, int LX, int TY, int R, int BB, bool PACKED>
__global__ void __launch_bounds__(kThreads) scan_fwd_kernel(ScanArgs g) {
  using G = Geo<LX, TY>;
  static_assert(LX * TY * BB == kThreads, "block shape");
  static_assert(BB == 1 || G::NW == 1, "several items per block only without block barriers");
  static_assert(!PACKED || G::NW > 1, "the one-warp tiles do not look at cuts");
  constexpr int NIN = P ? 3 : 2;
  constexpr int TT = TY * R;
  __shared__ float sA[2][G::NW][LX * VEC], sB[2][G::NW][LX * VEC];
  __shared__ int sF[2][G::NW];
  const int lane = threadIdx.x & 31;
  const int lx = threadIdx.x % LX, ty = (threadIdx.x / LX) % TY;
  const int grp = ty % G::GPW, wt = ty / G::GPW;  // group in the warp, warp along time
  const long long item = (long long)blockIdx.x * BB + threadIdx.x / (LX * TY);
  if (BB > 1 && item >= g.items) return;  // whole warps leave; no block barrier follows
  const int cb = (int)(item % g.chb);
  const long long rest = item / g.chb;
  const int seg = (int)(rest % g.launch_segs);
  const long long b = rest / g.launch_segs;
  const int ch = cb * LX * VEC + lx * VEC;
  const bool chok = ch < g.H;
  const int tile0 = seg * g.seg_tiles, tile1 = min(tile0 + g.seg_tiles, g.tiles);

  float cs[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) cs[v] = 0.f;
  if (P && chok) {
    load_f32(g.decay + ch, cs);
#pragma unroll
    for (int v = 0; v < VEC; ++v) cs[v] = -g.scale * softplus_of(cs[v]);
  }

  // state before the segment; in the folding launch (0, 1) so that carry and prod become B and A
  float carry[VEC], prod[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) { carry[v] = 0.f; prod[v] = 1.f; }
  bool cut_all = false;
  if (!g.fold_only && chok) {
    if (!PACKED && g.h0) load_f32(g.h0 + b * g.H + ch, carry);
    const float* ag = g.agg + (b * g.nseg * 2) * (long long)g.H + ch;
    for (int s = 0; s < seg; ++s, ag += 2 * (long long)g.H) {
      float fa[VEC], fb[VEC];
      load_f32(ag, fa);
      load_f32(ag + g.H, fb);
      const bool cut = PACKED && g.seg_cut[s] != 0;
#pragma unroll
      for (int v = 0; v < VEC; ++v) carry[v] = flow<PACKED>(cut, fa[v], carry[v], fb[v]);
    }
  }

  for (int tile = tile0; tile < tile1; ++tile) {
    const int t0 = tile * TT + ty * R;
    typename Raw<T, VEC>::type raw[NIN][R];
#pragma unroll
    for (int i = 0; i < NIN; ++i)
#pragma unroll
      for (int j = 0; j < R; ++j)
        raw[i][j] = load_raw<T, VEC>(g.in[i], b * g.sb[i] + (long long)(t0 + j) * g.st[i] + ch,
                                     chok && t0 + j < g.T);
    Marks m;
    if (PACKED) m = marks_of<R>(g.starts, g.S, t0, g.T);
    const unsigned cuts = PACKED ? m.first | m.out : 0u;
    if (!g.fold_only && g.bounds && ty == 0 && chok && tile > 0)
      store(g.bounds + (b * g.tiles + tile) * g.H + ch, carry);

    float a[R][VEC], bv[R][VEC], A[VEC], B[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) { A[v] = 1.f; B[v] = 0.f; }
#pragma unroll
    for (int j = 0; j < R; ++j) {
      float x[VEC], y[VEC], z[VEC];
      unpack(raw[0][j], x, T());
      unpack(raw[1][j], y, T());
      if (P) unpack(raw[NIN - 1][j], z, T());
      if (PACKED && ((m.out >> j) & 1u)) {  // whatever lies between and behind the sequences is not used
#pragma unroll
        for (int v = 0; v < VEC; ++v) x[v] = y[v] = z[v] = 0.f;
      }
      const bool live = t0 + j < g.T;
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        if (P) {
          const Gate q = gate_of<T>(y[v], z[v], cs[v]);
          a[j][v] = q.a;
          bv[j][v] = q.beta * q.sg * x[v];
        } else {
          a[j][v] = x[v];
          bv[j][v] = y[v];
        }
        if (!live) { a[j][v] = 1.f; bv[j][v] = 0.f; }
      }
      if (PACKED && live) {
        if ((m.out >> j) & 1u) {
#pragma unroll
          for (int v = 0; v < VEC; ++v) bv[j][v] = 0.f;
        } else if (((m.first >> j) & 1u) && g.h0 && chok) {
          float s[VEC];
          load_f32(g.h0 + (long long)seq_of(g.starts, g.S, t0 + j) * g.H + ch, s);
#pragma unroll
          for (int v = 0; v < VEC; ++v) bv[j][v] = fmaf(a[j][v], s[v], bv[j][v]);
        }
      }
      const bool cut = (cuts >> j) & 1u;
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        B[v] = flow<PACKED>(cut, a[j][v], B[v], bv[j][v]);
        A[v] *= a[j][v];
      }
    }
    int F = cuts != 0;  // the run holds a cut: its A counts for nothing

    // inclusive fold over the warp's time groups, then this thread's exclusive one
    float Ax[VEC], Bx[VEC];
#pragma unroll
    for (int d = 1; d < G::GPW; d *= 2) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const float pa = __shfl_up_sync(0xffffffffu, A[v], d * LX);
        const float pb = __shfl_up_sync(0xffffffffu, B[v], d * LX);
        if (grp >= d) {
          B[v] = flow<PACKED>(F, A[v], pb, B[v]);
          A[v] *= pa;
        }
      }
      if (PACKED) {
        const int pf = __shfl_up_sync(0xffffffffu, F, d * LX);
        if (grp >= d) F |= pf;
      }
    }
    const int Fx = PACKED && G::GPW > 1 ? __shfl_up_sync(0xffffffffu, F, LX % 32) : 0;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      Ax[v] = G::GPW > 1 ? __shfl_up_sync(0xffffffffu, A[v], LX % 32) : 1.f;
      Bx[v] = G::GPW > 1 ? __shfl_up_sync(0xffffffffu, B[v], LX % 32) : 0.f;
      if (grp == 0) { Ax[v] = 1.f; Bx[v] = 0.f; }
    }
    float h[VEC];
    if (G::NW > 1) {
      const int buf = tile & 1;  // the barrier of the next tile separates the reads from the next writes
      if (grp == G::GPW - 1) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          sA[buf][wt][lx * VEC + v] = A[v];
          sB[buf][wt][lx * VEC + v] = B[v];
        }
        if (PACKED && lx == 0) sF[buf][wt] = F;
      }
      __syncthreads();
#pragma unroll
      for (int w = 0; w < G::NW; ++w) {
        const bool cut = PACKED && sF[buf][w] != 0;
        cut_all = cut_all || cut;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          if (w == wt) h[v] = carry[v];
          const float wa = sA[buf][w][lx * VEC + v];
          carry[v] = flow<PACKED>(cut, wa, carry[v], sB[buf][w][lx * VEC + v]);
          prod[v] *= wa;
        }
      }
    } else {
      const int src = (lane & ~31) | ((G::GPW - 1) * LX + lx);
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const float wa = __shfl_sync(0xffffffffu, A[v], src);
        const float wb = __shfl_sync(0xffffffffu, B[v], src);
        h[v] = carry[v];
        carry[v] = fmaf(wa, carry[v], wb);
        prod[v] *= wa;
      }
    }
    if (g.fold_only) continue;

#pragma unroll
    for (int v = 0; v < VEC; ++v) h[v] = flow<PACKED>(Fx && grp > 0, Ax[v], h[v], Bx[v]);
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const bool cut = (cuts >> j) & 1u;
#pragma unroll
      for (int v = 0; v < VEC; ++v) h[v] = flow<PACKED>(cut, a[j][v], h[v], bv[j][v]);
      const int t = t0 + j;
      if (chok && t < g.T) {
        store(static_cast<T*>(g.h) + (b * g.T + t) * g.H + ch, h);
        if (PACKED && ((m.last >> j) & 1u))
          store(g.hT + (long long)seq_of(g.starts, g.S, t) * g.H + ch, h);
      }
    }
  }

  if (!chok) return;
  if (PACKED && !g.fold_only && seg == 0) {  // sequences without a token pass their first state on
    for (int n = ty; n < g.S; n += TY) {
      if (__ldg(g.starts + n) < __ldg(g.starts + n + 1)) continue;
      float s[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) s[v] = 0.f;
      if (g.h0) load_f32(g.h0 + (long long)n * g.H + ch, s);
      store(g.hT + (long long)n * g.H + ch, s);
    }
  }
  if (ty != 0) return;
  if (g.fold_only) {
    float* ag = g.agg + ((b * g.nseg + seg) * 2) * (long long)g.H + ch;
    store(ag, prod);
    store(ag + g.H, carry);
    if (PACKED) g.seg_cut[seg] = cut_all;  // the same from every block of channels
  } else if (!PACKED) {
    if (tile1 == g.tiles) store(g.hT + b * g.H + ch, carry);
  }
}

// ---- backward ----------------------------------------------------------------------
template <int P, typename T, int VEC, int LX, int TY, int R, int BB, bool PACKED>
__global__ void __launch_bounds__(kThreads) scan_bwd_kernel(ScanArgs g) {
  using G = Geo<LX, TY>;
  static_assert(LX * TY * BB == kThreads, "block shape");
  static_assert(BB == 1 || G::NW == 1, "several items per block only without block barriers");
  static_assert(!PACKED || G::NW > 1, "the one-warp tiles do not look at cuts");
  constexpr int NIN = P ? 3 : 2;
  constexpr int TT = TY * R;
  __shared__ float sA[2][G::NW][LX * VEC], sB[2][G::NW][LX * VEC], sC[2][G::NW][LX * VEC];
  __shared__ int sF[2][G::NW];
  const int lane = threadIdx.x & 31;
  const int lx = threadIdx.x % LX, ty = (threadIdx.x / LX) % TY;
  const int grp = ty % G::GPW, wt = ty / G::GPW;
  const long long item = (long long)blockIdx.x * BB + threadIdx.x / (LX * TY);
  if (BB > 1 && item >= g.items) return;
  const int cb = (int)(item % g.chb);
  const long long rest = item / g.chb;
  // the folding launch has no use for the first segment
  const int seg = (int)(rest % g.launch_segs) + (g.fold_only ? 1 : 0);
  const long long b = rest / g.launch_segs;
  const int ch = cb * LX * VEC + lx * VEC;
  const bool chok = ch < g.H;
  const int tile0 = seg * g.seg_tiles, tile1 = min(tile0 + g.seg_tiles, g.tiles);

  // decay gradient so far, and what its additions rounded away (a tile at a time)
  float cs[VEC], acc[VEC], lost[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) cs[v] = acc[v] = lost[v] = 0.f;
  if (P && chok) {
    load_f32(g.decay + ch, cs);
#pragma unroll
    for (int v = 0; v < VEC; ++v) cs[v] = -g.scale * softplus_of(cs[v]);
  }

  // c behind the segment
  float carry[VEC], prod[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) { carry[v] = 0.f; prod[v] = 1.f; }
  if (!g.fold_only && chok) {
    if (!PACKED && g.dhT) load_f32(g.dhT + b * g.H + ch, carry);
    for (int s = g.nseg - 1; s > seg; --s) {
      const float* ag = g.agg + ((b * g.nseg + s) * 2) * (long long)g.H + ch;
      float fa[VEC], fb[VEC];
      load_f32(ag, fa);
      load_f32(ag + g.H, fb);
      const bool cut = PACKED && g.seg_cut[s] != 0;
#pragma unroll
      for (int v = 0; v < VEC; ++v) carry[v] = flow<PACKED>(cut, fa[v], carry[v], fb[v]);
    }
  }
  bool cut_all = false;

  for (int tile = tile1 - 1; tile >= tile0; --tile) {
    const int t0 = tile * TT + ty * R;
    typename Raw<T, VEC>::type raw[NIN][R], rg[R];
#pragma unroll
    for (int i = 0; i < NIN; ++i) {
      // a folding launch needs the decay and the incoming gradient alone
      const bool need = !g.fold_only || (P ? i == 1 : i == 0);
#pragma unroll
      for (int j = 0; j < R; ++j)
        raw[i][j] = load_raw<T, VEC>(g.in[i], b * g.sb[i] + (long long)(t0 + j) * g.st[i] + ch,
                                     need && chok && t0 + j < g.T);
    }
#pragma unroll
    for (int j = 0; j < R; ++j)
      rg[j] = load_raw<T, VEC>(g.dh, b * g.sb[3] + (long long)(t0 + j) * g.st[3] + ch,
                               g.dh && chok && t0 + j < g.T);
    float h[VEC];  // state before the tile
#pragma unroll
    for (int v = 0; v < VEC; ++v) h[v] = 0.f;
    if (!g.fold_only && chok) {
      if (tile > 0) load_f32(g.bounds + (b * g.tiles + tile) * g.H + ch, h);
      else if (!PACKED && g.h0) load_f32(g.h0 + b * g.H + ch, h);
    }
    Marks m;
    if (PACKED) m = marks_of<R>(g.starts, g.S, t0, g.T);
    const unsigned cuts = PACKED ? m.first | m.out : 0u;

    // gates; forward fold (A, B) and reverse fold (A, C) of this thread's tokens
    float a[R][VEC], hp[R][VEC], sr[P ? R : 1][VEC], sg[P ? R : 1][VEC], be[P ? R : 1][VEC];
    float A[VEC], B[VEC], C[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) { A[v] = 1.f; B[v] = 0.f; C[v] = 0.f; }
#pragma unroll
    for (int j = 0; j < R; ++j) {
      float x[VEC], y[VEC], z[VEC];
      unpack(raw[0][j], x, T());
      unpack(raw[1][j], y, T());
      if (P) unpack(raw[NIN - 1][j], z, T());
      if (PACKED && ((m.out >> j) & 1u)) {  // whatever lies between and behind the sequences is not used
#pragma unroll
        for (int v = 0; v < VEC; ++v) x[v] = y[v] = z[v] = 0.f;
      }
      const bool live = t0 + j < g.T;
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        if (P) {
          const Gate q = gate_of<T>(y[v], z[v], cs[v]);
          a[j][v] = q.a;
          hp[j][v] = q.beta * q.sg * x[v];  // b_t, replaced below by the state before t
          sr[j][v] = q.sr;
          sg[j][v] = q.sg;
          be[j][v] = q.beta;
        } else {
          a[j][v] = x[v];
          hp[j][v] = y[v];
        }
        if (!live) { a[j][v] = 1.f; hp[j][v] = 0.f; }
      }
      if (PACKED && live) {
        if ((m.out >> j) & 1u) {
#pragma unroll
          for (int v = 0; v < VEC; ++v) hp[j][v] = 0.f;
        } else if (((m.first >> j) & 1u) && g.h0 && chok) {
          float s[VEC];
          load_f32(g.h0 + (long long)seq_of(g.starts, g.S, t0 + j) * g.H + ch, s);
#pragma unroll
          for (int v = 0; v < VEC; ++v) hp[j][v] = fmaf(a[j][v], s[v], hp[j][v]);
        }
      }
      const bool cut = (cuts >> j) & 1u;
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        B[v] = flow<PACKED>(cut, a[j][v], B[v], hp[j][v]);
        A[v] *= a[j][v];
      }
    }
    float gr[R][VEC];
#pragma unroll
    for (int j = R - 1; j >= 0; --j) {
      unpack(rg[j], gr[j], T());
      if (PACKED) {
        if ((m.out >> j) & 1u) {
#pragma unroll
          for (int v = 0; v < VEC; ++v) gr[j][v] = 0.f;
        } else if (((m.last >> j) & 1u) && g.dhT && chok) {
          float s[VEC];
          load_f32(g.dhT + (long long)seq_of(g.starts, g.S, t0 + j) * g.H + ch, s);
#pragma unroll
          for (int v = 0; v < VEC; ++v) gr[j][v] += s[v];
        }
      }
#pragma unroll
      for (int v = 0; v < VEC; ++v) C[v] = PACKED && ((cuts >> j) & 1u) ? 0.f : a[j][v] * (gr[j][v] + C[v]);
    }

    // folds over the warp's time groups: forward from the left, reverse from the right
    float Ax[VEC], Bx[VEC], Ar[VEC], Cx[VEC], At[VEC], Bt[VEC], Ct[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) Ar[v] = A[v];
    int F = cuts != 0, Fr = F;
#pragma unroll
    for (int d = 1; d < G::GPW; d *= 2) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const float pa = __shfl_up_sync(0xffffffffu, A[v], d * LX);
        const float pb = __shfl_up_sync(0xffffffffu, B[v], d * LX);
        const float na = __shfl_down_sync(0xffffffffu, Ar[v], d * LX);
        const float nc = __shfl_down_sync(0xffffffffu, C[v], d * LX);
        if (grp >= d) {
          B[v] = flow<PACKED>(F, A[v], pb, B[v]);
          A[v] *= pa;
        }
        if (grp + d < G::GPW) {
          C[v] = flow<PACKED>(Fr, Ar[v], nc, C[v]);
          Ar[v] *= na;
        }
      }
      if (PACKED) {
        const int pf = __shfl_up_sync(0xffffffffu, F, d * LX);
        const int nf = __shfl_down_sync(0xffffffffu, Fr, d * LX);
        if (grp >= d) F |= pf;
        if (grp + d < G::GPW) Fr |= nf;
      }
    }
    const int hi_lane = (G::GPW - 1) * LX + lx;
    const int Fx = PACKED && G::GPW > 1 ? __shfl_up_sync(0xffffffffu, F, LX % 32) : 0;
    const int Fy = PACKED && G::GPW > 1 ? __shfl_down_sync(0xffffffffu, Fr, LX % 32) : 0;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      // the warp's whole fold: forward at its last group, reverse at its first
      At[v] = __shfl_sync(0xffffffffu, A[v], hi_lane);
      Bt[v] = __shfl_sync(0xffffffffu, B[v], hi_lane);
      Ct[v] = __shfl_sync(0xffffffffu, C[v], lx);
      Ax[v] = G::GPW > 1 ? __shfl_up_sync(0xffffffffu, A[v], LX % 32) : 1.f;
      Bx[v] = G::GPW > 1 ? __shfl_up_sync(0xffffffffu, B[v], LX % 32) : 0.f;
      Ar[v] = G::GPW > 1 ? __shfl_down_sync(0xffffffffu, Ar[v], LX % 32) : 1.f;
      Cx[v] = G::GPW > 1 ? __shfl_down_sync(0xffffffffu, C[v], LX % 32) : 0.f;
      if (grp == 0) { Ax[v] = 1.f; Bx[v] = 0.f; }
      if (grp == G::GPW - 1) { Ar[v] = 1.f; Cx[v] = 0.f; }
    }
    float c[VEC];
    if (G::NW > 1) {
      const int buf = tile & 1;
      if (grp == 0) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          sA[buf][wt][lx * VEC + v] = At[v];
          sB[buf][wt][lx * VEC + v] = Bt[v];
          sC[buf][wt][lx * VEC + v] = Ct[v];
        }
        if (PACKED && lx == 0) sF[buf][wt] = Fr;  // the first group's: the whole warp's
      }
      __syncthreads();
#pragma unroll
      for (int w = 0; w < G::NW; ++w) {
        const bool cut = PACKED && sF[buf][w] != 0;
#pragma unroll
        for (int v = 0; v < VEC; ++v)
          if (w < wt) h[v] = flow<PACKED>(cut, sA[buf][w][lx * VEC + v], h[v], sB[buf][w][lx * VEC + v]);
      }
#pragma unroll
      for (int w = G::NW - 1; w >= 0; --w) {
        const bool cut = PACKED && sF[buf][w] != 0;
        cut_all = cut_all || cut;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          if (w == wt) c[v] = carry[v];
          const float wa = sA[buf][w][lx * VEC + v];
          carry[v] = flow<PACKED>(cut, wa, carry[v], sC[buf][w][lx * VEC + v]);
          prod[v] *= wa;
        }
      }
    } else {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        c[v] = carry[v];
        carry[v] = fmaf(At[v], carry[v], Ct[v]);
        prod[v] *= At[v];
      }
    }
    if (g.fold_only) continue;

    // states before each token, then the adjoint from the last token to the first
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      h[v] = flow<PACKED>(Fx && grp > 0, Ax[v], h[v], Bx[v]);
      c[v] = flow<PACKED>(Fy && grp < G::GPW - 1, Ar[v], c[v], Cx[v]);
    }
#pragma unroll
    for (int j = 0; j < R; ++j) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const float nx = flow<PACKED>((cuts >> j) & 1u, a[j][v], h[v], hp[j][v]);
        hp[j][v] = h[v];
        h[v] = nx;
      }
    }
    float tacc[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) tacc[v] = 0.f;
#pragma unroll
    for (int j = R - 1; j >= 0; --j) {
      const int t = t0 + j;
      const bool live = chok && t < g.T;
      float lam[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        lam[v] = gr[j][v] + c[v];
        c[v] = PACKED && ((cuts >> j) & 1u) ? 0.f : a[j][v] * lam[v];
      }
      if (PACKED) {
        if ((m.out >> j) & 1u) {
#pragma unroll
          for (int v = 0; v < VEC; ++v) lam[v] = hp[j][v] = 0.f;
        } else if ((m.first >> j) & 1u) {
          const long long n = seq_of(g.starts, g.S, t);
          float s[VEC];
#pragma unroll
          for (int v = 0; v < VEC; ++v) hp[j][v] = 0.f;
          if (g.h0 && chok) load_f32(g.h0 + n * g.H + ch, hp[j]);
          if (g.dh0 && live) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) s[v] = a[j][v] * lam[v];
            store(g.dh0 + n * g.H + ch, s);
          }
        }
      }
      if (!live) continue;
      const long long off = (b * g.T + t) * g.H + ch;
      if (P) {
        float x[VEC], d0[VEC], d1[VEC], d2[VEC];
        unpack(raw[0][j], x, T());
        if (PACKED && ((m.out >> j) & 1u)) {
#pragma unroll
          for (int v = 0; v < VEC; ++v) x[v] = 0.f;
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          const float s = sr[j][v], q = sg[j][v], bt = be[j][v], av = a[j][v];
          const float L = cs[v] * s, lb = lam[v] * bt, lq = lam[v] * q * x[v];
          d0[v] = lb * q;
          d2[v] = lb * x[v] * q * (1.f - q);
          // dL/dL_t = a dL/da + dL/dbeta * (-a^2 / beta); with beta = 0 (L = 0) its share of the
          // gradients below tends to 0
          float dl = lam[v] * hp[j][v] * av;
          if (bt > 0.f) dl = fmaf(-lq * av * av, rcp_approx(bt), dl);
          d1[v] = dl * L * (1.f - s);
          tacc[v] = fmaf(dl, s, tacc[v]);
        }
        store(static_cast<T*>(g.d[0]) + off, d0);
        store(static_cast<T*>(g.d[1]) + off, d1);
        store(static_cast<T*>(g.d[2]) + off, d2);
      } else {
        float d0[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) d0[v] = lam[v] * hp[j][v];
        store(static_cast<T*>(g.d[0]) + off, d0);
        store(static_cast<T*>(g.d[1]) + off, lam);
      }
    }
    if (P) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {  // compensated sum
        const float y = tacc[v] - lost[v], t = acc[v] + y;
        lost[v] = (t - acc[v]) - y;
        acc[v] = t;
      }
    }
  }

  if (g.fold_only) {
    if (chok && ty == 0) {
      float* ag = g.agg + ((b * g.nseg + seg) * 2) * (long long)g.H + ch;
      store(ag, prod);
      store(ag + g.H, carry);
      if (PACKED) g.seg_cut[seg] = cut_all;
    }
    return;
  }
  if (P) {  // decay gradient of this item: fixed order over the time groups
#pragma unroll
    for (int v = 0; v < VEC; ++v)
#pragma unroll
      for (int d = LX; d < 32; d *= 2) acc[v] += __shfl_xor_sync(0xffffffffu, acc[v], d);
    if (G::NW > 1) {
      __syncthreads();
      if (grp == 0) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) sA[0][wt][lx * VEC + v] = acc[v];
      }
      __syncthreads();
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        acc[v] = 0.f;
#pragma unroll
        for (int w = 0; w < G::NW; ++w) acc[v] += sA[0][w][lx * VEC + v];
      }
    }
    if (chok && ty == 0) store(g.part + (b * g.nseg + seg) * g.H + ch, acc);
  }
  if (!chok || seg != 0 || !g.dh0) return;
  if (!PACKED) {
    if (ty == 0) store(g.dh0 + b * g.H + ch, carry);
  } else {
    for (int n = ty; n < g.S; n += TY) {
      if (__ldg(g.starts + n) < __ldg(g.starts + n + 1)) continue;
      float s[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) s[v] = 0.f;
      if (g.dhT) load_f32(g.dhT + (long long)n * g.H + ch, s);
      store(g.dh0 + (long long)n * g.H + ch, s);
    }
  }
}

// d loss / d decay = -scale sigmoid(decay) * sum of the items' partial sums, in fixed order
__global__ void __launch_bounds__(1024) decay_finish_kernel(const float* part, long long rows, int H,
                                                            const float* decay, float scale, float* out) {
  __shared__ double s[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  double v = 0.0;
  if (c < H)
    for (long long r = threadIdx.y; r < rows; r += 32) v += part[r * H + c];
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  // column x of the block is summed by warp x: lanes over the 32 partial rows
  v = s[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  const int cc = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && cc < H) out[cc] = -scale * sigmoid_of<float>(decay[cc]) * (float)v;
}

// One token for each of B sequences: the whole call is one launch without any exchange.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) gated_step_kernel(ScanArgs g) {
  const int hv = g.H / VEC;
  const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
  if (i >= (long long)g.B * hv) return;
  const long long b = i / hv;
  const int ch = (int)(i - b * hv) * VEC;
  float x[VEC], r[VEC], q[VEC], d[VEC], s[VEC];
  unpack(load_raw<T, VEC>(g.in[0], b * g.sb[0] + ch, true), x, T());
  unpack(load_raw<T, VEC>(g.in[1], b * g.sb[1] + ch, true), r, T());
  unpack(load_raw<T, VEC>(g.in[2], b * g.sb[2] + ch, true), q, T());
  load_f32(g.decay + ch, d);
#pragma unroll
  for (int v = 0; v < VEC; ++v) s[v] = 0.f;
  if (g.h0) load_f32(g.h0 + b * g.H + ch, s);
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    const Gate k = gate_of<T>(r[v], q[v], -g.scale * softplus_of(d[v]));
    s[v] = fmaf(k.a, s[v], k.beta * k.sg * x[v]);
  }
  store(g.hT + b * g.H + ch, s);  // may be the array h0 was read from: same thread, same place
  store(static_cast<T*>(g.h) + b * g.H + ch, s);
}

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// whether every row can be read and written 4 channels at a time
bool vec_ok(const ScanArgs& a, int nin, int esize, bool bwd) {
  const size_t n = 4 * (size_t)esize;
  bool ok = a.H % 4 == 0;
  for (int i = 0; i < nin; ++i) ok = ok && aligned(a.in[i], n) && a.sb[i] % 4 == 0 && a.st[i] % 4 == 0;
  if (bwd) {
    ok = ok && aligned(a.dh, n) && a.sb[3] % 4 == 0 && a.st[3] % 4 == 0;
    for (int i = 0; i < nin; ++i) ok = ok && aligned(a.d[i], n);
  } else {
    ok = ok && aligned(a.h, n);
  }
  return ok && aligned(a.decay, 16) && aligned(a.h0, 16) && aligned(a.hT, 16) && aligned(a.dhT, 16) &&
         aligned(a.dh0, 16) && aligned(a.bounds, 16) && aligned(a.agg, 16) && aligned(a.part, 16);
}

template <int P, typename T, int VEC, int LX, int TY, int R, int BB, bool PACKED>
cudaError_t launch_one(ScanArgs a, bool bwd, cudaStream_t st) {
  a.chb = (a.H + LX * VEC - 1) / (LX * VEC);
  for (int pass = a.nseg > 1 ? 0 : 1; pass < 2; ++pass) {
    a.fold_only = pass == 0;
    a.launch_segs = pass == 0 ? a.nseg - 1 : a.nseg;  // one end segment is never folded
    a.items = (long long)a.B * a.launch_segs * a.chb;
    const long long blocks = (a.items + BB - 1) / BB;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    if (bwd) scan_bwd_kernel<P, T, VEC, LX, TY, R, BB, PACKED><<<(unsigned)blocks, kThreads, 0, st>>>(a);
    else scan_fwd_kernel<P, T, VEC, LX, TY, R, BB, PACKED><<<(unsigned)blocks, kThreads, 0, st>>>(a);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

template <int P, typename T>
cudaError_t launch_typed(const ScanArgs& a, bool bwd, cudaStream_t st) {
  const bool vec = vec_ok(a, P ? 3 : 2, (int)sizeof(T), bwd);
  if (a.starts)
    return vec ? launch_one<P, T, 4, 8, 16, 4, 1, true>(a, bwd, st) : launch_one<P, T, 1, 32, 4, 16, 1, true>(a, bwd, st);
  if (a.tile == kScanShortTile)
    return vec ? launch_one<P, T, 4, 8, 4, 4, 4, false>(a, bwd, st) : launch_one<P, T, 1, 32, 1, 16, 4, false>(a, bwd, st);
  return vec ? launch_one<P, T, 4, 8, 16, 4, 1, false>(a, bwd, st) : launch_one<P, T, 1, 32, 4, 16, 1, false>(a, bwd, st);
}

template <int P>
cudaError_t launch_policy(const ScanArgs& a, int dtype, bool bwd, cudaStream_t st) {
  switch (dtype) {
    case 0: return launch_typed<P, float>(a, bwd, st);
    case 1: return launch_typed<P, __nv_bfloat16>(a, bwd, st);
    default: return launch_typed<P, __half>(a, bwd, st);
  }
}

template <typename T>
cudaError_t launch_step(const ScanArgs& a, cudaStream_t st) {
  const bool vec = vec_ok(a, 3, (int)sizeof(T), false);
  const long long n = (long long)a.B * (vec ? a.H / 4 : a.H);
  const long long blocks = (n + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  if (vec) gated_step_kernel<T, 4><<<(unsigned)blocks, kThreads, 0, st>>>(a);
  else gated_step_kernel<T, 1><<<(unsigned)blocks, kThreads, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace

ScanPlan plan_scan(int B, int T, int H, bool packed, int num_sms) {
  ScanPlan p;
  const long long groups = (H + 31) / 32;  // a block or a warp covers 32 channels in every variant
  p.tile = !packed && T <= kScanShortTile ? kScanShortTile : kScanLongTile;
  p.tiles = (T + p.tile - 1) / p.tile;
  const long long chains = B * groups;
  const long long want = 4LL * num_sms;  // blocks that fill the GPU
  long long seg = 1;
  if (chains < want) seg = (want + chains - 1) / chains;
  const long long most = p.tiles / 4;  // at least 4 tiles a segment
  if (seg > most) seg = most;
  if (seg < 1) seg = 1;
  p.seg_tiles = (int)((p.tiles + seg - 1) / seg);
  p.nseg = (p.tiles + p.seg_tiles - 1) / p.seg_tiles;
  return p;
}

cudaError_t launch_scan(const ScanArgs& a, int policy, int dtype, bool bwd, cudaStream_t st) {
  const cudaError_t e = policy ? launch_policy<1>(a, dtype, bwd, st) : launch_policy<0>(a, dtype, bwd, st);
  if (e != cudaSuccess || !bwd || !policy) return e;
  decay_finish_kernel<<<(a.H + 31) / 32, dim3(32, 32), 0, st>>>(a.part, (long long)a.B * a.nseg, a.H, a.decay,
                                                               a.scale, a.ddecay);
  return cudaGetLastError();
}

cudaError_t launch_gated_step(const ScanArgs& a, int dtype, cudaStream_t st) {
  switch (dtype) {
    case 0: return launch_step<float>(a, st);
    case 1: return launch_step<__nv_bfloat16>(a, st);
    default: return launch_step<__half>(a, st);
  }
}

}  // namespace ltc
