// Linear recurrences over time, one independent chain per (sequence, channel):
//   linear scan   h_t = a_t h_{t-1} + b_t                     (a, b given)
//   gated scan    L_t = -scale softplus(decay) sigmoid(rate_t),  a_t = exp(L_t),
//                 b_t = sqrt(1 - a_t^2) sigmoid(gate_t) x_t   (gates computed here)
// and their backward pass, in fp32 whatever the type of the inputs.
//
// Mathematics.  A run of tokens maps the state before it to the state behind it,
// h -> A h + B, and two runs compose as (A2 A1, A2 B1 + B2).  With c_t = a_t lambda_t the
// adjoint lambda_t = dh_t + a_{t+1} lambda_{t+1} runs backwards by the same kind of map,
// c -> A c + C with C folded from the far end, over the SAME product A.
//
// Work split.  An item is one sequence x 32 channels.  A tile is TY x R tokens of it: a
// thread keeps R consecutive tokens of VEC channels in registers, folds them to one (A, B),
// the folds are combined over the tile's TY threads (a shuffle inside a warp, shared memory
// across warps), and the thread runs its tokens again from its own first state.  A group of
// threads marches over its tiles with the state in registers, so every input is read once;
// the next tile's loads are in flight while this one is combined and written.  Where there
// are too few items to fill the GPU, a cluster of up to 16 blocks takes one item, block r the
// tiles r, r + cl, ...: every round the blocks' folds go to every block's shared memory as
// messages that complete bytes on the receiver's mbarrier (bounded waits; a block whose wait
// expired sends and arms no more, so that the others' waits expire as well, and no block leaves
// before all are done).  All orders are
// fixed: results do not depend on scheduling.
//
// Backward.  The forward leaves the state before every 32nd token (fp32); the backward
// rebuilds the states of a tile from it in registers instead of reading h, which is both
// one tensor less and exact where h was rounded to 16 bits.
//
// Packed sequences: token t that starts sequence n is a cut, h_t = a_t h0[n] + b_t whatever came
// before, and a run that holds one is a constant map; tokens outside every sequence give
// h = 0 and zero gradients.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ltc_cluster.cuh"
#include "ltc_common.cuh"
#include "ltc_internal.h"

namespace cg = cooperative_groups;

namespace ltc {

namespace {

constexpr int kThreads = 128;
constexpr int kItem = 32;  // channels of an item, 16 in the narrow shapes

// ---- element types -------------------------------------------------------------
template <typename T, int VEC> struct Raw;  // VEC elements as loaded
template <> struct Raw<float, 2> { using type = float2; };
template <> struct Raw<float, 1> { using type = float; };
template <> struct Raw<__nv_bfloat16, 2> { using type = unsigned; };
template <> struct Raw<__nv_bfloat16, 1> { using type = unsigned short; };
template <> struct Raw<__half, 2> { using type = unsigned; };
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

// The channels of one token that a thread holds: one, or two in packed fp32 instructions.
template <int VEC> struct Chans;
template <> struct Chans<1> { using type = float; };
template <> struct Chans<2> { using type = float2; };

__device__ __forceinline__ float vfma(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float2 vfma(float2 a, float2 b, float2 c) { return fma2(a, b, c); }
__device__ __forceinline__ float vmul(float a, float b) { return a * b; }
__device__ __forceinline__ float2 vmul(float2 a, float2 b) { return mul2(a, b); }
__device__ __forceinline__ float vadd(float a, float b) { return a + b; }
__device__ __forceinline__ float2 vadd(float2 a, float2 b) { return add2(a, b); }
template <typename V> __device__ __forceinline__ V all_of(float x);
template <> __device__ __forceinline__ float all_of<float>(float x) { return x; }
template <> __device__ __forceinline__ float2 all_of<float2>(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 two(float x) { return make_float2(x, x); }
template <typename F> __device__ __forceinline__ float vmap(float x, F f) { return f(x); }
template <typename F> __device__ __forceinline__ float2 vmap(float2 x, F f) { return make_float2(f(x.x), f(x.y)); }
// lane exchange
__device__ __forceinline__ float vxor(float v, int d) { return __shfl_xor_sync(0xffffffffu, v, d); }
__device__ __forceinline__ float2 vxor(float2 v, int d) { return make_float2(vxor(v.x, d), vxor(v.y, d)); }

__device__ __forceinline__ void unpack(const float2& r, float2& v, float) { v = r; }
__device__ __forceinline__ void unpack(const float& r, float& v, float) { v = r; }
template <typename T>
__device__ __forceinline__ void unpack(const unsigned& r, float2& v, T) { v = up2(r, T()); }
template <typename T>
__device__ __forceinline__ void unpack(const unsigned short& r, float& v, T) { v = up2(r, T()).x; }

__device__ __forceinline__ void store(float* p, float2 v) { *reinterpret_cast<float2*>(p) = v; }
__device__ __forceinline__ void store(float* p, float v) { *p = v; }
template <typename T>
__device__ __forceinline__ void store(T* p, float2 v) { *reinterpret_cast<unsigned*>(p) = down2(v.x, v.y, T()); }
template <typename T>
__device__ __forceinline__ void store(T* p, float v) {
  *reinterpret_cast<unsigned short*>(p) = (unsigned short)(down2(v, 0.f, T()) & 0xffffu);
}
template <typename T, typename C>
__device__ __forceinline__ T* at(C* p, int j, int bytes) {
  return reinterpret_cast<T*>(p + (long long)j * bytes);
}
template <typename V>
__device__ __forceinline__ V load_f32(const float* p) { return *reinterpret_cast<const V*>(p); }
template <typename T, int VEC>
__device__ __forceinline__ typename Raw<T, VEC>::type load_raw(const T* p) {
  return __ldg(reinterpret_cast<const typename Raw<T, VEC>::type*>(p));
}

// ---- gates ---------------------------------------------------------------------
// On two elements at a time, in packed fp32 instructions.  The hardware's exp2, reciprocal
// and reciprocal root are off by about 2 ulp each, which leaves the results where a chain of
// correctly rounded operations has them (the tests' bounds count it).  With cu = scale
// softplus(decay) log2(e):  a = 2^-u,  u = cu sigmoid(rate) >= 0.
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kTinyOm = 1e-36f;  // keeps 1 / (1 - a^2) finite; b is 0 long before

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rsqrt_ftz(float x) {
  float y;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 ex2_2(float2 x) { return make_float2(ex2(x.x), ex2(x.y)); }
__device__ __forceinline__ float2 rcp_2(float2 x) { return make_float2(rcp_approx(x.x), rcp_approx(x.y)); }

// a = 2^-u and om = 1 - a^2 = c (2 - c), c = 1 - a.  Near 1, where a step of a is a large part of
// c and exp2's 2 ulp would shift the decay of a slow channel, c is the Taylor series y - y^2/2 +
// ... of 1 - exp(-y), y = ln(2) u, whose first left-out term is below 2^-24 of the sum for
// y < 1/4, and a its rounded complement; past it c is at least 0.22.
__device__ __forceinline__ void decay_of(float2 u, float2& a, float2& om) {
  constexpr double l = 0.6931471805599453;  // ln 2
  float2 p = fma2(u, two((float)(-l * l * l * l * l * l / 720)), two((float)(l * l * l * l * l / 120)));
  p = fma2(u, p, two((float)(-l * l * l * l / 24)));
  p = fma2(u, p, two((float)(l * l * l / 6)));
  p = fma2(u, p, two((float)(-l * l / 2)));
  p = mul2(fma2(u, p, two((float)l)), u);
  const float2 e = make_float2(ex2(-u.x), ex2(-u.y));
  constexpr float limit = (float)(0.25 / l);
  const float2 c = make_float2(u.x < limit ? p.x : 1.f - e.x, u.y < limit ? p.y : 1.f - e.y);
  a = make_float2(u.x < limit ? 1.f - p.x : e.x, u.y < limit ? 1.f - p.y : e.y);
  om = mul2(c, fma2(c, two(-1.f), two(2.f)));
}

__device__ __forceinline__ float softplus_of(float x) { return x > 20.f ? x : log1pf(expf(x)); }
__device__ __forceinline__ float sigmoid_of(float x) { return 1.f / (1.f + expf(-x)); }
__device__ __forceinline__ float rate_of(float decay, float scale) { return scale * softplus_of(decay) * kLog2e; }

// a, and w = sqrt(1 - a^2) sigmoid(gate) as (1 - a^2) rsqrt((1 - a^2) (1 + exp(-gate))^2): one
// instruction for the root and the reciprocal (a gate below -44 overflows the square and
// gives 0 instead of its 1e-19)
__device__ __forceinline__ void gate_fwd(float2 rate, float2 gate, float2 cu, float2& a, float2& w) {
  const float2 s = rcp_2(add2(ex2_2(mul2(rate, two(-kLog2e))), two(1.f)));
  const float2 u = mul2(cu, s);
  float2 om;
  decay_of(u, a, om);
  const float2 pg = add2(ex2_2(mul2(gate, two(-kLog2e))), two(1.f));
  const float2 q = mul2(mul2(make_float2(fmaxf(om.x, kTinyOm), fmaxf(om.y, kTinyOm)), pg), pg);
  w = mul2(om, make_float2(rsqrt_ftz(q.x), rsqrt_ftz(q.y)));
}
// the same with what the gradients need: s = sigmoid(rate), b = w x,
// k = -b a^2 / (1 - a^2) (dL/dL_t = lambda (a h_{t-1} + k)), m = b (1 - sigmoid(gate))
__device__ __forceinline__ void gate_bwd(float2 x, float2 rate, float2 gate, float2 cu, float2& a, float2& w,
                                         float2& s, float2& b, float2& k, float2& m) {
  s = rcp_2(add2(ex2_2(mul2(rate, two(-kLog2e))), two(1.f)));
  const float2 u = mul2(cu, s);
  float2 om;
  decay_of(u, a, om);
  const float2 sg = rcp_2(add2(ex2_2(mul2(gate, two(-kLog2e))), two(1.f)));
  const float2 rs = make_float2(rsqrt_ftz(fmaxf(om.x, kTinyOm)), rsqrt_ftz(fmaxf(om.y, kTinyOm)));
  w = mul2(mul2(om, rs), sg);
  b = mul2(w, x);
  const float2 ar = mul2(a, rs), nb = mul2(b, two(-1.f));
  k = mul2(mul2(nb, ar), ar);
  m = fma2(nb, sg, b);
}

// h -> a h + b, or b behind a cut: where a packed sequence starts, whatever the earlier one
// holds stops there, infinities and NaN too, which a zero factor would let through.  (An
// underflown product is no cut: a NaN goes on through it as in the definition.)
template <bool PACKED, typename V>
__device__ __forceinline__ V flow(bool cut, V a, V h, V b) {
  return PACKED && cut ? b : vfma(a, h, b);
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

// offset n as far as there are tokens
__device__ __forceinline__ int offset_of(const int* starts, int n, int T) {
  return min(max(__ldg(starts + n), 0), T);
}

struct Marks {         // of a thread's R tokens, one bit each
  unsigned first = 0;  // starts its sequence
  unsigned last = 0;   // ends it
  unsigned out = 0;    // belongs to none
  int nf = 0, nl = 0;  // sequences of the earliest first and of the earliest last one
};
// the sequence that token t0 + j starts or ends
__device__ __forceinline__ int seq_at(unsigned bits, int n, int j, const int* starts, int S, int t0) {
  return bits & ((1u << j) - 1) ? seq_of(starts, S, t0 + j) : n;
}

// Where a warp's tiles lie among the sequences.  Each lane keeps one of 32 evenly spread
// offsets, so that finding a tile's sequence takes one load (more past 1024 sequences)
// instead of a bisection's chain of them; nothing is looked up while the tiles stay inside
// one sequence.
struct Walk {
  const int* starts;
  int S, T, stride, pick, begin, end;
  int n = 0, s0 = 0, s1 = 0;  // sequence of the last tile, its tokens [s0, s1)

  __device__ __forceinline__ Walk(const int* starts_, int S_, int T_) : starts(starts_), S(S_), T(T_) {
    stride = (S + 31) / 32;
    const int at = (int)(threadIdx.x & 31) * stride;
    pick = at < S ? __ldg(starts + at) : 0x7fffffff;
    begin = offset_of(starts, 0, T);
    end = offset_of(starts, S, T);
  }
  // all lanes of a warp call it with the same tile
  __device__ __forceinline__ void find(int t) {
    const int block = max(__popc(__ballot_sync(0xffffffffu, pick <= t)) - 1, 0) * stride;
    int count = 0;
    for (int k = 0; k < stride; k += 32) {
      const int at = block + k + (int)(threadIdx.x & 31);
      const bool le = at < min(block + stride, S) && __ldg(starts + min(at, S)) <= t;
      count += __popc(__ballot_sync(0xffffffffu, le));
    }
    n = min(block + max(count - 1, 0), S - 1);
    LTC_CHECK(n >= 0 && n < S, 901);
    s0 = offset_of(starts, n, T);
    s1 = offset_of(starts, n + 1, T);
  }
  template <int R, int TT>
  __device__ __forceinline__ Marks marks(int tile_t0, int t0) {
    Marks m;
    if (!(s0 < tile_t0 && tile_t0 < s1)) find(tile_t0);
    if (s0 < tile_t0 && s1 > tile_t0 + TT && begin <= tile_t0 && end >= tile_t0 + TT) return m;
    // tokens before the first sequence and behind the last, then the ends that lie among the thread's tokens
    const int before = min(max(begin - t0, 0), R), behind = min(max(t0 + R - end, 0), R);
    m.out = ((1u << before) - 1) | (((1u << behind) - 1) << (R - behind));
    int k = n, a = s0, b = s1;
    while (true) {
      if (a < b) {
        if (a >= t0 && a < t0 + R && a < end) {
          if (!m.first) m.nf = k;
          m.first |= 1u << (a - t0);
        }
        if (b > t0 && b <= t0 + R && b <= end) {
          if (!m.last) m.nl = k;
          m.last |= 1u << (b - 1 - t0);
        }
      }
      if (b >= t0 + R || b >= end || k + 1 >= S) break;
      ++k;
      a = b;
      b = offset_of(starts, k + 1, T);
      if (b <= a) {  // no token: on to the last sequence that starts here, however many there are
        k = max(k, seq_of(starts, S, a));
        b = offset_of(starts, k + 1, T);
      }
    }
    return m;
  }
};
struct NoWalk {
  __device__ __forceinline__ NoWalk(const int*, int, int) {}
  template <int R, int TT>
  __device__ __forceinline__ Marks marks(int, int) { return Marks{}; }
};
template <bool PACKED> struct WalkOf { using type = NoWalk; };
template <> struct WalkOf<true> { using type = Walk; };

// A block's last act on the states of its channels, behind every other write to them: a sequence
// without a token passes `from` on (its first state; backward: the gradient of its final one).
// Offsets out of order leave sequences unvisited: then all rows become NaN, not what was in memory.
// All threads of the block call it.
template <typename V, int TY>
__device__ __forceinline__ void finish_sequences(const ScanArgs& g, float* to, const float* from, int ch, bool chok,
                                                 int ty) {
  bool disorder = false;
  for (int n = ty; n < g.S; n += TY) {
    disorder |= __ldg(g.starts + n) > __ldg(g.starts + n + 1);
    if (chok && offset_of(g.starts, n, g.T) >= offset_of(g.starts, n + 1, g.T))
      store(to + (long long)n * g.H + ch, from ? load_f32<V>(from + (long long)n * g.H + ch) : V{});
  }
  if (!__syncthreads_or(disorder) || !chok) return;
  for (int n = ty; n < g.S; n += TY) store(to + (long long)n * g.H + ch, all_of<V>(__int_as_float(0x7fffffff)));
}

// ---- shapes ----------------------------------------------------------------------
template <int VEC_, int R_, int TY_, int BB_, int ITEM_ = kItem>
struct Shape {
  static constexpr int VEC = VEC_, R = R_, TY = TY_, BB = BB_;
  static constexpr int ITEM = ITEM_;
  static constexpr int LX = ITEM / VEC;   // lanes side by side: one row of an item
  static constexpr int GPW = 32 / LX;     // time groups inside a warp
  static constexpr int NW = TY / GPW;     // warps along time
  static constexpr int TT = TY * R;       // tokens of a tile
  static constexpr int THREADS = LX * TY * BB;
  static_assert(TY % GPW == 0 && THREADS % 32 == 0, "whole warps along time");
  static_assert(BB == 1 || NW == 1, "several items per block only without block barriers");
  static_assert((R * VEC) % 2 == 0 && GPW <= 2, "pairs; one shuffle step");
};

// What the warps of a block, and the blocks of a cluster, tell each other about one round.
template <int NW, int NF, bool MANY>
struct alignas(16) Exchange {
  float w[2][NW][NF][kItem];   // per warp: A, then B (and C in the backward)
  int wf[2][NW];               // whether it holds a cut
  float2 x[2][MANY ? kScanMaxCluster : 1][kItem];  // per block: (A, B) or (A, C)
  float xf[2][MANY ? kScanMaxCluster : 1];         // not 0: it holds a cut
  unsigned long long bar[2];   // bytes of a round's messages
  int aborted;
};
__device__ int g_scan_wait_timeouts = 0;

__device__ __forceinline__ int message_bytes(int cl) { return cl * (kItem * (int)sizeof(float2) + (int)sizeof(float)); }

// before the first round: both slots expect the messages of all blocks
template <int NW, int NF>
__device__ __forceinline__ void exchange_begin(Exchange<NW, NF, true>& sh, int cl) {
  if (cl == 1) return;
  if (threadIdx.x == 0) {
    sh.aborted = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_addr(&sh.bar[i]), 1);
    }
    mbar_init_fence();
    for (int i = 0; i < 2; ++i) mbar_arm(smem_addr(&sh.bar[i]), message_bytes(cl));
  }
  cg::this_cluster().sync();
}

// behind the last round: no block leaves while another may still address its shared memory, which
// the message counts alone ensure only as long as no wait expires
__device__ __forceinline__ void exchange_end(int cl) {
  if (cl > 1) cg::this_cluster().sync();
}

// The warps' folds are in shared memory: makes them visible to the block and sends the block's
// fold (in time order) to all blocks of the cluster, each warp to its share of them.  The
// messages complete bytes on the receiver's barrier, so that no block waits for its own.  The slot of
// the round before is armed for the round behind here, away from the waits: its messages may come
// first, since the phase stays open for this arrival.
template <bool PACKED, bool REVERSE, int NW, int NF, bool MANY>
__device__ __forceinline__ void exchange_send(Exchange<NW, NF, MANY>& sh, int buf, int cl, int rank, bool first) {
  const int expired = MANY && cl > 1 ? *static_cast<volatile int*>(&sh.aborted) : 0;
  __syncthreads();
  if (!MANY || cl == 1 || expired) return;
  if (threadIdx.x == 0 && !first) mbar_arm(smem_addr(&sh.bar[buf ^ 1]), message_bytes(cl));
  const int ch = threadIdx.x & 31;  // a narrow item's upper half sends what nobody reads
  float A = 1.f, B = 0.f;
  int F = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    const int w = REVERSE ? NW - 1 - i : i;
    const float wa = sh.w[buf][w][0][ch];
    const bool cut = PACKED && sh.wf[buf][w] != 0;
    B = flow<PACKED>(cut, wa, B, sh.w[buf][w][NF - 1][ch]);
    A *= wa;
    F |= cut;
  }
  const unsigned to = smem_addr(&sh.x[buf][rank][ch]);
  const unsigned tf = smem_addr(&sh.xf[buf][rank]), bar = smem_addr(&sh.bar[buf]);
  for (int r = threadIdx.x / 32; r < cl; r += NW) {
    const unsigned rbar = cluster_map(bar, r);
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];" ::"r"(
                     cluster_map(to, r)), "r"(__float_as_uint(A)), "r"(__float_as_uint(B)), "r"(rbar) : "memory");
    if (ch == 0) st_async(cluster_map(tf, r), F ? 1.f : 0.f, rbar);
  }
}
// Waits for the round's messages.  A block writes a slot again two rounds later, after it has
// all messages of the round between, which every block sends behind a block barrier that
// follows its reads of the slot.
template <int NW, int NF, bool MANY>
__device__ __forceinline__ void exchange_wait(Exchange<NW, NF, MANY>& sh, int buf, int cl, int phase) {
  if (!MANY || cl == 1) return;
  const unsigned bar = smem_addr(&sh.bar[buf]);
  mbar_wait(bar, phase, &sh.aborted, &g_scan_wait_timeouts);
}

// (A, B) of this thread's channels
__device__ __forceinline__ void message(const float2* x, int lx, float& a, float& b) {
  const float2 v = x[lx];
  a = v.x;
  b = v.y;
}
__device__ __forceinline__ void message(const float2* x, int lx, float2& a, float2& b) {
  const float4 v = *reinterpret_cast<const float4*>(x + 2 * lx);
  a = make_float2(v.x, v.z);
  b = make_float2(v.y, v.w);
}

struct Item {
  long long b;
  int ch, rank;
  bool chok;
};
template <typename S, bool MANY>
__device__ __forceinline__ Item item_of(const ScanArgs& g, bool& out) {
  Item it;
  long long i = (long long)blockIdx.x;
  it.rank = 0;
  if (S::BB > 1) {
    i = i * S::BB + threadIdx.x / (S::LX * S::TY);
  } else if (MANY) {
    it.rank = (int)(i % g.cl);
    i /= g.cl;
  }
  out = S::BB > 1 && i >= g.items;
  it.b = i / g.chb;
  it.ch = (int)(i % g.chb) * S::ITEM + (int)(threadIdx.x % S::LX) * S::VEC;
  it.chok = it.ch < g.H;
  return it;
}

// One tensor's R elements (or pairs) of a thread.  Byte addresses with a 32-bit byte stride:
// one multiply-add each.  BRANCH: a whole run of tokens takes a path without tests, which the
// forward gains from (88 against 92 us at 8 x 2048 x 2560 bf16) and the backward does not (201, 196).
template <bool BRANCH, typename T, int VEC, int R>
__device__ __forceinline__ void fetch_run(typename Raw<T, VEC>::type (&raw)[R], const char* p, int st, int left) {
  if (BRANCH && left >= R) {
#pragma unroll
    for (int j = 0; j < R; ++j) raw[j] = load_raw<T, VEC>(at<const T>(p, j, st));
  } else {
#pragma unroll
    for (int j = 0; j < R; ++j) {
      raw[j] = typename Raw<T, VEC>::type{};
      if (j < left) raw[j] = load_raw<T, VEC>(at<const T>(p, j, st));
    }
  }
}

// A and B of a run of tokens
template <bool PACKED, typename V, int R>
__device__ __forceinline__ void fold_run(unsigned cuts, const V (&a)[R], const V (&b)[R], V& A, V& B) {
  A = all_of<V>(1.f);
  B = V{};
  if (PACKED && cuts) {
#pragma unroll
    for (int j = 0; j < R; ++j) {
      B = flow<true>((cuts >> j) & 1u, a[j], B, b[j]);
      A = vmul(A, a[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < R; ++j) {
      B = vfma(a[j], B, b[j]);
      A = vmul(A, a[j]);
    }
  }
}

// gates of a thread's elements: pairs of channels, or of tokens where it holds one channel
template <int R>
__device__ __forceinline__ void gates_fwd(const float2 (&x)[R], const float2 (&y)[R], const float2 (&z)[R], float2 cu,
                                          float2 (&a)[R], float2 (&b)[R]) {
#pragma unroll
  for (int j = 0; j < R; ++j) {
    float2 w;
    gate_fwd(y[j], z[j], cu, a[j], w);
    b[j] = mul2(w, x[j]);
  }
}
template <int R>
__device__ __forceinline__ void gates_fwd(const float (&x)[R], const float (&y)[R], const float (&z)[R], float cu,
                                          float (&a)[R], float (&b)[R]) {
#pragma unroll
  for (int j = 0; j < R; j += 2) {
    float2 fa, fw;
    gate_fwd(make_float2(y[j], y[j + 1]), make_float2(z[j], z[j + 1]), two(cu), fa, fw);
    fw = mul2(fw, make_float2(x[j], x[j + 1]));
    a[j] = fa.x; a[j + 1] = fa.y;
    b[j] = fw.x; b[j + 1] = fw.y;
  }
}
template <int R>
__device__ __forceinline__ void gates_bwd(const float2 (&x)[R], const float2 (&y)[R], const float2 (&z)[R], float2 cu,
                                          float2 (&a)[R], float2 (&w)[R], float2 (&s)[R], float2 (&b)[R],
                                          float2 (&k)[R], float2 (&m)[R]) {
#pragma unroll
  for (int j = 0; j < R; ++j) gate_bwd(x[j], y[j], z[j], cu, a[j], w[j], s[j], b[j], k[j], m[j]);
}
template <int R>
__device__ __forceinline__ void gates_bwd(const float (&x)[R], const float (&y)[R], const float (&z)[R], float cu,
                                          float (&a)[R], float (&w)[R], float (&s)[R], float (&b)[R], float (&k)[R],
                                          float (&m)[R]) {
#pragma unroll
  for (int j = 0; j < R; j += 2) {
    float2 fa, fw, fs, fb, fk, fm;
    gate_bwd(make_float2(x[j], x[j + 1]), make_float2(y[j], y[j + 1]), make_float2(z[j], z[j + 1]), two(cu), fa, fw,
             fs, fb, fk, fm);
    a[j] = fa.x; a[j + 1] = fa.y;
    w[j] = fw.x; w[j + 1] = fw.y;
    s[j] = fs.x; s[j + 1] = fs.y;
    b[j] = fb.x; b[j + 1] = fb.y;
    k[j] = fk.x; k[j + 1] = fk.y;
    m[j] = fm.x; m[j + 1] = fm.y;
  }
}

// ---- forward -----------------------------------------------------------------------
// blocks that an SM's registers have to hold
template <int P, typename T, typename S, bool MANY>
constexpr int fwd_blocks() {
  return MANY || (P && (sizeof(T) == 4 || S::VEC == 1)) ? 4 : 5;
}

template <int P, typename T, typename S, bool PACKED, bool MANY>
__global__ void __launch_bounds__(S::THREADS, (fwd_blocks<P, T, S, MANY>())) scan_fwd_kernel(ScanArgs g) {
  static_assert(!(PACKED || MANY) || S::NW > 1, "the one-warp tiles look at neither cuts nor other blocks");
  constexpr int NIN = P ? 3 : 2, VEC = S::VEC, R = S::R, NW = S::NW, LX = S::LX;
  using V = typename Chans<VEC>::type;
  __shared__ Exchange<NW, 2, MANY> sh;
  const int lx = threadIdx.x % LX, ty = (threadIdx.x / LX) % S::TY;
  const int grp = ty % S::GPW, wt = ty / S::GPW;  // group in the warp, warp along time
  bool out_of_items;
  const Item it = item_of<S, MANY>(g, out_of_items);
  if (out_of_items) return;  // whole warps leave; no block barrier follows
  const long long b = it.b;
  const int ch = it.ch, cl = MANY ? g.cl : 1;
  const bool chok = it.chok;
  const int cr = chok ? ch : 0;  // lanes past the last channel read the first one and write nothing

  V cu{}, carry{};  // carry: state before the round
  if (P) cu = vmap(load_f32<V>(g.decay + cr), [&](float d) { return rate_of(d, g.scale); });
  if (!PACKED && g.h0) carry = load_f32<V>(g.h0 + b * g.H + cr);

  if constexpr (MANY) exchange_begin(sh, cl);
  int t0 = it.rank * S::TT + ty * R;
  const char* in[NIN];
  typename Raw<T, VEC>::type raw[NIN][R];
#pragma unroll
  for (int i = 0; i < NIN; ++i) {
    in[i] = reinterpret_cast<const char*>(static_cast<const T*>(g.in[i]) + b * g.sb[i] + cr) + (long long)t0 * g.st[i];
    fetch_run<true, T, VEC, R>(raw[i], in[i], g.st[i], g.T - t0);
  }
  const int row = g.H * (int)sizeof(T);
  char* out = reinterpret_cast<char*>(static_cast<T*>(g.h) + (b * g.T + t0) * g.H + ch);

  // packed: marks and the first state that the tile needs, found while the tile before is at work
  typename WalkOf<PACKED>::type walk(g.starts, g.S, g.T);
  Marks m = walk.template marks<R, S::TT>(t0 - ty * R, t0);
  V hz{};
  if (PACKED && m.first && g.h0) hz = load_f32<V>(g.h0 + (long long)m.nf * g.H + cr);
  for (int round = 0; round < g.rounds; ++round, t0 += cl * S::TT) {
    const unsigned cuts = PACKED ? m.first | m.out : 0u;

    // factors and terms of this thread's tokens
    V a[R], bv[R];
    {
      V x[R], y[R], z[R];
#pragma unroll
      for (int j = 0; j < R; ++j) {
        unpack(raw[0][j], x[j], T());
        unpack(raw[1][j], y[j], T());
        if (P) unpack(raw[NIN - 1][j], z[j], T());
        if (PACKED && ((m.out >> j) & 1u)) x[j] = y[j] = z[j] = V{};  // what lies outside the sequences is not used
      }
      if constexpr (P != 0) {
        gates_fwd(x, y, z, cu, a, bv);
      } else {
#pragma unroll
        for (int j = 0; j < R; ++j) {
          a[j] = x[j];
          bv[j] = y[j];
        }
      }
    }
    if (round + 1 < g.rounds) {
#pragma unroll
      for (int i = 0; i < NIN; ++i) {
        in[i] += (long long)(cl * S::TT) * g.st[i];
        fetch_run<true, T, VEC, R>(raw[i], in[i], g.st[i], g.T - t0 - cl * S::TT);
      }
    }
    if (t0 + R > g.T) {  // behind the end the state stays
#pragma unroll
      for (int j = 0; j < R; ++j)
        if (t0 + j >= g.T) {
          a[j] = all_of<V>(1.f);
          bv[j] = V{};
        }
    }
    if (PACKED && cuts) {
#pragma unroll
      for (int j = 0; j < R; ++j) {
        if (t0 + j >= g.T) continue;
        if ((m.out >> j) & 1u) bv[j] = V{};
        else if (((m.first >> j) & 1u) && g.h0)
          bv[j] = vfma(a[j], m.first & ((1u << j) - 1)
                                 ? load_f32<V>(g.h0 + (long long)seq_of(g.starts, g.S, t0 + j) * g.H + cr) : hz, bv[j]);
      }
    }
    Marks next;

    // fold of this thread's tokens, over the warp, over the block
    V A, B, Ax = all_of<V>(1.f), Bx{};
    int F = cuts != 0, Fx = 0;  // a run with a cut is the constant B
    fold_run<PACKED>(cuts, a, bv, A, B);
    if (S::GPW > 1) {
      const V pa = vxor(A, LX % 32), pb = vxor(B, LX % 32);
      const int pf = PACKED ? __shfl_xor_sync(0xffffffffu, F, LX % 32) : 0;
      if (grp > 0) {
        Ax = pa;
        Bx = pb;
        Fx = pf;
        B = flow<PACKED>(F, A, pb, B);
        A = vmul(A, pa);
        F |= pf;
      }
    }
    V h;
    if (NW > 1) {
      const int buf = round & 1;  // the next round's barrier separates the reads from the writes after it
      if (grp == S::GPW - 1) {
        store(&sh.w[buf][wt][0][lx * VEC], A);
        store(&sh.w[buf][wt][1][lx * VEC], B);
        if (PACKED && lx == 0) sh.wf[buf][wt] = F;
      }
      exchange_send<PACKED, false>(sh, buf, cl, it.rank, round == 0);
      if (PACKED && round + 1 < g.rounds) {  // while the messages are on their way
        next = walk.template marks<R, S::TT>(t0 + cl * S::TT - ty * R, t0 + cl * S::TT);
        if (next.first && g.h0) hz = load_f32<V>(g.h0 + (long long)next.nf * g.H + cr);
      }
      exchange_wait(sh, buf, cl, (round >> 1) & 1);
      h = carry;
      if (MANY && cl > 1) {
        for (int r = 0; r < cl; ++r) {
          if (r == it.rank) h = carry;
          V xa, xb;
          message(sh.x[buf][r], lx, xa, xb);
          carry = flow<PACKED>(PACKED && sh.xf[buf][r] != 0.f, xa, carry, xb);
        }
      }
      V run = h;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        if (w == wt) h = run;
        run = flow<PACKED>(PACKED && sh.wf[buf][w] != 0, load_f32<V>(&sh.w[buf][w][0][lx * VEC]), run,
                           load_f32<V>(&sh.w[buf][w][1][lx * VEC]));
      }
      if (cl == 1) carry = run;
    } else {
      const int src = (S::GPW - 1) * LX + lx;
      h = carry;
      carry = vfma(vmap(A, [&](float v) { return __shfl_sync(0xffffffffu, v, src); }), carry,
                   vmap(B, [&](float v) { return __shfl_sync(0xffffffffu, v, src); }));
    }
    h = flow<PACKED>(Fx, Ax, h, Bx);
    if (g.bounds && t0 > 0 && t0 % kScanBound == 0 && t0 < g.T && chok)
      store(g.bounds + (b * g.nbounds + t0 / kScanBound - 1) * g.H + ch, h);

    const int left = chok ? g.T - t0 : 0;
    if (PACKED && cuts) {
#pragma unroll
      for (int j = 0; j < R; ++j) {
        h = flow<true>((cuts >> j) & 1u, a[j], h, bv[j]);
        a[j] = h;
      }
    } else {
#pragma unroll
      for (int j = 0; j < R; ++j) {
        h = vfma(a[j], h, bv[j]);
        a[j] = h;
      }
    }
    if (left >= R) {
#pragma unroll
      for (int j = 0; j < R; ++j) store(at<T>(out, j, row), a[j]);
    } else {
#pragma unroll
      for (int j = 0; j < R; ++j)
        if (j < left) store(at<T>(out, j, row), a[j]);
    }
    out += (long long)(cl * S::TT) * row;
    if (PACKED && m.last && chok) {
#pragma unroll
      for (int j = 0; j < R; ++j)
        if ((m.last >> j) & 1u)
          store(g.hT + (long long)seq_at(m.last, m.nl, j, g.starts, g.S, t0) * g.H + ch, a[j]);
    }
    m = next;
  }

  if constexpr (MANY) exchange_end(cl);
  if (it.rank != 0) return;
  if constexpr (PACKED) finish_sequences<V, S::TY>(g, g.hT, g.h0, ch, chok, ty);
  else if (chok && ty == 0) store(g.hT + b * g.H + ch, carry);
}

// blocks that an SM's registers have to hold; more spill (bf16 gated: 5 against 4 blocks 184 and 205 us at
// 8 x 2048 x 2560, the second a partial wave of blocks; fp32 spills at 5: 242 against 195 us at 1 x 32771 x 512)
template <int P, typename T, typename S, bool MANY>
constexpr int bwd_blocks() {
  if (MANY) return 3;
  if (!P) return S::R * S::VEC > 8 ? 4 : 5;
  if (S::R * S::VEC > 8 || sizeof(T) == 4) return 3;
  return 5;
}

// ---- backward ----------------------------------------------------------------------
template <int P, typename T, typename S, bool PACKED, bool MANY>
__global__ void __launch_bounds__(S::THREADS, (bwd_blocks<P, T, S, MANY>())) scan_bwd_kernel(ScanArgs g) {
  static_assert(!(PACKED || MANY) || S::NW > 1, "the one-warp tiles look at neither cuts nor other blocks");
  static_assert(S::NW == 1 || S::TT % kScanBound == 0, "a tile starts at a saved state");
  constexpr int NIN = P ? 3 : 2, VEC = S::VEC, R = S::R, NW = S::NW, LX = S::LX;
  using V = typename Chans<VEC>::type;
  __shared__ Exchange<NW, 3, MANY> sh;
  // what only the last step of a tile needs waits in shared memory, every thread in its own places, so that
  // five blocks fit an SM's registers instead of three
  __shared__ V parked[P ? 4 : 1][P ? R : 1][S::THREADS];
  const int lx = threadIdx.x % LX, ty = (threadIdx.x / LX) % S::TY;
  const int grp = ty % S::GPW, wt = ty / S::GPW;
  bool out_of_items;
  const Item it = item_of<S, MANY>(g, out_of_items);
  if (out_of_items) return;
  const long long b = it.b;
  const int ch = it.ch, cl = MANY ? g.cl : 1;
  const bool chok = it.chok;
  const int cr = chok ? ch : 0;

  // carry: c behind the round; acc: decay gradient so far, lost: what its additions rounded away
  V cu{}, carry{}, acc{}, lost{};
  if (P) cu = vmap(load_f32<V>(g.decay + cr), [&](float d) { return rate_of(d, g.scale); });
  const V cn = vmul(cu, all_of<V>(-0.6931471805599453f));
  if (!PACKED && g.dhT) carry = load_f32<V>(g.dhT + b * g.H + cr);

  if constexpr (MANY) exchange_begin(sh, cl);
  int t0 = ((g.rounds - 1) * cl + it.rank) * S::TT + ty * R;
  const char* in[NIN + 1];
  typename Raw<T, VEC>::type raw[NIN + 1][R];
  V hs;  // state before the tile
  auto first_state = [&](int tile_t0) {
    V v{};
    if (NW > 1 && tile_t0 > 0) {
      if (tile_t0 < g.T) v = load_f32<V>(g.bounds + (b * g.nbounds + tile_t0 / kScanBound - 1) * g.H + cr);
    } else if (!PACKED && g.h0) {
      v = load_f32<V>(g.h0 + b * g.H + cr);
    }
    return v;
  };
#pragma unroll
  for (int i = 0; i <= NIN; ++i) {
    const int st = g.st[i < NIN ? i : 3];
    in[i] = reinterpret_cast<const char*>(static_cast<const T*>(i < NIN ? g.in[i < NIN ? i : 0] : g.dh) +
                                          b * g.sb[i < NIN ? i : 3] + cr) + (long long)t0 * st;
    fetch_run<false, T, VEC, R>(raw[i], in[i], st, i < NIN || g.dh ? g.T - t0 : 0);
  }
  const int row = g.H * (int)sizeof(T);
  char* out[NIN];
#pragma unroll
  for (int i = 0; i < NIN; ++i)
    out[i] = reinterpret_cast<char*>(static_cast<T*>(g.d[i]) + (b * g.T + t0) * g.H + ch);
  hs = first_state(t0 - ty * R);

  typename WalkOf<PACKED>::type walk(g.starts, g.S, g.T);
  Marks m = walk.template marks<R, S::TT>(t0 - ty * R, t0);
  V hz{}, dz{};  // first state and final state's gradient that the tile needs
  if (PACKED && m.first && g.h0) hz = load_f32<V>(g.h0 + (long long)m.nf * g.H + cr);
  if (PACKED && m.last && g.dhT) dz = load_f32<V>(g.dhT + (long long)m.nl * g.H + cr);
  for (int round = g.rounds - 1; round >= 0; --round, t0 -= cl * S::TT) {
    const unsigned cuts = PACKED ? m.first | m.out : 0u;

    // gates; hp holds b_t until the states are known
    V a[R], hp[R], gr[R], h = hs;
    {
      V x[R], y[R], z[R];
#pragma unroll
      for (int j = 0; j < R; ++j) {
        unpack(raw[0][j], x[j], T());
        unpack(raw[1][j], y[j], T());
        if (P) unpack(raw[NIN - 1][j], z[j], T());
        unpack(raw[NIN][j], gr[j], T());
        if (PACKED && ((m.out >> j) & 1u)) x[j] = y[j] = z[j] = gr[j] = V{};
      }
      if constexpr (P != 0) {
        V s[R], w[R], k[R], mg[R];
        gates_bwd(x, y, z, cu, a, w, s, hp, k, mg);
#pragma unroll
        for (int j = 0; j < R; ++j) {
          parked[0][j][threadIdx.x] = s[j];
          parked[1][j][threadIdx.x] = w[j];
          parked[2][j][threadIdx.x] = k[j];
          parked[3][j][threadIdx.x] = mg[j];
        }
      } else {
#pragma unroll
        for (int j = 0; j < R; ++j) {
          a[j] = x[j];
          hp[j] = y[j];
        }
      }
    }
    if (round > 0) {
#pragma unroll
      for (int i = 0; i <= NIN; ++i) {
        const int st = g.st[i < NIN ? i : 3];
        in[i] -= (long long)(cl * S::TT) * st;
        fetch_run<false, T, VEC, R>(raw[i], in[i], st, i < NIN || g.dh ? g.T - t0 + cl * S::TT : 0);
      }
      hs = first_state(t0 - cl * S::TT - ty * R);
    }
    if (t0 + R > g.T) {
#pragma unroll
      for (int j = 0; j < R; ++j)
        if (t0 + j >= g.T) {
          a[j] = all_of<V>(1.f);
          hp[j] = V{};
        }
    }
    if (PACKED && (cuts | m.last)) {
#pragma unroll
      for (int j = 0; j < R; ++j) {
        if (t0 + j >= g.T) continue;
        if ((m.out >> j) & 1u) hp[j] = V{};
        if (((m.first >> j) & 1u) && g.h0)
          hp[j] = vfma(a[j], m.first & ((1u << j) - 1)
                                 ? load_f32<V>(g.h0 + (long long)seq_of(g.starts, g.S, t0 + j) * g.H + cr) : hz, hp[j]);
        if (((m.last >> j) & 1u) && g.dhT)
          gr[j] = vadd(gr[j], m.last & ((1u << j) - 1)
                                  ? load_f32<V>(g.dhT + (long long)seq_of(g.starts, g.S, t0 + j) * g.H + cr) : dz);
      }
    }
    const V h0f = hz;
    Marks next;

    // forward fold (A, B) and reverse fold (A, C) of this thread's tokens
    V A, B, C{};
    const int F = cuts != 0;
    fold_run<PACKED>(cuts, a, hp, A, B);
#pragma unroll
    for (int j = R - 1; j >= 0; --j) C = PACKED && ((cuts >> j) & 1u) ? V{} : vmul(a[j], vadd(gr[j], C));
    // the two groups of a warp: the first one's fold goes to the second's states, the second one's to the
    // first's adjoints, and both make the warp's
    V Ax = all_of<V>(1.f), Bx{}, Cx{}, At = A, Bt = B, Ct = C;
    int Fo = 0;
    if (S::GPW > 1) {
      if (PACKED) Fo = __shfl_xor_sync(0xffffffffu, F, LX % 32);
      Ax = vxor(A, LX % 32);
      Bx = vxor(B, LX % 32);
      Cx = vxor(C, LX % 32);
      At = vmul(A, Ax);
      if (grp == 0) {
        Bt = flow<PACKED>(Fo, Ax, B, Bx);
        Ct = flow<PACKED>(F, A, Cx, C);
      } else {
        Bt = flow<PACKED>(F, A, Bx, B);
        Ct = flow<PACKED>(Fo, Ax, C, Cx);
      }
    }
    V c;
    if (NW > 1) {
      const int buf = (g.rounds - 1 - round) & 1;
      if (grp == 0) {
        store(&sh.w[buf][wt][0][lx * VEC], At);
        store(&sh.w[buf][wt][1][lx * VEC], Bt);
        store(&sh.w[buf][wt][2][lx * VEC], Ct);
        if (PACKED && lx == 0) sh.wf[buf][wt] = F | Fo;
      }
      exchange_send<PACKED, true>(sh, buf, cl, it.rank, round == g.rounds - 1);
      if (PACKED && round > 0) {
        next = walk.template marks<R, S::TT>(t0 - cl * S::TT - ty * R, t0 - cl * S::TT);
        if (next.first && g.h0) hz = load_f32<V>(g.h0 + (long long)next.nf * g.H + cr);
        if (next.last && g.dhT) dz = load_f32<V>(g.dhT + (long long)next.nl * g.H + cr);
      }
      exchange_wait(sh, buf, cl, ((g.rounds - 1 - round) >> 1) & 1);
      c = carry;
      if (MANY && cl > 1) {
        for (int r = cl - 1; r >= 0; --r) {
          if (r == it.rank) c = carry;
          V xa, xb;
          message(sh.x[buf][r], lx, xa, xb);
          carry = flow<PACKED>(PACKED && sh.xf[buf][r] != 0.f, xa, carry, xb);
        }
      }
      V run = c;
#pragma unroll
      for (int u = NW - 1; u >= 0; --u) {
        const bool cut = PACKED && sh.wf[buf][u] != 0;
        const V wa = load_f32<V>(&sh.w[buf][u][0][lx * VEC]);
        if (u == wt) c = run;
        run = flow<PACKED>(cut, wa, run, load_f32<V>(&sh.w[buf][u][2][lx * VEC]));
      }
      if (cl == 1) carry = run;
#pragma unroll
      for (int u = 0; u < NW - 1; ++u)
        if (u < wt)
          h = flow<PACKED>(PACKED && sh.wf[buf][u] != 0, load_f32<V>(&sh.w[buf][u][0][lx * VEC]), h,
                           load_f32<V>(&sh.w[buf][u][1][lx * VEC]));
    } else {
      c = carry;
      carry = vfma(At, carry, Ct);
    }
    if (S::GPW > 1) {
      if (grp > 0) h = flow<PACKED>(Fo, Ax, h, Bx);
      else c = flow<PACKED>(Fo, Ax, c, Cx);
    }

    // states before each token, then the adjoint from the last token to the first
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const V nx = flow<PACKED>((cuts >> j) & 1u, a[j], h, hp[j]);
      hp[j] = h;
      h = nx;
    }
    V tacc{};
    const int left = chok ? g.T - t0 : 0;
    const bool whole = left >= R;
#pragma unroll
    for (int j = R - 1; j >= 0; --j) {
      V lam = vadd(gr[j], c);
      c = PACKED && ((cuts >> j) & 1u) ? V{} : vmul(a[j], lam);
      if (PACKED && ((cuts >> j) & 1u)) {
        hp[j] = V{};
        if ((m.out >> j) & 1u) {
          lam = V{};
        } else if (j < left) {
          const long long n = seq_at(m.first, m.nf, j, g.starts, g.S, t0);
          if (g.h0) hp[j] = m.first & ((1u << j) - 1) ? load_f32<V>(g.h0 + n * g.H + cr) : h0f;
          if (g.dh0) store(g.dh0 + n * g.H + ch, vmul(a[j], lam));
        }
      }
      const bool live = whole || j < left;
      if constexpr (P != 0) {
        // L_t (1 - s) = -ln(2) cu s (1 - s)
        const V s = parked[0][j][threadIdx.x];
        const V dl = vmul(lam, vfma(hp[j], a[j], parked[2][j][threadIdx.x]));
        const V cs = vmul(cn, s);
        const V d1 = vmul(dl, vfma(cs, vmul(s, all_of<V>(-1.f)), cs));
        if (live) {
          store(at<T>(out[0], j, row), vmul(lam, parked[1][j][threadIdx.x]));
          store(at<T>(out[1], j, row), d1);
          store(at<T>(out[NIN - 1], j, row), vmul(lam, parked[3][j][threadIdx.x]));
          tacc = vfma(dl, s, tacc);
        }
      } else if (live) {
        store(at<T>(out[0], j, row), vmul(lam, hp[j]));
        store(at<T>(out[1], j, row), lam);
      }
    }
#pragma unroll
    for (int i = 0; i < NIN; ++i) out[i] -= (long long)(cl * S::TT) * row;
    m = next;
    if (P) {  // compensated sum
      const V y = vfma(lost, all_of<V>(-1.f), tacc), t = vadd(acc, y);
      lost = vfma(y, all_of<V>(-1.f), vfma(acc, all_of<V>(-1.f), t));
      acc = t;
    }
  }

  if constexpr (MANY) exchange_end(cl);
  if (P) {  // decay gradient of this block or warp: fixed order over the time groups
    if (S::GPW > 1) acc = vadd(acc, vxor(acc, LX % 32));
    if (NW > 1) {
      __syncthreads();
      if (grp == 0) store(&sh.w[0][wt][0][lx * VEC], acc);
      __syncthreads();
      acc = V{};
#pragma unroll
      for (int u = 0; u < NW; ++u) acc = vadd(acc, load_f32<V>(&sh.w[0][u][0][lx * VEC]));
    }
    if (chok && ty == 0) store(g.part + (b * cl + it.rank) * g.H + ch, acc);
  }
  if (it.rank != 0 || !g.dh0) return;
  if constexpr (PACKED) finish_sequences<V, S::TY>(g, g.dh0, g.dhT, ch, chok, ty);
  else if (chok && ty == 0) store(g.dh0 + b * g.H + ch, carry);
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
  if (threadIdx.x == 0 && cc < H) out[cc] = -scale * sigmoid_of(decay[cc]) * (float)v;
}

// One token for each of B sequences: the whole call is one launch without any exchange.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) gated_step_kernel(ScanArgs g) {
  const int hv = g.H / VEC;
  const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
  if (i >= (long long)g.B * hv) return;
  const long long b = i / hv;
  const int ch = (int)(i - b * hv) * VEC;
  using V = typename Chans<VEC>::type;
  V x, r, q;
  unpack(load_raw<T, VEC>(static_cast<const T*>(g.in[0]) + b * g.sb[0] + ch), x, T());
  unpack(load_raw<T, VEC>(static_cast<const T*>(g.in[1]) + b * g.sb[1] + ch), r, T());
  unpack(load_raw<T, VEC>(static_cast<const T*>(g.in[2]) + b * g.sb[2] + ch), q, T());
  const V cu = vmap(load_f32<V>(g.decay + ch), [&](float d) { return rate_of(d, g.scale); });
  V s = g.h0 ? load_f32<V>(g.h0 + b * g.H + ch) : V{};
  if constexpr (VEC == 2) {
    float2 a, w;
    gate_fwd(r, q, cu, a, w);
    s = fma2(a, s, mul2(w, x));
  } else {
    float2 a, w;
    gate_fwd(two(r), two(q), two(cu), a, w);
    s = fmaf(a.x, s, w.x * x);
  }
  store(g.hT + b * g.H + ch, s);  // may be the array h0 was read from: same thread, same place
  store(static_cast<T*>(g.h) + b * g.H + ch, s);
}

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// whether every row can be read and written two channels at a time
bool pairs_ok(const ScanArgs& a, int nin, int esize, bool bwd) {
  const size_t n = 2 * (size_t)esize;
  bool ok = a.H % 2 == 0;
  for (int i = 0; i < nin; ++i) ok = ok && aligned(a.in[i], n) && a.sb[i] % 2 == 0 && a.st[i] % (int)n == 0;
  if (bwd) {
    ok = ok && aligned(a.dh, n) && a.sb[3] % 2 == 0 && a.st[3] % (int)n == 0;
    for (int i = 0; i < nin; ++i) ok = ok && aligned(a.d[i], n);
  } else {
    ok = ok && aligned(a.h, n);
  }
  return ok && aligned(a.decay, 8) && aligned(a.h0, 8) && aligned(a.hT, 8) && aligned(a.dhT, 8) &&
         aligned(a.dh0, 8) && aligned(a.bounds, 8) && aligned(a.part, 8);
}

template <typename S, typename K>
cudaError_t launch_one(K kernel, ScanArgs a, cudaStream_t st) {
  a.chb = (a.H + S::ITEM - 1) / S::ITEM;
  a.items = (long long)a.B * a.chb;
  if (S::BB > 1) a.cl = 1;
  const int tiles = (a.T + S::TT - 1) / S::TT;
  a.rounds = (tiles + a.cl - 1) / a.cl;
  const long long blocks = S::BB > 1 ? (a.items + S::BB - 1) / S::BB : a.items * a.cl;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(S::THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)a.cl;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = a.cl > 1 ? 1 : 0;
  if (a.cl > 8) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
  }
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

// VEC, tokens per thread, threads along time, items per block
using FwdPair = Shape<2, 8, 8, 1>;
using FwdOne = Shape<1, 16, 4, 1>;
using BwdPair = Shape<2, 4, 8, 1>;
using BwdOne = Shape<1, 8, 4, 1>;
// 16 channels of twice the tokens: twice as many items where there are very few
using FwdNarrow = Shape<1, 16, 8, 1, 16>;
using BwdNarrow = Shape<1, 8, 8, 1, 16>;
// rows of up to 16 and up to 8 tokens: a warp each
using ShortPair = Shape<2, 8, 2, 4>;
using ShortOne = Shape<1, 16, 1, 4>;
using TinyPair = Shape<2, 4, 2, 4>;
using TinyOne = Shape<1, 8, 1, 4>;

template <int P, typename T, typename PAIR, typename ONE, bool PACKED, bool MANY>
cudaError_t launch_dir(const ScanArgs& a, bool bwd, bool pair, cudaStream_t st) {
  if (bwd)
    return pair ? launch_one<PAIR>(scan_bwd_kernel<P, T, PAIR, PACKED, MANY>, a, st)
                : launch_one<ONE>(scan_bwd_kernel<P, T, ONE, PACKED, MANY>, a, st);
  return pair ? launch_one<PAIR>(scan_fwd_kernel<P, T, PAIR, PACKED, MANY>, a, st)
              : launch_one<ONE>(scan_fwd_kernel<P, T, ONE, PACKED, MANY>, a, st);
}
template <int P, typename T, typename F, typename B, bool PACKED, bool MANY>
cudaError_t launch_long(const ScanArgs& a, bool bwd, cudaStream_t st) {
  if (bwd) return launch_one<B>(scan_bwd_kernel<P, T, B, PACKED, MANY>, a, st);
  return launch_one<F>(scan_fwd_kernel<P, T, F, PACKED, MANY>, a, st);
}

template <int P, typename T>
cudaError_t launch_typed(const ScanArgs& a, bool bwd, cudaStream_t st) {
  const bool pair = pairs_ok(a, P ? 3 : 2, (int)sizeof(T), bwd);
  if (a.narrow && (a.starts || a.T > kScanShort))
    return a.starts ? launch_long<P, T, FwdNarrow, BwdNarrow, true, true>(a, bwd, st)
                    : launch_long<P, T, FwdNarrow, BwdNarrow, false, true>(a, bwd, st);
  if (a.starts)
    return pair ? launch_long<P, T, FwdPair, BwdPair, true, true>(a, bwd, st)
                : launch_long<P, T, FwdOne, BwdOne, true, true>(a, bwd, st);
  if (a.T <= TinyPair::TT) return launch_dir<P, T, TinyPair, TinyOne, false, false>(a, bwd, pair, st);
  if (a.T <= kScanShort) return launch_dir<P, T, ShortPair, ShortOne, false, false>(a, bwd, pair, st);
  if (a.cl > 1)
    return pair ? launch_long<P, T, FwdPair, BwdPair, false, true>(a, bwd, st)
                : launch_long<P, T, FwdOne, BwdOne, false, true>(a, bwd, st);
  return pair ? launch_long<P, T, FwdPair, BwdPair, false, false>(a, bwd, st)
              : launch_long<P, T, FwdOne, BwdOne, false, false>(a, bwd, st);
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
  const bool pair = pairs_ok(a, 3, (int)sizeof(T), false);
  const long long n = (long long)a.B * (pair ? a.H / 2 : a.H);
  const long long blocks = (n + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  if (pair) gated_step_kernel<T, 2><<<(unsigned)blocks, kThreads, 0, st>>>(a);
  else gated_step_kernel<T, 1><<<(unsigned)blocks, kThreads, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace

// Blocks of an item.  A block marches at the latency of its tiles, so few items are shared by
// clusters until the SMs have a few blocks each (4 fit in the forward, 3 in the backward), the
// smaller clusters first: their rounds are shorter.  Measured on a B200 with (items x blocks):
// forward, 16387 packed tokens x 2048 bf16: 64 x 4 211 us, x 8 140, x 16 214 (a second wave);
// 3 x 5000 x 1001 fp16: 96 x 4 35 us, x 8 37; both directions of 1 x 32771 x 512 fp32:
// 16 x 16 240 us, 16 x 8 330, in narrow items 32 x 8 208, 32 x 16 240.
ScanPlan plan_scan(int B, int T, int H, bool packed, int num_sms) {
  ScanPlan p;
  p.nbounds = (T - 1) / kScanBound;
  p.cl_fwd = p.cl_bwd = 1;
  p.narrow = false;
  if (!packed && T <= kScanShort) return p;
  long long items = (long long)B * ((H + kItem - 1) / kItem);
  if (8 * items < 2LL * num_sms) {
    p.narrow = true;
    items = (long long)B * ((H + kItem / 2 - 1) / (kItem / 2));
  }
  auto blocks = [&](int tile, int fit) {
    int cl = 1;
    while (cl < 8 && items * cl * 2 <= (long long)fit * num_sms && cl * 2 * tile <= T) cl *= 2;
    if (cl == 8 && items * 8 <= num_sms && 16 * tile <= T) cl = 16;
    return cl;
  };
  p.cl_fwd = blocks(p.narrow ? FwdNarrow::TT : FwdPair::TT, 4);
  p.cl_bwd = blocks(p.narrow ? BwdNarrow::TT : BwdPair::TT, 3);
  return p;
}

cudaError_t launch_scan(const ScanArgs& a, int policy, int dtype, bool bwd, cudaStream_t st) {
  const cudaError_t e = policy ? launch_policy<1>(a, dtype, bwd, st) : launch_policy<0>(a, dtype, bwd, st);
  if (e != cudaSuccess || !bwd || !policy) return e;
  decay_finish_kernel<<<(a.H + 31) / 32, dim3(32, 32), 0, st>>>(a.part, (long long)a.B * a.cl, a.H, a.decay,
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

int read_scan_wait_timeouts(int* count) {
  return (int)cudaMemcpyFromSymbol(count, g_scan_wait_timeouts, sizeof(int));
}

}  // namespace ltc
