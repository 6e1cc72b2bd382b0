// Gated linear recurrence over sequences (batch, steps, 3, dim): candidates z, gates g and output gates o,
//   f = sigmoid(g)     h_t = f_t (reset_t ? 0 : h_{t-1}) + (1 - f_t) z_t     y_t = sigmoid(o_t) h_t
// and its gradient, with e_t = what step t hands to the step before it:
//   dh_t = dy_t sigmoid(o_t) + e_{t+1}      e_t = (reset_t ? 0 : f_t) dh_t
//   dz = (1 - f) dh     dg = (h_{t-1} - z) f (1 - f) dh     do = dy h sigmoid(o) (1 - sigmoid(o))
// Both directions are scans of x -> a x + b.  A warp takes 64 channels of a chunk of consecutive steps, the warps of a CTA and the
// CTAs of a cluster take consecutive chunks, and a cluster walks along its sequence.  What a chunk does to a value that comes
// in, (product of a, result from 0), is a link; links are passed on before every warp walks its chunk again from the true
// value: between warps in shared memory, between CTAs by asynchronous stores into each other's shared memory.  The state is
// fp32 throughout; the forward leaves it in front of every eighth step for the backward, which rebuilds h from it.
//
// Bound: 8 bytes a value of h forward, 14 backward (16 bytes more for every 32 of them: the saved states).  The arithmetic is
// close behind, four operations of the special-function units a value in either direction, so the two gates' exponentials and
// reciprocals are formed once and everything else is packed.  Measured, bf16: 1 x 30011 x 2048 121 us forward (66 % of the
// copy rate) and 203 us backward (67 %); 8 x 1024 x 1024 25 and 34 us.  The comparisons further down were measured before the walks
// looked for closed gates and infinities, which takes 2 % of the forward and 5 % of the backward.
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>

#include "elem16.cuh"
#include "gemm_tcgen05.h"
#include "tc05.cuh"
#include "tensor_map.h"

extern int g_fbam_last_driver_error;   // defined in gemm_tcgen05.cu

namespace {

using namespace tc05;

constexpr int kSaved = 8;         // the forward keeps the state in front of every eighth step
constexpr int kFwdSteps = 16;     // of a chunk of the forward by TMA; all others have kSaved steps
constexpr int kMaxCtas = 16;      // of a cluster
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// A lane's channels: two packed values (sm_100 computes on two fp32 values per instruction) or one.
template <int VEC>
struct Vec;
template <>
struct Vec<1> {
  float v;
  __device__ __forceinline__ static Vec all(float a) { return {a}; }
  __device__ __forceinline__ float get(int) const { return v; }
};
template <>
struct Vec<2> {
  float2 v;
  __device__ __forceinline__ static Vec all(float a) { return {make_float2(a, a)}; }
  __device__ __forceinline__ float get(int j) const { return j ? v.y : v.x; }
};
__device__ __forceinline__ Vec<1> fma(Vec<1> a, Vec<1> b, Vec<1> c) { return {fmaf(a.v, b.v, c.v)}; }
__device__ __forceinline__ Vec<2> fma(Vec<2> a, Vec<2> b, Vec<2> c) { return {__ffma2_rn(a.v, b.v, c.v)}; }
__device__ __forceinline__ Vec<1> operator*(Vec<1> a, Vec<1> b) { return {a.v * b.v}; }
__device__ __forceinline__ Vec<2> operator*(Vec<2> a, Vec<2> b) { return {__fmul2_rn(a.v, b.v)}; }
__device__ __forceinline__ Vec<1> operator+(Vec<1> a, Vec<1> b) { return {a.v + b.v}; }
__device__ __forceinline__ Vec<2> operator+(Vec<2> a, Vec<2> b) { return {__fadd2_rn(a.v, b.v)}; }
template <int VEC>
__device__ __forceinline__ Vec<VEC> operator-(Vec<VEC> a, Vec<VEC> b) { return fma(b, Vec<VEC>::all(-1.0f), a); }
__device__ __forceinline__ Vec<1> minus(Vec<1> a) { return {-a.v}; }
__device__ __forceinline__ Vec<2> minus(Vec<2> a) { return {make_float2(-a.v.x, -a.v.y)}; }
__device__ __forceinline__ Vec<1> ex2(Vec<1> a) { return {ex2(a.v)}; }
__device__ __forceinline__ Vec<2> ex2(Vec<2> a) { return {make_float2(ex2(a.v.x), ex2(a.v.y))}; }
__device__ __forceinline__ Vec<1> rcp(Vec<1> a) { return {rcp(a.v)}; }
__device__ __forceinline__ Vec<2> rcp(Vec<2> a) { return {make_float2(rcp(a.v.x), rcp(a.v.y))}; }
__device__ __forceinline__ Vec<1> pick(bool c, Vec<1> a, Vec<1> b) { return {c ? a.v : b.v}; }
__device__ __forceinline__ Vec<2> pick(bool c, Vec<2> a, Vec<2> b) { return {make_float2(c ? a.v.x : b.v.x, c ? a.v.y : b.v.y)}; }
template <typename F>
__device__ __forceinline__ Vec<1> map(F f, Vec<1> a, Vec<1> b) { return {f(a.v, b.v)}; }
template <typename F>
__device__ __forceinline__ Vec<2> map(F f, Vec<2> a, Vec<2> b) { return {make_float2(f(a.v.x, b.v.x), f(a.v.y, b.v.y))}; }
template <typename F>
__device__ __forceinline__ Vec<1> map(F f, Vec<1> a, Vec<1> b, Vec<1> c) { return {f(a.v, b.v, c.v)}; }
template <typename F>
__device__ __forceinline__ Vec<2> map(F f, Vec<2> a, Vec<2> b, Vec<2> c) {
  return {make_float2(f(a.v.x, b.v.x, c.v.x), f(a.v.y, b.v.y, c.v.y))};
}
template <int VEC>
__device__ __forceinline__ Vec<VEC> magnitude(Vec<VEC> a) { return map([](float x, float) { return fabsf(x); }, a, a); }

// sigmoid(x) to full relative accuracy at both ends
template <int VEC>
__device__ __forceinline__ Vec<VEC> sigmoid(Vec<VEC> x) {
  return rcp(ex2(x * Vec<VEC>::all(-kLog2e)) + Vec<VEC>::all(1.0f));
}
// -sigmoid(-x), the same
template <int VEC>
__device__ __forceinline__ Vec<VEC> minus_sigmoid_minus(Vec<VEC> x) {
  return rcp(Vec<VEC>::all(-1.0f) - ex2(x * Vec<VEC>::all(kLog2e)));
}
__device__ __forceinline__ float below(float x, float most) {     // NaN stays NaN
  float a;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(x), "f"(most));
  return a;
}
__device__ __forceinline__ Vec<1> below(Vec<1> x, float most) { return {below(x.v, most)}; }
__device__ __forceinline__ Vec<2> below(Vec<2> x, float most) { return {make_float2(below(x.v.x, most), below(x.v.y, most))}; }
// With e = exp(x), kept finite for its product with 0, to full relative accuracy at both ends:
// nf = -sigmoid(x) and nf1 = -sigmoid(-x)
template <int VEC>
__device__ __forceinline__ void gates(Vec<VEC> x, Vec<VEC>& nf, Vec<VEC>& nf1) {
  const Vec<VEC> e = ex2(below(x * Vec<VEC>::all(kLog2e), 126.0f));
  nf1 = rcp(Vec<VEC>::all(-1.0f) - e);
  nf = e * nf1;
}
// s = sigmoid(x) and s1 = sigmoid(-x)
template <int VEC>
__device__ __forceinline__ void both_sigmoids(Vec<VEC> x, Vec<VEC>& s, Vec<VEC>& s1) {
  const Vec<VEC> e = ex2(below(x * Vec<VEC>::all(-kLog2e), 126.0f));
  s = rcp(e + Vec<VEC>::all(1.0f));
  s1 = e * s;
}

// What moves a state, to full relative accuracy whichever way the gate stands: -(1 - f), from h on, where f >= 1/2, and f, from z on,
// where f < 1/2.  The fast walks have -(1 - f) throughout, which is a weight in this sense too.
template <int VEC>
__device__ __forceinline__ Vec<VEC> weight(Vec<VEC> x) {
  const auto of = [](float a, float m) { return __uint_as_float(__float_as_uint(m) | (~__float_as_uint(a) & 0x80000000u)); };
  const Vec<VEC> e = ex2(magnitude(x) * Vec<VEC>::all(-kLog2e));
  return map(of, x, e * rcp(e + Vec<VEC>::all(1.0f)));               // min(f, 1 - f) with the sign of -x
}
// a where the weight counts from h, else b
template <int VEC>
__device__ __forceinline__ Vec<VEC> side(Vec<VEC> w, Vec<VEC> a, Vec<VEC> b) {
  return map([](float w, float a, float b) { return __float_as_int(w) < 0 ? a : b; }, w, a, b);
}
// f h + (1 - f) z, with d = h - z
template <int VEC>
__device__ __forceinline__ Vec<VEC> moved(Vec<VEC> w, Vec<VEC> d, Vec<VEC> h, Vec<VEC> z) { return fma(w, d, side(w, h, z)); }
// f x
template <int VEC>
__device__ __forceinline__ Vec<VEC> kept(Vec<VEC> w, Vec<VEC> x) { return fma(w, x, side(w, x, Vec<VEC>::all(0.0f))); }
// -(1 - f) x
template <int VEC>
__device__ __forceinline__ Vec<VEC> minus_taken(Vec<VEC> w, Vec<VEC> x) { return fma(w, x, side(w, Vec<VEC>::all(0.0f), minus(x))); }
// f (1 - f) x
template <int VEC>
__device__ __forceinline__ Vec<VEC> both(Vec<VEC> w, Vec<VEC> x) {
  const Vec<VEC> m = magnitude(w);
  return fma(minus(m), m, m) * x;
}

// The same where values may be infinite, or their difference.  A gate's share is above 0 however small it is in fp32.
__device__ __forceinline__ float share(float a) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(1.17549435e-38f));
  return r;
}
__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) < INFINITY; }
__device__ __forceinline__ float f_of(float w) { return __float_as_int(w) < 0 ? 1.0f + w : w; }
__device__ __forceinline__ float f1_of(float w) { return __float_as_int(w) < 0 ? -w : 1.0f - w; }
__device__ __forceinline__ float share_of(float a, float x) { return (is_finite(x) ? a : share(a)) * x; }
template <int VEC>
__device__ __forceinline__ Vec<VEC> share_of(Vec<VEC> a, Vec<VEC> x) {
  return map([](float a, float x) { return share_of(a, x); }, a, x);
}
template <int VEC>
__device__ __forceinline__ Vec<VEC> any_moved(Vec<VEC> w, Vec<VEC> h, Vec<VEC> z) {
  return map([](float w, float h, float z) {
    const float d = h - z;
    return is_finite(d) ? fmaf(w, d, __float_as_int(w) < 0 ? h : z) : fmaf(share(f_of(w)), h, share(f1_of(w)) * z);
  }, w, h, z);
}
template <int VEC>
__device__ __forceinline__ Vec<VEC> any_kept(Vec<VEC> w, Vec<VEC> x) {
  return map([](float w, float x) { return is_finite(x) ? fmaf(w, x, __float_as_int(w) < 0 ? x : 0.0f) : share(f_of(w)) * x; }, w, x);
}
template <int VEC>
__device__ __forceinline__ Vec<VEC> any_taken(Vec<VEC> w, Vec<VEC> x) {
  return map([](float w, float x) {
    return is_finite(x) ? -fmaf(w, x, __float_as_int(w) < 0 ? 0.0f : -x) : share(f1_of(w)) * x;
  }, w, x);
}
template <int VEC>
__device__ __forceinline__ Vec<VEC> any_both(Vec<VEC> w, Vec<VEC> x) {
  return map([](float w, float x) { return share_of(fmaf(-fabsf(w), fabsf(w), fabsf(w)), x); }, w, x);
}

// VEC elements as they lie in memory
template <int VEC>
struct Raw {
  uint32_t u;
  __device__ __forceinline__ void load(const elem_t* p) {
    if constexpr (VEC == 2) u = *reinterpret_cast<const uint32_t*>(p);
    else u = *reinterpret_cast<const uint16_t*>(p);
  }
  __device__ __forceinline__ Vec<VEC> get() const {
    if constexpr (VEC == 2) return {e22ff(*reinterpret_cast<const elem2_t*>(&u))};
    else {
      const uint16_t h = (uint16_t)u;
      return {e2f(*reinterpret_cast<const elem_t*>(&h))};
    }
  }
};
__device__ __forceinline__ void store(elem_t* p, Vec<2> r) { *reinterpret_cast<elem2_t*>(p) = ff2e2(r.v.x, r.v.y); }
__device__ __forceinline__ void store(elem_t* p, Vec<1> r) { *p = f2e(r.v); }
__device__ __forceinline__ void store(float* p, Vec<2> r) { p[0] = r.v.x; p[1] = r.v.y; }
__device__ __forceinline__ void store(float* p, Vec<1> r) { *p = r.v; }
template <int VEC>
__device__ __forceinline__ Vec<VEC> load(const float* p) {
  if constexpr (VEC == 2) return {make_float2(p[0], p[1])};
  else return {*p};
}

// What a chunk makes of a value that comes in.  A gain below 0 marks a chunk with a reset: nothing of what comes in goes on,
// not even as a product of 0 with an infinity or a NaN of the sequence before.  A gain is never 0, for the same reason: of an
// infinite value that comes in, however small a share is infinite.
constexpr float kLeastGain = 0x1p-149f;
template <int VEC>
__device__ __forceinline__ Vec<VEC> above_zero(Vec<VEC> gain) {      // a NaN, which is in from0 too, is not kept
  return map([](float a, float b) { return fmaxf(a, b); }, gain, Vec<VEC>::all(kLeastGain));
}
template <int VEC>
struct Link {
  Vec<VEC> gain, from0;
  __device__ __forceinline__ Vec<VEC> operator()(Vec<VEC> x) const {
    return pick(gain.get(0) < 0.0f, from0, fma(gain, x, from0));      // a mark is in all of a lane's channels
  }
  // this one, then `next`
  __device__ __forceinline__ Link then(const Link& next) const {
    return {pick(gain.get(0) < 0.0f || next.gain.get(0) < 0.0f, Vec<VEC>::all(-1.0f), gain * next.gain), next(from0)};
  }
  __device__ __forceinline__ Link above0() const { return {pick(gain.get(0) < 0.0f, gain, above_zero(gain)), from0}; }
};

struct Shape {
  int batch, steps, dim, states;    // states: saved ones of a sequence
  long long zb, zt, zk;             // strides of zgo: sequence, step, member
  long long yb, yt;                 // of y, or of dy in the backward
  long long rb, rt;                 // of the resets
};

// The reset flags of a chunk, one bit a step; the same in all lanes.
__device__ __forceinline__ uint32_t reset_bits(const uint8_t* resets, const Shape& s, int b, int t0, int n) {
  if (resets == nullptr) return 0;
  const int lane = threadIdx.x % 32;
  const bool r = lane < n && resets[b * s.rb + (t0 + lane) * s.rt] != 0;
  return __ballot_sync(0xffffffffu, r);
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Sends a link to the same place in the shared memory of CTA `rank`, counted on the barrier at the same place there.
__device__ __forceinline__ void push(const Link<2>* place, uint64_t* bar, uint32_t rank, const Link<2>& l) {
  uint32_t at, at_bar;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(place)), "r"(rank));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at_bar) : "r"(smem_u32(bar)), "r"(rank));
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(at), "f"(l.gain.v.x),
               "f"(l.gain.v.y), "f"(l.from0.v.x), "f"(l.from0.v.y), "r"(at_bar) : "memory");
}
__device__ __forceinline__ void push(const Link<1>* place, uint64_t* bar, uint32_t rank, const Link<1>& l) {
  uint32_t at, at_bar;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(place)), "r"(rank));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at_bar) : "r"(smem_u32(bar)), "r"(rank));
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(at), "f"(l.gain.v), "f"(l.from0.v),
               "r"(at_bar) : "memory");
}

// The links of a walk step: of the warps of this CTA, and of the CTAs of the cluster, each sent there by its CTA.  Two sets take
// turns: whoever writes a set again has passed the step between, to which every reader of the set has contributed.
template <int VEC, int WARPS>
struct __align__(16) Exchange {
  Link<VEC> warps[2][WARPS][32];
  uint64_t arrived[2];              // behind it in shared memory: the links of the cluster's CTAs
  __device__ __forceinline__ Link<VEC>* cta(int turn, int c) {
    return reinterpret_cast<Link<VEC>*>(this + 1) + (turn * (int)cluster_size() + c) * 32 + threadIdx.x % 32;
  }
  // before the first exchange
  __device__ __forceinline__ void init() {
    if (cluster_size() == 1) return;
    if (threadIdx.x == 0) {
      mbar_init(&arrived[0], 1);
      mbar_init(&arrived[1], 1);
      mbar_fence_init();
    }
    cluster_sync();
  }
};

// Links are passed on in two halves, between which a warp has work that needs nothing from the others.  Chunks follow one another
// by (place of the CTA, place of the warp); round: of this launch, from 0.
template <int VEC, int WARPS>
struct Passing {
  Link<VEC> before;                 // of the warps of the CTA before this one

  __device__ __forceinline__ void send(Exchange<VEC, WARPS>& ex, int round, const Link<VEC>& mine, int place, bool backwards) {
    const int lane = threadIdx.x % 32, turn = round & 1;
    const int ctas = (int)cluster_size(), rank = (int)cluster_rank();
    ex.warps[turn][place][lane] = mine;
    __syncthreads();
    before = Link<VEC>{Vec<VEC>::all(1.0f), Vec<VEC>::all(0.0f)};
    if (ctas > 1) {
#pragma unroll
      for (int w = 0; w < WARPS - 1; ++w)
        if (w < place) before = before.then(ex.warps[turn][w][lane]);
      before = before.above0();
      if (place == WARPS - 1) {                                       // of the CTA as a whole
        const Link<VEC> all = before.then(mine).above0();
        if (lane == 0) mbar_expect_tx(&ex.arrived[turn], ctas * 32 * (uint32_t)sizeof(Link<VEC>));
        const int here = backwards ? ctas - 1 - rank : rank;
        for (int c = 0; c < ctas; ++c) push(ex.cta(turn, here), &ex.arrived[turn], c, all);
      }
    }
  }

  // What comes in to this warp's chunk; `carry` is what comes in to the cluster's first chunk, and becomes what its last hands on.
  __device__ __forceinline__ Vec<VEC> take(Exchange<VEC, WARPS>& ex, int round, int place, bool backwards, Vec<VEC>& carry, int* status) {
    const int lane = threadIdx.x % 32, turn = round & 1;
    const int ctas = (int)cluster_size(), rank = (int)cluster_rank();
    Vec<VEC> in = carry;
    if (ctas == 1) {
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        if (w == place) in = carry;
        carry = ex.warps[turn][w][lane](carry);
      }
    } else {
      if (!mbar_wait(&ex.arrived[turn], (round >> 1) & 1) && lane == 0) atomicExch(status, GEMM_ERR_EPILOGUE_TIMEOUT);
      const int here = backwards ? ctas - 1 - rank : rank;
#pragma unroll
      for (int c = 0; c < kMaxCtas; ++c) {
        if (c >= ctas) break;
        if (c == here) in = carry;
        carry = (*ex.cta(turn, c))(carry);
      }
      in = before(in);
    }
    return in;
  }
};

// The walks over a chunk of STEPS steps.  z, g, o, d: functions of the step that give the inputs (0 behind the end), put: one that
// takes an output.
// MASKED: steps may be missing at the end, or start a new sequence.
// EXACT: gates may be closed.  The fast walks move by -(1 - f) only: 1 - f is known to its last bits where f is near 1, but f h is
// off by a unit of h, which is much of it where f is small.  A chunk with a gate below kClosed (f = 1 / 150) is walked again by
// `weight`, two selections more a step and channel; its warp begins the next chunks that way, until one has no gate below
// kClosed + 1.  us with gates around 3 | 0 | -2 (spread 1), 1 x 30011 x 2048 bf16: forward 121 | 121 | 152, backward 203 | 203 | 239 (by the
// fast walks alone 119 and 193).
constexpr float kClosed = -5.0f;
// What the walks find out for the whole warp: the lowest gate, and whether every value that they passed was finite and no
// difference of two beyond the largest number (`probe` stays 0, else it becomes NaN; looked at in front of a reset and at the end,
// since what is not finite stays so).  Where one was not, `any_forward` and `any_backward` do the chunk again.
template <int VEC>
struct Found {
  float least = 0.0f;
  Vec<VEC> probe = Vec<VEC>::all(0.0f);
  __device__ __forceinline__ void gate(Vec<VEC> g) { least = fminf(fminf(least, g.get(0)), g.get(VEC - 1)); }
  __device__ __forceinline__ void value(Vec<VEC> x) { probe = fma(x, Vec<VEC>::all(0.0f), probe); }
  __device__ __forceinline__ bool clean() const { return probe.get(0) == 0.0f && probe.get(VEC - 1) == 0.0f; }
  __device__ __forceinline__ bool all_clean() const { return __all_sync(0xffffffffu, clean()); }
  __device__ __forceinline__ bool all_open(float bound) const { return __all_sync(0xffffffffu, least >= bound); }
  __device__ __forceinline__ bool all_fast() const { return __all_sync(0xffffffffu, least >= kClosed && clean()); }
};
// A value that comes in to a chunk of finite ones: so far below the largest number that it moves no difference beyond it
template <int VEC>
__device__ __forceinline__ bool moderate(Vec<VEC> x) { return fabsf(x.get(0)) < 0x1p60f && fabsf(x.get(VEC - 1)) < 0x1p60f; }

template <bool MASKED, bool EXACT, int STEPS, int VEC, typename Z, typename G>
__device__ __forceinline__ Found<VEC> forward_in(Vec<VEC> (&w)[STEPS], Link<VEC>& link, int n, uint32_t bits, Z z, G g) {
  using V = Vec<VEC>;
  Found<VEC> found;
  link.gain = V::all(1.0f);
  link.from0 = V::all(0.0f);
#pragma unroll
  for (int t = 0; t < STEPS; ++t) {
    if (MASKED && ((bits >> t) & 1)) {
      found.value(link.from0);
      link.from0 = V::all(0.0f);
    }
    const V gate = g(t);
    found.gate(gate);
    w[t] = EXACT ? weight<VEC>(gate) : minus_sigmoid_minus<VEC>(gate);
    if (MASKED && t >= n) w[t] = V::all(-0.0f);             // behind the end nothing changes
    const V d = link.from0 - z(t);
    if constexpr (EXACT) {
      link.from0 = moved(w[t], d, link.from0, z(t));
      link.gain = kept(w[t], link.gain);
    } else {
      link.from0 = fma(w[t], d, link.from0);
      link.gain = fma(w[t], link.gain, link.gain);
    }
  }
  if (EXACT) link.gain = above_zero(link.gain);
  if (MASKED && bits) link.gain = V::all(-1.0f);
  found.value(link.from0);
  return found;
}

// Output gates are formed while links are on their way, but only the first kAhead of a chunk: they lie in registers until h is
// there.  us by kAhead, 16 steps to a chunk, bf16: 1 x 30011 x 2048  0: 123  4: 119  8: 120  16: 131; 1 x 60000 x 512  0: 158
// 4: 150  8: 145  16: 156.
constexpr int kAhead = 8;
template <int VEC, typename O>
__device__ __forceinline__ void forward_ahead(Vec<VEC> (&so)[kAhead], O o) {
#pragma unroll
  for (int t = 0; t < kAhead; ++t) so[t] = sigmoid<VEC>(o(t));
}

template <bool MASKED, bool EXACT, int STEPS, int VEC, typename Z, typename O, typename P>
__device__ __forceinline__ Found<VEC> forward_out(const Vec<VEC> (&w)[STEPS], const Vec<VEC> (&so)[kAhead], Vec<VEC>& h, float* saved, int dim,
                                                  int n, uint32_t bits, Z z, O o, P put) {
  using V = Vec<VEC>;
  Found<VEC> found;
#pragma unroll
  for (int t = 0; t < STEPS; ++t) {
    if (t % kSaved == 0 && saved != nullptr && (!MASKED || t < n)) store(saved + t / kSaved * dim, h);
    if (MASKED && ((bits >> t) & 1)) {
      found.value(h);
      h = V::all(0.0f);
    }
    const V d = h - z(t);
    if constexpr (EXACT) h = moved(w[t], d, h, z(t));
    else h = fma(w[t], d, h);
    put(t, (t < kAhead ? so[t] : sigmoid<VEC>(o(t))) * h);
  }
  found.value(h);
  return found;
}

// The link and the outputs of a chunk whose values may be infinite, in loops of few instructions.  What is finite of it has the bits
// of the walk that it stands for.
template <int VEC, typename Z, typename G>
__device__ __forceinline__ void any_forward_in(bool exact, Link<VEC>& link, int n, uint32_t bits, Z z, G g) {
  using V = Vec<VEC>;
  link.gain = V::all(1.0f);
  link.from0 = V::all(0.0f);
#pragma unroll 1
  for (int t = 0; t < n; ++t) {
    const V w = exact ? weight<VEC>(g(t)) : minus_sigmoid_minus<VEC>(g(t));
    if ((bits >> t) & 1) link.from0 = V::all(0.0f);
    link.from0 = any_moved<VEC>(w, link.from0, z(t));
    link.gain = kept(w, link.gain);
  }
  link.gain = bits ? V::all(-1.0f) : above_zero(link.gain);
}
template <int VEC, typename Z, typename G, typename O, typename P>
__device__ __forceinline__ void any_forward_out(bool exact, Vec<VEC>& h, float* saved, int dim, int n, uint32_t bits, Z z, G g, O o, P put) {
  using V = Vec<VEC>;
#pragma unroll 1
  for (int t = 0; t < n; ++t) {
    if (t % kSaved == 0 && saved != nullptr) store(saved + t / kSaved * dim, h);
    if ((bits >> t) & 1) h = V::all(0.0f);
    h = any_moved<VEC>(exact ? weight<VEC>(g(t)) : minus_sigmoid_minus<VEC>(g(t)), h, z(t));
    put(t, share_of(sigmoid<VEC>(o(t)), h));
  }
}

// What a link needs: w, nf = -f (not where EXACT), so1 = 1 - sigmoid(o), and dh0, the part of dh that a step's own y gives.
template <bool MASKED, bool EXACT, int STEPS, int VEC, typename G, typename O, typename D>
__device__ __forceinline__ Found<VEC> backward_in(Vec<VEC> (&w)[STEPS], Vec<VEC> (&nf)[STEPS], Vec<VEC> (&so1)[STEPS],
                                                  Vec<VEC> (&dh0)[STEPS], Link<VEC>& link, int n, uint32_t bits, G g, O o, D d) {
  using V = Vec<VEC>;
  Found<VEC> found;
#pragma unroll
  for (int t = 0; t < STEPS; ++t) {
    V so;
    const V gate = g(t);
    found.gate(gate);
    if constexpr (EXACT) w[t] = weight<VEC>(gate);
    else gates<VEC>(gate, nf[t], w[t]);
    both_sigmoids<VEC>(o(t), so, so1[t]);
    dh0[t] = d(t) * so;
    if (MASKED && t >= n) w[t] = V::all(-0.0f), dh0[t] = V::all(0.0f);      // behind the end e passes unchanged
  }
  link.gain = V::all(1.0f);
  link.from0 = V::all(0.0f);
#pragma unroll
  for (int t = STEPS - 1; t >= 0; --t) {
    const V dh = link.from0 + dh0[t];
    if constexpr (EXACT) {
      link.from0 = kept(w[t], dh);
      link.gain = kept(w[t], link.gain);
    } else {
      link.from0 = fma(w[t], dh, dh);
      link.gain = fma(w[t], link.gain, link.gain);
    }
    if (MASKED && ((bits >> t) & 1)) {
      found.value(link.from0);
      link.from0 = V::all(0.0f);
    }
  }
  if (EXACT) link.gain = above_zero(link.gain);
  if (MASKED && bits) link.gain = V::all(-1.0f);
  found.value(link.from0);
  return found;
}

// Forwards over the chunk from the state h in front of it: the gradient of the output gates, and u, the factor of dg, over nf.
template <bool MASKED, bool EXACT, int STEPS, int VEC, typename Z, typename P>
__device__ __forceinline__ Found<VEC> backward_states(const Vec<VEC> (&w)[STEPS], Vec<VEC> (&nf)[STEPS], const Vec<VEC> (&so1)[STEPS],
                                                      const Vec<VEC> (&dh0)[STEPS], Vec<VEC> h, uint32_t bits, Z z, P put) {
  using V = Vec<VEC>;
  Found<VEC> found;
#pragma unroll
  for (int t = 0; t < STEPS; ++t) {
    if (MASKED && ((bits >> t) & 1)) {
      found.value(h);
      h = V::all(0.0f);
    }
    const V step = h - z(t);
    if constexpr (EXACT) {
      h = moved(w[t], step, h, z(t));
      nf[t] = both(w[t], step);
    } else {
      h = fma(w[t], step, h);
      nf[t] = (step * nf[t]) * w[t];
    }
    put(t, (dh0[t] * h) * so1[t]);
  }
  found.value(h);
  return found;
}

template <bool MASKED, bool EXACT, int STEPS, int VEC, typename P, typename Q>
__device__ __forceinline__ Found<VEC> backward_out(const Vec<VEC> (&w)[STEPS], const Vec<VEC> (&u)[STEPS], const Vec<VEC> (&dh0)[STEPS],
                                                   Vec<VEC>& e, uint32_t bits, P put_z, Q put_g) {
  using V = Vec<VEC>;
  Found<VEC> found;
#pragma unroll
  for (int t = STEPS - 1; t >= 0; --t) {
    const V dh = e + dh0[t];
    put_g(t, u[t] * dh);
    if constexpr (EXACT) {
      put_z(t, minus(minus_taken(w[t], dh)));
      e = kept(w[t], dh);
    } else {
      put_z(t, minus(w[t] * dh));
      e = fma(w[t], dh, dh);
    }
    if (MASKED && ((bits >> t) & 1)) {
      found.value(e);
      e = V::all(0.0f);
    }
  }
  found.value(e);
  return found;
}

// The same for a chunk whose values may be infinite: its link, and all of its gradients.
template <int VEC, typename G, typename O, typename D>
__device__ __forceinline__ void any_backward_in(bool exact, Link<VEC>& link, int n, uint32_t bits, G g, O o, D d) {
  using V = Vec<VEC>;
  link.gain = V::all(1.0f);
  link.from0 = V::all(0.0f);
#pragma unroll 1
  for (int t = n - 1; t >= 0; --t) {
    V w, nf, so, so1;
    gates<VEC>(g(t), nf, w);
    if (exact) w = weight<VEC>(g(t));
    both_sigmoids<VEC>(o(t), so, so1);
    link.from0 = any_kept<VEC>(w, link.from0 + share_of(so, d(t)));
    if ((bits >> t) & 1) link.from0 = V::all(0.0f);
    link.gain = kept(w, link.gain);
  }
  link.gain = bits ? V::all(-1.0f) : above_zero(link.gain);
}
// h: in front of the chunk.  The state in front of a step is walked to anew for each.
template <int VEC, typename Z, typename G, typename O, typename D, typename P, typename Q, typename R>
__device__ __forceinline__ void any_backward(bool exact, const Vec<VEC> h, Vec<VEC>& e, int n, uint32_t bits, Z z, G g, O o, D d, P put_z,
                                             Q put_g, R put_o) {
  using V = Vec<VEC>;
#pragma unroll 1
  for (int t = n - 1; t >= 0; --t) {
    V at = h, before = h, w, nf;
#pragma unroll 1
    for (int q = 0; q <= t; ++q) {
      gates<VEC>(g(q), nf, w);
      if (exact) w = weight<VEC>(g(q));
      before = (bits >> q) & 1 ? V::all(0.0f) : at;
      at = any_moved<VEC>(w, before, z(q));
    }
    V so, so1;
    both_sigmoids<VEC>(o(t), so, so1);
    const V step = before - z(t), dh0 = share_of(so, d(t)), dh = e + dh0;
    const V fast = share_of(minus(w), share_of(minus(nf), step));
    put_o(t, share_of(so1, dh0 * at));
    put_g(t, (exact ? any_both<VEC>(w, step) : fast) * dh);
    put_z(t, any_taken<VEC>(w, dh));
    e = any_kept<VEC>(w, dh);
    if ((bits >> t) & 1) e = V::all(0.0f);
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Any alignment, and a few steps: inputs in registers by plain loads
// ---------------------------------------------------------------------------------------------------------------
// A lane's VEC channels in a row of them; a lane behind the last one computes it too, and stores nothing.
template <int VEC>
struct Channels {
  int ch;
  bool in;
  __device__ __forceinline__ Channels(int slab, int dim) {
    const int own = (slab * 32 + (int)threadIdx.x % 32) * VEC;
    in = own < dim;
    ch = in ? own : dim - VEC;
  }
  template <int STEPS>
  __device__ __forceinline__ void fetch(Raw<VEC> (&r)[STEPS], const elem_t* row, long long step, int n) const {
#pragma unroll
    for (int t = 0; t < STEPS; ++t) {
      r[t].u = 0;
      if (t < n) r[t].load(row + t * step + ch);
    }
  }
  __device__ __forceinline__ Vec<VEC> read(const elem_t* row) const {
    Raw<VEC> r;
    r.load(row + ch);
    return r.get();
  }
  __device__ __forceinline__ Vec<VEC> load(const float* row) const {
    if constexpr (VEC == 1) return {row[ch]};
    else return {make_float2(row[ch], row[ch + 1])};
  }
  template <typename T>
  __device__ __forceinline__ void put(T* row, Vec<VEC> v) const {
    if (in) store(row + ch, v);
  }
};

template <int VEC, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 2)
recurrence_fwd_kernel(const elem_t* __restrict__ zgo, const float* __restrict__ state_in, const uint8_t* __restrict__ resets,
                      elem_t* __restrict__ y, float* __restrict__ state_out, float* __restrict__ saved, int* status, const Shape s) {
  constexpr int STEPS = kSaved;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  Exchange<VEC, WARPS>& ex = *reinterpret_cast<Exchange<VEC, WARPS>*>(smem_raw);
  ex.init();
  const int warp = threadIdx.x / 32;
  const int ctas = (int)cluster_size(), rank = (int)cluster_rank();
  const int slabs = (s.dim + 32 * VEC - 1) / (32 * VEC), unit = blockIdx.x / ctas, b = unit / slabs;
  const Channels<VEC> c(unit % slabs, s.dim);
  Vec<VEC> carry = state_in != nullptr ? c.load(state_in + (long long)b * s.dim) : Vec<VEC>::all(0.0f);
  int round = 0;
  bool closed = false;              // gates of the last chunk
  for (int c0 = 0; c0 < s.states; c0 += ctas * WARPS, ++round) {
    const int chunk = c0 + rank * WARPS + warp, t0 = chunk * STEPS;
    const int n = min(STEPS, s.steps - t0);                 // may be below 0
    const uint32_t bits = reset_bits(resets, s, b, t0, n);
    const elem_t* src = zgo + b * s.zb + t0 * s.zt;
    Raw<VEC> z[STEPS], g[STEPS], o[STEPS];
    c.fetch(g, src + s.zk, s.zt, n);
    c.fetch(z, src, s.zt, n);
    c.fetch(o, src + 2 * s.zk, s.zt, n);
    const auto get_z = [&](int t) { return z[t].get(); };
    const auto get_g = [&](int t) { return g[t].get(); };
    const auto get_o = [&](int t) { return o[t].get(); };
    Vec<VEC> w[STEPS], so[kAhead];
    Link<VEC> link;
    Vec<VEC> h;
    bool exact = WARPS == 1 || closed;
    bool any = false;
    if (!exact) {
      const Found<VEC> found = forward_in<true, false>(w, link, n, bits, get_z, get_g);
      if (__builtin_expect(!found.all_fast(), 0)) {
        exact = !found.all_open(kClosed);
        any = !exact;
      }
    }
    if (exact) {
      const Found<VEC> found = forward_in<true, true>(w, link, n, bits, get_z, get_g);
      if constexpr (WARPS > 1) {
        closed = !found.all_open(kClosed + 1.0f);
        any = !found.all_clean();
      }
    }
    const auto mem_z = [&](int t) { return c.read(src + t * s.zt); };
    const auto mem_g = [&](int t) { return c.read(src + t * s.zt + s.zk); };
    const auto mem_o = [&](int t) { return c.read(src + t * s.zt + 2 * s.zk); };
    if constexpr (WARPS == 1) {                             // needs no link
      forward_ahead(so, get_o);
      h = carry;
    } else {
      if (__builtin_expect(any, 0)) any_forward_in<VEC>(exact, link, n, bits, mem_z, mem_g);
      Passing<VEC, WARPS> passing;
      passing.send(ex, round, link, warp, false);
      forward_ahead(so, get_o);
      h = passing.take(ex, round, warp, false, carry, status);
      any = any || !__all_sync(0xffffffffu, moderate(h));
    }
    elem_t* out = y + b * s.yb + t0 * s.yt;
    float* at = saved != nullptr && c.in ? saved + ((long long)b * s.states + chunk) * s.dim + c.ch : nullptr;
    const auto put = [&](int t, Vec<VEC> v) { if (t < n) c.put(out + t * s.yt, v); };
    if (!any) {
      if (!exact) forward_out<true, false>(w, so, h, at, s.dim, n, bits, get_z, get_o, put);
      else if (!forward_out<true, true>(w, so, h, at, s.dim, n, bits, get_z, get_o, put).all_clean() && WARPS == 1) any = true, h = carry;
    }
    if (__builtin_expect(any, 0)) any_forward_out<VEC>(exact, h, at, s.dim, n, bits, mem_z, mem_g, mem_o, put);
    if constexpr (WARPS == 1) carry = h;
    if (t0 + STEPS >= s.steps && n > 0) c.put(state_out + (long long)b * s.dim, h);
  }
  if (ctas > 1) cluster_sync();     // no CTA leaves while another may still read its links
}

template <int VEC, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 2)
recurrence_bwd_kernel(const elem_t* __restrict__ zgo, const uint8_t* __restrict__ resets, const float* __restrict__ saved,
                      const elem_t* __restrict__ dy, const float* __restrict__ d_state_out, elem_t* __restrict__ d_zgo,
                      float* __restrict__ d_state_in, int* status, const Shape s, long long db, long long dt) {
  constexpr int STEPS = kSaved;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  Exchange<VEC, WARPS>& ex = *reinterpret_cast<Exchange<VEC, WARPS>*>(smem_raw);
  ex.init();
  const int warp = threadIdx.x / 32;
  const int ctas = (int)cluster_size(), rank = (int)cluster_rank();
  const int slabs = (s.dim + 32 * VEC - 1) / (32 * VEC), unit = blockIdx.x / ctas, b = unit / slabs;
  const Channels<VEC> c(unit % slabs, s.dim);
  Vec<VEC> carry = d_state_out != nullptr ? c.load(d_state_out + (long long)b * s.dim) : Vec<VEC>::all(0.0f);
  const int per_step = ctas * WARPS, rounds = (s.states + per_step - 1) / per_step;
  bool closed = false;
  for (int round = 0; round < rounds; ++round) {
    const int chunk = (rounds - 1 - round) * per_step + rank * WARPS + warp, t0 = chunk * STEPS;
    const int n = min(STEPS, s.steps - t0);
    const uint32_t bits = reset_bits(resets, s, b, t0, n);
    const elem_t* src = zgo + b * s.zb + t0 * s.zt;
    elem_t* out = d_zgo + b * db + t0 * dt;
    Raw<VEC> z[STEPS], g[STEPS], o[STEPS], d[STEPS];
    c.fetch(g, src + s.zk, s.zt, n);
    c.fetch(z, src, s.zt, n);
    c.fetch(o, src + 2 * s.zk, s.zt, n);
    c.fetch(d, dy + b * s.yb + t0 * s.yt, s.yt, n);
    const Vec<VEC> h = n > 0 ? c.load(saved + ((long long)b * s.states + chunk) * s.dim) : Vec<VEC>::all(0.0f);
    const auto get_z = [&](int t) { return z[t].get(); };
    const auto get_g = [&](int t) { return g[t].get(); };
    const auto get_o = [&](int t) { return o[t].get(); };
    const auto get_d = [&](int t) { return d[t].get(); };
    const auto put_z = [&](int t, Vec<VEC> v) { if (t < n) c.put(out + t * dt, v); };
    const auto put_g = [&](int t, Vec<VEC> v) { if (t < n) c.put(out + t * dt + s.dim, v); };
    const auto put_o = [&](int t, Vec<VEC> v) { if (t < n) c.put(out + t * dt + 2 * s.dim, v); };
    Vec<VEC> w[STEPS], u[STEPS], so1[STEPS], dh0[STEPS];
    Link<VEC> link;
    bool exact = WARPS == 1 || closed;
    bool any = false;
    if (!exact) {
      const Found<VEC> found = backward_in<true, false>(w, u, so1, dh0, link, n, bits, get_g, get_o, get_d);
      if (__builtin_expect(!found.all_fast(), 0)) {
        exact = !found.all_open(kClosed);
        any = !exact;
      }
    }
    if (exact) {
      const Found<VEC> found = backward_in<true, true>(w, u, so1, dh0, link, n, bits, get_g, get_o, get_d);
      if constexpr (WARPS > 1) {
        closed = !found.all_open(kClosed + 1.0f);
        any = !found.all_clean();
      }
    }
    const auto mem_z = [&](int t) { return c.read(src + t * s.zt); };
    const auto mem_g = [&](int t) { return c.read(src + t * s.zt + s.zk); };
    const auto mem_o = [&](int t) { return c.read(src + t * s.zt + 2 * s.zk); };
    const auto mem_d = [&](int t) { return c.read(dy + b * s.yb + (t0 + t) * s.yt); };
    Passing<VEC, WARPS> passing;
    if constexpr (WARPS > 1) {
      if (__builtin_expect(any, 0)) any_backward_in<VEC>(exact, link, n, bits, mem_g, mem_o, mem_d);
      passing.send(ex, round, link, WARPS - 1 - warp, true);
    }
    Found<VEC> found = exact ? backward_states<true, true>(w, u, so1, dh0, h, bits, get_z, put_o)
                             : backward_states<true, false>(w, u, so1, dh0, h, bits, get_z, put_o);
    Vec<VEC> e = carry;
    if constexpr (WARPS > 1) {
      e = passing.take(ex, round, WARPS - 1 - warp, true, carry, status);
      any = any || !__all_sync(0xffffffffu, found.clean() && moderate(h) && moderate(e));
    }
    if (!any) {
      if (!exact) {
        backward_out<true, false>(w, u, dh0, e, bits, put_z, put_g);
      } else {
        const Found<VEC> last = backward_out<true, true>(w, u, dh0, e, bits, put_z, put_g);
        if (WARPS == 1 && !__all_sync(0xffffffffu, found.clean() && last.clean())) any = true, e = carry;
      }
    }
    if (__builtin_expect(any, 0)) any_backward<VEC>(exact, h, e, n, bits, mem_z, mem_g, mem_o, mem_d, put_z, put_g, put_o);
    if constexpr (WARPS == 1) carry = e;
  }
  if (rank == 0 && warp == 0 && d_state_in != nullptr) c.put(d_state_in + (long long)b * s.dim, carry);
  if (ctas > 1) cluster_sync();
}

// ---------------------------------------------------------------------------------------------------------------
// Rows of 16-byte pieces: tiles by TMA.  Each warp fetches the chunk of its next walk step while it works on this one, and
// writes results over the inputs that it has read, from where they leave by TMA; what lies behind the last step or channel is
// filled with zeros on the way in and clipped on the way out.
// ---------------------------------------------------------------------------------------------------------------
constexpr int kWarps = 8, kSlab = 64;       // channels of a tile: two a lane

// This lane's two channels of a row of a tile
__device__ __forceinline__ Vec<2> get(const elem_t* row) { return {e22ff(*reinterpret_cast<const elem2_t*>(row))}; }

template <int STEPS>
struct FwdSmem {
  alignas(128) elem_t tiles[kWarps][2][3][STEPS][kSlab];
  uint64_t full_zg[kWarps][2], full_o[kWarps][2];
  Exchange<2, kWarps> ex;           // the last one
};

template <int STEPS>
__global__ void __launch_bounds__(kWarps * 32, 2)
recurrence_fwd_tma_kernel(const __grid_constant__ CUtensorMap map_in, const __grid_constant__ CUtensorMap map_y,
                          const float* __restrict__ state_in, const uint8_t* __restrict__ resets, float* __restrict__ state_out,
                          float* __restrict__ saved, int* status, const Shape s) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  FwdSmem<STEPS>& sm = *reinterpret_cast<FwdSmem<STEPS>*>(smem_raw);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int ctas = (int)cluster_size(), rank = (int)cluster_rank();
  const int slabs = (s.dim + kSlab - 1) / kSlab, unit = blockIdx.x / ctas;
  const int b = unit / slabs, ch0 = unit % slabs * kSlab, ch = ch0 + 2 * lane;
  const bool in = ch < s.dim;
  if (lane == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.full_zg[warp][i], 1);
      mbar_init(&sm.full_o[warp][i], 1);
    }
    mbar_fence_init();
  }
  sm.ex.init();
  __syncwarp();
  auto issue_zg = [&](int t0, int buf) {                    // one lane
    mbar_expect_tx(&sm.full_zg[warp][buf], 2 * STEPS * kSlab * 2);
    for (int k = 0; k < 2; ++k) tma_load_4d(sm.tiles[warp][buf][k], &map_in, &sm.full_zg[warp][buf], ch0, k, t0, b);
  };
  auto issue_o = [&](int t0, int buf) {
    mbar_expect_tx(&sm.full_o[warp][buf], STEPS * kSlab * 2);
    tma_load_4d(sm.tiles[warp][buf][2], &map_in, &sm.full_o[warp][buf], ch0, 2, t0, b);
  };
  Vec<2> carry = Vec<2>::all(0.0f);
  if (in && state_in != nullptr) carry = load<2>(state_in + (long long)b * s.dim + ch);
  const int per_step = ctas * kWarps * STEPS;
  int t0 = (rank * kWarps + warp) * STEPS;
  if (lane == 0 && t0 < s.steps) {
    issue_zg(t0, 0);
    issue_o(t0, 0);
  }
  uint32_t next_bits = reset_bits(resets, s, b, t0, min(STEPS, s.steps - t0));
  bool closed = false;              // gates of the last chunk
  for (int base = 0, round = 0; base < s.steps; base += per_step, t0 += per_step, ++round) {
    const int turn = round & 1;
    const int n = min(STEPS, s.steps - t0);                 // may be below 0
    const uint32_t bits = next_bits;
    const bool whole = n == STEPS && bits == 0;
    const elem_t *zs = &sm.tiles[warp][turn][0][0][2 * lane], *gs = &sm.tiles[warp][turn][1][0][2 * lane];
    elem_t* oy = &sm.tiles[warp][turn][2][0][2 * lane];
    const bool more = t0 + per_step < s.steps;
    if (n > 0 && !mbar_wait(&sm.full_zg[warp][turn], (round >> 1) & 1) && lane == 0) atomicExch(status, GEMM_ERR_PRODUCER_TIMEOUT);
    if (more && lane == 0) issue_zg(t0 + per_step, turn ^ 1);
    if (more) next_bits = reset_bits(resets, s, b, t0 + per_step, min(STEPS, s.steps - t0 - per_step));
    auto z = [&](int t) { return get(zs + t * kSlab); };
    auto g = [&](int t) { return get(gs + t * kSlab); };
    auto o = [&](int t) { return get(oy + t * kSlab); };
    auto put = [&](int t, Vec<2> v) { store(oy + t * kSlab, v); };
    Vec<2> w[STEPS], so[kAhead];
    Link<2> link{Vec<2>::all(1.0f), Vec<2>::all(0.0f)};
    bool exact = closed || !whole;
    bool any = false;
    if (!exact) {
      const Found<2> found = forward_in<false, false>(w, link, n, bits, z, g);
      if (__builtin_expect(!found.all_fast(), 0)) {
        exact = !found.all_open(kClosed);
        any = !exact;
      }
    }
    if (__builtin_expect(exact && n > 0, 0)) {
      const Found<2> found = forward_in<true, true>(w, link, n, bits, z, g);
      closed = !found.all_open(kClosed + 1.0f);
      any = !found.all_clean();
    }
    if (__builtin_expect(any, 0)) any_forward_in<2>(exact, link, n, bits, z, g);
    Passing<2, kWarps> passing;
    passing.send(sm.ex, round, link, warp, false);
    // Results go over the output gates that they come from.  The ones of the step before take a while to leave the other buffer,
    // so its output gates, which are needed last, are fetched only now.
    if (more && lane == 0) {
      bulk_wait_group_read<0>();
      issue_o(t0 + per_step, turn ^ 1);
    }
    __syncwarp();
    if (n > 0) {
      if (!mbar_wait(&sm.full_o[warp][turn], (round >> 1) & 1) && lane == 0) atomicExch(status, GEMM_ERR_PRODUCER_TIMEOUT);
      forward_ahead(so, o);
    }
    Vec<2> h = passing.take(sm.ex, round, warp, false, carry, status);
    if (n <= 0) continue;
    float* at = saved != nullptr && in ? saved + ((long long)b * s.states + t0 / kSaved) * s.dim + ch : nullptr;
    if (any || !__all_sync(0xffffffffu, moderate(h))) any_forward_out<2>(exact, h, at, s.dim, n, bits, z, g, o, put);
    else if (exact) forward_out<true, true>(w, so, h, at, s.dim, n, bits, z, o, put);
    else forward_out<false, false>(w, so, h, at, s.dim, n, bits, z, o, put);
    if (in && t0 + STEPS >= s.steps) store(state_out + (long long)b * s.dim + ch, h);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      tma_store_3d(&map_y, sm.tiles[warp][turn][2], ch0, t0, b);
      bulk_commit_group();
    }
  }
  if (lane == 0) bulk_wait_group_all();
  if (ctas > 1) cluster_sync();     // no CTA leaves while another may still read its links
}

template <int STEPS>
struct BwdSmem {
  alignas(128) elem_t zgo[kWarps][2][STEPS][3][kSlab];
  alignas(128) elem_t dy[kWarps][2][STEPS][kSlab];
  alignas(128) elem_t results[kWarps][STEPS][3][kSlab];
  alignas(128) float states[kWarps][2][kSlab];
  uint64_t full[kWarps][2];
  Exchange<2, kWarps> ex;           // the last one
};

template <int STEPS>
__global__ void __launch_bounds__(kWarps * 32, 2)
recurrence_bwd_tma_kernel(const __grid_constant__ CUtensorMap map_in, const __grid_constant__ CUtensorMap map_dy,
                          const __grid_constant__ CUtensorMap map_out, const uint8_t* __restrict__ resets,
                          const float* __restrict__ saved, const float* __restrict__ d_state_out, float* __restrict__ d_state_in,
                          int* status, const Shape s) {
  static_assert(STEPS == kSaved, "a chunk starts from a saved state");
  extern __shared__ __align__(128) uint8_t smem_raw[];
  BwdSmem<STEPS>& sm = *reinterpret_cast<BwdSmem<STEPS>*>(smem_raw);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int ctas = (int)cluster_size(), rank = (int)cluster_rank();
  const int slabs = (s.dim + kSlab - 1) / kSlab, unit = blockIdx.x / ctas;
  const int b = unit / slabs, ch0 = unit % slabs * kSlab, ch = ch0 + 2 * lane;
  const bool in = ch < s.dim;
  if (lane == 0) {
    for (int i = 0; i < 2; ++i) mbar_init(&sm.full[warp][i], 1);
    mbar_fence_init();
  }
  sm.ex.init();
  __syncwarp();
  const int state_bytes = min(kSlab, s.dim - ch0) * 4;
  // One lane.  A chunk's three members come and go as one copy: 1 x 30011 x 2048 189 us, 197 as one each.  (The forward, which
  // fetches z and g as one copy and o as another, gains nothing: 119 | 119, and 1 x 60000 x 512 loses, 160 | 144.)
  auto issue = [&](int t0, int buf) {
    mbar_expect_tx(&sm.full[warp][buf], 4 * STEPS * kSlab * 2 + state_bytes);
    bulk_load(sm.states[warp][buf], saved + ((long long)b * s.states + t0 / kSaved) * s.dim + ch0, state_bytes, &sm.full[warp][buf]);
    tma_load_4d(sm.zgo[warp][buf], &map_in, &sm.full[warp][buf], ch0, 0, t0, b);
    tma_load_3d(sm.dy[warp][buf], &map_dy, &sm.full[warp][buf], ch0, t0, b);
  };
  Vec<2> carry = Vec<2>::all(0.0f);
  if (in && d_state_out != nullptr) carry = load<2>(d_state_out + (long long)b * s.dim + ch);
  const int per_step = ctas * kWarps * STEPS, rounds = (s.steps + per_step - 1) / per_step;
  int t0 = (rounds - 1) * per_step + (rank * kWarps + warp) * STEPS;
  if (lane == 0 && t0 < s.steps) issue(t0, 0);
  uint32_t next_bits = reset_bits(resets, s, b, t0, min(STEPS, s.steps - t0));
  uint32_t phases = 0;
  bool closed = false;
  for (int round = 0, stage = 0; round < rounds; ++round, t0 -= per_step, stage ^= 1) {
    const int n = min(STEPS, s.steps - t0);
    const uint32_t bits = next_bits;
    const bool whole = n == STEPS && bits == 0;
    const elem_t *zgo = &sm.zgo[warp][stage][0][0][2 * lane], *dy = &sm.dy[warp][stage][0][2 * lane];
    elem_t* result = &sm.results[warp][0][0][2 * lane];
    if (n > 0) {
      if (!mbar_wait(&sm.full[warp][stage], (phases >> stage) & 1) && lane == 0) atomicExch(status, GEMM_ERR_PRODUCER_TIMEOUT);
      phases ^= 1u << stage;
    }
    if (round + 1 < rounds) {
      if (lane == 0) issue(t0 - per_step, stage ^ 1);
      next_bits = reset_bits(resets, s, b, t0 - per_step, min(STEPS, s.steps - t0 + per_step));
    }
    auto z = [&](int t) { return get(zgo + 3 * t * kSlab); };
    auto g = [&](int t) { return get(zgo + (3 * t + 1) * kSlab); };
    auto o = [&](int t) { return get(zgo + (3 * t + 2) * kSlab); };
    auto d = [&](int t) { return get(dy + t * kSlab); };
    elem2_t dout[STEPS];
    auto put_z = [&](int t, Vec<2> v) { store(result + 3 * t * kSlab, v); };
    auto put_g = [&](int t, Vec<2> v) { store(result + (3 * t + 1) * kSlab, v); };
    auto put_o = [&](int t, Vec<2> v) { dout[t] = ff2e2(v.v.x, v.v.y); };
    Vec<2> w[STEPS], u[STEPS], so1[STEPS], dh0[STEPS];
    Link<2> link{Vec<2>::all(1.0f), Vec<2>::all(0.0f)};
    bool exact = closed || !whole;
    bool any = false;
    if (!exact) {
      const Found<2> found = backward_in<false, false>(w, u, so1, dh0, link, n, bits, g, o, d);
      if (__builtin_expect(!found.all_fast(), 0)) {
        exact = !found.all_open(kClosed);
        any = !exact;
      }
    }
    if (__builtin_expect(exact && n > 0, 0)) {
      const Found<2> found = backward_in<true, true>(w, u, so1, dh0, link, n, bits, g, o, d);
      closed = !found.all_open(kClosed + 1.0f);
      any = !found.all_clean();
    }
    if (__builtin_expect(any, 0)) any_backward_in<2>(exact, link, n, bits, g, o, d);
    Passing<2, kWarps> passing;
    passing.send(sm.ex, round, link, kWarps - 1 - warp, true);
    const Vec<2> h = load<2>(&sm.states[warp][stage][2 * lane]);
    Found<2> found;
    if (!exact) found = backward_states<false, false>(w, u, so1, dh0, h, bits, z, put_o);
    else if (n > 0) found = backward_states<true, true>(w, u, so1, dh0, h, bits, z, put_o);
    const bool ok = found.clean() && moderate(h);
    Vec<2> e = passing.take(sm.ex, round, kWarps - 1 - warp, true, carry, status);
    if (n <= 0) continue;
    if (lane == 0) bulk_wait_group_read<0>();               // the results of the step before have left
    __syncwarp();
    any = any || !__all_sync(0xffffffffu, !in || (ok && moderate(e)));
    if (any) {
      any_backward<2>(exact, h, e, n, bits, z, g, o, d, put_z, put_g, [&](int t, Vec<2> v) { store(result + (3 * t + 2) * kSlab, v); });
    } else {
#pragma unroll
      for (int t = 0; t < STEPS; ++t) *reinterpret_cast<elem2_t*>(result + (3 * t + 2) * kSlab) = dout[t];
      if (exact) backward_out<true, true>(w, u, dh0, e, bits, put_z, put_g);
      else backward_out<false, false>(w, u, dh0, e, bits, put_z, put_g);
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      tma_store_4d(&map_out, sm.results[warp], ch0, 0, t0, b);
      bulk_commit_group();
    }
  }
  if (in && rank == 0 && warp == 0 && d_state_in != nullptr) store(d_state_in + (long long)b * s.dim + ch, carry);
  if (lane == 0) bulk_wait_group_all();
  if (ctas > 1) cluster_sync();
}

template <int N>
using Int = std::integral_constant<int, N>;

// Two neighbouring channels per lane where they lie on 4-byte boundaries
bool pairs(const void* p, int dim, long long a, long long b, long long c) {
  return dim % 2 == 0 && ((a | b | c) & 1) == 0 && (reinterpret_cast<uintptr_t>(p) & 3) == 0;
}
// What a tensor map takes: rows and strides of 16-byte pieces
bool pieces(const void* p, int dim, long long a, long long b, long long c) {
  return dim % 8 == 0 && ((a | b | c) & 7) == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0 && a > 0 && b > 0 && c > 0 &&
         a < (1ll << 38) && b < (1ll << 38) && c < (1ll << 38);
}

// (batch, steps, 3, dim), or (batch, steps, dim) with members = 0, in boxes of `box` steps, `members` and kSlab channels
int encode(CUtensorMap* map, const void* p, const Shape& s, long long sb, long long st, long long sk, int members, int box) {
  auto enc = fbam_encode_tiled();
  if (!enc) return GEMM_ERR_DRIVER;
  fbam_bind_context_to_thread();
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  CUresult r;
  if (members) {
    const cuuint64_t dims[4] = {(cuuint64_t)s.dim, 3, (cuuint64_t)s.steps, (cuuint64_t)s.batch};
    const cuuint64_t strides[3] = {(cuuint64_t)sk * 2, (cuuint64_t)st * 2, (cuuint64_t)sb * 2};
    const cuuint32_t boxes[4] = {kSlab, (cuuint32_t)members, (cuuint32_t)box, 1};
    r = enc(map, ELEM_TMAP, 4, const_cast<void*>(p), dims, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  } else {
    const cuuint64_t dims[3] = {(cuuint64_t)s.dim, (cuuint64_t)s.steps, (cuuint64_t)s.batch};
    const cuuint64_t strides[2] = {(cuuint64_t)st * 2, (cuuint64_t)sb * 2};
    const cuuint32_t boxes[3] = {kSlab, (cuuint32_t)box, 1};
    r = enc(map, ELEM_TMAP, 3, const_cast<void*>(p), dims, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  }
  if (r != CUDA_SUCCESS) g_fbam_last_driver_error = (int)r;
  return r == CUDA_SUCCESS ? 0 : GEMM_ERR_TENSORMAP;
}

// A launch with the cluster that suits it: sequences and channels that do not fit on the machine at once run in waves, the larger
// the cluster the more of them, each of as many rounds as its warps need for the sequence, and one for its start; a round with
// links between CTAs takes half as long again.  us forward | backward by cluster size, bf16 (batch x steps x channels):
//   8 x 1024 x 1024    1: 26 | 38     2: 25 | 33     4: 30 | 39     8: 35 | 49
//   64 x 128 x 1024    1: 25 | 35     2: 47 | 49
//   3 x 8192 x 1024    4: 63 | 102    5: 55 | 88     6: 72 | 119    8: 62 | 101
//   1 x 16384 x 2368   6: 88 | 141    7: 80 | 124    8: 100 | 174
//   1 x 30011 x 2048   4: 141 | 262   7: 135 | 215   8: 121 | 190
//   1 x 60000 x 64     4: 270 | 510   8: 145 | 281   12: 107 | 203   16: 88 | 164
template <auto KERNEL, int VEC, int WARPS, int STEPS, typename... Args>
int launch(size_t smem, const Shape& s, cudaStream_t stream, Args... args) {
  constexpr size_t cta_links = 2 * 32 * sizeof(Link<VEC>);
  static std::atomic<int> held[kMaxCtas + 1];               // clusters of each size that the machine holds at once
  const long long units = (long long)((s.dim + 32 * VEC - 1) / (32 * VEC)) * s.batch;
  if (units * (WARPS > 1 ? kMaxCtas : 1) > 0x7fffffffll) return GEMM_ERR_SHAPE;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(WARPS * 32);
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  auto clusters_of = [&](int ctas) {
    cfg.gridDim = dim3((unsigned)(units * ctas));
    cfg.dynamicSmemBytes = smem + ctas * cta_links;
    attr.val.clusterDim = {(unsigned)ctas, 1, 1};
  };
  int best = 1;
  if (WARPS > 1) {
    if (held[1] == 0) {
      if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(smem + kMaxCtas * cta_links)) != cudaSuccess ||
          cudaFuncSetAttribute(KERNEL, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
        return GEMM_ERR_LAUNCH;
      for (int ctas = kMaxCtas; ctas > 0; --ctas) {
        int n = 0;
        clusters_of(ctas);
        if (cudaOccupancyMaxActiveClusters(&n, KERNEL, &cfg) != cudaSuccess) {      // more than eight are for the device to grant
          cudaGetLastError();
          n = 0;
        }
        held[ctas] = n;
      }
      if (held[1] == 0) return GEMM_ERR_LAUNCH;
    }
    double least = 0;
    for (int ctas = 1; ctas <= kMaxCtas && (ctas == 1 || (long long)(ctas - 1) * WARPS * STEPS < s.steps); ++ctas) {
      const int n = held[ctas];
      if (n == 0) continue;
      const long long waves = (units + n - 1) / n, rounds = (s.steps + ctas * WARPS * STEPS - 1) / (ctas * WARPS * STEPS);
      const double time = (double)waves * (rounds + 1) * (ctas > 1 ? 1.5 : 1.0);
      if (ctas == 1 || time < least) {
        best = ctas;
        least = time;
      }
    }
  }
  clusters_of(best);
  return cudaLaunchKernelEx(&cfg, KERNEL, args...) == cudaSuccess ? 0 : GEMM_ERR_LAUNCH;
}

}  // namespace

// Steps from one saved state to the next: the forward's `saved` has [batch][ceil(steps / this)][dim] fp32 values (null where no
// backward follows).
extern "C" int fbam_recurrence_chunk() { return kSaved; }

// zgo: strides zb, zt, zk (sequence, step, member; channels dense); y: yb, yt; resets (bytes, or null): rb, rt.  state_in
// (batch, dim) fp32 or null for zeros.
extern "C" int fbam_recurrence_fwd(const void* zgo, long long zb, long long zt, long long zk, const float* state_in,
                                   const uint8_t* resets, long long rb, long long rt, void* y, long long yb, long long yt,
                                   float* state_out, float* saved, int batch, int steps, int dim, int* status, void* stream) {
  if (batch <= 0 || steps <= 0 || dim <= 0 || steps > 0x3fffffff) return GEMM_ERR_SHAPE;
  const Shape s{batch, steps, dim, (steps + kSaved - 1) / kSaved, zb, zt, zk, yb, yt, rb, rt};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (steps > kSaved && pieces(zgo, dim, zb, zt, zk) && pieces(y, dim, yb, yt, 8)) {
    CUtensorMap in, out;
    int e = encode(&in, zgo, s, zb, zt, zk, 1, kFwdSteps);
    if (!e) e = encode(&out, y, s, yb, yt, 0, 0, kFwdSteps);
    if (e) return e;
    return launch<recurrence_fwd_tma_kernel<kFwdSteps>, 2, kWarps, kFwdSteps>(sizeof(FwdSmem<kFwdSteps>), s, st, in, out, state_in, resets,
                                                                              state_out, saved, status, s);
  }
  const bool two = pairs(zgo, dim, zb, zt, zk) && pairs(y, dim, yb, yt, 0);
  auto go = [&](auto vec, auto warps) {
    return launch<recurrence_fwd_kernel<vec(), warps()>, vec(), warps(), kSaved>(
        sizeof(Exchange<vec(), warps()>), s, st, (const elem_t*)zgo, state_in, resets, (elem_t*)y, state_out, saved, status, s);
  };
  if (steps > kSaved) return go(Int<1>(), Int<kWarps>());
  return two ? go(Int<2>(), Int<1>()) : go(Int<1>(), Int<1>());
}

// dy: strides yb, yt; d_zgo: db, dt and dense (3, dim) steps.  d_state_out and d_state_in (batch, dim) fp32 or null.
extern "C" int fbam_recurrence_bwd(const void* zgo, long long zb, long long zt, long long zk, const uint8_t* resets,
                                   long long rb, long long rt, const float* saved, const void* dy, long long yb, long long yt,
                                   const float* d_state_out, void* d_zgo, long long db, long long dt, float* d_state_in,
                                   int batch, int steps, int dim, int* status, void* stream) {
  if (batch <= 0 || steps <= 0 || dim <= 0 || steps > 0x3fffffff) return GEMM_ERR_SHAPE;
  const Shape s{batch, steps, dim, (steps + kSaved - 1) / kSaved, zb, zt, zk, yb, yt, rb, rt};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (steps > kSaved && pieces(zgo, dim, zb, zt, zk) && pieces(dy, dim, yb, yt, 8) && pieces(d_zgo, dim, db, dt, 8) &&
      (reinterpret_cast<uintptr_t>(saved) & 15) == 0) {
    CUtensorMap in, d, out;
    int e = encode(&in, zgo, s, zb, zt, zk, 3, kSaved);
    if (!e) e = encode(&d, dy, s, yb, yt, 0, 0, kSaved);
    if (!e) e = encode(&out, d_zgo, s, db, dt, dim, 3, kSaved);
    if (e) return e;
    return launch<recurrence_bwd_tma_kernel<kSaved>, 2, kWarps, kSaved>(sizeof(BwdSmem<kSaved>), s, st, in, d, out, resets, saved,
                                                                        d_state_out, d_state_in, status, s);
  }
  const bool two = pairs(zgo, dim, zb, zt, zk) && pairs(dy, dim, yb, yt, 0) && pairs(d_zgo, dim, db, dt, 0);
  auto go = [&](auto vec, auto warps) {
    return launch<recurrence_bwd_kernel<vec(), warps()>, vec(), warps(), kSaved>(
        sizeof(Exchange<vec(), warps()>), s, st, (const elem_t*)zgo, resets, saved, (const elem_t*)dy, d_state_out, (elem_t*)d_zgo,
        d_state_in, status, s, db, dt);
  };
  if (steps > kSaved) return go(Int<1>(), Int<kWarps>());
  return two ? go(Int<2>(), Int<1>()) : go(Int<1>(), Int<1>());
}
