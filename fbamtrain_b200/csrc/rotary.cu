// Rotary positions: pairs of channels of a head turned by an angle that grows with the position of its token.
//
//   y_a = m (x_a cos φ − x_b sin φ),  y_b = m (x_b cos φ + x_a sin φ),  φ = position · θ_i
//
// for pair i of the first `rotated` channels: (i, i + rotated / 2) in the half layout, (2 i, 2 i + 1) interleaved.  What lies
// behind them, and the heads behind the first `turned`, is copied.  The gradient is the same pass with −φ.
//
// Angles.  At position 10^6 an fp32 product position · θ is off by 0.03 of a radian.  A frequency is therefore kept as a 64-bit
// fraction of a TURN a position: the product with the position modulo 2^64 is exact, and what it drops are whole turns.  Its top 32
// bits go to sin and cos as fp32, which rounds them by up to 2^-26 of a turn, and the frequency's own rounding, 2^-65 of a turn, counts
// once for every position.  sin and cos are formed once for a (token, pair) and shared by all heads of the token.
//
// The append form is the same pass of a serving step: the heads of new tokens come as (tokens, query + key + value heads, D);
// turned queries go to a tensor, turned keys and the values into the pages of a cache.
//
// Bound by memory: each value is read and written once.  A thread has one piece of a head (in the half layout 8 channels and the 8 that
// they turn with) and walks the heads of its token, four at a time: it forms its sines and cosines once, in registers, and the heads'
// loads are on their way together.  A first form kept the angles of a few tokens in shared memory and gave pieces to threads in any
// order: a block's loads waited for its angles and every piece for two divisions (27 against 20 us at 8192 tokens of 48 heads of 64).
#include <cuda_runtime.h>
#include <stdint.h>
#include "elem16.cuh"

namespace {

constexpr int kMaxPairs = 128, kThreads = 256, kUnroll = 4;

struct RotaryParams {
  unsigned long long turns[kMaxPairs];  // fraction of a turn a position, times 2^64
  const elem_t* x;
  elem_t* y;
  long long x_sb, x_st, x_sh;           // of x (B, T, H, D); the inner stride is 1
  const void* positions;                // (B, T) with strides p_sb, p_st; int32 or int64
  long long p_sb, p_st;
  long long tokens;
  int positions64;
  int T, H, D, turned, pairs;
  int inverse;
  float magnitude;
  int pieces;                           // of a head
  int heads_each;                       // heads of a thread
  // append
  elem_t* k_pages;
  elem_t* v_pages;                      // (pages, page, kv_heads, D)
  long long k_sp, k_ss, k_sh, v_sp, v_ss, v_sh;
  const int* tables;                    // (B, max_pages)
  const int* lengths;                   // (B): tokens of each sequence, the new ones among them
  const int* offsets;                   // (B + 1) first rows of the sequences' new tokens; null: one each
  long long t_sb;
  int B, max_pages, page, pages, q_heads, kv_heads;
};

__device__ __forceinline__ float2 turn(unsigned long long per_position, long long position) {
  // the top 32 bits as a signed fraction of a turn in [-1/2, 1/2): x 2^-31 is the angle in units of pi
  const int top = (int)((per_position * (unsigned long long)position) >> 32);
  float s, c;
  sincospif((float)top * 4.656612873077393e-10f, &s, &c);
  return make_float2(c, s);
}

// The sequence of row n of the new tokens and its position there; -1 for a row of no sequence, or of one that is shorter.
__device__ __forceinline__ long long append_position(const RotaryParams& p, long long n, int& b) {
  long long first, count;
  if (p.offsets == nullptr) {
    b = (int)n;
    first = n;
    count = 1;
  } else {
    int lo = 0, hi = p.B;               // the last sequence that starts at n or before it
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.offsets[mid] <= n) lo = mid; else hi = mid;
    }
    b = lo;
    first = p.offsets[lo];
    count = min((long long)p.offsets[lo + 1], p.tokens) - first;
    if (n < first || n >= first + count) return -1;
  }
  return (long long)p.lengths[b] - count + (n - first);
}

__device__ __forceinline__ void rotate8(uint4& a, uint4& b, const float2* cs, float m) {
  elem2_t* ea = reinterpret_cast<elem2_t*>(&a);
  elem2_t* eb = reinterpret_cast<elem2_t*>(&b);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 va = e22ff(ea[i]), vb = e22ff(eb[i]);
    const float2 t0 = cs[2 * i], t1 = cs[2 * i + 1];
    ea[i] = ff2e2(m * (va.x * t0.x - vb.x * t0.y), m * (va.y * t1.x - vb.y * t1.y));
    eb[i] = ff2e2(m * (vb.x * t0.x + va.x * t0.y), m * (vb.y * t1.x + va.y * t1.y));
  }
}
__device__ __forceinline__ void rotate4(uint4& a, const float2* cs, float m) {
  elem2_t* ea = reinterpret_cast<elem2_t*>(&a);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = e22ff(ea[i]);
    const float2 t = cs[i];
    ea[i] = ff2e2(m * (v.x * t.x - v.y * t.y), m * (v.y * t.x + v.x * t.y));
  }
}

// Pieces of a head: in the half layout a piece of the rotated part is two vectors, 8 channels of the first half and the 8 they
// turn with; everything else, and all of the interleaved layout, is one vector.
template <bool APPEND, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
  const long long i = (long long)blockIdx.x * kThreads + threadIdx.x, n = i / p.pieces;
  if (n >= p.tokens) return;
  const int c = (int)(i - n * p.pieces);
  const int h0 = blockIdx.y * p.heads_each, h1 = min(p.H, h0 + p.heads_each);
  const bool turns = INTERLEAVED ? c * 8 < 2 * p.pairs : c * 8 < p.pairs, two = !INTERLEAVED && turns;
  const int ch = INTERLEAVED || turns ? c * 8 : c * 8 + p.pairs;          // first channel: behind both halves where nothing turns
  long long pos, src;
  long long dst_k = -1, dst_v = -1;
  if constexpr (APPEND) {
    int b;
    pos = append_position(p, n, b);
    src = n * p.x_st;
    if (pos >= 0 && pos / p.page < p.max_pages) {
      const int which = p.tables[b * p.t_sb + pos / p.page];
      if (which >= 0 && which < p.pages) {
        dst_k = which * p.k_sp + pos % p.page * p.k_ss;
        dst_v = which * p.v_sp + pos % p.page * p.v_ss;
      }
    }
  } else {
    const long long b = n / p.T, t = n - b * p.T, at = b * p.p_sb + t * p.p_st;
    src = b * p.x_sb + t * p.x_st;
    pos = p.positions64 ? ((const long long*)p.positions)[at] : (long long)((const int*)p.positions)[at];
  }
  const elem_t* x = p.x + src + ch;
  float2 cs[8];
  if (turns && h0 < p.turned) {
#pragma unroll
    for (int j = 0; j < (INTERLEAVED ? 4 : 8); ++j) {
      cs[j] = turn(p.turns[c * (INTERLEAVED ? 4 : 8) + j], pos);
      if (p.inverse) cs[j].y = -cs[j].y;
    }
  }
  for (int h = h0; h < h1; h += kUnroll) {
    uint4 a[kUnroll], b[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (h + u < h1) {
        a[u] = __ldcs(reinterpret_cast<const uint4*>(x + (h + u) * p.x_sh));
        if (two) b[u] = __ldcs(reinterpret_cast<const uint4*>(x + (h + u) * p.x_sh + p.pairs));
      }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (h + u < h1) {
        const int head = h + u;
        if (turns && head < p.turned) {
          if constexpr (INTERLEAVED) rotate4(a[u], cs, p.magnitude); else rotate8(a[u], b[u], cs, p.magnitude);
        }
        elem_t* dst;
        if constexpr (APPEND) {
          if (head < p.q_heads) {
            dst = p.y + (n * p.q_heads + head) * p.D;
            if (pos < 0) a[u] = b[u] = make_uint4(0u, 0u, 0u, 0u);
          } else {
            if (dst_k < 0) continue;
            dst = head < p.q_heads + p.kv_heads ? p.k_pages + dst_k + (head - p.q_heads) * p.k_sh
                                                : p.v_pages + dst_v + (head - p.q_heads - p.kv_heads) * p.v_sh;
          }
        } else {
          dst = p.y + (n * p.H + head) * p.D;
        }
        *reinterpret_cast<uint4*>(dst + ch) = a[u];
        if (two) *reinterpret_cast<uint4*>(dst + ch + p.pairs) = b[u];
      }
  }
}

// Any widths, strides and alignment: a thread per channel, or pair of channels.
template <bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) rotary_any_kernel(const __grid_constant__ RotaryParams p) {
  const int per_head = p.D - p.pairs;
  const long long all = p.tokens * p.H * per_head;
  for (long long i = (long long)blockIdx.x * kThreads + threadIdx.x; i < all; i += (long long)gridDim.x * kThreads) {
    const int c = (int)(i % per_head);
    const long long row = i / per_head;
    const int h = (int)(row % p.H);
    const long long n = row / p.H, b = n / p.T, t = n % p.T;
    const elem_t* src = p.x + b * p.x_sb + t * p.x_st + h * p.x_sh;
    elem_t* dst = p.y + row * p.D;
    if (c >= p.pairs) {
      dst[c + p.pairs] = src[c + p.pairs];
      continue;
    }
    const int ca = INTERLEAVED ? 2 * c : c, cb = INTERLEAVED ? 2 * c + 1 : c + p.pairs;
    if (h >= p.turned) {
      dst[ca] = src[ca];
      dst[cb] = src[cb];
      continue;
    }
    const long long at = b * p.p_sb + t * p.p_st;
    float2 v = turn(p.turns[c], p.positions64 ? ((const long long*)p.positions)[at] : (long long)((const int*)p.positions)[at]);
    if (p.inverse) v.y = -v.y;
    const float xa = e2f(src[ca]), xb = e2f(src[cb]);
    dst[ca] = f2e(p.magnitude * (xa * v.x - xb * v.y));
    dst[cb] = f2e(p.magnitude * (xb * v.x + xa * v.y));
  }
}

// Eight heads a thread, or fewer where there are so few tokens that the machine would not be full.
template <bool APPEND>
int launch(RotaryParams& p, bool interleaved, cudaStream_t s) {
  p.pieces = interleaved ? p.D / 8 : (p.D - p.pairs) / 8;
  const long long threads = p.tokens * p.pieces, blocks = (threads + kThreads - 1) / kThreads;
  p.heads_each = 8;
  while (p.heads_each > 1 && threads * ((p.H + p.heads_each - 1) / p.heads_each) < 148 * 1024) p.heads_each >>= 1;
  const int parts = (p.H + p.heads_each - 1) / p.heads_each;
  if (blocks > 0x7fffffffll || parts > 65535) return 1;
  const dim3 grid((unsigned)blocks, parts);
  if (interleaved)
    rotary_kernel<APPEND, true><<<grid, kThreads, 0, s>>>(p);
  else
    rotary_kernel<APPEND, false><<<grid, kThreads, 0, s>>>(p);
  return cudaGetLastError() == cudaSuccess ? 0 : 5;
}

}  // namespace

extern "C" {

// x (B, T, H, D) with strides, y contiguous; positions (B, T) with strides.  The first `turned` heads are turned in their first
// 2 · pairs channels.
int fbam_rotary(const void* x, long long sb, long long st, long long sh, void* y, const void* positions, int positions64,
                long long p_sb, long long p_st, const unsigned long long* turns, int pairs, float magnitude, int interleaved,
                int inverse, long long B, long long T, int H, int D, int turned, void* stream) {
  if (pairs < 0 || pairs > kMaxPairs || 2 * pairs > D || turned < 0 || turned > H || B < 1 || T < 1 || T > 0x7fffffffll || H < 1) return 1;
  RotaryParams p = {};
  for (int i = 0; i < pairs; ++i) p.turns[i] = turns[i];
  p.x = (const elem_t*)x;
  p.y = (elem_t*)y;
  p.x_sb = sb; p.x_st = st; p.x_sh = sh;
  p.positions = positions;
  p.positions64 = positions64;
  p.p_sb = p_sb; p.p_st = p_st;
  p.tokens = B * T;
  p.T = (int)T; p.H = H; p.D = D; p.turned = turned; p.pairs = pairs;
  p.inverse = inverse;
  p.magnitude = magnitude;
  cudaStream_t s = (cudaStream_t)stream;
  // whole 16-byte pieces everywhere; interleaved pairs come four to a piece, halves eight
  const bool pieces = D % 8 == 0 && pairs % (interleaved ? 4 : 8) == 0 && !(((uintptr_t)x | (uintptr_t)y) & 15) && sb % 8 == 0 &&
                      st % 8 == 0 && sh % 8 == 0;
  if (pieces) return launch<false>(p, interleaved != 0, s);
  const long long all = p.tokens * H * (D - pairs);
  const long long blocks = (all + kThreads - 1) / kThreads;
  const unsigned grid = (unsigned)(blocks < 148 * 64 ? blocks : 148 * 64);
  if (interleaved)
    rotary_any_kernel<true><<<grid, kThreads, 0, s>>>(p);
  else
    rotary_any_kernel<false><<<grid, kThreads, 0, s>>>(p);
  return cudaGetLastError() == cudaSuccess ? 0 : 5;
}

// qkv (tokens, q_heads + 2 kv_heads, D) with strides st, sh; q (tokens, q_heads, D) contiguous; pages with strides of pages,
// slots and heads.  D, and the strides, in multiples of 8.
int fbam_cache_append(const void* qkv, long long st, long long sh, void* q, void* k_pages, long long k_sp, long long k_ss, long long k_sh,
                      void* v_pages, long long v_sp, long long v_ss, long long v_sh, const int* tables, long long t_sb,
                      const int* lengths, const int* offsets, const unsigned long long* turns, int pairs, float magnitude,
                      int interleaved, long long tokens, int B, int max_pages, int page, int pages, int q_heads, int kv_heads, int D,
                      void* stream) {
  if (pairs < 0 || pairs > kMaxPairs || 2 * pairs > D || tokens < 1 || B < 1 || page < 1 || max_pages < 0) return 1;
  if (D % 8 || pairs % (interleaved ? 4 : 8)) return 1;
  if ((((uintptr_t)qkv | (uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages) & 15) || st % 8 || sh % 8 || k_sp % 8 || k_ss % 8 ||
      k_sh % 8 || v_sp % 8 || v_ss % 8 || v_sh % 8)
    return 2;
  RotaryParams p = {};
  for (int i = 0; i < pairs; ++i) p.turns[i] = turns[i];
  p.x = (const elem_t*)qkv;
  p.y = (elem_t*)q;
  p.x_st = st; p.x_sh = sh;
  p.tokens = tokens;
  p.H = q_heads + 2 * kv_heads; p.D = D; p.turned = q_heads + kv_heads; p.pairs = pairs;
  p.magnitude = magnitude;
  p.k_pages = (elem_t*)k_pages; p.v_pages = (elem_t*)v_pages;
  p.k_sp = k_sp; p.k_ss = k_ss; p.k_sh = k_sh; p.v_sp = v_sp; p.v_ss = v_ss; p.v_sh = v_sh;
  p.tables = tables; p.t_sb = t_sb; p.lengths = lengths; p.offsets = offsets;
  p.B = B; p.max_pages = max_pages; p.page = page; p.pages = pages; p.q_heads = q_heads; p.kv_heads = kv_heads;
  return launch<true>(p, interleaved != 0, (cudaStream_t)stream);
}

}  // extern "C"
