// Rotary positions: pairs of channels of a head turned by an angle that grows with the position of its token.
//
//   y_a = m (x_a cos φ − x_b sin φ),  y_b = m (x_b cos φ + x_a sin φ),  φ = position · θ_i
//
// for pair i of the first `rotated` channels: (i, i + rotated / 2) in the half layout, (2 i, 2 i + 1) interleaved.  What lies
// behind them, and the heads behind the first `turned`, is copied.  The gradient is the same pass with −φ.
//
// Angles.  At position 10^6 an fp32 product position · θ is off by 0.03 of a radian.  A frequency is therefore kept as a 64-bit
// fraction of a TURN a position: the product with the position modulo 2^64 is exact, what it drops are whole turns, and its top 32
// bits are the angle to 2^-32 of a turn.  sin and cos are formed once for a (token, pair) and shared by all heads of the token.
//
// The append form is the same pass of a serving step: the heads of new tokens come as (tokens, query + key + value heads, D);
// turned queries go to a tensor, turned keys and the values into the pages of a cache.
//
// Bound by memory: each value is read and written once.  A thread block takes a few tokens (some 2048 16-byte pieces), forms
// their angles in shared memory and walks the pieces, four loads in flight a thread.
#include <cuda_runtime.h>
#include <stdint.h>
#include "elem16.cuh"

namespace {

constexpr int kMaxPairs = 128, kThreads = 256, kMaxTokens = 32, kUnroll = 4;

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
  int per_block;                        // tokens of a thread block
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
    count = p.offsets[lo + 1] - first;
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
  extern __shared__ float2 cs[];        // (tokens, pairs)
  __shared__ long long src_at[kMaxTokens];
  __shared__ long long dst_k[kMaxTokens], dst_v[kMaxTokens];
  __shared__ long long pos[kMaxTokens];
  const long long n0 = (long long)blockIdx.x * p.per_block;
  const int tokens = (int)min((long long)p.per_block, p.tokens - n0);
  if (threadIdx.x < tokens) {
    const long long n = n0 + threadIdx.x;
    if constexpr (APPEND) {
      int b;
      const long long at = append_position(p, n, b);
      pos[threadIdx.x] = at;
      src_at[threadIdx.x] = n * p.x_st;
      long long dk = -1, dv = -1;
      if (at >= 0 && at / p.page < p.max_pages) {
        const int which = p.tables[b * p.t_sb + at / p.page];
        if (which >= 0 && which < p.pages) {
          dk = which * p.k_sp + at % p.page * p.k_ss;
          dv = which * p.v_sp + at % p.page * p.v_ss;
        }
      }
      dst_k[threadIdx.x] = dk;
      dst_v[threadIdx.x] = dv;
    } else {
      const long long b = n / p.T, t = n % p.T;
      src_at[threadIdx.x] = b * p.x_sb + t * p.x_st;
      const long long at = b * p.p_sb + t * p.p_st;
      pos[threadIdx.x] = p.positions64 ? ((const long long*)p.positions)[at] : (long long)((const int*)p.positions)[at];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < tokens * p.pairs; i += kThreads) {
    const int t = i / p.pairs;
    float2 v = turn(p.turns[i - t * p.pairs], pos[t]);
    if (p.inverse) v.y = -v.y;
    cs[i] = v;
  }
  __syncthreads();
  const int half = p.pairs >> 3;                                             // two-vector pieces (half layout)
  const int per_turned = INTERLEAVED ? p.D / 8 : p.D / 8 - half, per_plain = p.D / 8;
  const int in_turned = p.turned * per_turned, per_token = in_turned + (p.H - p.turned) * per_plain;
  const int all = tokens * per_token;
  for (int base = threadIdx.x; base < all; base += kThreads * kUnroll) {
    uint4 a[kUnroll], b[kUnroll];
    elem_t* dst[kUnroll];
    const float2* angle[kUnroll];
    int kind[kUnroll];                  // 0: nothing, 1: copy, 2: interleaved vector, 3: two vectors, 4: zeros
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int i = base + u * kThreads;
      kind[u] = 0;
      if (i < all) {
        const int t = i / per_token, r = i - t * per_token;
        int h, c;
        if (r < in_turned) {
          h = r / per_turned;
          c = r - h * per_turned;
        } else {
          h = (r - in_turned) / per_plain;
          c = r - in_turned - h * per_plain;
          h += p.turned;
        }
        const bool turned = h < p.turned;
        kind[u] = 1;
        int ch = c * 8;                 // first channel
        if (turned) {
          if (INTERLEAVED) {
            if (ch < 2 * p.pairs) { kind[u] = 2; angle[u] = cs + t * p.pairs + c * 4; }
          } else if (c < half) {
            kind[u] = 3;
            angle[u] = cs + t * p.pairs + c * 8;
          } else {
            ch += p.pairs;              // behind both halves
          }
        }
        if constexpr (APPEND) {
          const bool there = pos[t] >= 0;
          if (h < p.q_heads) {
            dst[u] = p.y + ((n0 + t) * p.q_heads + h) * p.D + ch;
            if (!there) kind[u] = kind[u] == 3 ? 5 : 4;
          } else if (h < p.q_heads + p.kv_heads) {
            dst[u] = p.k_pages + dst_k[t] + (h - p.q_heads) * p.k_sh + ch;
            if (dst_k[t] < 0) kind[u] = 0;
          } else {
            dst[u] = p.v_pages + dst_v[t] + (h - p.q_heads - p.kv_heads) * p.v_sh + ch;
            if (dst_k[t] < 0) kind[u] = 0;
          }
        } else {
          dst[u] = p.y + ((n0 + t) * p.H + h) * p.D + ch;
        }
        const elem_t* src = p.x + src_at[t] + h * p.x_sh + ch;
        if (kind[u] != 0) a[u] = __ldcs(reinterpret_cast<const uint4*>(src));
        if (kind[u] == 3) b[u] = __ldcs(reinterpret_cast<const uint4*>(src + p.pairs));
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (kind[u] == 0) continue;
      if (kind[u] == 2) rotate4(a[u], angle[u], p.magnitude);
      if (kind[u] == 3) rotate8(a[u], b[u], angle[u], p.magnitude);
      if (kind[u] >= 4) a[u] = b[u] = make_uint4(0u, 0u, 0u, 0u);
      *reinterpret_cast<uint4*>(dst[u]) = a[u];
      if (kind[u] == 3 || kind[u] == 5) *reinterpret_cast<uint4*>(dst[u] + p.pairs) = b[u];
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

// Pieces of a token and from them the tokens of a block: some 2048 pieces, but no fewer blocks than fill the machine twice.
template <bool APPEND>
int launch(RotaryParams& p, bool interleaved, cudaStream_t s) {
  const long long pieces = (long long)p.H * (p.D / 8);
  long long per = 2048 / (pieces < 1 ? 1 : pieces);
  const long long spread = p.tokens / 296;
  per = per < spread ? per : spread;
  p.per_block = (int)(per < 1 ? 1 : per > kMaxTokens ? kMaxTokens : per);
  const long long blocks = (p.tokens + p.per_block - 1) / p.per_block;
  if (blocks > 0x7fffffffll || pieces * p.per_block > 0x7fffffffll) return 1;
  const size_t smem = (size_t)p.per_block * (p.pairs < 1 ? 1 : p.pairs) * sizeof(float2);
  if (interleaved)
    rotary_kernel<APPEND, true><<<(unsigned)blocks, kThreads, smem, s>>>(p);
  else
    rotary_kernel<APPEND, false><<<(unsigned)blocks, kThreads, smem, s>>>(p);
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
