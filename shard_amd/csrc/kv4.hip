// Paged KV cache held in 4 bits: append (with RoPE), read back, attention.
//
// Format.  A page holds 64 tokens of every kv head, 68 * D bytes a head
// (D = head_dim 64 or 128): an element is an E2M1 code, 32 channels of a token
// share an E5M2 scale (its byte is the upper half of the fp16 number of the
// same value).  value = e2m1(code) * scale has at most 5 significant bits and
// a magnitude in {0} or 2^-17 .. 61440, so it is exact in fp16: the attention
// multiplies fp16 operands and rounds nothing of the cache.
// scale = the smallest E5M2 number >= amax / 6.5 (6.5 rather than 6: magnitudes
// in (6, 6.5] scales saturate by at most half a scale, and the finer scale
// pays elsewhere: relative rms error of Gaussian blocks 10.4% against 11.2%),
// from 2^-16 to 10240.  Codes round to the nearest, ties to the even code;
// magnitudes above 6 scales and infinities saturate, NaN is stored as 0.
//
// Within a page a head's bytes are laid out as the attention's MFMA operands
// (16x16x32, fp16) take them, so that a wave reads them as contiguous 16-byte
// lanes and nothing is transposed on the way:
//   K codes   [0, 32 D): lane (kq, r) of token group sub = t / 16, r = t % 16,
//             holds the D / 4 channels kq * D/4 .. of its token: 16 (D = 128) or
//             8 bytes (D = 64, two token groups side by side), even channel low.
//   K scales  [32 D, 34 D): [block][r][sub].
//   V codes   [34 D, 66 D): a 32-bit word holds one channel of 8 tokens, the
//             two runs of four that a lane's score registers hold: token
//             32 s + 16 (e / 4) + 4 kq + e % 4 in nibble e; words
//             [s][n / 4][kq][channel % 16][n % 4], n = channel / 16.
//   V scales  [66 D, 68 D): [kq][s][block][e].
//
// Batch: sequence b's new tokens are rows cu[b] .. cu[b + 1] - 1 (or row b
// alone) and the last of its seq_lens[b] tokens; token t of it lives in page
// block_table[b][t / 64], slot t % 64.  Everything read from device memory is
// checked where it is used: rows and lengths are clamped, positions outside
// the table or the phases and page numbers outside the cache are left out.
#include <math.h>
#include <stdio.h>

#include <algorithm>

#include "common.h"

namespace shard {
namespace {

constexpr int kPage = 64;

typedef __bf16 bf16_t;

struct Seq {
  int row0, n;      // its rows of q, k, v
  int len;          // tokens, as given
  int cap;          // tokens its block table can hold
};

__device__ __forceinline__ Seq seq_of(const shard_kv4_args& a, int b, int len) {
  Seq s;
  int c0 = b, c1 = b + 1;
  if (a.cu_seqlens) {
    c0 = a.cu_seqlens[b];
    c1 = a.cu_seqlens[b + 1];
  }
  c0 = min(max(c0, 0), a.n_tokens);
  c1 = min(max(c1, c0), a.n_tokens);
  s.row0 = c0;
  s.n = c1 - c0;
  s.len = max(len, 0);
  s.cap = a.table_width * kPage;
  return s;
}
__device__ __forceinline__ Seq seq_of(const shard_kv4_args& a, int b) { return seq_of(a, b, a.seq_lens[b]); }

// The page that holds token t of sequence b (t < cap), -1 if the table names none.
__device__ __forceinline__ int page_of(const shard_kv4_args& a, int b, int t) {
  const int p = a.block_table[(int64_t)b * a.table_stride + (t >> 6)];
  return (unsigned)p < (unsigned)a.n_pages ? p : -1;
}

template <int D>
__device__ __forceinline__ uint8_t* head_of(const shard_kv4_args& a, int page, int g) {
  return a.cache + (int64_t)page * a.page_stride + (int64_t)g * (68 * D);
}

// Byte offsets within a head's part of a page.
template <int D>
__device__ __forceinline__ int k_code_at(int slot, int kq) {  // of D / 8 bytes
  const int sub = slot >> 4, r = slot & 15;
  return D == 128 ? (sub * 64 + kq * 16 + r) * 16 : ((sub >> 1) * 64 + kq * 16 + r) * 16 + (sub & 1) * 8;
}
template <int D>
__device__ __forceinline__ int k_scale_at(int slot, int blk) {
  return 32 * D + (blk * 16 + (slot & 15)) * 4 + (slot >> 4);
}
template <int D>
__device__ __forceinline__ int v_word_at(int s, int kq, int ch) {  // of 4 bytes
  const int n = ch >> 4;
  return 34 * D + (((s * (D / 64) + (n >> 2)) * 64 + kq * 16 + (ch & 15)) * 4 + (n & 3)) * 4;
}
template <int D>
__device__ __forceinline__ int v_scale_at(int slot, int blk) {
  const int s = slot >> 5, u = slot & 31, e = ((u >> 4) << 2) | (u & 3), kq = (u >> 2) & 3;
  return 66 * D + ((kq * 2 + s) * (D / 32) + blk) * 8 + e;
}

__device__ __forceinline__ float e5m2(unsigned byte) { return h2f((uint16_t)(byte << 8)); }

// The scale byte of a block whose largest magnitude is `amax` (not NaN).
__device__ __forceinline__ unsigned scale_byte(float amax) {
  const unsigned c = f2h(amax * (1.0f / 6.5f)) >> 8;  // within one of the answer, from below
  unsigned b = c > 1u ? min(c, 113u) : 1u;
  b += 6.5f * e5m2(b) < amax ? 1u : 0u;               // 6.5 scale is exact: 7 significant bits
  b += 6.5f * e5m2(b) < amax ? 1u : 0u;
  return min(b, 113u);
}

// E2M1 code of x at scale s: nearest, ties to the even code.  s times a border
// has at most 6 significant bits, so every comparison is exact.
__device__ __forceinline__ unsigned code4(float x, float s) {
  const float a = fabsf(x);
  const unsigned b2 = a >= 1.75f * s;
  const unsigned b1 = a >= (b2 ? 3.5f : 0.75f) * s;
  const float t = b2 ? (b1 ? 5.0f : 2.5f) : (b1 ? 1.25f : 0.25f);
  const unsigned b0 = a > t * s;
  return (x < 0.f ? 8u : 0u) | b2 << 2 | b1 << 1 | b0;
}

// d in 32 bits, rounded to odd where it does not fit: compares with every
// number of fewer bits as d does.
__device__ __forceinline__ float to_odd(double d) {
  const float f = (float)d;
  uint32_t u = __float_as_uint(f);
  const double back = (double)f;
  if (back != d) {
    if (fabs(back) > fabs(d)) u -= 1u;
    u |= 1u;
  }
  return __uint_as_float(u);
}

__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, dpp_mov<kDppXor1>(v));
  return fmaxf(v, dpp_mov<kDppXor2>(v));
}

// 8 elements of a row at p (16-byte aligned) as floats.
template <class T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  typedef T vec8 __attribute__((ext_vector_type(8)));
  const vec8 v = *(const vec8*)p;
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  typedef T vec8 __attribute__((ext_vector_type(8)));
  vec8 v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (T)x[i];
  *(vec8*)p = v;
}

// --------------------------------------------------------------------------
// Append: rotation of q and k, 4-bit rounding of k and v, scatter into pages.
//
// A workgroup owns 32 aligned tokens of a sequence for one kv head (blockIdx.y
// < G): no other workgroup writes a word of its V codes, so words shared with
// earlier tokens are read, merged and written without atomics.  Further y
// rotate kHeadsQ query heads for the same tokens.
// k is rotated in 64 bits, (c, s) being fp32 inputs: codes next to a border
// come out as the formula's.  The products are exact there and the sum rounds
// once, so nothing depends on contraction.
// Measured (32 query heads on 8, head_dim 128, fp16): four prompts of 8,192
// tokens 179 us, 4.0 TB/s of the 724 MB it reads and writes (a large copy: 4.75),
// the vector pipe half busy with K's 64-bit rotation and the roundings; one token
// 6 us.  That is not its chain of memory accesses (arguments, length, table, page,
// store): the read has the same and takes 3.2.  Most likely it is the serial work of
// few lanes: 8 threads rotate, round and code 16 elements of K each, and 8 of a
// query workgroup take 4 heads one after the other.
// --------------------------------------------------------------------------
constexpr int kHeadsQ = 4;

template <class T, int D>
__global__ __launch_bounds__(256, 4)
void k_kv4_append(const shard_kv4_args a) {
  constexpr int PB = D / 64;  // pairs of 32-channel blocks: (pb, pb + PB)
  __shared__ __align__(4) uint8_t codes[32][D + 4];
  const int tid = threadIdx.x, b = blockIdx.z;
  const Seq s = seq_of(a, b);
  if (s.n == 0) return;
  const int start = s.len - s.n;                    // position of the first new token
  const bool is_q = blockIdx.y >= (unsigned)a.n_kv_heads;
  const int g0 = (is_q ? start : max(start, 0)) >> 5, g1 = (s.len - 1) >> 5;
  const int lq = tid & 3, pb = PB == 2 ? (tid >> 2) & 1 : 0;
  const int tok = PB == 2 ? tid >> 3 : tid >> 2;    // of the 32 (D = 64: threads 0..127)
  const int ch = pb * 32 + lq * 8;
  for (int grp = g0 + blockIdx.x; grp <= g1; grp += gridDim.x) {
    const int t0 = grp * 32;
    const int pos = t0 + tok, i = pos - start;
    const bool mine = tok < 32 && i >= 0 && i < s.n;
    const bool there = mine && pos >= 0 && pos < s.cap && pos < a.n_phases;
    float c[8], sn[8];
    if (there) {
      const float4* ph = (const float4*)(a.phases + ((int64_t)pos * (D / 2) + ch) * 2);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4 f = ph[j];
        c[2 * j] = f.x; sn[2 * j] = f.y; c[2 * j + 1] = f.z; sn[2 * j + 1] = f.w;
      }
    }
    if (is_q) {                                     // query heads; zeros where a token has no place
      if (!mine) continue;
      const int h0 = (blockIdx.y - a.n_kv_heads) * kHeadsQ, h1 = min(h0 + kHeadsQ, a.n_q_heads);
      for (int h = h0; h < h1; ++h) {
        float lo[8] = {}, hi[8] = {};
        if (there) {
          const T* q = (const T*)a.q + (int64_t)(s.row0 + i) * a.q_stride + (int64_t)h * a.q_head_stride + ch;
          float x[8], y[8];
          load8(q, x);
          load8(q + D / 2, y);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            lo[j] = x[j] * c[j] - y[j] * sn[j];
            hi[j] = y[j] * c[j] + x[j] * sn[j];
          }
        }
        T* o = (T*)a.q_out + ((int64_t)(s.row0 + i) * a.n_q_heads + h) * D + ch;
        store8(o, lo);
        store8(o + D / 2, hi);
      }
      continue;
    }
    if (t0 >= s.cap) return;                        // cap is a multiple of 32
    const int g = blockIdx.y;
    const int page = page_of(a, b, t0);
    if (page < 0) continue;
    uint8_t* base = head_of<D>(a, page, g);
    const int slot0 = t0 & 63, slot = slot0 + tok;
    const auto is_new = [&](int t) { return (unsigned)(t0 + t - start) < (unsigned)s.n && t0 + t < a.n_phases; };
    // all that the group reads, before anything waits: k, v, and the words of V
    // codes that earlier tokens share
    constexpr int VU = D / 64;                        // 8-channel pieces of V a thread, words a thread
    typedef T vec8 __attribute__((ext_vector_type(8)));
    vec8 kx{}, ky{}, vx[VU];
    uint32_t old[VU], keep[VU];
    if (there) {
      const T* k = (const T*)a.k + (int64_t)(s.row0 + i) * a.k_stride + (int64_t)g * a.k_head_stride + ch;
      kx = *(const vec8*)k;
      ky = *(const vec8*)(k + D / 2);
    }
#pragma unroll
    for (int n = 0; n < VU; ++n) {
      const int u = tid + 256 * n, vt = u / (D / 8), vc = (u % (D / 8)) * 8;
      if (is_new(vt))
        vx[n] = *(const vec8*)((const T*)a.v + (int64_t)(s.row0 + t0 + vt - start) * a.v_stride + (int64_t)g * a.v_head_stride + vc);
    }
#pragma unroll
    for (int n = 0; n < VU; ++n) {
      const int u = tid + 256 * n, kq = u / D, vc = u % D;
      keep[n] = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (!is_new(16 * (e >> 2) + 4 * kq + (e & 3))) keep[n] |= 15u << (4 * e);
      old[n] = 0;
      if (keep[n] != 0 && keep[n] != ~0u) old[n] = *(const uint32_t*)(base + v_word_at<D>(slot0 >> 5, kq, vc));
    }
    if (there) {
      float r[2][8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const double x = (double)(float)kx[j], y = (double)(float)ky[j];
        const double dl = x * c[j] - y * sn[j];
        const double dh = y * c[j] + x * sn[j];
        r[0][j] = dl == dl ? to_odd(dl) : 0.f;
        r[1][j] = dh == dh ? to_odd(dh) : 0.f;
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(r[half][j]));
        const unsigned sb = scale_byte(quad_max(m));
        const float sc = e5m2(sb);
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) w |= code4(r[half][j], sc) << (4 * j);
        const int cc = half * (D / 2) + ch;
        *(uint32_t*)(base + k_code_at<D>(slot, cc / (D / 4)) + (cc % (D / 4)) / 2) = w;
        if (lq == 0) base[k_scale_at<D>(slot, cc / 32)] = (uint8_t)sb;
      }
    }
    // V: codes into LDS by token, words of 8 tokens out
#pragma unroll
    for (int n = 0; n < VU; ++n) {  // quads of lanes share a block of 32 channels
      const int u = tid + 256 * n, vt = u / (D / 8), vc = (u % (D / 8)) * 8;
      if (is_new(vt)) {
        float x[8], m = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[j] = (float)vx[n][j];
          x[j] = x[j] == x[j] ? x[j] : 0.f;
          m = fmaxf(m, fabsf(x[j]));
        }
        const unsigned sb = scale_byte(quad_max(m));
        const float sc = e5m2(sb);
        uint32_t w[2] = {};
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j >> 2] |= code4(x[j], sc) << (8 * (j & 3));
        *(uint32_t*)&codes[vt][vc] = w[0];
        *(uint32_t*)&codes[vt][vc + 4] = w[1];
        if ((vc & 31) == 0) base[v_scale_at<D>(slot0 + vt, vc / 32)] = (uint8_t)sb;
      }
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < VU; ++n) {
      const int u = tid + 256 * n, kq = u / D, vc = u % D;
      if (keep[n] == ~0u) continue;
      uint32_t w = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) w |= (codes[16 * (e >> 2) + 4 * kq + (e & 3)][vc] & 15u) << (4 * e);  // whatever lies in the others
      *(uint32_t*)(base + v_word_at<D>(slot0 >> 5, kq, vc)) = (old[n] & keep[n]) | (w & ~keep[n]);
    }
    __syncthreads();
  }
}

// --------------------------------------------------------------------------
// Read: the K and V that the cache holds for the new tokens' positions.  V goes
// through LDS, by channel in, by token out.  32,768 tokens of 8 heads of 128: 35
// us, 4.9 TB/s of its 170 MB.
// --------------------------------------------------------------------------
__device__ __forceinline__ half2v fp4_pair(uint32_t w, int byte) {
  switch (byte) {
    case 0: return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 0);
    case 1: return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 1);
    case 2: return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 2);
    default: return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 3);
  }
}

template <class T, int D>
__global__ __launch_bounds__(256)
void k_kv4_read(const shard_kv4_args a) {
  __shared__ half_t rows[32][D + 2];
  const int tid = threadIdx.x, b = blockIdx.z, g = blockIdx.y;
  const Seq s = seq_of(a, b);
  if (s.n == 0) return;
  // rows that no token of the cache stands for (positions before 0 or past the table) are zero
  const int start = s.len - s.n;
  const int g0 = start >> 5, g1 = (s.len - 1) >> 5;  // floor, also below 0
  for (int grp = g0 + blockIdx.x; grp <= g1; grp += gridDim.x) {
    const int t0 = grp * 32;
    const int page = t0 >= 0 && t0 < s.cap ? page_of(a, b, t0) : -1;
    const uint8_t* base = page >= 0 ? head_of<D>(a, page, g) : nullptr;
    constexpr int U = D / 64;  // 8-channel pieces a thread, of K and of V; words of V codes
    uint32_t kw[U] = {}, vw[U] = {};
    uint8_t ksc[U] = {}, vsc[U] = {};
    if (base) {
#pragma unroll
      for (int n = 0; n < U; ++n) {
        const int u = tid + 256 * n, slot = (t0 & 63) + u / (D / 8), ch = (u % (D / 8)) * 8;
        kw[n] = *(const uint32_t*)(base + k_code_at<D>(slot, ch / (D / 4)) + (ch % (D / 4)) / 2);
        ksc[n] = base[k_scale_at<D>(slot, ch / 32)];
        vsc[n] = base[v_scale_at<D>(slot, ch / 32)];
        vw[n] = *(const uint32_t*)(base + v_word_at<D>((t0 & 63) >> 5, u / D, u % D));
      }
    }
#pragma unroll
    for (int n = 0; n < U; ++n) {
      const int u = tid + 256 * n, kq = u / D, vc = u % D;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const half2v p = fp4_pair(vw[n], j);
        const int vt = 16 * (j >> 1) + 4 * kq + 2 * (j & 1);
        rows[vt][vc] = p[0];
        rows[vt + 1][vc] = p[1];
      }
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < U; ++n) {
      const int u = tid + 256 * n, t = u / (D / 8), ch = (u % (D / 8)) * 8, i = t0 + t - start;
      if (i < 0 || i >= s.n) continue;
      const float ks = base ? e5m2(ksc[n]) : 0.f, vs = base ? e5m2(vsc[n]) : 0.f;
      float x[8], y[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const half2v p = fp4_pair(kw[n], j);
        x[2 * j] = (float)p[0] * ks;
        x[2 * j + 1] = (float)p[1] * ks;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = (float)rows[t][ch + j] * vs;
      const int64_t at = ((int64_t)(s.row0 + i) * a.n_kv_heads + g) * D + ch;
      store8((T*)a.k_out + at, x);
      store8((T*)a.v_out + at, y);
    }
    __syncthreads();
  }
}

// --------------------------------------------------------------------------
// Attention.
//
// Rows of (sequence, kv head): r = i * group + h for new token i and query
// head h of the group; row r sees the keys up to its own position.
// Scores are taken transposed, S^T = K Q^T (16 tokens x 16 rows an MFMA), so
// that a lane's score registers hold four tokens of ONE row, and after the
// softmax they are the right operand of O^T = V^T P^T as they stand.
// A row's weights are 2^(score - m), m at most kLead below the largest score so
// far and moved only where a weight would exceed 2^kMost: most pages rescale no
// sums, and the largest weight lies between 2^kLead and 2^kMost, fp16's upper end.
// P is rounded to fp16: 2^-11 of each weight down to 2^-(14 + kLead) of a row's
// largest, 2^-(25 + kLead) of that largest below, so that what many keys far
// below one key add up to is kept; the sums are fp32.  A longer lead moves m more
// often: a prompt of 8,192 tokens 570 us with m moved at 8 above it and no lead,
// 574 with leads of 7 and 11, 575 with 13; a chunk of 512 over 16K 163, 163.5, 165.7.
// The cache's values are exact.  bf16 queries are scaled by a power of two a row
// (their largest below 2) and are then exact in fp16 down to 2^-17 of that largest
// (below it they lose bits, 2^-26 of the largest at most); the power goes back
// in through the softmax scale.
// --------------------------------------------------------------------------
constexpr float kMostScale = 2e38f;  // times log2(e) it is finite
constexpr float kLead = 11.f, kMost = 15.f;
constexpr float kLeast = 1.17549435e-38f;  // a factor of scores is never 0: -inf stays what it is

// The reference that scores up to mx move a row's to; rounded by itself, as the
// differences below are.
__device__ __forceinline__ float reference(float m, float mx) {
#pragma clang fp contract(off)
  return fmaxf(m, mx - kLead);
}
// A weight's exponent, x sc - ref, rounded twice: the product as in the largest,
// so that none is above it.  Weights take it in one step, fma(x, sc, -ref), which
// is closer but leaves what the largest itself was rounded by: nothing that
// matters up to a reference of kFar, and beyond it as much as fp16 cannot hold.
constexpr float kFar = 4194304.f;   // 2^22: below it that is 2^-3 at most
__device__ __forceinline__ float far_exponent(float x, float sc, float ref) {
#pragma clang fp contract(off)
  const float s = x * sc;
  const float d = s - ref;
  return d > kMost ? kMost : d;      // NaN stays
}

struct AttnWork {
  float* m;      // [row][split], rows (token, query head)
  float* l;
  float* acc;    // [row][split][D]
  int n_splits, split_shift;    // a power of two
  int group, group_shift;       // query heads of a kv head; -1: no power of two
  int row_tiles;                // workgroups along a sequence's rows
  float sorted;                 // 16 / longest length where longer sequences go first, or 0
};

// Tiles (pages) a split of a sequence of `tiles` takes: at least kMinTiles, one
// for each wave of the workgroup.
constexpr int kMinTiles = 4;
__device__ __forceinline__ int tiles_per_split(const AttnWork& w, int tiles) {
  return max(kMinTiles, (tiles + w.n_splits - 1) >> w.split_shift);
}

// Token of a sequence's row, and its head within the group.  (An integer division
// costs a launch's first instructions about 150 cycles each.)
__device__ __forceinline__ int token_of(const AttnWork& w, int r) {
  return w.group_shift >= 0 ? r >> w.group_shift : r / w.group;
}

// The z-th sequence by length, longest first, of z's 64 (lengths in 16 classes,
// equal ones in their order), and its length.
__device__ __forceinline__ int by_length(const shard_kv4_args& a, const AttnWork& w, int z, int lane, int& len) {
  const int z0 = z & ~63, mine = z0 + lane < a.batch ? a.seq_lens[z0 + lane] : 0;
  const int of = z0 + lane < a.batch ? (int)fminf((float)max(mine, 0) * w.sorted, 15.f) : -1;
  int k = z & 63, c = 15;
  uint64_t in = __builtin_amdgcn_ballot_w64(of == c);
  for (int n; c > 0 && k >= (n = __builtin_popcountll(in)); in = __builtin_amdgcn_ballot_w64(of == --c)) k -= n;
  const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0));
  const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(of == c && before == k));
  len = __builtin_amdgcn_readlane(mine, at);
  return z0 + at;
}

// A split past a sequence's end: the merge reads that it has nothing.  Rows tid,
// tid + 256, ... of every 256 row_tiles.
__device__ __forceinline__ void nothing(const shard_kv4_args& a, const AttnWork& w, const Seq& s, int g, int split, int at) {
  for (int r = at * 256 + (int)threadIdx.x; r < s.n * w.group; r += w.row_tiles * 256) {
    const int i = token_of(w, r), h = g * w.group + r - i * w.group;
    const int64_t part = ((int64_t)(s.row0 + i) * a.n_q_heads + h) * w.n_splits + split;
    w.m[part] = -INFINITY;
    w.l[part] = 0.f;
  }
}

// A page's operands for one wave.
template <int D>
struct PageRegs {
  uint4 k[D / 32], v[D / 32], vs[D / 32];
  uint32_t ks;
  __device__ __forceinline__ void load_k(const uint8_t* base, int lane) {
    const uint4* pk = (const uint4*)base + lane;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) k[j] = pk[64 * j];
    ks = *(const uint32_t*)(base + 32 * D + ((D == 128 ? lane : (lane >> 5) * 16 + (lane & 15)) * 4));
  }
  __device__ __forceinline__ void load_v(const uint8_t* base, int lane) {
    const uint4* pv = (const uint4*)(base + 34 * D) + lane;
    const uint4* ps = (const uint4*)(base + 66 * D + (lane >> 4) * (D / 2));
#pragma unroll
    for (int j = 0; j < D / 32; ++j) v[j] = pv[64 * j];
#pragma unroll
    for (int j = 0; j < D / 64; ++j) { vs[2 * j] = ps[2 * j]; vs[2 * j + 1] = ps[2 * j + 1]; }
  }
};

__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

__device__ __forceinline__ half8 dequant(uint32_t w, half2v s01, half2v s23, half2v s45, half2v s67) {
  const half2v a = fp4_pair(w, 0) * s01, b = fp4_pair(w, 1) * s23;
  const half2v c = fp4_pair(w, 2) * s45, d = fp4_pair(w, 3) * s67;
  return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Scales of tokens (or of one token twice) from the bytes of w: fp16 pairs.
__device__ __forceinline__ half2v scale_pair(uint32_t w, int lo, int hi) {
  const uint32_t sel = 0x0c | (uint32_t)lo << 8 | 0x0c0000u | (uint32_t)hi << 24;
  return __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0u, w, sel));
}

__device__ __forceinline__ float across_quarters_max(float v) {
  float a, b;
  perm16_swap(v, a, b);
  v = fmaxf(a, b);
  perm32_swap(v, a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float across_quarters_sum(float v) {
  float a, b;
  perm16_swap(v, a, b);
  v = a + b;
  perm32_swap(v, a, b);
  return a + b;
}

// Few rows: a workgroup of 4 waves takes ROWS (4 to 32) rows and a split of the
// pages; every wave walks its own pages (registers only) and the waves are
// joined in LDS at the end.  The next page's K is loaded into the registers
// that the scores have just freed, its V into those of the output's product, so
// that each is on its way during the other half of the work.
// Up to 4 (8) rows stand in the 16 columns of a tile 4 (2) times: a column weighs
// the tokens of its own quarter (half) of every page, a softmax of its own that
// the end joins, and a lane forms 4 (8) exponentials a page, not 16.  The longer
// join is worth it from two pages a wave on: graph replays, us, with / without,
// 4 rows: 64 sequences of 128 to 8,192 tokens (head_dim 64) 24.7 / 26.5, 8 of 2K
// to 8K 16.9 / 17.4, one of 32K 14.7 / 14.9, one of 2,048 (a page a wave) 8.3 /
// 8.15; 8 rows: the 64 sequences 26.7 / 27.1, the 8 17.5 / 17.6.
// A page of a head costs a wave about 380 vector instructions at head_dim 128
// (256 of them expand and scale the 16,384 codes) and 32 matrix ones; three waves
// a SIMD hide the memory behind it.  Measured (32 query heads on 8 of 128, fp16,
// one token): 16 sequences of 16,384 tokens 53 us, 5.4 TB/s of 285 MB; one of
// 32,768 11 us, 3.3 TB/s, of 2,048 5.2 us: launch and the chain table -> page ->
// join.
// Not faster: 8 or 16 waves a workgroup without splits (one sequence of 2,048
// 13.4 us against 8.2 with the merge), work cut on the device by the sequences'
// lengths (the 64 sequences 27.7 us against 26.9 then).
template <class T, int D, int ROWS>
__global__ __launch_bounds__(256, (D == 128 ? 4 : 5) - (ROWS > 16 ? 2 : 1))
void k_kv4_attn_rows(const shard_kv4_args a, const AttnWork w) {
  constexpr int WAVES = 4;
  constexpr int NQ = ROWS > 16 ? ROWS / 16 : 1;     // tiles of 16 columns
  constexpr int F = ROWS < 16 ? 16 / ROWS : 1;      // columns of a row
  constexpr int NS = 4 / F;                         // quarters of a page whose tokens a lane weighs
  constexpr int ST = D / 32;  // k-steps of a score, 32-channel blocks
  constexpr int NT = D / 16;  // channel tiles of the output
  __shared__ float sh_acc[WAVES][16 * NQ][D + 4];
  __shared__ float sh_m[WAVES][16 * NQ], sh_l[WAVES][16 * NQ];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, kq = lane >> 4;
  const int g = blockIdx.y;
  const int split = blockIdx.x & (w.n_splits - 1), rt0 = blockIdx.x >> w.split_shift;
  int b = blockIdx.z, len;
  if (w.sorted != 0.f) b = by_length(a, w, b, lane, len);
  else len = a.seq_lens[b];
  const Seq s = seq_of(a, b, len);
  const int group = w.group;
  const int n_rows = s.n * group;
  const int keys = min(s.len, s.cap);
  const int tiles = (keys + kPage - 1) / kPage;
  const int per = tiles_per_split(w, tiles);
  const int first = split * per, last = min(first + per, tiles);
  if (w.n_splits > 1 && first >= tiles) return nothing(a, w, s, g, split, rt0);
  // the scale's sign goes into q, so that the largest product is the largest score
  const float scale2 = a.scale == 0.f ? 1.f : fmaxf(fabsf(a.scale) * 1.4426950408889634f, kLeast);
  const half_t sign = a.scale < 0.f ? (half_t)-1.f : a.scale == 0.f ? (half_t)0.f : (half_t)1.f;

  const int fold = F == 1 ? 0 : col / ROWS;         // the lane's share: quarters fold * NS + 0 .. NS - 1
  for (int rt = rt0; rt * ROWS < n_rows; rt += w.row_tiles) {
    typedef T vec8 __attribute__((ext_vector_type(8)));
    vec8 raw[NQ][ST];
    float sc[NQ], m[NQ], l[NQ];
    int lim[NQ];                      // keys that the lane's row sees
    float4v acc[NQ][NT];
    const int r0 = rt * ROWS, r1 = min(r0 + ROWS, n_rows) - 1;
    // of the tile's rows (uniform)
    const int lim_min = min(max(s.len - s.n + token_of(w, r0) + 1, 0), keys);
    const int lim_max = min(max(s.len - s.n + token_of(w, r1) + 1, 0), keys);
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
      const int r = min(r0 + 16 * t + (F == 1 ? col : col % ROWS), r1);   // columns behind the last row repeat it, unused
      const int i = token_of(w, r), h = r - i * group;
      lim[t] = min(max(s.len - s.n + i + 1, 0), keys);
      const T* qp = (const T*)a.q + (int64_t)(s.row0 + i) * a.q_stride + (int64_t)(g * group + h) * a.q_head_stride + kq * (D / 4);
#pragma unroll
      for (int j = 0; j < ST; ++j) raw[t][j] = *(const vec8*)(qp + 8 * j);
      m[t] = -INFINITY;
      l[t] = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[t][n] = float4v{0.f, 0.f, 0.f, 0.f};
    }

    const int stop = min(last, (lim_max + kPage - 1) / kPage);
    if (first + wave < stop) {
    PageRegs<D> pg;
    // pages of the wave's tile, of its next one and (on its way) the one after:
    // the last tile's again where there is none, page 0 where there is no page
    const auto page_near = [&](int tile) { return page_of(a, b, min(tile, stop - 1) * kPage); };
    int page = page_near(first + wave), ahead = page_near(first + wave + WAVES);
    pg.load_k(head_of<D>(a, max(page, 0), g), lane);
    pg.load_v(head_of<D>(a, max(page, 0), g), lane);
    __builtin_amdgcn_sched_barrier(0);  // q is not waited for before the first page is on its way
    half8 q[NQ][ST];
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
      if constexpr (__is_same(T, half_t)) {
        sc[t] = scale2;
#pragma unroll
        for (int j = 0; j < ST; ++j) q[t][j] = raw[t][j] * sign;
      } else {
        float mx = 0.f;
#pragma unroll
        for (int j = 0; j < ST; ++j)
#pragma unroll
          for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf((float)raw[t][j][e]));
        mx = across_quarters_max(mx);
        const int ex = mx > 0.f ? (int)(__float_as_uint(mx) >> 23) - 127 : 0;
#pragma unroll
        for (int j = 0; j < ST; ++j)
#pragma unroll
          for (int e = 0; e < 8; ++e) q[t][j][e] = (half_t)ldexpf((float)raw[t][j][e], -ex) * sign;
        sc[t] = fmaxf(ldexpf(scale2, ex), kLeast);
      }
    }
    for (int tile = first + wave; tile < stop; tile += WAVES) {
      const int lim_page = page < 0 ? 0 : lim_max;   // keys of no page are not seen
      const bool none = page < 0;
      const uint8_t* next = head_of<D>(a, max(ahead, 0), g);
      page = ahead;
      ahead = page_near(tile + 2 * WAVES);
      const int left = lim_page - tile * kPage;
      if (left < kPage) {
        // tokens behind the last key: whatever their bytes are, their V is finite
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
          for (int run = 0; run < 2; ++run) {
            const int t0 = 32 * s2 + 16 * run + 4 * kq;
            const int live = min(max(left - t0, 0), 4);
            const uint32_t msk = live == 4 ? ~0u : (1u << (8 * live)) - 1u;
#pragma unroll
            for (int bk = 0; bk < ST; ++bk) {
              const int at = (s2 * ST + bk) * 2 + run;   // word of the lane's scales
              uint32_t* p = (uint32_t*)&pg.vs[at >> 2] + (at & 3);
              *p &= msk;
            }
          }
      }
      float4v S[NQ][4];
#pragma unroll
      for (int sub = 0; sub < 4; ++sub) {
        const half2v ks = scale_pair(pg.ks, sub, sub);
#pragma unroll
        for (int t = 0; t < NQ; ++t) S[t][sub] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < ST; ++j) {
          const uint32_t kw = D == 128 ? word(pg.k[sub], j) : word(pg.k[sub >> 1], (sub & 1) * 2 + j);
          const half8 kk = dequant(kw, ks, ks, ks, ks);
#pragma unroll
          for (int t = 0; t < NQ; ++t) S[t][sub] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, q[t][j], S[t][sub], 0, 0, 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);  // K's registers are free from here on
      pg.load_k(next, lane);
      half8 P[NQ][2];
#pragma unroll
      for (int t = 0; t < NQ; ++t) {
        float4v X[NS];                                // the lane's own scores
        if constexpr (F == 4) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float lo = fold & 1 ? S[t][1][i] : S[t][0][i], hi = fold & 1 ? S[t][3][i] : S[t][2][i];
            X[0][i] = fold & 2 ? hi : lo;
          }
        } else {
#pragma unroll
          for (int u = 0; u < NS; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) X[u][i] = F == 2 && fold ? S[t][(u + NS) & 3][i] : S[t][u][i];
        }
        if (none || (tile + 1) * kPage > lim_min) {
          const int seen = (none ? 0 : lim[t]) - tile * kPage - 16 * NS * fold - 4 * kq;
#pragma unroll
          for (int u = 0; u < NS; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) X[u][i] = 16 * u + i < seen ? X[u][i] : -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int u = 0; u < NS; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) mx = fmaxf(mx, X[u][i]);
        mx = across_quarters_max(mx) * sc[t];
        if (__builtin_amdgcn_ballot_w64(mx > m[t] + kMost)) {
          const float to = reference(m[t], mx);
          const float alpha = __builtin_amdgcn_exp2f(m[t] - (to == -INFINITY ? 0.f : to));
          m[t] = to;
          l[t] *= alpha;
#pragma unroll
          for (int n = 0; n < NT; ++n) acc[t][n] *= alpha;
        }
        const float base = m[t] == -INFINITY ? 0.f : m[t];
        float by = sc[t], from = -base;
        if (__builtin_amdgcn_ballot_w64(fabsf(base) > kFar)) {
          const bool far = fabsf(base) > kFar;
#pragma unroll
          for (int u = 0; u < NS; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) X[u][i] = far ? far_exponent(X[u][i], sc[t], base) : X[u][i];
          by = far ? 1.f : by;
          from = far ? 0.f : from;
        }
        float sum = 0.f;
        uint32_t pairs[NS][2];
#pragma unroll
        for (int u = 0; u < NS; ++u)
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(X[u][i], by, from));
            const float p2 = __builtin_amdgcn_exp2f(__builtin_fmaf(X[u][i + 1], by, from));
            sum += p;
            sum += p2;
            pairs[u][i / 2] = __builtin_bit_cast(uint32_t, half2v{(half_t)p, (half_t)p2});
          }
        // the other quarters' tokens are not the column's: weights of 0
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) {
          uint4 words;
          words.x = F == 1 || fold == 2 * s2 / NS ? pairs[2 * s2 % NS][0] : 0u;
          words.y = F == 1 || fold == 2 * s2 / NS ? pairs[2 * s2 % NS][1] : 0u;
          words.z = F == 1 || fold == (2 * s2 + 1) / NS ? pairs[(2 * s2 + 1) % NS][0] : 0u;
          words.w = F == 1 || fold == (2 * s2 + 1) / NS ? pairs[(2 * s2 + 1) % NS][1] : 0u;
          P[t][s2] = __builtin_bit_cast(half8, words);
        }
        l[t] += sum;
      }
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
        for (int bk = 0; bk < ST; ++bk) {
          const int at = (s2 * ST + bk) * 2;
          const uint32_t w0 = word(pg.vs[at >> 2], at & 3), w1 = word(pg.vs[at >> 2], (at & 3) + 1);
          const half2v s01 = scale_pair(w0, 0, 1), s23 = scale_pair(w0, 2, 3);
          const half2v s45 = scale_pair(w1, 0, 1), s67 = scale_pair(w1, 2, 3);
#pragma unroll
          for (int n = 2 * bk; n < 2 * bk + 2; ++n) {
            const half8 vv = dequant(word(pg.v[s2 * (D / 64) + (n >> 2)], n & 3), s01, s23, s45, s67);
#pragma unroll
            for (int t = 0; t < NQ; ++t) acc[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv, P[t][s2], acc[t][n], 0, 0, 0);
          }
        }
      __builtin_amdgcn_sched_barrier(0);
      pg.load_v(next, lane);
    }
    }

    // join the waves
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
      const float lt = across_quarters_sum(l[t]);
      if (kq == 0) {
        sh_m[wave][16 * t + col] = m[t];
        sh_l[wave][16 * t + col] = lt;
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) *(float4v*)&sh_acc[wave][16 * t + col][16 * n + 4 * kq] = acc[t][n];
    }
    __syncthreads();
    const auto write = [&](int r, int ch, auto x, float M, float lt) {  // some channels of a row
      constexpr int N = sizeof(x) / sizeof(float);
      const int i = token_of(w, r), h = g * group + r - i * group;
      const int64_t row = (int64_t)(s.row0 + i) * a.n_q_heads + h;
      if (w.n_splits == 1) {
        const float inv = lt == 0.f ? 0.f : 1.f / lt;   // a row that sees no key: zeros
        typedef T vec __attribute__((ext_vector_type(N)));
        vec o;
#pragma unroll
        for (int j = 0; j < N; ++j) o[j] = (T)(x[j] * inv);
        *(vec*)((T*)a.out + row * D + ch) = o;
      } else {
        const int64_t part = row * w.n_splits + split;
        *(decltype(x)*)(w.acc + part * D + ch) = x;
        if (ch == 0) {
          w.m[part] = M;
          w.l[part] = lt;
        }
      }
    };
    if constexpr (F == 1) {
      typedef float float8v __attribute__((ext_vector_type(8)));
      for (int u = tid; u < ROWS * (D / 8); u += 64 * WAVES) {
        const int rr = u / (D / 8), ch = (u % (D / 8)) * 8;
        if (rt * ROWS + rr >= n_rows) continue;
        float M = sh_m[0][rr];
#pragma unroll
        for (int v = 1; v < WAVES; ++v) M = fmaxf(M, sh_m[v][rr]);
        const float base = M == -INFINITY ? 0.f : M;
        float8v x{};
        float lt = 0.f;
#pragma unroll
        for (int v = 0; v < WAVES; ++v) {
          const float k = __builtin_amdgcn_exp2f(sh_m[v][rr] - base);
          lt += k * sh_l[v][rr];
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] += k * sh_acc[v][rr][ch + j];
        }
        write(rt * ROWS + rr, ch, x, M, lt);
      }
    } else {
      // a row a wave, its weights in the lanes of 16
      typedef float pair __attribute__((ext_vector_type(D / 64)));
      const int p = lane % (WAVES * F), ch = lane * (D / 64);
      for (int rr = wave; rr < ROWS && rt * ROWS + rr < n_rows; rr += WAVES) {
        pair y[WAVES * F];
#pragma unroll
        for (int u = 0; u < WAVES * F; ++u) y[u] = *(const pair*)&sh_acc[u / F][rr + ROWS * (u % F)][ch];
        const float mp = sh_m[p / F][rr + ROWS * (p % F)], lp = sh_l[p / F][rr + ROWS * (p % F)];
        const float M = row16_reduce(mp, OpMax());
        const float k = __builtin_amdgcn_exp2f(mp - (M == -INFINITY ? 0.f : M));
        const float lt = row16_reduce((lane & 15) < WAVES * F ? k * lp : 0.f, OpAdd());
        pair x{};
#pragma unroll
        for (int u = 0; u < WAVES * F; ++u) x += __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(k), u)) * y[u];
        write(rt * ROWS + rr, ch, x, M, lt);
      }
    }
  }
}

// Many rows: a workgroup of 4 waves takes 128 rows, 32 a wave, and walks a split
// of the pages.  A page is dequantized once for all of them into LDS (fp16, two
// buffers) and read from there as 32x32x16 operands.  Rows are 16 bytes longer
// than their data: 8 lanes that read or write one 16-byte chunk of 8 rows use
// every bank once, and every read is an immediate offset from one address.
//
// A wave alternates two phases with a barrier after each: vector (the softmax of
// page n; V of page n + 1 and K of page n + 2 into LDS, from registers that were
// loaded a page earlier) and matrix (the output's product with V of page n, the
// scores of page n + 1).  The second workgroup of a CU runs one while the first
// runs the other.
//
// Measured: a whole prompt of 8,192 tokens, 32 heads on 8, 570 us, 0.96 PFLOP/s
// of its causal half; an 8192^3 fp16 product of the library reaches 1.17 on the
// same card.  The clock falls to 1.85 GHz under it; at that clock the matrix pipe
// is busy half the time.  Not faster: 256 rows in two groups of waves a phase
// apart (568 us against 560 then), 64 rows a wave (1,073: registers), scores of
// the next page between the maxima and the weights of this one (570).
// Byte offsets are formed once: the loop adds a page's address and a buffer's.
template <int W>
struct Words {
  uint32_t w[W];
};
template <int D>
struct KRegs {  // a thread's part of a page's K: a quarter of a token
  static constexpr int W = D / 32;
  static constexpr int kRow = 2 * D + 16, kBuffer = kPage * kRow;
  Words<W> k;
  uint32_t s;
  uint32_t from, s_from, to;
  __device__ __forceinline__ KRegs(int tid) {
    const int kq = (tid & 63) >> 4, slot = (tid >> 6) * 16 + (tid & 15);
    from = k_code_at<D>(slot, kq);
    s_from = k_scale_at<D>(slot, D == 128 ? kq : kq >> 1);
    to = slot * kRow + kq * W * 16;
  }
  __device__ __forceinline__ void load(const uint8_t* base) {
    s = base[s_from];
    __builtin_memcpy(&k, __builtin_assume_aligned(base + from, 4 * W), 4 * W);
  }
  // rows [token][channel]
  __device__ __forceinline__ void store(char* buffer) const {
    const half2v sc = scale_pair(s, 0, 0);
#pragma unroll
    for (int j = 0; j < W; ++j) *(half8*)(buffer + to + 16 * j) = dequant(k.w[j], sc, sc, sc, sc);
  }
};

template <int D>
struct VRegs {  // a thread's part of a page's V: W channels 16 apart of 8 tokens
  static constexpr int W = D / 32;
  static constexpr int B = D / 64;  // blocks of 32 channels among them
  static constexpr int kRow = 2 * kPage + 16, kBuffer = D * kRow;
  Words<W> v;
  Words<2 * B> s;
  uint32_t from, s_from, to;
  int t0;                           // first of its tokens
  __device__ __forceinline__ VRegs(int tid) {
    const int lane = tid & 63, kq = lane >> 4, sg = tid >> 7, x = (tid >> 6) & 1;
    from = 34 * D + (D == 128 ? ((sg * 2 + x) * 64 + lane) * 16 : (sg * 64 + lane) * 16 + x * 8);
    s_from = 66 * D + ((kq * 2 + sg) * (D / 32) + x * B) * 8;
    to = (x * (D / 2) + (lane & 15)) * kRow + (4 * sg + kq) * 16;
    t0 = 32 * sg + 4 * kq;
  }
  __device__ __forceinline__ void load(const uint8_t* base) {
    __builtin_memcpy(&v, __builtin_assume_aligned(base + from, 4 * W), 4 * W);
    __builtin_memcpy(&s, __builtin_assume_aligned(base + s_from, 8 * B), 8 * B);
  }
  // rows [channel][word: 8 tokens in the order of its codes].  Tokens from
  // `left` on get V = 0, whatever their bytes are.
  __device__ __forceinline__ void store(char* buffer, int left) {
    if (left < kPage) {
#pragma unroll
      for (int run = 0; run < 2; ++run) {
        const int n = min(max(left - (t0 + 16 * run), 0), 4);
        const uint32_t m = n == 4 ? ~0u : (1u << (8 * n)) - 1u;
#pragma unroll
        for (int k = 0; k < B; ++k) s.w[2 * k + run] &= m;
      }
    }
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const uint32_t w0 = s.w[(j >> 1) * 2], w1 = s.w[(j >> 1) * 2 + 1];
      *(half8*)(buffer + to + 16 * j * kRow) =
          dequant(v.w[j], scale_pair(w0, 0, 1), scale_pair(w0, 2, 3), scale_pair(w1, 0, 1), scale_pair(w1, 2, 3));
    }
  }
};

constexpr int kTileRows = 128;

template <class T, int D>
__global__ __launch_bounds__(256, 2)
void k_kv4_attn_tile(const shard_kv4_args a, const AttnWork w) {
  constexpr int QS = D / 16;        // k-steps of a score
  constexpr int CT = D / 32;        // channel tiles of the output
  typedef KRegs<D> K;
  typedef VRegs<D> V;
  __shared__ __align__(16) char sk[2 * K::kBuffer], sv[2 * V::kBuffer];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, hi = lane >> 5;
  // kv heads innermost: with 8 of them each has an XCD (workgroup id mod 8) and
  // its L2 to itself; long row tiles first
  const int g = blockIdx.x % a.n_kv_heads, b = blockIdx.y;
  const int unit = blockIdx.x / a.n_kv_heads;
  const int split = unit & (w.n_splits - 1), at = unit >> w.split_shift;
  const Seq s = seq_of(a, b);
  const int group = w.group;
  const int n_rows = s.n * group;
  const int keys = min(s.len, s.cap);
  const int tiles = (keys + kPage - 1) / kPage;
  const int per = tiles_per_split(w, tiles);
  const int first = split * per, end = min(first + per, tiles);
  if (w.n_splits > 1 && first >= tiles) return nothing(a, w, s, g, split, at);
  const int n_tiles = (n_rows + kTileRows - 1) / kTileRows;
  const auto limit = [&](int row) { return min(max(s.len - s.n + token_of(w, row) + 1, 0), keys); };

  for (int back = at; back < n_tiles; back += w.row_tiles) {
    const int rt = n_tiles - 1 - back;
    const int r0 = rt * kTileRows + wave * 32;                  // the wave's first row
    const int last = min(end, (limit(min(rt * kTileRows + kTileRows, n_rows) - 1) + kPage - 1) / kPage);
    // keys that every row of the wave sees: pages below need no mask
    const int lim_min = r0 + 32 <= n_rows ? limit(r0) : 0;
    const int r = r0 + col;
    const bool live = r < n_rows;
    const int i = live ? token_of(w, r) : 0, h = g * group + (live ? r - i * group : 0);
    const int lim = live ? limit(r) : 0;
    half8 q[QS];
    // the scale's sign goes into q, so that the largest product is the largest score
    const float sign = a.scale < 0.f ? -1.f : a.scale == 0.f ? 0.f : 1.f;
    float sc = a.scale == 0.f ? 1.f : fmaxf(fabsf(a.scale) * 1.4426950408889634f, kLeast);
    const T* qp = (const T*)a.q + (int64_t)(s.row0 + i) * a.q_stride + (int64_t)h * a.q_head_stride + 8 * hi;
    if constexpr (__is_same(T, half_t)) {
#pragma unroll
      for (int j = 0; j < QS; ++j) q[j] = live ? *(const half8*)(qp + 16 * j) * (half_t)sign : half8{};
    } else {
      float mx = 0.f;
#pragma unroll
      for (int j = 0; j < QS; ++j) {
        float x[8] = {};
        if (live) load8(qp + 16 * j, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(x[e]));
      }
      float other, mine;
      perm32_swap(mx, mine, other);
      mx = fmaxf(mine, other);
      const int ex = mx > 0.f ? (int)(__float_as_uint(mx) >> 23) - 127 : 0;
#pragma unroll
      for (int j = 0; j < QS; ++j) {
        float x[8] = {};
        if (live) load8(qp + 16 * j, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) q[j][e] = (half_t)(sign * ldexpf(x[e], -ex));
      }
      sc = fmaxf(ldexpf(sc, ex), kLeast);
    }
    float m = -INFINITY, l = 0.f;
    float16v acc[CT], S[2];
#pragma unroll
    for (int k = 0; k < CT; ++k)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[k][e] = 0.f;

    const auto scores = [&](uint32_t buffer) {
      const char* from = sk + buffer + col * K::kRow + 16 * hi;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int e = 0; e < 16; ++e) S[t][e] = 0.f;
#pragma unroll
        for (int j = 0; j < QS; ++j)
          S[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*(const half8*)(from + 32 * t * K::kRow + 32 * j), q[j], S[t], 0, 0, 0);
      }
    };

    __syncthreads();  // the buffers' readers of the row tile before
    if (first < last) {
      // pages of tiles n .. n + 3; past the last tile it again, page 0 where there is none
      const auto page_near = [&](int tile) { return page_of(a, b, min(tile, last - 1) * kPage); };
      const auto page_at = [&](int page) { return head_of<D>(a, max(page, 0), g); };
      const auto left = [&](int page, int tile) { return page < 0 ? 0 : keys - tile * kPage; };
      int p0 = page_near(first), p1 = page_near(first + 1), p2 = page_near(first + 2), p3 = page_near(first + 3);
      K kr(tid);
      V vr(tid);
      kr.load(page_at(p0));
      vr.load(page_at(p0));
      kr.store(sk);
      kr.load(page_at(p1));
      vr.store(sv, left(p0, first));
      vr.load(page_at(p1));
      kr.store(sk + K::kBuffer);
      kr.load(page_at(p2));
      __syncthreads();
      scores(0);
      __syncthreads();
      uint32_t k0 = 0, k1 = K::kBuffer, v0 = 0, v1 = V::kBuffer;  // buffers of pages n, n + 1
      for (int tile = first; tile < last; ++tile) {
        // vector phase
        vr.store(sv + v1, left(p1, tile + 1));
        vr.load(page_at(p2));
        kr.store(sk + k0);
        kr.load(page_at(p3));
        if (p0 < 0 || (tile + 1) * kPage > lim_min) {
          const int seen = p0 < 0 ? 0 : lim;          // keys of no page are not seen
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              S[t][e] = tile * kPage + 32 * t + 8 * (e >> 2) + 4 * hi + (e & 3) < seen ? S[t][e] : -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) mx = fmaxf(mx, S[t][e]);
        float other, mine;
        perm32_swap(mx, mine, other);
        mx = fmaxf(mine, other) * sc;
        if (__builtin_amdgcn_ballot_w64(mx > m + kMost)) {
          const float to = reference(m, mx);
          const float alpha = __builtin_amdgcn_exp2f(m - (to == -INFINITY ? 0.f : to));
          m = to;
          l *= alpha;
#pragma unroll
          for (int k = 0; k < CT; ++k)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[k][e] *= alpha;
        }
        const float base = m == -INFINITY ? 0.f : m;
        float by = sc, from_m = -base;
        if (__builtin_amdgcn_ballot_w64(fabsf(base) > kFar)) {
          const bool far = fabsf(base) > kFar;
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) S[t][e] = far ? far_exponent(S[t][e], sc, base) : S[t][e];
          by = far ? 1.f : by;
          from_m = far ? 0.f : from_m;
        }
        half8 P[4];
        float sum = 0.f;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(S[t][e], by, from_m));
            sum += p;
            P[2 * t + ((e >> 2) & 1)][(e & 3) + 4 * (e >> 3)] = (half_t)p;  // runs of tokens 0 2 | 1 3, as V's words
          }
        l += sum;
        p0 = p1;
        p1 = p2;
        p2 = p3;
        p3 = page_near(tile + 4);
        __builtin_amdgcn_sched_barrier(0);            // nothing of a phase moves into the other
        __syncthreads();
        // matrix phase; the scores past the last tile are those of it again, unused
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(1);
        const char* from = sv + v0 + col * V::kRow + 16 * hi;
#pragma unroll
        for (int st = 0; st < 4; ++st)
#pragma unroll
          for (int k = 0; k < CT; ++k)
            acc[k] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*(const half8*)(from + 32 * k * V::kRow + 32 * st), P[st], acc[k], 0, 0, 0);
        scores(k1);
        // operands six reads ahead of their products
        __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
        for (int k = 0; k < 4 * CT + 2 * QS; ++k) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          if (k < 4 * CT + 2 * QS - 6) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(0);
        __syncthreads();
        __builtin_amdgcn_sched_barrier(0);
        const uint32_t kt = k0, vt = v0;
        k0 = k1;
        k1 = kt;
        v0 = v1;
        v1 = vt;
      }
    }

    float other, mine;
    perm32_swap(l, mine, other);
    l = mine + other;
    if (live) {
      const int64_t row = (int64_t)(s.row0 + i) * a.n_q_heads + h;
      if (w.n_splits == 1) {
        const float inv = l == 0.f ? 0.f : 1.f / l;   // a row that sees no key: zeros
        typedef T vec4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int k = 0; k < CT; ++k)
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            vec4 o;
#pragma unroll
            for (int x = 0; x < 4; ++x) o[x] = (T)(acc[k][e + x] * inv);
            *(vec4*)((T*)a.out + row * D + 32 * k + 2 * e + 4 * hi) = o;
          }
      } else {
        const int64_t part = row * w.n_splits + split;
#pragma unroll
        for (int k = 0; k < CT; ++k)
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            *(float4v*)(w.acc + part * D + 32 * k + 2 * e + 4 * hi) =
                float4v{acc[k][e], acc[k][e + 1], acc[k][e + 2], acc[k][e + 3]};
        if (hi == 0) {
          w.m[part] = m;
          w.l[part] = l;
        }
      }
    }
  }
}

// Joins the splits of a row; 2.9 to 4.8 us, latency, up to 64 splits.  WAVES waves
// take a row's splits in turn, several a load (16 bytes a lane); every wave forms
// all weights itself (128 splits at most: two a lane).  Nothing here waits for
// lengths: splits without keys have a maximum of -inf, their sums are whatever
// was there and not used.
constexpr int kMaxSplits = 128;

template <class T, int D, int WAVES>
__device__ __forceinline__ void merge_row(const AttnWork& w, T* out, int64_t row, int wave, int lane, float4v* sh) {
  constexpr int LPS = D / 4;       // lanes of a split's row
  constexpr int SPL = 64 / LPS;    // splits a load
  const int n = w.n_splits;
  const float* pm = w.m + row * n;
  const float* pl = w.l + row * n;
  const float m0 = lane < n ? pm[lane] : -INFINITY, m1 = lane + 64 < n ? pm[lane + 64] : -INFINITY;
  const float l0 = lane < n ? pl[lane] : 0.f, l1 = lane + 64 < n ? pl[lane + 64] : 0.f;
  const float* pa = w.acc + row * n * D + (lane % LPS) * 4;
  constexpr int U = 4;             // loads in flight
  float4v v[U];
  const int s0 = wave * SPL + lane / LPS;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = s0 + u * SPL * WAVES;
    v[u] = i < n ? *(const float4v*)(pa + (int64_t)i * D) : float4v{0.f, 0.f, 0.f, 0.f};
  }
  // a row of NaN has NaN in its sums, not in its maxima
  const float M = wave64_reduce(fmaxf(m0, m1), OpMax());
  const float base = M == -INFINITY ? 0.f : M;
  const float f0 = exp2f(m0 - base), f1 = exp2f(m1 - base);
  const float l = wave64_reduce(f0 * l0 + f1 * l1, OpAdd());
  float4v x{0.f, 0.f, 0.f, 0.f};
  for (int at = 0; at < n; at += SPL * WAVES * U) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = at + s0 + u * SPL * WAVES;
      const float f = i < 64 ? __shfl(f0, i & 63) : __shfl(f1, i & 63);
      if (i < n && f != 0.f) x += f * v[u];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = at + s0 + (u + U) * SPL * WAVES;
      v[u] = i < n ? *(const float4v*)(pa + (int64_t)i * D) : float4v{0.f, 0.f, 0.f, 0.f};
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (LPS == 16) x[e] += xor_lane<16>(x[e]);
    x[e] += xor_lane<32>(x[e]);
  }
  if constexpr (WAVES > 1) {
    if (lane < LPS) sh[wave * LPS + lane] = x;
    __syncthreads();
    if (wave) return;
    if (lane < LPS)
#pragma unroll
      for (int k = 1; k < WAVES; ++k) x += sh[k * LPS + lane];
  }
  if (lane < LPS) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    typedef T vec4 __attribute__((ext_vector_type(4)));
    vec4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (T)(x[e] * inv);
    *(vec4*)(out + row * D + lane * 4) = o;
  }
}

// A row a workgroup (few rows or many splits: latency counts) or a row a wave.
template <class T, int D, int WAVES>
__global__ __launch_bounds__(256)
void k_kv4_merge(const shard_kv4_args a, const AttnWork w) {
  __shared__ float4v sh[WAVES > 1 ? WAVES * D / 4 : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t r = WAVES > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
  int t0 = 0, t1 = a.n_tokens;   // rows of sequences
  if (a.cu_seqlens) {
    t0 = max(a.cu_seqlens[0], 0);
    t1 = min(a.cu_seqlens[a.batch], a.n_tokens);
  }
  if (r >= (int64_t)t0 * a.n_q_heads && r < (int64_t)t1 * a.n_q_heads)
    merge_row<T, D, WAVES>(w, (T*)a.out, r, WAVES > 1 ? wave : 0, lane, sh);
}

// --------------------------------------------------------------------------
// host side
// --------------------------------------------------------------------------
int check_batch(const shard_kv4_args* a) {
  if (!a || !a->cache || !a->block_table || !a->seq_lens) return SHARD_ERR_ARG;
  if (a->batch <= 0 || a->n_tokens < 0 || a->n_kv_heads <= 0 || a->n_pages <= 0 || a->table_width <= 0)
    return SHARD_ERR_ARG;
  if (!a->cu_seqlens && a->n_tokens != a->batch) return SHARD_ERR_ARG;
  if (a->head_dim != 64 && a->head_dim != 128) return SHARD_ERR_SHAPE;
  if (a->dtype != SHARD_FP16 && a->dtype != SHARD_BF16) return SHARD_ERR_SHAPE;
  // positions are int32 and the grid's y and z 16 bits
  if (a->table_width > (INT32_MAX - 64) / kPage || a->batch > 65535 || a->n_kv_heads > 1024) return SHARD_ERR_SHAPE;
  if (a->page_stride < (int64_t)a->n_kv_heads * 68 * a->head_dim || a->page_stride % 16 || a->table_stride < a->table_width)
    return SHARD_ERR_ARG;
  if ((uintptr_t)a->cache % 16) return SHARD_ERR_ARG;
  return SHARD_OK;
}

bool rows_ok(const void* p, int64_t stride, int64_t head_stride) {
  return p && (uintptr_t)p % 16 == 0 && stride >= 0 && head_stride >= 0 && stride % 8 == 0 && head_stride % 8 == 0;
}

// 32-token groups that max_new tokens can touch; the kernels stride where a launch
// (2^32 - 1 threads) holds no more.
int groups_of(const shard_kv4_args* a) {
  const int n = !a->cu_seqlens ? 1 : a->max_new > 0 ? std::min(a->max_new, a->n_tokens) : a->n_tokens;
  return n <= 1 ? 1 : std::min((n - 1) / 32 + 2, 1 << 20);
}

// Row tiles and splits of an attention call.  Workgroups for two a CU (a split
// takes 4 tiles at least), and at most 64 tiles (4,096 tokens) a split of few
// rows, so that a batch of uneven lengths ends together.  Measured (graph
// replays, us; head_dim 128, 32 on 8 heads): 1 x 32K with 256 / 512 / 768
// workgroups 15.5 / 15.3 / 17.0, 8 sequences of 2K to 8K 20.9 / 17.3 / 18.5;
// 16 x 16K with 32 / 64 / 128 tiles at most 64.8 / 60.2 / 60.0.  Rows by rows or
// by tiles: 2 x 8,000 with 12 / 32 new tokens (48 / 128 rows) 20.3 / 27.1 by rows,
// 26.6 / 33.7 by tiles; 16 x 4,000 with 16 (64 rows) 40.8 / 52.1.
// With several workgroups a CU those of longer sequences start first, and 32
// tiles are a split's most where that makes 2,048 workgroups or fewer.  Without /
// with both: 64 sequences of 128 to 8,192 tokens at head_dim 64 24.9 / 23.9
// (either alone: 24.0 and 25.2), at 128 39.8 / 37.9, 256 of 62 to 4,000 74.5 /
// 67.3, 100 of 250 to 16,000 60.7 / 56.5; equal lengths, 128 of 3,000, 83.6 / 84.4.
// One choice for the call, by its longest sequence of new tokens: a prompt beside
// single tokens puts those into tiles of 128 rows, without splits of their own.  A
// prompt of 2,048 beside 32 single tokens at 8K to 32K 1,414 us (the two in calls
// of their own 181), a chunk of 512 at 8K beside them 1,391 (203), 40 new tokens
// 932 (144).
struct AttnPlan {
  int rows;       // of a workgroup: 4, 8, 16 or 32 (rows kernel), 128 (tile kernel)
  int row_tiles, n_splits, split_shift;
  float sorted;
};
AttnPlan plan_of(const shard_kv4_args* a) {
  AttnPlan p;
  const int group = a->n_q_heads / a->n_kv_heads;
  const int64_t n = a->max_new > 0 && a->max_new < a->n_tokens ? a->max_new : a->n_tokens;
  const int64_t rows = (a->cu_seqlens ? n : 1) * group;
  p.rows = rows <= 16 ? 16 : rows <= 128 ? 32 : 128;
  p.row_tiles = (int)((rows + p.rows - 1) / p.rows);
  const int64_t cap = (int64_t)a->table_width * kPage;
  const int64_t len = a->max_len > 0 && a->max_len < cap ? a->max_len : cap;
  const int64_t tiles = (len + kPage - 1) / kPage;
  const int64_t wg = (int64_t)a->batch * a->n_kv_heads * p.row_tiles;
  int64_t sp = (512 + wg - 1) / wg;
  int64_t even = (tiles + 63) / 64;
  if (wg >= 512 && even > 1 && 2 * even * wg <= 2048) even *= 2;  // room to even out
  if (p.rows != 128 && even > sp) sp = even;
  if (sp > (tiles + kMinTiles - 1) / kMinTiles) sp = (tiles + kMinTiles - 1) / kMinTiles;
  if (sp > kMaxSplits) sp = kMaxSplits;
  if ((int64_t)a->n_tokens * a->n_q_heads >= 1 << 24) sp = 1;  // more rows than a launch of the join takes
  // the nearest power of two
  p.split_shift = 0;
  while ((int64_t)2 << p.split_shift <= kMaxSplits && (int64_t)2 << (2 * p.split_shift) < sp * sp) ++p.split_shift;
  p.n_splits = 1 << p.split_shift;
  // several workgroups a CU: the longest first
  p.sorted = a->batch > 1 && wg * p.n_splits >= 1024 ? 16.f / len : 0.f;
  // few rows fold where a wave has more than a page (k_kv4_attn_rows)
  if (rows <= 8 && tiles > kMinTiles * p.n_splits) p.rows = rows <= 4 ? 4 : 8;
  return p;
}

int check_attn(const shard_kv4_args* a) {
  const int rc = check_batch(a);
  if (rc) return rc;
  if (a->n_q_heads <= 0 || a->n_q_heads % a->n_kv_heads) return SHARD_ERR_SHAPE;
  if ((int64_t)a->n_tokens * a->n_q_heads > INT32_MAX) return SHARD_ERR_SHAPE;  // rows are counted in 32 bits
  return SHARD_OK;
}

}  // namespace
}  // namespace shard

using namespace shard;

#define KV4_DISPATCH(KERNEL, grid, s, ...)                                                                      \
  do {                                                                                                          \
    if (a->dtype == SHARD_FP16) {                                                                               \
      if (a->head_dim == 128) hipLaunchKernelGGL((KERNEL<half_t, 128>), grid, dim3(256), 0, s, __VA_ARGS__);    \
      else hipLaunchKernelGGL((KERNEL<half_t, 64>), grid, dim3(256), 0, s, __VA_ARGS__);                        \
    } else {                                                                                                    \
      if (a->head_dim == 128) hipLaunchKernelGGL((KERNEL<bf16_t, 128>), grid, dim3(256), 0, s, __VA_ARGS__);    \
      else hipLaunchKernelGGL((KERNEL<bf16_t, 64>), grid, dim3(256), 0, s, __VA_ARGS__);                        \
    }                                                                                                           \
  } while (0)

#define KV4_DISPATCH_N(KERNEL, N, grid, s, ...)                                                              \
  do {                                                                                                                \
    if (a->dtype == SHARD_FP16) {                                                                                     \
      if (a->head_dim == 128) hipLaunchKernelGGL((KERNEL<half_t, 128, N>), grid, dim3(256), 0, s, __VA_ARGS__);   \
      else hipLaunchKernelGGL((KERNEL<half_t, 64, N>), grid, dim3(256), 0, s, __VA_ARGS__);                       \
    } else {                                                                                                          \
      if (a->head_dim == 128) hipLaunchKernelGGL((KERNEL<bf16_t, 128, N>), grid, dim3(256), 0, s, __VA_ARGS__);   \
      else hipLaunchKernelGGL((KERNEL<bf16_t, 64, N>), grid, dim3(256), 0, s, __VA_ARGS__);                       \
    }                                                                                                                 \
  } while (0)

extern "C" {

size_t shard_kv4_args_size(void) { return sizeof(shard_kv4_args); }
uint64_t shard_kv4_args_layout(void) { return SHARD_KV4_ARGS_LAYOUT; }

int64_t shard_kv4_page_bytes(int32_t n_kv_heads, int32_t head_dim) {
  if (n_kv_heads <= 0 || (head_dim != 64 && head_dim != 128)) return 0;
  return (int64_t)n_kv_heads * 68 * head_dim;
}

int shard_kv4_append(const shard_kv4_args* a, void* stream) {
  const int rc = check_batch(a);
  if (rc) return rc;
  if (!a->phases || (uintptr_t)a->phases % 16 || a->n_phases <= 0) return SHARD_ERR_ARG;
  if (!rows_ok(a->k, a->k_stride, a->k_head_stride) || !rows_ok(a->v, a->v_stride, a->v_head_stride)) return SHARD_ERR_ARG;
  int q_groups = 0;
  if (a->q) {
    if (!rows_ok(a->q, a->q_stride, a->q_head_stride) || !a->q_out || (uintptr_t)a->q_out % 16 || a->n_q_heads <= 0)
      return SHARD_ERR_ARG;
    q_groups = (a->n_q_heads + kHeadsQ - 1) / kHeadsQ;
    if (a->n_kv_heads + q_groups > 65535) return SHARD_ERR_SHAPE;
  }
  if (a->n_tokens == 0) return SHARD_OK;
  const dim3 grid(groups_of(a), a->n_kv_heads + q_groups, a->batch);
  KV4_DISPATCH(k_kv4_append, grid, (hipStream_t)stream, *a);
  SHARD_LAUNCH_CHECK("shard_kv4_append");
  return SHARD_OK;
}

int shard_kv4_read(const shard_kv4_args* a, void* stream) {
  const int rc = check_batch(a);
  if (rc) return rc;
  if (!a->k_out || !a->v_out || (uintptr_t)a->k_out % 16 || (uintptr_t)a->v_out % 16) return SHARD_ERR_ARG;
  if (a->n_tokens == 0) return SHARD_OK;
  const dim3 grid(groups_of(a), a->n_kv_heads, a->batch);
  KV4_DISPATCH(k_kv4_read, grid, (hipStream_t)stream, *a);
  SHARD_LAUNCH_CHECK("shard_kv4_read");
  return SHARD_OK;
}

size_t shard_kv4_attn_workspace(const shard_kv4_args* a) {
  if (check_attn(a) || a->n_tokens == 0) return 0;
  const AttnPlan p = plan_of(a);
  if (p.n_splits == 1) return 0;
  return (size_t)a->n_tokens * a->n_q_heads * p.n_splits * (a->head_dim + 2) * sizeof(float);
}

int shard_kv4_attn(const shard_kv4_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = check_attn(a);
  if (rc) return rc;
  if (!rows_ok(a->q, a->q_stride, a->q_head_stride) || !a->out || (uintptr_t)a->out % 16) return SHARD_ERR_ARG;
  if (!(fabsf(a->scale) <= kMostScale)) return SHARD_ERR_ARG;  // NaN, or infinite times log2(e)
  if (a->n_tokens == 0) return SHARD_OK;
  const AttnPlan p = plan_of(a);
  const int64_t rows = (int64_t)a->n_tokens * a->n_q_heads;
  AttnWork w{};
  w.n_splits = p.n_splits;
  w.split_shift = p.split_shift;
  w.sorted = p.sorted;
  w.group = a->n_q_heads / a->n_kv_heads;
  w.group_shift = w.group & (w.group - 1) ? -1 : __builtin_ctz(w.group);
  w.row_tiles = p.row_tiles;
  if ((int64_t)w.n_splits * w.row_tiles * a->n_kv_heads > INT32_MAX) return SHARD_ERR_SHAPE;
  if (p.n_splits > 1) {
    const size_t need = shard_kv4_attn_workspace(a);
    if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16) {
      char text[96];
      snprintf(text, sizeof(text), "shard_kv4_attn needs %zu bytes of workspace, 16-byte aligned", need);
      set_last_text(text);
      return SHARD_ERR_WORKSPACE;
    }
    w.acc = (float*)workspace;
    w.m = w.acc + rows * p.n_splits * a->head_dim;
    w.l = w.m + rows * p.n_splits;
  }
  const hipStream_t s = (hipStream_t)stream;
  const dim3 rows_grid((unsigned)(w.n_splits * w.row_tiles), a->n_kv_heads, a->batch);
  if (p.rows == 4) KV4_DISPATCH_N(k_kv4_attn_rows, 4, rows_grid, s, *a, w);
  else if (p.rows == 8) KV4_DISPATCH_N(k_kv4_attn_rows, 8, rows_grid, s, *a, w);
  else if (p.rows == 16) KV4_DISPATCH_N(k_kv4_attn_rows, 16, rows_grid, s, *a, w);
  else if (p.rows == 32) KV4_DISPATCH_N(k_kv4_attn_rows, 32, rows_grid, s, *a, w);
  else {
    const dim3 grid((unsigned)((int64_t)w.n_splits * w.row_tiles * a->n_kv_heads), a->batch);
    KV4_DISPATCH(k_kv4_attn_tile, grid, s, *a, w);
  }
  SHARD_LAUNCH_CHECK("shard_kv4_attn");
  if (p.n_splits > 1) {
    // up to 8 splits of a row are one load's; more, and few rows, spread over waves
    if (p.n_splits > 8) KV4_DISPATCH_N(k_kv4_merge, 4, dim3((unsigned)rows), s, *a, w);
    else KV4_DISPATCH_N(k_kv4_merge, 1, dim3((unsigned)((rows + 3) / 4)), s, *a, w);
    SHARD_LAUNCH_CHECK("shard_kv4_attn merge");
  }
  return SHARD_OK;
}

}  // extern "C"
