// Log probabilities of given tokens, entropy and the most probable tokens of
// each row of logits, in one pass over the row.
//
// A workgroup takes a part of a row.  Every thread keeps its own running
// maximum M with l = sum 2^d and t = sum d 2^d, d = (x - M) log2 e, and the
// place of its best element; then
//   lse = M + ln l,  logprob = x - lse,  entropy = ln l - ln2 t / l
// after the threads' (and the parts') sums are joined at a common maximum.
// The difference x - M is taken first, so that its rounding is relative to
// itself and a row of equal logits far from 0 loses nothing.
//
// M is the thread's true maximum, the row's after the joins.
//
// Top k: every thread also notes the largest logit of each eighth of its
// elements (a slot).  The k-th largest of the 256 threads' largest bounds the
// row's k-th largest from below, so only the slots that reach it (about k of
// 2,048) are read once more; their elements that reach it go into a list in
// LDS, where an element's rank is the number of larger ones.
// Elements are compared as (value, lower index first) in 64 bits, so no two
// are equal.  Where more than the list holds reach the bound (many equal
// logits), the list's own k-th largest is the next bound.
//
// Measured: 2,048 rows of 128,256 bf16 logits with 20 alternatives 110 us, 4.8
// TB/s, a large copy's rate, the vector pipe 87% busy; one fp16 row with 5, in 63
// parts, 5 us and 4 for the join, each a chain of latencies: load, sums, bound,
// list.
#include <stdio.h>

#include "common.h"

namespace shard {
namespace {

typedef __bf16 bf16_t;
typedef unsigned long long u64;

constexpr int kMaxTop = 64;
constexpr int kMaxParts = 64;
constexpr int kList = 1024;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLowest = -3.402823466e38f;

struct LogprobArgs {
  const void* logits;
  int64_t vocab, stride;
  const int64_t* tokens;
  int top, parts;
  int64_t granules;    // 16-byte granules of a part
  float* logprob;
  float* entropy;
  float* top_logprobs;
  int64_t* top_ids;
  u64* ws_keys;        // [row][part][top], descending, 0 = none
  float4* ws_stats;    // [row][part]: M, l, t
};

// Larger for larger values, for equal ones larger for lower indices; 0 for NaN.
__device__ __forceinline__ u64 key_of(float x, int64_t i) {
  return x == x ? (u64)f2ord(x + 0.f) << 32 | (uint32_t)(~(uint32_t)i) : 0;  // -0 counts as 0
}
__device__ __forceinline__ float value_of(u64 key) { return ord2f((uint32_t)(key >> 32)); }
__device__ __forceinline__ int64_t index_of(u64 key) { return (int64_t)(uint32_t)~(uint32_t)key; }

// A row seen as 16-byte granules from the aligned address at or before it.
template <class T>
struct Row {
  static constexpr int VEC = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(VEC)));
  const T* p;
  int64_t n;
  int mis;       // elements of the first granule that lie before the row
  int64_t count; // granules
  __device__ Row(const T* row, int64_t vocab) : p(row), n(vocab) {
    mis = (int)(((uintptr_t)row & 15) / sizeof(T));
    count = (n + mis + VEC - 1) / VEC;
  }
  // Granules lo .. hi - 1 lie wholly within the row.
  __device__ __forceinline__ int64_t lo() const { return mis ? 1 : 0; }
  __device__ __forceinline__ int64_t hi() const { return (n + mis) / VEC; }
  __device__ __forceinline__ vec raw(int64_t j) const { return *(const vec*)(p + (j * VEC - mis)); }
  // Elements outside the row are -inf.  Returns the index of x[0].
  __device__ __forceinline__ int64_t load(int64_t j, float (&x)[VEC]) const {
    const int64_t e0 = j * VEC - mis;
    if (e0 >= 0 && e0 + VEC <= n) {
      const vec v = *(const vec*)(p + e0);
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[i] = (float)v[i];
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[i] = e0 + i >= 0 && e0 + i < n ? (float)p[e0 + i] : -INFINITY;
    }
    return e0;
  }
};

// The largest b, its low 16 bits clear, such that at least k of the lanes' 4
// values are >= b (0 if none is).
__device__ __forceinline__ uint32_t kth_largest(const uint32_t (&v)[4], int k) {
  uint32_t b = 0;
  for (int bit = 31; bit >= 16; --bit) {
    const uint32_t t = b | 1u << bit;
    int n = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) n += __builtin_popcountll(__builtin_amdgcn_ballot_w64(v[i] >= t));
    if (n >= k) b = t;
  }
  return b;
}

struct Stats {
  float M, l, t;
};
// the sums at another maximum (no smaller than s.M)
__device__ __forceinline__ void move_to(Stats& s, float M) {
  const float d = fmaxf((s.M - M) * kLog2e, -1e4f);
  const float f = __builtin_amdgcn_exp2f(d);
  s.t = f * (s.t + d * s.l);
  s.l *= f;
  s.M = M;
}

__device__ __forceinline__ void write_row(const LogprobArgs& a, int64_t row, const Stats& s, float token_logit,
                                          int64_t token) {
  const float ln = logf(s.l);
  a.entropy[row] = ln - kLn2 * s.t / s.l;
  if (a.tokens)
    a.logprob[row] = token < 0 ? 0.f : token < a.vocab ? token_logit - s.M - ln : NAN;
}

constexpr int kSlots = 8;

template <class T>
__global__ __launch_bounds__(256)
void k_logprobs(const LogprobArgs a) {
  constexpr int VEC = Row<T>::VEC;
  __shared__ u64 list[kList];
  __shared__ uint32_t slot[kSlots][256], most[256];  // largest logits, ordered
  __shared__ uint16_t todo[kSlots * 256];
  __shared__ float sh_M[4], sh_l[4], sh_t[4];
  __shared__ u64 bound;
  __shared__ int found, n_todo;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const int part = blockIdx.y;
  const Row<T> r((const T*)a.logits + row * a.stride, a.vocab);
  const int64_t g0 = part * a.granules, g1 = g0 + a.granules < r.count ? g0 + a.granules : r.count;
  // the thread's i-th granule is g0 + 256 i + tid, slot q its granules from q * size on
  const int64_t own = (g1 - g0 + 255) / 256, size = own > kSlots ? (own + kSlots - 1) / kSlots : 1;

  Stats s{kLowest, 0.f, 0.f};
  float best = -INFINITY;
  // M is the largest so far, so that no term is above 1: an M further down would
  // make the sums of a row that one logit outweighs large and cancel them in the
  // end, 2^-24 of 8 nats instead of 2^-24.  2,048 rows of 128,256 bf16 logits 114.1
  // us in a graph, 113.2 with M moved only where the maximum is 8 ahead, 120.4 with
  // one maximum for four granules.
  const auto eat = [&](const float(&x)[VEC]) {
    float m = x[0];
#pragma unroll
    for (int i = 1; i < VEC; ++i) m = fmaxf(m, x[i]);
    best = fmaxf(best, m);
    if (m > s.M) move_to(s, m);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float d = (x[i] - s.M) * kLog2e;
      const float e = __builtin_amdgcn_exp2f(d);
      s.l += e;
      s.t += e * fmaxf(d, -1e4f);
    }
  };
  uint32_t all_best = 0;
  float only[VEC];   // the granule of a thread that has one alone
  const int slots = own > 1 ? kSlots : 1;
  for (int q = 0; q < slots; ++q) {
    best = -INFINITY;
    bool any = false;
    const int64_t i1 = (q + 1) * size < own ? (q + 1) * size : own;
    for (int64_t i = q * size; i < i1; ) {
      const int64_t j = g0 + 256 * i;   // of the first thread
      if (i + 4 <= i1 && j >= r.lo() && j + 4 * 256 <= (g1 < r.hi() ? g1 : r.hi())) {
        typename Row<T>::vec v[4];      // four granules in flight
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = r.raw(j + tid + u * 256);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          float x[VEC];
#pragma unroll
          for (int k = 0; k < VEC; ++k) x[k] = (float)v[u][k];
          eat(x);
        }
        any = true;
        i += 4;
      } else {
        if (j + tid < g1) {
          r.load(j + tid, only);
          eat(only);
          any = true;
        }
        ++i;
      }
    }
    // a slot without a granule (or of NaN alone) has nothing; -inf is something
    const uint32_t o = any ? f2ord(best + 0.f) : 0;
    slot[q][tid] = o;
    all_best = max(all_best, o);
  }

  // the row's (part's) sums
  float M = wave64_reduce(s.M, OpMax());
  if (lane == 0) sh_M[wave] = M;
  most[tid] = all_best;
  if (tid == 0) found = n_todo = 0;
  __syncthreads();
  M = fmaxf(fmaxf(sh_M[0], sh_M[1]), fmaxf(sh_M[2], sh_M[3]));
  move_to(s, M);
  const float l = wave64_reduce(s.l, OpAdd()), t = wave64_reduce(s.t, OpAdd());
  if (lane == 0) {
    sh_l[wave] = l;
    sh_t[wave] = t;
  }
  u64 need = 1;
  if (a.top) {
    const uint32_t v[4] = {most[lane], most[lane + 64], most[lane + 128], most[lane + 192]};
    const uint32_t b = kth_largest(v, a.top);
    if (b) need = (u64)b << 32;
    if (own > 1)
      for (int q = 0; q < kSlots; ++q)
        if (slot[q][tid] && slot[q][tid] >= b) todo[atomicAdd(&n_todo, 1)] = (uint16_t)(q * 256 + tid);
  }
  __syncthreads();
  const Stats all{M, (sh_l[0] + sh_l[1]) + (sh_l[2] + sh_l[3]), (sh_t[0] + sh_t[1]) + (sh_t[2] + sh_t[3])};
  if (tid == 0) {
    if (a.parts == 1) {
      const int64_t tok = a.tokens ? a.tokens[row] : -1;
      write_row(a, row, all, tok >= 0 && tok < a.vocab ? (float)r.p[tok] : 0.f, tok);
    } else {
      a.ws_stats[row * a.parts + part] = make_float4(all.M, all.l, all.t, 0.f);
    }
  }
  if (a.top == 0) return;

  int n;
  for (;;) {
    const auto collect = [&](const float(&x)[VEC], int64_t e0) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const u64 key = e0 + k >= 0 && e0 + k < a.vocab ? key_of(x[k], e0 + k) : 0;
        if (key >= need) {
          const int at = atomicAdd(&found, 1);
          if (at < kList) list[at] = key;
        }
      }
    };
    if (own == 1) {
      if (all_best && all_best >= (uint32_t)(need >> 32)) collect(only, (g0 + tid) * VEC - r.mis);
    } else {
      const uint32_t per = (uint32_t)size, items = n_todo * per;  // at most the part's granules and 2,048 more
      for (uint32_t it = tid; it < items; it += 256) {
        const int w = todo[it / per];
        const int64_t i = (w >> 8) * size + it % per, j = g0 + 256 * i + (w & 255);
        if (i >= own || j >= g1) continue;
        float x[VEC];
        const int64_t e0 = r.load(j, x);
        collect(x, e0);
      }
    }
    __syncthreads();
    n = found;
    if (n <= kList) break;
    // more than fit: kList of them are in the list, and its k-th largest lies
    // above the present bound, as kList > top
    __syncthreads();
    for (int u = tid; u < kList; u += 256) {
      const u64 key = list[u];
      int rank = 0;
      for (int i = 0; i < kList; ++i) rank += list[i] > key;
      if (rank == a.top - 1) bound = key;
    }
    if (tid == 0) found = 0;
    __syncthreads();
    need = bound;
  }
  // ranks of the list's elements; what a row does not have is 0
  const float ln = logf(all.l);
  for (int u = tid; u < n + a.top; u += 256) {
    u64 key = 0;
    int rank = u;  // u >= n: the empty places behind the n elements
    if (u < n) {
      key = list[u];
      rank = 0;
      for (int i = 0; i < n; ++i) rank += list[i] > key;
    }
    if (rank >= a.top) continue;
    if (a.parts > 1) {
      a.ws_keys[(row * a.parts + part) * a.top + rank] = key;
    } else {
      a.top_ids[row * a.top + rank] = key ? index_of(key) : -1;
      a.top_logprobs[row * a.top + rank] = key ? value_of(key) - all.M - ln : NAN;
    }
  }
}

// Joins the parts of a row.  A part's keys are in descending order; the largest
// of the parts' k-th bounds the row's k-th from below, and what reaches it is
// ranked by counting.
template <class T>
__global__ __launch_bounds__(256)
void k_logprobs_join(const LogprobArgs a) {
  extern __shared__ u64 list[];  // parts * top
  __shared__ float sh[2];
  __shared__ u64 bound;
  __shared__ int found;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const int k = a.top, n = a.parts * k;
  const u64* keys = a.ws_keys + row * n;
  u64 b = 0;
  for (int p = tid; k && p < a.parts; p += 256) b = keys[p * k + k - 1];   // parts <= 64: one a thread
  const int64_t tok = a.tokens ? a.tokens[row] : -1;
  const float logit = tok >= 0 && tok < a.vocab ? (float)((const T*)a.logits)[row * a.stride + tok] : 0.f;
  if (tid == 0) found = 0;
  if (wave == 0) {
    const uint32_t top32 = (uint32_t)(b >> 32);
    // the largest b: by its value, then by its index
    uint32_t hi = top32;
#pragma unroll
    for (int o = 32; o; o >>= 1) hi = max(hi, (uint32_t)__shfl_xor((int)hi, o));
    uint32_t lo = top32 == hi ? (uint32_t)b : 0;
#pragma unroll
    for (int o = 32; o; o >>= 1) lo = max(lo, (uint32_t)__shfl_xor((int)lo, o));
    float4 f = make_float4(kLowest, 0.f, 0.f, 0.f);
    if (lane < a.parts) f = a.ws_stats[row * a.parts + lane];
    Stats s{f.x, f.y, f.z};
    const float M = wave64_reduce(s.M, OpMax());
    move_to(s, M);
    const Stats all{M, wave64_reduce(s.l, OpAdd()), wave64_reduce(s.t, OpAdd())};
    if (lane == 0) {
      write_row(a, row, all, logit, tok);
      sh[0] = all.M;
      sh[1] = all.l;
      bound = (u64)hi << 32 | lo;
    }
  }
  if (k == 0) return;
  __syncthreads();
  const u64 need = bound ? bound : 1;
  for (int u = tid; u < n; u += 256) {
    const u64 key = keys[u];
    if (key >= need) list[atomicAdd(&found, 1)] = key;
  }
  __syncthreads();
  const int have = found;
  const float M = sh[0], ln = logf(sh[1]);
  for (int u = tid; u < have + k; u += 256) {
    u64 key = 0;
    int rank = u;  // u >= have: the places behind them
    if (u < have) {
      key = list[u];
      rank = 0;
      for (int i = 0; i < have; ++i) rank += list[i] > key;
    }
    if (rank >= k) continue;
    a.top_ids[row * k + rank] = key ? index_of(key) : -1;
    a.top_logprobs[row * k + rank] = key ? value_of(key) - M - ln : NAN;
  }
}

// Parts of a row: about 1,024 workgroups in all, a granule a thread at least.
int parts_of(int64_t rows, int64_t vocab) {
  const int64_t most = (vocab / 8 + 255) / 256;
  int64_t p = 1024 / rows;
  if (p > kMaxParts) p = kMaxParts;
  if (p > most) p = most;
  return p < 1 ? 1 : (int)p;
}

// A launch has at most 2^32 - 1 threads, a row 256.
bool sizes_ok(int64_t rows, int64_t vocab, int32_t top) {
  return rows > 0 && rows < 1 << 24 && vocab > 0 && vocab <= INT32_MAX && top >= 0 && top <= kMaxTop && top <= vocab;
}

}  // namespace
}  // namespace shard

using namespace shard;

template <class T>
static void launch_logprobs(const LogprobArgs& a, int64_t rows, hipStream_t s) {
  hipLaunchKernelGGL(k_logprobs<T>, dim3((unsigned)rows, a.parts), dim3(256), 0, s, a);
  if (a.parts > 1)
    hipLaunchKernelGGL(k_logprobs_join<T>, dim3((unsigned)rows), dim3(256), a.parts * a.top * sizeof(u64), s, a);
}

extern "C" {

size_t shard_token_logprobs_workspace(int64_t rows, int64_t vocab, int32_t top) {
  if (!sizes_ok(rows, vocab, top)) return 0;
  const int parts = parts_of(rows, vocab);
  return parts == 1 ? 0 : (size_t)rows * parts * (sizeof(float4) + top * sizeof(u64));
}

int shard_token_logprobs(const void* logits, int32_t dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                         const int64_t* tokens, int32_t top, float* logprob, float* entropy, float* top_logprobs,
                         int64_t* top_ids, void* workspace, size_t workspace_bytes, void* stream) {
  if (rows == 0) return SHARD_OK;
  if (!logits || !entropy || (tokens && !logprob) || (top > 0 && (!top_logprobs || !top_ids))) return SHARD_ERR_ARG;
  if (rows < 0 || vocab <= 0 || top < 0 || row_stride < 0) return SHARD_ERR_ARG;
  if (!sizes_ok(rows, vocab, top)) return SHARD_ERR_SHAPE;
  if (dtype != SHARD_FP16 && dtype != SHARD_BF16 && dtype != SHARD_FP32) return SHARD_ERR_SHAPE;
  if ((uintptr_t)logits % (dtype == SHARD_FP32 ? 4 : 2)) return SHARD_ERR_ARG;
  LogprobArgs a{};
  a.logits = logits;
  a.vocab = vocab;
  a.stride = row_stride;
  a.tokens = tokens;
  a.top = top;
  a.parts = parts_of(rows, vocab);
  const int vec = dtype == SHARD_FP32 ? 4 : 8;
  const int64_t granules = (vocab + 2 * vec - 2) / vec;  // of the worst aligned row
  a.granules = (granules + a.parts - 1) / a.parts;
  a.logprob = logprob;
  a.entropy = entropy;
  a.top_logprobs = top_logprobs;
  a.top_ids = top_ids;
  if (a.parts > 1) {
    const size_t need = shard_token_logprobs_workspace(rows, vocab, top);
    if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16) {
      char text[96];
      snprintf(text, sizeof(text), "shard_token_logprobs needs %zu bytes of workspace, 16-byte aligned", need);
      set_last_text(text);
      return SHARD_ERR_WORKSPACE;
    }
    a.ws_stats = (float4*)workspace;
    a.ws_keys = (u64*)(a.ws_stats + rows * a.parts);
  }
  const hipStream_t s = (hipStream_t)stream;
  if (dtype == SHARD_FP16) launch_logprobs<half_t>(a, rows, s);
  else if (dtype == SHARD_BF16) launch_logprobs<bf16_t>(a, rows, s);
  else launch_logprobs<float>(a, rows, s);
  SHARD_LAUNCH_CHECK("shard_token_logprobs");
  return SHARD_OK;
}

}  // extern "C"
