// Verification of drafted tokens against a target model's logits, from given
// random numbers (speculative sampling over trees).
//
// A sequence's walk starts at its row 0.  p = softmax(logits / temperature) of the
// row it is at; s = p.  The row's children are tried in their order, child c with
// token x and random number u:
//   without draft_probs   accepted where u sum(s) < s[x]; else s[x] = 0
//   drafted from q        accepted where u q[x] sum(s) < s[x]; else
//                         s = max(s / sum(s) - q, 0), where that leaves anything
// An accepted child is where the walk goes on; where none is, the answer is the
// first token at which the running sum of s exceeds u' sum(s).  Either way the
// tokens are distributed as the target's own.  Temperature 0: p is 1 at the
// largest logit.
//
// The answers are whole numbers that sums over the vocabulary border on, so every
// weight is formed in 64 bits (2^-48 of it): 32 bits move each of 128,256 borders
// by some 2^-25, which would change about one answer in a hundred.
//
// Rows are cut into parts of at most 64, a granule pair a thread or more.
//   k_verify_stats   a part of a row a workgroup: its largest logit M and
//                    sum exp2((x - M) log2(e) / t)
//   k_verify_walk    a sequence a workgroup: the walk, then the part that the
//                    answer lies in from the parts' sums, and in it the token
// With draft_probs s is another function of every token after a rejection, so a
// launch between the two sums its parts (k_verify_rest).
#include <math.h>
#include <stdio.h>

#include "common.h"
#include "rows.h"

namespace shard {
namespace {

constexpr int kMaxParts = 64;
constexpr int kThreads = 256;
constexpr double kLog2e = 1.4426950408889634074;

struct Part {
  double sum;    // of exp2((x - most) rate); NaN where the row has no distribution
  float most;
  int32_t at;    // of the largest logit, the first of equal ones
};
struct State {   // of a sequence whose walk has ended
  double total;  // sum of the last row's weights
  float most;
  int32_t at, row, rejected;   // row -1: nothing to answer
};

struct VerifyWork {
  int parts;
  int64_t granules;  // of a part
  Part* stats;       // [row][part]
  // with draft_probs
  State* state;      // [sequence]
  double* rest;      // [sequence][part]
  int32_t* rejected; // [row]: of each sequence its rejected rows from its first row's place on
  double* left;      // [row]: what their subtraction left, 0: nothing, so it was not made
};

// 2^y, y <= 0 or NaN, to 2^-50: Taylor's series of 2^r, |r| <= 1/2 (the first
// term left out is 7e-18 of the sum).
__device__ __forceinline__ double exp2_of(double y) {
  constexpr double ln2 = 0.69314718055994530942;
  constexpr double c1 = ln2, c2 = c1 * ln2 / 2, c3 = c2 * ln2 / 3, c4 = c3 * ln2 / 4, c5 = c4 * ln2 / 5, c6 = c5 * ln2 / 6,
                   c7 = c6 * ln2 / 7, c8 = c7 * ln2 / 8, c9 = c8 * ln2 / 9, c10 = c9 * ln2 / 10, c11 = c10 * ln2 / 11,
                   c12 = c11 * ln2 / 12, c13 = c12 * ln2 / 13;
  y = y < -1100.0 ? -1100.0 : y;
  const double k = rint(y), r = y - k;
  double p = c13;
  p = fma(p, r, c12);
  p = fma(p, r, c11);
  p = fma(p, r, c10);
  p = fma(p, r, c9);
  p = fma(p, r, c8);
  p = fma(p, r, c7);
  p = fma(p, r, c6);
  p = fma(p, r, c5);
  p = fma(p, r, c4);
  p = fma(p, r, c3);
  p = fma(p, r, c2);
  p = fma(p, r, c1);
  p = fma(p, r, 1.0);
  return ldexp(p, (int)k);
}
__device__ __forceinline__ float base_of(float most) { return most == -INFINITY ? 0.f : most; }
__device__ __forceinline__ double weight(float x, float most, double rate) {
  return exp2_of(((double)x - (double)base_of(most)) * rate);
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// log2(e) / temperature of a sequence; 0: greedy.
__device__ __forceinline__ double rate_of(const shard_verify_args& a, int b) {
  const float t = a.temperatures ? a.temperatures[b] : a.temperature;
  return t > 0.f ? kLog2e / (double)t : 0.0;
}

// The sequence that row r belongs to (any, where it is nobody's).
__device__ __forceinline__ int sequence_of(const shard_verify_args& a, int r, int lane) {
  if (!a.cu_seqlens) return r;
  int before = 0;
  for (int b = 0; b < a.batch; b += 64)
    before += __builtin_popcountll(__builtin_amdgcn_ballot_w64(b + lane < a.batch && a.cu_seqlens[b + lane] <= r));
  return max(before - 1, 0);
}

template <class T>
__global__ __launch_bounds__(kThreads)
void k_verify_stats(const shard_verify_args a, const VerifyWork w) {
  constexpr int VEC = Row<T>::VEC;
  __shared__ float sh_most[4];
  __shared__ int sh_at[4];
  __shared__ double sh_sum[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x, part = blockIdx.y;
  const double rate = rate_of(a, a.temperatures ? sequence_of(a, row, lane) : 0);
  const Row<T> r((const T*)a.logits + row * a.row_stride, a.vocab);
  const int64_t g0 = part * w.granules, g1 = min(g0 + w.granules, r.count);
  float most = -INFINITY;
  int at = INT32_MAX;
  double sum = 0.0;
  for (int64_t g = g0 + 2 * tid; g < g1; g += 2 * kThreads) {
    float x[2][VEC];
    int64_t e[2];
    e[0] = r.load(g, x[0]);
    e[1] = g + 1 < g1 ? r.load(g + 1, x[1]) : 0;
    if (g + 1 >= g1)
#pragma unroll
      for (int k = 0; k < VEC; ++k) x[1][k] = -INFINITY;
    float m = most;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        if (x[u][k] > m) at = (int)(e[u] + k);
        m = fmaxf(m, x[u][k]);
      }
    if (rate > 0.0) {
      if (m > most) sum *= weight(most, m, rate);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int k = 0; k < VEC; ++k) sum += weight(x[u][k], m, rate);
    } else {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int k = 0; k < VEC; ++k) sum = x[u][k] == x[u][k] ? sum : (double)NAN;
    }
    most = m;
  }
  const float M = wave64_reduce(most, OpMax());
  if (lane == 0) sh_most[wave] = M;
  __syncthreads();
  const float all = fmaxf(fmaxf(sh_most[0], sh_most[1]), fmaxf(sh_most[2], sh_most[3]));
  if (rate > 0.0 && sum != 0.0) sum *= weight(most, all, rate);
  sum = wave_sum(sum);
  int first = most == all ? at : INT32_MAX;
#pragma unroll
  for (int o = 32; o; o >>= 1) first = min(first, __shfl_xor(first, o));
  if (lane == 0) {
    sh_sum[wave] = sum;
    sh_at[wave] = first;
  }
  __syncthreads();
  if (tid == 0) {
    Part p;
    p.sum = (sh_sum[0] + sh_sum[1]) + (sh_sum[2] + sh_sum[3]);
    p.most = all;
    p.at = min(min(sh_at[0], sh_at[1]), min(sh_at[2], sh_at[3]));
    w.stats[(int64_t)row * w.parts + part] = p;
  }
}

// A row's parts joined, in every lane of a wave; `mine` is the lane's part at the
// row's maximum.
struct Joined {
  double sum, mine;
  float most;
  int at;
};
__device__ __forceinline__ Joined join(const VerifyWork& w, int64_t row, double rate, int lane) {
  Part p{0.0, -INFINITY, INT32_MAX};
  if (lane < w.parts) p = w.stats[row * w.parts + lane];
  Joined j;
  j.most = wave64_reduce(p.most, OpMax());
  int at = p.most == j.most ? p.at : INT32_MAX;
#pragma unroll
  for (int o = 32; o; o >>= 1) at = min(at, __shfl_xor(at, o));
  j.at = at;
  j.mine = rate > 0.0 && p.sum != 0.0 ? p.sum * weight(p.most, j.most, rate) : p.sum;
  j.sum = wave_sum(j.mine);
  return j;
}

// What a sequence's walk needs of its rows.
struct Nodes {
  int32_t up[SHARD_TREE_ROWS], token[SHARD_TREE_ROWS];   // token -1: none of the vocabulary
  float u[SHARD_TREE_ROWS], logit[SHARD_TREE_ROWS];      // of the token in its parent's row
  int32_t rejected[SHARD_TREE_ROWS];                     // rows, in their order
  double amount[SHARD_TREE_ROWS];                        // weights of their tokens; draft_probs: what they left
};

// s of a token before any normalisation by sums that are not known yet: the weight
// w / total, less the first n rejected rows' probabilities, each difference again
// relative to what it left.
template <class F>
__device__ __forceinline__ double residual(double s, const double* left, int n, F q) {
  for (int k = 0; k < n; ++k) {
    const double d = s - q(k);
    if (k == n - 1) return d > 0.0 ? d : 0.0;
    if (left[k] > 0.0) s = (d > 0.0 ? d : 0.0) / left[k];
  }
  return s;
}

struct Shared {
  Nodes n;
  double scan[4];
  State end;
  int count, pick_part, found, last;
  double before, target;
};

// The weights of a pair of granules of a row, 0 outside it.
template <class T, bool Q>
struct Weights {
  static constexpr int VEC = Row<T>::VEC;
  const shard_verify_args& a;
  const Row<T>& r;
  const Shared& sh;
  const int64_t row0;
  const double rate;
  int n;          // rejected rows that count
  __device__ __forceinline__ double pair(int64_t g, int64_t g1, double (&v)[2][VEC], int64_t (&e)[2]) const {
    double sum = 0.0;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float x[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) x[k] = -INFINITY;
      e[u] = g + u < g1 ? r.load(g + u, x) : -VEC;
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        double s = weight(x[k], sh.end.most, rate);
        const int64_t i = e[u] + k;
        if constexpr (Q) {
          if (i >= 0 && i < a.vocab)
            s = residual(s / sh.end.total, sh.n.amount, n,
                         [&](int j) { return (double)a.draft_probs[(row0 + sh.n.rejected[j]) * a.probs_stride + i]; });
        } else {
          for (int j = 0; j < n; ++j)
            if (sh.n.token[sh.n.rejected[j]] == i) s = 0.0;
        }
        v[u][k] = s;
        sum += s;
      }
    }
    return sum;
  }
};

// Sums over a workgroup: every thread's exclusive prefix, and the whole.
__device__ __forceinline__ double scan(double v, Shared& sh, double& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 63) sh.scan[wave] = x;
  __syncthreads();
  double before = 0.0;
  for (int k = 0; k < wave; ++k) before += sh.scan[k];
  all = (sh.scan[0] + sh.scan[1]) + (sh.scan[2] + sh.scan[3]);
  return before + (x - v);
}

// The walk.  Wave 0 decides; for Q, where sums over a row take the whole workgroup,
// every wave decides, from the same numbers in the same way.  Leaves sh.end, the
// rejected rows of the last row, and for Q what each but the last left.
template <class T, bool Q>
__device__ void walk(const shard_verify_args& a, const VerifyWork& w, Shared& sh, int b, bool write) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int c0 = b, c1 = b + 1;
  if (a.cu_seqlens) {
    c0 = a.cu_seqlens[b];
    c1 = a.cu_seqlens[b + 1];
  }
  c0 = min(max(c0, 0), a.n_tokens);
  c1 = min(max(c1, c0), a.n_tokens);
  const int n = min(c1 - c0, min(a.width, SHARD_TREE_ROWS));
  const double rate = rate_of(a, b);
  const T* logits = (const T*)a.logits + c0 * a.row_stride;
  for (int i = tid; i < n; i += kThreads) {
    const int p = a.parents[c0 + i];
    const int64_t t = a.tokens[c0 + i];
    const bool ok = p >= 0 && p < i && t >= 0 && t < a.vocab;
    sh.n.up[i] = p >= 0 && p < i ? p : -1;
    sh.n.token[i] = ok ? (int32_t)t : -1;
    sh.n.u[i] = a.uniforms[2 * (int64_t)(c0 + i)];
    sh.n.logit[i] = ok ? (float)logits[p * a.row_stride + t] : -INFINITY;
  }
  __syncthreads();
  int cur = 0, count = n > 0 ? 1 : 0, rejected = 0;
  int32_t* path = a.path + (int64_t)b * a.width;
  double total = 0.0;
  float most = 0.f;
  int at = -1;
  bool none = n == 0;
  // one row a turn; for Q a turn ends as well where a sum over the row is needed
  while ((Q || wave == 0) && !none) {
    const Joined j = join(w, c0 + cur, rate, lane);
    most = j.most;
    at = j.at;
    total = j.sum;
    rejected = 0;
    if (most == -INFINITY || !(total >= 0.0) || total == INFINITY) {   // no distribution
      none = true;
      break;
    }
    if (count > a.max_depth) break;
    double sum = total;     // of s; Q: of s / total, 1
    if (Q) sum = 1.0;
    int chosen = -1;
    for (int base = (cur + 1) & ~63; base < n && chosen < 0; base += 64) {
      const int i = base + lane;
      const bool child = i < n && sh.n.up[i] == cur;
      uint64_t todo = __builtin_amdgcn_ballot_w64(child);
      const double e = child && sh.n.token[i] >= 0 ? weight(sh.n.logit[i], most, rate) : 0.0;
      for (; todo && chosen < 0; todo &= todo - 1) {
        const int bit = __builtin_ctzll(todo), c = base + bit;
        const int token = sh.n.token[c];
        const double mine = __shfl(e, bit), u = (double)sh.n.u[c];
        if (token < 0) continue;
        if (rate == 0.0) {
          if (token == at) chosen = c;
          continue;
        }
        if constexpr (Q) {
          const auto q = [&](int k) {
            return (double)a.draft_probs[(int64_t)(c0 + (k < rejected ? sh.n.rejected[k] : c)) * a.probs_stride + token];
          };
          if (rejected) {   // what the last rejection left, which nobody has summed yet
            if (tid == 0) {
              sh.end.total = total;
              sh.end.most = most;
            }
            __syncthreads();
            const Row<T> r(logits + (int64_t)cur * a.row_stride, a.vocab);
            const Weights<T, Q> weights{a, r, sh, c0, rate, rejected};
            double own = 0.0;
            for (int64_t g = 2 * tid; g < r.count; g += 2 * kThreads) {
              double v[2][Row<T>::VEC];
              int64_t el[2];
              own += weights.pair(g, r.count, v, el);
            }
            double all;
            scan(own, sh, all);
            __syncthreads();
            if (tid == 0) sh.n.amount[rejected - 1] = all;
            __syncthreads();
          }
          double s = mine / total;
          for (int k = 0; k < rejected; ++k)
            if (sh.n.amount[k] > 0.0) {
              const double d = s - q(k);
              s = (d > 0.0 ? d : 0.0) / sh.n.amount[k];
            }
          if (u * q(rejected) < s) chosen = c;
          else {
            __syncthreads();
            if (tid == 0) sh.n.rejected[rejected] = c;
            ++rejected;
            __syncthreads();
          }
        } else {
          // a token that a sibling before has had rejected has nothing left
          bool again = false;
          for (int k = lane; k < rejected; k += 64) again |= sh.n.token[sh.n.rejected[k]] == token;
          if (__builtin_amdgcn_ballot_w64(again)) continue;
          if (u * sum < mine) chosen = c;
          else {
            if (lane == 0) {
              sh.n.rejected[rejected] = c;
              sh.n.amount[rejected] = mine;
            }
            ++rejected;
            sum -= mine;
          }
        }
      }
    }
    if (chosen < 0) break;
    cur = chosen;
    if (write && tid == 0 && count < a.width) path[count] = cur;
    ++count;
  }
  __syncthreads();
  if (tid == 0) {
    sh.end.total = total;
    sh.end.most = most;
    sh.end.at = at;
    sh.end.row = none ? -1 : c0 + cur;
    sh.end.rejected = rejected;
    sh.count = count;
    if (write) {
      a.counts[b] = count;
      if (n > 0) path[0] = 0;
    }
  }
  __syncthreads();
  if (write)
    for (int i = sh.count + tid; i < a.width; i += kThreads) path[i] = -1;
}

template <class T>
__global__ __launch_bounds__(kThreads)
void k_verify_rest(const shard_verify_args a, const VerifyWork w) {
  __shared__ Shared sh;
  const int tid = threadIdx.x, part = blockIdx.x, b = blockIdx.y;
  walk<T, true>(a, w, sh, b, part == 0);
  const State end = sh.end;
  int c0 = a.cu_seqlens ? min(max(a.cu_seqlens[b], 0), a.n_tokens) : b;
  if (part == 0) {
    if (tid == 0) w.state[b] = end;
    for (int k = tid; k < end.rejected; k += kThreads) {
      w.rejected[c0 + k] = sh.n.rejected[k];
      w.left[c0 + k] = k < end.rejected - 1 ? sh.n.amount[k] : 0.0;
    }
  }
  const double rate = rate_of(a, b);
  if (end.row < 0 || rate == 0.0) return;
  const Row<T> r((const T*)a.logits + (int64_t)end.row * a.row_stride, a.vocab);
  const Weights<T, true> weights{a, r, sh, c0, rate, end.rejected};
  const int64_t g0 = part * w.granules, g1 = min(g0 + w.granules, r.count);
  double own = 0.0;
  for (int64_t g = g0 + 2 * tid; g < g1; g += 2 * kThreads) {
    double v[2][Row<T>::VEC];
    int64_t e[2];
    own += weights.pair(g, g1, v, e);
  }
  double all;
  scan(own, sh, all);
  if (tid == 0) w.rest[(int64_t)b * w.parts + part] = all;
}

// The walk (Q: its state) and the answer.
template <class T, bool Q>
__global__ __launch_bounds__(kThreads)
void k_verify_walk(const shard_verify_args a, const VerifyWork w) {
  constexpr int VEC = Row<T>::VEC;
  __shared__ Shared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = blockIdx.x;
  const int c0 = a.cu_seqlens ? min(max(a.cu_seqlens[b], 0), a.n_tokens) : b;
  const double rate = rate_of(a, b);
  if constexpr (Q) {
    const State end = w.state[b];
    if (tid == 0) sh.end = end;
    for (int k = tid; k < end.rejected; k += kThreads) {
      sh.n.rejected[k] = w.rejected[c0 + k];
      sh.n.amount[k] = w.left[c0 + k];
    }
    __syncthreads();
  } else {
    walk<T, false>(a, w, sh, b, true);
  }
  const State end = sh.end;
  if (end.row < 0 || rate == 0.0) {
    if (tid == 0) a.next[b] = end.row < 0 ? -1 : end.at;
    return;
  }
  const Row<T> r((const T*)a.logits + (int64_t)end.row * a.row_stride, a.vocab);
  int rejected = end.rejected;
  const float u = a.uniforms[2 * (int64_t)end.row + 1];
  // the part that the answer lies in
  if (wave == 0) {
    double v;
    if constexpr (Q) {
      v = lane < w.parts ? w.rest[(int64_t)b * w.parts + lane] : 0.0;
    } else {
      v = join(w, end.row, rate, lane).mine;
      for (int k = 0; k < rejected; ++k) {
        const int64_t g = (sh.n.token[sh.n.rejected[k]] + r.mis) / VEC;
        if (g / w.granules == lane) v -= sh.n.amount[k];
      }
      v = v > 0.0 ? v : 0.0;
    }
    double x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double y = __shfl_up(x, o);
      if (lane >= o) x += y;
    }
    const double total = __shfl(x, 63), target = (double)u * total;
    const uint64_t over = __builtin_amdgcn_ballot_w64(x > target), some = __builtin_amdgcn_ballot_w64(v > 0.0);
    const int p = over ? __builtin_ctzll(over) : some ? 63 - __builtin_clzll(some) : -1;
    const double before = __shfl(x - v, max(p, 0));
    if (lane == 0) {
      sh.pick_part = p;
      sh.target = target - before;
      sh.found = INT32_MAX;
      sh.last = -1;
    }
  }
  __syncthreads();
  int64_t g0 = sh.pick_part * w.granules, g1 = min(g0 + w.granules, r.count);
  double target = sh.target;
  if (sh.pick_part < 0) {   // nothing is left of s
    if (!Q || rejected == 0) {
      if (tid == 0) a.next[b] = end.at;
      return;
    }
    // the last subtraction is not made; its row as a whole
    do --rejected;
    while (rejected && !(sh.n.amount[rejected - 1] > 0.0));
    g0 = 0;
    g1 = r.count;
    const Weights<T, Q> weights{a, r, sh, c0, rate, rejected};
    double own = 0.0, all;
    for (int64_t g = g0 + 2 * tid; g < g1; g += 2 * kThreads) {
      double v[2][VEC];
      int64_t e[2];
      own += weights.pair(g, g1, v, e);
    }
    scan(own, sh, all);
    target = (double)u * all;
  }
  const Weights<T, Q> weights{a, r, sh, c0, rate, rejected};
  double base = 0.0;
  for (int64_t at = g0; at < g1; at += 2 * kThreads) {
    double v[2][VEC], all;
    int64_t e[2];
    const double own = weights.pair(at + 2 * tid, g1, v, e);
    double run = base + scan(own, sh, all);
    // the first element at which the running sum is above the target, else the last that has any
    int pick = -1, some = -1;
#pragma unroll
    for (int k = 0; k < 2 * VEC; ++k) {
      const double s = v[k / VEC][k % VEC];
      run += s;
      if (s > 0.0) {
        some = (int)(e[k / VEC] + k % VEC);
        if (run > target && pick < 0) pick = some;
      }
    }
    if (pick >= 0) atomicMin(&sh.found, pick);
    if (some >= 0) atomicMax(&sh.last, some);
    __syncthreads();
    if (sh.found != INT32_MAX) break;
    base += all;
    __syncthreads();
  }
  __syncthreads();
  if (tid == 0) a.next[b] = sh.found != INT32_MAX ? sh.found : sh.last >= 0 ? sh.last : end.at;
}

// --------------------------------------------------------------------------
// host side
// --------------------------------------------------------------------------
bool plan(const shard_verify_args* a, VerifyWork& w, size_t& bytes) {
  if (a->n_tokens < 0 || a->n_tokens >= 1 << 24 || a->batch <= 0 || a->batch > 65535 || a->vocab <= 0 || a->vocab >= INT32_MAX - 64)
    return false;
  if (a->dtype != SHARD_FP16 && a->dtype != SHARD_BF16 && a->dtype != SHARD_FP32) return false;
  const int vec = a->dtype == SHARD_FP32 ? 4 : 8;
  const int64_t granules = (a->vocab + 2 * vec - 2) / vec;          // of the worst aligned row
  const int64_t parts = (granules + 2 * kThreads - 1) / (2 * kThreads);
  w.parts = (int)(parts < kMaxParts ? parts : kMaxParts);
  w.granules = (granules + w.parts - 1) / w.parts;
  w.granules += w.granules & 1;
  bytes = (size_t)a->n_tokens * w.parts * sizeof(Part);
  if (a->draft_probs)
    bytes += (size_t)a->batch * (sizeof(State) + w.parts * sizeof(double)) + (size_t)a->n_tokens * (sizeof(double) + sizeof(int32_t));
  return true;
}

}  // namespace
}  // namespace shard

using namespace shard;

template <class T>
static void launch_verify(const shard_verify_args& a, const VerifyWork& w, hipStream_t s) {
  hipLaunchKernelGGL(k_verify_stats<T>, dim3((unsigned)a.n_tokens, w.parts), dim3(kThreads), 0, s, a, w);
  if (a.draft_probs) {
    hipLaunchKernelGGL(k_verify_rest<T>, dim3(w.parts, a.batch), dim3(kThreads), 0, s, a, w);
    hipLaunchKernelGGL((k_verify_walk<T, true>), dim3(a.batch), dim3(kThreads), 0, s, a, w);
  } else {
    hipLaunchKernelGGL((k_verify_walk<T, false>), dim3(a.batch), dim3(kThreads), 0, s, a, w);
  }
}

extern "C" {

size_t shard_verify_args_size(void) { return sizeof(shard_verify_args); }

size_t shard_verify_drafts_workspace(const shard_verify_args* a) {
  VerifyWork w{};
  size_t bytes = 0;
  return a && plan(a, w, bytes) ? bytes : 0;
}

int shard_verify_drafts(const shard_verify_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (!a || !a->logits || !a->tokens || !a->parents || !a->uniforms || !a->path || !a->counts || !a->next) return SHARD_ERR_ARG;
  if (a->batch <= 0 || a->n_tokens < 0 || a->vocab <= 0 || a->width <= 0 || a->max_depth < 0 || a->row_stride < 0) return SHARD_ERR_ARG;
  if (!a->cu_seqlens && a->n_tokens != a->batch) return SHARD_ERR_ARG;
  if (a->draft_probs && (a->probs_stride < 0 || (uintptr_t)a->draft_probs % 4)) return SHARD_ERR_ARG;
  if (!a->temperatures && !(a->temperature >= 0.f && a->temperature < INFINITY)) return SHARD_ERR_ARG;
  VerifyWork w{};
  size_t need = 0;
  if (a->width > SHARD_TREE_ROWS || !plan(a, w, need)) return SHARD_ERR_SHAPE;
  if ((uintptr_t)a->logits % (a->dtype == SHARD_FP32 ? 4 : 2)) return SHARD_ERR_ARG;
  if (a->n_tokens && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)) {
    char text[96];
    snprintf(text, sizeof(text), "shard_verify_drafts needs %zu bytes of workspace, 16-byte aligned", need);
    set_last_text(text);
    return SHARD_ERR_WORKSPACE;
  }
  w.stats = (Part*)workspace;
  if (a->draft_probs) {
    w.state = (State*)(w.stats + (size_t)a->n_tokens * w.parts);
    w.rest = (double*)(w.state + a->batch);
    w.left = w.rest + (size_t)a->batch * w.parts;
    w.rejected = (int32_t*)(w.left + a->n_tokens);
  }
  const hipStream_t s = (hipStream_t)stream;
  if (a->n_tokens == 0) {
    // sequences of no rows: nothing is read
    hipLaunchKernelGGL((k_verify_walk<half_t, false>), dim3(a->batch), dim3(kThreads), 0, s, *a, w);
  } else if (a->dtype == SHARD_FP16) {
    launch_verify<half_t>(*a, w, s);
  } else if (a->dtype == SHARD_BF16) {
    launch_verify<bf16_t>(*a, w, s);
  } else {
    launch_verify<float>(*a, w, s);
  }
  SHARD_LAUNCH_CHECK("shard_verify_drafts");
  return SHARD_OK;
}

}  // extern "C"
