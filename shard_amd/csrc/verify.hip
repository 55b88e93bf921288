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
// Rows are cut into at most 64 parts.
//   k_verify_stats   a part of a row a wave: its largest logit M and
//                    sum exp2((x - M) log2(e) / t)
//   k_verify_walk    a sequence a workgroup: the walk, which takes rejected tokens
//                    out of the parts' sums (kVague), then the part that the
//                    answer lies in from those sums, and in it the token
// With draft_probs s is another function of every token after a rejection: the walk
// leaves its sum to k_verify_rest, which has the whole chip, and goes on in the next
// launch; k_verify_answer finds the token.  Many
// rows, few of which are on a path, go a launch a level instead (k_verify_level,
// k_verify_end), and only the rows on the paths are read.
//
// Measured, 128,256 logits a row, us: 5 rows of one sequence 4.9 + 5.8 (a chain of
// loads and reductions), 61 rows 10.3 + 7.0; 192 rows of 32 sequences with draft_probs
// 26 (vector issue: 20 64-bit instructions a weight) + 9 + 12 + 5; 1,190 rows of 64
// trees, 7 levels 1.7 to 7 each, the end 7.7.
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
  double sum;    // of exp2((x - most) rate)
  float most;    // the largest logit, NaN where one is
  int32_t at;    // greedy: of the largest logit, the first of equal ones
};
struct State {   // of a sequence whose walk has ended, or wants a sum
  double total;  // sum of the last row's weights
  float most;
  int32_t at, row, rejected;   // row -1: nothing to answer
  int32_t count, wants, round; // of the path; wants what its rejections have left; when it was written
};

struct Level {   // of a sequence's walk, a launch a level
  int32_t row, count, done;    // done: the level at which it was seen to end, or 0
};

struct VerifyWork {
  int levels;        // launches of a level each, 0: all rows at once
  int parts;
  int64_t granules;  // of a part
  Part* stats;       // [row][part]
  Level* level;      // [2][sequence]; stats: [2][sequence][part]
  // with draft_probs
  State* state;      // [sequence]
  double* rest;      // [sequence][part]
  int32_t* rejected; // [row]: of each sequence its rejected rows from its first row's place on
  double* left;      // [row]: what their subtraction left, 0: nothing, so it was not made
};

// 2^y to 2^-51, 0 below 2^-1074; y <= 1, a number or -inf.  y is split at the
// nearest whole number, whose bits the addition of 1.5 2^52 leaves in the low word;
// the polynomial is 2^r's interpolation at Chebyshev's points of [-1/2, 1/2],
// 3.2e-16 off at most.
__device__ __forceinline__ double exp2_of(double y) {
  constexpr double whole = 6755399441055744.0;
  y = fmax(y, -1100.0);
  const double t = y + whole;
  const double r = y - (t - whole);
  double p = 7.072585949269223e-09;
  p = fma(p, r, 1.0208690299958306e-07);
  p = fma(p, r, 1.321544258792169e-06);
  p = fma(p, r, 1.5252657260200837e-05);
  p = fma(p, r, 0.0001540353044173605);
  p = fma(p, r, 0.0013333558230164974);
  p = fma(p, r, 0.009618129107606888);
  p = fma(p, r, 0.05550410866444772);
  p = fma(p, r, 0.24022650695910097);
  p = fma(p, r, 0.69314718055995);
  p = fma(p, r, 1.0);
  return ldexp(p, __double2loint(t));
}
// A row's (or part's) weights 2^((x - most) rate), x not NaN.  The difference comes
// first: it is exact, or rounded relative to itself, however far from 0 the row lies.
struct Scale {
  double rate, from;
  __device__ __forceinline__ Scale(float most, double rate) : rate(rate), from(most == -INFINITY ? 0.0 : (double)most) {}
  __device__ __forceinline__ double operator()(float x) const { return exp2_of(((double)x - from) * rate); }
};

// Lanes' values without the LDS crossbar.
template <int CTRL>
__device__ __forceinline__ double dpp_mov(double v) {
  const int lo = __builtin_amdgcn_mov_dpp(__double2loint(v), CTRL, 0xF, 0xF, false);
  const int hi = __builtin_amdgcn_mov_dpp(__double2hiint(v), CTRL, 0xF, 0xF, false);
  return __hiloint2double(hi, lo);
}
__device__ __forceinline__ double wave_sum(double v) {
  v += dpp_mov<kDppXor1>(v);
  v += dpp_mov<kDppXor2>(v);
  v += dpp_mov<kDppHalfMirror>(v);
  v += dpp_mov<kDppMirror>(v);
  {
    const auto lo = __builtin_amdgcn_permlane16_swap(__double2loint(v), __double2loint(v), false, false);
    const auto hi = __builtin_amdgcn_permlane16_swap(__double2hiint(v), __double2hiint(v), false, false);
    v = __hiloint2double(hi[0], lo[0]) + __hiloint2double(hi[1], lo[1]);
  }
  const auto lo = __builtin_amdgcn_permlane32_swap(__double2loint(v), __double2loint(v), false, false);
  const auto hi = __builtin_amdgcn_permlane32_swap(__double2hiint(v), __double2hiint(v), false, false);
  return __hiloint2double(hi[0], lo[0]) + __hiloint2double(hi[1], lo[1]);
}
// A lane's sum of the lanes up to it.
template <int CTRL, int ROWS>
__device__ __forceinline__ double moved(double v) {   // 0 where nothing comes in
  const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, ROWS, 0xF, false);
  const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, ROWS, 0xF, false);
  return __hiloint2double(hi, lo);
}
__device__ __forceinline__ double wave_scan(double v) {
  v += moved<0x111, 0xF>(v);   // within rows of 16: from 1, 2, 4, 8 lanes below
  v += moved<0x112, 0xF>(v);
  v += moved<0x114, 0xF>(v);
  v += moved<0x118, 0xF>(v);
  v += moved<0x142, 0xA>(v);   // the last lane of rows 0 and 2 to rows 1 and 3
  v += moved<0x143, 0xC>(v);   // lane 31 to the upper half
  return v;
}
__device__ __forceinline__ double lane_value(double v, int lane) {   // lane is the same in all
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), lane), __builtin_amdgcn_readlane(__double2loint(v), lane));
}
__device__ __forceinline__ float max_of(float a, float b) { return __builtin_elementwise_maximum(a, b); }   // NaN stays
struct OpMaxOf { __device__ float operator()(float a, float b) const { return max_of(a, b); } };
// A row's largest logit says whether it has a distribution: a greedy one may be +inf.
__device__ __forceinline__ bool has_answer(float most, double rate) { return most > -INFINITY && (most < INFINITY || rate == 0.0); }

// log2(e) / temperature of a sequence; 0: greedy.  An infinite temperature leaves a
// rate that tells masked tokens from the others.
__device__ __forceinline__ double rate_of(const shard_verify_args& a, int b) {
  const float t = a.temperatures ? a.temperatures[b] : a.temperature;
  return t > 0.f ? fmax(kLog2e / (double)t, 1e-300) : 0.0;
}

// The sequence that row r belongs to (any, where it is nobody's).
__device__ __forceinline__ int sequence_of(const shard_verify_args& a, int r, int lane) {
  if (!a.cu_seqlens) return r;
  int before = 0;
  for (int b = 0; b < a.batch; b += 64)
    before += __builtin_popcountll(__builtin_amdgcn_ballot_w64(b + lane < a.batch && a.cu_seqlens[b + lane] <= r));
  return max(before - 1, 0);
}

// A part a wave: no barrier, nothing in LDS.  kTurn granules a turn; one that lies wholly
// within the part and the row is on its way before the first is looked at.  Any other
// (every one of half-precision rows below 131,072 logits: a part has 251 granules at 128,256)
// is loaded granule by granule and filled up with -inf, whose weights take as long as
// others: 2% more at 128,256, twice as many between 32,000 and 65,536, 1.7 times at 151,936.
constexpr int kTurn = 256;

template <class T>
__device__ __forceinline__ void part_of(const shard_verify_args& a, const VerifyWork& w, int row, int part, int sequence, Part* out) {
  constexpr int VEC = Row<T>::VEC, PER = kTurn / 64;
  const int lane = threadIdx.x & 63;
  const Row<T> r((const T*)a.logits + row * a.row_stride, a.vocab);
  const int64_t g0 = part * w.granules, g1 = min(g0 + w.granules, r.count);
  float most = -INFINITY;
  int at = INT32_MAX;
  double sum = 0.0, rate = -1.0;
  for (int64_t g = g0; g < g1; g += kTurn) {
    typename Row<T>::vec raw[PER];
    if (g >= r.lo() && g + kTurn <= min(g1, r.hi())) {
#pragma unroll
      for (int u = 0; u < PER; ++u) raw[u] = r.raw(g + 64 * u + lane);
    } else {
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        float x[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) x[k] = -INFINITY;
        if (g + 64 * u + lane < g1) r.load(g + 64 * u + lane, x);
#pragma unroll
        for (int k = 0; k < VEC; ++k) raw[u][k] = (T)x[k];   // as it was
      }
    }
    if (rate < 0.0) rate = rate_of(a, !a.temperatures ? 0 : sequence < 0 ? sequence_of(a, row, lane) : sequence);
    float m = most;
#pragma unroll
    for (int u = 0; u < PER; ++u)
#pragma unroll
      for (int k = 0; k < VEC; ++k) m = max_of(m, (float)raw[u][k]);
    m = wave64_reduce(m, OpMaxOf());
    // the logits are kept in their own type, half the registers, and widened again
#pragma unroll
    for (int u = 0; u < PER; ++u) asm volatile("" : "+v"(raw[u]));
    if (rate > 0.0) {
      const Scale scale(m, rate);
      if (g > g0) sum *= scale(most);
#pragma unroll
      for (int u = 0; u < PER; ++u)
#pragma unroll
        for (int k = 0; k < VEC; ++k) sum += scale((float)raw[u][k]);
    } else if (m > most) {
      at = INT32_MAX;
#pragma unroll
      for (int u = PER - 1; u >= 0; --u)
#pragma unroll
        for (int k = VEC - 1; k >= 0; --k)
          if ((float)raw[u][k] == m) at = (int)((g + 64 * u + lane) * VEC - r.mis + k);
    }
    most = m;
  }
  sum = wave_sum(sum);
  if (rate == 0.0)
#pragma unroll
    for (int o = 32; o; o >>= 1) at = min(at, __shfl_xor(at, o));
  if (lane == 0) *out = Part{sum, most, at};
}

template <class T>
__global__ __launch_bounds__(kThreads)
void k_verify_stats(const shard_verify_args a, const VerifyWork w) {
  const int part = blockIdx.y * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (part < w.parts) part_of<T>(a, w, blockIdx.x, part, -1, w.stats + (int64_t)blockIdx.x * w.parts + part);
}

// A row's parts joined, in every lane of a wave; `mine` is the lane's part at the
// row's maximum.
struct Joined {
  double sum, mine;
  float most;
  int at;
};
__device__ __forceinline__ Joined join(const Part* row, int parts, double rate, int lane) {
  Part p{0.0, -INFINITY, INT32_MAX};
  if (lane < parts) p = row[lane];
  Joined j;
  j.most = wave64_reduce(p.most, OpMaxOf());
  int at = INT32_MAX;
  if (rate == 0.0) {
    at = p.most == j.most ? p.at : INT32_MAX;
#pragma unroll
    for (int o = 32; o; o >>= 1) at = min(at, __shfl_xor(at, o));
  }
  j.at = at;
  j.mine = p.sum != 0.0 ? p.sum * Scale(j.most, rate)(p.most) : 0.0;
  j.sum = wave_sum(j.mine);
  return j;
}

// What a sequence's walk needs of its rows.
constexpr int kWalk = 1024;                              // threads of a walk, a row each
constexpr int kHeld = 2048;                              // parts of rows in LDS, where a sequence has no more
static_assert(SHARD_TREE_ROWS <= kWalk, "a thread a row");
struct Nodes {
  int32_t up[SHARD_TREE_ROWS], token[SHARD_TREE_ROWS];   // token -1: none of the vocabulary
  float u[SHARD_TREE_ROWS], after[SHARD_TREE_ROWS];      // random numbers
  float logit[SHARD_TREE_ROWS];                          // of the token in its parent's row
  float q[SHARD_TREE_ROWS];                              // of the token in what it was drawn from
};

struct Shared {
  int32_t rejected[SHARD_TREE_ROWS];                     // rows (Q) or tokens, in their order
  double amount[SHARD_TREE_ROWS];                        // Q: what they left
  double scan[kWalk / 64];
  State end;
  int count, pick_part, found, last;
  float u;
  double target;
};

// s of a row's tokens four at a time, 0 outside it: quad i holds elements 4 i - mis ..
// 4 i - mis + 3.  Q: the weights' shares, less the first n rejected rows'
// probabilities, each difference again relative to what it left, the last one as it is.
template <class T, bool Q>
struct Weights {
  const shard_verify_args& a;
  const Row<T> r;
  const Shared& sh;
  const int64_t row0;
  const Scale scale;
  const double each;
  int n;          // rejected rows that count
  __device__ __forceinline__ Weights(const shard_verify_args& a, const Shared& sh, int64_t row0, int64_t row, float most, double total,
                                     double rate, int n)
      : a(a), r((const T*)a.logits + row * a.row_stride, a.vocab), sh(sh), row0(row0), scale(most, rate), each(1.0 / total), n(n) {}
  struct Raw {
    float x[4], q[4];   // q: of the first rejected row
    int64_t e;          // the first element's index; all four lie in the row
    bool whole;
  };
  __device__ __forceinline__ void probs(int j, const Raw& raw, float (&q)[4]) const {
    const float* p = a.draft_probs + (row0 + sh.rejected[j]) * a.probs_stride + raw.e;
    if (raw.whole) {
#pragma unroll
      for (int k = 0; k < 4; ++k) q[k] = p[k];
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) q[k] = raw.e + k >= 0 && raw.e + k < r.n ? p[k] : 0.f;
    }
  }
  __device__ __forceinline__ Raw fetch(int64_t i, int64_t end) const {
    typedef T vec4 __attribute__((ext_vector_type(4)));
    Raw raw;
    raw.e = i < end ? 4 * i - r.mis : -4;
    raw.whole = raw.e >= 0 && raw.e + 4 <= r.n;
    if (raw.whole) {
      const vec4 v = *(const vec4*)(r.p + raw.e);
#pragma unroll
      for (int k = 0; k < 4; ++k) raw.x[k] = (float)v[k];
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) raw.x[k] = raw.e + k >= 0 && raw.e + k < r.n ? (float)r.p[raw.e + k] : -INFINITY;
    }
    if (Q && n > 0) probs(0, raw, raw.q);
    return raw;
  }
  // s of U quads, a rejected row for all of them after the other
  template <int U>
  __device__ __forceinline__ double values(Raw (&raw)[U], double (&v)[U][4]) const {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < 4; ++k) v[u][k] = scale(raw[u].x[k]);
    if constexpr (Q) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < 4; ++k) v[u][k] *= each;
      for (int j = 0; j < n; ++j) {
        const double left = j == n - 1 ? 1.0 : sh.amount[j], part = 1.0 / left;
        if (j)
#pragma unroll
          for (int u = 0; u < U; ++u) probs(j, raw[u], raw[u].q);
        if (left > 0.0)
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const double d = v[u][k] - (double)raw[u].q[k];
              v[u][k] = (d > 0.0 ? d : 0.0) * part;
            }
      }
    } else {
      for (int j = 0; j < n; ++j) {
        const int64_t token = sh.rejected[j];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int k = 0; k < 4; ++k) v[u][k] = token - raw[u].e == k ? 0.0 : v[u][k];
      }
    }
    double sum = 0.0;
#pragma unroll
    for (int u = 0; u < U; ++u) sum += (v[u][0] + v[u][1]) + (v[u][2] + v[u][3]);
    return sum;
  }
  // a part's quads
  __device__ __forceinline__ int64_t begin(const VerifyWork& w, int64_t part) const { return part * w.granules * (Row<T>::VEC / 4); }
  __device__ __forceinline__ int64_t end(const VerifyWork& w, int64_t part) const {
    return min((part + 1) * w.granules, r.count) * (Row<T>::VEC / 4);
  }
  // of quads i0 + `at`, i0 + at + stride, ..., U of them on their way together
  template <int U>
  __device__ __forceinline__ double sum(int64_t i0, int64_t i1, int at, int stride) const {
    double own = 0.0;
#pragma unroll 1
    for (int64_t i = i0; i < i1; i += U * stride) {
      Raw raw[U];
      double v[U][4];
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = fetch(i + u * stride + at, i1);
      own += values(raw, v);
    }
    return own;
  }
};

// Sums over a workgroup of kWalk threads: every thread's exclusive prefix, and the whole.
__device__ __forceinline__ double scan(double v, Shared& sh, double& all) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const double x = wave_scan(v);
  __syncthreads();
  if (lane == 63) sh.scan[wave] = x;
  __syncthreads();
  const double waves = wave_scan(lane < kWalk / 64 ? sh.scan[lane] : 0.0);
  all = lane_value(waves, kWalk / 64 - 1);
  return (wave ? lane_value(waves, max(wave - 1, 0)) : 0.0) + (x - v);
}

// The sum of a row's weights.
template <class T, bool Q>
__device__ __forceinline__ double sum_of(const Weights<T, Q>& weights, int64_t i0, int64_t i1, Shared& sh) {
  double all;
  const double own = weights.template sum<Q ? 3 : 4>(i0, i1, threadIdx.x, kWalk);   // 4 with Q: spills
  scan(own, sh, all);
  return all;
}

struct Rows {
  int first, n;   // of a sequence that are looked at
};
__device__ __forceinline__ Rows rows_of(const shard_verify_args& a, int b) {
  int c0 = b, c1 = b + 1;
  if (a.cu_seqlens) {
    c0 = a.cu_seqlens[b];
    c1 = a.cu_seqlens[b + 1];
  }
  c0 = min(max(c0, 0), a.n_tokens);
  c1 = min(max(c1, c0), a.n_tokens);
  return {c0, min(c1 - c0, min(a.width, SHARD_TREE_ROWS))};
}

template <class T>
__device__ __forceinline__ void load_nodes(const shard_verify_args& a, Nodes& nodes, const Rows& rows, int tid, int threads) {
  const T* logits = (const T*)a.logits + rows.first * a.row_stride;
  for (int i = tid; i < rows.n; i += threads) {
    const int64_t row = rows.first + i;
    const int p = a.parents[row];
    const int64_t t = a.tokens[row];
    const float* u = a.uniforms + 2 * row;          // 4-byte aligned
    const bool child = p >= 0 && p < i, ok = child && t >= 0 && t < a.vocab;
    nodes.up[i] = child ? p : -1;
    nodes.token[i] = ok ? (int32_t)t : -1;
    nodes.u[i] = u[0];
    nodes.after[i] = u[1];
    nodes.logit[i] = ok ? (float)logits[p * a.row_stride + t] : -INFINITY;
    if (a.draft_probs) nodes.q[i] = ok ? a.draft_probs[row * a.probs_stride + t] : 0.f;
  }
}

// A part's rejected weights are subtracted from its sum, which is off by some 2^-48 of
// what it was.  That may be all that is left of the part, and one that holds nothing must
// not have the answer; or more than is left of the row can bear.  A part of which less
// than kVague is left, or that was more than kMuch times what is left of the row, is
// summed again without them: 3.4 us at 128,256 logits, for a token with 15/16 of the
// weight or more, which is rejected one time in 16 at most.
constexpr double kVague = 0x1p-24, kMuch = 16.0;

// A row's children in their order, until one is accepted: its row, or -1.  Leaves
// the rejected ones in sh, stored by every lane: what a lane reads of them follows its
// own store.  A whole wave.  Q: kSum where another child comes after rejections of
// which only `known` have their sums in sh.amount.  Otherwise j.mine and j.sum are what
// the rejections leave of the lane's part and of the row.
constexpr int kSum = -2;
template <class T, bool Q>
__device__ __forceinline__ int turn(const shard_verify_args& a, const VerifyWork& w, const Nodes& nodes, Shared& sh, int c0, int n, int cur,
                                    Joined& j, double rate, int& rejected, int known = 0) {
  const int lane = threadIdx.x & 63;
  rejected = 0;
  const Scale scale(j.most, rate);
  double was = j.mine;                                  // the lane's part when it was last summed
  int chosen = -1;
  Weights<T, false> weights(a, sh, c0, c0 + cur, j.most, 1.0, rate, 0);
  for (int base = (cur + 1) & ~63; base < n && chosen < 0; base += 64) {
    const int i = base + lane;
    const bool child = i < n && nodes.up[i] == cur;
    uint64_t todo = __builtin_amdgcn_ballot_w64(child);
    const int token_i = child ? nodes.token[i] : -1;
    const float u_i = child ? nodes.u[i] : 0.f;
    const double e = token_i >= 0 ? scale(nodes.logit[i]) : 0.0;
    const int part_i = (int)((uint32_t)(max(token_i, 0) + weights.r.mis) / Row<T>::VEC / (uint32_t)w.granules);
    while (todo && chosen < 0) {
      const int bit = __builtin_ctzll(todo), c = base + bit;
      todo &= todo - 1;
      const int token = __builtin_amdgcn_readlane(token_i, bit);
      const double mine = lane_value(e, bit), u = (double)__int_as_float(__builtin_amdgcn_readlane(__float_as_int(u_i), bit));
      if (rate == 0.0) {
        if (token >= 0 && token == j.at) chosen = c;
      } else if (token < 0) {
        // passed over
      } else if constexpr (Q) {
        const auto q = [&](int k) { return (double)a.draft_probs[(int64_t)(c0 + sh.rejected[k]) * a.probs_stride + token]; };
        if (rejected > known) return kSum;
        double s = mine / j.sum;
        for (int k = 0; k < rejected; ++k)
          if (sh.amount[k] > 0.0) {
            const double d = s - q(k);
            s = (d > 0.0 ? d : 0.0) / sh.amount[k];
          }
        if (u * (double)nodes.q[c] < s) {
          chosen = c;
        } else {
          sh.rejected[rejected] = c;
          ++rejected;
        }
      } else {
        // a token that a sibling before has had rejected has nothing left
        bool again = false;
        for (int k = lane; k < rejected; k += 64) again |= sh.rejected[k] == token;
        if (!__builtin_amdgcn_ballot_w64(again)) {
          if (u * j.sum < mine) {
            chosen = c;
          } else {
            sh.rejected[rejected] = token;
            ++rejected;
            if (lane == __builtin_amdgcn_readlane(part_i, bit)) j.mine -= mine;
            for (;;) {
              j.sum = wave_sum(j.mine);
              const uint64_t vague = __builtin_amdgcn_ballot_w64(j.mine != was && (j.mine < kVague * was || was > kMuch * j.sum));
              if (!vague) break;
              const int part = __builtin_ctzll(vague);
              weights.n = rejected;
              const double left = wave_sum(weights.template sum<4>(weights.begin(w, part), weights.end(w, part), lane, 64));
              if (lane == part) j.mine = was = left;
            }
          }
        }
      }
    }
  }
  return chosen;
}

// What wave 0 found, for all, and the rest of the walk's outputs.
__device__ __forceinline__ void ended(const shard_verify_args& a, const Nodes& nodes, Shared& sh, int b, const Rows& rows, const Joined& j,
                                      bool none, int cur, int count, int rejected) {
  const int tid = threadIdx.x;
  int32_t* path = a.path + (int64_t)b * a.width;
  __syncthreads();
  if (tid == 0) {
    sh.end.total = j.sum;
    sh.end.most = j.most;
    sh.end.at = j.at;
    sh.end.row = none ? -1 : rows.first + cur;
    sh.end.rejected = rejected;
    sh.end.wants = 0;
    sh.count = count;
    sh.u = rows.n > 0 ? nodes.after[cur] : 0.f;
    a.counts[b] = count;
    if (rows.n > 0) path[0] = 0;
  }
  __syncthreads();
  for (int i = sh.count + tid; i < a.width; i += kWalk) path[i] = -1;
}

// The walk.  Wave 0 decides; for Q the whole workgroup sums what a rejection has
// left where another child comes after it, or (not `last`) leaves that to another
// launch and goes on `from` there.  Leaves sh.end, the rejected rows (tokens) of the
// last row, and for Q what each but the last left.  Returns the lane's part of the
// last row (wave 0).
template <class T, bool Q>
__device__ __forceinline__ double walk(const shard_verify_args& a, const VerifyWork& w, Nodes& nodes, Shared& sh, Part (&held_stats)[kHeld],
                                       int b, double rate, const State* from, bool last) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Rows rows = rows_of(a, b);
  const int c0 = rows.first, n = rows.n;
  const Part* stats = w.stats + (int64_t)c0 * w.parts;
  const bool held = n * w.parts <= kHeld;
  if (held)
#pragma unroll
    for (int i = tid; i < kHeld; i += kWalk)
      if (i < n * w.parts) held_stats[i] = stats[i];
  load_nodes<T>(a, nodes, rows, tid, kWalk);
  __syncthreads();
  int cur = 0, count = n > 0 ? 1 : 0, rejected = 0;
  int32_t* path = a.path + (int64_t)b * a.width;
  Joined j{0.0, 0.0, 0.f, -1};
  bool none = n == 0, wants = false;
  int known = 0;                                        // Q: rejections of the row whose sums are known
  if (Q && from) {
    cur = from->row - c0;
    count = from->count;
    known = from->rejected;
    for (int k = tid; k < known - 1; k += kWalk) sh.amount[k] = w.left[c0 + k];
    if (wave == 0) {
      j = join((held ? held_stats : stats) + cur * w.parts, w.parts, rate, lane);
      const double left = wave_sum(lane < w.parts ? w.rest[(int64_t)b * w.parts + lane] : 0.0);
      if (lane == 0) sh.amount[known - 1] = left;
    }
    __syncthreads();
  }
  do {
    if (wave == 0) {
      bool on = !none;
      while (on) {                                      // one row a turn
        if (known == 0) j = join((held ? held_stats : stats) + cur * w.parts, w.parts, rate, lane);
        rejected = 0;
        none = !has_answer(j.most, rate);
        const int chosen = none || count > a.max_depth ? -1 : turn<T, Q>(a, w, nodes, sh, c0, n, cur, j, rate, rejected, known);
        on = chosen >= 0;
        wants = chosen == kSum;
        if (on) {
          cur = chosen;
          if (lane == 0) path[count] = cur;
          ++count;
          known = 0;
        }
      }
      if (Q && lane == 0) {
        sh.end = State{j.sum, j.most, j.at, c0 + cur, rejected, count, wants, 0};
      }
    }
    if constexpr (Q) {
      __syncthreads();
      wants = sh.end.wants;
      if (wants && !last) return j.mine;                // k_verify_rest sums it
      if (wants) {                                      // what the last rejection left, and the turn once more
        known = sh.end.rejected;
        const Weights<T, Q> weights(a, sh, c0, sh.end.row, sh.end.most, sh.end.total, rate, known);
        const double all = sum_of(weights, 0, weights.r.count * (Row<T>::VEC / 4), sh);
        if (tid == 0) sh.amount[known - 1] = all;
        __syncthreads();
      }
    }
  } while (Q && wants);
  ended(a, nodes, sh, b, rows, j, none, cur, count, rejected);
  return j.mine;
}

// The answer of a walk that has ended at sh.end: the part that it lies in from the
// parts' sums of s, `part` in wave 0's lanes, then the token.
template <class T, bool Q>
__device__ __forceinline__ void answer(const shard_verify_args& a, const VerifyWork& w, Shared& sh, int b, int64_t c0, double rate,
                                       double part) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const State end = sh.end;
  if (end.row < 0 || rate == 0.0) {
    if (tid == 0) a.next[b] = end.row < 0 ? -1 : end.at;
    return;
  }
  Weights<T, Q> weights(a, sh, c0, end.row, end.most, end.total, rate, end.rejected);
  if (wave == 0) {
    const double x = wave_scan(part);
    const double target = (double)sh.u * lane_value(x, 63);
    const uint64_t over = __builtin_amdgcn_ballot_w64(x > target), some = __builtin_amdgcn_ballot_w64(part > 0.0);
    const int p = over ? __builtin_ctzll(over) : some ? 63 - __builtin_clzll(some) : -1;
    const double before = lane_value(x - part, max(p, 0));
    if (lane == 0) {
      sh.pick_part = p;
      sh.target = target - before;
      sh.found = INT32_MAX;
      sh.last = -1;
    }
  }
  __syncthreads();
  int64_t i0 = weights.begin(w, sh.pick_part), i1 = weights.end(w, sh.pick_part);
  double target = sh.target;
  if (sh.pick_part < 0) {           // nothing is left of s
    if (!Q || weights.n == 0) {     // of numbers that are not below 1
      if (tid == 0) a.next[b] = -1;
      return;
    }
    // the last subtraction is not made; its row as a whole
    do --weights.n;
    while (weights.n && !(sh.amount[weights.n - 1] > 0.0));
    i0 = 0;
    i1 = weights.r.count * (Row<T>::VEC / 4);
    target = (double)sh.u * sum_of(weights, i0, i1, sh);
  }
  double base = 0.0;
#pragma unroll 1
  for (int64_t at = i0; at < i1; at += kWalk) {
    double v[1][4], all;
    typename Weights<T, Q>::Raw raw[1] = {weights.fetch(at + tid, i1)};
    const double own = weights.values(raw, v);
    double run = base + scan(own, sh, all);
    // the first element at which the running sum is above the target, else the last that has any
    int pick = -1, some = -1;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      run += v[0][k];
      if (v[0][k] > 0.0) {
        some = (int)(4 * (at + tid) - weights.r.mis + k);
        if (run > target && pick < 0) pick = some;
      }
    }
    const uint64_t picks = __builtin_amdgcn_ballot_w64(pick >= 0), has = __builtin_amdgcn_ballot_w64(some >= 0);
    if (picks) {
      if (lane == __builtin_ctzll(picks)) atomicMin(&sh.found, pick);
    } else if (has && lane == 63 - __builtin_clzll(has)) {
      atomicMax(&sh.last, some);
    }
    __syncthreads();
    if (sh.found != INT32_MAX) break;
    base += all;
    __syncthreads();
  }
  if (tid == 0) a.next[b] = sh.found != INT32_MAX ? sh.found : sh.last;
}

// Many rows, few of them on a path: a launch a level.  Each workgroup takes its
// sequence's turn at the row of the level before (all of them the same one), then its
// parts of the row that this leads to.
template <class T>
__global__ __launch_bounds__(kThreads)
void k_verify_level(const shard_verify_args a, const VerifyWork w, int level) {
  __shared__ Nodes nodes;
  __shared__ Shared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int b = blockIdx.y, part = blockIdx.x * (kThreads / 64) + wave;
  const Rows rows = rows_of(a, b);
  if (rows.n == 0) return;
  Level s{0, 1, 0};
  if (level > 0) {
    s = w.level[(level - 1 & 1) * a.batch + b];
    const double rate = rate_of(a, b);
    if (s.done == 0) {
      const Part* stats = w.stats + ((int64_t)(level - 1 & 1) * a.batch + b) * w.parts;
      load_nodes<T>(a, nodes, rows, tid, kThreads);
      __syncthreads();
      if (wave == 0) {
        Joined j = join(stats, w.parts, rate, lane);
        int rejected, chosen = -1;
        if (has_answer(j.most, rate)) chosen = turn<T, false>(a, w, nodes, sh, rows.first, rows.n, s.row, j, rate, rejected);
        if (lane == 0) sh.found = chosen;
      }
      __syncthreads();
      if (sh.found < 0) {
        s.done = level;                                // its last row's parts are those of the level before
      } else {
        s.row = sh.found;
        if (tid == 0 && blockIdx.x == 0) a.path[(int64_t)b * a.width + s.count] = s.row;
        ++s.count;
      }
    }
  }
  if (tid == 0 && blockIdx.x == 0) w.level[(level & 1) * a.batch + b] = s;
  if (s.done == 0 && part < w.parts)
    part_of<T>(a, w, rows.first + s.row, part, b, w.stats + ((int64_t)(level & 1) * a.batch + b) * w.parts + part);
}

// After `levels` of them: the last turn again, which leads nowhere, and the answer.
template <class T>
__global__ __launch_bounds__(kWalk)
void k_verify_end(const shard_verify_args a, const VerifyWork w, int levels) {
  __shared__ Nodes nodes;
  __shared__ Shared sh;
  const int b = blockIdx.x, last = levels - 1;
  const double rate = rate_of(a, b);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Rows rows = rows_of(a, b);
  Level s{0, 0, 0};
  if (rows.n) s = w.level[(last & 1) * a.batch + b];
  const int of = s.done ? s.done - 1 : last;            // the level that took its last row's parts
  load_nodes<T>(a, nodes, rows, threadIdx.x, kWalk);
  __syncthreads();
  Joined j{0.0, 0.0, 0.f, -1};
  int rejected = 0;
  bool none = rows.n == 0;
  if (wave == 0 && rows.n) {
    j = join(w.stats + ((int64_t)(of & 1) * a.batch + b) * w.parts, w.parts, rate, lane);
    none = !has_answer(j.most, rate);
    if (!none && s.count <= a.max_depth) turn<T, false>(a, w, nodes, sh, rows.first, rows.n, s.row, j, rate, rejected);
  }
  ended(a, nodes, sh, b, rows, j, none, s.row, s.count, rejected);
  const int c0 = rows.first;
  const double mine = j.mine;
  answer<T, false>(a, w, sh, b, c0, rate, mine);
}

template <class T, bool Q>
__global__ __launch_bounds__(kWalk)
void k_verify_walk(const shard_verify_args a, const VerifyWork w, int round, bool last) {
  __shared__ Part stats[kHeld];
  __shared__ Nodes nodes;
  __shared__ Shared sh;
  const int tid = threadIdx.x, b = blockIdx.x;
  const double rate = rate_of(a, b);
  const int c0 = rows_of(a, b).first;
  if constexpr (Q) {
    State from;
    if (round) {
      from = w.state[b];
      if (!from.wants) return;
    }
    walk<T, Q>(a, w, nodes, sh, stats, b, rate, round ? &from : nullptr, last);
    __syncthreads();
    const int rejected = sh.end.rejected;
    if (tid == 0) {
      State end = sh.end;
      if (!end.wants) end.count = sh.count;
      end.round = round;
      w.state[b] = end;
    }
    for (int k = tid; k < rejected; k += kWalk) {
      w.rejected[c0 + k] = sh.rejected[k];
      w.left[c0 + k] = k < rejected - 1 ? sh.amount[k] : 0.0;
    }
  } else {
    const double mine = walk<T, Q>(a, w, nodes, sh, stats, b, rate, nullptr, true);
    answer<T, Q>(a, w, sh, b, c0, rate, mine);
  }
}

// With draft_probs: a walk's end from its state.  Sequences that share rows (offsets that
// do not ascend) write over each other's rejected rows: none of them leaves the sequence.
__device__ __forceinline__ void end_of(const shard_verify_args& a, const VerifyWork& w, Shared& sh, int b, const Rows& rows) {
  const int tid = threadIdx.x, c0 = rows.first;
  const State end = w.state[b];
  if (tid == 0) {
    sh.end = end;
    sh.u = end.row >= 0 ? a.uniforms[2 * (int64_t)end.row + 1] : 0.f;
  }
  for (int k = tid; k < end.rejected; k += blockDim.x) {
    sh.rejected[k] = min(w.rejected[c0 + k], rows.n - 1);
    sh.amount[k] = w.left[c0 + k];
  }
  __syncthreads();
}

template <class T>
__global__ __launch_bounds__(kThreads)
void k_verify_rest(const shard_verify_args a, const VerifyWork w, int round) {
  __shared__ Shared sh;
  const int part = blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int b = blockIdx.y;
  const Rows rows = rows_of(a, b);
  const int c0 = rows.first;
  const double rate = rate_of(a, b);
  end_of(a, w, sh, b, rows);
  if (sh.end.round != round || sh.end.row < 0 || rate == 0.0 || part >= w.parts) return;
  const Weights<T, true> weights(a, sh, c0, sh.end.row, sh.end.most, sh.end.total, rate, sh.end.rejected);
  double own = weights.template sum<4>(weights.begin(w, part), weights.end(w, part), lane, 64);
  own = wave_sum(own);
  if (lane == 0) w.rest[(int64_t)b * w.parts + part] = own;
}

template <class T>
__global__ __launch_bounds__(kWalk)
void k_verify_answer(const shard_verify_args a, const VerifyWork w) {
  __shared__ Shared sh;
  const int b = blockIdx.x;
  const Rows rows = rows_of(a, b);
  const double part = threadIdx.x < w.parts ? w.rest[(int64_t)b * w.parts + threadIdx.x] : 0.0;
  const double rate = rate_of(a, b);
  end_of(a, w, sh, b, rows);
  answer<T, true>(a, w, sh, b, rows.first, rate, part);
}

// --------------------------------------------------------------------------
// host side
// --------------------------------------------------------------------------
// Launches of a level each, or 0: all rows at once.  A row of 128,256 logits costs
// 0.12 us of the chip (its exponentials in 64 bits), a level 2.3 us; about three
// rows of a sequence are on its path.  All at once / by levels, us: 61 rows in 7
// levels 17.8 / 24.3, 4 such trees 40.9 / 29.3, 64 chains of 5 46.3 / 33.0, 64 trees
// of up to 26 134.5 / 47.2; 3,904 rows of 5,000 logits in 6 levels 47.4 / 39.4.
int levels_of(const shard_verify_args* a) {
  if (a->draft_probs) return 0;   // a turn may take sums over the row
  const int64_t levels = (int64_t)(a->max_depth < a->width - 1 ? a->max_depth : a->width - 1) + 1;
  return (a->n_tokens - 3 * (int64_t)a->batch) * a->vocab > 2500000 * levels ? (int)levels : 0;
}

// With draft_probs: launches of the walk, each with one that sums what rejections
// have left; a walk that wants more sums than they give takes them in its one
// workgroup (40 to 60 us each, the launches 15, 5 where nobody wants them).  A
// chain, whose depth is its rows, wants none; trees most often up to two.  Trees whose
// max_depth is not told pass for chains, and so does a batch with a chain as long as its
// largest tree: 2 / 3 / 4 children of one row rejected, us, told and not, one sequence
// 36.8 and 60.4 / 55.7 and 110 / 117 and 172, 16 sequences 51.9 and 81.5 / 77 and 140 /
// 158 and 214.  128,256
// tokens, the first of 4 children accepted / all 4 rejected, us: one sequence 23.6 / 154
// with two launches, 28.5 / 126 with three; 16 sequences 37.1 / 191, 42.2 / 159.
int rounds_of(const shard_verify_args* a) {
  const int spare = a->width - 1 - (a->max_depth < a->width - 1 ? a->max_depth : a->width - 1);
  return 1 + (spare < 2 ? spare : 2);
}

bool plan(const shard_verify_args* a, VerifyWork& w, size_t& bytes) {
  if (a->n_tokens < 0 || a->n_tokens >= 1 << 24 || a->batch <= 0 || a->batch > 65535 || a->vocab <= 0 || a->vocab >= INT32_MAX - 64)
    return false;
  if (a->dtype != SHARD_FP16 && a->dtype != SHARD_BF16 && a->dtype != SHARD_FP32) return false;
  const int vec = a->dtype == SHARD_FP32 ? 4 : 8;
  const int64_t granules = (a->vocab + 2 * vec - 2) / vec;          // of the worst aligned row
  w.granules = (granules + kMaxParts - 1) / kMaxParts;
  if (w.granules < kTurn / 2) w.granules = kTurn / 2;
  w.parts = (int)((granules + w.granules - 1) / w.granules);
  w.levels = levels_of(a);
  if (w.levels) {
    bytes = (size_t)2 * a->batch * (w.parts * sizeof(Part) + sizeof(Level));
    return true;
  }
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
  const unsigned groups = (w.parts + kThreads / 64 - 1) / (kThreads / 64);
  if (w.levels) {
    for (int i = 0; i < w.levels; ++i) hipLaunchKernelGGL(k_verify_level<T>, dim3(groups, a.batch), dim3(kThreads), 0, s, a, w, i);
    hipLaunchKernelGGL(k_verify_end<T>, dim3(a.batch), dim3(kWalk), 0, s, a, w, w.levels);
    return;
  }
  hipLaunchKernelGGL(k_verify_stats<T>, dim3((unsigned)a.n_tokens, groups), dim3(kThreads), 0, s, a, w);
  if (a.draft_probs) {
    const int rounds = rounds_of(&a);
    for (int i = 0; i < rounds; ++i) {
      hipLaunchKernelGGL((k_verify_walk<T, true>), dim3(a.batch), dim3(kWalk), 0, s, a, w, i, i == rounds - 1);
      hipLaunchKernelGGL(k_verify_rest<T>, dim3(groups, a.batch), dim3(kThreads), 0, s, a, w, i);
    }
    hipLaunchKernelGGL(k_verify_answer<T>, dim3(a.batch), dim3(kWalk), 0, s, a, w);
  } else {
    hipLaunchKernelGGL((k_verify_walk<T, false>), dim3(a.batch), dim3(kWalk), 0, s, a, w, 0, true);
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
  w.level = (Level*)(w.stats + (size_t)2 * a->batch * w.parts);
  if (a->draft_probs) {
    w.state = (State*)(w.stats + (size_t)a->n_tokens * w.parts);
    w.rest = (double*)(w.state + a->batch);
    w.left = w.rest + (size_t)a->batch * w.parts;
    w.rejected = (int32_t*)(w.left + a->n_tokens);
  }
  const hipStream_t s = (hipStream_t)stream;
  if (a->n_tokens == 0) {
    // sequences of no rows: nothing is read
    hipLaunchKernelGGL((k_verify_walk<half_t, false>), dim3(a->batch), dim3(kWalk), 0, s, *a, w, 0, true);
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
