// qe_op_verify_drafts and qe_op_verify_tree: drafted tokens checked against the target's probabilities, from given random
// numbers. It is qe_verify_greedy's rule for sampled decoding: what the accepted drafts and the
// token drawn after them follow is exactly the target's distribution. No reference counterpart.
//
// Row r of a sequence has the target's logits x after the tokens before it. With weights
// w_i = exp((x_i - max x) / T) and p_i = w_i / sum w, the draft d of the row is accepted if
// u q(d) < p(d) for the row's random number u and the draft model's probability q(d) (1 without
// draft probabilities: a draft rule such as prompt lookup proposes one token). The first row that
// does not accept draws from max(p - q, 0); the last row, which has no draft, draws from p. A draw
// is the smallest token whose running sum of weights is above v times their sum.
//
// Numerics: tokens are whole values, so the sums that decide them are held in 64 bits, where the
// running sum of 151,936 weights is off by some 1e-16 of a token's mean weight instead of the 1%
// that f32 would give. Without a distribution to subtract a draw uses the weights as they are, so
// equal ones are exactly equal.
//
// Bound by one read of the logits. k_draft_sums reads every row once, in chunks of 2048 tokens,
// and keeps each chunk's largest logit and its sum of weights relative to that one. k_draft_decide, a
// workgroup per sequence, joins the chunks of each row, accepts drafts (a gather each) and finds the
// row that draws; with no draft probabilities the chunk sums already hold the running sum at chunk
// borders, so it also draws, reading one chunk again. With them k_draft_rest sums max(p - q, 0) of the
// drawing rows by chunks and k_draft_draw draws.
//
// Measured: 250 rows of 151,936 logits with draft probabilities, 40 sequences of up to 7 drafts, 55 to 61 us,
// of which the sums take 31 to 35 (152 MB, 4.3 to 5 TB/s), decide 7.5, the rest 10 and the draw 5; 32 rows without
// drafts 14.0 (sums 8, bound by the 64-bit exponentials; decide 7); 5 rows of one sequence 11.4 in a graph. Decide and draw
// are chains: plan, sums, the row's total, its chunk, the logits there, the token; 0.5 to 1.5 us a link.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "../../include/qe.h"
#include "device_common.h"
#include "status.h"

namespace qe {
namespace {

// What a chunk of a row adds up to: weights relative to its own largest logit.
struct alignas(16) ChunkSum {
  double sum;
  float top;      // -inf: nothing above -inf
  uint32_t best;  // first index of top, of greedy rows
};

// The row a sequence draws from.
struct DrawRow {
  double total, inv_total, k;  // sum of weights, 1 / it; log2(e) / T
  uint32_t row;                // 0xFFFFFFFF: the sequence draws nothing here
  uint32_t best, draft;
  float top;
  uint32_t greedy;  // all the weight on `best`
};

struct DraftArgs {
  const float* logits;
  const float* probs;  // null: one drafted token without a distribution
  const int32_t* starts;
  const uint32_t* drafts;
  const float* accept;
  const float* sample;
  const float* temperature;  // null: 1
  uint32_t *tokens, *count;
  float* logprobs;  // null: not wanted
  uint64_t stride, probs_stride;
  uint32_t n_rows, n_seqs, vocab, chunks;
  ChunkSum* sums;  // [n_rows][chunks]
  double* rests;   // [n_seqs][chunks]
  DrawRow* draws;  // [n_seqs]
};

constexpr int kThreads = 512;
constexpr uint32_t kChunk = 2048, kNone = 0xFFFFFFFFu;
constexpr uint32_t kMostVocab = kThreads * kChunk;  // a thread of a draw has one chunk: 2^20
constexpr uint32_t kRowsAcross = 65535;              // a grid's limit in y and z

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

// 2^t in 64 bits for t <= 0 (6e-16; 0 below -1000 and for NaN): t = n + f with n the nearest whole number,
// and 2^f = 1 + f c(f) by Chebyshev interpolation of (2^f - 1) / f at 10 points of [-1/2, 1/2]; n goes
// straight into the exponent. 2^0 is exactly 1. (The library's exp is some 40 instructions on the same
// unit, which then bounds the pass instead of the memory.)
template <int N>
__device__ __forceinline__ void exp2_64(const double (&t)[N], double (&y)[N]) {
  constexpr double c[10] = {7.070977866508138e-09,  1.0205905413765595e-07, 1.3215451633221434e-06, 1.5252672924850737e-05,
                            0.00015403530424776529, 0.0013333558200794592,  0.009618129107618665,   0.05550410866465167,
                            0.24022650695910075,    0.6931471805599462};
  double n[N], f[N];
#pragma unroll
  for (int i = 0; i < N; i++) {
    n[i] = rint(t[i]);
    f[i] = t[i] - n[i];
    y[i] = c[0];
  }
  // y f + c with c in a scalar register (the compiler would copy it into the accumulator first, two moves
  // for each); N chains side by side, since each step waits for the one before
#pragma unroll
  for (int k = 1; k < 10; k++)
#pragma unroll
    for (int i = 0; i < N; i++) {
      const double x = y[i];
      asm("v_fma_f64 %0, %1, %2, %3" : "=v"(y[i]) : "v"(x), "v"(f[i]), "s"(c[k]));
    }
#pragma unroll
  for (int i = 0; i < N; i++) {
    const double z = fma(y[i], f[i], 1.0);
    y[i] = __hiloint2double(__double2hiint(z) + (int(fmax(n[i], -1000.0)) << 20), __double2loint(z));
    y[i] = t[i] >= -1000.0 ? y[i] : 0.0;
  }
}
__device__ __forceinline__ double exp2_64(double t) {
  const double x[1] = {t};
  double y[1];
  exp2_64<1>(x, y);
  return y[0];
}

// weight of logit x relative to the largest one, top: NaN and -inf weigh nothing, infinite ones share
__device__ __forceinline__ double weight(float x, float top, double k) {
  if (top == INFINITY) return x == top ? 1.0 : 0.0;
  return exp2_64((double(x) - double(top)) * k);
}

// log p of a token with logit x
__device__ __forceinline__ float log_weight(const DrawRow& d, float x, float t) {
  if (d.greedy) return 0.f;
  return float((x == d.top ? 0.0 : (double(x) - double(d.top)) / double(t)) - log(d.total));
}

__device__ __forceinline__ double wave_sum64(double v) { return from_lane(wave_scan(v), 63); }

// the row's sequence, or -1 (as paged rows are found: the last one that starts at or before it)
__device__ __forceinline__ int32_t sequence(const DraftArgs& a, int32_t r) {
  uint32_t lo = 0, hi = a.n_seqs;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (a.starts[mid] <= r) lo = mid;
    else hi = mid;
  }
  return a.starts[lo] <= r && r < a.starts[lo + 1] ? int32_t(lo) : -1;
}
__device__ __forceinline__ float temperature(const DraftArgs& a, uint32_t s) {
  return a.temperature ? a.temperature[s] : 1.f;
}
// log2(e) / T
__device__ __forceinline__ double rate(float t) { return 1.4426950408889634 / double(t); }

// N values of a row of n from c0 on: value 4 i + e of lane l is token c0 + 256 i + 4 l + e; `pad` behind the row.
// Non-temporal (four inputs in turn in a graph): 40 sequences of up to 7 drafts 62.6 us without, so 57.5; 32 rows
// 17.8 and 15.6.
template <int N>
__device__ __forceinline__ void load_values(const float* row, uint32_t c0, uint32_t n, float pad, float (&x)[N]) {
  const uint32_t lane = threadIdx.x & 63;
  if (c0 + 64 * N <= n) {
#pragma unroll
    for (int i = 0; i < N / 4; i++) {
      const f32x4u v = __builtin_nontemporal_load(reinterpret_cast<const f32x4u*>(row + c0 + 256 * i + 4 * lane));
#pragma unroll
      for (int e = 0; e < 4; e++) x[4 * i + e] = v[e];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const uint32_t t = c0 + 256 * i + 4 * lane + e;
        x[4 * i + e] = t < n ? row[t] : pad;
      }
  }
}

// A chunk's work goes to one wave (WAVES = 1) or to the four waves of a workgroup, so that few chunks reach all
// SIMDs: up to 4 for each of them (four inputs in turn in a graph: 5 rows 12.5 us with one wave, 11.4 with four; the
// whole of 40 x 7 with the rests of 40 rows by one 61.5, by four 57.5; with the sums of its 250 rows, 18,750
// chunks, by four 62.7).
constexpr uint64_t kFewChunks = 4096;

// The chunk's number, and the first token of the wave's share.
template <int WAVES>
__device__ __forceinline__ uint32_t chunk_of(uint32_t& c0) {
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t c = WAVES == 1 ? blockIdx.x * 4 + wave : blockIdx.x;
  c0 = c * kChunk + (WAVES == 1 ? 0 : wave * (kChunk / WAVES));
  return c;
}

// What the wave's values x (of WAVES = 4: with the workgroup's other three waves') add up to; of wave 0.
template <int WAVES, int N>
__device__ __forceinline__ ChunkSum chunk_sum(const float (&x)[N], uint32_t c0, float t, ChunkSum* shares) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < N; i++) m = fmaxf(m, x[i]);
  m = wave_max(m);
  if constexpr (WAVES > 1) {
    if (lane == 0) shares[wave].top = m;
    __syncthreads();
    for (int i = 0; i < WAVES; i++) m = fmaxf(m, shares[i].top);
  }
  double sum = 0.0;
  uint32_t at = kNone;
  if (t > 0.f && m > -INFINITY) {
    const double k = rate(t), top = double(m);
    if (m < INFINITY) {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        double t4[4], w[4];
#pragma unroll
        for (int e = 0; e < 4; e++) t4[e] = (double(x[i + e]) - top) * k;
        exp2_64<4>(t4, w);
        sum += (w[0] + w[1]) + (w[2] + w[3]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; i++) sum += x[i] == m ? 1.0 : 0.0;
    }
    sum = wave_sum64(sum);
  } else {  // greedy: the first place that holds the largest
#pragma unroll
    for (int i = N - 1; i >= 0; i--)
      if (x[i] == m) at = c0 + 256 * (i / 4) + 4 * lane + i % 4;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) at = min(at, uint32_t(__shfl_xor(int(at), d)));
  }
  if constexpr (WAVES > 1) {
    if (lane == 0) {
      shares[wave].sum = sum;
      shares[wave].best = at;
    }
    __syncthreads();
    if (threadIdx.x == 0)
      for (int i = 1; i < WAVES; i++) {
        sum += shares[i].sum;
        at = min(at, shares[i].best);
      }
  }
  return ChunkSum{sum, m, at};
}

// Row blockIdx.y + ..., a chunk of it.
template <int WAVES>
__global__ __launch_bounds__(256) void k_draft_sums(DraftArgs a) {
  constexpr int N = 32 / WAVES;
  __shared__ ChunkSum shares[WAVES];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = blockIdx.y + blockIdx.z * kRowsAcross;
  uint32_t c0;
  const uint32_t c = chunk_of<WAVES>(c0);
  if (c >= a.chunks || r >= a.n_rows) return;
  float x[N];
  load_values(a.logits + r * a.stride, c0, a.vocab, -INFINITY, x);
  const int32_t s = sequence(a, int32_t(r));
  if (s < 0) return;
  const ChunkSum sum = chunk_sum<WAVES>(x, c0, temperature(a, s), shares);
  if (lane == 0 && (WAVES == 1 || wave == 0)) a.sums[size_t(r) * a.chunks + c] = sum;
}

// ---- a workgroup's draw ----
struct Scratch {
  double wave[kThreads / 64];
  uint64_t some[kThreads / 64], over[kThreads / 64];  // lanes with any weight; of them those the aim lies below
};

// Of N items with weights w: the first with some whose running sum, from `run` on, is above `to` (else the
// last with some), and the running sum before it.
template <int N>
__device__ __forceinline__ uint32_t pick(const double (&w)[N], double run, double to, double& before) {
  uint32_t at = 0;
  bool found = false;
  before = run;
#pragma unroll
  for (int i = 0; i < N; i++) {
    if (!found && w[i] > 0.0) {
      at = i;
      before = run;
      found = run + w[i] > to;
    }
    run += w[i];
  }
  return at;
}

// sum of the chunk's weights from one logit to another: the chunk's largest to the row's
__device__ __forceinline__ double chunk_scale(float from, float top, double k) {
  return from == top ? 1.0 : top == INFINITY ? 0.0 : exp2_64((double(from) - double(top)) * k);
}

// A row's chunks over the lanes of a wave: lane l has n = ceil(chunks / 64) of them from n l on.
constexpr int kLaneChunks = kMostVocab / kChunk / 64;

// The first chunk whose running sum is above aim(sum of all), and the running sum before it; if rounding leaves
// none, the last with any weight; kNone if nothing has any. Every wave finds it for itself.
template <class Aim>
__device__ __forceinline__ uint32_t find_chunk(const double (&w)[kLaneChunks], uint32_t n, Aim aim, double& before) {
  const uint32_t lane = threadIdx.x & 63;
  double mine = 0.0;
#pragma unroll
  for (int i = 0; i < kLaneChunks; i++) mine += w[i];
  const double up_to = wave_scan(mine), to = aim(from_lane(up_to, 63));
  const uint64_t some = __ballot(mine > 0.0), over = __ballot(mine > 0.0 && up_to > to);
  before = 0.0;
  if (!some) return kNone;
  const int owner = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(some);
  const uint32_t at = lane * n + pick(w, up_to - mine, to, before);
  before = from_lane(before, owner);
  return from_lane(at, owner);
}

// The sums of max(p - q, 0) over a lane's chunks of sequence s.
__device__ __forceinline__ void load_rests(const DraftArgs& a, uint32_t s, double (&w)[kLaneChunks]) {
  const uint32_t n = (a.chunks + 63) / 64, c0 = (threadIdx.x & 63) * n;
#pragma unroll
  for (int i = 0; i < kLaneChunks; i++) w[i] = uint32_t(i) < n && c0 + i < a.chunks ? a.rests[size_t(s) * a.chunks + c0 + i] : 0.0;
}

// The token of row d.row whose running weight goes above `to`, by the thread that has it, into packed row
// at_row; a thread has N tokens from i0 on, with weights z and logits y.
typedef float f32x4 __attribute__((ext_vector_type(4)));
template <int N>
__device__ __forceinline__ void place_token(const DraftArgs& a, const DrawRow& d, uint32_t at_row, uint32_t i0, const double (&z)[N],
                                            f32x4 y, double to, float t, Scratch& sc) {
  static_assert(N == 4, "y holds 4");
  const float* x = a.logits + d.row * a.stride;
  const uint32_t tid = threadIdx.x;
  double mine = 0.0;
#pragma unroll
  for (int e = 0; e < N; e++) mine += z[e];
  const uint32_t lane = tid & 63, wave = tid >> 6;
  double up_to = wave_scan(mine);
  if (lane == 63) sc.wave[wave] = up_to;
  __syncthreads();
#pragma unroll
  for (uint32_t i = 0; i < kThreads / 64 - 1; i++)
    if (i < wave) up_to += sc.wave[i];
  const uint64_t some = __ballot(mine > 0.0), over = __ballot(mine > 0.0 && up_to > to);
  if (lane == 0) {
    sc.some[wave] = some;
    sc.over[wave] = over;
  }
  __syncthreads();
  uint32_t first = kNone, final = kNone;
#pragma unroll
  for (uint32_t i = 0; i < kThreads / 64; i++) {
    if (first == kNone && sc.over[i]) first = i * 64 + __builtin_ctzll(sc.over[i]);
    if (sc.some[i]) final = i * 64 + 63 - __builtin_clzll(sc.some[i]);
  }
  const uint32_t owner = first != kNone ? first : final;
  if (tid == (owner == kNone ? 0 : owner)) {
    double inner;
    const uint32_t at = pick(z, up_to - mine, to, inner);
    uint32_t token = i0 + at;
    float logit = at == 0 ? y[0] : at == 1 ? y[1] : at == 2 ? y[2] : y[3];
    if (owner == kNone) {
      token = d.best;
      logit = x[token];
    }
    a.tokens[at_row] = token;
    if (a.logprobs) a.logprobs[at_row] = log_weight(d, logit, t);
  }
}

// One token of row d.row: over the chunks by their sums, then within a chunk (4 tokens a thread). v, t: the
// sequence's random number and temperature. REST: from max(p - q, 0), whose sums by chunk are w. Else: the logit of
// the row's draft, and the row's sums by chunk relative to its largest logit where they are at hand (`kept`).
template <bool REST>
__device__ __forceinline__ void draw(const DraftArgs& a, const DrawRow& d, bool last, double v, float t, double (&w)[kLaneChunks],
                                     float drafted, const double* kept, Scratch& sc) {
  constexpr int N = kChunk / kThreads;
  const float* x = a.logits + d.row * a.stride;
  const uint32_t tid = threadIdx.x, n = (a.chunks + 63) / 64, c0 = (tid & 63) * n;
  const uint32_t skip = last || a.probs ? kNone : d.draft;  // a drafted token that has all of q
  auto token_weight = [&](uint32_t i, float xi) -> double {
    return d.greedy ? (i == d.best ? 1.0 : 0.0) : weight(xi, d.top, d.k);
  };
  auto plain_chunks = [&](const double* kept) {
    if (kept && !d.greedy) {
#pragma unroll
      for (int i = 0; i < kLaneChunks; i++) w[i] = uint32_t(i) < n && c0 + i < a.chunks ? kept[c0 + i] : 0.0;
      return;
    }
    ChunkSum p[kLaneChunks];
#pragma unroll
    for (int i = 0; i < kLaneChunks; i++)
      if (uint32_t(i) < n) p[i] = a.sums[size_t(d.row) * a.chunks + min(c0 + i, a.chunks - 1)];
#pragma unroll
    for (int i = 0; i < kLaneChunks; i++) {
      w[i] = 0.0;
      if (uint32_t(i) < n) {
        if (d.greedy) w[i] = d.best / kChunk == c0 + i ? 1.0 : 0.0;
        else if (c0 + i < a.chunks) w[i] = p[i].sum * chunk_scale(p[i].top, d.top, d.k);
      }
    }
  };
  double before, aim = 0.0;
  auto share = [&](double all) { return aim = v * all; };
  if constexpr (!REST) {
    plain_chunks(kept);
    // (a draft is refused where u < 1 is at least p(d): what is left is 2^-24 of the row or more, and the
    // difference is off by 2^-29 of that at most)
#pragma unroll
    for (int i = 0; i < kLaneChunks; i++)
      if (uint32_t(i) < n && skip < a.vocab && skip / kChunk == c0 + i) w[i] = fmax(w[i] - token_weight(skip, drafted), 0.0);
  }
  uint32_t c = find_chunk(w, n, share, before);
  bool plain = false;
  if (c == kNone) {  // nothing is left of p - q: from p
    plain = true;
    plain_chunks(kept);
    c = find_chunk(w, n, share, before);
  }
  double z[N];
  f32x4 y;
  const uint32_t i0 = c * kChunk + tid * N;
  const double to = aim - before;
#pragma unroll
  for (int e = 0; e < N; e++) {
    z[e] = 0.0;
    y[e] = 0.f;
    const uint32_t i = i0 + e;
    if (c != kNone && i < a.vocab) {
      y[e] = x[i];
      z[e] = token_weight(i, y[e]);
      if (!plain) {
        if (REST) {
          const float q = a.probs[d.row * a.probs_stride + i];
          z[e] = z[e] * d.inv_total - (q > 0.f ? double(q) : 0.0);
          z[e] = z[e] > 0.0 ? z[e] : 0.0;
        } else if (i == skip) {
          z[e] = 0.0;
        }
      }
    }
  }
  place_token(a, d, d.row, i0, z, y, to, t, sc);
}

// A workgroup per sequence: a wave joins the chunks of one row after another.
__global__ __launch_bounds__(kThreads) void k_draft_decide(DraftArgs a) {
  constexpr uint32_t BATCH = 64, WAVES = kThreads / 64;
  __shared__ Scratch sc;
  __shared__ DrawRow rows[BATCH];
  __shared__ float drafted[BATCH];  // the draft's logit
  __shared__ uint32_t taken[BATCH];
  __shared__ double kept[WAVES][128];  // of each wave's last row: its sums by chunk (the first 128)
  const uint32_t s = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t r0 = max(a.starts[s], 0), r1 = min(int64_t(a.starts[s + 1]), int64_t(a.n_rows));
  const float t = temperature(a, s), v = a.sample[s];
  if (r1 <= r0) {
    if (threadIdx.x == 0) {
      a.count[s] = 0;
      if (a.probs) a.draws[s].row = kNone;
    }
    return;
  }
  const double k = rate(t);
  int64_t stop = -1;
  const double* at_hand = nullptr;
  for (int64_t b = r0; stop < 0; b += BATCH) {
    const uint32_t n = uint32_t(min(r1 - b, int64_t(BATCH)));
    for (uint32_t i = wave; i < n; i += WAVES) {
      const uint32_t r = uint32_t(b) + i;
      // (the loads that wait for nothing first)
      const ChunkSum* const sums = a.sums + size_t(r) * a.chunks;
      ChunkSum z[2];
#pragma unroll
      for (uint32_t e = 0; e < 2; e++) z[e] = sums[min(lane + 64 * e, a.chunks - 1)];
      DrawRow d;
      d.k = k;
      d.row = r;
      d.draft = a.drafts[r];
      const bool has = r + 1 < r1 && d.draft < a.vocab;
      const float x = has ? a.logits[r * a.stride + d.draft] : 0.f, u = a.accept[r];
      float qd = 1.f;
      if (has && a.probs) qd = a.probs[r * a.probs_stride + d.draft];
      float top = -INFINITY;
#pragma unroll
      for (uint32_t e = 0; e < 2; e++) {
        if (lane + 64 * e >= a.chunks) z[e] = ChunkSum{0.0, -INFINITY, kNone};
        top = fmaxf(top, z[e].top);
      }
      for (uint32_t c = lane + 128; c < a.chunks; c += 64) top = fmaxf(top, sums[c].top);
      d.top = wave_max(top);
      d.greedy = !(t > 0.f) || !(d.top > -INFINITY);
      uint32_t best = kNone;
      double sum = 1.0;
      if (d.greedy) {
        auto first = [&](const ChunkSum& z) {
          if (z.top == d.top) best = min(best, z.best);
        };
#pragma unroll
        for (uint32_t e = 0; e < 2; e++) first(z[e]);
        for (uint32_t c = lane + 128; c < a.chunks; c += 64) first(sums[c]);
#pragma unroll
        for (int e = 1; e < 64; e *= 2) best = min(best, uint32_t(__shfl_xor(int(best), e)));
      } else {
        sum = 0.0;
#pragma unroll
        for (uint32_t e = 0; e < 2; e++) {
          const double w = z[e].top > -INFINITY ? z[e].sum * chunk_scale(z[e].top, d.top, k) : 0.0;
          kept[wave][lane + 64 * e] = w;
          sum += w;
        }
        for (uint32_t c = lane + 128; c < a.chunks; c += 64)
          if (sums[c].top > -INFINITY) sum += sums[c].sum * chunk_scale(sums[c].top, d.top, k);
        sum = wave_sum64(sum);
      }
      d.best = best < a.vocab && d.top > -INFINITY && d.greedy ? best : 0;
      d.total = sum;
      d.inv_total = 1.0 / sum;
      if (lane == 0) {
        const double w = d.greedy ? (d.draft == d.best ? 1.0 : 0.0) : weight(x, d.top, k);
        rows[i] = d;
        drafted[i] = x;
        taken[i] = has && double(u) * (qd > 0.f ? double(qd) : 0.0) < w * d.inv_total;
      }
    }
    __syncthreads();
    uint32_t first = 0;
    while (first < n && taken[first]) first++;
    if (threadIdx.x < first) {
      a.tokens[b + threadIdx.x] = rows[threadIdx.x].draft;
      if (a.logprobs) a.logprobs[b + threadIdx.x] = log_weight(rows[threadIdx.x], drafted[threadIdx.x], t);
    }
    if (first < n) {
      stop = b + first;
      if (first + WAVES >= n && a.chunks <= 128) at_hand = kept[first % WAVES];
    } else {
      __syncthreads();
    }
  }
  const DrawRow d = rows[(stop - r0) % BATCH];
  for (int64_t e = stop + 1 + threadIdx.x; e < r1; e += kThreads) {
    a.tokens[e] = kNone;
    if (a.logprobs) a.logprobs[e] = 0.f;
  }
  const bool last = stop + 1 == r1, rest = a.probs && !last;
  if (threadIdx.x == 0) {
    a.count[s] = uint32_t(stop - r0 + 1);
    if (a.probs) {
      a.draws[s] = d;
      if (!rest) a.draws[s].row = kNone;
    }
  }
  if (!rest) {
    double w[kLaneChunks];
    draw<false>(a, d, last, double(v), t, w, drafted[(stop - r0) % BATCH], at_hand, sc);
  }
}

// The sum of max(p - q, 0) over a chunk of the row that sequence blockIdx.y draws from.
template <int WAVES>
__global__ __launch_bounds__(256) void k_draft_rest(DraftArgs a) {
  constexpr int N = 32 / WAVES;
  __shared__ double shares[WAVES];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, s = blockIdx.y;
  uint32_t c0;
  const uint32_t c = chunk_of<WAVES>(c0);
  if (c >= a.chunks) return;
  const DrawRow d = a.draws[s];
  if (d.row == kNone) return;
  float x[N], q[N];
  load_values(a.logits + d.row * a.stride, c0, a.vocab, -INFINITY, x);
  load_values(a.probs + d.row * a.probs_stride, c0, a.vocab, 0.f, q);
  double sum = 0.0;
  const uint32_t greedy = __builtin_amdgcn_readfirstlane(d.greedy);
  const bool usual = !greedy && d.top < INFINITY;
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    double w[4];
    if (usual) {
      double t4[4];
#pragma unroll
      for (int e = 0; e < 4; e++) t4[e] = (double(x[i + e]) - double(d.top)) * d.k;
      exp2_64<4>(t4, w);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) w[e] = (greedy ? c0 + 64 * i + 4 * lane + e == d.best : x[i + e] == d.top) ? 1.0 : 0.0;
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
      w[e] = w[e] * d.inv_total - (q[i + e] > 0.f ? double(q[i + e]) : 0.0);
      sum += w[e] > 0.0 ? w[e] : 0.0;
    }
  }
  sum = wave_sum64(sum);
  if constexpr (WAVES > 1) {
    if (lane == 0) shares[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0)
      for (int i = 1; i < WAVES; i++) sum += shares[i];
  }
  if (lane == 0 && (WAVES == 1 || wave == 0)) a.rests[size_t(s) * a.chunks + c] = sum;
}

__global__ __launch_bounds__(kThreads) void k_draft_draw(DraftArgs a) {
  __shared__ Scratch sc;
  const uint32_t s = blockIdx.x;
  double w[kLaneChunks];  // (of no use, and of any value, where nothing is drawn)
  load_rests(a, s, w);
  const float t = temperature(a, s), v = a.sample[s];
  const DrawRow d = a.draws[s];
  if (d.row == kNone) return;
  draw<true>(a, d, false, double(v), t, w, 0.f, nullptr, sc);
}

// ---- trees (qe_op_verify_tree) ----
// From a sequence's root on, with p the target at the node and R = 1: its children in order, child c with token d is
// accepted if u_c R < p(d), else R -= p(d) and d has no p left; if none is, the token is drawn from what is left of p. Given
// the ones tried before, child c is accepted with p(d) / R, which is d's share of what is left; so the token that
// comes out has p, whatever the children are.
// The sums of p are k_draft_sums', or a level's. A draw takes the tokens tried out of their chunks' sums, and sums a chunk
// anew of which that leaves next to nothing.
// Measured (151,936 tokens): a tree of 13 nodes 14 us, two launches (sums 5; the walk 2 a step, the draw 4, links of dependent
// loads); 24 trees of up to 48 nodes by levels 50, 8 launches of 2 to 7 and the draw 9.
//
// Where a walk is: at node `cur` of depth `depth`, or (done) it ended there.
struct Walk {
  uint32_t cur, depth, done, pad;
};
struct TreeArgs {
  DraftArgs d;  // drafts: the nodes' tokens; sums: [n_rows][chunks], or by level: [2][n_seqs][chunks]
  const int32_t* parents;
  int32_t* path;  // [n_seqs][QE_TREE_NODES]
  Walk* walks;    // by level: [2][n_seqs]
  uint32_t max_depth;
};

// The sum of a row's weights from its chunks' sums, and what a draw needs of it, by each wave for itself.
__device__ __forceinline__ DrawRow row_of(const DraftArgs& a, const ChunkSum* sums, uint32_t r, float t) {
  const uint32_t lane = threadIdx.x & 63;
  ChunkSum z[2];  // (the first 128 chunks: most vocabularies' all)
#pragma unroll
  for (uint32_t e = 0; e < 2; e++) z[e] = sums[min(lane + 64 * e, a.chunks - 1)];
  DrawRow d;
  d.k = rate(t);
  d.row = r;
  d.draft = kNone;
  float top = -INFINITY;
#pragma unroll
  for (uint32_t e = 0; e < 2; e++) {
    if (lane + 64 * e >= a.chunks) z[e] = ChunkSum{0.0, -INFINITY, kNone};
    top = fmaxf(top, z[e].top);
  }
  for (uint32_t c = lane + 128; c < a.chunks; c += 64) top = fmaxf(top, sums[c].top);
  d.top = wave_max(top);
  d.greedy = !(t > 0.f) || !(d.top > -INFINITY);
  uint32_t best = kNone;
  double sum = 0.0;
  auto add = [&](const ChunkSum& z) __attribute__((always_inline)) {
    if (d.greedy) {
      if (z.top == d.top) best = min(best, z.best);
    } else if (z.top > -INFINITY) {
      sum += z.sum * chunk_scale(z.top, d.top, d.k);
    }
  };
#pragma unroll
  for (uint32_t e = 0; e < 2; e++) add(z[e]);
  for (uint32_t c = lane + 128; c < a.chunks; c += 64) add(sums[c]);
  d.best = 0;
  if (d.greedy) {
#pragma unroll
    for (int e = 1; e < 64; e *= 2) best = min(best, uint32_t(__shfl_xor(int(best), e)));
    if (best < a.vocab && d.top > -INFINITY) d.best = best;
  }
  d.total = d.greedy ? 1.0 : wave_sum64(sum);
  d.inv_total = 1.0 / d.total;
  return d;
}

// The weight of token i, whose logit is x, in row d (its share times d.total)
__device__ __forceinline__ double row_weight(const DrawRow& d, uint32_t i, float x) {
  return d.greedy ? (i == d.best ? 1.0 : 0.0) : weight(x, d.top, d.k);
}

// The nodes of a sequence, one a lane; rows r0 .. r1 - 1.
struct Nodes {
  int64_t r0, r1;
  int32_t parent;
  uint32_t token;
  float accept, t;  // t: the sequence's temperature
};
__device__ __forceinline__ Nodes nodes_of(const TreeArgs& tree, uint32_t s) {
  const DraftArgs& a = tree.d;
  const uint32_t lane = threadIdx.x & 63;
  Nodes n;
  n.r0 = max(a.starts[s], 0);
  n.r1 = min(int64_t(a.starts[s + 1]), int64_t(a.n_rows));
  const bool node = lane < n.r1 - n.r0;
  n.parent = node ? tree.parents[n.r0 + lane] : -1;
  n.token = node ? a.drafts[n.r0 + lane] : kNone;
  n.accept = node ? a.accept[n.r0 + lane] : 0.f;
  n.t = temperature(a, s);
  return n;
}

// Whether the lane's node is tried after node `cur` of depth `depth`, and its token's logit there (loaded before the
// row's sums are waited for).
__device__ __forceinline__ bool is_child(const TreeArgs& tree, const Nodes& n, uint32_t cur, uint32_t depth, float& x) {
  const DraftArgs& a = tree.d;
  const uint32_t lane = threadIdx.x & 63;
  const bool child = depth < tree.max_depth && lane > cur && n.parent == int32_t(cur);
  x = child && n.token < a.vocab ? a.logits[uint64_t(n.r0 + cur) * a.stride + n.token] : 0.f;
  return child;
}
// One step of a walk by each wave for itself: the first child that is accepted, or kNone. d: the node's row; child, x:
// is_child's; tried: the children; w: their tokens' weights, 0 for a token tried before.
__device__ __forceinline__ uint32_t next_node(const TreeArgs& tree, const Nodes& n, const DrawRow& d, bool child, float x,
                                              uint64_t& tried, double& w) {
  const DraftArgs& a = tree.d;
  const uint32_t lane = threadIdx.x & 63;
  tried = __ballot(child);
  w = child && n.token < a.vocab ? row_weight(d, n.token, x) : 0.0;
  double left = 1.0;
  for (uint64_t rest = tried; rest; rest &= rest - 1) {
    const int c = __builtin_ctzll(rest);
    const uint32_t is = from_lane(n.token, c);
    const uint64_t before = __ballot(child && n.token == is) & ((1ull << c) - 1);
    if (before && int(lane) == c) w = 0.0;
    const double p = from_lane(w, c) * d.inv_total;
    if (double(from_lane(n.accept, c)) * left < p) return uint32_t(c);
    left -= p;
  }
  return kNone;
}
// What an accepted child leaves: its token, at depth `depth` of the path before it; by the lane that has it.
__device__ __forceinline__ void take_node(const TreeArgs& tree, const Nodes& n, const DrawRow& d, uint32_t depth, float x) {
  const DraftArgs& a = tree.d;
  a.tokens[n.r0 + depth] = n.token;
  if (a.logprobs) a.logprobs[n.r0 + depth] = log_weight(d, x, n.t);
}

// Level `level` of the walks, of trees too large for every row's sums: the workgroups of a sequence, one or four chunks
// each as k_draft_sums has them, all take the step from the level before, and then sum the row it led to. So a level
// is one launch and reads one row a sequence.
template <int WAVES>
__global__ __launch_bounds__(256) void k_tree_level(TreeArgs tree, uint32_t level) {
  constexpr int N = 32 / WAVES;
  __shared__ ChunkSum shares[WAVES];
  const DraftArgs& a = tree.d;
  const uint32_t s = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t c0;
  const uint32_t c = chunk_of<WAVES>(c0);
  const bool first = blockIdx.x == 0;
  const int64_t r0 = max(a.starts[s], 0), r1 = min(int64_t(a.starts[s + 1]), int64_t(a.n_rows));
  if (r1 <= r0) return;
  uint32_t cur = 0;
  if (level) {
    const Walk at = tree.walks[(level - 1 & 1) * a.n_seqs + s];
    uint32_t next = kNone;
    if (!at.done) {
      const Nodes n = nodes_of(tree, s);
      float x;
      const bool child = is_child(tree, n, at.cur, at.depth, x);
      const DrawRow d = row_of(a, a.sums + (size_t(level - 1 & 1) * a.n_seqs + s) * a.chunks, uint32_t(r0) + at.cur, n.t);
      uint64_t tried;
      double w;
      next = next_node(tree, n, d, child, x, tried, w);
      if (first && threadIdx.x == next) {
        take_node(tree, n, d, at.depth, x);
        tree.path[size_t(s) * QE_TREE_NODES + level] = int32_t(next);
      }
    }
    if (first && threadIdx.x == 0)
      tree.walks[(level & 1) * a.n_seqs + s] = next != kNone ? Walk{next, level, 0, 0} : Walk{at.cur, at.depth, 1, 0};
    if (next == kNone) return;
    cur = next;
  } else if (first && threadIdx.x == 0) {
    tree.walks[s] = Walk{0, 0, 0, 0};
  }
  ChunkSum sum;
  const uint32_t r = uint32_t(r0) + cur;
  if (c >= a.chunks) return;  // (a wave that shares nothing, or, of WAVES > 1, none)
  float x[N];
  load_values(a.logits + r * a.stride, c0, a.vocab, -INFINITY, x);
  sum = chunk_sum<WAVES>(x, c0, temperature(a, s), shares);
  if (lane == 0 && (WAVES == 1 || wave == 0)) a.sums[(size_t(level & 1) * a.n_seqs + s) * a.chunks + c] = sum;
}

// A workgroup per sequence walks its tree (LEVELS: it is where k_tree_level left it, and only draws): every wave walks
// for itself, and all of them draw at the end.
template <bool LEVELS>
__global__ __launch_bounds__(kThreads) void k_tree_decide(TreeArgs tree, uint32_t levels) {
  constexpr int N = kChunk / kThreads;
  __shared__ Scratch sc;
  const DraftArgs& a = tree.d;
  const uint32_t s = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  int32_t* const path = tree.path + size_t(s) * QE_TREE_NODES;
  const Nodes nodes = nodes_of(tree, s);
  const int64_t r0 = nodes.r0, r1 = nodes.r1;
  if (r1 <= r0) {
    if (tid == 0) a.count[s] = 0;
    if (tid < QE_TREE_NODES) path[tid] = -1;
    return;
  }
  const float t = nodes.t;
  const uint32_t token = nodes.token;
  Walk at{};
  if constexpr (LEVELS) at = tree.walks[(levels - 1 & 1) * a.n_seqs + s];
  uint32_t cur = at.cur, depth = at.depth, mine = lane == 0 ? 0u : kNone;  // mine: the path's row at depth `lane`
  DrawRow d;
  const ChunkSum* sums;
  uint64_t tried;
  double w;
  while (true) {
    sums = a.sums + (LEVELS ? size_t(depth & 1) * a.n_seqs + s : size_t(r0) + cur) * a.chunks;
    float x;
    const bool child = is_child(tree, nodes, cur, depth, x);
    d = row_of(a, sums, uint32_t(r0) + cur, t);
    const uint32_t next = next_node(tree, nodes, d, child, x, tried, w);
    if (LEVELS || next == kNone) break;
    // (a wave for each, so that none waits for more than one logarithm)
    if (tid / 64 == depth % (kThreads / 64) && lane == next) take_node(tree, nodes, d, depth, x);
    depth++;
    if (lane == depth) mine = next;
    cur = next;
  }
  if (LEVELS && lane > 0 && lane <= depth) mine = uint32_t(path[lane]);
  if (tid < QE_TREE_NODES) path[tid] = int32_t(mine);
  if (tid == 0) a.count[s] = depth + 1;
  for (int64_t e = r0 + depth + 1 + tid; e < r1; e += kThreads) {
    a.tokens[e] = kNone;
    if (a.logprobs) a.logprobs[e] = 0.f;
  }
  // the draw: the chunks' sums without the tokens tried, then a chunk's tokens
  const uint32_t n = (a.chunks + 63) / 64, c0 = lane * n;
  double chunk[kLaneChunks], gone[kLaneChunks] = {}, before, aim = 0.0;
  auto plain_chunks = [&] {
#pragma unroll
    for (int i = 0; i < kLaneChunks; i++) {
      chunk[i] = 0.0;
      if (uint32_t(i) < n && c0 + i < a.chunks) {
        const ChunkSum z = sums[c0 + i];
        if (d.greedy) chunk[i] = d.best / kChunk == c0 + i ? 1.0 : 0.0;
        else chunk[i] = z.sum * chunk_scale(z.top, d.top, d.k);
      }
    }
  };
  // weights z and logits y of this thread's tokens of chunk c, those tried weigh nothing
  double z[N];
  f32x4 y;
  auto load_chunk = [&](uint32_t c) __attribute__((always_inline)) {
    const uint32_t i0 = c * kChunk + tid * N;
#pragma unroll
    for (int e = 0; e < N; e++) {
      z[e] = 0.0;
      y[e] = 0.f;
      if (c != kNone && i0 + e < a.vocab) {
        y[e] = a.logits[d.row * a.stride + i0 + e];
        z[e] = row_weight(d, i0 + e, y[e]);
      }
    }
    for (uint64_t rest = tried; rest; rest &= rest - 1) {
      const uint32_t is = from_lane(token, __builtin_ctzll(rest));
#pragma unroll
      for (int e = 0; e < N; e++)
        if (is == i0 + e) z[e] = 0.0;
    }
  };
  auto share = [&](double all) { return aim = double(a.sample[s]) * all; };
  plain_chunks();
  for (uint64_t rest = tried; rest; rest &= rest - 1) {
    const int c = __builtin_ctzll(rest);
    const uint32_t is = from_lane(token, c);
    const double less = from_lane(w, c);
#pragma unroll
    for (int i = 0; i < kLaneChunks; i++)
      if (uint32_t(i) < n && is < a.vocab && is / kChunk == c0 + i) gone[i] += less;
  }
  // A difference is off by some 2^-50 of the chunk's sum, so where 2^-26 of it or less is left (or the chunk weighs so
  // little that its other tokens may weigh 0) what is left is summed anew: no chunk has weight that its tokens have not.
  uint32_t thin = 0;
#pragma unroll
  for (int i = 0; i < kLaneChunks; i++) {
    const double whole = chunk[i];
    if (gone[i] > 0.0) chunk[i] = whole - gone[i];
    if (gone[i] > 0.0 && !(chunk[i] > 0x1p-26 * whole && whole > 0x1p-900)) thin |= 1u << i;
  }
  while (const uint64_t lanes = __ballot(thin)) {  // (every wave has the same)
    const int at = __builtin_ctzll(lanes);
    const uint32_t i = uint32_t(from_lane(uint32_t(__builtin_ctz(thin | 1u << 31)), at));
    load_chunk(uint32_t(at) * n + i);
    const double mine = wave_sum64((z[0] + z[1]) + (z[2] + z[3]));
    if (lane == 0) sc.wave[tid / 64] = mine;
    __syncthreads();
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < kThreads / 64; k++) sum += sc.wave[k];
    __syncthreads();
    if (int(lane) == at) {
      thin &= thin - 1;
#pragma unroll
      for (int k = 0; k < kLaneChunks; k++)
        if (uint32_t(k) == i) chunk[k] = sum;
    }
  }
  uint32_t c = find_chunk(chunk, n, share, before);
  if (c == kNone) {  // nothing is left: from p
    tried = 0;
    plain_chunks();
    c = find_chunk(chunk, n, share, before);
  }
  load_chunk(c);
  const uint32_t i0 = c * kChunk + tid * N;
  place_token(a, d, uint32_t(r0) + depth, i0, z, y, aim - before, t, sc);
}

struct DraftWork {
  uint64_t chunks, sums, rests, draws, bytes;  // byte offsets
};
DraftWork draft_work(uint64_t n_rows, uint64_t n_seqs, uint64_t vocab) {
  DraftWork w{};
  w.chunks = (vocab + kChunk - 1) / kChunk;
  w.rests = n_rows * w.chunks * sizeof(ChunkSum);
  w.draws = w.rests + n_seqs * w.chunks * sizeof(double);
  w.bytes = w.draws + n_seqs * sizeof(DrawRow);
  return w;
}

static_assert(2 * sizeof(Walk) <= sizeof(DrawRow), "a check by levels keeps its walks where draws lie");
// Whether a check goes level by level, a launch each that reads one row a sequence (5 us, 2 where every walk has ended), or
// sums all rows first (8 KB a chunk at 4.8 TB/s). Measured with 151,936 tokens and 8 levels, all rows and by levels: 8 trees
// of up to 26 nodes (173 rows, 22 us of reading) 34 and 39 us; 8 of up to 48 (325 rows, 42) 53 and 46; 24 of up to 48
// (881 rows, 113) 127 and 51. So from 4 us of reading for each level.
bool by_levels(uint64_t n_rows, uint64_t n_seqs, uint64_t chunks, uint64_t levels) {
  return n_rows >= 2 * n_seqs && double(n_rows * chunks) * 8192 / 4.8e6 > 4.0 * double(levels);
}

}  // namespace
}  // namespace qe

extern "C" {

uint64_t qe_op_verify_drafts_work_bytes(uint64_t n_rows, uint64_t n_seqs, uint64_t vocab) {
  if (vocab == 0 || vocab > qe::kMostVocab || n_rows > 0x7FFFFFFFull || n_seqs > 65535) return 0;
  return qe::draft_work(n_rows, n_seqs, vocab).bytes;
}

int qe_op_verify_drafts(const float* logits, uint64_t n_rows, uint64_t vocab, uint64_t row_stride,
                        const int32_t* starts, uint64_t n_seqs, const uint32_t* drafts, const float* draft_probs,
                        uint64_t probs_stride, const float* accept, const float* sample, const float* temperature,
                        uint32_t* tokens_out, uint32_t* count_out, float* logprobs_out, void* work,
                        uint64_t work_bytes, void* stream) {
  if (!starts || !sample || !count_out) return qe::set_error(QE_ERR_ARG, "null argument");
  if (n_seqs == 0 || n_seqs > 65535) return qe::set_error(QE_ERR_ARG, "n_seqs must be 1..65535");
  if (n_rows > 0x7FFFFFFFull) return qe::set_error(QE_ERR_ARG, "need n_rows < 2^31");
  if (!work) return qe::set_error(QE_ERR_ARG, "null argument");
  if (n_rows && (!logits || !drafts || !accept || !tokens_out)) return qe::set_error(QE_ERR_ARG, "null argument");
  if (vocab == 0 || vocab > qe::kMostVocab) return qe::set_error(QE_ERR_ARG, "vocab must be 1..%u", qe::kMostVocab);
  if (row_stride < vocab || (draft_probs && probs_stride < vocab) || row_stride > 0xFFFFFFFFull ||
      probs_stride > 0xFFFFFFFFull)
    return qe::set_error(QE_ERR_ARG, "row strides must be at least vocab and below 2^32");
  if (work_bytes < qe_op_verify_drafts_work_bytes(n_rows, n_seqs, vocab))
    return qe::set_error(QE_ERR_ARG, "work holds %llu bytes, fewer than qe_op_verify_drafts_work_bytes gives",
                         (unsigned long long)work_bytes);
  if (reinterpret_cast<uintptr_t>(work) % 16) return qe::set_error(QE_ERR_ARG, "work must be 16-byte aligned");
  const qe::DraftWork w = qe::draft_work(n_rows, n_seqs, vocab);
  uint8_t* const base = static_cast<uint8_t*>(work);
  qe::DraftArgs a{logits, draft_probs, starts, drafts, accept, sample, temperature, tokens_out, count_out,
                  logprobs_out, row_stride, probs_stride, uint32_t(n_rows), uint32_t(n_seqs), uint32_t(vocab),
                  uint32_t(w.chunks), reinterpret_cast<qe::ChunkSum*>(base), reinterpret_cast<double*>(base + w.rests),
                  reinterpret_cast<qe::DrawRow*>(base + w.draws)};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const uint32_t waves4 = qe::ceil_div(a.chunks, 4u);
  // (`rows` rows of chunks at hand: four waves for each)
  auto few = [&](uint64_t rows) { return rows * a.chunks <= qe::kFewChunks; };
  if (n_rows) {
    const uint32_t y = a.n_rows < qe::kRowsAcross ? a.n_rows : qe::kRowsAcross;
    const dim3 grid(few(a.n_rows) ? a.chunks : waves4, y, qe::ceil_div(a.n_rows, qe::kRowsAcross));
    (few(a.n_rows) ? qe::k_draft_sums<4> : qe::k_draft_sums<1>)<<<grid, 256, 0, st>>>(a);
  }
  qe::k_draft_decide<<<a.n_seqs, qe::kThreads, 0, st>>>(a);
  if (a.probs && n_rows) {
    (few(a.n_seqs) ? qe::k_draft_rest<4> : qe::k_draft_rest<1>)<<<dim3(few(a.n_seqs) ? a.chunks : waves4, a.n_seqs), 256, 0, st>>>(a);
    qe::k_draft_draw<<<a.n_seqs, qe::kThreads, 0, st>>>(a);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return qe::set_error(QE_ERR_HIP, "verify drafts launch failed: %s", hipGetErrorString(e));
  return QE_OK;
}

uint64_t qe_op_verify_tree_work_bytes(uint64_t n_rows, uint64_t n_seqs, uint64_t vocab) {
  return qe_op_verify_drafts_work_bytes(n_rows, n_seqs, vocab);
}

int qe_op_verify_tree(const float* logits, uint64_t n_rows, uint64_t vocab, uint64_t row_stride, const int32_t* starts,
                      uint64_t n_seqs, const int32_t* parents, const uint32_t* nodes, const float* accept,
                      const float* sample, const float* temperature, uint64_t max_depth, uint32_t* tokens_out,
                      int32_t* path_out, uint32_t* count_out, float* logprobs_out, void* work, uint64_t work_bytes,
                      void* stream) {
  if (!starts || !sample || !count_out || !path_out || !work) return qe::set_error(QE_ERR_ARG, "null argument");
  if (n_seqs == 0 || n_seqs > 65535) return qe::set_error(QE_ERR_ARG, "n_seqs must be 1..65535");
  if (n_rows > 0x7FFFFFFFull) return qe::set_error(QE_ERR_ARG, "need n_rows < 2^31");
  if (n_rows && (!logits || !parents || !nodes || !accept || !tokens_out)) return qe::set_error(QE_ERR_ARG, "null argument");
  if (vocab == 0 || vocab > qe::kMostVocab) return qe::set_error(QE_ERR_ARG, "vocab must be 1..%u", qe::kMostVocab);
  if (row_stride < vocab || row_stride > 0xFFFFFFFFull)
    return qe::set_error(QE_ERR_ARG, "row_stride must be at least vocab and below 2^32");
  if (work_bytes < qe_op_verify_tree_work_bytes(n_rows, n_seqs, vocab))
    return qe::set_error(QE_ERR_ARG, "work holds %llu bytes, fewer than qe_op_verify_tree_work_bytes gives",
                         (unsigned long long)work_bytes);
  if (reinterpret_cast<uintptr_t>(work) % 16) return qe::set_error(QE_ERR_ARG, "work must be 16-byte aligned");
  for (const void* p : {(const void*)logits, (const void*)starts, (const void*)parents, (const void*)nodes, (const void*)accept,
                        (const void*)sample, (const void*)temperature, (const void*)tokens_out, (const void*)path_out,
                        (const void*)count_out, (const void*)logprobs_out})
    if (reinterpret_cast<uintptr_t>(p) % 4) return qe::set_error(QE_ERR_ARG, "arrays must be 4-byte aligned");
  const qe::Bytes out[] = {{tokens_out, 4 * n_rows}, {path_out, 4 * QE_TREE_NODES * n_seqs}, {count_out, 4 * n_seqs},
                           {logprobs_out, 4 * n_rows}, {work, work_bytes}};
  const qe::Bytes in[] = {{logits, n_rows ? 4 * ((n_rows - 1) * row_stride + vocab) : 0}, {starts, 4 * (n_seqs + 1)},
                          {parents, 4 * n_rows}, {nodes, 4 * n_rows}, {accept, 4 * n_rows}, {sample, 4 * n_seqs},
                          {temperature, 4 * n_seqs}};
  for (int i = 0; i < 5; i++) {
    for (const qe::Bytes& b : in)
      if (out[i].meets(b)) return qe::set_error(QE_ERR_ARG, "outputs and work must not overlap the inputs");
    for (int j = 0; j < i; j++)
      if (out[i].meets(out[j])) return qe::set_error(QE_ERR_ARG, "outputs and work must not overlap each other");
  }
  const qe::DraftWork w = qe::draft_work(n_rows, n_seqs, vocab);
  uint8_t* const base = static_cast<uint8_t*>(work);
  qe::TreeArgs a{};
  a.d.logits = logits;
  a.d.starts = starts;
  a.d.drafts = nodes;
  a.d.accept = accept;
  a.d.sample = sample;
  a.d.temperature = temperature;
  a.d.tokens = tokens_out;
  a.d.count = count_out;
  a.d.logprobs = logprobs_out;
  a.d.stride = row_stride;
  a.d.n_rows = uint32_t(n_rows);
  a.d.n_seqs = uint32_t(n_seqs);
  a.d.vocab = uint32_t(vocab);
  a.d.chunks = uint32_t(w.chunks);
  a.d.sums = reinterpret_cast<qe::ChunkSum*>(base);
  a.parents = parents;
  a.path = path_out;
  a.max_depth = max_depth && max_depth < QE_TREE_NODES ? uint32_t(max_depth) : QE_TREE_NODES - 1;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const uint64_t levels = a.max_depth + 1;
  if (qe::by_levels(n_rows, n_seqs, w.chunks, levels)) {
    a.walks = reinterpret_cast<qe::Walk*>(base + w.draws);
    const bool few = n_seqs * w.chunks <= qe::kFewChunks;
    const dim3 grid(few ? a.d.chunks : qe::ceil_div(a.d.chunks, 4u), a.d.n_seqs);
    for (uint32_t l = 0; l < levels; l++) (few ? qe::k_tree_level<4> : qe::k_tree_level<1>)<<<grid, 256, 0, st>>>(a, l);
    qe::k_tree_decide<true><<<a.d.n_seqs, qe::kThreads, 0, st>>>(a, uint32_t(levels));
  } else {
    if (n_rows) {
      const bool few = n_rows * w.chunks <= qe::kFewChunks;
      const uint32_t y = a.d.n_rows < qe::kRowsAcross ? a.d.n_rows : qe::kRowsAcross;
      const dim3 grid(few ? a.d.chunks : qe::ceil_div(a.d.chunks, 4u), y, qe::ceil_div(a.d.n_rows, qe::kRowsAcross));
      (few ? qe::k_draft_sums<4> : qe::k_draft_sums<1>)<<<grid, 256, 0, st>>>(a.d);
    }
    qe::k_tree_decide<false><<<a.d.n_seqs, qe::kThreads, 0, st>>>(a, 0);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return qe::set_error(QE_ERR_HIP, "verify tree launch failed: %s", hipGetErrorString(e));
  return QE_OK;
}

}  // extern "C"
