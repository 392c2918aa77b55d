// qe_op_verify_drafts: drafted tokens checked against the target's probabilities, from given random
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
// Bound by one read of the logits. k_draft_sums reads every row once, a wave per chunk of 2048 tokens,
// and keeps each chunk's largest logit and its sum of weights relative to that one. k_draft_decide, a
// workgroup per sequence, joins the chunks of each row, accepts drafts (a gather each) and finds the
// row that draws; with no draft probabilities the chunk sums already hold the running sum at chunk
// borders, so it also draws, reading one chunk again. With them k_draft_rest sums max(p - q, 0) of the
// drawing rows by chunks and k_draft_draw draws.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "../../include/qe.h"
#include "device_common.h"
#include "status.h"

namespace qe {
namespace {

// What a chunk of a row adds up to: weights relative to its own largest logit.
struct ChunkSum {
  double sum;
  float top;      // -inf: nothing above -inf
  uint32_t best;  // first index of top
};

// The row a sequence draws from.
struct DrawRow {
  double inv_total, k;  // 1 / sum of weights; log2(e) / T
  double log_total;
  uint32_t row;         // 0xFFFFFFFF: the sequence draws nothing here
  uint32_t best, draft;
  float top, inv_t;
  uint32_t greedy;
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

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

// 2^t in 64 bits for t <= 0 (6e-16; 0 below -1075): t = n + f with n the nearest whole number, and
// 2^f = 1 + f c(f) by Chebyshev interpolation of (2^f - 1) / f at 10 points of [-1/2, 1/2]. 2^0 is
// exactly 1. (The library's exp is some 40 instructions on the same unit, which then bounds the pass
// instead of the memory.)
__device__ __forceinline__ double exp2_64(double t) {
  t = fmax(t, -1100.0);
  const double n = rint(t), f = t - n;
  double c = 7.070977866508138e-09;
  c = fma(c, f, 1.0205905413765595e-07);
  c = fma(c, f, 1.3215451633221434e-06);
  c = fma(c, f, 1.5252672924850737e-05);
  c = fma(c, f, 0.00015403530424776529);
  c = fma(c, f, 0.0013333558200794592);
  c = fma(c, f, 0.009618129107618665);
  c = fma(c, f, 0.05550410866465167);
  c = fma(c, f, 0.24022650695910075);
  c = fma(c, f, 0.6931471805599462);
  return ldexp(fma(c, f, 1.0), int(n));
}

// weight of logit x relative to the largest one, top: NaN and -inf weigh nothing, infinite ones share
__device__ __forceinline__ double weight(float x, float top, double k) {
  if (x == top) return 1.0;
  if (!(x > -INFINITY) || top == INFINITY) return 0.0;
  return exp2_64((double(x) - double(top)) * k);
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
  return v;
}

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

// 32 values of a chunk of a row of n: value 4 i + e of lane l is token c0 + 256 i + 4 l + e; `pad` behind the row
__device__ __forceinline__ void load_chunk(const float* row, uint32_t c0, uint32_t n, float pad, float (&x)[32]) {
  const uint32_t lane = threadIdx.x & 63;
  if (c0 + kChunk <= n) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const f32x4u v = *reinterpret_cast<const f32x4u*>(row + c0 + 256 * i + 4 * lane);
#pragma unroll
      for (int e = 0; e < 4; e++) x[4 * i + e] = v[e];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const uint32_t t = c0 + 256 * i + 4 * lane + e;
        x[4 * i + e] = t < n ? row[t] : pad;
      }
  }
}

// A wave per (row, chunk).
__global__ __launch_bounds__(256) void k_draft_sums(DraftArgs a) {
  const uint32_t lane = threadIdx.x & 63;
  const uint32_t c = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)), r = blockIdx.y + blockIdx.z * 32768;
  if (c >= a.chunks || r >= a.n_rows) return;
  float x[32];
  load_chunk(a.logits + r * a.stride, c * kChunk, a.vocab, -INFINITY, x);
  const int32_t s = sequence(a, int32_t(r));
  if (s < 0) return;
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < 32; i++) m = fmaxf(m, x[i]);
  m = wave_max(m);
  uint32_t at = kNone;  // the first place that holds it
#pragma unroll
  for (int i = 31; i >= 0; i--)
    if (x[i] == m) at = c * kChunk + 256 * (i / 4) + 4 * lane + i % 4;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) at = min(at, uint32_t(__shfl_xor(int(at), d)));
  const float t = temperature(a, s);
  double sum = 0.0;
  if (t > 0.f && m > -INFINITY) {
    const double k = rate(t);
#pragma unroll
    for (int i = 0; i < 32; i++) sum += weight(x[i], m, k);
    sum = wave_sum64(sum);
  }
  if (lane == 0) a.sums[size_t(r) * a.chunks + c] = ChunkSum{sum, m, at};
}

// ---- a workgroup's own sums ----
struct Scratch {
  double wave[kThreads / 64];
  double of[kThreads];
  uint32_t pick, some;
  double before;
  double without;
};

// running sum of v over the threads up to and with this one, and the sum of all
__device__ double running_sum(double v, Scratch& sc, double& all) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const double u = __shfl_up(v, d);
    if (int(lane) >= d) v += u;
  }
  __syncthreads();
  if (lane == 63) sc.wave[wave] = v;
  __syncthreads();
  double before = 0.0;
  all = 0.0;
#pragma unroll
  for (uint32_t i = 0; i < kThreads / 64; i++) {
    if (i < wave) before += sc.wave[i];
    all += sc.wave[i];
  }
  return before + v;
}

// The first of n items (item i weighs w(i), thread t asks for a contiguous range of them) whose running
// sum is above goal(sum of all), and the running sum before it. If rounding leaves none, the last with
// any weight; kNone if nothing has any.
template <class W, class Goal>
__device__ uint32_t find_item(uint32_t n, W w, Goal goal, Scratch& sc, double& before, double& all) {
  const uint32_t per = (n + kThreads - 1) / kThreads, i0 = min(threadIdx.x * per, n), i1 = min(i0 + per, n);
  double mine = 0.0;
  uint32_t some = kNone;
  for (uint32_t i = i0; i < i1; i++) {
    const double v = w(i);
    mine += v;
    if (v > 0.0) some = i;
  }
  const double up_to = running_sum(mine, sc, all);
  const double aim = goal(all);
  if (threadIdx.x == 0) {
    sc.pick = kNone;
    sc.some = 0;
  }
  __syncthreads();
  if (some != kNone) atomicMax(&sc.some, some + 1);
  if (some != kNone && up_to > aim) atomicMin(&sc.pick, threadIdx.x);
  __syncthreads();
  const uint32_t owner = sc.pick, last = sc.some;
  __syncthreads();
  if (owner == kNone) {  // not above the aim anywhere: the last item that has weight
    if (last != 0 && last - 1 >= i0 && last - 1 < i1) sc.before = up_to - w(last - 1);
    __syncthreads();
    before = sc.before;
    return last == 0 ? kNone : last - 1;
  }
  if (threadIdx.x == owner) {
    double run = up_to - mine;
    for (uint32_t i = i0; i < i1; i++) {
      const double v = w(i);
      if (v > 0.0 && (run + v > aim || i == some)) {
        sc.pick = i;
        sc.before = run;
        break;
      }
      run += v;
    }
  }
  __syncthreads();
  before = sc.before;
  return sc.pick;
}

// sum of the chunk's weights from one logit to another: the chunk's largest to the row's
__device__ __forceinline__ double chunk_scale(float from, const DrawRow& d) {
  if (from == d.top) return 1.0;
  if (!(from > -INFINITY) || d.top == INFINITY) return 0.0;
  return exp2_64((double(from) - double(d.top)) * d.k);
}

// One token of row d.row: over the chunks by their sums, then within a chunk. REST: from max(p - q, 0).
template <bool REST>
__device__ void draw(const DraftArgs& a, uint32_t s, const DrawRow& d, bool last, Scratch& sc) {
  const float* x = a.logits + d.row * a.stride;
  const float* q = REST ? a.probs + d.row * a.probs_stride : nullptr;
  const uint32_t skip = last || a.probs ? kNone : d.draft;  // a drafted token that has all of q
  const double v = double(a.sample[s]);
  auto token_weight = [&](uint32_t i) -> double {
    if (d.greedy) return i == d.best ? 1.0 : 0.0;
    return weight(x[i], d.top, d.k);
  };
  auto rest_weight = [&](uint32_t i) -> double {
    if (i == skip) return 0.0;
    const double w = token_weight(i);
    if constexpr (REST) {
      const float qi = q[i];
      return qi > 0.f ? fmax(w * d.inv_total - double(qi), 0.0) : w * d.inv_total;
    }
    return w;
  };
  auto plain_chunk = [&](uint32_t c) -> double {
    if (d.greedy) return d.best / kChunk == c ? 1.0 : 0.0;
    const ChunkSum p = a.sums[size_t(d.row) * a.chunks + c];
    return p.sum * chunk_scale(p.top, d);
  };
  if (skip < a.vocab) {  // its chunk's sum without it
    const uint32_t c0 = skip / kChunk * kChunk, n = min(kChunk, a.vocab - c0);
    double mine = 0.0, all;
    for (uint32_t i = threadIdx.x * (kChunk / kThreads); i < min((threadIdx.x + 1) * (kChunk / kThreads), n); i++)
      mine += rest_weight(c0 + i);
    running_sum(mine, sc, all);
    if (threadIdx.x == 0) sc.without = all;
    __syncthreads();
  }
  const double without = sc.without;
  double before, all, inner, unused;
  auto chunk_weight = [&](uint32_t c) -> double {
    if constexpr (REST) return a.rests[size_t(s) * a.chunks + c];
    return skip < a.vocab && skip / kChunk == c ? without : plain_chunk(c);
  };
  double aim = 0.0;
  auto goal = [&](double sum) { return aim = v * sum; };
  uint32_t c = find_item(a.chunks, chunk_weight, goal, sc, before, all);
  bool plain = false;
  if (c == kNone) {  // nothing is left of p - q: from p
    plain = true;
    c = find_item(a.chunks, plain_chunk, goal, sc, before, all);
  }
  const uint32_t c0 = c == kNone ? 0 : c * kChunk, n = c == kNone ? 0 : min(kChunk, a.vocab - c0);
  const double to = aim - before;
  const uint32_t i = find_item(
      n, [&](uint32_t k) { return plain ? token_weight(c0 + k) : rest_weight(c0 + k); },
      [&](double) { return to; }, sc, inner, unused);
  if (threadIdx.x == 0) {
    const uint32_t token = i == kNone ? d.best : c0 + i;
    a.tokens[d.row] = token;
    if (a.logprobs)
      a.logprobs[d.row] =
          d.greedy ? 0.f : float((x[token] == d.top ? 0.0 : (double(x[token]) - double(d.top)) / double(temperature(a, s))) - d.log_total);
  }
}

// A workgroup per sequence: a wave joins the chunks of one row after another.
__global__ __launch_bounds__(kThreads) void k_draft_decide(DraftArgs a) {
  constexpr uint32_t BATCH = 64, WAVES = kThreads / 64;
  __shared__ Scratch sc;
  __shared__ DrawRow rows[BATCH];
  __shared__ float logp[BATCH];
  __shared__ uint32_t taken[BATCH];
  const uint32_t s = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t r0 = max(a.starts[s], 0), r1 = min(int64_t(a.starts[s + 1]), int64_t(a.n_rows));
  if (r1 <= r0) {
    if (threadIdx.x == 0) {
      a.count[s] = 0;
      a.draws[s].row = kNone;
    }
    return;
  }
  const float t = temperature(a, s);
  const double k = rate(t);
  int64_t stop = -1;
  for (int64_t b = r0; stop < 0; b += BATCH) {
    const uint32_t n = uint32_t(min(r1 - b, int64_t(BATCH)));
    for (uint32_t i = wave; i < n; i += WAVES) {
      const uint32_t r = uint32_t(b) + i;
      const ChunkSum* p = a.sums + size_t(r) * a.chunks;
      float top = -INFINITY;
      for (uint32_t c = lane; c < a.chunks; c += 64) top = fmaxf(top, p[c].top);
      top = wave_max(top);
      DrawRow d;
      d.top = top;
      d.k = k;
      d.greedy = !(t > 0.f) || !(top > -INFINITY);
      d.row = r;
      d.draft = a.drafts[r];
      uint32_t best = kNone;
      double sum = 0.0;
      for (uint32_t c = lane; c < a.chunks; c += 64) {
        const ChunkSum z = p[c];
        if (z.top == top && top > -INFINITY) best = min(best, z.best);
        if (!d.greedy) sum += z.sum * chunk_scale(z.top, d);
      }
#pragma unroll
      for (int e = 1; e < 64; e *= 2) best = min(best, uint32_t(__shfl_xor(int(best), e)));
      d.best = best < a.vocab ? best : 0;  // (top is -inf: the first token)
      sum = d.greedy ? 1.0 : wave_sum64(sum);
      d.inv_total = 1.0 / sum;
      d.log_total = log(sum);
      if (lane == 0) {
        rows[i] = d;
        bool yes = false;
        if (r + 1 < r1 && d.draft < a.vocab) {
          const float x = a.logits[r * a.stride + d.draft];
          const double w = d.greedy ? (d.draft == d.best ? 1.0 : 0.0) : weight(x, top, k);
          double qd = 1.0;
          if (a.probs) {
            const float y = a.probs[r * a.probs_stride + d.draft];
            qd = y > 0.f ? double(y) : 0.0;
          }
          yes = double(a.accept[r]) * qd < w * d.inv_total;
          logp[i] = d.greedy ? 0.f : float((x == top ? 0.0 : (double(x) - double(top)) / double(t)) - d.log_total);
        }
        taken[i] = yes;
      }
    }
    __syncthreads();
    uint32_t first = 0;
    while (first < n && taken[first]) first++;
    for (uint32_t i = threadIdx.x; i < first; i += kThreads) {
      a.tokens[b + i] = rows[i].draft;
      if (a.logprobs) a.logprobs[b + i] = logp[i];
    }
    if (first < n) stop = b + first;
    else __syncthreads();
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
  if (!rest) draw<false>(a, s, d, last, sc);
}

// A wave per (sequence, chunk): the sum of max(p - q, 0) over a chunk of the row that draws.
__global__ __launch_bounds__(256) void k_draft_rest(DraftArgs a) {
  const uint32_t lane = threadIdx.x & 63;
  const uint32_t c = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)), s = blockIdx.y;
  if (c >= a.chunks) return;
  const DrawRow d = a.draws[s];
  if (d.row == kNone) return;
  float x[32], q[32];
  load_chunk(a.logits + d.row * a.stride, c * kChunk, a.vocab, -INFINITY, x);
  load_chunk(a.probs + d.row * a.probs_stride, c * kChunk, a.vocab, 0.f, q);
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < 32; i++) {
    const uint32_t token = c * kChunk + 256 * (i / 4) + 4 * lane + i % 4;
    const double w = (d.greedy ? (token == d.best ? 1.0 : 0.0) : weight(x[i], d.top, d.k)) * d.inv_total;
    sum += q[i] > 0.f ? fmax(w - double(q[i]), 0.0) : w;
  }
  sum = wave_sum64(sum);
  if (lane == 0) a.rests[size_t(s) * a.chunks + c] = sum;
}

__global__ __launch_bounds__(kThreads) void k_draft_draw(DraftArgs a) {
  __shared__ Scratch sc;
  const uint32_t s = blockIdx.x;
  const DrawRow d = a.draws[s];
  if (d.row == kNone) return;
  draw<true>(a, s, d, false, sc);
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

}  // namespace
}  // namespace qe

extern "C" {

uint64_t qe_op_verify_drafts_work_bytes(uint64_t n_rows, uint64_t n_seqs, uint64_t vocab) {
  if (vocab == 0 || vocab > 0x7FFFFFFFull || n_rows > 0x7FFFFFFFull || n_seqs > 65535) return 0;
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
  if (vocab == 0 || vocab > 0x7FFFFFFFull) return qe::set_error(QE_ERR_ARG, "need 0 < vocab < 2^31");
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
  if (n_rows) {
    const uint32_t y = a.n_rows < 32768 ? a.n_rows : 32768;
    qe::k_draft_sums<<<dim3(waves4, y, qe::ceil_div(a.n_rows, 32768u)), 256, 0, st>>>(a);
  }
  qe::k_draft_decide<<<a.n_seqs, qe::kThreads, 0, st>>>(a);
  if (a.probs && n_rows) {
    qe::k_draft_rest<<<dim3(waves4, a.n_seqs), 256, 0, st>>>(a);
    qe::k_draft_draw<<<a.n_seqs, qe::kThreads, 0, st>>>(a);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return qe::set_error(QE_ERR_HIP, "verify drafts launch failed: %s", hipGetErrorString(e));
  return QE_OK;
}

}  // extern "C"
