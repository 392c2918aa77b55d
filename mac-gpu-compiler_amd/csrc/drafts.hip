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
// that f32 would give.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "../../include/qe.h"
#include "device_common.h"
#include "status.h"

namespace qe {
namespace {

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
  uint32_t n_rows, n_seqs, vocab;
};

constexpr int kThreads = 256;

// sum of the workgroup's values in a fixed order, to every thread
__device__ double block_sum(double v, double* smem) {
  const int t = threadIdx.x;
  __syncthreads();
  smem[t] = v;
  __syncthreads();
  for (int n = kThreads / 2; n > 0; n /= 2) {
    if (t < n) smem[t] += smem[t + n];
    __syncthreads();
  }
  return smem[0];
}

// What a row's logits say: NaN counts as -inf; with nothing above -inf token 0 has all the weight.
struct Row {
  const float* x;
  float top;       // largest logit
  uint32_t best;   // its first index
  bool greedy;     // all the weight on `best`
  double inv_t, total;
  // weight of token i relative to the largest
  __device__ double weight(uint32_t i) const {
    if (greedy) return i == best ? 1.0 : 0.0;
    const float v = x[i];
    if (v == top) return 1.0;  // +inf too
    if (!(v > -INFINITY) || top == INFINITY) return 0.0;
    return exp((double(v) - double(top)) * inv_t);
  }
};

__device__ Row read_row(const DraftArgs& a, uint32_t r, float temp, double* smem) {
  Row row;
  row.x = a.logits + r * a.stride;
  float m = -INFINITY;
  uint32_t mi = 0;
  for (uint32_t i = threadIdx.x; i < a.vocab; i += kThreads) {
    const float v = row.x[i];
    if (v > m) {
      m = v;
      mi = i;
    }
  }
  __shared__ float fm[kThreads];
  __shared__ uint32_t fi[kThreads];
  __syncthreads();
  fm[threadIdx.x] = m;
  fi[threadIdx.x] = mi;
  __syncthreads();
  for (int n = kThreads / 2; n > 0; n /= 2) {
    if (int(threadIdx.x) < n && cand_better(fm[threadIdx.x + n], fi[threadIdx.x + n], fm[threadIdx.x], fi[threadIdx.x])) {
      fm[threadIdx.x] = fm[threadIdx.x + n];
      fi[threadIdx.x] = fi[threadIdx.x + n];
    }
    __syncthreads();
  }
  row.top = fm[0];
  row.best = row.top > -INFINITY ? fi[0] : 0;
  row.greedy = !(temp > 0.f) || !(row.top > -INFINITY);
  row.inv_t = 1.0 / double(temp);
  double sum = 0.0;
  if (!row.greedy)
    for (uint32_t i = threadIdx.x; i < a.vocab; i += kThreads) sum += row.weight(i);
  row.total = block_sum(sum, smem);
  if (row.greedy) row.total = 1.0;
  return row;
}

// One workgroup per sequence, its rows one after the other.
__global__ __launch_bounds__(kThreads) void k_verify_drafts(DraftArgs a) {
  __shared__ double smem[kThreads];
  __shared__ uint32_t pick;
  const uint32_t s = blockIdx.x;
  const int64_t r0 = max(a.starts[s], 0), r1 = min(int64_t(a.starts[s + 1]), int64_t(a.n_rows));
  if (r1 <= r0) {
    if (threadIdx.x == 0) a.count[s] = 0;
    return;
  }
  const float temp = a.temperature ? a.temperature[s] : 1.f;
  for (int64_t r = r0; r < r1; r++) {
    const Row row = read_row(a, uint32_t(r), temp, smem);
    const bool last = r == r1 - 1;
    const float* q = a.probs && !last ? a.probs + r * a.probs_stride : nullptr;
    const uint32_t d = a.drafts[r];
    const double inv = 1.0 / row.total;
    if (!last && d < a.vocab) {
      const double w = row.weight(d), qd = q ? (q[d] > 0.f ? double(q[d]) : 0.0) : 1.0;
      if (double(a.accept[r]) * qd < w * inv) {
        if (threadIdx.x == 0) {
          a.tokens[r] = d;
          if (a.logprobs) a.logprobs[r] = float(log(w) - log(row.total));
        }
        continue;
      }
    }
    // without a distribution to subtract the weights stay as they are: equal ones are exactly equal
    auto rest = [&](uint32_t i) -> double {
      const double w = row.weight(i);
      if (last) return w;
      if (!a.probs) return i == d ? 0.0 : w;
      const float qi = q[i];
      return qi > 0.f ? fmax(w * inv - double(qi), 0.0) : w * inv;
    };
    // thread t owns a contiguous range of tokens
    const uint32_t per = (a.vocab + kThreads - 1) / kThreads, i0 = min(threadIdx.x * per, a.vocab),
                   i1 = min(i0 + per, a.vocab);
    bool plain = false;
    double mine = 0.0;
    for (uint32_t i = i0; i < i1; i++) mine += rest(i);
    if (!(block_sum(mine, smem) > 0.0)) {  // p and q are the same: from p
      plain = true;
      mine = 0.0;
      for (uint32_t i = i0; i < i1; i++) mine += row.weight(i);
    }
    __syncthreads();
    smem[threadIdx.x] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
      double all = 0.0;
      for (int t = 0; t < kThreads; t++) all += smem[t];
      const double goal = double(a.sample[s]) * all;
      double before = 0.0;
      int at = -1, some = 0;
      for (int t = 0; t < kThreads && at < 0; t++) {
        if (smem[t] > 0.0) some = t;
        if (before + smem[t] > goal) at = t;
        else before += smem[t];
      }
      if (at < 0) at = some;
      uint32_t tok = 0;
      for (uint32_t i = at * per; i < min((at + 1) * per, a.vocab); i++) {
        const double w = plain ? row.weight(i) : rest(i);
        before += w;
        if (w > 0.0) tok = i;
        if (w > 0.0 && before > goal) break;
      }
      pick = tok;
      a.tokens[r] = tok;
      a.count[s] = uint32_t(r - r0 + 1);
      if (a.logprobs) a.logprobs[r] = float(log(row.weight(tok)) - log(row.total));
    }
    for (int64_t e = r + 1 + threadIdx.x; e < r1; e += kThreads) {
      a.tokens[e] = 0xFFFFFFFFu;
      if (a.logprobs) a.logprobs[e] = 0.f;
    }
    return;
  }
}

}  // namespace
}  // namespace qe

extern "C" {

uint64_t qe_op_verify_drafts_work_bytes(uint64_t n_rows, uint64_t n_seqs, uint64_t vocab) {
  (void)n_rows;
  (void)n_seqs;
  (void)vocab;
  return 256;
}

int qe_op_verify_drafts(const float* logits, uint64_t n_rows, uint64_t vocab, uint64_t row_stride,
                        const int32_t* starts, uint64_t n_seqs, const uint32_t* drafts, const float* draft_probs,
                        uint64_t probs_stride, const float* accept, const float* sample, const float* temperature,
                        uint32_t* tokens_out, uint32_t* count_out, float* logprobs_out, void* work,
                        uint64_t work_bytes, void* stream) {
  if (!starts || !sample || !count_out) return qe::set_error(QE_ERR_ARG, "null argument");
  if (n_seqs == 0 || n_seqs > 65535) return qe::set_error(QE_ERR_ARG, "n_seqs must be 1..65535");
  if (n_rows > 0x7FFFFFFFull) return qe::set_error(QE_ERR_ARG, "need n_rows < 2^31");
  if (n_rows && (!logits || !drafts || !accept || !tokens_out || !work)) return qe::set_error(QE_ERR_ARG, "null argument");
  if (vocab == 0 || vocab > 0x7FFFFFFFull) return qe::set_error(QE_ERR_ARG, "need 0 < vocab < 2^31");
  if (row_stride < vocab || (draft_probs && probs_stride < vocab) || row_stride > 0xFFFFFFFFull ||
      probs_stride > 0xFFFFFFFFull)
    return qe::set_error(QE_ERR_ARG, "row strides must be at least vocab and below 2^32");
  if (work_bytes < qe_op_verify_drafts_work_bytes(n_rows, n_seqs, vocab))
    return qe::set_error(QE_ERR_ARG, "work holds %llu bytes, fewer than qe_op_verify_drafts_work_bytes gives",
                         (unsigned long long)work_bytes);
  qe::DraftArgs a{logits, draft_probs, starts, drafts, accept, sample, temperature, tokens_out, count_out,
                  logprobs_out, row_stride, probs_stride, uint32_t(n_rows), uint32_t(n_seqs), uint32_t(vocab)};
  qe::k_verify_drafts<<<uint32_t(n_seqs), qe::kThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return qe::set_error(QE_ERR_HIP, "verify drafts launch failed: %s", hipGetErrorString(e));
  return QE_OK;
}

}  // extern "C"
