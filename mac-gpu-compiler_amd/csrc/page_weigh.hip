// qe_op_page_weigh: the softmax weight that each cached position gets from new tokens, added up per
// sequence and KV head. No reference counterpart.
//
//   mass[s][h][j] += sum over rows t, q heads g of KV head h of w_tg(j),
//   w_tg(j) = exp(x_tg(j) - m_tg) / sum_i exp(x_tg(i) - m_tg),  x_tg(j) = q[t][g] . k_j / sqrt(128)
//
// k_weigh_rows takes each row's maximum and sum, k_weigh_mass each position's weights, in row order:
// one thread owns an entry of mass, so sums are the same every time.
#include "pages.h"

#include "device_common.h"
#include "status.h"

#include <cmath>

namespace qe {
namespace {

struct WeighArgs {
  PagePlan p;
  PageStore st;
  const uint8_t* q;
  uint64_t q_stride;
  float* mass;
  uint64_t mass_stride;
  float2* rows;  // [n_rows][heads]: maximum, 1 / sum
  uint32_t n_rows, group;
  float c;  // log2(e) / sqrt(128)
};

struct Span {
  int64_t first;      // position of its first row
  int32_t row0, rows;  // packed rows
};
__device__ __forceinline__ Span span_of(const WeighArgs& a, uint32_t s) {
  const int64_t b = a.p.starts[s], e = a.p.starts[s + 1], lo = b < 0 ? 0 : b, hi = e < a.n_rows ? e : a.n_rows;
  return {int64_t(a.p.lens[s]) - (e - lo), int32_t(lo), hi > lo ? int32_t(hi - lo) : 0};
}

template <bool FP8, bool BF16_ROWS>
__device__ float score(const WeighArgs& a, uint32_t t, uint32_t h, size_t row) {
  float s = 0.f;
  const uint64_t e = uint64_t(t) * a.q_stride + h * kPageDim;
  for (uint32_t d = 0; d < kPageDim; d++) {
    const float q = BF16_ROWS ? bf16f(reinterpret_cast<const uint16_t*>(a.q)[e + d]) : reinterpret_cast<const float*>(a.q)[e + d];
    const float k = FP8 ? __builtin_amdgcn_cvt_f32_fp8(a.st.k[row * kPageDim + d], 0)
                        : bf16f(reinterpret_cast<const uint16_t*>(a.st.k)[row * kPageDim + d]);
    s = fmaf(q, k, s);
  }
  return (FP8 ? s * exp_scale(a.st.k_exp[row]) : s) * a.c;
}

// a wave for each row and q head
template <bool FP8, bool BF16_ROWS>
__global__ __launch_bounds__(64) void k_weigh_rows(WeighArgs a) {
  const uint32_t heads = a.group * a.p.n_kv, t = blockIdx.x / heads, h = blockIdx.x - t * heads, lane = threadIdx.x;
  uint32_t lo = 0, hi = a.p.n_seqs;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (a.p.starts[mid] <= int32_t(t)) lo = mid;
    else hi = mid;
  }
  const Span q = span_of(a, lo);
  if (int32_t(t) < q.row0 || int32_t(t) >= q.row0 + q.rows) return;
  const int64_t end = min(q.first + (int32_t(t) - q.row0) + 1, capacity_of(a.p));
  float m = -INFINITY, l = 0.f;
  for (int64_t x = 0; x < end; x += 64) {
    const int64_t j = x + lane;
    const int32_t page = j < end ? page_of(a.p, lo, j) : -1;
    float s = -INFINITY;
    if (page >= 0) s = score<FP8, BF16_ROWS>(a, t, h, page_row(a.p, page, h / a.group, uint32_t(j) & ((1u << a.p.page_shift) - 1)));
    const float top = fmaxf(m, wave_max(s));
    l = l * (m == top ? 1.f : exp2f(m - top)) + wave_sum(s == -INFINITY ? 0.f : exp2f(s - top));
    m = top;
  }
  if (lane == 0) a.rows[uint64_t(t) * heads + h] = make_float2(m, l == 0.f ? 0.f : 1.f / l);
}

// a thread for each position of a sequence and KV head
template <bool FP8, bool BF16_ROWS>
__global__ __launch_bounds__(256) void k_weigh_mass(WeighArgs a, uint32_t blocks) {
  const uint32_t item = blockIdx.x / blocks, s = item / a.p.n_kv, kv = item - s * a.p.n_kv;
  const int64_t j = int64_t(blockIdx.x - item * blocks) * 256 + threadIdx.x;
  const Span q = span_of(a, s);
  if (j >= capacity_of(a.p) || j >= q.first + q.rows) return;
  const int32_t page = page_of(a.p, s, j);
  if (page < 0) return;
  const size_t row = page_row(a.p, page, kv, uint32_t(j) & ((1u << a.p.page_shift) - 1));
  float sum = 0.f;
  for (int32_t i = j < q.first ? 0 : int32_t(j - q.first); i < q.rows; i++)
    for (uint32_t g = 0; g < a.group; g++) {
      const uint32_t t = uint32_t(q.row0 + i), h = kv * a.group + g;
      const float2 r = a.rows[uint64_t(t) * a.group * a.p.n_kv + h];
      const float x = score<FP8, BF16_ROWS>(a, t, h, row);
      sum += x == -INFINITY && r.x == -INFINITY ? 0.f : exp2f(x - r.x) * r.y;
    }
  a.mass[(uint64_t(s) * a.p.n_kv + kv) * a.mass_stride + j] += sum;
}

}  // namespace
}  // namespace qe

extern "C" {

uint64_t qe_op_page_weigh_work_bytes(uint64_t n_rows, uint64_t n_heads, uint64_t n_kv_heads, uint64_t n_seqs,
                                     uint64_t positions, uint64_t max_new) {
  if (!n_kv_heads || !n_heads || n_heads % n_kv_heads) return 0;
  return n_rows * n_heads * sizeof(float2);
}

int qe_op_page_weigh(const qe_pages* pages, const void* q, uint64_t n_rows, uint64_t n_heads, uint64_t q_stride,
                     uint64_t max_new, int dtype, float* mass, uint64_t mass_stride, void* work, uint64_t work_bytes,
                     void* stream) {
  qe::WeighArgs a{};
  if (int rc = qe::check_pages(pages, &a.p, &a.st)) return rc;
  if (dtype != QE_KV_F32 && dtype != QE_KV_BF16) return qe::set_error(QE_ERR_ARG, "rows are QE_KV_F32 or QE_KV_BF16");
  if (n_heads == 0 || n_heads % a.p.n_kv || n_heads > 65536)
    return qe::set_error(QE_ERR_ARG, "n_heads must be a multiple of n_kv_heads, at most 65536");
  if (n_rows == 0) return QE_OK;
  if (!q || !mass || !work) return qe::set_error(QE_ERR_ARG, "null argument");
  if (n_rows > 0x7FFFFFFFull / n_heads) return qe::set_error(QE_ERR_ARG, "need n_rows * n_heads < 2^31");
  const uint64_t el = dtype == QE_KV_F32 ? 4 : 2, capacity = pages->table_stride * pages->page_size;
  if (q_stride < n_heads * qe::kPageDim || q_stride > 0xFFFFFFFFull || q_stride * el % 16)
    return qe::set_error(QE_ERR_ARG, "q_stride must be at least n_heads * 128 elements and a multiple of 16 bytes");
  if (mass_stride < capacity || mass_stride > 0x7FFFFFFFull)
    return qe::set_error(QE_ERR_ARG, "mass_stride must be at least table_stride * page_size, and below 2^31");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(work)) % 16 || reinterpret_cast<uintptr_t>(mass) % 4)
    return qe::set_error(QE_ERR_ARG, "q and work must be 16-byte aligned, mass 4-byte");
  if (work_bytes < qe_op_page_weigh_work_bytes(n_rows, n_heads, a.p.n_kv, a.p.n_seqs, capacity, max_new))
    return qe::set_error(QE_ERR_ARG, "work holds %llu bytes, fewer than qe_op_page_weigh_work_bytes gives",
                         (unsigned long long)work_bytes);
  const qe::Bytes to{mass, 4 * mass_stride * a.p.n_seqs * a.p.n_kv};
  const uint64_t page_bytes = qe_page_bytes(pages->n_pages, pages->page_size, pages->n_kv_heads, pages->kv_dtype);
  const bool fp8 = pages->kv_dtype == QE_KV_FP8;
  if (to.meets({q, ((n_rows - 1) * q_stride + n_heads * qe::kPageDim) * el}) || to.meets({pages->k, page_bytes}) ||
      to.meets({pages->v, page_bytes}) || to.meets({work, work_bytes}) ||
      (fp8 && (to.meets({pages->k_exp, page_bytes / qe::kPageDim}) || to.meets({pages->v_exp, page_bytes / qe::kPageDim}))))
    return qe::set_error(QE_ERR_ARG, "mass must not overlap q, the pages or work");
  a.q = static_cast<const uint8_t*>(q);
  a.q_stride = q_stride;
  a.mass = mass;
  a.mass_stride = mass_stride;
  a.rows = static_cast<float2*>(work);
  a.n_rows = uint32_t(n_rows);
  a.group = uint32_t(n_heads / a.p.n_kv);
  a.c = 1.44269504f / sqrtf(float(qe::kPageDim));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const uint32_t blocks = uint32_t((capacity + 255) / 256);
  auto go = [&](auto* rows, auto* sums) {
    rows<<<uint32_t(n_rows * n_heads), 64, 0, st>>>(a);
    sums<<<blocks * a.p.n_seqs * a.p.n_kv, 256, 0, st>>>(a, blocks);
  };
  const bool bf16 = dtype == QE_KV_BF16;
  if (fp8 && bf16) go(qe::k_weigh_rows<true, true>, qe::k_weigh_mass<true, true>);
  else if (fp8) go(qe::k_weigh_rows<true, false>, qe::k_weigh_mass<true, false>);
  else if (bf16) go(qe::k_weigh_rows<false, true>, qe::k_weigh_mass<false, true>);
  else go(qe::k_weigh_rows<false, false>, qe::k_weigh_mass<false, false>);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return qe::set_error(QE_ERR_HIP, "page weigh launch failed: %s", hipGetErrorString(e));
  return QE_OK;
}

}  // extern "C"
