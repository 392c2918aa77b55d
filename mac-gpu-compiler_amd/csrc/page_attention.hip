// qe_op_page_attention: causal GQA attention of packed new tokens over the paged K/V cache. No
// reference counterpart (its attention reads one sequence's contiguous cache, one token at a time:
// cpu_inference.rs:144-162).
//
//   out[t][h] = sum_j w_j v_j / sum_j w_j,  w_j = exp(q[t][h] . k_j / sqrt(128)),  j = 0 .. pos(t),
//
// over the positions j whose page is there; a row that has none gives zeros.
#include "pages.h"

#include "device_common.h"
#include "status.h"

namespace qe {
namespace {

// A wave per (row, q head): lane l holds dims 2 l and 2 l + 1. One position at a time with the
// running maximum and sum of the softmax in f32.
template <bool FP8, bool BF16_ROWS>
__global__ __launch_bounds__(256) void k_page_attention(PagePlan p, PageStore st, const uint8_t* q, uint8_t* out,
                                                        uint32_t n_rows, uint32_t n_heads, uint64_t q_stride,
                                                        uint64_t out_stride, float scale) {
  const uint32_t lane = threadIdx.x & 63;
  const uint64_t unit = uint64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const uint32_t t = uint32_t(unit / n_heads), h = uint32_t(unit % n_heads), head = h / (n_heads / p.n_kv);
  if (t >= n_rows) return;
  const int32_t s = sequence_of(p, int32_t(t));
  if (s < 0) return;
  const int64_t last = position_of(p, s, int32_t(t)), cap = capacity_of(p);
  const int64_t end = last + 1 < cap ? last + 1 : cap;
  float q0, q1;
  if constexpr (BF16_ROWS) {
    const uint32_t u = reinterpret_cast<const uint32_t*>(q + (t * q_stride + h * kPageDim) * 2)[lane];
    q0 = __uint_as_float(u << 16);
    q1 = __uint_as_float(u & 0xFFFF0000u);
  } else {
    const float2 u = reinterpret_cast<const float2*>(q + (t * q_stride + h * kPageDim) * 4)[lane];
    q0 = u.x;
    q1 = u.y;
  }
  float m = -INFINITY, l = 0.f, a0 = 0.f, a1 = 0.f;
  for (int64_t j = 0; j < end; j++) {
    const int32_t page = page_of(p, s, j);
    if (page < 0) continue;
    const uint32_t off = uint32_t(j) & ((1u << p.page_shift) - 1);
    const size_t row = page_row(p, page, head, off), ve = v_element(p, page, head, off);
    float k0, k1, v0, v1;
    if constexpr (FP8) {
      const float ks = exp_scale(st.k_exp[row]), vs = exp_scale(st.v_exp[row]);
      const uint32_t u = reinterpret_cast<const uint16_t*>(st.k + row * kPageDim)[lane];
      const uint32_t w = st.v[ve + 32 * lane] | uint32_t(st.v[ve + 32 * lane + 16]) << 8;
      k0 = __builtin_amdgcn_cvt_f32_fp8(int(u), 0) * ks;
      k1 = __builtin_amdgcn_cvt_f32_fp8(int(u), 1) * ks;
      v0 = __builtin_amdgcn_cvt_f32_fp8(int(w), 0) * vs;
      v1 = __builtin_amdgcn_cvt_f32_fp8(int(w), 1) * vs;
    } else {
      const uint32_t u = reinterpret_cast<const uint32_t*>(st.k + row * kPageDim * 2)[lane];
      const uint16_t* o = reinterpret_cast<const uint16_t*>(st.v) + ve + 32 * lane;
      k0 = __uint_as_float(u << 16);
      k1 = __uint_as_float(u & 0xFFFF0000u);
      v0 = bf16f(o[0]);
      v1 = bf16f(o[16]);
    }
    const float x = wave_sum(fmaf(q0, k0, q1 * k1)) * scale;
    const float mn = fmaxf(m, x);
    const float c = m == -INFINITY ? 0.f : expf(m - mn), w = x == -INFINITY ? 0.f : expf(x - mn);
    l = fmaf(l, c, w);
    a0 = fmaf(a0, c, w * v0);
    a1 = fmaf(a1, c, w * v1);
    m = mn;
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  a0 *= inv;
  a1 *= inv;
  if constexpr (BF16_ROWS) {
    reinterpret_cast<uint32_t*>(out + (t * out_stride + h * kPageDim) * 2)[lane] =
        f32_to_bf16(a0) | uint32_t(f32_to_bf16(a1)) << 16;
  } else {
    reinterpret_cast<float2*>(out + (t * out_stride + h * kPageDim) * 4)[lane] = make_float2(a0, a1);
  }
}

}  // namespace
}  // namespace qe

extern "C" {

uint64_t qe_op_page_attention_work_bytes(uint64_t n_heads, uint64_t n_kv_heads, uint64_t max_new) {
  (void)max_new;
  if (!n_kv_heads || !n_heads || n_heads % n_kv_heads) return 0;
  return 256;
}

int qe_op_page_attention(const qe_pages* pages, const void* q, void* out, uint64_t n_rows, uint64_t n_heads,
                         uint64_t q_stride, uint64_t out_stride, uint64_t max_new, int dtype, void* work,
                         uint64_t work_bytes, void* stream) {
  qe::PagePlan p;
  qe::PageStore st;
  if (int rc = qe::check_pages(pages, &p, &st)) return rc;
  if (dtype != QE_KV_F32 && dtype != QE_KV_BF16) return qe::set_error(QE_ERR_ARG, "rows are QE_KV_F32 or QE_KV_BF16");
  if (n_heads == 0 || n_heads % p.n_kv || n_heads > 65536)
    return qe::set_error(QE_ERR_ARG, "n_heads must be a multiple of n_kv_heads, at most 65536");
  if (n_rows == 0) return QE_OK;
  if (!q || !out || !work) return qe::set_error(QE_ERR_ARG, "null argument");
  if (n_rows > 0x7FFFFFFFull / n_heads) return qe::set_error(QE_ERR_ARG, "need n_rows * n_heads < 2^31");
  const uint64_t el = dtype == QE_KV_F32 ? 4 : 2;
  for (uint64_t stride : {q_stride, out_stride})
    if (stride < n_heads * qe::kPageDim || stride > 0xFFFFFFFFull || stride * el % 16)
      return qe::set_error(QE_ERR_ARG, "row strides must be at least n_heads * 128 elements and multiples of 16 bytes");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(work)) % 16)
    return qe::set_error(QE_ERR_ARG, "q, out and work must be 16-byte aligned");
  if (work_bytes < qe_op_page_attention_work_bytes(n_heads, p.n_kv, max_new))
    return qe::set_error(QE_ERR_ARG, "work holds %llu bytes, fewer than qe_op_page_attention_work_bytes gives",
                         (unsigned long long)work_bytes);
  const uint32_t grid = qe::ceil_div(uint32_t(n_rows) * uint32_t(n_heads), 4u);
  const bool fp8 = pages->kv_dtype == QE_KV_FP8, bf16 = dtype == QE_KV_BF16;
  auto* kern = fp8 ? (bf16 ? qe::k_page_attention<true, true> : qe::k_page_attention<true, false>)
                   : (bf16 ? qe::k_page_attention<false, true> : qe::k_page_attention<false, false>);
  kern<<<grid, 256, 0, static_cast<hipStream_t>(stream)>>>(p, st, static_cast<const uint8_t*>(q),
                                                           static_cast<uint8_t*>(out), uint32_t(n_rows),
                                                           uint32_t(n_heads), q_stride, out_stride,
                                                           1.0f / sqrtf(float(qe::kPageDim)));
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return qe::set_error(QE_ERR_HIP, "page attention launch failed: %s", hipGetErrorString(e));
  return QE_OK;
}

}  // extern "C"
