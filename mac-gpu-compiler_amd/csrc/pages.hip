// The paged K/V cache's own operators: rows of new tokens into pages (qe_op_page_append) and rows
// of pages back out (qe_op_page_read). No reference counterpart (its cache is one buffer per layer).
//
// e4m3 rows carry one power-of-two scale 2^e each, with e the smallest for which the row's largest
// finite magnitude is at most 448 = 1.75 x 2^8 (the largest e4m3 value). A power of two leaves the
// mantissas alone, so x 2^-e is exact and the only rounding is the one to e4m3's 4 significant
// bits (half a step: 2^-4 of the value, 2^-10 x 2^e for the smallest).
#include "pages.h"

#include "device_common.h"
#include "status.h"

namespace qe {
namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// 2 elements from a row of f32 or bf16
template <bool BF16>
__device__ __forceinline__ f32x2 load2(const void* row, uint32_t i) {
  if constexpr (BF16) {
    const uint32_t u = reinterpret_cast<const uint32_t*>(row)[i];
    return f32x2{__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u)};
  } else {
    return reinterpret_cast<const f32x2*>(row)[i];
  }
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}

// |x| where it is finite, else 0
__device__ __forceinline__ float finite_magnitude(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;
}

// Exponent byte of a row whose largest finite magnitude is amax: 127 (scale 1) for a row of zeros.
__device__ __forceinline__ uint32_t row_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  if (u == 0) return 127;
  const int e = int(u >> 23) - 8 + ((u & 0x7FFFFFu) > 0x600000u);  // mantissa above 1.75: one more
  return uint32_t(max(e, 1));
}

// two e4m3 bytes of a and b times inv (a power of two); what is not finite becomes NaN
__device__ __forceinline__ uint32_t pack_fp8(float a, float b, float inv) {
  const float x = a * inv, y = b * inv;
  uint32_t u = uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(x, y, 0, false)) & 0xFFFFu;
  if (!(fabsf(x) <= 448.f)) u = (u & 0xFF00u) | 0x7Fu;
  if (!(fabsf(y) <= 448.f)) u = (u & 0x00FFu) | 0x7F00u;
  return u;
}

// A wave per (row, KV head): lane l holds dims 2 l and 2 l + 1 of K and of V.
template <bool FP8, bool BF16_ROWS>
__global__ __launch_bounds__(256) void k_page_append(PagePlan p, PageStore st, const uint8_t* k, const uint8_t* v,
                                                     uint32_t n_rows, uint64_t stride) {
  const uint32_t lane = threadIdx.x & 63;
  const uint64_t unit = uint64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const uint32_t t = uint32_t(unit / p.n_kv), head = uint32_t(unit % p.n_kv);
  if (t >= n_rows) return;
  const int32_t s = sequence_of(p, int32_t(t));
  if (s < 0) return;
  const int64_t pos = position_of(p, s, int32_t(t));
  if (pos < 0 || pos >= capacity_of(p)) return;
  const int32_t page = page_of(p, s, pos);
  if (page < 0) return;
  const uint32_t off = uint32_t(pos) & ((1u << p.page_shift) - 1);
  const size_t src = (t * stride + head * kPageDim) * (BF16_ROWS ? 2 : 4);
  const f32x2 x = load2<BF16_ROWS>(k + src, lane), y = load2<BF16_ROWS>(v + src, lane);
  const size_t row = page_row(p, page, head, off), ve = v_element(p, page, head, off);
  if constexpr (FP8) {
    const uint32_t kx = row_exponent(wave_max(fmaxf(finite_magnitude(x[0]), finite_magnitude(x[1]))));
    const uint32_t vx = row_exponent(wave_max(fmaxf(finite_magnitude(y[0]), finite_magnitude(y[1]))));
    reinterpret_cast<uint16_t*>(st.k + row * kPageDim)[lane] = uint16_t(pack_fp8(x[0], x[1], exp_scale(254 - kx)));
    const uint32_t u = pack_fp8(y[0], y[1], exp_scale(254 - vx));
    st.v[ve + 32 * lane] = uint8_t(u);
    st.v[ve + 32 * lane + 16] = uint8_t(u >> 8);
    if (lane == 0) {
      st.k_exp[row] = uint8_t(kx);
      st.v_exp[row] = uint8_t(vx);
    }
  } else {
    reinterpret_cast<uint32_t*>(st.k + row * kPageDim * 2)[lane] = pack_bf16(x[0], x[1]);
    const uint32_t u = pack_bf16(y[0], y[1]);
    uint16_t* o = reinterpret_cast<uint16_t*>(st.v) + ve + 32 * lane;
    o[0] = uint16_t(u);
    o[16] = uint16_t(u >> 16);
  }
}

template <bool BF16>
__device__ __forceinline__ void store2(void* row, uint32_t i, float a, float b) {
  if constexpr (BF16) reinterpret_cast<uint32_t*>(row)[i] = pack_bf16(a, b);
  else reinterpret_cast<f32x2*>(row)[i] = f32x2{a, b};
}

// A wave per (row, KV head), the same lanes; a position without a page reads as zeros.
template <bool FP8, bool BF16_ROWS>
__global__ __launch_bounds__(256) void k_page_read(PagePlan p, PageStore st, uint8_t* k, uint8_t* v, uint32_t n_rows,
                                                   uint64_t stride) {
  const uint32_t lane = threadIdx.x & 63;
  const uint64_t unit = uint64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const uint32_t t = uint32_t(unit / p.n_kv), head = uint32_t(unit % p.n_kv);
  if (t >= n_rows) return;
  const int32_t s = sequence_of(p, int32_t(t));
  if (s < 0) return;
  const int64_t pos = position_of(p, s, int32_t(t));
  const int32_t page = pos < 0 || pos >= capacity_of(p) ? -1 : page_of(p, s, pos);
  const size_t dst = (t * stride + head * kPageDim) * (BF16_ROWS ? 2 : 4);
  float a = 0.f, b = 0.f, c = 0.f, d = 0.f;
  if (page >= 0) {
    const uint32_t off = uint32_t(pos) & ((1u << p.page_shift) - 1);
    const size_t row = page_row(p, page, head, off), ve = v_element(p, page, head, off);
    if constexpr (FP8) {
      const float ks = exp_scale(st.k_exp[row]), vs = exp_scale(st.v_exp[row]);
      const uint32_t u = reinterpret_cast<const uint16_t*>(st.k + row * kPageDim)[lane];
      const uint32_t w = st.v[ve + 32 * lane] | uint32_t(st.v[ve + 32 * lane + 16]) << 8;
      a = __builtin_amdgcn_cvt_f32_fp8(int(u), 0) * ks;
      b = __builtin_amdgcn_cvt_f32_fp8(int(u), 1) * ks;
      c = __builtin_amdgcn_cvt_f32_fp8(int(w), 0) * vs;
      d = __builtin_amdgcn_cvt_f32_fp8(int(w), 1) * vs;
    } else {
      const uint32_t u = reinterpret_cast<const uint32_t*>(st.k + row * kPageDim * 2)[lane];
      const uint16_t* o = reinterpret_cast<const uint16_t*>(st.v) + ve + 32 * lane;
      a = __uint_as_float(u << 16);
      b = __uint_as_float(u & 0xFFFF0000u);
      c = bf16f(o[0]);
      d = bf16f(o[16]);
    }
  }
  store2<BF16_ROWS>(k + dst, lane, a, b);
  store2<BF16_ROWS>(v + dst, lane, c, d);
}

}  // namespace

int check_pages(const qe_pages* p, PagePlan* plan, PageStore* store) {
  if (!p) return set_error(QE_ERR_ARG, "null argument");
  if (p->kv_dtype != QE_KV_BF16 && p->kv_dtype != QE_KV_FP8)
    return set_error(QE_ERR_UNSUPPORTED, "pages hold QE_KV_BF16 or QE_KV_FP8");
  if (!p->k || !p->v || !p->table || !p->lens || !p->starts) return set_error(QE_ERR_ARG, "null pointer in qe_pages");
  if (p->kv_dtype == QE_KV_FP8 && (!p->k_exp || !p->v_exp))
    return set_error(QE_ERR_ARG, "QE_KV_FP8 pages need k_exp and v_exp");
  if (p->page_size < kPageRun || p->page_size > 65536 || (p->page_size & (p->page_size - 1)))
    return set_error(QE_ERR_ARG, "page_size must be a power of two from 16 to 65536");
  if (p->n_pages == 0 || p->n_pages > 0x7FFFFFFFull) return set_error(QE_ERR_ARG, "need 0 < n_pages < 2^31");
  if (p->n_kv_heads == 0 || p->n_kv_heads > 1024) return set_error(QE_ERR_ARG, "n_kv_heads must be 1..1024");
  if (p->n_seqs == 0 || p->n_seqs > 65536) return set_error(QE_ERR_ARG, "n_seqs must be 1..65536");
  // positions are held in 32 bits
  if (p->table_stride == 0 || p->table_stride > 0x7FFFFFFFull / p->page_size)
    return set_error(QE_ERR_ARG, "need table_stride > 0 and table_stride * page_size < 2^31");
  if ((reinterpret_cast<uintptr_t>(p->k) | reinterpret_cast<uintptr_t>(p->v)) % 16)
    return set_error(QE_ERR_ARG, "pages must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(p->table) | reinterpret_cast<uintptr_t>(p->lens) |
       reinterpret_cast<uintptr_t>(p->starts)) % 4)
    return set_error(QE_ERR_ARG, "table, lens and starts must be 4-byte aligned");
  if (p->kv_dtype == QE_KV_FP8 &&
      (reinterpret_cast<uintptr_t>(p->k_exp) | reinterpret_cast<uintptr_t>(p->v_exp)) % 16)
    return set_error(QE_ERR_ARG, "k_exp and v_exp must be 16-byte aligned");
  plan->table = p->table;
  plan->lens = p->lens;
  plan->starts = p->starts;
  plan->n_seqs = uint32_t(p->n_seqs);
  plan->n_pages = uint32_t(p->n_pages);
  plan->n_kv = uint32_t(p->n_kv_heads);
  plan->page_shift = uint32_t(__builtin_ctzll(p->page_size));
  plan->table_stride = uint32_t(p->table_stride);
  store->k = static_cast<uint8_t*>(p->k);
  store->v = static_cast<uint8_t*>(p->v);
  store->k_exp = p->k_exp;
  store->v_exp = p->v_exp;
  return QE_OK;
}

namespace {

// the checks of append and read, which take the same arguments
int check_rows(const qe_pages* pages, const void* k, const void* v, uint64_t n_rows, uint64_t stride, int dtype,
               PagePlan* plan, PageStore* store) {
  if (int rc = check_pages(pages, plan, store)) return rc;
  if (dtype != QE_KV_F32 && dtype != QE_KV_BF16) return set_error(QE_ERR_ARG, "rows are QE_KV_F32 or QE_KV_BF16");
  if (n_rows == 0) return QE_OK;
  if (!k || !v) return set_error(QE_ERR_ARG, "null argument");
  const uint64_t el = dtype == QE_KV_F32 ? 4 : 2;
  if (n_rows > 0x7FFFFFFFull / plan->n_kv) return set_error(QE_ERR_ARG, "need n_rows * n_kv_heads < 2^31");
  if (stride < uint64_t(plan->n_kv) * kPageDim || stride > 0xFFFFFFFFull || stride * el % 16)
    return set_error(QE_ERR_ARG, "row_stride must be at least n_kv_heads * 128 elements and a multiple of 16 bytes");
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16)
    return set_error(QE_ERR_ARG, "k and v must be 16-byte aligned");
  return QE_OK;
}

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(QE_ERR_HIP, "%s launch failed: %s", what, hipGetErrorString(e));
  return QE_OK;
}

}  // namespace
}  // namespace qe

extern "C" {

uint64_t qe_page_bytes(uint64_t n_pages, uint64_t page_size, uint64_t n_kv_heads, int kv_dtype) {
  if (kv_dtype != QE_KV_BF16 && kv_dtype != QE_KV_FP8) return 0;
  return n_pages * page_size * n_kv_heads * qe::kPageDim * (kv_dtype == QE_KV_BF16 ? 2 : 1);
}

int qe_op_page_append(const qe_pages* pages, const void* k, const void* v, uint64_t n_rows, uint64_t row_stride,
                      int dtype, void* stream) {
  qe::PagePlan p;
  qe::PageStore st;
  if (int rc = qe::check_rows(pages, k, v, n_rows, row_stride, dtype, &p, &st)) return rc;
  if (n_rows == 0) return QE_OK;
  const uint32_t grid = qe::ceil_div(uint32_t(n_rows) * p.n_kv, 4u);
  const bool fp8 = pages->kv_dtype == QE_KV_FP8, bf16 = dtype == QE_KV_BF16;
  auto* kern = fp8 ? (bf16 ? qe::k_page_append<true, true> : qe::k_page_append<true, false>)
                   : (bf16 ? qe::k_page_append<false, true> : qe::k_page_append<false, false>);
  kern<<<grid, 256, 0, static_cast<hipStream_t>(stream)>>>(p, st, static_cast<const uint8_t*>(k),
                                                           static_cast<const uint8_t*>(v), uint32_t(n_rows), row_stride);
  return qe::launched("page append");
}

int qe_op_page_read(const qe_pages* pages, void* k, void* v, uint64_t n_rows, uint64_t row_stride, int dtype,
                    void* stream) {
  qe::PagePlan p;
  qe::PageStore st;
  if (int rc = qe::check_rows(pages, k, v, n_rows, row_stride, dtype, &p, &st)) return rc;
  if (n_rows == 0) return QE_OK;
  const uint32_t grid = qe::ceil_div(uint32_t(n_rows) * p.n_kv, 4u);
  const bool fp8 = pages->kv_dtype == QE_KV_FP8, bf16 = dtype == QE_KV_BF16;
  auto* kern = fp8 ? (bf16 ? qe::k_page_read<true, true> : qe::k_page_read<true, false>)
                   : (bf16 ? qe::k_page_read<false, true> : qe::k_page_read<false, false>);
  kern<<<grid, 256, 0, static_cast<hipStream_t>(stream)>>>(p, st, static_cast<uint8_t*>(k), static_cast<uint8_t*>(v),
                                                           uint32_t(n_rows), row_stride);
  return qe::launched("page read");
}

}  // extern "C"
