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
typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}

// ---- which rows a workgroup takes ----
// V lies transposed in runs of 16 positions, so the rows of one run are written together. The workgroup of
// window x (and a KV head) takes the runs whose first new row is one of the packed rows 16 x .. 16 x + 15: a
// window of a long chunk is one whole run whatever the alignment of the chunk, a window of decode rows is 16
// runs of one row. Those rows are contiguous and at most 31. The heads of a window come one after another:
// their parts of the packed rows lie side by side (head after head over all rows, 143 MB
// took 39.4 us for 35.2, four inputs in turn in a graph).
struct Rows {
  uint32_t window, first, count;  // packed rows
  bool whole;                     // one run, all 16 positions of it
  int64_t slot;  // of lane i < 32: where packed row window + i lies (row index in the pages), -1 no page, -2 no sequence
};

constexpr uint32_t kStartsInLds = 1024;

__device__ __forceinline__ Rows rows_of(const PagePlan& p, uint32_t n_rows, uint32_t window, uint32_t head, int32_t* starts) {
  const uint32_t tid = threadIdx.x, lane = tid & 63, t0 = window * 16, t = t0 + (lane & 31);
  // the search in `starts` is a chain of loads: from LDS where it fits
  const bool in_lds = p.n_seqs < kStartsInLds;
  if (in_lds) {
    for (uint32_t i = tid; i <= p.n_seqs; i += blockDim.x) starts[i] = p.starts[i];
    __syncthreads();
  }
  const int32_t* at = in_lds ? starts : p.starts;
  Rows r;
  r.slot = -2;
  bool begins = true;  // a run (rows of no sequence are one each)
  if (t < n_rows) {
    uint32_t lo = 0, hi = p.n_seqs;
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (at[mid] <= int32_t(t)) lo = mid;
      else hi = mid;
    }
    const int32_t a = at[lo], e = at[lo + 1];
    if (a <= int32_t(t) && int32_t(t) < e) {
      const int64_t pos = int64_t(p.lens[lo]) - (int64_t(e) - t);
      begins = a == int32_t(t) || (pos & (kPageRun - 1)) == 0;
      r.slot = -1;
      if (pos >= 0 && pos < capacity_of(p)) {
        const int32_t page = page_of(p, lo, pos);
        if (page >= 0) r.slot = int64_t(page_row(p, page, head, uint32_t(pos) & ((1u << p.page_shift) - 1)));
      }
    }
  }
  const uint32_t marks = uint32_t(__ballot(begins)) & 0xFFFFFFFFu;
  const uint32_t here = marks & 0xFFFFu, next = marks >> 16;
  // (of 16 consecutive rows one begins a run, so both are there; a plan whose starts decrease may lack it)
  const uint32_t from = here ? __builtin_ctz(here) : 16, to = 16 + (next ? __builtin_ctz(next) : 16);
  r.first = t0 + from;
  r.window = t0;
  r.count = here ? min(to, n_rows > t0 ? n_rows - t0 : 0u) - min(from, n_rows > t0 ? n_rows - t0 : 0u) : 0;
  const int64_t s = __shfl(r.slot, from & 31);
  r.whole = __builtin_popcount(here) == 1 && r.count == 16 && s >= 0 && (s & (kPageRun - 1)) == 0;
  return r;
}
// slot of row i of r.first ..
__device__ __forceinline__ int64_t slot_of(const Rows& r, uint32_t i) {
  return __shfl(r.slot, int(r.first + i - r.window) & 31);
}

// ---- values ----
template <bool BF16>
__device__ __forceinline__ void load8(const uint8_t* row, uint32_t d, float (&x)[8]) {
  if constexpr (BF16) {
    const u32x4_t u = *reinterpret_cast<const u32x4_t*>(row + 2 * d);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      x[2 * i] = __uint_as_float(u[i] << 16);
      x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
  } else {
    const f32x4 u = *reinterpret_cast<const f32x4*>(row + 4 * d), v = *reinterpret_cast<const f32x4*>(row + 4 * d + 16);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      x[i] = u[i];
      x[i + 4] = v[i];
    }
  }
}
template <bool BF16>
__device__ __forceinline__ void store8(uint8_t* row, uint32_t d, const float (&x)[8]) {
  if constexpr (BF16) {
    u32x4_t u;
#pragma unroll
    for (int i = 0; i < 4; i++) u[i] = pack_bf16(x[2 * i], x[2 * i + 1]);
    __builtin_nontemporal_store(u, reinterpret_cast<u32x4_t*>(row + 2 * d));
  } else {
    __builtin_nontemporal_store(f32x4{x[0], x[1], x[2], x[3]}, reinterpret_cast<f32x4*>(row + 4 * d));
    __builtin_nontemporal_store(f32x4{x[4], x[5], x[6], x[7]}, reinterpret_cast<f32x4*>(row + 4 * d + 16));
  }
}

// Maximum over each 16 lanes, to all of them (quad xor 1, quad xor 2, half-row mirror, row mirror).
__device__ __forceinline__ float max16(float v) {
  v = fmaxf(v, dpp<0xB1>(v));
  v = fmaxf(v, dpp<0x4E>(v));
  v = fmaxf(v, dpp<0x141>(v));
  return fmaxf(v, dpp<0x140>(v));
}

// Exponent byte of a row whose largest finite magnitude is amax: 127 (scale 1) for a row of zeros.
__device__ __forceinline__ uint32_t row_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  if (u == 0) return 127;
  const int e = int(u >> 23) - 8 + ((u & 0x7FFFFFu) > 0x600000u);  // mantissa above 1.75: one more
  return uint32_t(max(e, 1));
}

// 8 values of a row held by 16 lanes as e4m3 (o[0], o[1]), and the row's exponent byte.
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], uint32_t (&o)[4]) {
  float a = 0.f;
  bool fine = true;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float y = fabsf(x[i]);
    fine &= y < INFINITY;
    a = fmaxf(a, y < INFINITY ? y : 0.f);
  }
  const uint32_t e = row_exponent(max16(a));
  const float inv = exp_scale(254 - e);
#pragma unroll
  for (int i = 0; i < 2; i++) {
    int u = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i] * inv, x[4 * i + 1] * inv, 0, false);
    u = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2] * inv, x[4 * i + 3] * inv, u, true);
    o[i] = uint32_t(u);
  }
  if (!fine) {  // infinities and NaN become NaN
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (!(fabsf(x[i]) < INFINITY)) o[i / 4] |= 0x7Fu << (8 * (i & 3));
  }
  return e;
}

// A workgroup per (16 packed rows, KV head), see Rows: thread (tid / 16, tid % 16) has a row and 8 dims of it.
// Bound by the rows read and written: 13,900 rows of 8 heads, f32 to e4m3 (143 MB), 33.1 us (4.3 TB/s; a large
// copy 4.9); a row each of 48 sequences 5.0 us, a launch and the chain starts, lens, table, row.
template <bool FP8, bool BF16_ROWS>
__global__ __launch_bounds__(256) void k_page_append(PagePlan p, PageStore st, const uint8_t* k, const uint8_t* v,
                                                     uint32_t n_rows, uint64_t stride) {
  constexpr uint32_t EL = FP8 ? 1 : 2, IN = BF16_ROWS ? 2 : 4;
  __shared__ int32_t starts[kStartsInLds + 1];
  __shared__ __align__(16) uint8_t run[kPageRun * kPageDim * EL];  // V of a run as it lies in the page
  const uint32_t tid = threadIdx.x, window = blockIdx.x / p.n_kv, head = blockIdx.x - window * p.n_kv, d = (tid & 15) * 8;
  const Rows r = rows_of(p, n_rows, window, head, starts);
  for (uint32_t b = 0; b < r.count; b += 16) {
    const uint32_t i = b + tid / 16;
    const int64_t slot = slot_of(r, i);
    const bool real = i < r.count && slot >= 0;
    float x[8] = {}, y[8] = {};
    if (real) {
      const size_t src = (size_t(r.first + i) * stride + head * kPageDim) * IN;
      load8<BF16_ROWS>(k + src, d, x);
      load8<BF16_ROWS>(v + src, d, y);
    }
    uint32_t kq[4], vq[4], ke = 0, ve = 0;
    if constexpr (FP8) {
      ke = quantise8(x, kq);
      ve = quantise8(y, vq);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        kq[e] = pack_bf16(x[2 * e], x[2 * e + 1]);
        vq[e] = pack_bf16(y[2 * e], y[2 * e + 1]);
      }
    }
    auto v_byte_or_half = [&](int e) { return FP8 ? vq[e / 4] >> (8 * (e & 3)) : vq[e / 2] >> (16 * (e & 1)); };
    if (real) {
      uint8_t* o = st.k + (size_t(slot) * kPageDim + d) * EL;
      if constexpr (FP8) *reinterpret_cast<uint2*>(o) = make_uint2(kq[0], kq[1]);
      else *reinterpret_cast<uint4*>(o) = make_uint4(kq[0], kq[1], kq[2], kq[3]);
      if (FP8 && d == 0) {
        st.k_exp[slot] = uint8_t(ke);
        st.v_exp[slot] = uint8_t(ve);
      }
    }
    if (r.whole) {  // (then b is 0 and row i is position i of the run)
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const uint32_t at = (d + e) * kPageRun + i;
        if constexpr (FP8) run[at] = uint8_t(v_byte_or_half(e));
        else reinterpret_cast<uint16_t*>(run)[at] = uint16_t(v_byte_or_half(e));
      }
      __syncthreads();
      const int64_t base = slot_of(r, 0);
      if (tid < sizeof(run) / 16)
        reinterpret_cast<uint4*>(st.v + size_t(base) * kPageDim * EL)[tid] = reinterpret_cast<const uint4*>(run)[tid];
    } else if (real) {
      const size_t at = size_t(slot & ~int64_t(kPageRun - 1)) * kPageDim + (slot & (kPageRun - 1)) + d * kPageRun;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        if constexpr (FP8) st.v[at + e * kPageRun] = uint8_t(v_byte_or_half(e));
        else reinterpret_cast<uint16_t*>(st.v)[at + e * kPageRun] = uint16_t(v_byte_or_half(e));
      }
    }
  }
}

// The same rows the other way; a position without a page reads as zeros. Pages and rows pass by once, with
// non-temporal loads and stores: 18,400 bf16 rows out of bf16 pages (151 MB) 33.7 us (4.5 TB/s);
// four inputs in turn in a graph 38.8 without, so 35.5. (The rows that an append reads lose by it, 35.2 and 37.6 us,
// and the pages it writes are read next.)
template <bool FP8, bool BF16_ROWS>
__global__ __launch_bounds__(256) void k_page_read(PagePlan p, PageStore st, uint8_t* k, uint8_t* v, uint32_t n_rows,
                                                   uint64_t stride) {
  constexpr uint32_t EL = FP8 ? 1 : 2, OUT = BF16_ROWS ? 2 : 4;
  __shared__ int32_t starts[kStartsInLds + 1];
  __shared__ __align__(16) uint8_t run[kPageRun * kPageDim * EL];
  const uint32_t tid = threadIdx.x, window = blockIdx.x / p.n_kv, head = blockIdx.x - window * p.n_kv, d = (tid & 15) * 8;
  const Rows r = rows_of(p, n_rows, window, head, starts);
  for (uint32_t b = 0; b < r.count; b += 16) {
    const uint32_t i = b + tid / 16;
    const int64_t slot = slot_of(r, i);
    uint32_t kq[4] = {}, vq[4] = {};
    float ks = 1.f, vs = 1.f;
    const bool there = i < r.count && slot >= 0;
    if (there) {
      const uint8_t* o = st.k + (size_t(slot) * kPageDim + d) * EL;
      if constexpr (FP8) {
        const uint2 u = *reinterpret_cast<const uint2*>(o);
        kq[0] = u.x;
        kq[1] = u.y;
        ks = exp_scale(st.k_exp[slot]);
        vs = exp_scale(st.v_exp[slot]);
      } else {
        const u32x4_t u = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(o));
        kq[0] = u[0]; kq[1] = u[1]; kq[2] = u[2]; kq[3] = u[3];
      }
    }
    if (r.whole) {
      const int64_t base = slot_of(r, 0);
      if (tid < sizeof(run) / 16)
        reinterpret_cast<u32x4_t*>(run)[tid] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(st.v + size_t(base) * kPageDim * EL) + tid);
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const uint32_t at = (d + e) * kPageRun + i;
        if constexpr (FP8) vq[e / 4] |= uint32_t(run[at]) << (8 * (e & 3));
        else vq[e / 2] |= uint32_t(reinterpret_cast<const uint16_t*>(run)[at]) << (16 * (e & 1));
      }
    } else if (there) {
      const size_t at = size_t(slot & ~int64_t(kPageRun - 1)) * kPageDim + (slot & (kPageRun - 1)) + d * kPageRun;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        if constexpr (FP8) vq[e / 4] |= uint32_t(st.v[at + e * kPageRun]) << (8 * (e & 3));
        else vq[e / 2] |= uint32_t(reinterpret_cast<const uint16_t*>(st.v)[at + e * kPageRun]) << (16 * (e & 1));
      }
    }
    if (i >= r.count || slot == -2) continue;
    auto widen = [&](const uint32_t (&q)[4], float scale, float (&x)[8]) {
      if constexpr (FP8) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(int(q[e]), false), c = __builtin_amdgcn_cvt_pk_f32_fp8(int(q[e]), true);
          x[4 * e] = a[0] * scale;
          x[4 * e + 1] = a[1] * scale;
          x[4 * e + 2] = c[0] * scale;
          x[4 * e + 3] = c[1] * scale;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          x[2 * e] = __uint_as_float(q[e] << 16);
          x[2 * e + 1] = __uint_as_float(q[e] & 0xFFFF0000u);
        }
      }
    };
    float x[8], y[8];
    widen(kq, ks, x);
    widen(vq, vs, y);
    const size_t dst = (size_t(r.first + i) * stride + head * kPageDim) * OUT;
    store8<BF16_ROWS>(k + dst, d, x);
    store8<BF16_ROWS>(v + dst, d, y);
  }
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
  // (a launch has fewer than 2^32 threads, 256 for each 16 rows of a head)
  if (n_rows >= 1ull << 28 || ceil_div(uint32_t(n_rows), 16u) * uint64_t(plan->n_kv) >= 1ull << 24)
    return set_error(QE_ERR_ARG, "need n_rows * n_kv_heads < 2^28, n_rows rounded up to a multiple of 16");
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
  const uint32_t grid = qe::ceil_div(uint32_t(n_rows), 16u) * p.n_kv;
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
  const uint32_t grid = qe::ceil_div(uint32_t(n_rows), 16u) * p.n_kv;
  const bool fp8 = pages->kv_dtype == QE_KV_FP8, bf16 = dtype == QE_KV_BF16;
  auto* kern = fp8 ? (bf16 ? qe::k_page_read<true, true> : qe::k_page_read<true, false>)
                   : (bf16 ? qe::k_page_read<false, true> : qe::k_page_read<false, false>);
  kern<<<grid, 256, 0, static_cast<hipStream_t>(stream)>>>(p, st, static_cast<uint8_t*>(k), static_cast<uint8_t*>(v),
                                                           uint32_t(n_rows), row_stride);
  return qe::launched("page read");
}

}  // extern "C"
